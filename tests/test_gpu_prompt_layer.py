"""A layer of a prompt chunk of more pairs than pulsar_moe_group_csr takes, as it
is documented: pulsar_router_logits_q8, pulsar_router_select_groups,
pulsar_moe_group_ids, the grouped expert stages with a bound of their pairs, the
slot sum. Every stage against the oracle or 64 bits on the inputs that the GPU's
own stages gave it, for a sample of the tokens."""
import numpy as np
import pytest
import torch

import oracle
from pulsar_amd import formats as fm
from pulsar_amd import kernels as K
from pulsar_amd import synth
from pulsar_amd.formats import QUANT_Q4_K, QUANT_Q6_K, SCORE_SIGMOID, SCORE_SOFTMAX, row_bytes
from tests.gpu_util import assert_rows_close, down, up, up_f32, zeros_f32, zeros_u8
from tests.test_gpu_group_ids import want_long
from tests.test_gpu_grouped_choice import ROW16
from tests.test_gpu_router_groups import want_route
from tests.test_gpu_tile import rows_want

pytestmark = pytest.mark.gpu
GQ, DQ = QUANT_Q4_K, QUANT_Q6_K


# tokens, experts, winners, groups, kept groups, shared slots, whether the bias
# leaves fewer candidates than winners: the grouping in two launches; in one, with
# empty slots; in two, with more groups than the wide tile takes
@pytest.mark.parametrize("T,E,k,G,kept,n_shared,empty,score", [
    (8300, 64, 8, 8, 4, 1, False, SCORE_SIGMOID), (700, 48, 6, 8, 1, 2, True, SCORE_SOFTMAX),
    (3300, 1024, 8, 1, 1, 1, False, SCORE_SOFTMAX), (9000, 16, 8, 4, 4, 0, False, SCORE_SOFTMAX)])
def test_layer(dev, T, E, k, G, kept, n_shared, empty, score):
    hidden, ffn, scale, slots = 512, 256, 1.5, k + n_shared
    rng = np.random.default_rng(T)
    grb, drb = row_bytes(GQ, hidden), row_bytes(DQ, ffn)
    kinds = min(E + n_shared, 61)  # matrices of their own, dealt out in turn
    of = np.arange(E + n_shared) % kinds
    gate, upw = (synth.quant_matrix(GQ, kinds * ffn, hidden, rng).reshape(kinds, ffn, grb) for _ in range(2))
    dn = synth.quant_matrix(DQ, kinds * hidden, ffn, rng).reshape(kinds, hidden, drb)
    dg, du, dd = (up(m[of]) for m in (gate, upw, dn))
    gs, ds = ffn * grb, hidden * drb
    bank = K.ExpertBank(dg.data_ptr(), du.data_ptr(), dd.data_ptr(), None, None, None, gs, gs, ds, 0, 0, 0)
    shared = [(dg.data_ptr() + e * gs, du.data_ptr() + e * gs, dd.data_ptr() + e * ds) for e in range(E, E + n_shared)]
    wr = (rng.standard_normal((E, hidden)) / np.sqrt(hidden)).astype(np.float32)
    x = rng.standard_normal((T, hidden)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    if empty:
        bias[::E // G] = -np.inf  # one of the experts of every group: 5 are left for 6 winners

    n, groups = T * slots, E + n_shared
    logits, xq = zeros_f32((T, E)), zeros_u8(T * 2 * 292)
    ids, rw = torch.full((T, k), -7, dtype=torch.int32, device=dev), zeros_f32((T, k))
    gptrs, starts = zeros_u8(groups * 48), torch.zeros(groups + 1, dtype=torch.int32, device=dev)
    pairs, sw = torch.zeros(n, dtype=torch.int32, device=dev), zeros_f32((T, slots))
    mid, midq, part, out = zeros_f32((n, ffn)), zeros_u8(n * 292), zeros_f32((n, hidden)), zeros_f32((T, hidden))
    K.router_logits_q8(logits, xq, up_f32(x), up_f32(wr), None, hidden, E, T)
    K.router_select_groups(ids, rw, logits, up_f32(bias), E, k, G, kept, 2, score, True, scale, T)
    K.moe_group_ids(gptrs, starts, pairs, sw, ids, rw, bank, E, shared, T, k)
    K.moe_pair_swiglu_grouped(mid, gptrs, starts, pairs, sw, xq, hidden, ffn, slots, groups, grb, GQ, 0)
    K.quantize_q8_k(midq, mid, ffn, n)
    K.moe_down_grouped(part, gptrs, starts, pairs, midq, ffn, hidden, slots, groups, drb, DQ)
    K.moe_slot_sum(out, part, hidden, slots, T)

    sel, wts, sums = down(ids), down(sw), down(out)
    at = np.unique(np.concatenate([[0, 1, T // 2, T - 2, T - 1], rng.integers(0, T, 24)]))
    pick = torch.from_numpy(at).to(dev)
    hl, hx = down(logits[pick]), down(xq.view(T, -1)[pick])
    hmid, hmq, hpart = (down(t.view(T, slots, -1)[pick]) for t in (mid, midq, part))
    # the router's logits: sum of products in another order
    bound = np.abs(x[at]).astype(np.float64) @ np.abs(wr).astype(np.float64).T
    assert_rows_close(hl, x[at].astype(np.float64) @ wr.T.astype(np.float64), bound, "logits")
    assert np.array_equal(hx, oracle.quantize_q8_k(x[at]))
    want, w, tol = want_route(hl, bias, k, G, kept, 2, score, True, scale)
    assert np.array_equal(sel[at], want) and (np.abs(wts[at, :k] - w) <= tol).all()
    assert (wts[:, k:] == 1.0).all() and ((sel == -1).any(1) == empty).all()
    want_starts, want_pairs = want_long(sel, E, n_shared)
    assert np.array_equal(down(starts), want_starts)
    assert np.array_equal(down(pairs)[:len(want_pairs)], want_pairs)
    for i, t in enumerate(at):
        for s in range(slots):
            e = sel[t, s] if s < k else E + s - k
            if e < 0:
                assert not hmid[i, s].any() and not hpart[i, s].any()
                continue
            m, (g, _, bg), (u, _, bu) = of[e], *(rows_want(GQ, a[of[e]], grb, hx[i:i + 1], hidden, 1) for a in (gate, upw))
            g, u, bg, bu = (v.reshape(-1).astype(np.float64) for v in (g, u, 1e-5 * bg, 1e-5 * bu))
            silu, wt = g / (1 + np.exp(-g)), float(wts[t, s])
            # |silu'| <= 1.1; the device's exp, division and two products: 1e-6
            bound = wt * (1.1 * bg * (np.abs(u) + bu) + np.abs(silu) * bu + 1e-6 * np.abs(silu * u)) + 1e-30
            assert (np.abs(hmid[i, s] - silu * u * wt) <= bound).all(), ("mid", t, s, e)
            v, _, bound = rows_want(DQ, dn[m], drb, hmq[i, s:s + 1], ffn, 1)
            assert_rows_close(hpart[i, s], v.reshape(-1), bound.reshape(-1), f"down {t} {s} {e}")
    total, size = hpart.astype(np.float64).sum(1), np.abs(hpart.astype(np.float64)).sum(1)
    assert (np.abs(sums[at] - total) <= slots * 2.0**-24 * size).all()  # a rounding an addition


@pytest.mark.parametrize("quant", ROW16, ids=lambda q: fm.NAMES[q])
def test_stages_in_slices_of_the_groups(dev, quant):
    """1024 experts and two shared slots, the grouped stages called on 1024 groups
    and on the two behind them, whose starts go on where the others' end: the rows
    of one call on all, bit for bit where both calls' kernels sum alike."""
    T, E, k, n_shared, hidden, ffn = 3300, 1024, 4, 2, 512, 256
    rng = np.random.default_rng(5)
    slots, groups, n = k + n_shared, E + n_shared, T * (k + n_shared)
    rbs, kinds = (row_bytes(quant, hidden), row_bytes(quant, ffn)), 23
    of = np.arange(groups) % kinds
    dg, du = (up(synth.quant_matrix(quant, kinds * ffn, hidden, rng).reshape(kinds, -1)[of]) for _ in range(2))
    dd = up(synth.quant_matrix(quant, kinds * hidden, ffn, rng).reshape(kinds, -1)[of])
    gs, ds = ffn * rbs[0], hidden * rbs[1]
    bank = K.ExpertBank(dg.data_ptr(), du.data_ptr(), dd.data_ptr(), None, None, None, gs, gs, ds, 0, 0, 0)
    shared = [(dg.data_ptr() + e * gs, du.data_ptr() + e * gs, dd.data_ptr() + e * ds) for e in range(E, groups)]
    ids = torch.from_numpy(rng.integers(0, E, (T, k)).astype(np.int32)).to(dev)
    gptrs, starts = zeros_u8(groups * 48), torch.zeros(groups + 1, dtype=torch.int32, device=dev)
    pairs, sw, xq = torch.zeros(n, dtype=torch.int32, device=dev), zeros_f32((T, slots)), zeros_u8(T * 2 * 292)
    K.moe_group_ids(gptrs, starts, pairs, sw, ids, up_f32(rng.random((T, k)) + 0.1), bank, E, shared, T, k)
    K.quantize_q8_k(xq, up_f32(rng.standard_normal((T, hidden))), hidden, T)
    midq = up(oracle.quantize_q8_k(rng.standard_normal((n, ffn)).astype(np.float32)))
    got = []
    for slices in ([(0, groups)], [(0, 1024), (1024, groups)]):
        mid, part = zeros_f32((n, ffn)), zeros_f32((n, hidden))
        for a, b in slices:
            K.moe_pair_swiglu_grouped(mid, gptrs[48 * a:], starts[a:], pairs, sw, xq, hidden, ffn, slots, b - a, rbs[0],
                                      quant, 0)
            K.moe_down_grouped(part, gptrs[48 * a:], starts[a:], pairs, midq, ffn, hidden, slots, b - a, rbs[1], quant)
        got.append((down(mid), down(part)))
    for one, two in zip(*got):
        assert one.any(1).all() and np.array_equal(one.view(np.uint32), two.view(np.uint32))
