"""pulsar_moe_group_ids against a plain grouping on the host, and a whole layer
of a long chunk: routing with expert groups, the grouping, the expert stages and
dense products with an epilogue."""
import numpy as np
import pytest
import torch

import oracle
from pulsar_amd import kernels as K
from pulsar_amd import runtime, synth
from pulsar_amd.formats import (EPI_NONE, EPI_SILU, QUANT_Q4_K, QUANT_Q6_K, SCORE_SIGMOID, row_bytes)
from tests.gpu_util import assert_rows_close, down, up, up_f32, zeros_f32, zeros_u8

pytestmark = pytest.mark.gpu


def want_groups(ids, experts, n_shared):
    T, k = ids.shape
    lists = [[] for _ in range(experts + n_shared)]
    for t in range(T):
        for s in range(k):
            if 0 <= ids[t, s] < experts:
                lists[ids[t, s]].append(t << 4 | s)
    for i in range(n_shared):
        lists[experts + i] = [t << 4 | k + i for t in range(T)]
    starts = np.cumsum([0] + [len(p) for p in lists]).astype(np.uint32)
    return starts, np.array([p for part in lists for p in part], np.uint32)


BANK = dict(gate=1 << 40, up=2 << 40, down=3 << 40, gate_b=4 << 40, up_b=5 << 40, down_b=6 << 40)


def bank_of(biases):
    b = {n: v for n, v in BANK.items() if biases or not n.endswith("_b")}
    return K.ExpertBank(*[b.get(n) for n in BANK], 1000, 2000, 3000, 100, 200, 300)


def want_ptrs(experts, shared, biases):
    rows = [[BANK["gate"] + 1000 * e, BANK["up"] + 2000 * e, BANK["down"] + 3000 * e]
            + ([BANK["gate_b"] + 400 * e, BANK["up_b"] + 800 * e, BANK["down_b"] + 1200 * e] if biases else [0] * 3)
            for e in range(experts)]
    return np.array(rows + [list(s) + [0] * (6 - len(s)) for s in shared], np.uint64)


def check(dev, ids, experts, n_shared=0, biases=False, weights=True):
    T, k = ids.shape
    slots, groups = k + n_shared, experts + n_shared
    shared = [tuple((7 << 40) + 16 * (8 * i + j) for j in range(6 if i % 2 else 3)) for i in range(n_shared)]
    gptrs = torch.full((groups + 1, 6), -5, dtype=torch.int64, device=dev)
    starts = torch.full((groups + 2,), -5, dtype=torch.int32, device=dev)
    pairs = torch.full((T * slots + 1,), -5, dtype=torch.int32, device=dev)
    sw = torch.full((T * slots + 1,), -5.0, device=dev)
    rw = np.random.default_rng(1).random((T, k)).astype(np.float32)
    K.moe_group_ids(gptrs, starts, pairs, sw if weights else None, torch.from_numpy(ids).to(dev),
                    up_f32(rw) if weights else None, bank_of(biases), experts, shared, T, k)
    want_starts, want_pairs = want_groups(ids, experts, n_shared)
    got, p = down(starts).view(np.uint32), down(pairs).view(np.uint32)
    assert np.array_equal(got[:-1], want_starts)
    n = len(want_pairs)
    assert np.array_equal(p[:n], want_pairs)
    assert (p[n:].view(np.int32) == -5).all() and down(starts)[-1] == -5  # behind the last pair: as it was
    g = down(gptrs)
    assert np.array_equal(g[:-1].view(np.uint64), want_ptrs(experts, shared, biases)) and (g[-1] == -5).all()
    s = down(sw)
    assert s[-1] == -5.0
    if weights:
        want = np.concatenate([rw, np.ones((T, n_shared), np.float32)], 1).reshape(-1)
        assert np.array_equal(s[:-1], want)
    else:
        assert (s == -5.0).all()


@pytest.mark.parametrize("T,k,experts,n_shared", [
    (1, 1, 1, 0), (1, 8, 256, 1), (3, 2, 5, 2), (31, 2, 6, 1), (32, 8, 64, 0), (64, 4, 32, 0), (257, 1, 7, 4),
    (301, 8, 256, 1), (1000, 16, 1024, 0), (1621, 10, 13, 2), (4096, 8, 128, 0), (2500, 12, 300, 4),
    (2049, 15, 512, 1)])
def test_shapes(dev, T, k, experts, n_shared):
    rng = np.random.default_rng(T)
    ids = np.stack([rng.permutation(max(experts, k))[:k] % experts for _ in range(T)]).astype(np.int32)
    check(dev, ids, experts, n_shared)
    # ids of no expert, the same expert twice in a token
    ids[rng.random(ids.shape) < 0.2] = -1
    ids[rng.random(ids.shape) < 0.05] = experts
    ids[rng.random(ids.shape) < 0.05] = np.iinfo(np.int32).min
    ids[rng.random(ids.shape) < 0.3] = experts // 2
    check(dev, ids, experts, n_shared, biases=True, weights=T % 2 == 0)


def test_no_pair_at_all(dev):
    check(dev, np.full((300, 8), -1, np.int32), 64, 1)
    check(dev, np.full((300, 8), 64, np.int32), 64, 0)


def test_one_expert_takes_all(dev):
    check(dev, np.full((5000, 4), 3, np.int32), 8, 0)


def want_long(ids, experts, n_shared):
    """want_groups for long chunks, by numpy's stable sort."""
    T, k = ids.shape
    flat = ids.reshape(-1)
    order = np.argsort(flat, kind="stable")
    order = order[(flat[order] >= 0) & (flat[order] < experts)]
    starts = np.searchsorted(flat[order], np.arange(experts + 1))
    token = np.arange(T)
    pairs = np.concatenate([(order // k) << 4 | order % k] + [token << 4 | k + i for i in range(n_shared)])
    return np.concatenate([starts, starts[-1] + T * np.arange(1, n_shared + 1)]), pairs


@pytest.mark.parametrize("T,k,experts,n_shared,kind", [
    (30001, 3, 96, 0, "even"), (80001, 6, 96, 1, "even"), (80001, 7, 96, 0, "even"), (65536, 8, 96, 0, "even"),
    (65537, 8, 96, 0, "none"), (131072, 8, 96, 0, "even"), (16384, 8, 256, 0, "even"), (16383, 12, 1024, 4, "even"),
    (9000, 8, 1, 2, "one"), (70000, 1, 1000, 3, "one"), (20000, 8, 8, 1, "skewed"), (5462, 12, 33, 1, "skewed"),
    (5461, 12, 512, 0, "even"), (4096, 16, 300, 0, "skewed"), (4097, 16, 300, 0, "skewed"), (66000, 1, 2, 0, "last")])
def test_long_chunks(dev, T, k, experts, n_shared, kind):
    """Chunks on both sides of the length from which the grouping takes two
    launches, up to a million ids: even, uneven, one expert's, none's."""
    rng = np.random.default_rng(T)
    ids = rng.integers(-1, experts + 1, (T, k)).astype(np.int32)
    if kind == "one":
        ids[:] = experts - 1
    elif kind == "none":
        ids[:] = -1
    elif kind == "skewed":
        ids[rng.random((T, k)) < 0.9] = experts // 3
    elif kind == "last":
        ids[:-1] = experts
    groups = experts + n_shared
    shared = [tuple((7 << 40) + 16 * (3 * i + j) for j in range(3)) for i in range(n_shared)]
    want_starts, want_pairs = want_long(ids, experts, n_shared)
    rw = rng.random((T, k)).astype(np.float32)
    for _ in range(2):
        gptrs = torch.full((groups + 1, 6), -5, dtype=torch.int64, device=dev)
        starts = torch.full((groups + 2,), -5, dtype=torch.int32, device=dev)
        pairs = torch.full((T * (k + n_shared) + 1,), -5, dtype=torch.int32, device=dev)
        sw = torch.full((T * (k + n_shared) + 1,), -5.0, device=dev)
        K.moe_group_ids(gptrs, starts, pairs, sw, torch.from_numpy(ids).to(dev), up_f32(rw), bank_of(False), experts,
                        shared, T, k)
        n, p = len(want_pairs), down(pairs)
        assert np.array_equal(down(starts)[:-1], want_starts) and down(starts)[-1] == -5
        assert np.array_equal(p[:n], want_pairs) and (p[n:] == -5).all()
        assert np.array_equal(down(gptrs)[:-1].view(np.uint64), want_ptrs(experts, shared, False))
        assert (down(gptrs)[-1] == -5).all()
        want = np.concatenate([rw, np.ones((T, n_shared), np.float32)], 1).reshape(-1)
        assert np.array_equal(down(sw)[:-1], want) and down(sw)[-1] == -5.0


def test_matches_group_csr(dev):
    """Where both take the chunk: the same pairs per expert as moe_group_csr."""
    T, k, E = 100, 8, 32
    ids = np.stack([np.random.default_rng(t).permutation(E)[:k] for t in range(T)]).astype(np.int32)
    bank, sel = bank_of(False), torch.from_numpy(ids).to(dev)
    rw = up_f32(np.ones((T, k), np.float32))
    ptrs, sw = zeros_u8(T * k * 48), zeros_f32((T, k))
    K.moe_route_ptrs(ptrs, sw, sel, rw, bank, E, [], T, k)
    out = []
    for call in (lambda g, s, p: K.moe_group_csr(g, s, p, ptrs, T, k, E),
                 lambda g, s, p: K.moe_group_ids(g, s, p, None, sel, None, bank, E, [], T, k)):
        g = torch.zeros((E, 6), dtype=torch.int64, device=dev)
        s, p = torch.zeros(E + 1, dtype=torch.int32, device=dev), torch.zeros(T * k, dtype=torch.int32, device=dev)
        call(g, s, p)
        g, s, p = down(g), down(s), down(p)
        out.append({tuple(g[e]): p[s[e]:s[e + 1]].tolist() for e in range(E)})
    assert out[0] == out[1]


@pytest.mark.parametrize("T", [700, 20000])
def test_captured(dev, T):
    k, E = 4, 40
    rng = np.random.default_rng(9)
    sel = torch.zeros((T, k), dtype=torch.int32, device=dev)
    g = torch.zeros((E + 1, 6), dtype=torch.int64, device=dev)
    s, p = torch.zeros(E + 2, dtype=torch.int32, device=dev), torch.zeros(T * 5, dtype=torch.int32, device=dev)
    shared = [(16, 32, 48)]
    torch.cuda.synchronize()
    graph = runtime.Graph.capture(lambda: K.moe_group_ids(g, s, p, None, sel, None, bank_of(True), E, shared, T, k))
    for _ in range(3):
        ids = rng.integers(0, E, (T, k)).astype(np.int32)
        sel.copy_(torch.from_numpy(ids))
        torch.cuda.synchronize()
        graph.launch()
        runtime.sync()
        starts, pairs = want_long(ids, E, 1)
        assert np.array_equal(down(s), starts) and np.array_equal(down(p), pairs)


@pytest.mark.parametrize("T", [700, 20000])
def test_own_stream(dev, T):
    k, E = 4, 40
    ids = np.random.default_rng(10).integers(0, E, (T, k)).astype(np.int32)
    sel = torch.from_numpy(ids).to(dev)
    g = torch.zeros((E, 6), dtype=torch.int64, device=dev)
    s, p = torch.zeros(E + 1, dtype=torch.int32, device=dev), torch.zeros(T * k, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    K.set_stream(stream)
    try:
        K.moe_group_ids(g, s, p, None, sel, None, bank_of(False), E, None, T, k)
    finally:
        K.set_stream(None)
    stream.synchronize()
    starts, pairs = want_long(ids, E, 0)
    assert np.array_equal(down(s), starts) and np.array_equal(down(p), pairs)


def test_wrapper_refuses_short_tensors(dev):
    z = torch.zeros(4096, dtype=torch.int32, device=dev)
    good = dict(gptrs=z, starts=z, pairs=z, slot_weights=z, selected=z, router_weights=z)
    for name, n in (("gptrs", 33 * 12 - 1), ("starts", 33), ("pairs", 10 * 9 - 1), ("slot_weights", 10 * 9 - 1),
                    ("selected", 79), ("router_weights", 79)):
        with pytest.raises(ValueError, match=f"{name} has to be contiguous"):
            K.moe_group_ids(bank=bank_of(False), n_expert=32, shared=[(16, 32, 48)], n_tok=10, k_used=8,
                            **{**good, name: z[:n]})


@pytest.mark.parametrize("T", [300, 1])
def test_layer_of_a_long_chunk(dev, T):
    """Routing, grouping, the expert stages, then a dense branch whose last
    product adds the experts' output as its residual, in place. Every stage
    against the oracle on the inputs the GPU's own stages gave it."""
    hidden, ffn, E, k, G, kept, scale = 512, 256, 16, 4, 4, 2, 2.5
    rng = np.random.default_rng(T)
    gq, dq = QUANT_Q4_K, QUANT_Q6_K
    grb, drb = row_bytes(gq, hidden), row_bytes(dq, ffn)
    gate, upw = (synth.quant_matrix(gq, E * ffn, hidden, rng).reshape(E, ffn, grb) for _ in range(2))
    dn = synth.quant_matrix(dq, E * hidden, ffn, rng).reshape(E, hidden, drb)
    w1, w2 = synth.quant_matrix(gq, ffn, hidden, rng), synth.quant_matrix(dq, hidden, ffn, rng)
    b1 = rng.standard_normal(ffn).astype(np.float32)
    x = rng.standard_normal((T, hidden)).astype(np.float32)
    logits = rng.standard_normal((T, E)).astype(np.float32)
    rbias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    dg, du, dd, d1, d2 = up(gate), up(upw), up(dn), up(w1), up(w2)
    bank = K.ExpertBank(dg.data_ptr(), du.data_ptr(), dd.data_ptr(), None, None, None, ffn * grb, ffn * grb,
                        hidden * drb, 0, 0, 0)
    ids, rw = torch.zeros((T, k), dtype=torch.int32, device=dev), zeros_f32((T, k))
    K.router_select_groups(ids, rw, up_f32(logits), up_f32(rbias), E, k, G, kept, 2, SCORE_SIGMOID, True, scale, T)
    gptrs, starts = zeros_u8(E * 48), torch.zeros(E + 1, dtype=torch.int32, device=dev)
    pairs = torch.zeros(T * k, dtype=torch.int32, device=dev)
    K.moe_group_ids(gptrs, starts, pairs, None, ids, None, bank, E, [], T, k)
    xq, midq, hq = zeros_u8(T * 2 * 292), zeros_u8(T * k * 292), zeros_u8(T * 292)
    mid, part, out, h = zeros_f32((T * k, ffn)), zeros_f32((T * k, hidden)), zeros_f32((T, hidden)), zeros_f32((T, ffn))
    K.quantize_q8_k(xq, up_f32(x), hidden, T)
    K.moe_pair_swiglu_grouped(mid, gptrs, starts, pairs, rw, xq, hidden, ffn, k, E, grb, gq, 0)
    K.quantize_q8_k(midq, mid, ffn, T * k)
    K.moe_down_grouped(part, gptrs, starts, pairs, midq, ffn, hidden, k, E, drb, dq)
    K.moe_slot_sum(out, part, hidden, k, T)
    moe = down(out).copy()
    K.matmul_kq_fused(h, d1, xq, up_f32(b1), None, hidden, ffn, T, grb, gq, EPI_SILU)
    K.quantize_q8_k(hq, h, ffn, T)
    K.matmul_kq_fused(out, d2, hq, None, out, ffn, hidden, T, drb, dq, EPI_NONE)

    sel, wts = down(ids), down(rw)
    assert (sel >= 0).all() and np.allclose(wts.sum(1), scale, rtol=1e-6)
    hx, hm, hh = (down(t).reshape(-1) for t in (xq, midq, hq))
    hx, hm, hh = hx.reshape(T, -1), hm.reshape(T, k, -1), hh.reshape(T, -1)
    ptrs = oracle.host_ptrs([(gate[e], upw[e], dn[e]) for e in sel.reshape(-1)])
    want_mid = oracle.moe_pair_swiglu(ptrs, wts, hx, hidden, ffn, k, T, grb, gq, 0)
    assert np.allclose(down(mid).reshape(want_mid.shape), want_mid, rtol=1e-4, atol=1e-4 * np.abs(want_mid).max())
    want = oracle.moe_down(ptrs, hm.reshape(T * k, -1), ffn, hidden, k, T, drb, dq)
    assert np.allclose(moe, want, rtol=1e-4, atol=1e-5 * np.abs(want).max())
    v, _ = oracle.rows_dot(w1, grb, ffn, hx, hidden, T, gq, 8)
    v = v.reshape(T, ffn).astype(np.float64) + b1
    want_h = v / (1 + np.exp(-v))
    assert np.allclose(down(h), want_h, rtol=1e-4, atol=1e-5 * np.abs(want_h).max())
    v, sc = oracle.rows_dot(w2, drb, hidden, hh, ffn, T, dq, 8)
    assert_rows_close(down(out), v.reshape(T, hidden).astype(np.float64) + moe,
                      sc.reshape(T, hidden) + np.abs(moe), "product with residual")
