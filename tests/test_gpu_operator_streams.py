"""The routing with expert groups, the grouping by ids and the fused product in
the order of the stream that pulsar_set_stream chose: their inputs are stale until
work queued ahead on that stream has ended, and their outputs are copied by work
queued behind. A launch on any other stream would read the stale inputs."""
import numpy as np
import pytest
import torch

from pulsar_amd import formats as fm
from pulsar_amd import kernels as K
from pulsar_amd.formats import EPI_SILU, SCORE_SIGMOID
from tests.gpu_util import zeros_f32
from tests.test_gpu_group_ids import bank_of, want_long
from tests.test_gpu_product_fused import Case, assert_epilogue
from tests.test_gpu_router_groups import want_route

pytestmark = pytest.mark.gpu


def in_order(dev, call, fresh, outs):
    """Copies of outs, made on a stream of its own behind: some ms of work, the
    copies of `fresh` ((buffer, values) pairs), call()."""
    a = torch.full((4096, 4096), 1.0 / 4096, device=dev)
    b, staged = torch.empty_like(a), [(to, torch.from_numpy(np.ascontiguousarray(v)).to(dev)) for to, v in fresh]
    kept = [torch.empty_like(o) for o in outs]
    torch.mm(a, a, out=b)  # the library's own start
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ahead = torch.cuda.Event()
    with torch.cuda.stream(stream):
        for _ in range(40):
            torch.mm(a, a, out=b)
        for to, v in staged:
            to.copy_(v)
        ahead.record()
        K.set_stream(stream)
        try:
            early = not ahead.query()
            call()
        finally:
            K.set_stream(None)
        for k, o in zip(kept, outs):
            k.copy_(o)
    stream.synchronize()
    assert early, "the work ahead had ended before the call: nothing was checked"
    return [k.cpu().numpy() for k in kept]


@pytest.mark.parametrize("experts,groups", [(256, 8), (320, 20)])
def test_routing(dev, experts, groups):
    rng = np.random.default_rng(experts)
    T, k = 600, 6
    logits = rng.standard_normal((T, experts)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    x, b = zeros_f32((T, experts)), zeros_f32(experts)
    ids, w = torch.full((T, k), -7, dtype=torch.int32, device=dev), zeros_f32((T, k))
    how = (k, groups, 3, 2, SCORE_SIGMOID, True, 1.0)
    got, gw = in_order(dev, lambda: K.router_select_groups(ids, w, x, b, experts, *how, T), [(x, logits), (b, bias)],
                       [ids, w])
    want, ww, tol = want_route(logits, bias, *how)
    assert np.array_equal(got, want) and (np.abs(gw - ww) <= tol).all()


@pytest.mark.parametrize("T", [700, 20000])  # one launch, two
def test_grouping(dev, T):
    k, E = 4, 40
    rng = np.random.default_rng(T)
    real, rw = rng.integers(0, E, (T, k)).astype(np.int32), rng.random((T, k)).astype(np.float32)
    ids, w, sw = torch.zeros((T, k), dtype=torch.int32, device=dev), zeros_f32((T, k)), zeros_f32((T, k + 1))
    g, s = torch.zeros((E + 1, 6), dtype=torch.int64, device=dev), torch.zeros(E + 2, dtype=torch.int32, device=dev)
    p = torch.zeros(T * (k + 1), dtype=torch.int32, device=dev)
    gs, gp, gw = in_order(dev, lambda: K.moe_group_ids(g, s, p, sw, ids, w, bank_of(True), E, [(16, 32, 48)], T, k),
                          [(ids, real), (w, rw)], [s, p, sw])
    starts, pairs = want_long(real, E, 1)
    assert np.array_equal(gs, starts) and np.array_equal(gp, pairs)
    assert np.array_equal(gw, np.concatenate([rw, np.ones((T, 1), np.float32)], 1))


@pytest.mark.parametrize("quant,rows,n,T", [
    (fm.QUANT_Q4_K, 300, 512, 1), (fm.QUANT_Q6_K, 301, 512, 4), (fm.QUANT_Q5_K, 500, 768, 40),
    (fm.QUANT_Q4_K, 16500, 768, 12), (fm.QUANT_Q4_K, 4130, 256, 500)])  # lane kernels, K split, 16-row kernel, tile
def test_product(dev, quant, rows, n, T):
    c = Case(quant, rows, n, T)
    bias, res, out = zeros_f32(rows), zeros_f32((T, rows)), zeros_f32((T, rows))
    real = c.x.reshape(T, -1)
    c.dx = torch.zeros(real.size, dtype=torch.uint8, device=dev)
    got, = in_order(dev, lambda: c.run(out, bias, res, EPI_SILU),
                    [(bias, c.bias), (res, c.res), (c.dx, real.view(np.uint8).reshape(-1))], [out])
    assert_epilogue(got, c.dots, c.bias, EPI_SILU, c.res, quant)
