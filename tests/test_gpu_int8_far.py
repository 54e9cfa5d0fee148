"""The norm to 8-bit rows, the int8 quantizer and the int8 product past 32-bit offsets, on
a stream of their caller's, two at once on two streams, and at the largest counts."""
import numpy as np
import pytest
import torch

from pulsar_amd import kernels as K
from pulsar_amd.formats import ACT_SILU, EPI_NONE, EPI_SILU, ROWS_I8, ROWS_Q8_K, TYPE_BF16, TYPE_F32
from tests.gpu_util import down, up_f32, zeros_f32
from tests.test_gpu_operator_streams import in_order
from tests.test_gpu_product_i8 import Case, i8, out_of
from tests.test_gpu_rows8 import NAMES, TORCH, Norm, dev_rows, glu64, host, quant_check, rounded

pytestmark = pytest.mark.gpu


def far_rows(rows, dim, stride, dtype):
    """[rows, dim] views of an array whose last row starts past 4 GiB."""
    t = torch.empty((rows - 1) * stride + dim, dtype=dtype, device="cuda:0")
    return t.as_strided((rows, dim), (stride, 1))


@pytest.mark.parametrize("kind", [TYPE_F32, TYPE_BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim", [1000, 16500])
def test_norm_rows_far_apart(dev, dim, kind):
    rows, stride = 70, (2**32 // 60) // (4 if kind == TYPE_F32 else 2)
    n = Norm(rows, dim, kind)
    x, r, s = (far_rows(rows, dim, stride, TORCH[kind]) for _ in range(3))
    q = far_rows(rows, dim, 2**26, torch.int8)
    x.copy_(dev_rows(n.x, kind)), r.copy_(dev_rows(n.r, kind))
    sc, y = up_f32(np.zeros(rows)), torch.zeros((rows, dim), dtype=TORCH[kind], device=dev)
    n.call((q, sc, y, s, x, r, up_f32(n.g)), ROWS_I8, x_stride=stride, res_stride=stride, sum_stride=stride,
           q_stride=2**26)
    n.check(s.contiguous(), y, q.contiguous(), sc, ROWS_I8)


def test_norm_blocks_past_4_gib(dev):
    """15 million rows of 256 values in q8_K."""
    rows = 2**32 // 292 + 9
    x = torch.zeros((rows, 256), dtype=torch.bfloat16, device=dev)
    q = torch.empty(rows * 292, dtype=torch.uint8, device=dev)
    at = [0, 1, rows // 2, rows - 9, rows - 2, rows - 1]
    n = Norm(len(at), 256, TYPE_BF16, residual=False)
    x[at] = dev_rows(n.x, TYPE_BF16)
    K.rms_norm_q8(q, None, None, None, x, None, up_f32(n.g), 256, rows, n.eps, TYPE_BF16, ROWS_Q8_K)
    n.check(None, None, q.view(rows, 292)[at].reshape(-1), None, ROWS_Q8_K)


@pytest.mark.parametrize("dim,op", [(900, ACT_SILU), (900, None), (17000, ACT_SILU)])
def test_quantize_rows_far_apart(dev, dim, op):
    rows, stride = 70, 2**30 // 15
    rng = np.random.default_rng(dim)
    hx, hu = (rounded(rng.standard_normal((rows, dim)), TYPE_F32) for _ in range(2))
    x, u, q = far_rows(rows, dim, stride, torch.float32), far_rows(rows, dim, stride, torch.float32), far_rows(
        rows, dim, 2**26, torch.int8)
    x.copy_(dev_rows(hx, TYPE_F32)), u.copy_(dev_rows(hu, TYPE_F32))
    sc = up_f32(np.zeros(rows))
    K.quantize_i8(q, sc, x, None if op is None else u, dim, rows, op or 0, TYPE_F32, stride, stride, 2**26)
    quant_check(hx if op is None else glu64(hx, hu, op), q.contiguous(), sc, dim)


# rows, columns, tokens: lane kernel, tiles with and without whole 16-byte pieces
@pytest.mark.parametrize("rows,cols,T", [(600, 512, 2), (600, 1024, 20), (600, 1000, 20), (520, 512, 520), (520, 500, 520),
                                         (600, 256, 5000)])
def test_product_rows_far_apart(dev, rows, cols, T):
    """Rows of x and w 2^23 bytes apart, the most there may be, rows of out and residual
    past 4 GiB."""
    c = Case(rows, cols, T)
    ws = xs = 2**23
    if T > 1000:
        xs = cols
    x, w = far_rows(T, cols, xs, torch.int8), far_rows(rows, cols, ws, torch.int8)
    x.copy_(i8(c.x)), w.copy_(i8(c.w))
    so = max(rows, 2**30 // max(T - 5, 1) + 7)
    out, res = far_rows(T, rows, so, torch.float32), far_rows(T, rows, so, torch.float32)
    res.copy_(dev_rows(c.res, TYPE_F32))
    K.matmul_i8(out, w, up_f32(c.sw), x, up_f32(c.sx), up_f32(c.bias), res, cols, rows, T, EPI_SILU, TYPE_F32, ws, xs, so, so)
    c.check(host(out), True, EPI_SILU, True)


@pytest.mark.parametrize("rows,T", [(3, 300_000), (300_000, 3), (1_100_000, 1)])
def test_product_of_many_rows(dev, rows, T):
    c = Case(rows, 64, T)
    out = out_of(c)
    K.matmul_i8(out, *c.buffers(), None, None, 64, rows, T)
    c.check(host(out), False, EPI_NONE, False)


def test_in_the_order_of_a_chosen_stream(dev):
    n, T, dim = Norm(60, 700, TYPE_F32), 60, 700
    x, r = zeros_f32((T, dim)), zeros_f32((T, dim))
    a = list(n.arrays(ROWS_I8))
    a[4], a[5] = x, r
    got = in_order(dev, lambda: n.call(a, ROWS_I8), [(x, n.x.astype(np.float32)), (r, n.r.astype(np.float32))],
                   [a[3], a[2], a[0], a[1]])
    back = [torch.from_numpy(g).to(dev) for g in got]
    n.check(back[0], back[1], back[2], back[3], ROWS_I8)
    q, sc = torch.zeros((T, dim), dtype=torch.int8, device=dev), zeros_f32(T)
    gq, gs = in_order(dev, lambda: K.quantize_i8(q, sc, x, r, dim, T), [(x, n.x.astype(np.float32)), (r, n.r.astype(np.float32))],
                      [q, sc])
    quant_check(glu64(n.x, n.r, ACT_SILU), torch.from_numpy(gq).to(dev), torch.from_numpy(gs).to(dev), "stream")
    for rows, cols, tok in ((300, 512, 1), (300, 512, 40), (300, 500, 40), (700, 512, 500)):
        c = Case(rows, cols, tok)
        w, sw, _, sx = c.buffers()
        xq, out = torch.zeros((tok, cols), dtype=torch.int8, device=dev), out_of(c)
        got, = in_order(dev, lambda: K.matmul_i8(out, w, sw, xq, sx, None, None, cols, rows, tok), [(xq, c.x)], [out])
        c.check(got.astype(np.float64), False, EPI_NONE, False)


def test_two_at_once(dev):
    """The same calls on two streams that run at once, on buffers of their own: nothing
    is shared between them."""
    cases = [Case(1500, 1024, T, seed=T) for T in (30, 300)]
    norms = [Norm(400, 3000, TYPE_F32, seed=i) for i in range(2)]
    bufs, outs, arrays = [c.buffers() for c in cases], [out_of(c) for c in cases], [n.arrays(ROWS_I8) for n in norms]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, b, o, n, a, s in zip(cases, bufs, outs, norms, arrays, streams):
            K.set_stream(s)
            try:
                n.call(a, ROWS_I8)
                K.matmul_i8(o, *b, None, None, c.cols, c.rows, c.T)
            finally:
                K.set_stream(None)
    torch.cuda.synchronize()
    for c, o, n, a in zip(cases, outs, norms, arrays):
        c.check(host(o), False, EPI_NONE, False)
        n.check(a[3], a[2], a[0], a[1], ROWS_I8)


@pytest.mark.parametrize("rows,cols,T", [(2000, 2048, 40), (700, 4096, 9), (3000, 512, 700)])
def test_same_bits_every_time(dev, rows, cols, T):
    c = Case(rows, cols, T)
    b, first = c.buffers(), None
    for _ in range(4):
        out = out_of(c)
        K.matmul_i8(out, *b, up_f32(c.bias), None, cols, rows, T, EPI_SILU)
        got = down(out)
        first = got if first is None else first
        assert np.array_equal(first.view(np.uint32), got.view(np.uint32))


def test_more_threads_than_an_axis_holds(dev):
    """2^26 waves and more: rows of one value, channels of one token."""
    n = 2**26 + 5003
    x, q, sc = torch.ones((n, 1), device=dev), torch.zeros((n, 1), dtype=torch.int8, device=dev), zeros_f32(n)
    K.rms_norm_q8(q, sc, None, None, x, None, up_f32(np.full(1, 2.0)), 1, n, 0.0, TYPE_F32, ROWS_I8)
    torch.cuda.synchronize()
    assert (q == 127).all() and (sc == float(np.float32(2 / 127))).all()
    q.zero_()
    for up in (None, x):
        torch.cuda.synchronize()
        K.quantize_i8(q, sc, x, up, 1, n)
        torch.cuda.synchronize()
        assert (q == 127).all()
        q.zero_()
    w, ws, out = torch.ones((n, 3), dtype=torch.int8, device=dev), torch.ones(n, device=dev), zeros_f32((2, n))
    x = torch.tensor([[1, 2, 3], [4, 5, -6]], dtype=torch.int8, device=dev)
    torch.cuda.synchronize()
    for T in (1, 2):
        K.matmul_i8(out, w, ws, x, up_f32(np.ones(2)), None, None, 3, n, T)
        torch.cuda.synchronize()
        assert (out[0] == 6).all() and (out[1] == (3 if T == 2 else 0)).all()


# tokens times the tiles' threads past 2^32: rows at any byte, and whole pieces
@pytest.mark.parametrize("T,cols", [(2**30 + 1000, 1), (2**31 - 1, 16)])
def test_more_tiles_than_an_axis_holds(dev, T, cols):
    x, sx, out = torch.ones((T, cols), dtype=torch.int8, device=dev), torch.ones(T, device=dev), zeros_f32((T, 1))
    torch.cuda.synchronize()
    K.matmul_i8(out, torch.ones((1, cols), dtype=torch.int8, device=dev), up_f32(np.ones(1)), x, sx, None, None, cols, 1, T)
    torch.cuda.synchronize()
    assert (out == cols).all()
