"""pulsar_matmul_i8: its sums as the exact integers they are, its epilogue within its
roundings, at the chunk lengths, channel counts, row lengths and alignments where the
product changes its kernel; and a layer of it with the norm and the quantizer around."""
import numpy as np
import pytest
import torch

from pulsar_amd import kernels as K
from pulsar_amd import runtime
from pulsar_amd.formats import (ACT_SILU, EPI_GELU, EPI_NONE, EPI_RELU, EPI_SIGMOID, EPI_SILU, ROWS_I8, TYPE_BF16,
                                TYPE_F16, TYPE_F32)
from tests.gpu_util import down, up_f32
from tests.test_gpu_product_fused import act64
from tests.test_gpu_rows8 import HALF, NAMES, TINY, TORCH, codes64, dev_rows, glu64, host, near, rounded

pytestmark = pytest.mark.gpu
ACTS = [EPI_NONE, EPI_SILU, EPI_GELU, EPI_RELU, EPI_SIGMOID]
TYPES = [TYPE_F32, TYPE_F16, TYPE_BF16]


def i8(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int8)).to("cuda:0")


def int_dots(x, w):
    """Exact: every partial sum of f64 integers is below 2^53."""
    return x.astype(np.float64) @ w.astype(np.float64).T


class Case:
    def __init__(self, rows, cols, T, kind=TYPE_F32, seed=0):
        rng = np.random.default_rng(rows * 7 + cols + T + kind + seed)
        self.rows, self.cols, self.T, self.kind = rows, cols, T, kind
        self.x, self.w = (rng.integers(-128, 128, (n, cols)).astype(np.int8) for n in (T, rows))
        self.sx = (rng.random(T) + 0.5).astype(np.float32)
        self.sw = ((rng.random(rows) + 0.5) / (5476 * np.sqrt(cols))).astype(np.float32)
        self.bias = (0.5 * rng.standard_normal(rows)).astype(np.float32)
        self.res = rounded(rng.standard_normal((T, rows)), kind)
        self.v = int_dots(self.x, self.w) * self.sx[:, None].astype(np.float64) * self.sw.astype(np.float64)

    def buffers(self):
        return i8(self.w), up_f32(self.sw), i8(self.x), up_f32(self.sx)

    def check(self, got, bias, act, res, what=()):
        """Roundings of 2^-24: the sum to f32, two products, the bias add: 4 of v and
        bias, which an activation of slope <= 1.13 passes on; the activation's own 8 of
        its value, GELU's exponent 4 of 1 (tests/test_gpu_product_fused.py); the
        residual add 1 of out; then the rows' type."""
        b, r = self.bias.astype(np.float64) if bias else 0.0, self.res if res else 0.0
        v = self.v + b
        a = act64(act, v)
        want = a + r
        tol = 2.0**-24 * (4.5 * np.abs(self.v) + 1.2 * np.abs(v) + 8 * np.abs(a) + 4 * (act != EPI_NONE) + np.abs(want))
        if self.kind != TYPE_F32:
            tol = tol + HALF[self.kind] * (np.abs(want) + tol) + TINY[self.kind]
        err = np.abs(got - want)
        assert (err <= tol).all(), (self.rows, self.cols, self.T, NAMES[self.kind], act, what, float(err.max()),
                                    np.argwhere(~(err <= tol))[:4].tolist())


def out_of(c):
    return torch.full((c.T, c.rows), 77.0, dtype=TORCH[c.kind], device="cuda:0")


# rows, columns, tokens
SHAPES = [(1, 1, 1), (3, 15, 1), (64, 16, 2), (65, 17, 3), (300, 1000, 4), (500, 4096, 1), (33, 5000, 5), (130, 2047, 7),
          (257, 128, 16), (100, 4096, 17), (1000, 144, 31), (513, 512, 32), (96, 3000, 33), (4100, 64, 48),
          (300, 1040, 64), (127, 640, 65), (1500, 96, 100), (200, 2048, 128), (260, 384, 130), (129, 20000, 129),
          (700, 272, 255), (512, 512, 256), (1025, 160, 300), (2049, 131, 257), (300, 130, 1000), (4352, 256, 1100),
          (70, 64, 5000), (8, 131071, 3), (40, 131071, 70), (300, 65536, 140)]


@pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols,T", SHAPES)
def test_shapes(dev, rows, cols, T, kind):
    c = Case(rows, cols, T, kind)
    bufs = c.buffers()
    out = out_of(c)
    K.matmul_i8(out, *bufs, None, None, cols, rows, T, EPI_NONE, kind)
    c.check(host(out), False, EPI_NONE, False)
    act = ACTS[(rows + T + kind) % 5]
    K.matmul_i8(out, *bufs, up_f32(c.bias), dev_rows(c.res, kind), cols, rows, T, act, kind)
    c.check(host(out), True, act, True)


@pytest.mark.parametrize("rows,cols,T", [(200, 512, 1), (300, 512, 20), (300, 512, 70), (600, 512, 600)])
def test_sums_are_exact(dev, rows, cols, T):
    """Scales of 1: sums below 2^24 come out as they are."""
    c = Case(rows, cols, T)
    w, _, x, _ = c.buffers()
    out, ones = out_of(c), lambda n: up_f32(np.ones(n))  # noqa: E731
    K.matmul_i8(out, w, ones(rows), x, ones(T), None, None, cols, rows, T)
    assert np.array_equal(host(out), int_dots(c.x, c.w))


@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_the_largest_sums(dev, T):
    """131071 products of 128 x 128, the most that 32 bits hold, and their negative."""
    n = 131071
    x, w = np.full((T, n), -128, np.int8), np.full((3, n), -128, np.int8)
    w[1] = 127
    out = torch.zeros((T, 3), device=dev)
    K.matmul_i8(out, i8(w), up_f32(np.ones(3)), i8(x), up_f32(np.ones(T)), None, None, n, 3, T)
    want = np.array([n * 16384, -n * 128 * 127, n * 16384])
    assert (host(out) == np.float32(want)).all()


@pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols,T", [(70, 512, 3), (300, 512, 33), (300, 512, 200), (520, 384, 600), (130, 301, 90)])
@pytest.mark.parametrize("shift", [0, 1, 4, 16])
def test_columns_of_wider_arrays(dev, rows, cols, T, kind, shift):
    """Rows of x and w from byte `shift` on, at strides that are and are not multiples
    of 16, out and residual columns of one array; what lies between the rows stays."""
    c = Case(rows, cols, T, kind)
    pad = 32 if shift in (0, 16) and cols % 16 == 0 else 37
    w, x = (torch.full((n, cols + pad), 101, dtype=torch.int8, device=dev) for n in (rows, T))
    w[:, shift:shift + cols], x[:, shift:shift + cols] = i8(c.w), i8(c.x)
    wide = torch.full((T, 2 * rows + 9), 5.0, dtype=TORCH[kind], device=dev)
    out, res = wide[:, 1:1 + rows], wide[:, rows + 4:2 * rows + 4]
    res.copy_(dev_rows(c.res, kind))
    K.matmul_i8(out, w[:, shift:shift + cols], up_f32(c.sw), x[:, shift:shift + cols], up_f32(c.sx), up_f32(c.bias), res,
                cols, rows, T, EPI_SILU, kind, cols + pad, cols + pad, 2 * rows + 9, 2 * rows + 9)
    got = host(wide)
    c.check(got[:, 1:1 + rows], True, EPI_SILU, True)
    assert np.array_equal(got[:, rows + 4:2 * rows + 4], c.res)
    for a, b in ((0, 1), (1 + rows, rows + 4), (2 * rows + 4, 2 * rows + 9)):
        assert (got[:, a:b] == 5).all()


@pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols,T", [(300, 256, 1), (700, 256, 40), (900, 256, 300)])
def test_residual_in_place(dev, rows, cols, T, kind):
    c = Case(rows, cols, T, kind)
    out = dev_rows(c.res, kind)
    K.matmul_i8(out, *c.buffers(), up_f32(c.bias), out, cols, rows, T, EPI_NONE, kind)
    c.check(host(out), True, EPI_NONE, True)


@pytest.mark.parametrize("rows,cols,T", [(70, 300, 2), (70, 304, 9), (300, 304, 90), (300, 304, 700)])
def test_what_is_not_finite(dev, rows, cols, T):
    """A token's scale of NaN or infinity, as the quantizer gives it to a row that is
    not finite, shows in that token alone."""
    c = Case(rows, cols, T)
    w, sw, x, _ = c.buffers()
    sx = c.sx.copy()
    sx[0] = np.nan
    x[0] = 0
    sx[T - 1] = np.inf
    x[T - 1] = 0
    out = out_of(c)
    K.matmul_i8(out, w, sw, x, up_f32(sx), None, None, cols, rows, T)
    got = host(out)
    assert np.isnan(got[[0, T - 1]]).all()
    if T > 2:
        c.v[[0, T - 1]] = got[[0, T - 1]] = 0
        c.check(got, False, EPI_NONE, False)


@pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("T,hidden,ffn", [(1, 512, 1000), (37, 500, 777), (300, 1024, 1536)])
def test_dense_ffn(dev, T, hidden, ffn, kind):
    """A dense layer as it would run: the norm with the residual, gate and up in one
    product, the quantizer of their combine, the down product back onto the sum; each
    step against 64 bits on what the step before it gave. Captured and replayed."""
    rng = np.random.default_rng(T)
    wu, wd = rng.integers(-127, 128, (2 * ffn, hidden)).astype(np.int8), rng.integers(-127, 128, (hidden, ffn)).astype(np.int8)
    su, sd = ((rng.random(n) + 0.5).astype(np.float32) / (74 * np.sqrt(k)).astype(np.float32)
              for n, k in ((2 * ffn, hidden), (hidden, ffn)))
    gain = np.exp(0.2 * rng.standard_normal(hidden)).astype(np.float32)
    new = lambda *s: torch.zeros(s, dtype=TORCH[kind], device=dev)  # noqa: E731
    q8 = lambda n: torch.zeros((T, n), dtype=torch.int8, device=dev)  # noqa: E731
    x, r, s, gu, out = new(T, hidden), new(T, hidden), new(T, hidden), new(T, 2 * ffn), new(T, hidden)
    q, sc, mq, msc, dgain = q8(hidden), up_f32(np.zeros(T)), q8(ffn), up_f32(np.zeros(T)), up_f32(gain)
    dwu, dsu, dwd, dsd = i8(wu), up_f32(su), i8(wd), up_f32(sd)

    def layer():
        K.rms_norm_q8(q, sc, None, s, x, r, dgain, hidden, T, 1e-5, kind, ROWS_I8)
        K.matmul_i8(gu, dwu, dsu, q, sc, None, None, hidden, 2 * ffn, T, EPI_NONE, kind)
        K.quantize_i8(mq, msc, gu, gu[:, ffn:], ffn, T, ACT_SILU, kind, 2 * ffn, 2 * ffn)
        K.matmul_i8(out, dwd, dsd, mq, msc, None, s, ffn, hidden, T, EPI_NONE, kind)

    layer()
    torch.cuda.synchronize()
    graph = runtime.Graph.capture(layer)
    for seed in range(3):
        hx, hr = rounded(rng.standard_normal((T, hidden)), kind), rounded(rng.standard_normal((T, hidden)), kind)
        x.copy_(dev_rows(hx, kind)), r.copy_(dev_rows(hr, kind))
        torch.cuda.synchronize()
        graph.launch()
        runtime.sync()
        hs = rounded(hx + hr, kind)
        assert np.array_equal(host(s), hs)
        p = hs * gain.astype(np.float64)
        root = 1 / np.sqrt((hs * hs).mean(1, keepdims=True) + np.float64(np.float32(1e-5)))
        top = np.abs(p).max(1, keepdims=True)
        hq, hsc = down(q), down(sc)
        assert np.array_equal(hq, codes64(p, top))
        near(hsc, (top * root / 127)[:, 0], 2.0**-23, 0, "scales")
        want = int_dots(hq, wu) * hsc[:, None].astype(np.float64) * su
        near(host(gu), want, 3.1 * 2.0**-24 + 1.01 * HALF[kind], TINY[kind], "gate and up")
        hg = host(gu)
        v = glu64(hg[:, :ffn], hg[:, ffn:], ACT_SILU)
        top = np.abs(v).max(1, keepdims=True)
        hmq, hmsc = down(mq), down(msc)
        assert np.abs(hmq - codes64(v, top)).sum() <= 1  # a value on a half to 2^-40
        near(hmsc, top[:, 0] / 127, 2.0**-23, 0, "mid scales")
        dots = int_dots(hmq, wd) * hmsc[:, None].astype(np.float64) * sd
        tol = 2.0**-24 * (3.1 * np.abs(dots) + 1.1 * np.abs(dots + hs)) + HALF[kind] * 1.01 * np.abs(dots + hs) + TINY[kind]
        assert (np.abs(host(out) - (dots + hs)) <= tol).all()


# a shape for each kernel of rows at any byte, with row ends in every place of a word,
# a 16-byte piece and a step of 128
@pytest.mark.parametrize("rows,cols,T", [(700, 1501, 5), (512, 4099, 16), (500, 261, 40), (600, 1026, 33), (6000, 131, 60),
                                         (5001, 1027, 61), (5001, 255, 130), (5000, 390, 200), (2049, 257, 1000),
                                         (2048, 513, 1023), (2100, 642, 2100)])
@pytest.mark.parametrize("x_at,w_at,x_pad,w_pad", [(0, 1, 1, 3), (1, 2, 2, 1), (2, 3, 3, 2), (3, 0, 0, 0), (0, 0, 4, 1)])
def test_rows_at_any_byte(dev, rows, cols, T, x_at, w_at, x_pad, w_pad):
    """Bytes between the rows are -128 and 127, and the arrays end with the last row."""
    c = Case(rows, cols, T, TYPE_BF16)

    def placed(a, at, pad, fill):
        n = a.shape[0]
        t = torch.full((at + (n - 1) * (cols + pad) + cols,), fill, dtype=torch.int8, device=dev)
        v = t[at:].as_strided((n, cols), (cols + pad, 1))
        v.copy_(i8(a))
        return v

    x, w = placed(c.x, x_at, x_pad, -128), placed(c.w, w_at, w_pad, 127)
    out = out_of(c)
    K.matmul_i8(out, w, up_f32(c.sw), x, up_f32(c.sx), up_f32(c.bias), dev_rows(c.res, c.kind), cols, rows, T, EPI_SILU,
                c.kind, cols + w_pad, cols + x_pad)
    c.check(host(out), True, EPI_SILU, True)


# more channels than a round of the tiles that fit few tokens
@pytest.mark.parametrize("kind", [TYPE_F32, TYPE_BF16], ids=NAMES.get)
@pytest.mark.parametrize("rows,cols,T", [(17000, 304, 3), (17000, 1040, 32), (33000, 144, 33), (33000, 272, 64),
                                         (33000, 144, 65), (33000, 143, 9), (33000, 77, 64), (33000, 45, 65)])
def test_many_channels(dev, rows, cols, T, kind):
    c = Case(rows, cols, T, kind)
    out = out_of(c)
    K.matmul_i8(out, *c.buffers(), up_f32(c.bias), dev_rows(c.res, kind), cols, rows, T, EPI_RELU, kind)
    c.check(host(out), True, EPI_RELU, True)


# tiles whose groups outnumber the parts of their sums, all tokens and channels of a tile there
@pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols,T", [(256, 1024, 160), (256, 1025, 160), (1024, 2048, 224), (1030, 2048, 200),
                                         (64, 4096, 16), (2048, 2064, 32)])
def test_residual_that_ends_with_its_memory(dev, rows, cols, T, kind):
    """Residual and output in the last bytes of allocations of whole pages."""
    c = Case(rows, cols, T, kind)
    res, out = (torch.zeros(2**25 // TORCH[kind].itemsize, dtype=TORCH[kind], device=dev)[-T * rows:].view(T, rows)
                for _ in range(2))
    res.copy_(dev_rows(c.res, kind))
    bufs, bias = c.buffers(), up_f32(c.bias)
    K.matmul_i8(out, *bufs, bias, res, cols, rows, T, EPI_GELU, kind)
    c.check(host(out), True, EPI_GELU, True)


@pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols,T", [(2050, 2048, 200), (2050, 2064, 200), (4096, 4112, 256), (4096, 2064, 192)])
def test_two_groups_of_64(dev, rows, cols, T, kind):
    """On both sides of the row length from which two groups share a 64 x 64 tile."""
    c = Case(rows, cols, T, kind)
    out = out_of(c)
    K.matmul_i8(out, *c.buffers(), up_f32(c.bias), dev_rows(c.res, kind), cols, rows, T, EPI_GELU, kind)
    c.check(host(out), True, EPI_GELU, True)
