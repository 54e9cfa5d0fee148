"""pulsar_rms_norm_q8 and pulsar_quantize_i8 against their formulas in 64 bits: sums
and codes exactly, norms and scales within their roundings; rows from one value to
those that no block holds, every element type, strides, NaN and infinity, graphs."""
import numpy as np
import pytest
import torch

from pulsar_amd import formats as fm
from pulsar_amd import kernels as K
from pulsar_amd import runtime
from pulsar_amd.formats import ACT_SILU, ACT_SWIGLU_OAI, ROWS_I8, ROWS_Q8_K, TYPE_BF16, TYPE_F16, TYPE_F32
from tests.gpu_util import down, up_f32

pytestmark = pytest.mark.gpu
TYPES = [TYPE_F32, TYPE_F16, TYPE_BF16]
TORCH = {TYPE_F32: torch.float32, TYPE_F16: torch.float16, TYPE_BF16: torch.bfloat16}
HALF = {t: torch.finfo(TORCH[t]).eps / 2 for t in TYPES}  # a rounding's share of the value
TINY = {t: torch.finfo(TORCH[t]).smallest_normal * torch.finfo(TORCH[t]).eps for t in TYPES}  # and below the normal ones
NAMES = {TYPE_F32: "f32", TYPE_F16: "f16", TYPE_BF16: "bf16"}
by_type = pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)


def rounded(a, kind):
    """The rows' type nearest to a, as f64."""
    return torch.from_numpy(np.asarray(a, np.float32)).to(TORCH[kind]).double().numpy()


def dev_rows(a, kind):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TORCH[kind]).to("cuda:0")


def host(t):
    return down(t.double())


def codes64(v, top):
    """[..] values, [.., 1] largest sizes: the nearest integers, halves up in size."""
    with np.errstate(invalid="ignore", divide="ignore"):
        t = np.where(top > 0, np.abs(v) / top, 0.0) * 127.0
        return (np.sign(v) * np.floor(t + 0.5 + 2.0**-40)).astype(np.int64)


def near(got, want, rel, tiny, what):
    """Within rel of the value, or a step of the type's least numbers."""
    bad = ~(np.abs(got - want) <= rel * np.abs(want) + tiny)
    assert not bad.any(), (what, np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


def split_blocks(q, rows, dim):
    b = down(q).reshape(rows, -(-dim // 256), 292)
    d = np.ascontiguousarray(b[..., :4]).view(np.float32)
    sums = np.ascontiguousarray(b[..., 260:]).view(np.int16)
    return d.astype(np.float64), b[..., 4:260].view(np.int8).astype(np.int64), sums.astype(np.int64)


# a rounding to f32 before the one to the type, and 2^-50 for the sums in 64 bits
def rel_of(kind):
    return HALF[kind] + (0 if kind == TYPE_F32 else 2.0**-24) + 2.0**-50


class Norm:
    """Rows and what the formula makes of them."""

    def __init__(self, rows, dim, kind, residual=True, eps=1e-5, seed=0, size=1.0):
        rng = np.random.default_rng(rows * 31 + dim + kind + seed)
        self.rows, self.dim, self.kind, self.eps = rows, dim, kind, eps
        wide = np.exp(0.5 * rng.standard_normal(dim))
        self.x = rounded(size * rng.standard_normal((rows, dim)) * wide, kind)
        self.r = rounded(size * rng.standard_normal((rows, dim)), kind) if residual else None
        self.g = np.exp(0.3 * rng.standard_normal(dim)).astype(np.float32)

    def want(self):
        s = self.x if self.r is None else rounded((self.x.astype(np.float32) + self.r.astype(np.float32)), self.kind)
        p = s * self.g.astype(np.float64)
        root = 1.0 / np.sqrt((s * s).mean(1, keepdims=True) + np.float64(np.float32(self.eps)))
        return s, p, root

    def check(self, s, y, q, scales, fmt):
        """Arrays of the call (None: left out) against the formula."""
        ws, p, root = self.want()
        what = (self.rows, self.dim, NAMES[self.kind], fmt)
        if s is not None:
            assert np.array_equal(host(s), ws), what
        if y is not None:
            near(host(y), p * root, rel_of(self.kind), TINY[self.kind], (what, "y"))
        if q is None:
            return
        if fmt == ROWS_I8:
            top = np.abs(p).max(1, keepdims=True)
            near(down(scales).astype(np.float64), (top * root / 127)[:, 0], rel_of(TYPE_F32), TINY[TYPE_F32],
                 (what, "scales"))
            assert np.array_equal(down(q), codes64(p, top)), what
            return
        nb = -(-self.dim // 256)
        blocks = np.zeros((self.rows, 256 * nb))
        blocks[:, :self.dim] = p
        blocks = blocks.reshape(self.rows, nb, 256)
        top = np.abs(blocks).max(2, keepdims=True)
        d, codes, sums = split_blocks(q, self.rows, self.dim)
        near(d, top * root[..., None] / 127, rel_of(TYPE_F32), TINY[TYPE_F32], (what, "d"))
        assert np.array_equal(codes, codes64(blocks, top)), what
        assert np.array_equal(sums, codes.reshape(self.rows, nb, 16, 16).sum(-1)), what

    def arrays(self, fmt):
        x, r = dev_rows(self.x, self.kind), None if self.r is None else dev_rows(self.r, self.kind)
        s, y = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
        if fmt == ROWS_I8:
            q, sc = torch.full((self.rows, self.dim), 99, dtype=torch.int8, device=x.device), up_f32(np.full(self.rows, 7))
        else:
            q, sc = torch.full((self.rows * -(-self.dim // 256) * 292,), 99, dtype=torch.uint8, device=x.device), None
        return q, sc, y, s, x, r, up_f32(self.g)

    def call(self, arrays, fmt, **kw):
        K.rms_norm_q8(*arrays, self.dim, self.rows, self.eps, self.kind, fmt, **kw)


# one value; rows inside a chunk of 256, on its edge and past it; one to 16 waves of one,
# two and four chunks; the longest that a block holds and the next
DIMS = [1, 3, 64, 255, 256, 257, 1000, 2880, 4095, 4096, 4097, 5001, 8192, 8193, 14336, 16384, 16385, 20001]


@pytest.mark.parametrize("fmt", [ROWS_Q8_K, ROWS_I8])
@by_type
@pytest.mark.parametrize("dim", DIMS)
def test_norm(dev, dim, kind, fmt):
    n = Norm(3, dim, kind)
    a = n.arrays(fmt)
    n.call(a, fmt)
    n.check(a[3], a[2], a[0], a[1], fmt)


@by_type
@pytest.mark.parametrize("rows,dim", [(1, 4096), (700, 300), (70000, 8), (40, 16390)])
def test_norm_rows(dev, rows, dim, kind):
    for fmt in (ROWS_Q8_K, ROWS_I8):
        n = Norm(rows, dim, kind)
        a = n.arrays(fmt)
        n.call(a, fmt)
        n.check(a[3], a[2], a[0], a[1], fmt)


@pytest.mark.parametrize("dim", [1000, 17000])
@pytest.mark.parametrize("left_out", ["residual", "sum", "y", "q", "residual sum", "residual sum y", "sum q"])
def test_norm_leaves_out(dev, left_out, dim):
    for fmt in (ROWS_Q8_K, ROWS_I8):
        n = Norm(5, dim, TYPE_F32, residual="residual" not in left_out)
        a = list(n.arrays(fmt))
        for i, name in ((0, "q"), (1, "q"), (2, "y"), (3, "sum"), (5, "residual")):
            if name in left_out.split():
                a[i] = None
        n.call(a, fmt)
        n.check(a[3], a[2], a[0], a[1], fmt)


@by_type
@pytest.mark.parametrize("dim", [301, 8000, 17001])
@pytest.mark.parametrize("onto", [4, 5])  # x, residual
def test_norm_sum_in_place(dev, onto, dim, kind):
    n = Norm(6, dim, kind)
    a = list(n.arrays(ROWS_I8))
    a[3] = a[onto]
    n.call(a, ROWS_I8)
    n.check(a[3], a[2], a[0], a[1], ROWS_I8)


@by_type
@pytest.mark.parametrize("dim", [37, 1001, 16500])
def test_norm_columns_of_wider_arrays(dev, dim, kind):
    """Every array at a stride of its own, from an odd element on; what lies between
    the rows stays."""
    n = Norm(7, dim, kind)
    x, r, s = (torch.full((7, dim + k), 3.0, dtype=TORCH[kind], device=dev) for k in (3, 5, 8))
    q = torch.full((7, dim + 2), 55, dtype=torch.int8, device=dev)
    x[:, 1:1 + dim], r[:, 3:3 + dim] = dev_rows(n.x, kind), dev_rows(n.r, kind)
    sc, y = up_f32(np.zeros(7)), torch.zeros((7, dim), dtype=TORCH[kind], device=dev)
    n.call((q[:, 1:1 + dim], sc, y, s[:, 5:5 + dim], x[:, 1:1 + dim], r[:, 3:3 + dim], up_f32(n.g)), ROWS_I8,
           x_stride=dim + 3, res_stride=dim + 5, sum_stride=dim + 8, q_stride=dim + 2)
    n.check(s[:, 5:5 + dim].contiguous(), y, q[:, 1:1 + dim].contiguous(), sc, ROWS_I8)
    assert (host(s[:, :5]) == 3).all() and (host(s[:, 5 + dim:]) == 3).all()
    assert (down(q[:, 0]) == 55).all() and (down(q[:, 1 + dim:]) == 55).all()


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_norm_blocks_at_any_byte(dev, shift):
    n = Norm(3, 700, TYPE_F32)
    a = list(n.arrays(ROWS_Q8_K))
    buf = torch.full((a[0].numel() + 8,), 77, dtype=torch.uint8, device=dev)
    a[0] = buf[shift:shift + a[0].numel()]
    n.call(a, ROWS_Q8_K)
    n.check(a[3], a[2], a[0], None, ROWS_Q8_K)
    assert (down(buf[:shift]) == 77).all() and (down(buf[shift + a[0].numel():]) == 77).all()


@by_type
def test_norm_halves_and_the_largest(dev, kind):
    """Values that are half the largest (63.5 steps, up in size) and 1/254 of it, of
    both signs, with gains that are powers of two; blocks of one size, of zeros."""
    dim = 1024
    x = np.zeros((4, dim), np.float32)
    x[0, :6] = [254, 127, -127, 1, -1, 3]
    x[1, 256:262] = [-2, 1, -1, 0.5, 0.25, 2]
    x[2, 512:] = 1.0
    n = Norm(4, dim, kind, residual=False)
    n.x, n.g = rounded(x, kind), np.exp2(np.arange(dim) % 3).astype(np.float32)
    n.g[:6] = 1
    for fmt in (ROWS_Q8_K, ROWS_I8):
        a = n.arrays(fmt)
        n.call(a, fmt)
        n.check(None, a[2], a[0], a[1], fmt)
    q = down(a[0])
    assert q[0, :6].tolist() == [127, 64, -64, 1, -1, 2] and not q[3].any()


def test_norm_of_zeros(dev):
    for eps in (0.0, 1e-6):
        n = Norm(3, 600, TYPE_F32, residual=False, eps=eps)
        n.x[:] = 0
        for fmt in (ROWS_Q8_K, ROWS_I8):
            a = n.arrays(fmt)
            n.call(a, fmt)
            assert not down(a[2]).any() and not down(a[0]).any() and not down(a[3]).any()
            assert fmt == ROWS_Q8_K or not down(a[1]).any()


@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e18, 1e30])
def test_norm_sizes(dev, size):
    """Squares beyond f32 on both sides."""
    n = Norm(4, 1500, TYPE_F32, eps=0.0, size=size)
    for fmt in (ROWS_Q8_K, ROWS_I8):
        a = n.arrays(fmt)
        n.call(a, fmt)
        n.check(a[3], a[2], a[0], a[1], fmt)


@pytest.mark.parametrize("dim", [900, 18000])
@by_type
def test_norm_of_what_is_not_finite(dev, dim, kind):
    """A NaN or an infinity is seen in its row's scales and nowhere else."""
    for fmt in (ROWS_Q8_K, ROWS_I8):
        n = Norm(4, dim, kind)
        n.x[1, 300], n.x[2, 301] = np.nan, np.inf
        a = n.arrays(fmt)
        n.call(a, fmt)
        y = host(a[2])
        assert np.isnan(y[1]).all() and np.isnan(y[2, 301]) and not y[2, :301].any() and not y[2, 302:].any()
        if fmt == ROWS_I8:
            sc = down(a[1])
            assert np.isnan(sc[1:3]).all() and not down(a[0])[1:3].any()
        else:
            d, codes, _ = split_blocks(a[0], 4, dim)
            assert np.isnan(d[1]).all() and np.isnan(d[2, 1]) and not codes[1:3, 1].any() and not d[2, 0].any()
        keep = [0, 3]
        m = Norm(4, dim, kind)
        m.rows, m.x, m.r = 2, m.x[keep], m.r[keep]
        q = a[0][keep] if fmt == ROWS_I8 else a[0].view(4, -1)[keep].reshape(-1)
        m.check(a[3][keep], a[2][keep], q, None if a[1] is None else a[1][keep], fmt)


# -------------------------------------------------------------- quantizer --

def glu64(g, u, op):
    a = 1.0
    if op == ACT_SWIGLU_OAI:
        a, g, u = 1.702, np.minimum(g, 7.0), np.clip(u, -7.0, 7.0) + 1.0
    e = np.exp(-np.abs(a * g))
    return g * u * (np.where(g < 0, e, 1.0) / (1.0 + e))


def quant_check(v, q, scales, what):
    top = np.abs(v).max(1, keepdims=True)
    near(down(scales).astype(np.float64), top[:, 0] / 127, 2.0**-24 + 2.0**-49, TINY[TYPE_F32], what)
    got, want = down(q).astype(np.int64), codes64(v, top)
    bad = got != want
    # the combine's 64-bit values are within some 2^-50 of one another on both sides: an
    # argument of up to 127 moves by 2^-42
    with np.errstate(invalid="ignore", divide="ignore"):
        t = np.where(top > 0, np.abs(v) / top, 0.0) * 127.0
    border = np.abs(t - np.floor(t) - 0.5) <= 2.0**-39
    assert not (bad & ~border).any(), (what, np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


OPS = [None, ACT_SILU, ACT_SWIGLU_OAI]


@pytest.mark.parametrize("op", OPS)
@by_type
@pytest.mark.parametrize("dim", DIMS)
def test_quantize(dev, dim, kind, op):
    rows = 3
    rng = np.random.default_rng(dim + kind)
    x, u = rounded(3 * rng.standard_normal((rows, dim)), kind), rounded(3 * rng.standard_normal((rows, dim)), kind)
    q, sc = torch.full((rows, dim), 99, dtype=torch.int8, device=dev), up_f32(np.full(rows, 9))
    K.quantize_i8(q, sc, dev_rows(x, kind), None if op is None else dev_rows(u, kind), dim, rows, op or 0, kind)
    quant_check(x if op is None else glu64(x, u, op), q, sc, (dim, NAMES[kind], op))


@by_type
@pytest.mark.parametrize("rows,dim", [(1, 14336), (900, 300), (70000, 5), (33, 17000)])
def test_quantize_columns(dev, rows, dim, kind):
    """Gate and up as columns of one array, codes at a stride; what lies between the
    rows stays."""
    rng = np.random.default_rng(rows + kind)
    both = rounded(2 * rng.standard_normal((rows, 2 * dim + 3)), kind)
    q, sc = torch.full((rows, dim + 5), 99, dtype=torch.int8, device=dev), up_f32(np.full(rows, 9))
    b = dev_rows(both, kind)
    g, u = b[:, 1:1 + dim], b[:, 1 + dim:1 + 2 * dim]
    K.quantize_i8(q[:, 2:2 + dim], sc, g, u, dim, rows, ACT_SILU, kind, 2 * dim + 3, 2 * dim + 3, dim + 5)
    quant_check(glu64(both[:, 1:1 + dim], both[:, 1 + dim:1 + 2 * dim], ACT_SILU), q[:, 2:2 + dim].contiguous(), sc,
                (rows, dim))
    assert (down(q[:, :2]) == 99).all() and (down(q[:, 2 + dim:]) == 99).all()


@by_type
def test_quantize_halves_far_gates_and_zeros(dev, kind):
    """Exact halves; gates so far out that a sigmoid is 0 or 1 in 64 bits; rows of 0."""
    x = np.zeros((5, 300), np.float32)
    x[0, :6] = [254, 127, -127, 1, -1, 3]
    x[1, 5:9] = [8, 4, -4, 2]
    q, sc = torch.zeros((5, 300), dtype=torch.int8, device=dev), up_f32(np.zeros(5))
    K.quantize_i8(q, sc, dev_rows(x, kind), None, 300, 5, 0, kind)
    quant_check(rounded(x, kind), q, sc, "halves")
    assert down(q)[0, :6].tolist() == [127, 64, -64, 1, -1, 2] and down(q)[1, 5:9].tolist() == [127, 64, -64, 32]
    assert not down(q)[2:].any() and not down(sc)[2:].any()
    g = np.linspace(-40, 40, 300)[None] * np.array([[1], [5], [20], [50], [200]])
    u = np.cos(np.arange(300.0))[None].repeat(5, 0)
    g, u = rounded(g, kind), rounded(u, kind)
    for op in (ACT_SILU, ACT_SWIGLU_OAI):
        K.quantize_i8(q, sc, dev_rows(g, kind), dev_rows(u, kind), 300, 5, op, kind)
        quant_check(glu64(g, u, op), q, sc, ("far", op))
    far = rounded(np.full((5, 300), -60000.0), kind)
    K.quantize_i8(q, sc, dev_rows(far, kind), dev_rows(u, kind), 300, 5, ACT_SILU, kind)
    assert not down(q).any() and not down(sc).any()


@pytest.mark.parametrize("dim", [700, 17000])
@pytest.mark.parametrize("op", OPS)
@by_type
def test_quantize_what_is_not_finite(dev, op, kind, dim):
    rng = np.random.default_rng(dim)
    x, u = (rounded(rng.standard_normal((4, dim)), kind) for _ in range(2))
    x[1, 300], x[2, 301] = np.nan, np.inf
    if op == ACT_SWIGLU_OAI:
        x[2, 301], u[2, 301] = 1.0, np.nan  # its clamps leave no infinity
    elif op is not None:
        u[2, 301] = 1.0
    q, sc = torch.full((4, dim), 99, dtype=torch.int8, device=dev), up_f32(np.zeros(4))
    K.quantize_i8(q, sc, dev_rows(x, kind), None if op is None else dev_rows(u, kind), dim, 4, op or 0, kind)
    s = down(sc)
    assert np.isnan(s[1]) and (np.isnan(s[2]) if op == ACT_SWIGLU_OAI else np.isposinf(s[2]))
    assert not down(q)[1:3].any()
    keep = [0, 3]
    v = x if op is None else glu64(np.where(np.isfinite(x), x, 0), np.where(np.isfinite(u), u, 0), op)
    quant_check(v[keep], q[keep], sc[keep], op)


def test_replayed(dev):
    """Both calls in a graph, replayed on new inputs between eager work."""
    n = Norm(9, 1000, TYPE_F32)
    a = n.arrays(ROWS_I8)
    q, sc = torch.zeros((9, 1000), dtype=torch.int8, device=dev), up_f32(np.zeros(9))

    def work():
        n.call(a, ROWS_I8)
        K.quantize_i8(q, sc, a[2], a[3], 1000, 9)

    work()
    torch.cuda.synchronize()
    g = runtime.Graph.capture(work)
    for seed in range(1, 5):
        m = Norm(9, 1000, TYPE_F32, seed=seed)
        a[4].copy_(dev_rows(m.x, TYPE_F32)), a[5].copy_(dev_rows(m.r, TYPE_F32)), a[6].copy_(up_f32(m.g))
        torch.cuda.synchronize()
        g.launch()
        runtime.sync()
        m.check(a[3], a[2], a[0], a[1], ROWS_I8)
        quant_check(glu64(host(a[2]), host(a[3]), ACT_SILU), q, sc, seed)


def test_feeds_the_products(dev):
    """q8_K rows of the norm through pulsar_matmul_kq: the oracle's dots of those
    bytes."""
    import oracle
    from pulsar_amd import synth
    from tests.gpu_util import assert_rows_close, up, zeros_f32

    n = Norm(3, 768, TYPE_F32)
    a = n.arrays(ROWS_Q8_K)
    n.call(a, ROWS_Q8_K)
    w = synth.quant_matrix(fm.QUANT_Q4_K, 65, 768, np.random.default_rng(1))
    out = zeros_f32((3, 65))
    rb = fm.row_bytes(fm.QUANT_Q4_K, 768)
    K.matmul_kq(out, up(w), a[0], 768, 65, 3, rb, fm.QUANT_Q4_K)
    x = down(a[0]).reshape(3, -1)
    want, scale = oracle.rows_dot(w, rb, 65, x, 768, 3, fm.QUANT_Q4_K, 8)
    assert_rows_close(down(out), want.reshape(3, 65), scale.reshape(3, 65), "dots")


@pytest.mark.parametrize("kind", [TYPE_F32, TYPE_BF16], ids=NAMES.get)
@pytest.mark.parametrize("dim", [300, 5000])
def test_quantize_least_gates(dev, dim, kind):
    """Gates at the lowest end of the type, below its normal values too, under values of
    up that bring the products back to the middle of the range."""
    rng = np.random.default_rng(dim + kind)
    e = np.arange(dim) % 25
    g = rounded(np.ldexp(1 + rng.random((3, dim)), -122 - e), kind)
    u = rounded(np.ldexp(rng.standard_normal((3, dim)), 100 + e), kind)
    assert ((g > 0) & (g < 2.0**-126)).any() and np.isfinite(u).all()
    q, sc = torch.full((3, dim), 99, dtype=torch.int8, device=dev), up_f32(np.full(3, 9))
    K.quantize_i8(q, sc, dev_rows(g, kind), dev_rows(u, kind), dim, 3, ACT_SILU, kind)
    quant_check(glu64(g, u, ACT_SILU), q, sc, (dim, NAMES[kind]))


@pytest.mark.parametrize("dim", [300, 4096])
def test_norm_blocks_and_the_f32_quantizer(dev, dim):
    """The norm's q8_K rows against pulsar_quantize_q8_K of its y: a code differs only
    where y's rounding and the f32 decision (2^-24 of an argument of up to 127 for y, its
    block's largest, 1 / d and the product each: 2^-15 together) reach a half, and by 1."""
    rows = 64
    n = Norm(rows, dim, TYPE_F32)
    a = n.arrays(ROWS_Q8_K)
    n.call(a, ROWS_Q8_K)
    other = torch.zeros_like(a[0])
    K.quantize_q8_k(other, a[2], dim, rows)
    d, codes, _ = split_blocks(a[0], rows, dim)
    d2, codes2, _ = split_blocks(other, rows, dim)
    near(d2, d, 4 * 2.0**-24, 0.0, "d")
    _, p, _ = n.want()
    nb = -(-dim // 256)
    blocks = np.zeros((rows, 256 * nb))
    blocks[:, :dim] = p
    blocks = blocks.reshape(rows, nb, 256)
    t = np.abs(blocks) / np.abs(blocks).max(2, keepdims=True) * 127
    border = np.abs(t - np.floor(t) - 0.5) <= 2.0**-15
    differ = codes != codes2
    assert (np.abs(codes - codes2) <= 1).all() and not (differ & ~border).any(), int(differ.sum())


# what a quantizer's block holds and the next; many rows, of as many waves as one row
# leaves to a second on a CU, and more
@pytest.mark.parametrize("op", OPS)
@by_type
@pytest.mark.parametrize("rows,dim", [(2, 32768), (2, 32769), (3, 40001), (256, 6144), (256, 6145), (257, 12288),
                                      (257, 12289), (300, 24577)])
def test_quantize_shapes(dev, rows, dim, kind, op):
    rng = np.random.default_rng(rows + dim + kind)
    x, u = (rounded(3 * rng.standard_normal((rows, dim), dtype=np.float32), kind) for _ in range(2))
    q, sc = torch.full((rows, dim), 99, dtype=torch.int8, device=dev), up_f32(np.full(rows, 9))
    K.quantize_i8(q, sc, dev_rows(x, kind), None if op is None else dev_rows(u, kind), dim, rows, op or 0, kind)
    quant_check(x if op is None else glu64(x, u, op), q, sc, (rows, dim, NAMES[kind], op))


@by_type
@pytest.mark.parametrize("rows,dim", [(256, 6144), (257, 6145), (256, 12289)])
def test_norm_shapes(dev, rows, dim, kind):
    for fmt in (ROWS_Q8_K, ROWS_I8):
        n = Norm(rows, dim, kind)
        a = n.arrays(fmt)
        n.call(a, fmt)
        n.check(a[3], a[2], a[0], a[1], fmt)
