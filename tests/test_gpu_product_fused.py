"""pulsar_matmul_kq_fused: its dots against the oracle, its epilogue against 64
bits on those dots, at the chunk lengths and row counts where the product changes
its kernel."""
import numpy as np
import pytest
import torch

import oracle
from pulsar_amd import formats as fm
from pulsar_amd import kernels as K
from pulsar_amd import runtime, synth
from pulsar_amd.formats import EPI_GELU, EPI_NONE, EPI_RELU, EPI_SIGMOID, EPI_SILU, row_bytes
from tests.gpu_util import assert_rows_close, down, up, up_f32, zeros_f32

pytestmark = pytest.mark.gpu
ACTS = [EPI_NONE, EPI_SILU, EPI_GELU, EPI_RELU, EPI_SIGMOID]


def act64(act, v):
    with np.errstate(over="ignore"):
        if act == EPI_SILU:
            return v / (1 + np.exp(-v))
        if act == EPI_GELU:
            return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v**3)))
        if act == EPI_RELU:
            return np.maximum(v, 0)
        return 1 / (1 + np.exp(-v)) if act == EPI_SIGMOID else v


def assert_epilogue(got, dots, bias, act, res, what):
    """f32 steps of 2^-24 each: the bias add moves v by |v| steps, which an
    activation of slope <= 1.13 passes on; the activation's own exp (2), sum,
    division and products: 8 of its value, and GELU's exponent 2z, 5 roundings
    of it, |v| s (1 - s) 2z <= 0.7 of a step each; the residual add: 1 of out."""
    v = dots.astype(np.float64) + (0.0 if bias is None else bias.astype(np.float64))
    a = act64(act, v)
    want = a + (0.0 if res is None else res.astype(np.float64))
    tol = 2.0**-24 * (1.2 * np.abs(v) + 8 * np.abs(a) + 4 + np.abs(want))
    err = np.abs(got - want)
    assert (err <= tol).all(), (what, float(err.max()), np.argwhere(err > tol)[:4].tolist())


class Case:
    def __init__(self, quant, rows, n, T, seed=0):
        rng = np.random.default_rng(rows * 7 + n + T + seed)
        self.quant, self.rows, self.n, self.T, self.rb = quant, rows, n, T, row_bytes(quant, n)
        self.w = synth.quant_matrix(quant, rows, n, rng)
        self.x = oracle.quantize_q8_k(rng.standard_normal((T, n)).astype(np.float32))
        self.dw, self.dx = up(self.w), up(self.x)
        # the bare dots; the epilogue is applied to the same sums
        self.dots = down(self.run(zeros_f32((T, rows)), None, None, EPI_NONE))
        # bias and residual of the dots' size, so that each term shows
        size = max(float(np.abs(self.dots).mean()), 1e-3)
        self.bias = (size * rng.standard_normal(rows)).astype(np.float32)
        self.res = (size * rng.standard_normal((T, rows))).astype(np.float32)

    def check_dots(self):
        """The dots against the oracle, a sample of the rows around the tiles'
        edges and of the tokens: exact integers per super-block on both sides, at
        most 6 roundings of each product's size where the two products of a format
        with mins cancel (P, M below), 1e-5 sum |f_b| for the sums' order. Where a
        super-block is itself a sum of up to 16 f32 terms, of 16 or 32 values each,
        that may cancel: 2 roundings of each term and 15 additions on either side,
        34 2^-24 of the terms' sizes."""
        at = sorted({r for e in (0, 16, 32, 64, 128, self.rows // 2, self.rows) for r in range(e - 2, e + 3)
                     if 0 <= r < self.rows})
        tok = sorted({t for e in (0, 16, 32, 48, 64, 128, self.T) for t in range(e - 2, e + 2) if 0 <= t < self.T})
        w, x = np.ascontiguousarray(self.w[at]), np.ascontiguousarray(self.x[tok])
        want, scale = oracle.rows_dot(w, self.rb, len(at), x, self.n, len(tok), self.quant, 8)
        bound = scale
        if self.quant in (fm.QUANT_Q4_K, fm.QUANT_Q5_K, fm.QUANT_Q2_K):
            w0, off = w.copy(), 82 if self.quant == fm.QUANT_Q2_K else 2
            w0.reshape(-1, fm.BLOCK_LAYOUT[self.quant][1])[:, off:off + 2] = 0
            _, p = oracle.rows_dot(w0, self.rb, len(at), x, self.n, len(tok), self.quant, 8)
            bound = scale + 6 * 2.0**-24 / 1e-5 * (2 * p + scale)
        if self.quant in (fm.QUANT_IQ4_NL, fm.QUANT_NVFP4):
            v = np.stack([oracle.dequant_row(self.quant, r, self.n) for r in w]).astype(np.float64)
            b = x.reshape(len(tok), -1, 292)
            y = np.ascontiguousarray(b[..., 4:260]).view(np.int8) * np.ascontiguousarray(b[..., :4]).view(np.float32)
            terms = np.einsum("tgi,rgi->trg", y.reshape(len(tok), -1, 16).astype(np.float64), v.reshape(len(at), -1, 16))
            bound = bound + 34 * 2.0**-24 / 1e-5 * np.abs(terms).sum(-1).reshape(bound.shape)
        assert_rows_close(self.dots[np.ix_(tok, at)], want.reshape(len(tok), len(at)),
                          bound.reshape(len(tok), len(at)), (self.quant, self.rows, self.n, self.T))

    def run(self, out, bias, res, act, **kw):
        K.matmul_kq_fused(out, self.dw, self.dx, bias, res, self.n, self.rows, self.T, self.rb, self.quant, act, **kw)
        return out


# rows, values, tokens: the lane kernels (1 to 4 tokens, several rows to a wave,
# rows of more than 8 units a lane), the 16-row kernel, the wide tile, the K split
# (each form of these two for each format: tests/test_gpu_product_forms.py)
SHAPES = [(1, 256, 1), (33, 512, 1), (500, 4096, 1), (5000, 256, 1), (65, 33024, 1), (40, 33024, 3), (130, 8448, 2),
          (70, 16640, 4), (301, 768, 3), (16500, 512, 2), (100, 512, 5), (8200, 256, 16), (16500, 768, 12),
          (513, 1024, 31), (70, 4352, 14), (4129, 512, 33), (8300, 512, 49), (1000, 768, 70), (1100, 2816, 100),
          (2049, 2304, 33), (4096, 2048, 31), (1500, 256, 64), (8300, 256, 130), (4130, 256, 500), (14400, 256, 300),
          (17, 2304, 400)]


@pytest.mark.parametrize("quant", fm.DENSE_QUANTS)
@pytest.mark.parametrize("rows,n,T", SHAPES)
def test_shapes(dev, quant, rows, n, T):
    c = Case(quant, rows, n, T)
    c.check_dots()
    act = ACTS[(rows + T + quant) % 5]
    got = down(c.run(zeros_f32((T, rows)), up_f32(c.bias), up_f32(c.res), act))
    assert_epilogue(got, c.dots, c.bias, act, c.res, (quant, act))


@pytest.mark.parametrize("rows,n,T", [(16500, 512, 12), (4130, 256, 500), (14400, 256, 300), (500, 4096, 1)])
def test_same_kernel_same_bits(dev, rows, n, T):
    """Where both run the same kernel: pulsar_matmul_kq's dots bit for bit."""
    c = Case(fm.QUANT_Q4_K, rows, n, T)
    dots = zeros_f32((T, rows))
    K.matmul_kq(dots, c.dw, c.dx, n, rows, T, c.rb, c.quant)
    assert np.array_equal(down(dots).view(np.uint32), c.dots.view(np.uint32))


@pytest.mark.parametrize("quant", fm.DENSE_QUANTS)
@pytest.mark.parametrize("rows,n,T", [(200, 2816, 5), (65, 5120, 40), (129, 256, 64)])
def test_integer_stage_exact(dev, quant, rows, n, T):
    """Unit scales and whole q8 values, one super-block's sum at a time: exact."""
    if quant not in (fm.QUANT_Q4_K, fm.QUANT_Q5_K, fm.QUANT_Q2_K, fm.QUANT_Q6_K, fm.QUANT_Q3_K, fm.QUANT_IQ4_XS):
        pytest.skip("no whole weight scale")
    rng = np.random.default_rng(n)
    w = synth.quant_matrix(quant, rows, n, rng)
    blk = w.reshape(-1, fm.BLOCK_LAYOUT[quant][1])
    for off in {fm.QUANT_Q4_K: (0, 2), fm.QUANT_Q5_K: (0, 2), fm.QUANT_Q2_K: (80, 82), fm.QUANT_Q6_K: (208,),
                fm.QUANT_Q3_K: (108,), fm.QUANT_IQ4_XS: (0,)}[quant]:
        blk[:, off], blk[:, off + 1] = 0x00, 0x3C  # 1.0
    qs = rng.integers(-9, 10, (T, n // 256, 256)).astype(np.int8)  # sums stay below 2^24
    x = np.zeros((T, n // 256, 292), np.uint8)
    x[..., 0:4] = np.array([1.0], np.float32).view(np.uint8)
    x[..., 4:260] = qs.view(np.uint8)
    x[..., 260:] = qs.reshape(T, -1, 16, 16).astype(np.int16).sum(-1).astype(np.int16).view(np.uint8).reshape(T, -1, 32)
    x = x.reshape(T, -1)
    out = zeros_f32((T, rows))
    K.matmul_kq_fused(out, up(w), up(x), None, None, n, rows, T, row_bytes(quant, n), quant, EPI_NONE)
    want, _ = oracle.rows_dot(w, row_bytes(quant, n), rows, x, n, T, quant, 8)
    assert np.array_equal(down(out), want.reshape(T, rows))


@pytest.mark.parametrize("T", [1, 3, 9, 33, 260])
@pytest.mark.parametrize("act", ACTS)
def test_terms(dev, act, T):
    c = Case(fm.QUANT_Q4_K, 300, 512, T)
    for bias, res in ((None, None), (c.bias, None), (None, c.res), (c.bias, c.res)):
        got = down(c.run(zeros_f32((T, 300)), None if bias is None else up_f32(bias),
                         None if res is None else up_f32(res), act))
        assert_epilogue(got, c.dots, bias, act, res, act)


def test_against_the_oracle(dev):
    c = Case(fm.QUANT_Q6_K, 700, 1024, 37)
    got = down(c.run(zeros_f32((37, 700)), up_f32(c.bias), up_f32(c.res), EPI_NONE))
    want, scale = oracle.rows_dot(c.w, c.rb, 700, c.x, 1024, 37, c.quant, 8)
    want, scale = want.reshape(37, 700), scale.reshape(37, 700)
    assert_rows_close(got, want + c.bias.astype(np.float64) + c.res, scale + np.abs(c.bias) + np.abs(c.res), "fused")


@pytest.mark.parametrize("T", [1, 2, 7, 40, 300])
def test_in_place_and_strided(dev, T):
    rows = 200
    c = Case(fm.QUANT_Q4_K, rows, 512, T)
    want = down(c.run(zeros_f32((T, rows)), up_f32(c.bias), up_f32(c.res), EPI_SILU))
    out = up_f32(c.res)
    c.run(out, up_f32(c.bias), out, EPI_SILU)
    assert np.array_equal(down(out), want)
    # out and residual as columns of one wider array, apart and the same
    wide = torch.full((T, 700), -3.0, device=dev)
    wide[:, 450:450 + rows] = up_f32(c.res)
    before = down(wide).copy()
    c.run(wide[:, 100:100 + rows], up_f32(c.bias), wide[:, 450:450 + rows], EPI_SILU, out_stride=700, res_stride=700)
    got = down(wide)
    assert np.array_equal(got[:, 100:100 + rows], want)
    before[:, 100:100 + rows] = want
    assert np.array_equal(got, before)  # the floats between the rows: as they were
    c.run(wide[:, 450:450 + rows], up_f32(c.bias), wide[:, 450:450 + rows], EPI_SILU, out_stride=700, res_stride=700)
    assert np.array_equal(down(wide)[:, 450:450 + rows], want)


def test_infinities_and_nan(dev):
    """Of the residual and the bias: they come out where they went in."""
    rows, T = 96, 6
    c = Case(fm.QUANT_Q5_K, rows, 256, T)
    bias, res = c.bias.copy(), c.res.copy()
    bias[3], bias[5], bias[7] = np.inf, -np.inf, np.nan
    res[2, 10], res[4, 11], res[5, 12] = np.inf, -np.inf, np.nan
    for act in ACTS:
        got = down(c.run(zeros_f32((T, rows)), up_f32(bias), up_f32(res), act))
        v = c.dots.astype(np.float64) + bias
        with np.errstate(invalid="ignore"):
            want = {EPI_NONE: v, EPI_RELU: np.maximum(v, 0)}.get(act, act64(act, v)) + res
        plain = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~plain & ~np.isnan(want)], want[~plain & ~np.isnan(want)].astype(np.float32))


def test_large_values_of_the_activations(dev):
    """Biases that take the activations to their ends: no NaN from exp's overflow."""
    rows, T = 64, 5
    c = Case(fm.QUANT_Q4_K, rows, 256, T)
    bias = np.repeat(np.array([-1e30, -1e4, -200, -90, 90, 200, 1e4, 1e30], np.float32), 8)
    for act in ACTS:
        got = down(c.run(zeros_f32((T, rows)), up_f32(bias), None, act))
        v = c.dots.astype(np.float64) + bias
        with np.errstate(over="ignore", invalid="ignore"):
            want = np.nan_to_num(act64(act, v), nan=0.0)
        assert np.isfinite(got).all()
        assert np.allclose(got, want, rtol=1e-5, atol=1e-30)


def test_unaligned_operands(dev):
    """xq and w at odd byte addresses, as pulsar_matmul_kq takes them."""
    for T in (1, 20, 64):
        c = Case(fm.QUANT_Q4_K, 130, 512, T)
        w, x = up(np.concatenate([np.zeros(3, np.uint8), c.w.reshape(-1)])), up(np.concatenate([np.zeros(5, np.uint8), c.x.reshape(-1)]))
        out = zeros_f32((T, 130))
        K.matmul_kq_fused(out, w[3:], x[5:], None, up_f32(c.res), 512, 130, T, c.rb, c.quant)
        want, scale = oracle.rows_dot(c.w, c.rb, 130, c.x, 512, T, c.quant, 8)
        assert_rows_close(down(out), want.reshape(T, 130) + c.res.astype(np.float64),
                          scale.reshape(T, 130) + np.abs(c.res), T)


@pytest.mark.parametrize("T", [1, 12, 64])
def test_captured(dev, T):
    rows = 260
    c = Case(fm.QUANT_Q4_K, rows, 512, T)
    bias, res, out = up_f32(c.bias), zeros_f32((T, rows)), zeros_f32((T, rows))
    torch.cuda.synchronize()
    graph = runtime.Graph.capture(lambda: c.run(out, bias, res, EPI_GELU))
    for i in range(3):
        fresh = (c.res * (i + 1)).astype(np.float32)
        res.copy_(torch.from_numpy(fresh))
        torch.cuda.synchronize()
        graph.launch()
        runtime.sync()
        assert_epilogue(down(out), c.dots, c.bias, EPI_GELU, fresh, i)


def test_own_stream(dev):
    c = Case(fm.QUANT_Q4_K, 300, 512, 4)
    want = down(c.run(zeros_f32((4, 300)), up_f32(c.bias), up_f32(c.res), EPI_NONE))
    out, bias, res = zeros_f32((4, 300)), up_f32(c.bias), up_f32(c.res)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    K.set_stream(stream)
    try:
        c.run(out, bias, res, EPI_NONE)
    finally:
        K.set_stream(None)
    stream.synchronize()
    assert np.array_equal(down(out), want)


@pytest.mark.parametrize("T", [4, 5, 33])
def test_rows_past_32_bit_offsets(dev, T):
    """Rows of out and residual so far apart that the last one starts behind 4 GiB."""
    c = Case(fm.QUANT_Q6_K, 100, 512, T)
    stride = 2**30 // (T - 1) + 7  # floats
    wide = torch.zeros((T - 1) * stride + 100, device=dev)
    out = wide.as_strided((T, 100), (stride, 1))
    out.copy_(up_f32(c.res))
    torch.cuda.synchronize()
    c.run(out, up_f32(c.bias), out, EPI_NONE, out_stride=stride, res_stride=stride)
    runtime.sync()
    assert_epilogue(down(out.contiguous()), c.dots, c.bias, EPI_NONE, c.res, T)
    assert not wide[100:stride].any()


def test_wrapper_refuses_short_tensors(dev):
    c = Case(fm.QUANT_Q4_K, 64, 256, 4)
    z = torch.zeros((4, 64), device=dev)
    for out, bias, res in ((z[:3], None, None), (z, z[0, :63], None), (z, None, z[:, :63]), (z, None, z[:3])):
        with pytest.raises(ValueError, match="has to"):
            c.run(out, bias, res, EPI_NONE)
    with pytest.raises(ValueError, match="f32"):
        c.run(z.double(), None, None, EPI_NONE)
    c.dw = c.dw.reshape(-1)[:-1]  # the last row, but for a byte
    with pytest.raises(ValueError, match="w has to"):
        c.run(z, None, None, EPI_NONE)
