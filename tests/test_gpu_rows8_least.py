"""pulsar_quantize_i8 of gated combines below what 64 bits hold with all their bits: gates
so far below 0 that e^gate leaves the normal numbers. The formula in 80 bits."""
import numpy as np
import pytest
import torch

from pulsar_amd import kernels as K
from pulsar_amd.formats import ACT_SILU, ACT_SWIGLU_OAI, TYPE_BF16, TYPE_F32
from tests.gpu_util import down, up_f32
from tests.test_gpu_rows8 import NAMES, by_type, codes64, dev_rows, glu64, quant_check, rounded

pytestmark = pytest.mark.gpu
assert np.finfo(np.longdouble).minexp < -16000, "numbers far below those of 64 bits"


def quantized(g, u, op, kind):
    rows, dim = g.shape
    q, sc = torch.full((rows, dim), 99, dtype=torch.int8, device="cuda:0"), up_f32(np.full(rows, 9))
    K.quantize_i8(q, sc, dev_rows(g, kind), dev_rows(u, kind), dim, rows, op, kind)
    return q, sc


def check(g, u, op, kind):
    """Codes of rows whose scale is below f32's numbers. The argument of up to 127 is off by
    2^-42 as elsewhere; a clamped combine's 1.702 gate, of up to 745, is rounded to 2^-53 of
    it, which e^ makes 2^-43.4 of a value, 2^-42.4 of a quotient: 2^-35.4 of an argument."""
    q, sc = quantized(g, u, op, kind)
    v = glu64(g.astype(np.longdouble), u.astype(np.longdouble), op)
    top = np.abs(v).max(1, keepdims=True)
    assert ((top > 0) & (top < 1e-60)).all() and not down(sc).any()
    got, want = down(q).astype(np.int64), codes64(v, top)
    t = np.abs(v) / top * 127.0
    border = np.abs(t - np.floor(t) - 0.5) <= (2.0**-39 if op == ACT_SILU else 2.0**-35)
    bad = (got != want) & ~border
    assert not bad.any(), (g.shape, NAMES[kind], op, np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])
    assert (np.abs(got).max(1) == 127).all()


# rows that a block holds, and longer ones
@pytest.mark.parametrize("dim", [1, 300, 5000, 17000, 33000])
@pytest.mark.parametrize("op", [ACT_SILU, ACT_SWIGLU_OAI])
@by_type
def test_least_values(dev, kind, op, dim):
    rng = np.random.default_rng(dim + kind)
    a = 1.0 if op == ACT_SILU else 1.702
    g = -(705 + 25 * rng.random((5, dim))) / a
    g[2, 1:] = -(730 + 400 * rng.random(dim - 1)) / a  # most of the row below 64 bits altogether
    half = max(dim // 2, 1)
    g[3, half:] = -(360 + 900 * rng.random(dim - half)) / a
    u = rng.standard_normal((5, dim)) + np.copysign(0.1, rng.standard_normal((5, dim)))
    u[:, 0] = 1.0
    if dim > 1:
        g[4, 1::2], u[4, 1::2] = 3.0, 0.0 if op == ACT_SILU else -1.0  # values of 0 among them
    check(rounded(g, kind), rounded(u, kind), op, kind)


@pytest.mark.parametrize("dim", [300, 17000])
@pytest.mark.parametrize("kind", [TYPE_F32, TYPE_BF16], ids=NAMES.get)
def test_least_sigmoids_under_large_ups(dev, kind, dim):
    """Values inside the range of 64 bits whose e^gate is not."""
    rng = np.random.default_rng(dim)
    g = rounded(-(700 + 44 * rng.random((4, dim))), kind)
    u = rounded(1e36 * rng.standard_normal((4, dim)), kind)
    check(g, u, ACT_SILU, kind)


@by_type
def test_below_64_bits_altogether(dev, kind):
    """e^gate is 0 in 64 bits: rows of zeros. Beside them a row that is not."""
    g = np.full((3, 700), -800.0)
    g[1] = np.linspace(-800, 5, 700)
    u = np.ones((3, 700))
    g, u = rounded(g, kind), rounded(u, kind)
    q, sc = quantized(g, u, ACT_SILU, kind)
    assert not down(q)[[0, 2]].any() and not down(sc)[[0, 2]].any()
    quant_check(glu64(g, u, ACT_SILU)[1:2], q[1:2], sc[1:2], NAMES[kind])
