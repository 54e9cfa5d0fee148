"""The activations of pulsar_matmul_kq_fused alone: weights whose scales are 0, so
that every dot is 0 and each output is the activation of its bias, in 64 bits."""
import numpy as np
import pytest

from pulsar_amd import formats as fm
from pulsar_amd import kernels as K
from pulsar_amd.formats import EPI_GELU, EPI_NONE, EPI_RELU, EPI_SIGMOID, EPI_SILU, row_bytes
from tests.gpu_util import down, up, up_f32, zeros_f32

pytestmark = pytest.mark.gpu
ULP = 2.0**-23  # of a value, at most


def values():
    rng = np.random.default_rng(1)
    v = [rng.uniform(-105, 105, 6000), rng.standard_normal(3000) * 3, np.linspace(-1, 1, 2001),
         rng.standard_normal(500) * 1e-6, 10.0 ** rng.uniform(-38, 38, 400) * rng.choice([-1, 1], 400),
         [0.0, -0.0, 88.5, -88.5, 89.0, -89.0, 87.3, -87.3, 104.0, -104.0, 3e38, -3e38]]
    return np.concatenate(v).astype(np.float32)


# the lane kernels, the K split, the 16-row kernel and the wide tile at these rows
@pytest.mark.parametrize("T", [1, 4, 12, 20, 64, 140])
@pytest.mark.parametrize("act", [EPI_NONE, EPI_SILU, EPI_GELU, EPI_RELU, EPI_SIGMOID])
def test_activation_of_the_bias(dev, act, T):
    """sigmoid: e^-x within 2 units in the last place, the sum's half, the
    reciprocal's 1, each of a part of the value that is no larger; below 2^-126,
    where the reciprocal has no value, 0. SiLU: the product's half more. GELU: v x
    sigmoid(y), y from 5 roundings of half a unit each, which move sigmoid(y) by
    (1 - sigmoid(y)) |y| of itself."""
    v = values()
    rows, n = len(v), 256
    rb = row_bytes(fm.QUANT_Q4_K, n)
    w = np.random.default_rng(2).integers(0, 256, (rows, rb), dtype=np.uint8)
    w[:, :4] = 0  # both scales
    x = np.zeros((T, 292), np.uint8)
    x[:, :4] = np.array([1.0], np.float32).view(np.uint8)
    out = zeros_f32((T, rows))
    K.matmul_kq_fused(out, up(w), up(x), up_f32(v), None, n, rows, T, rb, fm.QUANT_Q4_K, act)
    got, d = down(out).astype(np.float64), v.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore", under="ignore"):
        if act == EPI_NONE:
            want, tol = d, 0 * d
        elif act == EPI_RELU:
            want, tol = np.maximum(d, 0), 0 * d
        else:
            y = np.sqrt(8 / np.pi) * (d + 0.044715 * d**3) if act == EPI_GELU else d
            s = np.where(y >= 0, 1 / (1 + np.exp(-y)), np.exp(np.minimum(y, 0)) / (1 + np.exp(np.minimum(y, 0))))
            by = 1.0 if act == EPI_SIGMOID else d
            want = np.where(s == 0, 0.0, by * s)
            steps = 3.5 + (0.5 if act != EPI_SIGMOID else 0)
            if act == EPI_GELU:
                steps = steps + np.where(s < 1, (1 - s) * np.abs(y) * 2.5, 0)
            tol = steps * ULP * np.abs(want) + np.abs(by) * 2.0**-126
    assert np.isfinite(got).all()
    worst = np.abs(got - want) - tol
    assert (worst <= 0).all(), (v[np.argmax(worst.max(0))], got[:, np.argmax(worst.max(0))][0], want[np.argmax(worst.max(0))])
