"""The weights of pulsar_router_select_groups, to the last bit that f32 can hold."""
import numpy as np
import pytest
import torch

from pulsar_amd.formats import SCORE_SIGMOID, SCORE_SOFTMAX
from tests.test_gpu_router_groups import run, want_route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spread", [0.01, 1.5, 8.0])
@pytest.mark.parametrize("experts,k,groups,kept", [(8, 2, 1, 1), (32, 4, 1, 1), (128, 8, 1, 1), (256, 8, 8, 4),
                                                   (483, 6, 7, 3), (512, 16, 4, 4), (512, 10, 32, 9), (1000, 4, 1, 1)])
def test_softmax_without_renormalisation(dev, experts, k, groups, kept, spread):
    """A weight e^(l - m) / z is rounded to f32 once: half a step, 2^-24 of it, and
    2^-32 for a sum whose terms are each within 2^-33 of themselves, an exp, the
    quotient and the scale in 64 bits. A sum in f32 is off by several steps. Logits
    next to one another give z all its terms."""
    rng = np.random.default_rng(experts)
    for T, group_top, with_bias, scale in ((1, 1, False, 1.0), (300, 1, False, 2.5), (130, 2, False, 1.0),
                                           (130, 1, True, 1.0), (131, 2, True, 0.3)):
        logits = (spread * rng.standard_normal((T, experts)) - 0.5).astype(np.float32)
        logits[rng.random((T, experts)) < 0.05] = -np.inf
        logits[:, :k] = np.where(np.isinf(logits[:, :k]), np.float32(0), logits[:, :k])
        bias = (0.1 * rng.standard_normal(experts)).astype(np.float32) if with_bias else None
        how = (k, groups, kept, group_top, SCORE_SOFTMAX, False)
        ids, w = run(dev, logits, bias, *how, scale)
        want, wts, _ = want_route(logits, bias, *how, float(np.float32(scale)))
        assert np.array_equal(ids, want)
        err = np.abs(w - wts)
        bound = wts * (2.0**-24 + 2.0**-32) + 2.0**-149
        assert (err <= bound).all(), float((err / np.maximum(wts, 1e-300)).max() * 2**24)


@pytest.mark.parametrize("experts,groups,kept", [(64, 8, 2), (1000, 1, 1)])
@pytest.mark.parametrize("score", [SCORE_SIGMOID, SCORE_SOFTMAX])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("scale", [np.inf, -np.inf, np.nan])
def test_empty_slots_under_any_scale(dev, experts, groups, kept, score, renorm, scale):
    """A slot that no expert is left for is -1 with weight 0, times whatever."""
    logits = np.full((5, experts), -np.inf, np.float32)
    logits[1, 3], logits[2, [1, 2]], logits[3] = 1.0, 0.5, np.nan
    for bias in (None, np.zeros(experts, np.float32)):
        ids, w = run(dev, logits, bias, 4, groups, kept, 1, score, renorm, scale)
        assert (ids[[0, 3, 4]] == -1).all() and ids[1].tolist() == [3, -1, -1, -1] and ids[2].tolist() == [1, 2, -1, -1]
        assert (w[ids == -1] == 0.0).all(), w
        won = w[ids >= 0]
        assert np.isnan(won).all() if np.isnan(scale) else (won == scale).all()
