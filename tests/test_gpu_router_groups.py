"""pulsar_router_select_groups against a plain 64-bit implementation."""
import math

import numpy as np
import pytest
import torch

from pulsar_amd import kernels as K
from pulsar_amd import runtime
from pulsar_amd.formats import SCORE_SIGMOID, SCORE_SOFTMAX
from tests.gpu_util import down, up_f32

pytestmark = pytest.mark.gpu
BIG = float(np.finfo(np.float32).max)


def want_route(logits, bias, k, groups, top_groups, group_top, score, renorm, scale):
    """ids, weights and each weight's bound. The kernel may form a weight in
    f32: the logits' difference to the maximum (|l - m| steps of exp's
    argument), an exp, a sum of up to 1024 terms in a tree, a division, the sum
    of k weights, a division and the scale: at most k + 40 + |l - m| roundings
    of 2^-24."""
    T, E = logits.shape
    l = logits.astype(np.float64)
    b = np.zeros(E) if bias is None else bias.astype(np.float64)
    ids, wts, tol = np.full((T, k), -1, np.int32), np.zeros((T, k)), np.zeros((T, k))
    size = E // groups
    for t in range(T):
        part = ~(np.isnan(l[t]) | (l[t] == -np.inf))
        v = np.clip(l[t], -BIG, BIG)
        m = v[part].max() if part.any() else 0.0
        s = np.zeros(E)
        with np.errstate(over="ignore", under="ignore"):
            if score == SCORE_SOFTMAX:
                s[part] = np.exp(v[part] - m)
                s[part] /= s[part].sum() if part.any() else 1.0
            else:
                e = np.exp(-np.abs(v[part]))
                s[part] = np.where(v[part] >= 0, 1.0, e) / (1.0 + e)
        c = s + b
        ok = part & ~(np.isnan(b) | (b == -np.inf))
        stand = []
        for g in range(groups):
            best = sorted((c[e] for e in range(g * size, (g + 1) * size) if ok[e]), reverse=True)[:group_top]
            if best:
                stand.append((-sum(best), g))
        kept = {g for _, g in sorted(stand)[:top_groups]}
        order = sorted((-c[e], e) for e in range(E) if ok[e] and e // size in kept)[:k]
        win = [e for _, e in order]
        ids[t, :len(win)] = win
        w = s[win]
        if renorm and len(win):
            total = w.sum()
            total = max(total, 2.0**-14) if score == SCORE_SIGMOID else total
            w = w / total if total > 0 else 0 * w
        wts[t, :len(win)] = w * scale
        away = np.abs(v[win] - m) if score == SCORE_SOFTMAX else 0.0
        tol[t, :len(win)] = np.abs(w * scale) * (k + 40 + away) * 2.0**-24 + 2.0**-149
    return ids, wts, tol


def run(dev, logits, bias, k, groups, top_groups, group_top, score, renorm, scale):
    T, E = logits.shape
    ids = torch.full((T, k), -7, dtype=torch.int32, device=dev)
    w = torch.full((T, k), math.nan, device=dev)
    K.router_select_groups(ids, w, up_f32(logits), None if bias is None else up_f32(bias), E, k, groups, top_groups,
                           group_top, score, renorm, scale, T)
    return down(ids), down(w)


def check(dev, logits, bias, *how):
    ids, w = run(dev, logits, bias, *how)
    want, wts, tol = want_route(logits, bias, *how)
    bad = np.argwhere(ids != want)
    assert bad.size == 0, (bad[:4].tolist(), ids[bad[0][0]].tolist(), want[bad[0][0]].tolist())
    err = np.abs(w - wts)
    assert (err <= tol).all(), (err.max(), np.argwhere(err > tol)[:4].tolist())
    return ids, w


# experts, k, groups, kept groups
SHAPES = [(1, 1, 1, 1), (8, 2, 4, 2), (32, 4, 1, 1), (64, 6, 8, 3), (91, 13, 1, 1), (104, 13, 8, 2), (128, 8, 1, 1),
          (160, 6, 8, 3), (182, 7, 14, 7), (240, 3, 8, 7), (256, 8, 8, 4), (256, 8, 1, 1), (256, 64, 8, 8),
          (45, 4, 5, 2), (99, 5, 9, 4), (100, 6, 2, 1), (300, 9, 12, 5), (390, 5, 13, 6), (480, 8, 15, 7),
          (483, 6, 7, 3), (500, 16, 10, 4), (256, 8, 16, 5), (256, 16, 32, 9), (256, 8, 2, 1), (384, 8, 1, 1), (392, 7, 8, 3), (512, 10, 4, 2),
          (1000, 16, 8, 3), (1024, 64, 64, 11)]


@pytest.mark.parametrize("experts,k,groups,kept", SHAPES)
@pytest.mark.parametrize("score", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_shapes(dev, experts, k, groups, kept, score):
    rng = np.random.default_rng(experts * 7 + groups)
    for T, group_top, with_bias, renorm in ((1, 1, True, True), (5, 2, False, False), (67, 2, True, False),
                                            (300, 1, False, True)):
        logits = (1.5 * rng.standard_normal((T, experts)) - 0.5).astype(np.float32)
        bias = (0.1 * rng.standard_normal(experts)).astype(np.float32) if with_bias else None
        check(dev, logits, bias, k, groups, kept, group_top, score, renorm, 2.5)


@pytest.mark.parametrize("experts,k,groups,kept", [(256, 8, 8, 4), (128, 8, 1, 1), (96, 5, 3, 2)])
@pytest.mark.parametrize("score", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_many_tokens(dev, experts, k, groups, kept, score):
    rng = np.random.default_rng(experts + score)
    logits = (1.5 * rng.standard_normal((4099, experts)) - 1.0).astype(np.float32)
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    check(dev, logits, bias, k, groups, kept, 2, score, True, 1.0)
    check(dev, logits, None, k, groups, kept, 1, score, False, 1.0)


@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3), (32, 20)])
@pytest.mark.parametrize("score", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_next_to_a_border(dev, groups, kept, score):
    """Scores that f32 rounds to one value, or whose order it swaps, and exact
    ties, which go to the lower id."""
    rng = np.random.default_rng(groups)
    experts, T = 256, 96
    logits = np.zeros((T, experts), np.float32)
    for t in range(T):
        kind = t % 6
        base = np.float32(rng.uniform(-3, 3))
        if kind == 0:  # steps of one unit in the last place
            logits[t] = base + np.float32(np.spacing(base)) * rng.integers(-3, 4, experts)
        elif kind == 1:  # a few values, many ties
            logits[t] = rng.integers(-2, 3, experts)
        elif kind == 2:  # all equal
            logits[t] = base
        elif kind == 3:  # saturated: 1 - s below an f32 step
            logits[t] = rng.uniform(14, 19, experts)
        elif kind == 4:  # far below 1
            logits[t] = rng.uniform(-60, -50, experts)
        else:
            logits[t] = rng.standard_normal(experts) * 1e-5
    none = None
    near = (np.float32(0.5) + np.float32(2.0**-25) * rng.integers(0, 4, experts)).astype(np.float32)
    for bias in (none, near):
        for group_top in (1, 2):
            check(dev, logits, bias, 8, groups, kept, group_top, score, True, 1.0)


@pytest.mark.parametrize("experts,groups,kept", [(256, 8, 4), (120, 6, 2), (256, 16, 15), (60, 2, 1)])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("score", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_groups_next_to_a_border(dev, experts, groups, kept, group_top, score):
    """Groups whose scores are those of another group, in another order, or a few
    units in the last place beside them."""
    rng = np.random.default_rng(experts + group_top)
    T, size = 120, experts // groups
    logits = (1.5 * rng.standard_normal((T, groups, size)) - 1.0).astype(np.float32)
    for t in range(T):
        a, b = rng.permutation(groups)[:2]
        logits[t, b] = rng.permutation(logits[t, a])
        best = np.argsort(logits[t, b])[-group_top:]
        ulps = [0, 1, -1, 3, -20][t % 5]
        logits[t, b, best[0]] += ulps * np.spacing(np.abs(logits[t, b, best[0]]))
        if t % 3 == 1:  # several of the group's best next to one another
            logits[t, b, rng.permutation(size)[:6]] = logits[t, b, best[-1]] * np.float32(1 + 2.0**-22)
        if t % 8 == 7:  # all of them
            logits[t] = logits[t, a]
    logits = logits.reshape(T, experts)
    same = np.full(experts, 0.25, np.float32)
    near = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    for bias in (None, same, near, near - np.float32(3), same - np.float32(2)):
        check(dev, logits, bias, 6, groups, kept, group_top, score, True, 1.0)


@pytest.mark.parametrize("groups,kept,group_top", [(1, 1, 1), (8, 2, 2), (8, 8, 1), (4, 1, 2), (32, 3, 2)])
@pytest.mark.parametrize("score", [SCORE_SIGMOID, SCORE_SOFTMAX])
@pytest.mark.parametrize("experts", [64, 256, 512])
def test_masks(dev, groups, kept, group_top, score, experts):
    """Logits and biases that take experts out, rows and groups that leave
    none, the type's lowest and infinite values."""
    rng = np.random.default_rng(experts + groups)
    T = 40
    logits = (2 * rng.standard_normal((T, experts))).astype(np.float32)
    for t in range(T):
        at = rng.random(experts) < rng.choice([0.1, 0.5, 0.97])
        logits[t, at] = [np.nan, -np.inf, -BIG, np.inf, BIG, -30000.0][t % 6]
    logits[3], logits[9], logits[10], logits[11] = np.nan, -np.inf, -BIG, np.inf
    logits[12, 1:] = np.nan
    logits[13, :experts // groups] = -np.inf
    logits[14, :-1] = -np.inf
    bias = (0.3 * rng.standard_normal(experts)).astype(np.float32)
    gone = bias.copy()
    gone[rng.random(experts) < 0.3] = -np.inf
    gone[rng.random(experts) < 0.1] = np.nan
    gone[rng.random(experts) < 0.02] = np.inf
    for b in (None, bias, gone):
        for renorm in (True, False):
            check(dev, logits, b, 4, groups, kept, group_top, score, renorm, 1.5)


def test_equals_router_select(dev):
    """One group, sigmoid and a bias, renormalised: pulsar_router_select's mode
    0; softmax: its mode 1 (the same ids, weights within the f32 roundings)."""
    rng = np.random.default_rng(3)
    T, E, k = 130, 256, 8
    logits, bias = rng.standard_normal((T, E)).astype(np.float32), (0.1 * rng.standard_normal(E)).astype(np.float32)
    for mode, b in ((0, bias), (1, np.zeros(E, np.float32))):
        ids, w = run(dev, logits, b, k, 1, 1, 1, mode, True, 1.0)
        sel, rw = torch.zeros((T, k), dtype=torch.int32, device=dev), torch.zeros((T, k), device=dev)
        K.router_select(sel, rw, up_f32(logits), up_f32(b), E, k, 1.0, T, mode, 0)
        assert (down(sel) == ids).all()
        assert np.allclose(down(rw), w, rtol=(k + 45) * 2.0**-23, atol=0)


def test_neighbours_untouched_and_repeatable(dev):
    rng = np.random.default_rng(4)
    T, E, k = 33, 256, 8
    x = up_f32(rng.standard_normal((T, E)).astype(np.float32))
    got = []
    for _ in range(2):
        ids = torch.full((T + 2, k), -9, dtype=torch.int32, device=dev)
        w = torch.full((T + 2, k), -9.0, device=dev)
        K.router_select_groups(ids[1:-1], w[1:-1], x, None, E, k, 8, 4, 2, SCORE_SIGMOID, True, 1.0, T)
        got.append((down(ids), down(w)))
    for ids, w in got:
        assert (ids[[0, -1]] == -9).all() and (w[[0, -1]] == -9.0).all()
    assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all()


def test_captured(dev):
    rng = np.random.default_rng(5)
    T, E, k = 70, 256, 8
    x = torch.zeros((T, E), device=dev)
    ids, w = torch.zeros((T, k), dtype=torch.int32, device=dev), torch.zeros((T, k), device=dev)
    torch.cuda.synchronize()
    how = (E, k, 8, 4, 2, SCORE_SIGMOID, True, 1.0, T)
    graph = runtime.Graph.capture(lambda: K.router_select_groups(ids, w, x, None, *how))
    for _ in range(3):
        fresh = rng.standard_normal((T, E)).astype(np.float32)
        x.copy_(torch.from_numpy(fresh))
        torch.cuda.synchronize()
        graph.launch()
        runtime.sync()
        want, wts = run(dev, fresh, None, k, 8, 4, 2, SCORE_SIGMOID, True, 1.0)
        assert (down(ids) == want).all() and (down(w) == wts).all()


def test_own_stream(dev):
    rng = np.random.default_rng(6)
    T, E, k = 70, 256, 8
    logits = rng.standard_normal((T, E)).astype(np.float32)
    want, wts = run(dev, logits, None, k, 8, 4, 2, SCORE_SIGMOID, True, 1.0)
    x, ids, w = up_f32(logits), torch.zeros((T, k), dtype=torch.int32, device=dev), torch.zeros((T, k), device=dev)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    K.set_stream(stream)
    try:
        K.router_select_groups(ids, w, x, None, E, k, 8, 4, 2, SCORE_SIGMOID, True, 1.0, T)
    finally:
        K.set_stream(None)
    stream.synchronize()
    assert (down(ids) == want).all() and (down(w) == wts).all()


@pytest.mark.parametrize("groups", [8, 32])
def test_logits_past_32_bit_offsets(dev, groups):
    T, E, k = 2**21 + 5, 512, 4
    x = torch.empty((T, E), device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(7))
    ids, w = torch.full((T, k), -7, dtype=torch.int32, device=dev), torch.full((T, k), math.nan, device=dev)
    torch.cuda.synchronize()
    how = (k, groups, 3, 2, SCORE_SOFTMAX, True, 1.0)
    K.router_select_groups(ids, w, x, None, E, *how, T)
    runtime.sync()
    at = [0, 2**20 - 1, 2**21 - 1, 2**21, T - 1]
    want, wts, tol = want_route(down(x[at]), None, *how)
    assert (down(ids[at]) == want).all()
    assert (np.abs(down(w[at]) - wts) <= tol).all()
    assert int(ids.min()) >= 0


def test_wrapper_refuses_short_tensors(dev):
    z = torch.zeros(4 * 32, device=dev)
    ids = torch.zeros(4 * 4, dtype=torch.int32, device=dev)
    how = (32, 4, 8, 2, 2, SCORE_SIGMOID, True, 1.0)
    for bad in ((ids[:-1], z, z, None), (ids, z[:15], z, None), (ids, z, z[:-1], None), (ids, z, z, z[:31]),
                (ids, z, torch.zeros((32, 4), device=dev).T, None)):
        with pytest.raises(ValueError, match="has to be contiguous"):
            K.router_select_groups(*bad, *how, 4)
