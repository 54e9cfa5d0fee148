"""pulsar_matmul_i8, every tile of its matrix-core kernels on purpose: tiles that are whole
and that are not, rows of fewer steps than a tile keeps on their way, of one more, and of
many. Which kernel a call takes is read from a captured graph, so that a shape that has
come to another tile is seen. The products in 64 bits on the device."""
import ctypes
import math
import re

import pytest
import torch

from pulsar_amd import kernels as K
from pulsar_amd import runtime
from pulsar_amd.formats import EPI_GELU, EPI_NONE, EPI_RELU, EPI_SIGMOID, EPI_SILU, TYPE_BF16, TYPE_F16, TYPE_F32
from tests.test_gpu_grouped_choice import launches
from tests.test_gpu_rows8 import HALF, NAMES, TINY, TORCH

pytestmark = pytest.mark.gpu
KINDS = [TYPE_F32, TYPE_F16, TYPE_BF16]
ACTS = [EPI_SILU, EPI_GELU, EPI_RELU, EPI_SIGMOID, EPI_NONE]


def kernel_of(call):
    """The name of the one kernel that a call launches (nothing runs)."""
    node, = launches(call)
    name = runtime._hip().hipKernelNameRefByPtr
    name.argtypes, name.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_char_p
    return name(node.func, runtime.STREAM_PER_THREAD).decode()


def tile_of(name):
    """(MF, BM, BN, WM, WN, WK, KB, S, DMA) of a mangled i8_tile_kernel."""
    return tuple(int(v) for v in re.findall(r"L[jb](\d+)E", name.split("I8TileI")[1]))


def tile(mf, bm, bn, wm, wn, wk, kb, s, dma=1):
    return mf, bm, bn, wm, wn, wk, kb, s, dma


# tile: (channels, tokens) of whole tiles and of others, row lengths. Rows of whole 16
# bytes: 2 steps of KB values, S + 1, 11, and 17 with a part of one; of tiles that split
# the row over WK groups so many for a group
TILES = [
    (tile(16, 16, 16, 1, 1, 8, 128, 4), [(4096, 16), (1000, 55)], [1024, 2064, 5120, 11280]),
    (tile(16, 32, 32, 2, 1, 4, 128, 4), [(4096, 64), (1500, 130)], [1040, 2560, 5632, 8720]),
    (tile(16, 32, 32, 2, 2, 1, 128, 4), [(4096, 64), (1500, 130), (17000, 32), (17003, 27)], [256, 640]),
    (tile(16, 32, 32, 2, 2, 1, 128, 4), [(17024, 32), (17003, 27)], [1408, 2064]),
    (tile(16, 32, 64, 2, 2, 2, 128, 4), [(4096, 128), (2011, 250)], [512, 1280, 2816, 4240]),
    (tile(32, 64, 64, 2, 2, 2, 128, 4), [(4096, 256), (2000, 490)], [2064, 2560, 2816, 4240]),
    (tile(32, 64, 64, 2, 2, 1, 128, 4), [(4096, 256), (2000, 490)], [256, 640, 1408, 2032]),
    (tile(32, 64, 64, 2, 2, 1, 128, 4), [(33024, 64), (33003, 50)], [256, 640, 1408, 2064]),
    (tile(16, 64, 128, 2, 4, 1, 128, 4), [(4096, 512), (4090, 500)], [256, 640, 1408, 2064]),
    (tile(16, 128, 128, 4, 2, 1, 128, 4), [(4096, 1024), (4090, 1000)], [256, 640, 1408, 2064]),
    (tile(32, 128, 256, 2, 4, 1, 128, 3), [(4352, 1152), (4345, 1100)], [128, 256, 512, 1408, 2064]),
    (tile(16, 256, 256, 2, 4, 1, 64, 4), [(8192, 2048), (28600, 500)], [128, 320, 704, 1040]),
]
# rows at any byte
ODD_TILES = [
    (tile(16, 16, 16, 1, 1, 8, 128, 2, 0), [(4096, 16), (1000, 55)], [1025, 2063, 5119, 11278]),
    (tile(16, 32, 32, 2, 2, 2, 128, 4, 0), [(4096, 64), (1500, 130)], [511, 1281, 2815, 4239]),
    (tile(16, 32, 64, 2, 2, 2, 128, 4, 0), [(4096, 128), (2011, 250)], [511, 1281, 2815, 4239]),
    (tile(16, 64, 64, 2, 4, 1, 128, 4, 0), [(4096, 256), (2000, 490)], [255, 641, 1407, 2063]),
    (tile(16, 64, 128, 2, 4, 1, 128, 4, 0), [(4096, 512), (4090, 500), (33024, 64), (33003, 50)], [255, 641, 1407, 2063]),
    (tile(16, 128, 128, 4, 4, 1, 128, 4, 0), [(4096, 1024), (4090, 1000)], [255, 641, 1407, 2063]),
    (tile(32, 128, 128, 4, 2, 1, 128, 2, 0), [(4352, 1152), (4345, 1100)], [127, 255, 385, 1407, 2063]),
]
CASES = [(t, n, T, k) for t, shapes, dims in TILES + ODD_TILES for n, T in shapes for k in dims]
IDS = [f"{'' if t[8] else 'odd_'}{t[1]}x{t[2]}x{t[5]}-{n}x{k}-{T}" for t, n, T, k in CASES]
cases = pytest.mark.parametrize("want,rows,T,cols", CASES, ids=IDS)


def gen(dev, *seed):
    g = torch.Generator(device=dev)
    g.manual_seed(hash(seed) % 2**31)
    return g


def codes(g, n, cols, most, dev):
    return torch.randint(-most, most, (n, cols), generator=g, device=dev, dtype=torch.int8)


def dots(x, w):
    """Exact: sums of whole numbers below 2^53."""
    return torch.mm(x.double(), w.double().t().contiguous())


def act64(act, v):
    if act == EPI_SILU:
        return v * torch.sigmoid(v)
    if act == EPI_GELU:
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v**3)))
    if act == EPI_RELU:
        return v.clamp_min(0.0)
    return torch.sigmoid(v) if act == EPI_SIGMOID else v


def takes(want, call):
    name = kernel_of(call)
    assert "i8_tile_kernel" in name and tile_of(name) == want, (name, want)


@cases
def test_sums_are_exact(dev, want, rows, T, cols):
    """Scales of 1: sums of up to 2^12 cols, below 2^24, come out as they are."""
    most = 64 if cols < 4096 else 32
    g = gen(dev, rows, T, cols)
    x, w = codes(g, T, cols, most, dev), codes(g, rows, cols, most, dev)
    ones, out = torch.ones(max(rows, T), device=dev), torch.full((T, rows), 0.5, device=dev)
    torch.cuda.synchronize()
    call = lambda: K.matmul_i8(out, w, ones, x, ones, None, None, cols, rows, T)  # noqa: E731
    takes(want, call)
    call()
    torch.cuda.synchronize()
    assert torch.equal(out.double(), dots(x, w))


@pytest.mark.parametrize("kind", KINDS, ids=NAMES.get)
@cases
def test_epilogue(dev, want, rows, T, cols, kind):
    """Bias, activation and residual; codes to the ends of their range. Roundings of 2^-24,
    as tests/test_gpu_product_i8.py counts them: of the sum and its two products and the
    bias 4.5 of v, an activation's slope of 1.13 on them, its own 8 of its value and 4 of 1,
    the residual's addition; then the rows' type."""
    g = gen(dev, rows, T, cols, kind)
    x, w = codes(g, T, cols, 128, dev), codes(g, rows, cols, 128, dev)
    sx = torch.rand(T, generator=g, device=dev) + 0.5
    sw = (torch.rand(rows, generator=g, device=dev) + 0.5) / (5476 * math.sqrt(cols))
    bias = 0.5 * torch.randn(rows, generator=g, device=dev)
    res = torch.randn((T, rows), generator=g, device=dev).to(TORCH[kind])
    act = ACTS[(rows + T + cols + kind) % 5]
    out = torch.full((T, rows), 77.0, dtype=TORCH[kind], device=dev)
    torch.cuda.synchronize()
    call = lambda: K.matmul_i8(out, w, sw, x, sx, bias, res, cols, rows, T, act, kind)  # noqa: E731
    takes(want, call)
    call()
    torch.cuda.synchronize()
    v = dots(x, w) * sx[:, None].double() * sw.double()
    b = v + bias.double()
    a = act64(act, b)
    exact = a + res.double()
    tol = 2.0**-24 * (4.5 * v.abs() + 1.2 * b.abs() + 8 * a.abs() + 4 * (act != EPI_NONE) + exact.abs())
    if kind != TYPE_F32:
        tol = tol + HALF[kind] * (exact.abs() + tol) + TINY[kind]
    bad = ~((out.double() - exact).abs() <= tol)
    assert not bad.any(), (want, act, int(bad.sum()), bad.nonzero()[:4].tolist())
