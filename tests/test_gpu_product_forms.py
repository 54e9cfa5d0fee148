"""pulsar_matmul_kq_fused on each form of its two matrix-core kernels: the K split
(csrc/ksplit.hip) with token tiles of 16 to 64 and 8 or 16 waves, and the wide tile
(csrc/tile.hip) in its four shapes, for the seven formats that have both. Which
form a shape takes is read from its recorded launch, so a rule that sends it
elsewhere fails here rather than leave a form unchecked."""
import numpy as np
import pytest

from pulsar_amd import formats as fm
from tests.gpu_util import down, up_f32, zeros_f32
from tests.test_gpu_grouped_choice import launches
from tests.test_gpu_product_fused import ACTS, Case, assert_epilogue
from tests.test_gpu_tile import FORMATS

pytestmark = pytest.mark.gpu

# (rows, tokens, waves) of a block of the K split, (rows, tokens) of the tile
SPLIT = [(16, 16, 8), (16, 16, 16), (16, 32, 8), (16, 48, 8), (16, 64, 8)]
TILE = [(32, 32), (64, 64), (128, 64), (128, 128)]

# form, rows, values, tokens: ragged in rows and tokens, with fewer super-blocks
# than a K split has waves and with a remainder over them, one and more per K part
# of the tile
SHAPES = [(SPLIT[0], 145, 256, 20), (SPLIT[0], 301, 768, 21), (SPLIT[0], 18, 2304, 68), (SPLIT[1], 17, 4352, 68),
          (SPLIT[1], 90, 4864, 39), (SPLIT[2], 2049, 256, 17), (SPLIT[2], 2093, 2304, 17), (SPLIT[3], 2745, 256, 33),
          (SPLIT[3], 4090, 512, 45), (SPLIT[3], 2743, 2304, 35), (SPLIT[4], 2119, 256, 51), (SPLIT[4], 4090, 768, 61),
          (SPLIT[4], 2081, 2304, 49), (TILE[0], 12425, 256, 17), (TILE[0], 12371, 2304, 19), (TILE[1], 8247, 256, 33),
          (TILE[1], 8491, 2304, 37), (TILE[2], 11019, 256, 129), (TILE[2], 10954, 2304, 132), (TILE[3], 11093, 256, 321),
          (TILE[3], 11093, 1280, 325)]


def launch_of(form, rows, tokens):
    """Blocks, padded to the 8 XCDs, and threads of one."""
    r, t = form[:2]
    return (-(-rows // r) * -(-tokens // t) + 7) & ~7, 64 * form[2] if len(form) == 3 else 256


def test_every_form_is_listed():
    assert {s[0] for s in SHAPES} == {*SPLIT, *TILE}


@pytest.mark.parametrize("quant", FORMATS, ids=lambda q: fm.NAMES[q])
@pytest.mark.parametrize("form,rows,n,T", SHAPES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_form(dev, quant, form, rows, n, T):
    want = launch_of(form, rows, T)
    fits = [f for f in SPLIT if f[1] < T + 16] + TILE  # the K split takes no token tile wider than its tokens
    assert [launch_of(f, rows, T) for f in fits].count(want) == 1
    c = Case(quant, rows, n, T)
    bias, res, out = up_f32(c.bias), up_f32(c.res), zeros_f32((T, rows))
    nodes = launches(lambda: c.run(out, bias, res, ACTS[0]))
    assert [(k.grid[0], k.grid[1], k.grid[2], k.block[0]) for k in nodes] == [(want[0], 1, 1, want[1])]
    c.check_dots()
    act = ACTS[(rows + T + quant) % 5]
    got = down(c.run(out, bias, res, act))
    assert_epilogue(got, c.dots, c.bias, act, c.res, (quant, act))
    # in place, and no element but its own: the rows of a wider array
    wide = np.full((T, rows + 9), -3.0, np.float32)
    wide[:, 4:4 + rows] = c.res
    d = up_f32(wide)
    c.run(d[:, 4:4 + rows], bias, d[:, 4:4 + rows], act, out_stride=rows + 9, res_stride=rows + 9)
    wide[:, 4:4 + rows] = got
    assert np.array_equal(down(d), wide)
