"""What the norm to 8-bit rows, the int8 quantizer and the int8 product refuse: numbers and
tensors in the wrappers, numbers and overlaps in the library, all before any launch (no
GPU: addresses and stand-ins that are never read)."""
import pytest
import torch

from pulsar_amd import _lib
from pulsar_amd import kernels as K
from pulsar_amd.formats import ACT_SILU, ACT_SWIGLU_OAI, EPI_SIGMOID, ROWS_I8, ROWS_Q8_K, TYPE_BF16, TYPE_F16, TYPE_F32
from tests.test_operator_arguments import Placed

A = [0x10000000 * (i + 1) for i in range(8)]  # addresses far apart
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    return _lib.load()


NORM = dict(q=A[0], scales=A[1], y=A[2], sum_out=A[3], x=A[4], residual=A[5], gain=A[6], dim=300, n_rows=3, eps=1e-5,
            type=TYPE_F32, fmt=ROWS_I8)
QUANT = dict(q=A[0], scales=A[1], x=A[2], up=A[3], dim=300, n_rows=3, act_op=ACT_SILU, type=TYPE_F32)
PRODUCT = dict(out=A[0], w=A[1], w_scales=A[2], x=A[3], x_scales=A[4], bias=A[5], residual=A[6], in_dim=300, out_dim=64,
               n_tok=3, act=0, type=TYPE_F32)


def norm(**change):
    K.rms_norm_q8(**{**NORM, **change})


def quant(**change):
    K.quantize_i8(**{**QUANT, **change})


def product(**change):
    K.matmul_i8(**{**PRODUCT, **change})


def said(capfd, call):
    """What the refusal of the call prints; empty where it came to a launch."""
    capfd.readouterr()
    with pytest.raises(K.KernelError):
        call()
    err = capfd.readouterr().err
    return err if "invalid arguments" in err else ""


@pytest.mark.parametrize("change", [
    dict(x=0), dict(gain=0), dict(q=0, scales=0, y=0), dict(q=0), dict(scales=0), dict(dim=0), dict(dim=2**24 + 1),
    dict(n_rows=0), dict(n_rows=2**31), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(fmt=2),
    dict(fmt=ROWS_Q8_K), dict(fmt=ROWS_Q8_K, scales=0, q_stride=300), dict(q=0, scales=0, q_stride=300),
    dict(x_stride=299), dict(res_stride=299), dict(sum_stride=299), dict(q_stride=299), dict(x_stride=2**32),
    dict(q_stride=2**40)])
def test_norm_refuses(capfd, change):
    assert "rms_norm_q8" in said(capfd, lambda: norm(**change))


@pytest.mark.parametrize("change", [
    dict(q=0), dict(scales=0), dict(x=0), dict(dim=0), dict(dim=2**24 + 1), dict(n_rows=0), dict(n_rows=2**31),
    dict(act_op=1), dict(act_op=3), dict(up=0, act_op=ACT_SWIGLU_OAI), dict(x_stride=299), dict(up_stride=299),
    dict(q_stride=299), dict(up_stride=2**32)])
def test_quantize_refuses(capfd, change):
    assert "quantize_i8" in said(capfd, lambda: quant(**change))


@pytest.mark.parametrize("change", [
    dict(out=0), dict(w=0), dict(w_scales=0), dict(x=0), dict(x_scales=0), dict(in_dim=0), dict(in_dim=131072),
    dict(out_dim=0), dict(out_dim=2**31), dict(n_tok=0), dict(n_tok=2**31), dict(act=EPI_SIGMOID + 1), dict(w_stride=299),
    dict(x_stride=299), dict(out_stride=63), dict(res_stride=63), dict(w_stride=2**23 + 1), dict(x_stride=2**23 + 1),
    dict(out_stride=2**32), dict(res_stride=2**32)])
def test_product_refuses(capfd, change):
    assert "matmul_i8" in said(capfd, lambda: product(**change))


@pytest.mark.parametrize("call,names,wide", [
    (norm, ("dim", "n_rows", "type", "fmt"), ("x_stride", "res_stride", "sum_stride", "q_stride")),
    (quant, ("dim", "n_rows", "act_op", "type"), ("x_stride", "up_stride", "q_stride")),
    (product, ("in_dim", "out_dim", "n_tok", "act", "type"), ("w_stride", "x_stride", "out_stride", "res_stride"))])
def test_refuses_numbers_that_the_library_would_read_as_others(call, names, wide):
    for name in names + wide:
        bits = 64 if name in wide else 32
        for value in (-1, -256, 2**bits, 2**bits + 1):
            with pytest.raises(ValueError, match="out of range"):
                call(**{name: value})
    with pytest.raises(ValueError, match="out of range"):
        call(type=3)


def apart(sizes):
    """Addresses in a row with nothing between the arrays."""
    at, out = 1 << 40, {}
    for name, n in sizes.items():
        out[name], at = at, at + n
    return out


@pytest.mark.parametrize("kind,size", [(TYPE_F32, 4), (TYPE_F16, 2), (TYPE_BF16, 2)])
@pytest.mark.parametrize("call,args,outs", [
    (norm, dict(q="b", scales="r", y="e", sum_out="e", x="e", residual="e", gain="g"), ("q", "scales", "y", "sum_out")),
    (quant, dict(q="b", scales="r", x="e", up="e"), ("q", "scales")),
    (product, dict(out="o", w="w", w_scales="c", x="b", x_scales="r", bias="c", residual="o"), ("out",))])
def test_refuses_outputs_over_its_arrays(capfd, call, args, outs, kind, size):
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    n = dict(b=3 * 300, r=3 * 4, e=3 * 300 * size, g=300 * 4, o=3 * 64 * size, w=64 * 300, c=64 * 4)
    sizes = {name: n[what] for name, what in args.items()}
    at = apart(sizes)
    assert not said(capfd, lambda: call(type=kind, **at))
    for a in outs:
        for b in sizes:
            if b == a:
                continue
            same = (a, b) in (("sum_out", "x"), ("sum_out", "residual"), ("out", "residual"))
            for address in (at[b], at[b] + sizes[b] - size, at[b] - sizes[a] + size):
                allowed = same and address == at[b]
                got = said(capfd, lambda: call(type=kind, **{**at, a: address}))
                assert bool(got) != allowed and (allowed or "(overlap)" in got), (a, b, address - at[b])


def test_rows_in_place_have_one_stride(capfd):
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    for change in (dict(sum_out=A[4]), dict(sum_out=A[5]), dict(sum_out=A[4], x_stride=310, sum_stride=310),
                   dict(sum_out=A[5], residual=A[5], x=A[5])):
        assert not said(capfd, lambda: norm(**change))
    for change in (dict(sum_out=A[4], x_stride=310), dict(sum_out=A[5], sum_stride=310),
                   dict(sum_out=A[4], residual=A[4] + 4)):
        assert "(overlap)" in said(capfd, lambda: norm(**change))
    for change in (dict(residual=A[0]), dict(residual=A[0], out_stride=70, res_stride=70),
                   dict(residual=A[0] + 4 * 64, out_stride=128, res_stride=128)):  # columns side by side
        assert not said(capfd, lambda: product(**change))
    for change in (dict(residual=A[0], out_stride=70), dict(residual=A[0] + 4),
                   dict(residual=A[0] + 4 * 63, out_stride=128, res_stride=128)):
        assert "(overlap)" in said(capfd, lambda: product(**change))
    # an array that is left out overlaps nothing
    assert not said(capfd, lambda: norm(sum_out=0, y=A[5], residual=0))
    assert not said(capfd, lambda: norm(fmt=ROWS_Q8_K, scales=0))


# ---------------------------------------------------------------- tensors --

def norm_t(**change):
    a = dict(q=Placed((3, 300), I8), scales=Placed((3,), F32), y=Placed((3, 300), F32), sum_out=Placed((3, 300), F32),
             x=Placed((3, 300), F32), residual=Placed((3, 300), F32), gain=Placed((300,), F32))
    norm(**{**a, **change})


def quant_t(**change):
    a = dict(q=Placed((3, 300), I8), scales=Placed((3,), F32), x=Placed((3, 300), F32), up=Placed((3, 300), F32))
    quant(**{**a, **change})


def product_t(**change):
    a = dict(out=Placed((3, 64), F32), w=Placed((64, 300), I8), w_scales=Placed((64,), F32), x=Placed((3, 300), I8),
             x_scales=Placed((3,), F32), bias=Placed((64,), F32), residual=Placed((3, 64), F32))
    product(**{**a, **change})


@pytest.mark.parametrize("call", [norm_t, quant_t, product_t])
def test_sound_tensors_reach_the_library(call):
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    with pytest.raises(K.KernelError):
        call()


@pytest.mark.parametrize("call,name,shape", [
    (norm_t, "q", (3, 300)), (norm_t, "y", (3, 300)), (norm_t, "sum_out", (3, 300)), (norm_t, "x", (3, 300)),
    (norm_t, "residual", (3, 300)), (norm_t, "scales", (3,)), (norm_t, "gain", (300,)), (quant_t, "q", (3, 300)),
    (quant_t, "x", (3, 300)), (quant_t, "up", (3, 300)), (quant_t, "scales", (3,)), (product_t, "out", (3, 64)),
    (product_t, "w", (64, 300)), (product_t, "x", (3, 300)), (product_t, "residual", (3, 64)),
    (product_t, "w_scales", (64,)), (product_t, "x_scales", (3,)), (product_t, "bias", (64,))])
def test_refuses_other_types_and_short_tensors(call, name, shape):
    with pytest.raises(ValueError, match=f"{name} has to be"):
        call(**{name: Placed(shape, torch.float64)})
    for other in (BF16, F16, torch.int32):  # where large enough
        with pytest.raises(ValueError, match=f"{name} has to be"):
            call(**{name: Placed((2 * shape[0], *shape[1:]), other)})
    mine = I8 if name in ("q", "w") or (call is product_t and name == "x") else F32
    with pytest.raises(ValueError, match=f"{name} has to"):
        call(**{name: Placed((shape[0] - 1, *shape[1:]), mine)})


@pytest.mark.parametrize("kind,mine", [(TYPE_F16, F16), (TYPE_BF16, BF16)])
def test_rows_are_of_the_type_they_are_said_to_be(kind, mine):
    for call, names in ((norm_t, ("x", "residual", "y", "sum_out")), (quant_t, ("x", "up")),
                        (product_t, ("out", "residual"))):
        shape = (3, 64) if call is product_t else (3, 300)
        good = {n: Placed(shape, mine) for n in names}
        if not torch.cuda.is_available():
            with pytest.raises(K.KernelError):
                call(type=kind, **good)
        for n in names:
            with pytest.raises(ValueError, match=f"{n} has to be {'f16' if mine is F16 else 'bf16'}"):
                call(type=kind, **{**good, n: Placed(shape, F32)})


def test_blocks_want_room():
    x = {n: Placed((3, 300), F32) for n in ("y", "sum_out", "x", "residual")}
    for rows, ok in ((3, True), (2, False)):
        q = Placed((rows * 2 * 292,), torch.uint8)
        with pytest.raises(K.KernelError if ok and not torch.cuda.is_available() else ValueError):
            if ok and torch.cuda.is_available():
                raise ValueError
            norm_t(q=q, scales=None, fmt=ROWS_Q8_K, **x)


def test_columns_of_a_wider_array():
    """A view has to have the stride that it is said to have."""
    wide = torch.empty((3, 700), dtype=F32, device="meta")

    class View(Placed):
        def __init__(self, t):
            self.t = t
            Placed.taken += 1
            self.address = Placed.taken << 32

    ok = View(wide[:, 5:305])
    if not torch.cuda.is_available():
        with pytest.raises(K.KernelError):
            quant_t(x=ok, x_stride=700)
    for stride in (0, 300, 701):
        with pytest.raises(ValueError, match="x has to hold"):
            quant_t(x=ok, x_stride=stride)
    with pytest.raises(ValueError, match="x has to hold"):
        quant_t(x=View(wide[:, ::2][:, :300]), x_stride=700)
    with pytest.raises(ValueError, match="x has to hold"):
        quant_t(x=View(wide[:2, 5:305]), x_stride=700)


def test_refuses_host_tensors():
    t = torch.zeros(4096)
    for call, name in ((norm, "x"), (norm, "gain"), (quant, "x"), (product, "out"), (product, "w_scales")):
        with pytest.raises(ValueError, match="host tensor"):
            call(**{name: t})


def test_product_refuses_more_tiles_than_a_grid(capfd):
    """2^27 tokens by 2^31 - 1 channels, out where no other array is."""
    call = lambda: product(out=1 << 62, residual=0, out_dim=2**31 - 1, n_tok=2**27, type=TYPE_BF16)  # noqa: E731
    assert "matmul_i8 (size)" in said(capfd, call)
