"""What the wrappers of the routing with expert groups, the grouping by ids and the
product with an epilogue refuse of a tensor or a number, before the library is
called (no GPU: stand-ins for device tensors, whose memory is never read)."""
import pytest
import torch

from pulsar_amd import _lib
from pulsar_amd import kernels as K
from pulsar_amd.formats import DENSE_QUANTS, QUANT_A4_OK, QUANT_Q4_K, row_bytes


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    return _lib.load()


class Placed:
    """A tensor without memory, on the current device at an address of its own."""

    is_cuda = True
    taken = 0

    def __init__(self, shape, dtype):
        self.t = torch.empty(shape, dtype=dtype, device="meta")
        Placed.taken += 1
        self.address = Placed.taken << 32

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return K._device()

    def data_ptr(self):
        return self.address


I32, F32 = torch.int32, torch.float32
T, E, N = 3, 32, 4


def route(**change):
    a = dict(selected=Placed((T, N), I32), weights=Placed((T, N), F32), logits=Placed((T, E), F32),
             bias=Placed((E,), F32), n_expert=E, k_used=N, n_group=8, topk_group=2, group_top=2, score=0, renorm=True,
             weight_scale=1.0, n_tok=T)
    K.router_select_groups(**{**a, **change})


def group(**change):
    a = dict(gptrs=Placed((E, 6), torch.int64), starts=Placed((E + 1,), I32), pairs=Placed((T * N,), I32),
             slot_weights=Placed((T, N), F32), selected=Placed((T, N), I32), router_weights=Placed((T, N), F32),
             bank=K.ExpertBank(1 << 20, 2 << 20, 3 << 20, None, None, None, 64, 64, 64, 0, 0, 0), n_expert=E,
             shared=[], n_tok=T, k_used=N)
    K.moe_group_ids(**{**a, **change})


ROWS, COLS, RB = 64, 512, 288


def product(**change):
    a = dict(out=Placed((T, ROWS), F32), w=Placed((ROWS, RB), torch.uint8), xq=Placed((T, 584), torch.uint8),
             bias=Placed((ROWS,), F32), residual=Placed((T, ROWS), F32), in_dim=COLS, out_dim=ROWS, n_tok=T,
             row_bytes=RB, quant=QUANT_Q4_K)
    K.matmul_kq_fused(**{**a, **change})


@pytest.mark.parametrize("call", [route, group, product])
def test_sound_arguments_reach_the_library(call):
    """What the refusals below are told apart from: without a GPU the launch
    itself fails."""
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    with pytest.raises(K.KernelError):
        call()


def test_raw_bytes_reach_the_library():
    """A buffer of bytes stands for any array but the product's rows."""
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    raw = lambda n: Placed((n,), torch.uint8)  # noqa: E731
    for call in (lambda: route(selected=raw(4 * T * N), weights=raw(4 * T * N), logits=raw(4 * T * E), bias=raw(4 * E)),
                 lambda: group(gptrs=raw(48 * E), starts=raw(4 * E + 4), pairs=raw(4 * T * N), selected=raw(4 * T * N),
                               slot_weights=raw(4 * T * N), router_weights=raw(4 * T * N)),
                 lambda: product(bias=raw(4 * ROWS))):
        with pytest.raises(K.KernelError):
            call()


WIDE = [(route, "selected", (T, N), torch.int64), (route, "selected", (T, N), F32),
        (route, "weights", (T, N), torch.float64), (route, "weights", (T, 2 * N), torch.float16),
        (route, "logits", (T, E), torch.float64), (route, "logits", (T, 2 * E), torch.bfloat16),
        (route, "bias", (E,), torch.float64), (route, "bias", (E,), I32),
        (group, "starts", (E + 1,), torch.int64), (group, "pairs", (T * N,), torch.int64),
        (group, "selected", (T, N), torch.int64), (group, "selected", (T, 2 * N), torch.int16),
        (group, "router_weights", (T, N), torch.float64), (group, "router_weights", (T, 2 * N), torch.bfloat16),
        (group, "slot_weights", (T, N), torch.float64), (group, "slot_weights", (T, N), I32),
        (product, "bias", (ROWS,), torch.float64), (product, "bias", (2 * ROWS,), torch.float16),
        (product, "out", (T, ROWS), I32), (product, "residual", (T, ROWS), I32)]


@pytest.mark.parametrize("call,name,shape,dtype", WIDE)
def test_refuses_other_element_types(call, name, shape, dtype):
    """Large enough, but of a type whose bytes are not the operator's numbers:
    torch.topk's int64 ids are the case that a router meets."""
    with pytest.raises(ValueError, match=f"{name} has to be"):
        call(**{name: Placed(shape, dtype)})


@pytest.mark.parametrize("flag", [0, QUANT_A4_OK])
@pytest.mark.parametrize("quant", DENSE_QUANTS)
def test_refuses_weights_short_of_their_last_row(quant, flag):
    """With and without the flag beside the format's code, which the library
    takes off before it reads the rows."""
    rb = row_bytes(quant, COLS)
    xq = Placed((T, 584), torch.uint8)
    for n in ((ROWS - 1) * rb, ROWS * rb - 1):
        with pytest.raises(ValueError, match="w has to be contiguous"):
            product(w=Placed((n,), torch.uint8), xq=xq, row_bytes=rb, quant=quant | flag)


@pytest.mark.parametrize("call,names", [
    (route, ("n_expert", "k_used", "n_group", "topk_group", "group_top", "score", "n_tok")),
    (group, ("n_expert", "n_tok", "k_used")),
    (product, ("in_dim", "out_dim", "n_tok", "row_bytes", "quant", "act", "out_stride", "res_stride"))])
def test_refuses_numbers_that_the_library_would_read_as_others(call, names):
    """Below 0 every array is large enough, and the library reads the low bits:
    -1 token as 4294967295, 2^32 + 1 as one."""
    with_u64 = {"row_bytes", "out_stride", "res_stride"}
    for name in names:
        bits = 64 if name in with_u64 else 32
        for value in (-1, -256, 2**bits, 2**bits + 1):
            with pytest.raises(ValueError, match="out of range"):
                call(**{name: value})
            # of raw addresses too, whose sizes nothing else checks
            with pytest.raises(ValueError, match="out of range"):
                call(**{name: value, **{a: 1 << 40 for a in ("weights", "selected", "logits", "bias") if call is route},
                        **{a: 1 << 40 for a in ("out", "w", "xq") if call is product}})


# what an entry point says of overlapping arrays on stderr, before any launch
def refused(capfd, call):
    capfd.readouterr()
    with pytest.raises(K.KernelError):
        call()
    return "(overlap): invalid arguments" in capfd.readouterr().err


def apart(sizes):
    """Addresses in a row with nothing between the arrays."""
    at, out = 1 << 40, {}
    for name, n in sizes.items():
        out[name], at = at, at + n
    return out


def test_grouping_refuses_arrays_over_one_another(capfd):
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    shared = [(16, 32, 48)]
    slots = N + 1
    size = dict(gptrs=48 * (E + 1), starts=4 * (E + 2), pairs=4 * T * slots, slot_weights=4 * T * slots,
                selected=4 * T * N, router_weights=4 * T * N)
    at = apart(size)
    assert not refused(capfd, lambda: group(shared=shared, **at))
    outs = ("gptrs", "starts", "pairs", "slot_weights")
    for a in outs:
        for b in size:
            if b == a:
                continue
            for address in (at[b], at[b] + size[b] - 4, at[b] - size[a] + 4):
                call = {**at, a: address}
                assert refused(capfd, lambda: group(shared=shared, **call)), (a, b, address - at[b])
    # a copy onto itself is none where every slot is the router's
    own = {**at, "slot_weights": at["router_weights"]}
    assert not refused(capfd, lambda: group(shared=[], **own))
    assert refused(capfd, lambda: group(shared=shared, **own))
    # weights that are not asked for are not read
    own = {**at, "slot_weights": 0, "router_weights": at["pairs"]}
    assert not refused(capfd, lambda: group(shared=shared, **own))


def test_routing_refuses_outputs_over_its_arrays(capfd):
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    size = dict(selected=4 * T * N, weights=4 * T * N, logits=4 * T * E, bias=4 * E)
    at = apart(size)
    assert not refused(capfd, lambda: route(**at))
    for a in ("selected", "weights"):
        for b in size:
            if b == a:
                continue
            for address in (at[b], at[b] + size[b] - 4, at[b] - size[a] + 4):
                call = {**at, a: address}
                assert refused(capfd, lambda: route(**call)), (a, b, address - at[b])
    at["bias"] = 0
    assert not refused(capfd, lambda: route(**at))
    at["bias"] = at["logits"] + 4 * E  # a row of the logits, which is only read
    assert not refused(capfd, lambda: route(**at))
