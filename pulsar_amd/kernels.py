"""Host-side mirror of the reference's kernel wrappers (crates/kernels/src/lib.rs).

Each function has the reference wrapper's name and argument order, takes
device buffers (torch CUDA tensors or raw device addresses as ints) and raises
KernelError(op) where the Rust wrapper returns Err(Error(op)) (the C entry
point returned 0; crates/kernels/src/lib.rs:212-218). Launches are
asynchronous on the calling thread's per-thread default stream (the
reference's --default-stream=per-thread); call runtime.sync() or
torch.cuda.synchronize() (the reference's kernels::sync) before reading
results on the host.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from .formats import BLOCK_LAYOUT, EXPERT_PTRS_BYTES, QUANT_A4_OK


class KernelError(RuntimeError):
    """A kernel entry point returned 0 (crates/kernels/src/lib.rs:8-20)."""

    def __init__(self, op: str):
        super().__init__(f"hip kernel op failed: {op}")
        self.op = op


def _ptr(buf) -> int:
    if buf is None:
        return 0
    if isinstance(buf, int):
        return buf
    if hasattr(buf, "data_ptr"):
        if not buf.is_cuda:
            raise ValueError("device buffer expected (got a host tensor)")
        return buf.data_ptr()
    raise TypeError(f"cannot take a device address of {type(buf)!r}")


def _check(ret: int, op: str) -> None:
    if ret == 0:
        raise KernelError(op)


def quantize_q8_k(out, x, in_dim: int, n_rows: int) -> None:
    _check(_lib.load().pulsar_quantize_q8_K(_ptr(out), _ptr(x), in_dim, n_rows), "quantize_q8_k")


def matmul_kq(out, w, xq, in_dim: int, out_dim: int, n_tok: int, row_bytes: int, quant: int) -> None:
    _check(
        _lib.load().pulsar_matmul_kq(_ptr(out), _ptr(w), _ptr(xq), in_dim, out_dim, n_tok, row_bytes, quant),
        "matmul_kq",
    )


# element types of an array of f32 or of 32-bit integers: its own, or raw bytes
_F32 = (_lib.torch.float32, _lib.torch.uint8) if _lib.torch else ()
_I32 = (_lib.torch.int32, _lib.torch.uint32, _lib.torch.uint8) if _lib.torch else ()


def _room(buf, nbytes: int, op: str, what: str, device: int, types=None) -> int:
    """The device address of `buf`, which the launch uses the first nbytes
    bytes of; a tensor has to be contiguous, that large, on the current device
    and of `types` (a raw address is the caller's word for all four)."""
    if buf is None or not hasattr(buf, "data_ptr"):
        return _ptr(buf)
    if buf.get_device() != device:
        _misplaced(buf, op, what)
    if buf.nbytes < nbytes or not buf.is_contiguous():
        raise ValueError(f"{op}: {what} has to be contiguous and hold {nbytes} bytes")
    if types is not None and buf.dtype not in types:
        _other_type(buf, op, what, types)
    return buf.data_ptr()


def _other_type(buf, op: str, what: str, types) -> None:
    """Of a wider type it is large enough, but its bytes are other numbers."""
    raise ValueError(f"{op}: {what} has to be {'f32' if types is _F32 else 'int32'} (got {buf.dtype})")


def _out_of_range(op: str) -> None:
    """A number that ctypes would cut to its low bits, -1 to the largest one."""
    raise ValueError(f"{op}: a size or code is out of range")


def _misplaced(buf, op: str, what: str) -> None:
    _ptr(buf)  # a host tensor
    raise ValueError(f"{op}: {what} is not on the current device")


def _device() -> int:
    """The current device, -2 (no tensor's) before the GPU is first used."""
    cuda = _lib.torch.cuda
    return cuda.current_device() if cuda.is_initialized() else -2


def _rows(buf, n_rows: int, dim: int, stride: int, op: str, what: str, device: int) -> int:
    """The device address of n_rows rows of dim floats, `stride` floats apart.
    A tensor may be a view of columns of a wider array: it has to be f32 [..,
    dim] with that stride, or contiguous and large enough."""
    if buf is None or not hasattr(buf, "data_ptr"):
        return _ptr(buf)
    if buf.get_device() != device:
        _misplaced(buf, op, what)
    if buf.dtype != _lib.torch.float32:
        raise ValueError(f"{op}: {what} has to be f32 (got {buf.dtype})")
    if buf.is_contiguous():
        ok = buf.numel() >= (n_rows - 1) * stride + dim
    else:
        ok = (buf.dim() == 2 and buf.shape[0] >= n_rows and buf.shape[1] >= dim and buf.stride(1) == 1
              and buf.stride(0) == stride)
    if not ok:
        raise ValueError(f"{op}: {what} has to hold {n_rows} rows of {dim} f32 values {stride} apart")
    return buf.data_ptr()


def matmul_kq_fused(out, w, xq, bias, residual, in_dim: int, out_dim: int, n_tok: int, row_bytes: int, quant: int,
                    act: int = 0, out_stride: int = 0, res_stride: int = 0) -> None:
    """matmul_kq with its epilogue in the same launch: out[t] = act(W x_t +
    bias) + residual[t] (formats.EPI_* codes; bias and residual may be None).
    Strides in floats, 0 for packed rows; residual may be out itself."""
    op, dev = "matmul_kq_fused", _device()
    if (in_dim | out_dim | n_tok | quant | act) >> 32 or (row_bytes | out_stride | res_stride) >> 64:
        _out_of_range(op)
    block, block_bytes = BLOCK_LAYOUT.get(quant & ~QUANT_A4_OK, (1, 0))
    w_bytes = (out_dim - 1) * row_bytes + in_dim // block * block_bytes
    xq_bytes, so, sr = n_tok * -(-in_dim // 256) * 292, out_stride or out_dim, res_stride or out_dim
    _check(
        _lib.load().pulsar_matmul_kq_fused(
            _rows(out, n_tok, out_dim, so, op, "out", dev), _room(w, w_bytes, op, "w", dev),
            _room(xq, xq_bytes, op, "xq", dev), _room(bias, 4 * out_dim, op, "bias", dev, _F32),
            _rows(residual, n_tok, out_dim, sr, op, "residual", dev), in_dim, out_dim, n_tok, row_bytes, quant, act,
            out_stride, res_stride),
        op,
    )


def moe_pair_swiglu(mid, ptrs, weights, x, in_dim: int, mid_dim: int, n_used: int, n_tok: int,
                    row_bytes: int, quant: int, act_op: int) -> None:
    _check(
        _lib.load().pulsar_moe_pair_swiglu(_ptr(mid), _ptr(ptrs), _ptr(weights), _ptr(x), in_dim, mid_dim,
                                           n_used, n_tok, row_bytes, quant, act_op),
        "moe_pair_swiglu",
    )


def moe_down(out, ptrs, mid, mid_dim: int, out_dim: int, n_used: int, n_tok: int, row_bytes: int,
             quant: int) -> None:
    _check(
        _lib.load().pulsar_moe_down(_ptr(out), _ptr(ptrs), _ptr(mid), mid_dim, out_dim, n_used, n_tok,
                                    row_bytes, quant),
        "moe_down",
    )


def _capacity(pairs) -> int:
    """The most pairs a CSR over `pairs` can list (a raw address: unknown)."""
    if not hasattr(pairs, "data_ptr"):
        return 0xFFFFFFFF
    return min(pairs.numel() * pairs.element_size() // 4, 0xFFFFFFFF)


def moe_pair_swiglu_grouped(mid, gptrs, starts, pairs, weights, xq, in_dim: int, mid_dim: int,
                            n_used: int, n_group: int, row_bytes: int, quant: int, act_op: int) -> None:
    _check(
        _lib.load().pulsar_moe_pair_swiglu_grouped_bounded(_ptr(mid), _ptr(gptrs), _ptr(starts), _ptr(pairs),
                                                           _ptr(weights), _ptr(xq), in_dim, mid_dim, n_used,
                                                           n_group, row_bytes, quant, act_op, _capacity(pairs)),
        "moe_pair_swiglu_grouped",
    )


def moe_down_grouped(partial, gptrs, starts, pairs, midq, mid_dim: int, out_dim: int, n_used: int,
                     n_group: int, row_bytes: int, quant: int) -> None:
    _check(
        _lib.load().pulsar_moe_down_grouped_bounded(_ptr(partial), _ptr(gptrs), _ptr(starts), _ptr(pairs),
                                                    _ptr(midq), mid_dim, out_dim, n_used, n_group, row_bytes,
                                                    quant, _capacity(pairs)),
        "moe_down_grouped",
    )


def moe_slot_sum(out, partial, out_dim: int, n_used: int, n_tok: int) -> None:
    _check(_lib.load().pulsar_moe_slot_sum(_ptr(out), _ptr(partial), out_dim, n_used, n_tok), "moe_slot_sum")


def moe_down_bias(out, ptrs, weights, out_dim: int, n_used: int, n_tok: int) -> None:
    _check(
        _lib.load().pulsar_moe_down_bias(_ptr(out), _ptr(ptrs), _ptr(weights), out_dim, n_used, n_tok),
        "moe_down_bias",
    )


def add_bias_rows(x, bias, dim: int, rows: int) -> None:
    _check(_lib.load().pulsar_add_bias_rows(_ptr(x), _ptr(bias), dim, rows), "add_bias_rows")


def router_select(selected, weights, logits, bias, n_expert: int, k_used: int, weight_scale: float,
                  n_tok: int, mode: int, n_shexp: int) -> None:
    _check(
        _lib.load().pulsar_router_select(_ptr(selected), _ptr(weights), _ptr(logits), _ptr(bias), n_expert,
                                         k_used, weight_scale, n_tok, mode, n_shexp),
        "router_select",
    )


def router_select_groups(selected, weights, logits, bias, n_expert: int, k_used: int, n_group: int, topk_group: int,
                         group_top: int, score: int, renorm: bool, weight_scale: float, n_tok: int) -> None:
    """Top-k of the experts of the topk_group best of n_group expert groups
    (a group's score: its group_top largest score + bias; formats.SCORE_*),
    the weights the winners' scores, renormalised if renorm, times weight_scale."""
    op, dev = "router_select_groups", _device()
    if (n_expert | k_used | n_group | topk_group | group_top | score | n_tok) >> 32:
        _out_of_range(op)
    _check(
        _lib.load().pulsar_router_select_groups(
            _room(selected, 4 * n_tok * k_used, op, "selected", dev, _I32),
            _room(weights, 4 * n_tok * k_used, op, "weights", dev, _F32),
            _room(logits, 4 * n_tok * n_expert, op, "logits", dev, _F32),
            _room(bias, 4 * n_expert, op, "bias", dev, _F32), n_expert, k_used, n_group, topk_group, group_top, score,
            int(bool(renorm)), weight_scale, n_tok),
        op,
    )


def matmul_f32(out, w, x, in_dim: int, out_dim: int, n_tok: int) -> None:
    _check(_lib.load().pulsar_matmul_f32(_ptr(out), _ptr(w), _ptr(x), in_dim, out_dim, n_tok), "matmul_f32")


class ExpertBank(ctypes.Structure):
    """pulsar_expert_bank (include/pulsar_moe.h): expert e's projection starts
    at base + e * stride bytes, its bias at b_base + e * b_stride floats."""

    _fields_ = [
        ("gate", ctypes.c_void_p), ("up", ctypes.c_void_p), ("down", ctypes.c_void_p),
        ("gate_b", ctypes.c_void_p), ("up_b", ctypes.c_void_p), ("down_b", ctypes.c_void_p),
        ("gate_stride", ctypes.c_uint64), ("up_stride", ctypes.c_uint64), ("down_stride", ctypes.c_uint64),
        ("gate_b_stride", ctypes.c_uint64), ("up_b_stride", ctypes.c_uint64), ("down_b_stride", ctypes.c_uint64),
    ]


class _Ptrs6(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("gate", "up", "down", "gate_b", "up_b", "down_b")]


def moe_route_ptrs(ptrs, slot_weights, selected, router_weights, bank: ExpertBank, n_expert: int,
                   shared, n_tok: int, k_used: int) -> None:
    """Device-side pointer build (no reference counterpart entry point; it
    replaces the host build of crates/engine/src/lib.rs:8255-8344).
    `shared` is a list of (gate, up, down[, biases]) address tuples."""
    shared = list(shared or [])
    arr = (_Ptrs6 * max(1, len(shared)))()
    for i, e in enumerate(shared):
        e = tuple(e) + (0,) * (6 - len(e))
        arr[i] = _Ptrs6(*[int(v) or None for v in e])
    _check(
        _lib.load().pulsar_moe_route_ptrs(_ptr(ptrs), _ptr(slot_weights), _ptr(selected), _ptr(router_weights),
                                          ctypes.byref(bank), n_expert, ctypes.cast(arr, ctypes.c_void_p),
                                          len(shared), n_tok, k_used),
        "moe_route_ptrs",
    )


def moe_group_csr(gptrs, starts, pairs, ptrs, n_tok: int, n_used: int, max_groups: int) -> None:
    """Device-side CSR by expert (replaces crates/engine/src/lib.rs:8357-8392)."""
    _check(
        _lib.load().pulsar_moe_group_csr(_ptr(gptrs), _ptr(starts), _ptr(pairs), _ptr(ptrs), n_tok, n_used,
                                         max_groups),
        "moe_group_csr",
    )


def moe_group_ids(gptrs, starts, pairs, slot_weights, selected, router_weights, bank: ExpertBank, n_expert: int,
                  shared, n_tok: int, k_used: int) -> None:
    """The CSR by expert of a chunk of any length from the router's ids: group e
    is bank expert e, then one group per shared slot; the grouped stages take it
    with n_group = n_expert + len(shared), in two calls where that is above 1024
    (gptrs and starts of the groups behind 1024 in the second): one leaves their
    fast path. slot_weights (None: left out) gets router_weights and the shared
    slots' ones."""
    op, dev = "moe_group_ids", _device()
    if (n_expert | n_tok | k_used) >> 32:
        _out_of_range(op)
    arr, n_shared = _shared_array(shared)
    groups, slots = n_expert + n_shared, k_used + n_shared
    gptrs = _room(gptrs, EXPERT_PTRS_BYTES * groups, op, "gptrs", dev)
    starts = _room(starts, 4 * (groups + 1), op, "starts", dev, _I32)
    pairs = _room(pairs, 4 * n_tok * slots, op, "pairs", dev, _I32)
    weights = _room(slot_weights, 4 * n_tok * slots, op, "slot_weights", dev)
    selected = _room(selected, 4 * n_tok * k_used, op, "selected", dev, _I32)
    router_weights = _room(router_weights, 4 * n_tok * k_used, op, "router_weights", dev, _F32)
    if hasattr(slot_weights, "data_ptr") and slot_weights.dtype not in _F32:  # behind every size
        _other_type(slot_weights, op, "slot_weights", _F32)
    _check(_lib.load().pulsar_moe_group_ids(gptrs, starts, pairs, weights, selected, router_weights,
                                            ctypes.byref(bank), n_expert, arr, n_shared, n_tok, k_used), op)


def moe_slot_sum_bias(out, partial, ptrs, weights, out_dim: int, n_used: int, n_tok: int) -> None:
    """moe_slot_sum + moe_down_bias in one launch (bit-identical)."""
    _check(_lib.load().pulsar_moe_slot_sum_bias(_ptr(out), _ptr(partial), _ptr(ptrs), _ptr(weights), out_dim,
                                                n_used, n_tok), "moe_slot_sum_bias")


def moe_route_group(selected, weights, ptrs, slot_weights, gptrs, starts, pairs, logits, router_bias,
                    n_expert: int, k_used: int, weight_scale: float, softmax_mode: int, bank: "ExpertBank", shared,
                    n_tok: int, max_groups: int) -> None:
    """router_select (modes 0/1) + moe_route_ptrs + moe_group_csr in one launch."""
    arr, n_shared = _shared_array(shared)
    _check(_lib.load().pulsar_moe_route_group(
        _ptr(selected), _ptr(weights), _ptr(ptrs), _ptr(slot_weights), _ptr(gptrs), _ptr(starts), _ptr(pairs),
        _ptr(logits), _ptr(router_bias), n_expert, k_used, weight_scale, softmax_mode, ctypes.byref(bank),
        ctypes.cast(arr, ctypes.c_void_p), n_shared, n_tok, max_groups), "moe_route_group")


def moe_route(selected, weights, ptrs, slot_weights, active, logits, router_bias, n_expert: int, k_used: int,
              weight_scale: float, softmax_mode: int, bank: "ExpertBank", shared, n_tok: int) -> None:
    """router_select (modes 0/1) + moe_route_ptrs in one launch (equal
    outputs), plus `active` (uint32 [2 + n_expert]): the count of distinct
    selected experts, the count of NULL slots, the expert ids in order of
    first appearance in (token, slot) order."""
    arr, n_shared = _shared_array(shared)
    _check(_lib.load().pulsar_moe_route(
        _ptr(selected), _ptr(weights), _ptr(ptrs), _ptr(slot_weights), _ptr(active), _ptr(logits), _ptr(router_bias),
        n_expert, k_used, weight_scale, softmax_mode, ctypes.byref(bank), ctypes.cast(arr, ctypes.c_void_p),
        n_shared, n_tok), "moe_route")


def moe_pair_swiglu_experts(mid, selected, active, slot_weights, xq, bank: "ExpertBank", n_expert: int, shared,
                            n_tok: int, k_used: int, in_dim: int, mid_dim: int, row_bytes: int, quant: int,
                            act_op: int) -> None:
    """The grouped gate/up stage with one group per selected expert, grouped
    on the device from moe_route's outputs (rows equal
    moe_pair_swiglu_grouped's, for Q3_K, IQ4_XS and very wide rows where both
    have short groups or neither has; unrouted slots get rows of 0)."""
    arr, n_shared = _shared_array(shared)
    _check(_lib.load().pulsar_moe_pair_swiglu_experts(
        _ptr(mid), _ptr(selected), _ptr(active), _ptr(slot_weights), _ptr(xq), ctypes.byref(bank), n_expert,
        ctypes.cast(arr, ctypes.c_void_p), n_shared, n_tok, k_used, in_dim, mid_dim, row_bytes, quant, act_op),
        "moe_pair_swiglu_experts")


def moe_down_experts(partial, selected, active, midq, bank: "ExpertBank", n_expert: int, shared, n_tok: int,
                     k_used: int, mid_dim: int, out_dim: int, row_bytes: int, quant: int) -> None:
    """The grouped down stage with one group per selected expert; writes
    every row of partial (0 for unrouted slots)."""
    arr, n_shared = _shared_array(shared)
    _check(_lib.load().pulsar_moe_down_experts(
        _ptr(partial), _ptr(selected), _ptr(active), _ptr(midq), ctypes.byref(bank), n_expert,
        ctypes.cast(arr, ctypes.c_void_p), n_shared, n_tok, k_used, mid_dim, out_dim, row_bytes, quant),
        "moe_down_experts")


def _shared_array(shared):
    shared = [tuple(map(int, e)) for e in shared or ()]
    return (_Ptrs6 * max(1, len(shared)))(*shared), len(shared)


# ---- fused decode layer (extensions; each equals the separate calls it replaces)

def router_logits_q8(logits, xq, x, w_r, bias, in_dim: int, n_expert: int, n_tok: int) -> None:
    """matmul_f32 [+ add_bias_rows] + quantize_q8_k(x) in one launch."""
    _check(_lib.load().pulsar_router_logits_q8(_ptr(logits), _ptr(xq), _ptr(x), _ptr(w_r), _ptr(bias), in_dim,
                                               n_expert, n_tok), "router_logits_q8")


def moe_pair_routed(mid, ptrs, slot_weights, selected, weights, logits, router_bias, n_expert: int, k_used: int,
                    weight_scale: float, softmax_mode: int, bank: ExpertBank, shared, xq, in_dim: int,
                    mid_dim: int, n_tok: int, row_bytes: int, quant: int, act_op: int) -> None:
    """router_select (modes 0/1) + moe_route_ptrs + moe_pair_swiglu in one launch."""
    arr, n_shared = _shared_array(shared)
    _check(_lib.load().pulsar_moe_pair_routed(
        _ptr(mid), _ptr(ptrs), _ptr(slot_weights), _ptr(selected), _ptr(weights), _ptr(logits), _ptr(router_bias),
        n_expert, k_used, weight_scale, softmax_mode, ctypes.byref(bank), ctypes.cast(arr, ctypes.c_void_p),
        n_shared, _ptr(xq), in_dim, mid_dim, n_tok, row_bytes, quant, act_op), "moe_pair_routed")


def moe_down_f32(out, ptrs, slot_weights, mid, mid_dim: int, out_dim: int, n_used: int, n_tok: int,
                 row_bytes: int, quant: int, add_bias: bool) -> None:
    """quantize_q8_k(mid) + moe_down [+ moe_down_bias] in one launch."""
    _check(_lib.load().pulsar_moe_down_f32(_ptr(out), _ptr(ptrs), _ptr(slot_weights), _ptr(mid), mid_dim, out_dim,
                                           n_used, n_tok, row_bytes, quant, int(bool(add_bias))), "moe_down_f32")


def moe_down_biased(out, ptrs, weights, midq, mid_dim: int, out_dim: int, n_used: int, n_tok: int, row_bytes: int,
                    quant: int) -> None:
    """moe_down + moe_down_bias in one launch."""
    _check(_lib.load().pulsar_moe_down_biased(_ptr(out), _ptr(ptrs), _ptr(weights), _ptr(midq), mid_dim, out_dim,
                                              n_used, n_tok, row_bytes, quant), "moe_down_biased")


def moe_selftest() -> bool:
    """pulsar_moe_selftest (klib:1563): the MoE path per format against host mirrors."""
    return bool(_lib.load().pulsar_moe_selftest())


def router_selftest() -> bool:
    """pulsar_router_selftest (klib:1559)."""
    return bool(_lib.load().pulsar_router_selftest())


def set_stream(stream) -> None:
    """Routes later launches from this thread to `stream` (a torch Stream or
    a raw hipStream_t int); None (or torch's null stream) restores the
    per-thread default stream."""
    handle = 0 if stream is None else (stream if isinstance(stream, int) else stream.cuda_stream)
    _check(_lib.load().pulsar_set_stream(handle or None), "set_stream")


def bw_read(buf, nbytes: int, sink) -> None:
    _check(_lib.load().pulsar_bw_read(_ptr(buf), nbytes, _ptr(sink)), "bw_read")


EXPERT_PTRS_DTYPE = np.dtype(
    [("gate", "<u8"), ("up", "<u8"), ("down", "<u8"), ("gate_b", "<u8"), ("up_b", "<u8"), ("down_b", "<u8")]
)
assert EXPERT_PTRS_DTYPE.itemsize == EXPERT_PTRS_BYTES


def expert_ptrs(entries) -> np.ndarray:
    """Packs (gate, up, down[, gate_b, up_b, down_b]) address tuples (0 = NULL)
    into the 48-byte pulsar_expert_ptrs layout (crates/kernels/src/lib.rs:21-49)."""
    arr = np.zeros(len(entries), dtype=EXPERT_PTRS_DTYPE)
    for i, e in enumerate(entries):
        e = tuple(e) + (0,) * (6 - len(e))
        arr[i] = tuple(int(v) for v in e)
    return arr
