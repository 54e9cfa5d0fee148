"""What the routing with expert groups, the grouping by ids and the product with
an epilogue refuse, before any launch (no GPU: the addresses are never read)."""
import ctypes

import pytest
import torch

from pulsar_amd import _lib
from pulsar_amd import kernels as K
from pulsar_amd.formats import EPI_SIGMOID, QUANT_MXFP4, QUANT_Q4_K, QUANT_Q8_0

A = [0x10000000 * (i + 1) for i in range(8)]  # addresses far apart


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    return _lib.load()


ROUTE = dict(selected=A[0], weights=A[1], logits=A[2], bias=A[3], n_expert=32, k_used=4, n_group=8, topk_group=2,
             group_top=2, score=0, renorm=True, weight_scale=1.0, n_tok=3)


@pytest.mark.parametrize("change", [
    dict(selected=0), dict(weights=0), dict(logits=0), dict(n_tok=0), dict(n_tok=2**25 + 1), dict(n_expert=0), dict(n_expert=1032),
    dict(n_group=0), dict(n_group=5), dict(n_group=128, n_expert=1024), dict(topk_group=0), dict(topk_group=9),
    dict(group_top=0), dict(group_top=3), dict(k_used=0), dict(k_used=9), dict(k_used=65, n_expert=512, topk_group=8),
    dict(score=2)])
def test_router_select_groups_refuses(change):
    with pytest.raises(K.KernelError, match="router_select_groups"):
        K.router_select_groups(**{**ROUTE, **change})


def bank():
    return K.ExpertBank(A[5], A[6], A[7], None, None, None, 64, 64, 64, 0, 0, 0)


IDS = dict(gptrs=A[0], starts=A[1], pairs=A[2], slot_weights=A[3], selected=A[4], router_weights=A[5], n_expert=32,
           shared=[], n_tok=300, k_used=8)


@pytest.mark.parametrize("change", [
    dict(gptrs=0), dict(starts=0), dict(pairs=0), dict(selected=0), dict(router_weights=0), dict(n_expert=0),
    dict(n_expert=1025), dict(n_tok=0), dict(n_tok=2**28 + 1, k_used=1), dict(n_tok=2**28, k_used=8), dict(k_used=0),
    dict(k_used=17), dict(k_used=16, shared=[(A[5], A[6], A[7])]), dict(shared=[(A[5], A[6], A[7])] * 5)])
def test_moe_group_ids_refuses(change):
    with pytest.raises(K.KernelError, match="moe_group_ids"):
        K.moe_group_ids(bank=bank(), **{**IDS, **change})


def test_moe_group_ids_refuses_null_bank_and_shared(lib):
    args = [A[0], A[1], A[2], A[3], A[4], A[5]]
    assert lib.pulsar_moe_group_ids(*args, None, 32, None, 0, 300, 8) == 0
    assert lib.pulsar_moe_group_ids(*args, ctypes.addressof(bank()), 32, None, 1, 300, 8) == 0


PRODUCT = dict(out=A[0], w=A[1], xq=A[2], bias=A[3], residual=A[4], in_dim=512, out_dim=64, n_tok=3, row_bytes=288,
               quant=QUANT_Q4_K, act=0)


@pytest.mark.parametrize("change", [
    dict(out=0), dict(w=0), dict(xq=0), dict(in_dim=0), dict(in_dim=300), dict(out_dim=0), dict(n_tok=0),
    dict(row_bytes=0), dict(act=EPI_SIGMOID + 1), dict(quant=QUANT_MXFP4), dict(quant=QUANT_Q8_0),
    dict(quant=QUANT_Q8_0, n_tok=40), dict(quant=99), dict(out_stride=63), dict(res_stride=63),
    dict(out_stride=2**63),
    # out over an operand
    dict(out=A[1] + 8), dict(out=A[2]), dict(out=A[3] + 252), dict(bias=A[0] + 4 * 191),
    # residual rows that share floats with out's, but are not out's
    dict(residual=A[0] + 4), dict(residual=A[0], res_stride=128), dict(residual=A[0] + 4 * 40, out_stride=100, res_stride=100),
    dict(residual=A[0] - 4 * 99, out_stride=100, res_stride=100)])
def test_matmul_kq_fused_refuses(change):
    with pytest.raises(K.KernelError, match="matmul_kq_fused"):
        K.matmul_kq_fused(**{**PRODUCT, **change})


def test_wrappers_refuse_host_tensors():
    t = torch.zeros(4096)
    with pytest.raises(ValueError, match="host tensor"):
        K.matmul_kq_fused(**{**PRODUCT, "residual": t})
    with pytest.raises(ValueError, match="host tensor"):
        K.router_select_groups(**{**ROUTE, "logits": t})
    with pytest.raises(ValueError, match="host tensor"):
        K.moe_group_ids(bank=bank(), **{**IDS, "pairs": t})
