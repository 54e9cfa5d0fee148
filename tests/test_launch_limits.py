"""Rows of which one axis of a launch does not hold the threads (fewer than 2^32) are
refused by the stages whose other axes are taken, before any launch (no GPU: addresses that
are never read)."""
import pytest
import torch

from pulsar_amd import kernels as K
from pulsar_amd.formats import (ACT_SILU, QUANT_IQ4_XS, QUANT_MXFP4, QUANT_Q2_K, QUANT_Q3_K, QUANT_Q4_K, TYPE_BF16, TYPE_F16,
                                TYPE_F32, row_bytes)
from tests.test_int8_arguments import A, lib, product, said  # noqa: F401
from tests.test_operator_refusals import bank

COLS = 4096  # a row is a wave's


def down(out_dim, quant=QUANT_Q4_K):
    K.moe_down(A[0], A[1], A[2], COLS, out_dim, 1, 1, row_bytes(quant, COLS), quant)


def down_biased(out_dim, quant=QUANT_Q4_K):
    K.moe_down_biased(A[0], A[1], A[2], A[3], COLS, out_dim, 1, 1, row_bytes(quant, COLS), quant)


def down_f32(out_dim, quant=QUANT_Q4_K):
    K.moe_down_f32(A[0], A[1], A[2], A[3], COLS, out_dim, 1, 1, row_bytes(quant, COLS), quant, False)


def pair(mid_dim, quant=QUANT_Q4_K):
    K.moe_pair_swiglu(A[0], A[1], A[2], A[3], COLS, mid_dim, 1, 1, row_bytes(quant, COLS), quant, ACT_SILU)


def pair_routed(mid_dim, quant=QUANT_Q4_K):
    K.moe_pair_routed(A[0], A[1], A[2], A[3], A[4], A[5], 0, 32, 1, 1.0, 0, bank(), [], A[6], COLS, mid_dim, 1,
                      row_bytes(quant, COLS), quant, ACT_SILU)


def pair_grouped(mid_dim, quant=QUANT_Q4_K):
    K.moe_pair_swiglu_grouped(A[0], A[1], A[2], A[3], A[4], A[5], COLS, mid_dim, 1, 1, row_bytes(quant, COLS), quant,
                              ACT_SILU)


def down_grouped(out_dim, quant=QUANT_Q4_K):
    K.moe_down_grouped(A[0], A[1], A[2], A[3], A[4], COLS, out_dim, 1, 1, row_bytes(quant, COLS), quant)


def pair_experts(mid_dim, quant=QUANT_Q4_K, n_tok=1):
    K.moe_pair_swiglu_experts(A[0], A[1], A[2], A[3], A[4], bank(), 1, [], n_tok, 1, COLS, mid_dim,
                              row_bytes(quant, COLS), quant, ACT_SILU)


def down_experts(out_dim, quant=QUANT_Q4_K, n_tok=1):
    K.moe_down_experts(A[0], A[1], A[2], A[3], bank(), 1, [], n_tok, 1, COLS, out_dim, row_bytes(quant, COLS), quant)


LANE, WIDE = QUANT_Q3_K, dict(n_tok=2000)  # one group of many pairs: the wide tile


@pytest.mark.parametrize("call,rows,kw", [
    (down, 2**24, {}), (down_biased, 2**24, {}), (down_f32, 2**31, {}), (pair, 2**27, {}), (pair_routed, 2**26, {}),
    (pair_grouped, 2**31, {}), (down_grouped, 2**31, {}), (pair_grouped, 2**31, dict(quant=LANE)),
    (down_grouped, 2**31, dict(quant=LANE)), (pair_grouped, 2**31, dict(quant=QUANT_MXFP4)),
    (down_grouped, 2**31, dict(quant=QUANT_Q2_K)), (pair_experts, 2**31, {}), (down_experts, 2**31, {}),
    (pair_experts, 2**31, WIDE), (down_experts, 2**31 + 2**27, WIDE), (pair_experts, 2**31, dict(quant=LANE)),
    (down_experts, 2**31, dict(quant=QUANT_IQ4_XS))])
def test_stages_refuse(capfd, call, rows, kw):
    assert "(size)" in said(capfd, lambda: call(rows, **kw))


@pytest.mark.parametrize("call,rows", [(down, 2**24 - 1), (down_biased, 2**24 - 1), (pair, 2**27 - 8), (pair_routed, 2**26 - 4)])
def test_the_most_rows_reach_a_launch(capfd, call, rows):
    if torch.cuda.is_available():
        pytest.skip("these addresses are nobody's")
    assert not said(capfd, lambda: call(rows))


@pytest.mark.parametrize("call", [
    lambda: K.quantize_q8_k(A[0], A[1], 2**32 - 1, 1), lambda: K.quantize_q8_k(A[0], A[1], 512, 2**32 - 1),
    lambda: K.matmul_f32(A[0], A[1], A[2], 2**32 - 255, 1, 1), lambda: K.matmul_f32(A[0], A[1], A[2], 4, 1, 2**32 - 1),
    lambda: K.router_logits_q8(A[0], A[1], A[2], A[3], 0, 2**32 - 1, 1, 1),
    lambda: K.router_logits_q8(A[0], A[1], A[2], A[3], 0, 4, 1, 2**32 - 1),
    lambda: K.router_logits_q8(A[0], A[1], A[2], A[3], 0, 1280, 1, 2**30),
    lambda: K.router_select(A[0], A[1], A[2], 0, 1, 1, 1.0, 2**31, 0, 0), lambda: K.add_bias_rows(A[0], A[1], 2**20, 2**19),
    lambda: K.moe_slot_sum(A[0], A[1], 2**20, 1, 2**19), lambda: K.moe_down_bias(A[0], A[1], A[2], 2**20, 1, 2**19),
    lambda: K.moe_slot_sum_bias(A[0], A[1], A[2], A[3], 2**20, 1, 2**19),
    lambda: K.moe_route_ptrs(A[0], A[1], A[2], A[3], bank(), 32, [], 2**31, 2**8)])
def test_sizes_past_two_axes(capfd, call):
    assert said(capfd, call)


@pytest.mark.parametrize("in_dim", [300, 304])  # rows that are not on 16 bytes, and that are
@pytest.mark.parametrize("kind", [TYPE_F32, TYPE_F16, TYPE_BF16])
def test_int8_product_refuses_2_31_tiles(capfd, in_dim, kind):
    """Of 128 tokens x 128 channels, whatever tile the product would take."""
    call = lambda T, n: product(out=1 << 61, residual=0, in_dim=in_dim, out_dim=n, n_tok=T, type=kind)  # noqa: E731
    for T, n in ((128 * 127 + 1, 2**31 - 1), (2**31 - 1, 128 * 127 + 1), (128 * 2**15 + 1, 128 * (2**16 - 1))):
        assert "matmul_i8 (size)" in said(capfd, lambda: call(T, n))
    if torch.cuda.is_available():
        return  # these addresses are nobody's
    for T, n in ((128 * 127, 2**31 - 1), (2**31 - 1, 128 * 127), (128 * 2**15, 128 * (2**16 - 1)), (2, 2**31 - 1)):
        assert not said(capfd, lambda: call(T, n))
