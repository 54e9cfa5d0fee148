"""Calls of more blocks than one axis of a launch holds (fewer than 2^32 threads, so 2^24
blocks of 256): every row of theirs is done, the first and the last ones too."""
import numpy as np
import pytest
import torch

from pulsar_amd import kernels as K
from pulsar_amd import synth
from pulsar_amd.formats import QUANT_IQ4_NL, QUANT_NVFP4, QUANT_Q4_K, row_bytes
from tests.gpu_util import up_f32, zeros_f32

pytestmark = pytest.mark.gpu
AXIS = 2**24  # blocks of 256 threads
SUM_TOK, SUM_DIM = 2**16 + 3, 2**16  # a value a thread


def small(shape, seed, dev):
    """Whole numbers: sums of their products are exact in f32."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=g, device=dev).float()


@pytest.fixture(autouse=True)
def leave_no_memory():
    yield
    torch.cuda.empty_cache()


def test_quantize_q8_k(dev):
    """4 blocks of q8_K a block: rows of one value, whose code is 127 or -127."""
    n = 4 * AXIS + 9
    x = torch.arange(n, device=dev).remainder_(1000).sub_(500).float()
    out = torch.full((n, 292), 0xAB, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    K.quantize_q8_k(out, x, 1, n)
    torch.cuda.synchronize()
    code = (127 * torch.sign(x)).to(torch.int8)
    assert torch.equal(out[:, 4].contiguous().view(torch.int8), code)
    assert torch.equal(out[:, 260:262].contiguous().view(torch.int16).view(-1), code.to(torch.int16))
    d = out[:, :4].contiguous().view(torch.float32).view(-1)
    assert ((d - x.abs() / 127).abs() <= 2.0**-23 * d).all()
    assert not out[:, 5:260].any() and not out[:, 262:].any()


@pytest.mark.parametrize("out_dim,n_tok", [(4096, 8200), (4097, 8203), (2049, 16400), (AXIS + 5, 1)])
def test_matmul_f32(dev, out_dim, n_tok):
    """A block is a row and two tokens."""
    assert out_dim * ((n_tok + 1) // 2) > AXIS
    w, x = small((out_dim, 4), 1, dev), small((n_tok, 4), 2, dev)
    out = torch.full((n_tok, out_dim), 1e30, device=dev)
    torch.cuda.synchronize()
    K.matmul_f32(out, w, x, 4, out_dim, n_tok)
    torch.cuda.synchronize()
    assert torch.equal(out, x @ w.T)


@pytest.mark.parametrize("n_expert,n_tok", [(256, 131078), (257, 131073)])
def test_router_logits_q8(dev, n_expert, n_tok):
    dim = 260
    w, x, bias = small((n_expert, dim), 1, dev), small((n_tok, dim), 2, dev), small((n_expert,), 3, dev)
    logits = torch.full((n_tok, n_expert), 1e30, device=dev)
    xq, want = (torch.full((n_tok * 2 * 292,), 0xAB, dtype=torch.uint8, device=dev) for _ in range(2))
    torch.cuda.synchronize()
    K.router_logits_q8(logits, xq, x, w, bias, dim, n_expert, n_tok)
    K.quantize_q8_k(want, x, dim, n_tok)
    torch.cuda.synchronize()
    assert torch.equal(logits, x @ w.T + bias) and torch.equal(xq, want)


def test_add_bias_rows(dev):
    x, bias = torch.ones((SUM_TOK, SUM_DIM), device=dev), small((SUM_DIM,), 1, dev)
    torch.cuda.synchronize()
    K.add_bias_rows(x, bias, SUM_DIM, SUM_TOK)
    torch.cuda.synchronize()
    assert (x == bias + 1).all()


def test_slot_sums(dev):
    """Sums of one slot, a bias, and both in one call."""
    bias = small((SUM_DIM,), 1, dev)
    row = np.zeros((SUM_TOK, 6), np.uint64)
    row[:, 5] = bias.data_ptr()
    ptrs, weights = torch.from_numpy(row.view(np.int64)).to(dev), torch.full((SUM_TOK,), 2.0, device=dev)
    partial = torch.arange(SUM_TOK, device=dev).remainder_(1000).float()[:, None].expand(-1, SUM_DIM).contiguous()
    out = torch.full((SUM_TOK, SUM_DIM), 1e30, device=dev)
    torch.cuda.synchronize()
    K.moe_slot_sum(out, partial, SUM_DIM, 1, SUM_TOK)
    torch.cuda.synchronize()
    assert torch.equal(out, partial)
    K.moe_down_bias(out, ptrs, weights, SUM_DIM, 1, SUM_TOK)
    torch.cuda.synchronize()
    assert (out == partial + 2 * bias).all()
    out.fill_(1e30)
    torch.cuda.synchronize()
    K.moe_slot_sum_bias(out, partial, ptrs, weights, SUM_DIM, 1, SUM_TOK)
    torch.cuda.synchronize()
    assert (out == partial + 2 * bias).all()


def test_router_select(dev):
    """A block of 64 threads a token: 2^26 of them."""
    n = 4 * AXIS + 7
    logits = small((n, 2), 1, dev)
    selected = torch.full((n, 1), -5, dtype=torch.int32, device=dev)
    weights = zeros_f32((n, 1))
    torch.cuda.synchronize()
    K.router_select(selected, weights, logits, up_f32(np.array([0.0, 0.0])), 2, 1, 2.5, n, 1, 0)
    torch.cuda.synchronize()
    assert torch.equal(selected[:, 0], (logits[:, 1] > logits[:, 0]).int())  # the first of equal ones
    assert (weights == 2.5).all()  # a softmax over one winner


@pytest.mark.parametrize("quant,n_tok", [(QUANT_IQ4_NL, 300_001), (QUANT_NVFP4, 2_200_001), (QUANT_Q4_K, 2_200_001)])
def test_products_of_many_tokens(dev, quant, n_tok):
    """More token groups than 2^16: the tokens repeat, so do the rows of the product."""
    rows, cols, period = 16, 256, 1000
    w = torch.from_numpy(synth.quant_matrix(quant, rows, cols, np.random.default_rng(1)).view(np.uint8).reshape(-1)).to(dev)
    x = small((period, cols), 1, dev)
    xq = torch.zeros((period, 292), dtype=torch.uint8, device=dev)
    K.quantize_q8_k(xq, x, cols, period)
    torch.cuda.synchronize()
    many = xq.repeat(-(-n_tok // period), 1)[:n_tok].contiguous()
    out = torch.full((n_tok, rows), 1e30, device=dev)
    torch.cuda.synchronize()
    K.matmul_kq(out, w, many, cols, rows, n_tok, row_bytes(quant, cols), quant)
    torch.cuda.synchronize()
    assert (out[:period].abs() < 1e6).all()
    whole = n_tok // period * period
    assert (out[:whole].view(-1, period, rows) == out[:period]).all() and torch.equal(out[whole:], out[:n_tok - whole])
