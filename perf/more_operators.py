"""What the steps of a dense layer in 8-bit integers cost: the norm with the
residual's addition, whose rows come out in 8 bits (q8_K blocks, or int8 with a
scale a row), the quantizer behind a gated activation, and the product of int8
rows with scales of tokens and channels. Each runs in its plain form (torch
operations on the whole arrays) or, with `own` set, through pulsar_amd.kernels."""
import math

import numpy as np
import torch

own = False
DEV = "cuda:0"
EPS = 1e-6
TYPES = {"f32": (torch.float32, 0, 4), "f16": (torch.float16, 1, 2), "bf16": (torch.bfloat16, 2, 2)}
ACTS = {"none": 0, "silu": 1, "gelu": 2, "relu": 3, "sigmoid": 4}
GLUS = {"none": 0, "silu": 0, "swiglu_oai": 2}
# nearer than this to a half, a code's argument counts as on it (and goes up)
NEAR = 2.0**-40


def listed():
    return [
        # one decoded token between attention and a routed layer: the sum goes on,
        # the router reads the f32 row, the experts the q8_K blocks
        dict(name="norm_1_q8k", op="norm", rows=1, dim=4096, type="f32", residual=True, y=True, out="q8k"),
        # a batch of decoding sequences of an odd size, int8 rows for a dense layer
        dict(name="norm_33_i8", op="norm", rows=33, dim=2880, type="bf16", residual=True, y=False, out="i8"),
        # a prompt chunk in front of the routed layer
        dict(name="norm_512_q8k", op="norm", rows=512, dim=4096, type="f32", residual=True, y=True, out="q8k"),
        # a long prompt in front of a dense layer
        dict(name="norm_8192_i8", op="norm", rows=8192, dim=4096, type="bf16", residual=True, y=False, out="i8"),
        # one decoded token's gated activations, f32
        dict(name="glu_1", op="quant", rows=1, dim=14336, type="f32", glu="silu"),
        # a ragged chunk of rows that end inside a vector load, clamped gate
        dict(name="glu_250_odd", op="quant", rows=250, dim=1419, type="bf16", glu="swiglu_oai"),
        # a long prompt's gated activations
        dict(name="glu_4096", op="quant", rows=4096, dim=14336, type="bf16", glu="silu"),
        # decode: the projection back to the hidden size, added to the residual
        dict(name="i8_1", op="product", tokens=1, rows=4096, cols=4096, type="f32", bias=False, act="none",
             residual=True),
        # a batch of decoding sequences through a wide projection
        dict(name="i8_16", op="product", tokens=16, rows=8192, cols=4096, type="bf16", bias=True, act="none",
             residual=False),
        # a ragged chunk, rows of an odd number of bytes
        dict(name="i8_130_odd", op="product", tokens=130, rows=5001, cols=2047, type="f32", bias=True, act="gelu",
             residual=False),
        # a prompt chunk through the gate and up projections at once
        dict(name="i8_512", op="product", tokens=512, rows=28672, cols=4096, type="bf16", bias=False, act="none",
             residual=False),
        # a long prompt through the down projection, added to the residual
        dict(name="i8_4096", op="product", tokens=4096, rows=4096, cols=14336, type="bf16", bias=True, act="none",
             residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quant", "product", "product"])
    kind = rng.choice(list(TYPES))
    if op == "product":
        rows, cols = _log(rng, 64, 28672), _log(rng, 64, 16384)
        if rng.random() < 0.7:  # most models' sizes
            rows, cols = -(-rows // 64) * 64, -(-cols // 64) * 64
        tokens = _log(rng, 1, max(1, min(8192, 200_000_000_000 // (rows * cols))))
        return dict(op=op, tokens=tokens, rows=rows, cols=cols, type=kind, bias=rng.random() < 0.5,
                    act=rng.choice(["none", "none", "silu", "gelu", "relu", "sigmoid"]), residual=rng.random() < 0.5)
    dim = _log(rng, 64, 16384)
    if rng.random() < 0.7:
        dim = -(-dim // 32) * 32
    rows = _log(rng, 1, min(16384, 32_000_000 // dim))
    if op == "quant":
        return dict(op=op, rows=rows, dim=dim, type=kind, glu=rng.choice(["silu", "swiglu_oai", "none"]))
    return dict(op=op, rows=rows, dim=dim, type=kind, residual=rng.random() < 0.8, y=rng.random() < 0.5,
                out=rng.choice(["q8k", "i8"]))


# ------------------------------------------------------------------ inputs --

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _zeros(shape, dtype):
    return torch.zeros(shape, dtype=dtype, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, s = case, {"case": case}
    kind, n = TYPES[c["type"]][0], c["rows"]
    if c["op"] == "product":
        T, K = c["tokens"], c["cols"]
        # codes of rows quantized by their largest value: a third of them in the
        # outer half, both ends among them
        s["x"] = (38.0 * _randn(g, T, K)).round_().clamp_(-127, 127).to(torch.int8)
        s["w"] = (38.0 * _randn(g, n, K)).round_().clamp_(-127, 127).to(torch.int8)
        s["x_scales"] = (torch.rand(T, generator=g, device=DEV) + 0.5) / 38.0
        s["w_scales"] = (torch.rand(n, generator=g, device=DEV) + 0.5) / (38.0 * math.sqrt(K))
        s["bias"] = 0.5 * _randn(g, n) if c["bias"] else None
        s["residual"] = _randn(g, T, n).to(kind) if c["residual"] else None
        s["out"] = _zeros((T, n), kind)
        return s
    dim = c["dim"]
    if c["op"] == "quant":
        s["x"] = (1.5 * _randn(g, n, dim)).to(kind)
        s["up"] = _randn(g, n, dim).to(kind) if c["glu"] != "none" else None
    else:
        # a residual stream: channels of their own size, a few of them large
        wide = torch.exp(0.5 * _randn(g, dim)) * torch.where(torch.rand(dim, generator=g, device=DEV) < 0.01, 12.0, 1.0)
        s["x"] = (_randn(g, n, dim) * wide).to(kind)
        s["residual"] = (0.5 * _randn(g, n, dim)).to(kind) if c["residual"] else None
        s["gain"] = torch.exp(0.2 * _randn(g, dim))
        s["sum"] = _zeros((n, dim), kind) if c["residual"] else None
        s["y"] = _zeros((n, dim), kind) if c["y"] else None
    if c.get("out") == "q8k":
        s["blocks"] = _zeros((n, -(-dim // 256), 292), torch.uint8)
    else:
        s["q"], s["scales"] = _zeros((n, dim), torch.int8), _zeros(n, torch.float32)
    # the values that the codes stand for, in the rows' type
    s["values"] = _zeros((n, -(-dim // 256), 256) if c.get("out") == "q8k" else (n, dim), kind)
    return s


# ------------------------------------------------------- the plain forms ----

def _codes(p, largest):
    """Integers of p / largest * 127, halves away from 0, in 64 bits: an
    argument can lie next to a half."""
    t = torch.where(largest > 0, p / largest, 0.0) * 127.0
    return torch.trunc(t + torch.copysign(torch.full((), 0.5 + NEAR, dtype=t.dtype, device=DEV), t))


def _norm(s):
    c, x = s["case"], s["x"]
    got = {}
    if s["residual"] is not None:
        x = (x.float() + s["residual"].float()).to(x.dtype)
        got["sum"] = x
    v = x.double()
    p = v * s["gain"].double()
    rs = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + float(np.float32(EPS)))
    if s["y"] is not None:
        got["y"] = (p * rs).to(x.dtype)
    if c["out"] == "q8k":
        pad = -c["dim"] % 256
        p = torch.nn.functional.pad(p, (0, pad)).view(c["rows"], -1, 256)
        rs = rs[..., None]
    largest = p.abs().amax(-1, keepdim=True)
    q, d = _codes(p, largest), (largest * rs / 127.0).float()
    got["values"] = (q.float() * d).to(x.dtype)
    if c["out"] == "q8k":
        got["sums"] = q.view(c["rows"], -1, 16, 16).sum(-1).to(torch.int16)
    return got


def _quant(s):
    v = s["x"].double()
    if s["case"]["glu"] == "silu":
        v = v / (1.0 + torch.exp(-v)) * s["up"].double()
    elif s["case"]["glu"] == "swiglu_oai":
        v = v.clamp_max(7.0)
        v = v / (1.0 + torch.exp(-1.702 * v)) * (s["up"].double().clamp(-7.0, 7.0) + 1.0)
    largest = v.abs().amax(1, keepdim=True)
    d = (largest / 127.0).float()
    return {"values": (_codes(v, largest).float() * d).to(s["x"].dtype)}


def _act(name, v):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "relu":
        return v.clamp_min(0.0)
    return 1.0 / (1.0 + torch.exp(-v)) if name == "sigmoid" else v


def _product(s):
    v = s["x"].float() @ s["w"].float().T
    v = v * s["x_scales"][:, None] * s["w_scales"]
    if s["bias"] is not None:
        v = v + s["bias"]
    v = _act(s["case"]["act"], v)
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["out"].dtype)


# -------------------------------------------------------------------- run --

def _values(s, codes, scales):
    """The codes' values, computed on the stream that the calls go to: on torch's
    own each pass would change streams twice, and wait for it."""
    from pulsar_amd import runtime

    if "stream" not in s:
        s["stream"] = torch.cuda.ExternalStream(runtime.STREAM_PER_THREAD)
    with torch.cuda.stream(s["stream"]):
        return torch.mul(codes, scales, out=s["values"])


def _call(s):
    from pulsar_amd import kernels as K

    c, kind = s["case"], TYPES[s["case"]["type"]][1]
    if c["op"] == "product":
        K.matmul_i8(s["out"], s["w"], s["w_scales"], s["x"], s["x_scales"], s["bias"], s["residual"], c["cols"],
                    c["rows"], c["tokens"], ACTS[c["act"]], kind)
        return s["out"]
    if c["op"] == "quant":
        K.quantize_i8(s["q"], s["scales"], s["x"], s["up"], c["dim"], c["rows"], GLUS[c["glu"]], kind)
        return {"values": _values(s, s["q"], s["scales"][:, None])}
    got = {k: s[k] for k in ("sum", "y") if s[k] is not None}
    if c["out"] == "i8":
        K.rms_norm_q8(s["q"], s["scales"], s["y"], s["sum"], s["x"], s["residual"], s["gain"], c["dim"], c["rows"], EPS,
                      kind, 1)
        got["values"] = _values(s, s["q"], s["scales"][:, None])
        return got
    b = s["blocks"]
    K.rms_norm_q8(b, None, s["y"], s["sum"], s["x"], s["residual"], s["gain"], c["dim"], c["rows"], EPS, kind, 0)
    got["values"] = _values(s, b[..., 4:260].view(torch.int8), b[..., :4].view(torch.float32))
    got["sums"] = b[..., 260:].view(torch.int16)
    return got


def run(s):
    if own:
        return _call(s)
    return {"norm": _norm, "quant": _quant, "product": _product}[s["case"]["op"]](s)


def work(c):
    size, n = TYPES[c["type"]][2], c["rows"]
    if c["op"] == "product":
        T, K = c["tokens"], c["cols"]
        out = size * T * n * (2 if c["residual"] else 1)
        return {"bytes": n * K + T * K + 4 * T + 4 * n + out + (4 * n if c["bias"] else 0), "flops": 2 * T * n * K}
    m = n * c["dim"]
    if c["op"] == "quant":
        return {"bytes": m * (size * (1 if c["glu"] == "none" else 2) + 1) + 4 * n, "flops": 16 * m}
    codes = n * -(-c["dim"] // 256) * 292 if c["out"] == "q8k" else m + 4 * n
    arrays = 1 + (2 if c["residual"] else 0) + (1 if c["y"] else 0)
    return {"bytes": arrays * size * m + 4 * c["dim"] + codes, "flops": 8 * m}


# ------------------------------------------------------------------ exact --

def _host(t):
    return None if t is None else t.detach().float().cpu().numpy().astype(np.float64)


def _rounded(v, kind):
    return torch.from_numpy(v).to(kind).double().numpy()


def _levels(p, top):
    """The 8-bit numbers nearest to 127 p / top: how many halves below lie under it."""
    with np.errstate(invalid="ignore", divide="ignore"):
        a = np.where(top == 0, 0.0, np.abs(p) / top)
    return np.sign(p) * np.floor(a * 127.0 + (0.5 + NEAR))


def _exact_norm(c, s):
    x, r, g = _host(s["x"]), _host(s["residual"]), _host(s["gain"])
    got = {}
    if r is not None:
        x = got["sum"] = _rounded(x + r, s["x"].dtype)
    n, dim = x.shape
    norm = np.sqrt(np.einsum("ij,ij->i", x, x) / dim + np.float64(np.float32(EPS)))[:, None]
    p = x * g
    if s["y"] is not None:
        got["y"] = p / norm
    if c["out"] == "i8":
        top = np.abs(p).max(1)[:, None]
        got["values"] = _levels(p, top) * (top / norm / 127.0)
    else:
        nb = -(-dim // 256)
        values, sums = np.zeros((n, nb, 256)), np.zeros((n, nb, 16), np.int16)
        for b in range(nb):
            part = p[:, 256 * b:256 * b + 256]
            top = np.abs(part).max(1)[:, None]
            q = np.zeros((n, 256))
            q[:, :part.shape[1]] = _levels(part, top)
            values[:, b] = q * (top / norm / 127.0)
            sums[:, b] = np.add.reduceat(q, np.arange(0, 256, 16), axis=1)
        got["values"], got["sums"] = values, sums
    return {k: torch.from_numpy(v) for k, v in got.items()}


def _exact_quant(c, s):
    v = _host(s["x"])
    if c["glu"] != "none":
        u, a = _host(s["up"]), 1.0
        if c["glu"] == "swiglu_oai":
            a, v, u = 1.702, np.minimum(v, 7.0), 1.0 + np.minimum(np.maximum(u, -7.0), 7.0)
        e = np.exp(-np.abs(a * v))
        v = v * u * (np.where(v < 0, e, 1.0) / (1.0 + e))
    top = np.abs(v).max(1)[:, None]
    return {"values": torch.from_numpy(_levels(v, top) * (top / 127.0))}


def _exact_product(c, s):
    """Channels in parts, sums in 64 bits."""
    x, (T, n) = s["x"].double(), s["out"].shape
    out = torch.empty((T, n), dtype=torch.float64, device=DEV)
    step = max(1, 32_000_000 // c["cols"])
    for r in range(0, n, step):
        w = s["w"][r:r + step].double() * s["w_scales"][r:r + step, None].double()
        out[:, r:r + step] = torch.mm(x, w.t())
    out *= s["x_scales"].double()[:, None]
    if s["bias"] is not None:
        out += s["bias"].double()
    if c["act"] == "silu":
        out = out * torch.special.expit(out)
    elif c["act"] == "gelu":
        out = 0.5 * out * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (out + 0.044715 * out**3)))
    elif c["act"] == "relu":
        out = torch.where(out > 0, out, 0.0)
    elif c["act"] == "sigmoid":
        out = torch.special.expit(out)
    return out if s["residual"] is None else out + s["residual"].double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "quant": _exact_quant, "product": _exact_product}[case["op"]](case, s)
