"""What the operators around the routed experts cost: routing with expert
groups, grouping a long chunk's pairs by expert, and the dense quantized
product with its epilogue. Each runs in its plain form (torch operations on
the whole arrays) or, with `own` set, through pulsar_amd.kernels."""
import math

import numpy as np
import torch

own = False
DEV = "cuda:0"

# quant code, bytes per 256 values, byte offset of the f16 scale, rms of
# weight / scale over random blocks, offset of the f16 min scale, its ratio to
# the scale that centres the codes
FMT = {"Q2_K": (0, 84, 80, 13.0, 82, 1.5), "Q4_K": (2, 144, 0, 250.0, 2, 7.5), "Q5_K": (3, 176, 0, 500.0, 2, 15.5),
       "Q6_K": (4, 210, 208, 1370.0, None, 0.0), "Q3_K": (5, 110, 108, 42.0, None, 0.0),
       "IQ4_XS": (11, 136, 0, 1200.0, None, 0.0)}
ACTS = {"none": 0, "silu": 1, "gelu": 2, "relu": 3, "sigmoid": 4}
SCORES = {"sigmoid": 0, "softmax": 1}


def listed():
    return [
        # one token of a decode step: sigmoid scores with a balance bias, the
        # best 4 of 8 groups of experts by their two best, renormalised
        dict(name="route_1", op="route", tokens=1, experts=256, k=8, groups=8, top_groups=4, group_top=2,
             score="sigmoid", bias=True, renorm=True),
        # a batch of decoding sequences, softmax scores of a layer of few
        # experts, weights left as probabilities
        dict(name="route_130_softmax", op="route", tokens=130, experts=32, k=4, groups=1, top_groups=1, group_top=1,
             score="softmax", bias=False, renorm=False),
        # a prompt chunk, 128 experts without groups
        dict(name="route_4096_softmax", op="route", tokens=4096, experts=128, k=8, groups=1, top_groups=1, group_top=1,
             score="softmax", bias=False, renorm=True),
        # a long prompt of several sequences, groups and bias
        dict(name="route_16384_groups", op="route", tokens=16384, experts=256, k=8, groups=8, top_groups=4, group_top=2,
             score="sigmoid", bias=True, renorm=True),
        # the smallest chunk that no longer groups in one block, ragged, with a
        # shared expert beside the routed ones
        dict(name="group_301_shared", op="group", tokens=301, experts=256, k=8, shared=1),
        # a long prompt
        dict(name="group_16384", op="group", tokens=16384, experts=256, k=8, shared=0),
        # decode: the projection back to the hidden size, added to the residual
        dict(name="proj_q4k_1", op="product", fmt="Q4_K", rows=4096, cols=4096, tokens=1, bias=False, act="none",
             residual=True),
        # four speculative tokens through a 6-bit projection with a bias
        dict(name="proj_q6k_4", op="product", fmt="Q6_K", rows=8192, cols=4096, tokens=4, bias=True, act="none",
             residual=False),
        # a short chunk, one more token than a tile of 32
        dict(name="proj_q5k_33", op="product", fmt="Q5_K", rows=4096, cols=4096, tokens=33, bias=True, act="none",
             residual=True),
        # a ragged prompt chunk through a codebook format, bias and GELU
        dict(name="up_iq4xs_250", op="product", fmt="IQ4_XS", rows=8192, cols=2816, tokens=250, bias=True, act="gelu",
             residual=False),
        # a prompt chunk through a wide up projection
        dict(name="up_q4k_512", op="product", fmt="Q4_K", rows=14336, cols=4096, tokens=512, bias=False, act="silu",
             residual=False),
        # a long prompt through the down projection, bias and residual
        dict(name="down_q4k_2048", op="product", fmt="Q4_K", rows=4096, cols=14336, tokens=2048, bias=True, act="none",
             residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route", "group", "product", "product", "product"])
    if op == "route":
        size = _log(rng, 4, 128)  # experts of a group
        groups = rng.randint(1, max(1, min(32, 512 // size)))
        if rng.random() < 0.35:
            groups = 8 if 8 * size <= 512 else 1
        top = rng.randint(1, groups)
        k = rng.randint(1, min(16, top * size))
        most = min(32768, 16384 * 256 // (size * groups))
        return dict(op=op, tokens=_log(rng, 1, most), experts=size * groups, k=k, groups=groups, top_groups=top,
                    group_top=rng.choice([1, 2]), score=rng.choice(["sigmoid", "softmax"]),
                    bias=rng.random() < 0.6, renorm=rng.random() < 0.6)
    if op == "group":
        experts, k = _log(rng, 4, 512), rng.randint(1, 12)
        k = min(k, experts)
        return dict(op=op, tokens=_log(rng, 1, 131072 // k), experts=experts, k=k, shared=rng.choice([0, 0, 1, 2]))
    fmt = rng.choice(list(FMT))
    rows, cols = _log(rng, 256, 16000), 256 * _log(rng, 1, 56)
    tokens = _log(rng, 1, max(1, min(4096, 120_000_000_000 // (rows * cols))))
    act = rng.choice(["none", "none", "silu", "gelu", "relu", "sigmoid"])
    return dict(op=op, fmt=fmt, rows=rows, cols=cols, tokens=tokens, bias=rng.random() < 0.5, act=act,
                residual=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs --

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _weights(fmt, rows, cols, g):
    """uint8 [rows * row bytes]: random blocks whose rows' dots with N(0, 1)
    activations are about N(0, 1), as in a trained layer."""
    _, size, d_at, rms, m_at, ratio = FMT[fmt]
    n = rows * (cols // 256) * size
    raw = torch.empty((n + 3) // 4, dtype=torch.int32, device=DEV).random_(-2**31, 2**31 - 1, generator=g)
    blocks = raw.view(torch.uint8)[:n].view(-1, size)
    d = 1.0 / (rms * math.sqrt(cols))
    for at, r in ((d_at, 1.0), (m_at, ratio)):
        if at is not None:
            v = (torch.rand(blocks.shape[0], generator=g, device=DEV) + 0.5) * (d * r)
            blocks[:, at:at + 2] = v.half().view(torch.uint8).view(-1, 2)
    return blocks.view(-1)


def _q8k(x):
    """The activations as q8_K blocks: f32 scale, 256 int8 values, 16 int16
    sums of 16 values each."""
    b = x.view(x.shape[0], -1, 256)
    amax = b.abs().amax(-1, keepdim=True)
    q = (b * (127.0 / amax)).round().clamp(-127, 127)
    sums = q.view(*q.shape[:2], 16, 16).sum(-1).to(torch.int16).contiguous()
    parts = [(amax / 127.0).contiguous().view(torch.uint8), q.to(torch.int8).view(torch.uint8), sums.view(torch.uint8)]
    return torch.cat(parts, -1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, s = case, {"case": case}
    T = c["tokens"]
    if c["op"] == "route":
        # a trained router: experts of different popularity, logits of a few units
        s["logits"] = 1.5 * _randn(g, T, c["experts"]) + 0.5 * _randn(g, c["experts"]) - 1.0
        s["bias"] = 0.1 * _randn(g, c["experts"]) if c["bias"] else None
        s["ids"] = torch.zeros((T, c["k"]), dtype=torch.int32, device=DEV)
        s["weights"] = torch.zeros((T, c["k"]), device=DEV)
    elif c["op"] == "group":
        E, k, n = c["experts"], c["k"], c["experts"] + c["shared"]
        pop = 0.7 * _randn(g, E)
        s["ids"] = torch.topk(_randn(g, T, E) + pop, k, dim=1).indices.int()
        s["router_weights"] = torch.softmax(_randn(g, T, k), 1)
        # slabs of 1.5 MiB per matrix at addresses the call only computes with
        s["base"] = [1 << 40, 2 << 40, 3 << 40]
        s["stride"] = 3 << 19
        s["shared"] = [tuple((4 << 40) + (3 * i + j) * s["stride"] for j in range(3)) for i in range(c["shared"])]
        s["gptrs"] = torch.zeros((n, 6), dtype=torch.int64, device=DEV)
        s["starts"] = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
        s["pairs"] = torch.zeros(T * (k + c["shared"]), dtype=torch.int32, device=DEV)
        s["slot_weights"] = torch.zeros((T, k + c["shared"]), device=DEV)
    else:
        s["w"] = _weights(c["fmt"], c["rows"], c["cols"], g)
        s["xq"] = _q8k(_randn(g, T, c["cols"]))
        s["bias"] = 0.5 * _randn(g, c["rows"]) if c["bias"] else None
        s["residual"] = _randn(g, T, c["rows"]) if c["residual"] else None
        s["out"] = torch.zeros((T, c["rows"]), device=DEV)
    return s


# ------------------------------------------------------- the plain forms ----

def _route(s):
    """Scores, group scores and order in 64 bits: two experts' scores can lie
    next to each other."""
    c, l = s["case"], s["logits"].double()
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-l))
    else:
        e = torch.exp(l - l.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    key = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        by_group = key.view(len(key), c["groups"], -1)
        best = torch.sort(by_group, dim=-1, descending=True).values[..., :c["group_top"]].sum(-1)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(keep[..., None], by_group, -math.inf).view_as(key)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :c["k"]]
    w = torch.gather(score, 1, ids)
    if c["renorm"]:
        total = w.sum(1, keepdim=True)
        w = w / (total.clamp_min(2.0**-14) if c["score"] == "sigmoid" else total)
    return {"ids": ids.int(), "weights": (w * _scale(c)).float()}


def _scale(c):
    return 2.5 if c["score"] == "sigmoid" else 1.0


def _group(s):
    c, ids = s["case"], s["ids"]
    (T, k), E, extra = ids.shape, c["experts"], c["shared"]
    flat = ids.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    token = torch.arange(T, device=DEV)
    parts = [(order // k) << 4 | order % k] + [token << 4 | k + i for i in range(extra)]
    experts = torch.arange(E + 1, device=DEV)
    starts = torch.searchsorted(flat[order], experts)
    starts = torch.cat([starts] + [starts[-1:] + (i + 1) * T for i in range(extra)])
    gptrs = torch.zeros((E + extra, 6), dtype=torch.int64, device=DEV)
    for j in range(3):
        gptrs[:E, j] = s["base"][j] + experts[:E] * s["stride"]
        for i in range(extra):
            gptrs[E + i, j] = s["shared"][i][j]
    w = torch.cat([s["router_weights"], torch.ones((T, extra), device=DEV)], 1)
    return {"gptrs": gptrs, "starts": starts.int(), "pairs": torch.cat(parts).int(), "slot_weights": w}


def _f16(b, at):
    return b[..., at:at + 2].contiguous().view(torch.float16).float()


_IQ4 = [-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113]


def _kscales(b):
    """The 8 six-bit scales and mins packed in 12 bytes."""
    lo, mid, hi = b[..., 4:8], b[..., 8:12], b[..., 12:16]
    sc = torch.cat([lo & 63, (hi & 15) | (lo >> 6) << 4], -1)
    mn = torch.cat([mid & 63, (hi >> 4) | (mid >> 6) << 4], -1)
    return sc.float(), mn.float()


def _dequant(fmt, raw, rows, cols):
    """f32 [rows][cols] of the format's blocks."""
    b = raw.view(rows, cols // 256, FMT[fmt][1])
    n = b.shape[:2]
    two = torch.tensor([0, 2, 4, 6], dtype=torch.uint8, device=DEV).view(4, 1)
    bit = torch.arange(8, dtype=torch.uint8, device=DEV).view(8, 1)
    if fmt in ("Q4_K", "Q5_K"):
        q = b[..., -128:].reshape(*n, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], -2).reshape(*n, 8, 32)
        if fmt == "Q5_K":
            q = q + ((b[..., None, 16:48] >> bit & 1) << 4)
        sc, mn = _kscales(b)
        w = (_f16(b, 0) * sc)[..., None] * q - (_f16(b, 2) * mn)[..., None]
    elif fmt == "Q2_K":
        q = (b[..., 16:80].reshape(*n, 2, 1, 32) >> two & 3).reshape(*n, 16, 16)
        sc = b[..., :16]
        w = (_f16(b, 80) * (sc & 15))[..., None] * q - (_f16(b, 82) * (sc >> 4))[..., None]
    elif fmt == "Q3_K":
        q = b[..., 32:96].reshape(*n, 2, 1, 32) >> two & 3
        high = (b[..., None, :32] >> bit & 1).reshape(*n, 2, 4, 32)
        q = (q + 4 * high).float().reshape(*n, 16, 16) - 4
        sc = b[..., 96:108]
        low = torch.cat([sc[..., :8] & 15, sc[..., :8] >> 4], -1)
        top = torch.cat([sc[..., 8:] >> 2 * j & 3 for j in range(4)], -1)
        w = (_f16(b, 108) * ((low | top << 4).float() - 32))[..., None] * q
    elif fmt == "Q6_K":
        low = b[..., :128].reshape(*n, 2, 1, 64)
        low = torch.cat([low & 15, low >> 4], -2).reshape(*n, 2, 4, 32)
        top = b[..., 128:192].reshape(*n, 2, 1, 32) >> two & 3
        q = ((low | top << 4).float() - 32).reshape(*n, 16, 16)
        w = (_f16(b, 208) * b[..., 192:208].contiguous().view(torch.int8))[..., None] * q
    else:  # IQ4_XS
        q = b[..., 8:].reshape(*n, 8, 16)
        q = torch.tensor(_IQ4, dtype=torch.float32, device=DEV)[torch.cat([q & 15, q >> 4], -1).int()]
        low = torch.stack([b[..., 4:8] & 15, b[..., 4:8] >> 4], -1).reshape(*n, 8)
        top = torch.cat([b[..., 2 + j // 4:3 + j // 4] >> 2 * (j % 4) & 3 for j in range(8)], -1)
        w = (_f16(b, 0) * ((low | top << 4).float() - 32))[..., None] * q
    return w.reshape(rows, cols)


def _act(name, v):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "gelu":
        return v / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "relu":
        return v.clamp_min(0.0)
    return 1.0 / (1.0 + torch.exp(-v)) if name == "sigmoid" else v


def _product(s):
    c, b = s["case"], s["xq"]
    x = b[..., :4].contiguous().view(torch.float32) * b[..., 4:260].contiguous().view(torch.int8)
    v = x.view(c["tokens"], c["cols"]) @ _dequant(c["fmt"], s["w"], c["rows"], c["cols"]).T
    if s["bias"] is not None:
        v = v + s["bias"]
    v = _act(c["act"], v)
    return v if s["residual"] is None else v + s["residual"]


# -------------------------------------------------------------------- run --

def _call(s):
    from pulsar_amd import kernels as K

    c = s["case"]
    if c["op"] == "route":
        K.router_select_groups(s["ids"], s["weights"], s["logits"], s["bias"], c["experts"], c["k"], c["groups"],
                               c["top_groups"], c["group_top"], SCORES[c["score"]], c["renorm"], _scale(c), c["tokens"])
        return {"ids": s["ids"], "weights": s["weights"]}
    if c["op"] == "group":
        if "bank" not in s:
            s["bank"] = K.ExpertBank(*s["base"], None, None, None, *[s["stride"]] * 3, 0, 0, 0)
        K.moe_group_ids(s["gptrs"], s["starts"], s["pairs"], s["slot_weights"], s["ids"], s["router_weights"],
                        s["bank"], c["experts"], s["shared"], c["tokens"], c["k"])
        return {n: s[n] for n in ("gptrs", "starts", "pairs", "slot_weights")}
    code, size = FMT[c["fmt"]][:2]
    K.matmul_kq_fused(s["out"], s["w"], s["xq"], s["bias"], s["residual"], c["cols"], c["rows"], c["tokens"],
                      c["cols"] // 256 * size, code, ACTS[c["act"]])
    return s["out"]


def run(s):
    if own:
        return _call(s)
    return {"route": _route, "group": _group, "product": _product}[s["case"]["op"]](s)


def work(c):
    T = c["tokens"]
    if c["op"] == "route":
        E = c["experts"]
        return {"bytes": 4 * T * E + 8 * T * c["k"] + (4 * E if c["bias"] else 0), "flops": 8 * T * E}
    if c["op"] == "group":
        slots, groups = c["k"] + c["shared"], c["experts"] + c["shared"]
        return {"bytes": 8 * T * c["k"] + 8 * T * slots + 52 * groups, "flops": 4 * T * slots}
    rows, cols = c["rows"], c["cols"]
    out = 4 * T * rows * (2 if c["residual"] else 1)
    return {"bytes": rows * (cols // 256) * FMT[c["fmt"]][1] + T * (cols // 256) * 292 + out
            + (4 * rows if c["bias"] else 0), "flops": 2 * T * rows * cols}


# ------------------------------------------------------------------ exact --

def _exact_route(c, s):
    l = s["logits"].cpu().numpy().astype(np.float64)
    e = np.exp(-np.abs(l))
    if c["score"] == "sigmoid":
        score = np.where(l >= 0, 1.0, e) / (1.0 + e)
    else:
        score = np.exp(l - l.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    key = score + (0.0 if s["bias"] is None else s["bias"].cpu().numpy().astype(np.float64))
    T, E = key.shape
    row, size = np.arange(T), E // c["groups"]
    if c["groups"] > 1:
        parted = np.sort(key.reshape(T, c["groups"], size), axis=2)
        total = parted[..., -min(size, c["group_top"]):].sum(2)
        kept = np.zeros(total.shape, bool)
        for _ in range(c["top_groups"]):  # argmax: the first of equals
            at = total.argmax(1)
            kept[row, at], total[row, at] = True, -np.inf
        key = np.where(np.repeat(kept, size, 1), key, -np.inf)
    ids = np.zeros((T, c["k"]), np.int32)
    for j in range(c["k"]):
        ids[:, j] = key.argmax(1)
        key[row, ids[:, j]] = -np.inf
    w = score[row[:, None], ids]
    if c["renorm"]:
        total = w.sum(1, keepdims=True)
        w = w / (np.maximum(total, 2.0**-14) if c["score"] == "sigmoid" else total)
    return {"ids": torch.from_numpy(ids), "weights": torch.from_numpy(w * _scale(c))}


def _exact_group(c, s):
    ids = s["ids"].cpu().numpy()
    T, k = ids.shape
    lists = [[] for _ in range(c["experts"] + c["shared"])]
    for t, row in enumerate(ids.tolist()):
        for slot, e in enumerate(row):
            lists[e].append(t << 4 | slot)
    for i in range(c["shared"]):
        lists[c["experts"] + i] = [t << 4 | k + i for t in range(T)]
    starts = np.cumsum([0] + [len(p) for p in lists])
    at = [[b + e * s["stride"] for b in s["base"]] + [0] * 3 for e in range(c["experts"])]
    at += [list(p) + [0] * 3 for p in s["shared"]]
    w = np.ones((T, k + c["shared"]))
    w[:, :k] = s["router_weights"].cpu().numpy()
    return {"gptrs": torch.tensor(at, dtype=torch.int64), "starts": torch.from_numpy(starts.astype(np.int32)),
            "pairs": torch.tensor([p for part in lists for p in part], dtype=torch.int32),
            "slot_weights": torch.from_numpy(w)}


def _codes(fmt):
    """Per value 0..255 of a block: the byte its low bits are in, their shift
    and mask, the byte of its high bits (-1: none), their shift, mask and
    weight, its scale group."""
    v = np.arange(256)
    none = np.full(256, -1)
    if fmt in ("Q4_K", "Q5_K"):
        high = (16 + v % 32, v // 32, 1, 16) if fmt == "Q5_K" else (none, 0 * v, 0, 0)
        return (FMT[fmt][1] - 128 + v // 64 * 32 + v % 32, v // 32 % 2 * 4, 15, *high, v // 32)
    if fmt == "Q2_K":
        return (16 + v // 128 * 32 + v % 32, v // 32 % 4 * 2, 3, none, 0 * v, 0, 0, v // 16)
    if fmt == "Q3_K":
        return (32 + v // 128 * 32 + v % 32, v // 32 % 4 * 2, 3, v % 32, v // 32, 1, 4, v // 16)
    if fmt == "Q6_K":
        return (v // 128 * 64 + v % 64, v // 64 % 2 * 4, 15, 128 + v // 128 * 32 + v % 32, v // 32 % 4 * 2, 3, 16, v // 16)
    return (8 + v // 32 * 16 + v % 16, v // 16 % 2 * 4, 15, none, 0 * v, 0, 0, v // 32)


def _scale_bits(fmt, b):
    """float64 [blocks][groups]: scales and mins of every group, with the
    block's own factors."""
    at = lambda j: b[:, j].double()  # noqa: E731
    low = lambda j, n: at(j).remainder(n)  # noqa: E731
    top = lambda j, n: torch.floor(at(j) / n)  # noqa: E731
    half = lambda j: b[:, j:j + 2].contiguous().view(torch.float16).double()  # noqa: E731
    if fmt in ("Q4_K", "Q5_K"):
        sc = [low(4 + j, 64) if j < 4 else low(8 + j, 16) + 16 * top(j, 64) for j in range(8)]
        mn = [low(8 + j, 64) if j < 4 else top(8 + j, 16) + 16 * top(4 + j, 64) for j in range(8)]
        return half(0) * torch.stack(sc, 1), half(2) * torch.stack(mn, 1)
    if fmt == "Q2_K":
        return (half(80) * torch.stack([low(j, 16) for j in range(16)], 1),
                half(82) * torch.stack([top(j, 16) for j in range(16)], 1))
    if fmt == "Q3_K":
        four = [low(96 + j, 16) if j < 8 else top(88 + j, 16) for j in range(16)]
        two = [torch.floor(at(104 + j % 4) / 4 ** (j // 4)).remainder(4) for j in range(16)]
        return half(108) * (torch.stack(four, 1) + 16 * torch.stack(two, 1) - 32), None
    if fmt == "Q6_K":
        return half(208) * b[:, 192:208].contiguous().view(torch.int8).double(), None
    four = [low(4 + j // 2, 16) if j % 2 == 0 else top(4 + j // 2, 16) for j in range(8)]
    two = [torch.floor(at(2 + j // 4) / 4 ** (j % 4)).remainder(4) for j in range(8)]
    return half(0) * (torch.stack(four, 1) + 16 * torch.stack(two, 1) - 32), None


def _exact_product(c, s):
    """Rows in parts: the codes gathered value by value, the sums in 64 bits."""
    fmt, (T, rows, cols) = c["fmt"], (c["tokens"], c["rows"], c["cols"])
    idx = [torch.as_tensor(a, device=DEV) for a in _codes(fmt)]
    byte, shift, mask, hbyte, hshift, hmask, hweight, group = idx
    xb = s["xq"]
    x = xb[..., 4:260].contiguous().view(torch.int8).double() * xb[..., :4].contiguous().view(torch.float32).double()
    x = x.view(T, cols)
    out = torch.empty((T, rows), dtype=torch.float64, device=DEV)
    step = max(1, 16_000_000 // cols)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        per = cols // 256 * FMT[fmt][1]
        b = s["w"][r * per:(r + n) * per].view(-1, FMT[fmt][1])
        code = (b[:, byte].int() >> shift) & mask
        if int(hweight):
            code = code + ((b[:, hbyte].int() >> hshift) & hmask) * hweight
        if fmt == "IQ4_XS":
            code = torch.tensor(_IQ4, dtype=torch.float64, device=DEV)[code]
        else:
            code = code.double() - {"Q6_K": 32, "Q3_K": 4}.get(fmt, 0)
        sc, mn = _scale_bits(fmt, b)
        w = sc[:, group] * code
        if mn is not None:
            w = w - mn[:, group]
        out[:, r:r + n] = x @ w.view(n, cols).T
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
    return {"route": _exact_route, "group": _exact_group, "product": _exact_product}[case["op"]](case, s)
