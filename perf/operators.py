"""The operators around the expert layer, as measurable cases: each in its plain form (elementary torch operations) and
through this package.

  route   moe_route_grouped: sigmoid or softmax scores, a balance bias, groups of experts, top-k, gates.
  norm    add_rms_norm: the residual's addition, the root-mean-square norm, rows in 16 or in 8 bits.
  linear  quant_matmul: int8 rows and weights with a scale for each token and each channel.
  block   add_rms_norm with int8 rows, then quant_matmul on them: the entry of a quantised layer.

Ranges: 1 to 65536 tokens over 8 to 512 experts; 1 to 32768 rows of 64 to 8192 columns; products of 1 to 8192 rows,
16 to 16384 deep, up to 32768 wide.
"""
import math

import torch

own = False
DEV = "cuda:0"
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
QUANT = {"none": 0, "int8": 2, "fp8": 3}
EPS = 1e-6


def listed():
    return [
        # the next token of a single user: a launch and nothing else
        dict(name="route_one_token", kind="route", T=1, E=256, K=8, G=8, KG=4, score="sigmoid", group="top2", bias=True,
             renorm=True, scaling=2.5, dtype="fp32"),
        # a decode batch on softmax scores, the best of each group counts, gates as they are; bf16 logits, whose ties
        # fall to the lower id
        dict(name="route_decode_softmax", kind="route", T=128, E=160, K=6, G=8, KG=3, score="softmax", group="max",
             bias=False, renorm=False, scaling=16.0, dtype="bf16"),
        # a long prefill in one call: the largest token count that the routing takes
        dict(name="route_long_prefill", kind="route", T=65536, E=256, K=8, G=8, KG=4, score="sigmoid", group="top2",
             bias=True, renorm=True, scaling=2.5, dtype="fp32"),
        # the rows of a small decode batch, in int8 for the product behind them
        dict(name="norm_decode_int8", kind="norm", T=16, H=7168, stride=7168, residual=True, quant="int8", dtype="bf16"),
        # the compressed part of wider rows: a slice with a stride of its own and no residual
        dict(name="norm_slice", kind="norm", T=4096, H=512, stride=576, residual=False, quant="none", dtype="bf16"),
        # a prefill chunk in e4m3 with scales for 128 columns, as the fp8 expert GEMMs read it
        dict(name="norm_prefill_fp8", kind="norm", T=4096, H=7168, stride=7168, residual=True, quant="fp8", dtype="bf16"),
        # a long prefill, rows kept in 16 bits
        dict(name="norm_long_prefill", kind="norm", T=32768, H=7168, stride=7168, residual=True, quant="none",
             dtype="bf16"),
        # one token through a projection: the weights' stream
        dict(name="linear_one_token", kind="linear", M=1, K=7168, N=4096, bias=False, out="bf16"),
        # a decode batch of 128 sequences through the same projection
        dict(name="linear_decode", kind="linear", M=128, K=7168, N=4096, bias=False, out="bf16"),
        # a ragged prompt, an odd width, a bias, fp16 out
        dict(name="linear_ragged", kind="linear", M=1021, K=5120, N=5001, bias=True, out="fp16"),
        # both halves of a wide MLP's first product over a prefill chunk: bound by the matrix cores
        dict(name="linear_prefill", kind="linear", M=8192, K=4096, N=28672, bias=False, out="bf16"),
        # the entry of a quantised layer in a decode step: the norm's int8 rows go into a product
        dict(name="block_decode", kind="block", T=64, H=7168, N=4096, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one_draw(rng):
    kind = rng.choice(["route", "route", "norm", "norm", "linear", "linear", "linear", "block"])
    if kind == "route":
        E = rng.choice([8, 16, 60, 64, 72, 128, 160, 256, 384, 512])
        G = rng.choice([g for g in (1, 2, 3, 4, 6, 8, 16) if E % g == 0 and E // g >= 4])
        KG = rng.randint(1, G)
        return dict(kind=kind, T=_log_int(rng, 1, 65536), E=E, K=rng.randint(1, min(16, KG * (E // G))), G=G, KG=KG,
                    score=rng.choice(["sigmoid", "softmax"]), group=rng.choice(["top2", "max"]),
                    bias=rng.random() < 0.6, renorm=rng.random() < 0.6, scaling=rng.choice([1.0, 2.5, 16.0]),
                    dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
    if kind == "norm":
        quant = rng.choice(["none", "none", "int8", "fp8"])
        H = _log_int(rng, 64, 8192)
        H = 128 * max(1, H // 128) if quant == "fp8" else 8 * max(8, H // 8) if rng.random() < 0.6 else H
        return dict(kind=kind, T=_log_int(rng, 1, 32768), H=H, stride=H + rng.choice([0, 0, 64, 8 * rng.randint(1, 64)]),
                    residual=rng.random() < 0.7, quant=quant, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "linear":
        return dict(kind=kind, M=_log_int(rng, 1, 8192), K=16 * _log_int(rng, 1, 1024), N=_log_int(rng, 1, 32768),
                    bias=rng.random() < 0.4, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    return dict(kind=kind, T=_log_int(rng, 1, 4096), H=16 * _log_int(rng, 4, 512), N=_log_int(rng, 16, 16384),
                dtype=rng.choice(["bf16", "fp16"]))


def draw(rng):
    most = [work(c) for c in listed()]
    top = {q: max(w[q] for w in most) for q in ("bytes", "flops")}
    while True:
        c = _one_draw(rng)
        w = work(c)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rows(T, H, g, dtype):
    """Activations: a scale for each token, and a few columns that are far larger than the others."""
    x = torch.randn(T, H, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(T, 1, generator=g, device=DEV))
    return (x * torch.exp(0.6 * torch.randn(1, H, generator=g, device=DEV))).to(DTYPE[dtype])


def _int8_rows(T, K, g):
    x = torch.randn(T, K, generator=g, device=DEV) * torch.exp(0.4 * torch.randn(1, K, generator=g, device=DEV))
    s = x.abs().amax(dim=1).clamp(min=1e-6) / 127.0
    return x.div_(s[:, None]).round_().clamp_(-127, 127).to(torch.int8), s


def _int8_weight(N, K, g):
    w = torch.randn(N, K, generator=g, device=DEV).mul_(0.02)
    s = w.abs().amax(dim=1).clamp(min=1e-6) / 127.0
    return w.div_(s[:, None]).round_().clamp_(-127, 127).to(torch.int8), s


def _norm_weight(H, g, dtype):
    return (1.0 + 0.2 * torch.randn(H, generator=g, device=DEV)).to(DTYPE[dtype])


def prepare(c, seed):
    g = _gen(seed)
    kind = c["kind"]
    s = {"c": c}
    if kind == "route":
        s["logits"] = (torch.randn(c["T"], c["E"], generator=g, device=DEV) * 1.5).to(DTYPE[c["dtype"]])
        s["bias"] = 0.1 * torch.randn(c["E"], generator=g, device=DEV) if c["bias"] else None
    elif kind == "norm":
        s["x"] = _rows(c["T"], c["stride"], g, c["dtype"])[:, :c["H"]]
        s["residual"] = _rows(c["T"], c["H"], g, c["dtype"]) if c["residual"] else None
        s["weight"] = _norm_weight(c["H"], g, c["dtype"])
    elif kind == "linear":
        s["x"], s["xs"] = _int8_rows(c["M"], c["K"], g)
        s["w"], s["ws"] = _int8_weight(c["N"], c["K"], g)
        s["bias"] = torch.randn(c["N"], generator=g, device=DEV) if c["bias"] else None
    else:
        s["x"] = _rows(c["T"], c["H"], g, c["dtype"])
        s["residual"] = _rows(c["T"], c["H"], g, c["dtype"])
        s["weight"] = _norm_weight(c["H"], g, c["dtype"])
        s["w"], s["ws"] = _int8_weight(c["N"], c["H"], g)
    return s


# ---------------------------------------------------------------- the plain forms
def _plain_route(c, logits, bias):
    """In 64 bits: which of two experts comes first can hang on the last bits of their scores."""
    T, E, K, G = c["T"], c["E"], c["K"], c["G"]
    l = logits.double()
    if c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        e = torch.exp(l - l.amax(dim=1, keepdim=True))
        s = e / e.sum(dim=1, keepdim=True)
    order = s if bias is None else s + bias.double()
    if G > 1:
        by_group = order.view(T, G, E // G)
        best = by_group.sort(dim=2, descending=True).values[:, :, : 2 if c["group"] == "top2" else 1].sum(dim=2)
        kept = torch.zeros(T, G, dtype=torch.bool, device=l.device)
        kept.scatter_(1, best.sort(dim=1, descending=True, stable=True).indices[:, : c["KG"]], True)
        order = torch.where(kept[:, :, None], by_group, -math.inf).view(T, E)
    idx = order.sort(dim=1, descending=True, stable=True).indices[:, :K]
    w = s.gather(1, idx)
    if c["renorm"]:
        w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return idx.int(), (w * c["scaling"]).float()


def _plain_norm(x, residual, weight, quant):
    """(rows or codes in 32 bits, scales or None, the new residual or None)."""
    v = x.float() if residual is None else x.float() + residual.float()
    r = torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS)
    t = v * weight.float()
    new = None if residual is None else v.to(x.dtype)
    if quant == "none":
        return (t * r).to(x.dtype), None, new
    if quant == "int8":
        a = t.abs().amax(dim=1, keepdim=True)
        return torch.round(t * (torch.full_like(a, 127.0) / a)), (a / 127.0 * r)[:, 0], new
    b = t.view(x.shape[0], -1, 128)
    a = b.abs().amax(dim=2, keepdim=True)
    return (b * (torch.full_like(a, 448.0) / a)).view_as(t), a[:, :, 0] / 448.0 * r, new


def _plain_linear(x, xs, w, ws, bias, dtype):
    y = (x.float() @ w.float().t()) * ws * xs[:, None]
    return (y if bias is None else y + bias).to(dtype)


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["c"]
    kind = c["kind"]
    if own:
        from umdk_amd import add_rms_norm, moe_route_grouped, quant_matmul
    if kind == "route":
        if own:
            return moe_route_grouped(s["logits"], s["bias"], c["K"], c["G"], c["KG"], c["score"], c["group"], c["renorm"],
                                     c["scaling"])
        return _plain_route(c, s["logits"], s["bias"])
    if kind == "norm":
        if own:
            y, scale, new = add_rms_norm(s["x"], s["residual"], s["weight"], EPS, QUANT[c["quant"]])
        else:
            y, scale, new = _plain_norm(s["x"], s["residual"], s["weight"], c["quant"])
        r = {} if s["residual"] is None else {"residual": new}
        if c["quant"] == "int8":  # as the values that the codes stand for, in the rows' own type
            r["y"] = torch.mul(y, scale[:, None], out=torch.empty_like(s["x"], memory_format=torch.contiguous_format))
        else:
            r["y"] = y if c["quant"] == "none" else y.to(torch.float8_e4m3fn)
        if c["quant"] != "none":
            r["scale"] = scale
        return r
    if kind == "linear":
        if own:
            return quant_matmul(s["x"], s["xs"], s["w"], s["ws"], s["bias"], DTYPE[c["out"]])
        return _plain_linear(s["x"], s["xs"], s["w"], s["ws"], s["bias"], DTYPE[c["out"]])
    if own:
        q, scale, new = add_rms_norm(s["x"], s["residual"], s["weight"], EPS, QUANT["int8"])
        return {"residual": new, "out": quant_matmul(q, scale, s["w"], s["ws"], None, DTYPE[c["dtype"]])}
    q, scale, new = _plain_norm(s["x"], s["residual"], s["weight"], "int8")
    return {"residual": new, "out": _plain_linear(q, scale, s["w"], s["ws"], None, DTYPE[c["dtype"]])}


# ---------------------------------------------------------------- what a pass cannot do without
def _norm_bytes(T, H, residual, quant):
    return T * H * (2 + (4 if residual else 0)) + T * {"none": 2 * H, "int8": H + 4, "fp8": H + H // 32}[quant] + 2 * H


def _linear_bytes(M, N, K, size):
    return M * K + N * K + M * N * size + 4 * (M + N)


def work(c):
    if c["kind"] == "route":
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": c["T"] * (size * c["E"] + 8 * c["K"]) + (4 * c["E"] if c["bias"] else 0),
                "flops": c["T"] * c["E"] * 4}
    if c["kind"] == "norm":
        return {"bytes": _norm_bytes(c["T"], c["H"], c["residual"], c["quant"]), "flops": 5 * c["T"] * c["H"]}
    if c["kind"] == "linear":
        return {"bytes": _linear_bytes(c["M"], c["N"], c["K"], 4 if c["out"] == "fp32" else 2),
                "flops": 2 * c["M"] * c["N"] * c["K"]}
    T, H, N = c["T"], c["H"], c["N"]
    return {"bytes": T * H * 6 + 2 * H + N * H + 4 * N + 2 * T * N, "flops": 5 * T * H + 2 * T * N * H}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def _exact_route(c, s):
    T, E, K, G = c["T"], c["E"], c["K"], c["G"]
    l = s["logits"].to(torch.float64)
    score = torch.sigmoid(l) if c["score"] == "sigmoid" else torch.softmax(l, dim=1)
    rank = score.clone() if s["bias"] is None else score + s["bias"].to(torch.float64)
    expert = torch.arange(E, device=l.device)
    if G > 1:
        group = torch.empty(T, G, dtype=torch.float64, device=l.device)
        for i in range(G):
            part = rank[:, i * (E // G):(i + 1) * (E // G)]
            group[:, i] = part.topk(2 if c["group"] == "top2" else 1, dim=1).values.sum(dim=1)
        allowed = torch.zeros(T, E, dtype=torch.bool, device=l.device)
        for _ in range(c["KG"]):
            best = group.max(dim=1).indices  # the first of equal ones
            allowed |= (expert // (E // G))[None, :] == best[:, None]
            group.scatter_(1, best[:, None], -math.inf)
        rank.masked_fill_(~allowed, -math.inf)
    ids = torch.empty(T, K, dtype=torch.int64, device=l.device)
    for k in range(K):
        ids[:, k] = rank.max(dim=1).indices
        rank.scatter_(1, ids[:, k:k + 1], -math.inf)
    gate = torch.gather(score, 1, ids)
    if c["renorm"]:
        gate = gate / gate.sum(dim=1, keepdim=True)
    return ids.to(torch.int32), gate * c["scaling"]


def _exact_norm(s, quant):
    v = s["x"].to(torch.float64)
    if s["residual"] is not None:
        v = v + s["residual"].to(torch.float64)
    y = v / torch.sqrt((v * v).sum(dim=1, keepdim=True) / v.shape[1] + EPS) * s["weight"].to(torch.float64)
    if quant == "none":
        return y, None, v
    width, most = (v.shape[1], 127.0) if quant == "int8" else (128, 448.0)
    blocks = y.reshape(y.shape[0], -1, width)
    step = blocks.abs().amax(dim=2, keepdim=True) / most
    codes = blocks / step
    codes = torch.round(codes) if quant == "int8" else codes.to(torch.float32).to(torch.float8_e4m3fn).to(torch.float64)
    return codes.reshape(y.shape), step[:, :, 0], v


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "route":
        return _exact_route(c, s)
    if c["kind"] == "norm":
        y, step, v = _exact_norm(s, c["quant"])
        r = {} if s["residual"] is None else {"residual": v}
        r["y"] = y * step if c["quant"] == "int8" else y
        if c["quant"] != "none":
            r["scale"] = step[:, 0] if c["quant"] == "int8" else step
        return r
    if c["kind"] == "linear":
        y = torch.matmul(s["x"].to(torch.float64), s["w"].to(torch.float64).t().contiguous())
        y.mul_(s["ws"].to(torch.float64)[None, :]).mul_(s["xs"].to(torch.float64)[:, None])
        return y if s["bias"] is None else y.add_(s["bias"].to(torch.float64)[None, :])
    q, step, v = _exact_norm(s, "int8")
    y = torch.matmul(q, s["w"].to(torch.float64).t().contiguous())
    return {"residual": v, "out": y * s["ws"].to(torch.float64)[None, :] * step}
