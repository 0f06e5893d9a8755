"""The operators of a decode step of a few requests, as measurable cases: each in its plain form (elementary torch
operations) and through this package.

  layer   moe_decode_layer: a whole expert layer (router product, grouped routing, experts, shared expert) of 1 to 16 tokens.
  lora    lora_add: the low-rank adapters of many requests beside a shared projection.
  entry   add_rms_norm with int8 rows, quant_matmul on them, and lora_add on the same rows: a quantised projection whose
          requests have adapters.

Ranges: 1 to 16 tokens through 8 to 256 experts of 128 to 14336 by 512 to 8192, weights in bf16, int8 or fp8; 1 to 16384
rows with 1 to 64 adapters of rank 8 to 256, projections 16 to 16384 deep and 1 to 16384 wide.
"""
import math

import torch

own = False
DEV = "cuda:0"
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # the next token of a single user on a small model: launches and latency
        dict(name="layer_one_token_small", kind="layer", T=1, H=1024, E=8, K=2, I=512, shared=0, G=1, KG=1, score="softmax",
             group="max", bias=False, router="fp32", dtype="bf16"),
        # the next token of a single user on a large one: the stream of its experts' weights
        dict(name="layer_one_token_fp8", kind="layer", T=1, H=7168, E=64, K=8, I=2048, shared=2048, G=8, KG=4,
             score="sigmoid", group="top2", bias=True, router="fp32", dtype="fp8"),
        # a few users of a model with few wide experts
        dict(name="layer_wide_int8", kind="layer", T=4, H=4096, E=8, K=2, I=14336, shared=0, G=1, KG=1, score="softmax",
             group="max", bias=False, router="bf16", dtype="int8"),
        # a draft of a few tokens to verify, many narrow experts and a shared one, widths that are no power of two
        dict(name="layer_ragged_bf16", kind="layer", T=7, H=5120, E=160, K=6, I=1408, shared=2816, G=8, KG=3, score="softmax",
             group="max", bias=False, router="fp32", dtype="bf16"),
        # the largest batch that the operator takes: most experts have a token or two
        dict(name="layer_batch_fp8", kind="layer", T=16, H=7168, E=64, K=8, I=2048, shared=2048, G=8, KG=4, score="sigmoid",
             group="top2", bias=True, router="bf16", dtype="fp8"),
        # one request's adapter at one token
        dict(name="lora_one_token", kind="lora", M=1, K=4096, N=4096, L=8, R=16, rows="bf16", base="bf16", dtype="bf16",
             spread="token", none=0.0),
        # a decode batch on int8 rows, about as many adapters as there are, the projection not yet rounded
        dict(name="lora_decode_int8", kind="lora", M=64, K=7168, N=4096, L=32, R=16, rows="int8", base="fp32", dtype="bf16",
             spread="token", none=0.1),
        # a larger decode batch, higher rank, odd width, fp16, a third of the requests without an adapter
        dict(name="lora_decode_ragged", kind="lora", M=200, K=5120, N=5001, L=20, R=64, rows="fp16", base="fp16",
             dtype="fp16", spread="token", none=0.33),
        # a handful of prompts in one batch, each with its adapter
        dict(name="lora_prompts", kind="lora", M=1021, K=4096, N=4096, L=6, R=32, rows="bf16", base="bf16", dtype="bf16",
             spread="prompt", none=0.2),
        # a long prefill through the widest projection
        dict(name="lora_long_prefill", kind="lora", M=16384, K=4096, N=14336, L=8, R=64, rows="bf16", base="bf16",
             dtype="bf16", spread="prompt", none=0.1),
        # the entry of a quantised layer in a decode step whose requests have adapters
        dict(name="entry_decode", kind="entry", M=32, K=7168, N=4096, L=16, R=32, dtype="bf16", spread="token", none=0.2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one_draw(rng):
    kind = rng.choice(["layer", "layer", "layer", "lora", "lora", "lora", "entry"])
    if kind == "layer":
        E = rng.choice([8, 16, 32, 60, 64, 72, 128, 160, 256])
        G = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 4])
        KG = rng.randint(1, G)
        dtype = rng.choice(["bf16", "int8", "fp8"])
        unit = 128 if dtype == "fp8" else 64
        return dict(kind=kind, T=rng.randint(1, 16), H=unit * _log_int(rng, 512 // unit, 8192 // unit), E=E,
                    K=rng.randint(1, min(8, KG * (E // G))), I=unit * _log_int(rng, 128 // unit, 14336 // unit),
                    shared=unit * _log_int(rng, 128 // unit, 4096 // unit) if rng.random() < 0.5 else 0, G=G, KG=KG,
                    score=rng.choice(["sigmoid", "softmax"]), group=rng.choice(["top2", "max"]), bias=rng.random() < 0.5,
                    router=rng.choice(["fp32", "bf16"]), dtype=dtype)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    spread = rng.choice(["token", "token", "prompt"])
    c = dict(kind=kind, M=_log_int(rng, 1, 512) if spread == "token" else _log_int(rng, 64, 16384),
             K=16 * _log_int(rng, 1, 1024), N=_log_int(rng, 1, 16384), L=rng.randint(1, 64), R=8 * _log_int(rng, 1, 32),
             dtype=dtype, spread=spread, none=rng.choice([0.0, 0.1, 0.5]))
    if kind == "entry":
        c["K"] = min(c["K"], 16384)
        c["M"] = min(c["M"], 512)
        return c
    return dict(c, rows=rng.choice([dtype, "int8"]), base=rng.choice([dtype, dtype, "fp32"]))


def _kept_bytes(c):
    """What the weights of a case take."""
    if c["kind"] != "layer":
        return 2 * c["L"] * c["R"] * (c["K"] + c["N"])
    return 3 * c["H"] * (c["E"] * c["I"] + c["shared"]) * (2 if c["dtype"] == "bf16" else 1)


def draw(rng):
    most = [work(c) for c in listed()]
    top = {q: max(w[q] for w in most) for q in ("bytes", "flops")}
    kept = max(_kept_bytes(c) for c in listed())
    while True:
        c = _one_draw(rng)
        w = work(c)
        # (all adapters' products, as the plain form takes them, stay within a few times the largest listed case's)
        if (w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and _kept_bytes(c) <= kept
                and (c["kind"] == "layer" or c["M"] * c["L"] * c["R"] <= 1 << 24)):
            return c


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rows(T, H, g, dtype):
    """Rows as a norm leaves them: the same size for every token, some columns larger than others."""
    x = torch.randn(T, H, generator=g, device=DEV)
    return (x * torch.exp(0.4 * torch.randn(1, H, generator=g, device=DEV))).to(DTYPE[dtype])


def _int8_rows(T, H, g):
    x = torch.randn(T, H, generator=g, device=DEV) * torch.exp(0.4 * torch.randn(1, H, generator=g, device=DEV))
    s = x.abs().amax(dim=1).clamp(min=1e-6) / 127.0
    return x.div_(s[:, None]).round_().clamp_(-127, 127).to(torch.int8), s


def _weight(lead, n, k, dtype, g):
    """[lead..., n, k] weights ~ N(0, 1 / k) and their scales: int8 per channel, fp8 per 128 x 128 block."""
    count = max(1, math.prod(lead))
    w = torch.empty(count, n, k, device=DEV, dtype={"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}[dtype])
    s = None if dtype == "bf16" else torch.empty((count, n) if dtype == "int8" else (count, n // 128, k // 128), device=DEV)
    for e in range(count):
        v = torch.randn(n, k, generator=g, device=DEV).mul_(k ** -0.5)
        if dtype == "int8":
            s[e] = v.abs().amax(dim=1) / 127.0
            v = v.div_(s[e][:, None]).round_()
        elif dtype == "fp8":
            b = v.view(n // 128, 128, k // 128, 128)
            s[e] = b.abs().amax(dim=(1, 3)) / 448.0
            v = b.div_(s[e][:, None, :, None]).view(n, k)
        w[e] = v.to(w.dtype)
    return w.view(*lead, n, k), None if s is None else s.view(*lead, *s.shape[1:])


def _adapters(c, g):
    """The adapter of each row: drawn for every row, or for every prompt of a batch (runs of rows); -1: none."""
    M, L = c["M"], c["L"]
    if c["spread"] == "token":
        owner = torch.arange(M, device=DEV)
    else:
        ends = torch.rand(max(1, min(12, M // 40)) - 1, generator=g, device=DEV).mul_(M).long()
        owner = (torch.arange(M, device=DEV)[:, None] >= ends[None, :]).sum(dim=1)
    ids = torch.randint(0, L, (M,), generator=g, device=DEV)
    ids = torch.where(torch.rand(M, generator=g, device=DEV) < c["none"], -1, ids)
    return ids[owner].to(torch.int32)


def prepare(c, seed):
    g = _gen(seed)
    s = {"c": c}
    if c["kind"] == "layer":
        H, E, I, sh, dt = c["H"], c["E"], c["I"], c["shared"], c["dtype"]
        s["x"] = _rows(c["T"], H, g, "bf16")
        s["router"] = torch.randn(E, H, generator=g, device=DEV).mul_(1.2 * H ** -0.5).to(DTYPE[c["router"]])
        s["bias"] = 0.1 * torch.randn(E, generator=g, device=DEV) if c["bias"] else None
        s["w1"], s["s1"] = _weight((E,), 2 * I, H, dt, g)
        s["w2"], s["s2"] = _weight((E,), H, I, dt, g)
        s["sw1"], s["ss1"] = _weight((), 2 * sh, H, dt, g) if sh else (None, None)
        s["sw2"], s["ss2"] = _weight((), H, sh, dt, g) if sh else (None, None)
        return s
    M, K, N, L, R, dt = c["M"], c["K"], c["N"], c["L"], c["R"], DTYPE[c["dtype"]]
    s["a"] = torch.randn(L, R, K, generator=g, device=DEV).mul_(K ** -0.5).to(dt)
    s["b"] = torch.randn(L, N, R, generator=g, device=DEV).mul_(0.5 * R ** -0.5).to(dt)
    s["ids"] = _adapters(c, g)
    s["scaling"] = torch.rand(L, generator=g, device=DEV) * 2
    if c["kind"] == "entry":
        s["x"] = _rows(M, K, g, c["dtype"])
        s["residual"] = _rows(M, K, g, c["dtype"])
        s["weight"] = (1.0 + 0.2 * torch.randn(K, generator=g, device=DEV)).to(dt)
        w, ws = _weight((), N, K, "int8", g)
        s["w"], s["ws"] = w, ws.contiguous()
        return s
    s["x"], s["xs"] = _int8_rows(M, K, g) if c["rows"] == "int8" else (_rows(M, K, g, c["rows"]), None)
    s["base"] = torch.randn(M, N, generator=g, device=DEV).to(DTYPE[c["base"]])
    return s


# ---------------------------------------------------------------- the plain forms
def _plain_route(c, l, bias):
    """In 64 bits: which of two experts comes first can hang on the last bits of their scores."""
    T, E, K, G = c["T"], c["E"], c["K"], c["G"]
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
    ids = order.sort(dim=1, descending=True, stable=True).indices[:, :K]
    w = s.gather(1, ids)
    w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return ids, w * _scaling(c)


def _scaling(c):
    return 2.5 if c["score"] == "sigmoid" else 1.0


def _values(w, s):
    """[..., n, k] codes as the values that they stand for, in 32 bits."""
    v = w.float()
    if s is None:
        return v
    if w.dtype == torch.int8:
        return v.mul_(s[..., None])
    n, k = v.shape[-2:]
    return v.view(*v.shape[:-2], n // 128, 128, k // 128, 128).mul_(s[..., :, None, :, None]).view(v.shape)


def _plain_expert(x, w1, s1, w2, s2):
    """x [B, 1, H] through weights [B, 2I, H] and [B, H, I]: [B, H]."""
    p = torch.bmm(x, _values(w1, s1).transpose(1, 2))
    gate, up = p.chunk(2, dim=2)
    h = gate / (1.0 + torch.exp(-gate)) * up
    return torch.bmm(h, _values(w2, s2).transpose(1, 2))


def _plain_layer(s):
    c, x = s["c"], s["x"]
    T, H, K = c["T"], c["H"], c["K"]
    logits = (x.double() @ s["router"].double().t()).float()  # (as the routing takes them)
    ids, w = _plain_route(c, logits.double(), s["bias"])
    pick = ids.flatten()
    some = lambda t: None if t is None else t[pick]  # noqa: E731
    # (bytes are picked as such: the codes of every pick's expert)
    codes = lambda t: t.view(torch.uint8)[pick].view(t.dtype) if t.element_size() == 1 else t[pick]  # noqa: E731
    rows = x.float().repeat_interleave(K, dim=0)[:, None, :]
    y = _plain_expert(rows, codes(s["w1"]), some(s["s1"]), codes(s["w2"]), some(s["s2"])).view(T, K, H)
    out = (y * w.float()[:, :, None]).sum(dim=1)
    if c["shared"]:
        one = lambda t: None if t is None else t[None]  # noqa: E731
        out = out + _plain_expert(x.float()[None], one(s["sw1"]), one(s["ss1"]), one(s["sw2"]), one(s["ss2"]))[0]
    return {"out": out.bfloat16(), "ids": ids.int(), "gates": w.float()}


def _plain_lora(base, x, xs, a, b, ids, scaling, dtype):
    """All adapters' products, of which each row keeps its own."""
    L, R, K = a.shape
    z = (x.float() @ a.float().view(L * R, K).t()).view(-1, L, R)
    z = z * ((ids[:, None] == torch.arange(L, device=ids.device)) * scaling)[:, :, None]
    if xs is not None:
        z = z * xs[:, None, None]
    return (base.float() + z.view(-1, L * R) @ b.float().transpose(1, 2).reshape(L * R, -1)).to(dtype)


def _plain_norm(x, residual, weight):
    """(int8 codes in 32 bits, scales, the new residual)."""
    v = x.float() + residual.float()
    r = torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS)
    t = v * weight.float()
    m = t.abs().amax(dim=1, keepdim=True)
    return torch.round(t * (torch.full_like(m, 127.0) / m)), (m / 127.0 * r)[:, 0], v.to(x.dtype)


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["c"]
    if own:
        from umdk_amd import add_rms_norm, lora_add, moe_decode_layer, quant_matmul
    if c["kind"] == "layer":
        if own:
            out, ids, gates = moe_decode_layer(
                s["x"], s["router"], s["bias"], s["w1"], s["s1"], s["w2"], s["s2"], c["K"], c["G"], c["KG"], c["score"],
                c["group"], True, _scaling(c), s["sw1"], s["ss1"], s["sw2"], s["ss2"])
            return {"out": out, "ids": ids, "gates": gates}
        return _plain_layer(s)
    dtype = DTYPE[c["dtype"]]
    if c["kind"] == "lora":
        if own:
            return lora_add(s["base"], s["x"], s["a"], s["b"], s["ids"], s["scaling"], s["xs"], dtype)
        return _plain_lora(s["base"], s["x"], s["xs"], s["a"], s["b"], s["ids"], s["scaling"], dtype)
    if own:
        q, qs, new = add_rms_norm(s["x"], s["residual"], s["weight"], EPS, 2)
        base = quant_matmul(q, qs, s["w"], s["ws"], None, torch.float32)
        return {"residual": new, "out": lora_add(base, q, s["a"], s["b"], s["ids"], s["scaling"], qs, dtype)}
    q, qs, new = _plain_norm(s["x"], s["residual"], s["weight"])
    base = (q @ s["w"].float().t()) * s["ws"] * qs[:, None]
    return {"residual": new, "out": _plain_lora(base, q, qs, s["a"], s["b"], s["ids"], s["scaling"], dtype)}


# ---------------------------------------------------------------- what a pass cannot do without
def _adapters_in_use(c):
    """Rows that have an adapter, and how many different adapters they have, on average."""
    draws = c["M"] if c["spread"] == "token" else max(1, min(12, c["M"] // 40))
    return c["M"] * (1.0 - c["none"]), c["L"] * (1.0 - (1.0 - (1.0 - c["none"]) / c["L"]) ** draws)


def work(c):
    if c["kind"] == "layer":
        T, H, E, K, I, sh = c["T"], c["H"], c["E"], c["K"], c["I"], c["shared"]
        size = 2 if c["dtype"] == "bf16" else 1
        used = E * (1.0 - (1.0 - K / E) ** T)  # experts with a token, on average
        return {"bytes": int(used * 3 * H * I * size + 3 * H * sh * size + E * H * (4 if c["router"] == "fp32" else 2)
                             + 4 * T * H + 8 * T * K),
                "flops": 6 * T * H * (K * I + sh) + 2 * T * E * H}
    M, K, N, R = c["M"], c["K"], c["N"], c["R"]
    rows, used = _adapters_in_use(c)
    both = {"bytes": int(2 * used * R * (K + N)) + 4 * M, "flops": int(2 * rows * R * (K + N))}
    if c["kind"] == "lora":
        one = {"bf16": 2, "fp16": 2, "int8": 1, "fp32": 4}
        both["bytes"] += M * (K * one[c["rows"]] + N * (one[c["base"]] + 2))
        return both
    return {"bytes": both["bytes"] + 6 * M * K + N * K + 2 * M * N, "flops": both["flops"] + 2 * M * N * K + 5 * M * K}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def _exact_route(c, l, bias):
    T, E, K, G = c["T"], c["E"], c["K"], c["G"]
    score = torch.sigmoid(l) if c["score"] == "sigmoid" else torch.softmax(l, dim=1)
    rank = score.clone() if bias is None else score + bias.to(torch.float64)
    if G > 1:
        expert = torch.arange(E, device=l.device)
        group = torch.stack([part.topk(2 if c["group"] == "top2" else 1, dim=1).values.sum(dim=1)
                             for part in rank.split(E // G, dim=1)], dim=1)
        allowed = torch.zeros(T, E, dtype=torch.bool, device=l.device)
        for _ in range(c["KG"]):
            best = group.max(dim=1).indices
            allowed |= (expert // (E // G))[None, :] == best[:, None]
            group.scatter_(1, best[:, None], -math.inf)
        rank.masked_fill_(~allowed, -math.inf)
    ids = torch.empty(T, K, dtype=torch.int64, device=l.device)
    for k in range(K):
        ids[:, k] = rank.max(dim=1).indices
        rank.scatter_(1, ids[:, k:k + 1], -math.inf)
    gate = torch.gather(score, 1, ids)
    return ids, gate / gate.sum(dim=1, keepdim=True) * _scaling(c)


def _exact_matrix(w, s):
    v = w.to(torch.float64)
    if s is None:
        return v
    if s.shape == w.shape[:1]:
        return v * s.to(torch.float64)[:, None]
    return v * s.to(torch.float64).repeat_interleave(128, dim=0).repeat_interleave(128, dim=1)


def _exact_expert(x, w1, s1, w2, s2):
    p = torch.matmul(x, _exact_matrix(w1, s1).t().contiguous())
    half = p.shape[1] // 2
    return torch.matmul(torch.nn.functional.silu(p[:, :half]) * p[:, half:], _exact_matrix(w2, s2).t().contiguous())


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "layer":
        x = s["x"].to(torch.float64)
        ids, gate = _exact_route(c, torch.matmul(x, s["router"].to(torch.float64).t().contiguous()), s["bias"])
        out = torch.zeros_like(x)
        at = lambda t, e: None if t is None else t[e]  # noqa: E731
        for e in sorted(set(ids.flatten().tolist())):
            t, k = torch.nonzero(ids == e, as_tuple=True)
            y = _exact_expert(x[t], s["w1"][e], at(s["s1"], e), s["w2"][e], at(s["s2"], e))
            out.index_add_(0, t, y * gate[t, k][:, None])
        if c["shared"]:
            out += _exact_expert(x, s["sw1"], s["ss1"], s["sw2"], s["ss2"])
        return {"out": out, "ids": ids.to(torch.int32), "gates": gate}
    if c["kind"] == "entry":
        v = s["x"].to(torch.float64) + s["residual"].to(torch.float64)
        y = v / torch.sqrt((v * v).sum(dim=1, keepdim=True) / v.shape[1] + EPS) * s["weight"].to(torch.float64)
        step = y.abs().amax(dim=1, keepdim=True) / 127.0
        x = torch.round(y / step) * step
        out = torch.matmul(x, (s["w"].to(torch.float64) * s["ws"].to(torch.float64)[:, None]).t().contiguous())
    else:
        x = s["x"].to(torch.float64)
        if s["xs"] is not None:
            x = x * s["xs"].to(torch.float64)[:, None]
        out = s["base"].to(torch.float64)
    for e in sorted(set(s["ids"].tolist()) - {-1}):
        t = torch.nonzero(s["ids"] == e)[:, 0]
        z = torch.matmul(x[t], s["a"][e].to(torch.float64).t().contiguous()) * s["scaling"][e].to(torch.float64)
        out.index_add_(0, t, torch.matmul(z, s["b"][e].to(torch.float64).t().contiguous()))
    return {"residual": v, "out": out} if c["kind"] == "entry" else out
