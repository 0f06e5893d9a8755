"""moe_decode_layer against its definition in 64 bits.

Tolerances.  With E = 2^-24 and d(n) = n / 8 + 40 additions on the longest path of a sum of n products (eight waves at least
share a sum; their sums, lanes and scales add fewer than 40), fp32 sums are within d(n) E sum |products|.  That bounds g and
u; |silu'| <= 1.1; h is held to 2^-16 and the exponential to 2^-20; the second product's sum likewise; the output's rounding
is 2^-8 of it.  Element by element that is a loose bound, so the norm of the error is held too: roundings to bf16 that
are uniform within half a step have a root mean square of at most 2^-8 / sqrt(3) of the value, and nothing else reaches a
hundredth of that; a tenth is left for the few outputs."""
import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E32 = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def weight(lead, n, k, dtype, g):
    """(codes, scales, values in 64 bits)"""
    w = torch.randn(*lead, n, k, generator=g) * k ** -0.5
    if dtype == "bf16":
        w = w.bfloat16()
        return w, None, w.double()
    if dtype == "int8":
        s = w.abs().amax(-1) / 127
        q = torch.round(w / s[..., None]).to(torch.int8)
        return q, s, q.double() * s.double()[..., None]
    b = w.view(*lead, n // 128, 128, k // 128, 128)
    s = (b.abs().amax((-3, -1)) / 448) * torch.exp(torch.randn(b.abs().amax((-3, -1)).shape, generator=g) * 0.3)
    q = (b / s[..., :, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(w.shape), s.contiguous(), (q.double() * s.double()[..., :, None, :, None]).view(w.shape)


def make(T, H, E, I, Is, dtype, router="fp32", seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    d = dict(x=torch.randn(T, H, generator=g).bfloat16(), bias=0.1 * torch.randn(E, generator=g) if bias else None,
             router=(torch.randn(E, H, generator=g) * 1.2 * H ** -0.5).to(torch.float32 if router == "fp32" else torch.bfloat16))
    d["w1"], d["s1"], d["W1"] = weight((E,), 2 * I, H, dtype, g)
    d["w2"], d["s2"], d["W2"] = weight((E,), H, I, dtype, g)
    for n in ("sw1", "ss1", "SW1", "sw2", "ss2", "SW2"):
        d[n] = None
    if Is:
        d["sw1"], d["ss1"], d["SW1"] = weight((), 2 * Is, H, dtype, g)
        d["sw2"], d["ss2"], d["SW2"] = weight((), H, Is, dtype, g)
    for n in ("x", "bias", "router", "w1", "s1", "w2", "s2", "sw1", "ss1", "sw2", "ss2"):
        d[n] = None if d[n] is None else d[n].to(DEV)
    return d


def call(d, K, x=None, mask=None, **kw):
    return umdk_amd.moe_decode_layer(d["x"] if x is None else x, d["router"], d["bias"], d["w1"], d["s1"], d["w2"], d["s2"], K,
                                     share_gmm1_weight=d["sw1"], share_gmm1_weight_scale=d["ss1"],
                                     share_gmm2_weight=d["sw2"], share_gmm2_weight_scale=d["ss2"], x_active_mask=mask, **kw)


def steps(n):
    return (n / 8 + 40) * E32


def expert(x, w1, w2):
    """(E(x), a bound of its error) in 64 bits, of x [H]."""
    H, I = x.shape[0], w2.shape[1]
    p, size = w1 @ x, w1.abs() @ x.abs()
    g, u = p[:I], p[I:]
    dg, du = steps(H) * size[:I], steps(H) * size[I:]
    s = torch.sigmoid(g) * g
    h = s * u
    dh = 1.1 * dg * (u.abs() + du) + s.abs() * du + h.abs() * (2.0 ** -16 + 2.0 ** -20)
    return w2 @ h, w2.abs() @ dh + steps(I) * (w2.abs() @ (h.abs() + dh))


def check(d, K, got, mask=None, **kw):
    out, ids, gates = got
    T, H = d["x"].shape
    x = d["x"].cpu().double()
    logits = (x @ d["router"].cpu().double().t()).float()
    if mask is not None:
        logits[~mask.cpu()] = float("nan")
    wids, wgates = umdk_amd.moe_route_grouped(logits.to(DEV), d["bias"], K, **kw)
    assert torch.equal(ids, wids) and torch.equal(gates, wgates)
    want, bound = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        if mask is not None and not mask[t]:
            continue
        picks = [(d["W1"][e], d["W2"][e], w) for e, w in zip(ids[t].tolist(), gates[t].double().tolist()) if e >= 0]
        if d["SW1"] is not None:
            picks.append((d["SW1"], d["SW2"], 1.0))
        for w1, w2, w in picks:
            y, b = expert(x[t], w1, w2)
            want[t] += w * y
            bound[t] += abs(w) * (b + 20 * E32 * y.abs())
    got = out.cpu().double()
    assert got.isfinite().all()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + bound * (1 + 2.0 ** -8) + 1e-30).all()
    if want.norm() > 0:
        assert (got - want).norm() <= 1.1 * 2.0 ** -8 / 3 ** 0.5 * want.norm()


GROUPED = dict(n_group=4, topk_group=2, score_func="sigmoid", group_score="top2", renormalize=True, routed_scaling=2.5)


@pytest.mark.parametrize("dtype", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("T,H,E,I,Is,K,kw", [
    (1, 1024, 8, 512, 0, 2, {}),                      # a small model's next token
    (1, 128, 1, 128, 0, 1, {}),                       # the least of everything
    (16, 128, 4, 128, 128, 4, {}),                    # every expert has every token
    (3, 640, 16, 384, 256, 4, GROUPED),
    (7, 1920, 12, 1408, 2816, 3, {}),                 # widths that are no power of two, a shared expert wider than the others
    (16, 2048, 64, 256, 0, 8, GROUPED),
    (5, 7168, 8, 256, 128, 4, GROUPED),
    (2, 8192, 4, 128, 0, 2, {}),                      # the widest rows
    (4, 512, 4, 14336, 0, 2, {}),                     # the widest experts that are usual
    (13, 256, 512, 128, 0, 16, dict(n_group=8, topk_group=4)),   # many experts, all picks
    (9, 384, 60, 128, 640, 6, dict(n_group=5, topk_group=3, group_score="max")),
])
def test_against_the_definition(dtype, T, H, E, I, Is, K, kw):
    d = make(T, H, E, I, Is, dtype, router="fp32" if T % 2 else "bf16", seed=T)
    check(d, K, call(d, K, **kw), **kw)


@pytest.mark.parametrize("dtype,H,I", [("bf16", 64, 64), ("int8", 64, 64), ("int8", 192, 320), ("bf16", 448, 192), ("int8", 4160, 704)])
def test_widths_of_64(dtype, H, I):
    d = make(6, H, 8, I, 64, dtype, seed=3)
    check(d, 3, call(d, 3))


def test_wide_shared_expert_of_narrow_experts():
    d = make(2, 256, 4, 64, 9024, "int8", seed=5)
    check(d, 2, call(d, 2))


@pytest.mark.parametrize("T", range(1, 17))
def test_every_batch_and_each_token_alone(T):
    """A token's results do not hang on the tokens beside it."""
    d = make(T, 1152, 24, 256, 128, "fp8", seed=40 + T)
    got = call(d, 4, **GROUPED)
    check(d, 4, got, **GROUPED)
    for t in {0, T // 2, T - 1}:
        alone = call(d, 4, x=d["x"][t:t + 1].contiguous(), **GROUPED)
        for a, b in zip(alone, got):
            assert torch.equal(a[0], b[t])


def test_no_tokens():
    d = make(1, 256, 4, 128, 0, "bf16")
    out, ids, gates = call(d, 2, x=d["x"][:0])
    assert out.shape == (0, 256) and ids.shape == (0, 2) and gates.shape == (0, 2)


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("mask", [[1, 1, 0, 0, 0], [0, 1, 0, 1, 0], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1]])
def test_tokens_that_are_not_active(dtype, mask):
    d = make(5, 512, 16, 256, 128, dtype, seed=9)
    m = torch.tensor(mask, dtype=torch.bool, device=DEV)
    d["x"][~m] = float("nan")   # padding holds anything
    got = call(d, 4, mask=m)
    assert (got[0][~m] == 0).all() and (got[1][~m] == -1).all() and (got[2][~m] == 0).all()
    whole = call(d, 4, x=torch.where(m[:, None], d["x"], 1.0))
    for a, b in zip(got, whole):
        assert torch.equal(a[m], b[m])


def test_experts_that_nobody_may_pick():
    d = make(6, 512, 8, 128, 0, "int8", seed=11)
    d["bias"][:] = float("-inf")
    d["bias"][5] = 0.0
    got = call(d, 4)
    assert (got[1][:, 0] == 5).all() and (got[1][:, 1:] == -1).all() and (got[2][:, 1:] == 0).all()
    check(d, 4, got)
    d["bias"][5] = float("-inf")   # none at all
    out, ids, gates = call(d, 4)
    assert (ids == -1).all() and (gates == 0).all() and (out == 0).all()


def test_weights_that_no_token_uses_are_not_read_into_the_sums():
    d = make(4, 512, 16, 256, 0, "bf16", seed=12)
    ids = call(d, 2)[1]
    unused = [e for e in range(16) if not (ids == e).any()]
    want = call(d, 2)[0]
    d["w1"][unused] = float("nan")
    d["w2"][unused] = float("inf")
    assert unused and torch.equal(call(d, 2)[0], want)


def test_infinities_and_nan_stay_in_their_token():
    d = make(4, 512, 16, 256, 128, "fp8", seed=13)
    want = call(d, 4)
    x = d["x"].clone()
    x[1, 7] = float("nan")
    x[2, 3] = float("inf")
    out, ids, gates = call(d, 4, x=x)
    assert (ids[1] == -1).all() and out[1].isnan().all()        # no logit, no expert; the shared expert's row is NaN
    assert torch.equal(out[0], want[0][0]) and torch.equal(out[3], want[0][3])
    assert torch.equal(ids[0], want[1][0]) and torch.equal(gates[3], want[2][3])
    assert not out[2].isfinite().all()


def test_large_values_do_not_pass_the_range_on_the_way():
    """h far past what fp16 holds, gates of a large scaling."""
    d = make(2, 512, 4, 256, 0, "bf16", seed=14)
    d["x"] *= 1024
    check(d, 2, call(d, 2, routed_scaling=16.0), routed_scaling=16.0)


def test_captured_and_replayed():
    d = make(5, 1024, 32, 256, 128, "fp8", seed=15)
    mask = torch.ones(5, dtype=torch.bool, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(d, 4, mask=mask)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = call(d, 4, mask=mask)
        second = call(d, 4, x=first[0], mask=mask)   # two layers in one graph
    for seed in range(5):
        d["x"].copy_(torch.randn(5, 1024, generator=torch.Generator().manual_seed(seed)).bfloat16())
        mask[4] = bool(seed % 2)
        graph.replay()
        a = call(d, 4, mask=mask)
        b = call(d, 4, x=a[0], mask=mask)
        torch.cuda.synchronize()
        for p, q in zip(first + second, a + b):
            assert torch.equal(p, q), seed


def test_calls_on_several_streams_at_once():
    d = make(8, 2048, 32, 512, 256, "int8", seed=16)
    want = [call(d, 4, x=d["x"].roll(i, 0)) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    xs = [d["x"].roll(i, 0).contiguous() for i in range(4)]
    torch.cuda.synchronize()
    got = [[] for _ in streams]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(d, 4, x=xs[i]))
    torch.cuda.synchronize()
    for i in range(4):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_guard_bands():
    """Nothing is written outside the outputs: a workspace of exactly the size asked for, in the middle of a buffer."""
    from umdk_amd import _lib
    d = make(3, 512, 16, 256, 128, "fp8", seed=17)
    want = call(d, 4)
    args = [d[n].data_ptr() for n in ("x", "router", "bias", "w1", "s1", "w2", "s2", "sw1", "ss1", "sw2", "ss2")] + [None]
    args += [3, 512, 16, 512, 256, 4, 3, 4, 1, 1, 0, 2, 1, 1.0]
    need = _lib.workspace_size("camhipMoeDecodeLayer", *args, 0x1000, 0x1000, 0x1000)
    ws = torch.full((need + 512,), 0xA5, dtype=torch.uint8, device=DEV)
    bufs = [torch.full((n + 512,), 0x5A, dtype=torch.uint8, device=DEV) for n in (3 * 512 * 2, 48, 48)]
    _lib.launch("camhipMoeDecodeLayer", *args, *[b.data_ptr() + 256 for b in bufs], workspace=ws[256:256 + need])
    torch.cuda.synchronize()
    assert (ws[:256] == 0xA5).all() and (ws[-256:] == 0xA5).all()
    for b, w in zip(bufs, want):
        assert (b[:256] == 0x5A).all() and (b[-256:] == 0x5A).all()
        assert torch.equal(b[256:-256], w.view(torch.uint8).flatten())


def test_weights_past_4_gib():
    """Expert offsets past 32 bits: 80 experts of 100 MB each."""
    g = torch.Generator(device=DEV).manual_seed(1)
    E, H, I = 80, 4096, 4096
    w1 = torch.randint(-100, 100, (E, 2 * I, H), generator=g, device=DEV, dtype=torch.int8)
    w2 = torch.randint(-100, 100, (E, H, I), generator=g, device=DEV, dtype=torch.int8)
    s1, s2 = (torch.rand(E, n, generator=g, device=DEV) * 1e-3 for n in (2 * I, H))
    x = torch.randn(2, H, generator=g, device=DEV).bfloat16()
    router = torch.zeros(E, H, device=DEV)
    bias = torch.zeros(E, device=DEV)
    bias[[0, 41, 79]] = torch.tensor([1.0, 2.0, 3.0], device=DEV)
    out, ids, gates = umdk_amd.moe_decode_layer(x, router, bias, w1, s1, w2, s2, 3)
    assert ids.tolist() == [[79, 41, 0]] * 2
    want = torch.zeros(2, H, dtype=torch.float64, device=DEV)
    for k, e in enumerate((79, 41, 0)):
        p = (x.double() @ w1[e].double().t().contiguous()) * s1[e].double()
        h = torch.nn.functional.silu(p[:, :I]) * p[:, I:]
        want += gates[:, k:k + 1].double() * (h @ w2[e].double().t().contiguous()) * s2[e].double()
    assert (out.double() - want).norm() <= 1.1 * 2.0 ** -8 / 3 ** 0.5 * want.norm()


def test_the_operator_entry_and_defaults():
    d = make(3, 512, 8, 128, 0, "bf16", seed=18, bias=False)
    a = torch.ops.umdk_cam_op_lib.moe_decode_layer(d["x"], d["router"], None, d["w1"], None, d["w2"], None, 2)
    for p, q in zip(a, call(d, 2)):
        assert torch.equal(p, q)
    check(d, 2, a)


def test_gradients_are_refused_not_dropped():
    d = make(2, 256, 4, 128, 0, "bf16")
    for name in ("x", "router", "bias", "w1", "w2"):
        t = d[name]
        d[name] = t.detach().clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            call(d, 2)
        with torch.no_grad():
            call(d, 2)
        d[name] = t


@pytest.mark.parametrize("dtype,T,H,E,I,Is,K", [
    ("int8", 16, 768, 32, 192, 0, 5), ("int8", 2, 5824, 16, 320, 0, 4), ("int8", 3, 3904, 16, 256, 1344, 8),
    ("bf16", 5, 8192, 32, 64, 0, 6), ("bf16", 16, 8128, 16, 64, 64, 4), ("bf16", 1, 8192, 2, 64, 4160, 1),
    ("int8", 9, 8192, 24, 64, 8256, 3), ("bf16", 8, 4160, 12, 448, 64, 2), ("fp8", 12, 8064, 20, 128, 1920, 3),
    ("bf16", 4, 1088, 8, 8256, 0, 2), ("fp8", 7, 1152, 6, 8320, 128, 2),
])
def test_narrow_and_wide_experts_share_out_tiles(dtype, T, H, E, I, Is, K):
    """Items of 1 to 32 tiles, shared experts by other numbers, parts whose tiles do not come out even."""
    d = make(T, H, E, I, Is, dtype, seed=T + I)
    check(d, K, call(d, K))


@pytest.mark.parametrize("dtype,Is", [("bf16", 64), ("int8", 4160), ("fp8", 4224)])
@pytest.mark.parametrize("T", [1, 9])
def test_the_shared_expert_alone(dtype, Is, T):
    """No token has an expert: every score is NaN."""
    d = make(T, 1024, 4, 128, Is, dtype, seed=T)
    d["router"].fill_(float("nan"))
    out, ids, gates = call(d, 2)
    assert (ids == -1).all() and not gates.any()
    x = d["x"].cpu().double()
    for t in range(T):
        want, bound = expert(x[t], d["SW1"], d["SW2"])
        assert ((out[t].cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + bound * (1 + 2.0 ** -8) + 20 * E32 * want.abs()).all()
