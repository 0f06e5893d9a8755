"""The operators around the expert layer together with it, as a decoder layer uses them: norm -> router product -> grouped
routing -> experts, and norm -> int8 product beside them."""
import pytest
import torch

import umdk_amd
from tests.test_gpu_norm import rows, weights
from tests.test_gpu_route_grouped import reference as route_reference
from umdk_amd.plan import MoeLayerPlan, MoePrefillPlan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OPS = torch.ops.umdk_cam_op_lib
GATING = dict(n_group=4, topk_group=2, score_func="sigmoid", group_score="top2", renormalize=True, routed_scaling=2.5)


def int8_weight(*shape, seed=0):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * 0.02
    s = w.abs().amax(dim=-1) / 127.0
    return torch.round(w / s[..., None]).to(torch.int8).to(DEV), s.to(DEV)


def make(T, H=1024, E=32, I=256, N=640, seed=0):
    g = torch.Generator().manual_seed(seed)
    w1, s1 = int8_weight(E, 2 * I, H, seed=1)
    w2, s2 = int8_weight(E, H, I, seed=2)
    wd, sd = int8_weight(N, H, seed=3)
    return dict(x=rows(T, H, seed + 5, torch.bfloat16), res=rows(T, H, seed + 6, torch.bfloat16),
                g=weights(H, torch.bfloat16), router=(torch.randn(E, H, generator=g) * 0.05).to(DEV),
                bias=(0.05 * torch.randn(E, generator=g)).to(DEV), w1=w1, s1=s1, w2=w2, s2=s2, wd=wd, sd=sd, E=E, K=4)


def layer(d):
    y, _, new = OPS.add_rms_norm(d["x"], d["res"], d["g"], 1e-6, 0)
    q, qs, _ = OPS.add_rms_norm(d["x"], d["res"], d["g"], 1e-6, 2)
    dense = OPS.quant_matmul(q, qs, d["wd"], d["sd"])
    logits = y.float() @ d["router"].t()
    idx, w = OPS.moe_route_grouped(logits, d["bias"], d["K"], **GATING)
    out, _, counts = OPS.fused_deep_moe(y, idx, [d["w1"].transpose(1, 2)], [d["s1"]], [d["w2"].transpose(1, 2)], [d["s2"]], w,
                                        None, None, None, None, None, None, None, "ep", 1, 0, d["E"], 0, y.shape[0])
    return dict(y=y, new=new, dense=dense, logits=logits, idx=idx, w=w, out=out, counts=counts)


@pytest.mark.parametrize("T", [1, 48, 200])
def test_layer(T):
    d = make(T)
    r = layer(d)
    ids, w = route_reference(r["logits"], d["bias"], d["K"], G=4, KG=2, score="sigmoid", scaling=2.5)
    assert torch.equal(r["idx"].cpu(), ids)
    assert torch.equal(r["counts"].cpu(), torch.bincount(ids.flatten().long(), minlength=d["E"]))
    # the dense branch against real numbers: a code is off by at most half a step of its row (norm = steps of 1/127 of the
    # row's largest), a weight by its own, which w * s already holds; the product's rounding to bf16 is 2^-8 of it
    v = d["x"].cpu().double() + d["res"].cpu().double()
    y = v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-6) * d["g"].cpu().double()
    wd = d["wd"].cpu().double() * d["sd"].cpu().double()[:, None]
    want = y @ wd.t()
    half = y.abs().amax(1, keepdim=True) / 254 * wd.abs().sum(1)[None, :]
    assert ((r["dense"].cpu().double() - want).abs() <= half * (1 + 2.0 ** -7) + want.abs() * 2.0 ** -8 + 1e-6).all()
    # the experts' branch against the fused op's definition in 64 bits: int8 rows, h requantised in int8.  Each expert's
    # output and their sum are rounded to bf16 (2^-8 of it at most); h in fp32 is within some 2^-20 of its 64-bit value, so
    # less than a thousandth of its codes, those within 127 2^-20 of a tie, are off by one step, a 127th of the row's
    # largest: sqrt(1e-3) / 127 of that, which is at most sqrt(256) = 16 times the row's rms, 4e-3 of h
    quant = lambda m: (torch.round(m * (127.0 / m.abs().max())), m.abs().max() / 127.0)  # noqa: E731
    out = torch.zeros(T, d["x"].shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    w1, s1, w2, s2 = (d[n].cpu().double() for n in ("w1", "s1", "w2", "s2"))
    I = w2.shape[2]
    for t in range(T):
        q, step = quant(r["y"][t].cpu().double())
        for k in range(d["K"]):
            e = int(ids[t, k])
            p = (w1[e] @ q) * s1[e] * step
            hq, hstep = quant(torch.nn.functional.silu(p[:I]) * p[I:])
            o = float(w[t, k]) * (w2[e] @ hq) * s2[e] * hstep
            out[t] += o
            size[t] += o.abs()
    err = (r["out"].cpu().double() - out).norm()
    assert err <= 2.0 ** -8 * (size.norm() + out.norm()) + 4e-3 * size.norm(), float(err / out.norm())


def test_layer_captured_and_replayed():
    d = make(64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer(d)
    for seed in range(4):
        d["x"].copy_(rows(64, 1024, 70 + seed, torch.bfloat16))
        graph.replay()
        eager = layer(d)
        torch.cuda.synchronize()
        for k in held:
            assert torch.equal(held[k], eager[k]), (k, seed)


def test_fp8_rows_feed_the_grouped_products():
    T, H, I = 130, 1024, 256
    x, res, g = rows(T, H, 1, torch.bfloat16), rows(T, H, 2, torch.bfloat16), weights(H, torch.bfloat16)
    q, s, _ = umdk_amd.add_rms_norm(x, res, g, 1e-6, 3)
    gen = torch.Generator().manual_seed(3)
    w = (torch.randn(2, 2 * I, H, generator=gen) * 3).to(torch.float8_e4m3fn)
    ws = torch.rand(2, 2 * I // 128, H // 128, generator=gen) * 0.01
    groups = torch.tensor([50, 80], device=DEV)
    h, _ = umdk_amd.grouped_matmul_swiglu(q, s, groups, w.to(DEV), ws.to(DEV), 0)
    a = (q.cpu().double().view(T, -1, 128) * s.cpu().double()[:, :, None]).view(T, H)
    wf = w.double().view(2, 2 * I // 128, 128, H // 128, 128) * ws.double()[:, :, None, :, None]
    wf = wf.view(2, 2 * I, H)
    p = torch.cat([a[:50] @ wf[0].t(), a[50:] @ wf[1].t()])
    want = torch.nn.functional.silu(p[:, :I]) * p[:, I:]
    assert (h.cpu().double() - want).norm() / want.norm() < 5e-3   # bf16 h and fp32 sums


@pytest.mark.parametrize("T", [7, 300])
def test_plan_routes_by_groups(T):
    H, E, K = 1024, 32, 4
    plan = MoePrefillPlan(T, H, E, K, quant_mode=0)
    g = torch.Generator().manual_seed(T)
    logits, bias = torch.randn(T, E, generator=g).to(DEV), (0.1 * torch.randn(E, generator=g)).to(DEV)
    logits[0, 2:] = float("-inf")   # two experts for four slots: the others are not routed
    x = rows(T, H, 1, torch.bfloat16)
    plan.route_grouped(logits, bias, **GATING)
    plan.layout()
    plan.dispatch(x)
    out = plan.combine(plan.expand_x)   # identity experts
    ids, w = route_reference(logits, bias, K, G=4, KG=2, score="sigmoid", scaling=2.5)
    assert torch.equal(plan.topk_idx.cpu(), ids) and torch.equal(plan.topk_idx64.cpu(), ids.long())
    n = int((ids >= 0).sum())
    assert int(plan.recv_count[-1]) == n == T * K - 2
    wf = plan.topk_w.cpu()
    want = torch.zeros(T, H)
    for k in range(K):   # multiply, then add, in pick order: the combine's own arithmetic
        want = want + torch.where(ids[:, k:k + 1] >= 0, x.cpu().float() * wf[:, k:k + 1], torch.zeros(1))
    assert torch.equal(out.cpu(), want.bfloat16())


def test_the_long_way_gives_the_same():
    """Calls that the native caller of tensors leaves to Python: numbers of other types, other strides."""
    d = make(9)
    logits = torch.randn(9, 64, device=DEV)
    a = umdk_amd.moe_route_grouped(logits, None, 4, 8, 2, "sigmoid", "max", True, 2.0)
    for b in (umdk_amd.moe_route_grouped(logits, None, 4, 8, 2, "sigmoid", "max", True, 2),
              umdk_amd.moe_route_grouped(logits, None, 4, 8, 2, "sigmoid", "max", 1, 2.0),
              umdk_amd.moe_route_grouped(logits.t().contiguous().t(), None, 4, 8, 2, "sigmoid", "max", True, 2.0),
              OPS.moe_route_grouped(logits, None, 4, 8, 2, "sigmoid", "max", True, 2.0)):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for quant in (0, 2, 3):
        a = umdk_amd.add_rms_norm(d["x"], d["res"], d["g"], 1.0, quant)
        for b in (umdk_amd.add_rms_norm(d["x"], d["res"], d["g"], 1, quant),
                  umdk_amd.add_rms_norm(d["x"].t().contiguous().t(), d["res"].t().contiguous().t(), d["g"], 1.0, quant),
                  umdk_amd.add_rms_norm(d["x"], d["res"], d["g"].repeat_interleave(2)[::2], 1.0, quant)):
            for p, q in zip(a, b):
                assert p.dtype == q.dtype and p.shape == q.shape and p.stride() == q.stride()
                assert torch.equal(p.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))


def test_parameters_without_a_gradient_to_record():
    d = make(5)
    g = torch.nn.Parameter(d["g"])
    q, s, new = umdk_amd.add_rms_norm(d["x"], d["res"], d["g"], 1e-6, 2)
    for guard in (torch.no_grad, torch.inference_mode):
        with guard():
            for a, b in zip(umdk_amd.add_rms_norm(d["x"], d["res"], g, 1e-6, 2), (q, s, new)):
                assert torch.equal(a, b) and type(a) is torch.Tensor and not a.requires_grad
    with pytest.raises(RuntimeError, match="no backward"):
        umdk_amd.add_rms_norm(d["x"], d["res"], g, 1e-6, 2)
    logits = torch.randn(5, 32, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        umdk_amd.moe_route_grouped(logits, None, 4)
    assert umdk_amd.moe_route_grouped(logits.detach(), None, 4)[0].shape == (5, 4)


def test_negated_views_and_batched_tensors_are_refused():
    z = torch.randn(4, 32, dtype=torch.complex64, device=DEV)
    view = torch.conj(z).imag
    assert view.is_neg()
    with pytest.raises(RuntimeError, match="negated"):
        umdk_amd.moe_route_grouped(view, None, 4)
    ids, _ = umdk_amd.moe_route_grouped(view.resolve_neg(), None, 4)
    assert torch.equal(ids, (-z.imag).topk(4, dim=1).indices.int())
    with pytest.raises(RuntimeError):
        torch.vmap(lambda l: umdk_amd.moe_route_grouped(l, None, 4))(torch.randn(3, 4, 32, device=DEV))


def test_plan_refuses_other_logits():
    plan = MoePrefillPlan(8, 1024, 32, 4, quant_mode=0)
    good, bias = torch.zeros(8, 32, device=DEV), torch.zeros(32, device=DEV)
    for logits, b, kw in [(good[:7], bias, {}), (good[:, :16], bias[:16], {}), (good.t().contiguous().t(), bias, {}),
                          (good.cpu(), bias, {}), (good, bias.cpu(), {}), (good, bias.double(), {}), (good, bias[:31], {}),
                          (good.double(), bias, {}), (good, bias, dict(score_func="relu")), (good, bias, dict(n_group=5))]:
        with pytest.raises(RuntimeError):
            plan.route_grouped(logits, b, **kw)
    plan.route_grouped(torch.zeros(8, 48, device=DEV)[:, :32], bias, n_group=4, topk_group=2)   # rows of a wider tensor


def test_layer_plan_takes_the_gating():
    T, H, E, K, I = 130, 1024, 32, 4, 256
    d = make(T, H, E, I)
    plan = MoeLayerPlan(T, H, E, K, E, I, dtype="int8")
    logits = torch.randn(T, E, device=DEV)
    out = plan.forward_op_chain(d["x"], logits, d["bias"], d["w1"], d["s1"], d["w2"], d["s2"], gating=GATING).clone()
    idx, w = umdk_amd.moe_route_grouped(logits, d["bias"], K, **GATING)
    assert torch.equal(plan.topk_idx, idx) and torch.equal(plan.topk_w, w)
    nte, sti = umdk_amd.get_dispatch_layout(idx, E, 1)
    ex, sc, src, rc, n = umdk_amd.moe_dispatch_prefill(d["x"], idx, w, nte, sti, "ep", 0, 1, True)
    h, hs = umdk_amd.grouped_matmul_swiglu(ex, sc, n, d["w1"], d["s1"], 2)
    y = umdk_amd.grouped_matmul(h, hs, n, d["w2"], d["s2"])
    assert torch.equal(out, umdk_amd.moe_combine_prefill(y, idx, w, src, rc, "ep", 0, 1))


def test_forward_mode_gradients_are_refused():
    """The tensors are on the GPU, where the native caller takes the call."""
    fwd = torch.autograd.forward_ad
    d = make(5)
    logits = torch.randn(5, 32, device=DEV)
    q, s, _ = umdk_amd.add_rms_norm(d["x"], d["res"], d["g"], 1e-6, 2)
    plan = MoePrefillPlan(5, 1024, 32, 4, quant_mode=0)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: umdk_amd.moe_route_grouped(dual(logits), None, 4),
                     lambda: umdk_amd.moe_route_grouped(logits, dual(d["bias"]), 4),
                     lambda: plan.route_grouped(dual(logits), None),
                     lambda: umdk_amd.add_rms_norm(dual(d["x"]), d["res"], d["g"]),
                     lambda: umdk_amd.add_rms_norm(d["x"], dual(d["res"]), d["g"]),
                     lambda: umdk_amd.add_rms_norm(d["x"], d["res"], dual(d["g"])),
                     lambda: umdk_amd.quant_matmul(q, dual(s), d["wd"], d["sd"]),
                     lambda: umdk_amd.quant_matmul(q, s, d["wd"], dual(d["sd"]))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        x = dual(logits)
        with torch.inference_mode():   # none is asked for there
            ids, _ = umdk_amd.moe_route_grouped(x, None, 4)
        assert torch.equal(ids, umdk_amd.moe_route_grouped(logits, None, 4)[0])
