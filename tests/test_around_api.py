"""What the operators around the expert layer refuse, and their shape functions: host logic, no kernel runs."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

import umdk_amd
from umdk_amd import _lib
from umdk_amd.plan import MoePrefillPlan

P = 0x1000  # a non-NULL stand-in pointer: never dereferenced by the first phase


def first_phase(name, *args):
    L = _lib.lib()
    ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(0)
    st = getattr(L, name + "GetWorkspaceSize")(*args, ctypes.byref(ws), ctypes.byref(ex))
    if st == 0:
        L.camhipReleaseExecutor(ex)
    return st, ws.value, L.camhipGetLastErrorMsg().decode()


def route(logits=P, bias=None, T=4, E=64, K=4, dtype=4, stride=64, G=8, KG=4, score=0, group=2, renorm=1, scaling=1.0,
          idx=P, w=P):
    return first_phase("camhipMoeRouteGrouped", logits, bias, T, E, K, dtype, stride, G, KG, score, group, renorm, scaling,
                       idx, w, None)


@pytest.mark.parametrize("kw,frag", [
    (dict(T=-1), "numTokens"), (dict(T=65537), "numTokens"), (dict(E=0), "numExperts"), (dict(E=520, stride=520), "numExperts"),
    (dict(K=0), "topK"), (dict(K=17), "topK"), (dict(E=8, G=1, KG=1, K=9), "topK"), (dict(dtype=3), "logitsDtype"),
    (dict(G=0), "numGroups"), (dict(G=5), "numGroups"), (dict(E=130, stride=130, G=65), "numGroups"),
    (dict(KG=0), "topkGroups"), (dict(KG=9), "topkGroups"), (dict(KG=1, K=9), "exceeds"), (dict(score=2), "scoreFunc"),
    (dict(group=0), "groupScore"), (dict(renorm=2), "renormalize"), (dict(stride=63), "logitsRowStride"),
    (dict(stride=1 << 50), "logitsRowStride"), (dict(logits=P + 2), "aligned"), (dict(bias=P + 1), "aligned"),
])
def test_route_grouped_rejects(kw, frag):
    st, _, msg = route(**kw)
    assert st == 161001 and frag in msg, msg


def test_misaligned_outputs_are_refused():
    args = (P, None, 4, 64, 4, 4, 64, 8, 4, 0, 2, 1, 1.0)
    for out in ((P + 2, P, None), (P, P + 1, None), (P, P, P + 4)):
        st, _, msg = first_phase("camhipMoeRouteGrouped", *args, *out)
        assert st == 161001 and "aligned" in msg, msg
    for kw in (dict(y=P + 1), dict(quant=2, scales=P + 2), dict(res=P, out=P + 1)):
        st, _, msg = norm(**kw)
        assert st == 161001 and "aligned" in msg, msg
    assert norm(quant=2, y=P + 1)[0] == 0   # bytes go anywhere


@pytest.mark.parametrize("kw", [dict(logits=None), dict(idx=None), dict(w=None)])
def test_route_grouped_null_pointers(kw):
    assert route(**kw)[0] == 161002
    assert route(**kw, T=0)[0] == 0


def norm(x=P, res=None, w=P, T=4, H=256, stride=256, dtype=0, wdtype=0, quant=0, eps=1e-6, y=P, scales=P, out=None):
    return first_phase("camhipAddRmsNorm", x, res, w, T, H, stride, dtype, wdtype, quant, eps, y, scales, out)


@pytest.mark.parametrize("kw,frag", [
    (dict(T=-1), "numTokens"), (dict(H=0), "hidden"), (dict(H=32769, stride=32769), "hidden"), (dict(dtype=4), "dtype"),
    (dict(wdtype=1), "weightDtype"), (dict(quant=3), "outQuant"), (dict(quant=5, H=250), "multiple of 128"),
    (dict(stride=255), "xRowStride"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=P + 1), "aligned"),
    (dict(wdtype=4, w=P + 2), "aligned"),
])
def test_norm_rejects(kw, frag):
    st, _, msg = norm(**kw)
    assert st == 161001 and frag in msg, msg


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(y=None), dict(quant=2, scales=None), dict(res=P, out=None)])
def test_norm_null_pointers(kw):
    assert norm(**kw)[0] == 161002


def qmm(x=P, xs=P, w=P, ws=P, bias=None, m=4, n=64, k=64, dtype=0, out=P):
    return first_phase("camhipQuantMatmul", x, xs, w, ws, bias, m, n, k, dtype, out)


@pytest.mark.parametrize("kw,frag", [
    (dict(m=-1), "m "), (dict(m=(1 << 20) + 1), "m "), (dict(n=0), "n "), (dict(n=(1 << 20) + 1), "n "), (dict(k=0), "k "),
    (dict(k=24), "k "), (dict(k=131072), "k "), (dict(dtype=2), "outDtype"), (dict(x=P + 8), "aligned"),
    (dict(w=P + 4), "aligned"), (dict(out=P + 1), "aligned"), (dict(dtype=4, out=P + 2), "aligned"),
])
def test_quant_matmul_rejects(kw, frag):
    st, _, msg = qmm(**kw)
    assert st == 161001 and frag in msg, msg


@pytest.mark.parametrize("kw", [dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(out=None)])
def test_quant_matmul_null_pointers(kw):
    assert qmm(**kw)[0] == 161002


bf, f32, i8 = torch.bfloat16, torch.float32, torch.int8
z = lambda *shape, dtype=f32: torch.zeros(*shape, dtype=dtype)  # noqa: E731


@pytest.mark.parametrize("call", [
    lambda: umdk_amd.moe_route_grouped(z(4, 8, dtype=torch.float64), None, 2),
    lambda: umdk_amd.moe_route_grouped(z(8), None, 2),
    lambda: umdk_amd.moe_route_grouped(z(4, 8), z(7), 2),
    lambda: umdk_amd.moe_route_grouped(z(4, 8), z(8, dtype=bf), 2),
    lambda: umdk_amd.moe_route_grouped(z(4, 8), None, 2, score_func="relu"),
    lambda: umdk_amd.moe_route_grouped(z(4, 8), None, 2, group_score="mean"),
    lambda: umdk_amd.moe_route_grouped(z(4, 0), None, 2),
    lambda: umdk_amd.add_rms_norm(z(4, 8), None, z(8)),
    lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), None, z(7, dtype=bf)),
    lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), None, z(8, dtype=torch.float16)),
    lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), z(4, 8), z(8)),
    lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), z(1, 8, dtype=bf), z(8)),
    lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), None, z(8), 1e-6, 1),
    lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), None, z(8), 1e-6, 3),
    lambda: umdk_amd.add_rms_norm(z(4, 0, dtype=bf), None, z(0)),
    lambda: umdk_amd.quant_matmul(z(4, 32), z(4), z(8, 32, dtype=i8), z(8)),
    lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), z(4), z(8, 48, dtype=i8), z(8)),
    lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), z(3), z(8, 32, dtype=i8), z(8)),
    lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), z(4), z(8, 32, dtype=i8), z(8, dtype=bf)),
    lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), z(4), z(32, 8, dtype=i8).t(), z(8)),
    lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), z(4), z(8, 32, dtype=i8), z(8), z(8, dtype=bf)),
    lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), z(4), z(8, 32, dtype=i8), z(8), None, i8),
    # well-formed, but not on a GPU
    lambda: umdk_amd.moe_route_grouped(z(4, 8), None, 2),
    lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), None, z(8)),
    lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), z(4), z(8, 32, dtype=i8), z(8)),
])
def test_python_checks(call):
    with pytest.raises(RuntimeError):
        call()


def test_gradients_are_refused_not_dropped():
    x = z(4, 8, dtype=bf).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        umdk_amd.add_rms_norm(x, None, z(8))
    with pytest.raises(RuntimeError, match="no backward"):
        umdk_amd.moe_route_grouped(z(4, 8).requires_grad_(), None, 2)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
        umdk_amd.add_rms_norm(x, None, z(8))


def test_shape_functions():
    ops = torch.ops.umdk_cam_op_lib
    m = lambda *shape, dtype=f32: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    idx, w = ops.moe_route_grouped(m(5, 64), m(64), 4, 8, 2, "sigmoid")
    assert idx.shape == (5, 4) and idx.dtype == torch.int32 and w.shape == (5, 4) and w.dtype == f32
    y, s, r = ops.add_rms_norm(m(5, 256, dtype=bf), m(5, 256, dtype=bf), m(256), 1e-6, 3)
    assert y.dtype == torch.float8_e4m3fn and s.shape == (5, 2) and s.stride() == (1, 5) and r.shape == (5, 256)
    y, s, r = ops.add_rms_norm(m(5, 256, dtype=bf), None, m(256, dtype=bf), 1e-6, 2)
    assert y.dtype == i8 and s.shape == (5,) and r.numel() == 0
    out = ops.quant_matmul(m(5, 32, dtype=i8), m(5), m(7, 32, dtype=i8), m(7), None, torch.float16)
    assert out.shape == (5, 7) and out.dtype == torch.float16
    assert ops.quant_matmul(m(5, 32, dtype=i8), m(5), m(7, 32, dtype=i8), m(7)).dtype == bf


def test_the_plan_refuses_gradients_and_negated_views():
    plan = MoePrefillPlan(4, 1024, 8, 2, quant_mode=0, device="cpu")   # (its host side: nothing is launched)
    good = z(4, 8)
    for logits, bias, why in [(good.requires_grad_(), z(8), "no backward"), (z(4, 8), z(8).requires_grad_(), "no backward"),
                              (torch._neg_view(z(4, 8)), z(8), "negated"), (z(4, 8), torch._neg_view(z(8)), "negated"),
                              (z(4, 8), z(8), "GPU only")]:
        with pytest.raises(RuntimeError, match=why):
            plan.route_grouped(logits, bias)


def test_forward_mode_gradients_are_refused_not_dropped():
    dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
    plan = MoePrefillPlan(4, 1024, 8, 2, quant_mode=0, device="cpu")
    with fwd.dual_level():
        for call in (lambda: umdk_amd.moe_route_grouped(dual(z(4, 8)), None, 2),
                     lambda: umdk_amd.moe_route_grouped(z(4, 8), dual(z(8)), 2),
                     lambda: plan.route_grouped(dual(z(4, 8)), None),
                     lambda: umdk_amd.add_rms_norm(dual(z(4, 8, dtype=bf)), None, z(8)),
                     lambda: umdk_amd.add_rms_norm(z(4, 8, dtype=bf), None, dual(z(8))),
                     lambda: umdk_amd.quant_matmul(z(4, 32, dtype=i8), dual(z(4)), z(8, 32, dtype=i8), z(8))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        x = dual(z(4, 8))
        with torch.inference_mode(), pytest.raises(RuntimeError, match="GPU only"):
            umdk_amd.moe_route_grouped(x, None, 2)   # nothing is asked for there
