"""What the operators of a decode step of a few requests refuse, and their shape functions: host logic, no kernel runs."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import umdk_amd
from tests.test_around_api import P, first_phase

bf, f16, f32, i8, fp8 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
z = lambda *shape, dtype=f32: torch.zeros(*shape, dtype=dtype)  # noqa: E731


def layer(x=P, router=P, bias=None, w1=P, s1=None, w2=P, s2=None, sw1=None, ss1=None, sw2=None, ss2=None, mask=None, T=4, H=256,
          E=16, n1=256, ns=0, K=4, wtype=0, rtype=4, G=4, KG=2, score=0, group=2, renorm=1, scaling=1.0, out=P, idx=P, w=P):
    return first_phase("camhipMoeDecodeLayer", x, router, bias, w1, s1, w2, s2, sw1, ss1, sw2, ss2, mask, T, H, E, n1, ns, K,
                       wtype, rtype, G, KG, score, group, renorm, scaling, out, idx, w)


@pytest.mark.parametrize("kw,frag", [
    (dict(T=-1), "numTokens"), (dict(T=17), "numTokens"), (dict(H=0), "hidden"), (dict(H=96), "hidden"),
    (dict(H=8256), "hidden"), (dict(wtype=3, s1=P, s2=P, H=192), "hidden"), (dict(n1=0), "gmm1HiddenSize"),
    (dict(n1=192), "gmm1HiddenSize"), (dict(n1=65664), "gmm1HiddenSize"), (dict(wtype=3, s1=P, s2=P, n1=128), "gmm1HiddenSize"),
    (dict(ns=-128), "shareGmm1HiddenSize"), (dict(ns=100, sw1=P, sw2=P), "shareGmm1HiddenSize"), (dict(E=0), "numExperts"),
    (dict(E=513, G=1, KG=1), "numExperts"), (dict(K=0), "topK"), (dict(K=17), "topK"), (dict(E=2, G=1, KG=1, K=3), "topK"),
    (dict(KG=1, K=5), "exceeds"), (dict(G=3), "numGroups"), (dict(G=0), "numGroups"), (dict(KG=5), "topkGroups"),
    (dict(wtype=1), "weightDtype"), (dict(wtype=4), "weightDtype"), (dict(rtype=1), "routerDtype"), (dict(score=2), "scoreFunc"),
    (dict(group=0), "groupScore"), (dict(renorm=2), "renormalize"), (dict(x=P + 8), "aligned"), (dict(w1=P + 8), "aligned"),
    (dict(w2=P + 4), "aligned"), (dict(router=P + 4), "aligned"), (dict(out=P + 2), "aligned"), (dict(idx=P + 2), "aligned"),
    (dict(w=P + 1), "aligned"), (dict(bias=P + 2), "aligned"),
])
def test_layer_rejects(kw, frag):
    st, _, msg = layer(**kw)
    assert st == 161001 and frag in msg, msg


@pytest.mark.parametrize("kw", [dict(x=None), dict(router=None), dict(w1=None), dict(w2=None), dict(out=None), dict(idx=None),
                                dict(w=None), dict(wtype=2, s1=P), dict(wtype=2, s2=P), dict(ns=128, sw1=P), dict(ns=128, sw2=P),
                                dict(wtype=2, s1=P, s2=P, ns=128, sw1=P, sw2=P, ss1=P)])
def test_layer_null_pointers(kw):
    assert layer(**kw)[0] == 161002
    assert layer(**kw, T=0)[0] == 0


def lora(base=P, x=P, xs=None, a=P, b=P, ids=P, scaling=None, m=4, n=64, k=64, r=16, L=2, bstep=64, xstep=64, bt=0, xt=0, lt=0, ot=0,
         out=P):
    return first_phase("camhipLoraAdd", base, x, xs, a, b, ids, scaling, m, n, k, r, L, bstep, xstep, bt, xt, lt, ot, out)


@pytest.mark.parametrize("kw,frag", [
    (dict(m=-1), "m "), (dict(m=(1 << 20) + 1), "m "), (dict(n=0), "n "), (dict(n=(1 << 20) + 1, bstep=1 << 21), "n "),
    (dict(k=0), "k "), (dict(k=24), "k "), (dict(k=131072, xstep=131072), "k "), (dict(r=0), "rank"), (dict(r=12), "rank"),
    (dict(r=264), "rank"), (dict(L=0), "numAdapters"), (dict(L=65537), "numAdapters"), (dict(bt=2), "baseDtype"),
    (dict(lt=4), "loraDtype"), (dict(xt=1), "xDtype"), (dict(xt=4), "xDtype"), (dict(ot=4), "outDtype"),
    (dict(bstep=63), "baseRowStride"), (dict(xstep=63), "xRowStride"), (dict(bstep=1 << 40), "baseRowStride"),
    (dict(a=P + 8), "aligned"), (dict(b=P + 2), "aligned"), (dict(x=P + 8), "aligned"), (dict(xstep=68), "aligned"), (dict(bt=4, base=P + 2), "aligned"),
    (dict(ids=P + 2), "aligned"), (dict(out=P + 1), "aligned"), (dict(scaling=P + 1), "aligned"),
])
def test_lora_rejects(kw, frag):
    st, _, msg = lora(**kw)
    assert st == 161001 and frag in msg, msg


@pytest.mark.parametrize("kw", [dict(base=None), dict(x=None), dict(a=None), dict(b=None), dict(ids=None), dict(out=None),
                                dict(xt=2, xs=None)])
def test_lora_null_pointers(kw):
    assert lora(**kw)[0] == 161002
    assert lora(**kw, m=0)[0] == 0


def test_a_short_workspace_is_refused():
    import ctypes
    from umdk_amd import _lib
    L = _lib.lib()
    for name, args in (("camhipLoraAdd", [P, P, None, P, P, P, None, 4, 64, 64, 16, 2, 64, 64, 0, 0, 0, 0, P]),
                       ("camhipMoeDecodeLayer", [P, P, None, P, None, P] + [None] * 6 + [4, 256, 16, 256, 0, 4, 0, 4, 4, 2, 0, 2, 1,
                                                                                         1.0, P, P, P])):
        ws, ex = ctypes.c_uint64(0), ctypes.c_void_p(0)
        assert getattr(L, name + "GetWorkspaceSize")(*args, ctypes.byref(ws), ctypes.byref(ex)) == 0 and ws.value > 0
        assert getattr(L, name)(P, ws.value - 1, ex, None) == 161003


def decode(x=None, router=None, bias=None, w1=None, s1=None, w2=None, s2=None, K=2, **kw):
    x = z(2, 128, dtype=bf) if x is None else x
    router = z(4, 128) if router is None else router
    w1 = z(4, 256, 128, dtype=bf) if w1 is None else w1
    w2 = z(4, 128, 128, dtype=bf) if w2 is None else w2
    return umdk_amd.moe_decode_layer(x, router, bias, w1, s1, w2, s2, K, **kw)


@pytest.mark.parametrize("kw,frag", [
    (dict(x=z(2, 128)), "bfloat16"), (dict(x=z(17, 128, dtype=bf)), "at most 16"), (dict(x=z(128, dtype=bf)), "x must"),
    (dict(x=z(2, 256, dtype=bf)[:, ::2]), "contiguous"), (dict(router=z(4, 64)), "router"), (dict(router=z(4, 128, dtype=f16)), "router"),
    (dict(bias=z(5)), "bias"), (dict(bias=z(4, dtype=bf)), "bias"), (dict(w1=z(4, 256, 128)), "weights must"),
    (dict(w1=z(3, 256, 128, dtype=bf)), "gmm1_weight"), (dict(w1=z(4, 128, 256, dtype=bf).transpose(1, 2)), "contiguous"),
    (dict(w2=z(4, 128, 64, dtype=bf)), "gmm2_weight"), (dict(w2=z(4, 128, 128, dtype=i8)), "gmm2_weight"),
    (dict(s1=z(4, 256)), "no scales"), (dict(w1=z(4, 256, 128, dtype=i8), w2=z(4, 128, 128, dtype=i8)), "scale missing"),
    (dict(w1=z(4, 256, 128, dtype=i8), w2=z(4, 128, 128, dtype=i8), s1=z(4, 128), s2=z(4, 128)), "gmm1_weight_scale"),
    (dict(w1=z(4, 256, 128, dtype=fp8), w2=z(4, 128, 128, dtype=fp8), s1=z(4, 2, 1), s2=z(4, 128)), "gmm2_weight_scale"),
    (dict(share_gmm1_weight=z(128, 128, dtype=bf)), "together"), (dict(share_gmm1_weight_scale=z(128)), "without share weights"),
    (dict(share_gmm1_weight=z(128, 128, dtype=bf), share_gmm2_weight=z(128, 128, dtype=bf)), "share_gmm2_weight"),
    (dict(x_active_mask=z(2)), "x_active_mask"), (dict(x_active_mask=z(3, dtype=torch.bool)), "x_active_mask"),
    (dict(score_func="relu"), "score_func"), (dict(group_score="mean"), "group_score"), (dict(), "GPU only"),
])
def test_layer_python_checks(kw, frag):
    with pytest.raises(RuntimeError, match=frag):
        decode(**kw)


def add(base=None, x=None, a=None, b=None, ids=None, scaling=None, xs=None, out=None):
    return umdk_amd.lora_add(z(4, 32, dtype=bf) if base is None else base, z(4, 64, dtype=bf) if x is None else x,
                             z(2, 8, 64, dtype=bf) if a is None else a, z(2, 32, 8, dtype=bf) if b is None else b,
                             z(4, dtype=torch.int32) if ids is None else ids, scaling, xs, out)


@pytest.mark.parametrize("kw,frag", [
    (dict(base=z(3, 32, dtype=bf)), "base must"), (dict(base=z(4, 32, dtype=torch.float64)), "base must"), (dict(x=z(64, dtype=bf)), "x "),
    (dict(x=z(4, 64)), "x must"), (dict(x=z(4, 64, dtype=i8)), "x_scale"), (dict(x=z(4, 64, dtype=i8), xs=z(3)), "x_scale"),
    (dict(xs=z(4)), "without int8"), (dict(a=z(2, 8, 64)), "lora_a"), (dict(a=z(2, 8, 32, dtype=bf)), "lora_a"),
    (dict(a=z(2, 64, 8, dtype=bf).transpose(1, 2)), "lora_a"), (dict(b=z(2, 8, 32, dtype=bf)), "lora_b"),
    (dict(b=z(2, 32, 8, dtype=f16)), "lora_b"), (dict(ids=z(4)), "adapter_ids"), (dict(ids=z(3, dtype=torch.int32)), "adapter_ids"),
    (dict(scaling=z(3)), "scaling"), (dict(scaling=z(2, dtype=bf)), "scaling"), (dict(out=f32), "out_dtype"), (dict(), "GPU only"),
])
def test_lora_python_checks(kw, frag):
    with pytest.raises(RuntimeError, match=frag):
        add(**kw)


def test_gradients_are_refused_not_dropped():
    with pytest.raises(RuntimeError, match="no backward"):
        decode(x=z(2, 128, dtype=bf).requires_grad_())
    with pytest.raises(RuntimeError, match="no backward"):
        add(a=z(2, 8, 64, dtype=bf).requires_grad_())
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        with pytest.raises(RuntimeError, match="forward-mode"):
            decode(router=dual(z(4, 128)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            add(base=dual(z(4, 32, dtype=bf)))
    with pytest.raises(RuntimeError, match="negated"):
        add(base=torch._neg_view(z(4, 32, dtype=bf)))


def test_shape_functions():
    ops = torch.ops.umdk_cam_op_lib
    m = lambda *shape, dtype=f32: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    out, idx, w = ops.moe_decode_layer(m(3, 256, dtype=bf), m(8, 256), m(8), m(8, 256, 256, dtype=fp8), m(8, 2, 2),
                                       m(8, 256, 128, dtype=fp8), m(8, 2, 1), 4)
    assert out.shape == (3, 256) and out.dtype == bf and idx.shape == (3, 4) and idx.dtype == torch.int32 and w.dtype == f32
    args = lambda base, t: (m(5, 32, dtype=base), m(5, 64, dtype=t), m(2, 8, 64, dtype=t), m(2, 32, 8, dtype=t),  # noqa: E731
                            m(5, dtype=torch.int32))
    assert ops.lora_add(*args(bf, bf)).dtype == bf and ops.lora_add(*args(f32, f16)).dtype == f16
    assert ops.lora_add(*args(f32, bf), out_dtype=f16).dtype == f16 and ops.lora_add(*args(f16, bf)).shape == (5, 32)
