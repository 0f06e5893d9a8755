"""A decode step of a few requests, some with adapters, as a layer runs it: norm with int8 rows -> int8 projection -> adapters
on the same rows -> norm -> whole expert layer.  Each operator is held to its definition in 64 bits on what it was given."""
import pytest
import torch

import tests.test_gpu_lora as A
import tests.test_gpu_moe_decode as E
import umdk_amd
from tests.test_gpu_norm import rows, weights
from umdk_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OPS = torch.ops.umdk_cam_op_lib
GATING = dict(E.GROUPED)


def make(T, H=640, K=4, adapters=5, rank=16, dtype="fp8", seed=0):
    d = E.make(T, H, 16, 384, 256, dtype, seed=seed)
    a = A.make(T, H, H, adapters, rank, "bf16", "int8", "fp32", seed=seed)
    wd = torch.randint(-127, 128, (H, H), generator=torch.Generator().manual_seed(seed + 1), dtype=torch.int8).to(DEV)
    return dict(h=rows(T, H, seed + 2, torch.bfloat16), res=rows(T, H, seed + 3, torch.bfloat16), g1=weights(H, torch.bfloat16),
                g2=weights(H, torch.bfloat16), wd=wd, sd=torch.rand(H, generator=torch.Generator().manual_seed(seed)).to(DEV) * 1e-3,
                lora=a, moe=d, K=K, mask=torch.ones(T, dtype=torch.bool, device=DEV))


def layer(d):
    q, qs, res = OPS.add_rms_norm(d["h"], d["res"], d["g1"], 1e-6, 2)
    base = OPS.quant_matmul(q, qs, d["wd"], d["sd"], None, torch.float32)
    a, m = d["lora"], d["moe"]
    y = OPS.lora_add(base, q, a["a"], a["b"], a["ids"], a["scaling"], qs)
    x, _, res2 = OPS.add_rms_norm(y, res, d["g2"], 1e-6, 0)
    out, ids, gates = OPS.moe_decode_layer(x, m["router"], m["bias"], m["w1"], m["s1"], m["w2"], m["s2"], d["K"],
                                           share_gmm1_weight=m["sw1"], share_gmm1_weight_scale=m["ss1"],
                                           share_gmm2_weight=m["sw2"], share_gmm2_weight_scale=m["ss2"],
                                           x_active_mask=d["mask"], **GATING)
    return dict(q=q, qs=qs, base=base, y=y, x=x, res=res2, out=out, ids=ids, gates=gates)


@pytest.mark.parametrize("dtype", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("T", [1, 5, 16])
def test_layer(T, dtype):
    d = make(T, dtype=dtype, seed=T)
    if T > 1:
        d["mask"][T // 2] = False
    r = layer(d)
    # base: the sum is exact, the two products are rounded to 24 bits; the norm: fp32 throughout, then 2^-8 of it
    want = (r["q"].double() @ d["wd"].double().t().contiguous()) * d["sd"].double() * r["qs"].double()[:, None]
    assert ((r["base"].double() - want).abs() <= want.abs() * 4 * A.E32).all()
    A.check(dict(d["lora"], base=r["base"], x=r["q"], xs=r["qs"]), r["y"])
    v = r["y"].double() + umdk_amd.add_rms_norm(d["h"], d["res"], d["g1"], 1e-6, 2)[2].double()
    x = v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-6) * d["g2"].double()
    assert ((r["x"].double() - x).abs() <= x.abs() * (2.0 ** -8 + 2.0 ** -16)).all()
    E.check(dict(d["moe"], x=r["x"]), d["K"], (r["out"], r["ids"], r["gates"]), mask=d["mask"], **GATING)
    assert not r["out"][~d["mask"]].any()


def test_steps_captured_and_replayed():
    T = 12
    d = make(T, seed=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # two layers in a row, the second on what the first gave
        held = layer(d)
        again = layer(dict(d, h=held["out"], res=held["res"]))
    for seed in range(5):
        new = make(T, seed=20 + seed)
        for n in ("h", "res"):
            d[n].copy_(new[n])
        d["lora"]["ids"].copy_(new["lora"]["ids"])
        d["mask"].copy_(torch.rand(T, generator=torch.Generator().manual_seed(seed)) < 0.8)
        graph.replay()
        eager = layer(d)
        second = layer(dict(d, h=eager["out"], res=eager["res"]))
        torch.cuda.synchronize()
        for n in eager:
            assert torch.equal(held[n], eager[n]) and torch.equal(again[n], second[n]), (seed, n)


class Absent:
    """No call takes the native way from tensors to the launch."""
    def __getattr__(self, name):
        return lambda *args: None


def test_both_ways_to_the_launch_give_the_same(monkeypatch):
    d = make(6, seed=5)
    want = layer(d)
    lora = A.make(70, 256, 96, 4, 16, "fp16", "fp16", "fp32", seed=6)
    wants = [A.call(lora), A.call(lora, torch.bfloat16), A.call(lora, scaling=None)]
    wide = dict(lora, ids=lora["ids"].long(), a=lora["a"], base=lora["base"].t().contiguous().t())
    got = [A.call(wide), A.call(wide, torch.bfloat16), A.call(wide, scaling=None)]
    for p, q in zip(got, wants):
        assert torch.equal(p, q)
    monkeypatch.setattr(_lib, "_tensor_caller", Absent())
    for n, t in layer(d).items():
        assert torch.equal(t, want[n]), n
    for p, q in zip([A.call(lora), A.call(lora, torch.bfloat16), A.call(lora, scaling=None)], wants):
        assert torch.equal(p, q)


def test_ids_past_32_bits_are_no_adapters():
    d = A.make(40, 64, 48, 3, 8, none=0.0)
    ids = d["ids"].long()
    ids[::2] += 2 ** 32
    got = A.call(d, ids=ids)
    assert torch.equal(got[::2], d["base"][::2])
    ids[::2] = -1
    assert torch.equal(got, A.call(d, ids=ids.int()))


@pytest.mark.parametrize("M,L,R", [(256, 300, 8), (700, 700, 256), (600, 2, 200), (9000, 2000, 16), (8300, 4, 160)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_many_adapters_and_wide_ranks(M, L, R, dtype):
    """More chunks in a window than blocks that share it, a window of one adapter a row, ranks of several groups."""
    d = A.make(M, 144, 72, L, R, dtype, none=0.05, seed=M)
    if L >= 300:  # nearly a chunk for every row
        d["ids"] = torch.randperm(max(M, L), generator=torch.Generator().manual_seed(1))[:M].remainder(L).int().to(DEV)
    A.check(d, A.call(d))


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwAD
    a = A.make(4, 64, 32, 2, 8)
    m = E.make(2, 256, 4, 128, 0, "bf16")
    with fwAD.dual_level():
        for name in ("base", "x", "a", "b", "scaling"):
            with pytest.raises(RuntimeError, match="no backward|forward"):
                A.call(a, **{name: fwAD.make_dual(a[name], torch.ones_like(a[name]))})
        for name in ("x", "router", "bias", "w1", "w2"):
            with pytest.raises(RuntimeError, match="no backward|forward"):
                E.call(dict(m, **{name: fwAD.make_dual(m[name], torch.ones_like(m[name]))}), 2)


def test_negated_views_are_refused():
    """Their sign is held beside their numbers, which is all that a kernel reads."""
    a = A.make(4, 64, 32, 2, 8, dtype="fp16", base="fp32")
    with pytest.raises(RuntimeError, match="negated view"):
        A.call(a, base=torch._neg_view(a["base"]))
    m = E.make(2, 256, 4, 128, 0, "bf16")
    with pytest.raises(RuntimeError, match="negated view"):
        E.call(m, 2, x=torch._neg_view(m["x"]))
