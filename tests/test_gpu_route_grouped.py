"""moe_route_grouped against its definition in 64 bits: ids equal, gates within a rounding of fp32 and one of the scaling
factor's (2 x 2^-24)."""
import math

import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def reference(logits, bias, K, G=1, KG=1, score="softmax", group="top2", renorm=True, scaling=1.0):
    l = logits.detach().cpu().double()
    T, E = l.shape
    there = ~torch.isnan(l) & (l > -math.inf)
    l = torch.where(there, l, torch.full_like(l, -math.inf))
    if score == "sigmoid":
        s = torch.sigmoid(l)
    else:
        mx = l.amax(dim=1, keepdim=True)
        e = torch.where(there, torch.exp(l - torch.where(mx > -math.inf, mx, torch.zeros_like(mx))), torch.zeros_like(l))
        s = e / e.sum(dim=1, keepdim=True).clamp(min=1e-300)
    b = torch.zeros(E, dtype=torch.float64) if bias is None else bias.cpu().double()
    # without a bias the order is the logits' own, which no rounding of s can hide
    c = (l if bias is None and (G == KG or group == "max") else s + b).clone()
    c[~there | torch.isnan(c) | (c == -math.inf)] = -math.inf
    if KG < G:
        by = c.view(T, G, E // G).sort(dim=2, descending=True).values
        gs = by[:, :, 0].clone()
        if group == "top2" and E // G > 1:
            gs += torch.where(by[:, :, 1] > -math.inf, by[:, :, 1], torch.zeros_like(gs))
        order = gs.sort(dim=1, descending=True, stable=True)
        kept = torch.zeros(T, G, dtype=torch.bool)
        kept.scatter_(1, order.indices[:, :KG], order.values[:, :KG] > -math.inf)
        c = torch.where(kept.repeat_interleave(E // G, dim=1), c, torch.full_like(c, -math.inf))
    top = c.sort(dim=1, descending=True, stable=True)
    ids = torch.where(top.values[:, :K] > -math.inf, top.indices[:, :K], torch.full((T, K), -1))
    w = torch.where(ids >= 0, s.gather(1, ids.clamp(min=0)), torch.zeros(T, K, dtype=torch.float64))
    if renorm:
        w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return ids.int(), w * scaling


def check(logits, bias, K, **kw):
    own = dict(n_group=kw.get("G", 1), topk_group=kw.get("KG", 1), score_func=kw.get("score", "softmax"),
               group_score=kw.get("group", "top2"), renormalize=kw.get("renorm", True),
               routed_scaling=kw.get("scaling", 1.0))
    ids, w = umdk_amd.moe_route_grouped(logits, bias, K, **own)
    rids, rw = reference(logits, bias, K, **kw)
    assert torch.equal(ids.cpu(), rids), (ids.cpu() != rids).any(dim=1).nonzero()[:5]
    err = (w.cpu().double() - rw).abs()
    assert (err <= 2 * U * rw.abs() + 2.0 ** -150).all(), float((err / rw.abs().clamp(min=1e-300)).max())
    return ids, w


def data(T, E, seed, dtype=torch.float32, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * spread).to(dtype).to(DEV), (0.1 * torch.randn(E, generator=g)).to(DEV)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K,G,KG,group", [
    (1, 256, 8, 8, 4, "top2"), (3, 160, 6, 8, 3, "max"), (129, 64, 6, 1, 1, "top2"), (64, 72, 5, 6, 2, "top2"),
    (37, 512, 16, 64, 2, "top2"), (5, 8, 2, 1, 1, "max"), (9, 60, 4, 3, 3, "top2"), (70, 384, 8, 1, 1, "max"),
    (33, 1, 1, 1, 1, "top2"), (17, 7, 7, 7, 7, "max"), (4097, 256, 8, 8, 4, "top2"), (5000, 160, 6, 8, 3, "max"),
    (4100, 512, 16, 1, 1, "top2"), (4099, 60, 6, 5, 2, "top2"), (6001, 33, 9, 11, 4, "top2"), (4111, 8, 8, 1, 1, "max"),
    (4500, 480, 8, 5, 2, "top2"), (4097, 320, 8, 1, 1, "max"), (4097, 384, 6, 4, 2, "max"),
    # 8 lanes a token, with as many experts a lane as its kernels take, and 16 or 64 beside them
    (6, 64, 8, 8, 4, "top2"), (8195, 160, 6, 8, 3, "max"), (8193, 100, 5, 5, 2, "top2"), (24577, 256, 8, 8, 4, "top2"),
    (24580, 192, 7, 1, 1, "max"), (24579, 250, 6, 2, 1, "top2"), (24581, 256, 4, 4, 2, "top2"), (24578, 256, 9, 8, 3, "max"),
])
def test_against_the_definition(T, E, K, G, KG, group, score):
    for i, (dtype, with_bias, renorm) in enumerate([(torch.float32, True, True), (torch.bfloat16, False, False),
                                                    (torch.float16, True, False), (torch.float32, False, True)]):
        logits, bias = data(T, E, 7 * T + i, dtype)
        check(logits, bias if with_bias else None, K, G=G, KG=KG, score=score, group=group, renorm=renorm,
              scaling=[1.0, 16.0, 2.5, 0.3][i])


@pytest.mark.parametrize("T,E,K,G,KG", [
    (3, 96, 6, 1, 1), (2049, 96, 6, 1, 1), (8193, 96, 7, 1, 1), (130, 150, 6, 5, 2), (2050, 150, 6, 5, 2), (2300, 512, 8, 16, 4),
    (2600, 384, 8, 6, 2), (4097, 512, 12, 16, 4), (8200, 192, 8, 1, 1), (2048, 144, 4, 1, 1), (2049, 144, 4, 1, 1),
    (7, 36, 5, 3, 2), (9, 300, 8, 3, 2), (5, 468, 9, 13, 5), (11, 20, 5, 1, 1), (8192, 20, 5, 1, 1), (6, 44, 3, 11, 4),
])
@pytest.mark.parametrize("off", [0, 1, 4])
def test_lanes_that_are_not_full_and_slices(T, E, K, G, KG, off):
    for i, dtype in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        wide, bias = data(T, E + 16, 3 * T + i, dtype)
        part, b = wide[:, off:off + E], bias[off:off + E]
        check(part, b, K, G=G, KG=KG, score="sigmoid")
        check(part, None, K, G=G, KG=KG, score="softmax", group="max", renorm=False)


@pytest.mark.parametrize("T,E,G,KG", [
    (5, 256, 1, 1), (5, 256, 8, 4), (1025, 256, 8, 4), (7, 512, 16, 4), (3001, 512, 1, 1), (3, 510, 34, 3), (9, 64, 4, 2),
    (9, 128, 1, 1), (1030, 160, 8, 3), (1026, 384, 1, 1), (1, 384, 6, 2), (8200, 40, 5, 4), (300, 17, 1, 1), (4, 450, 5, 3),
])
def test_many_picks_and_few_experts_left(T, E, G, KG):
    for K in (9, 12, 16):
        logits, bias = data(T, E, T + K)
        logits[0, 5:] = -math.inf                      # fewer experts than picks
        logits[-1, ::3] = math.nan
        logits[T // 2, :] = -1.0                       # ties throughout
        bias[E // 2] = -math.inf
        check(logits, bias, K, G=G, KG=KG, score="sigmoid")
        check(logits, bias - 3.0, K, G=G, KG=KG, score="softmax", group="max", renorm=False)
        check(logits, None, K, G=G, KG=KG, score="softmax", group="max")
        # the best ones all in one lane: every pick from one list
        logits[0] = torch.arange(E, device=DEV) * -1e-3
        check(logits, None, K, G=G, KG=KG, score="sigmoid")


@pytest.mark.parametrize("K", [5, 8])
@pytest.mark.parametrize("T,E,G,KG", [(3, 512, 1, 1), (3, 512, 16, 4), (1000, 384, 1, 1), (1025, 384, 1, 1), (3, 450, 5, 3),
                                      (3, 510, 34, 3), (3002, 512, 16, 4), (2, 352, 1, 1)])
def test_five_to_eight_picks_of_many_experts(T, E, G, KG, K):
    logits, bias = data(T, E, T + K)
    logits[0, 3:] = -math.inf
    check(logits, bias, K, G=G, KG=KG, score="sigmoid")
    check(logits, None, K, G=G, KG=KG, score="softmax", group="max", renorm=False)


@pytest.mark.parametrize("T", [6, 4200])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_fall_to_the_lower_id(score, T):
    # three values only, so that nearly every choice of an expert and of a group is a tie
    g = torch.Generator().manual_seed(3)
    logits = torch.randint(-1, 2, (T, 96), generator=g).float().to(DEV)
    check(logits, None, 8, G=8, KG=3, score=score, group="max")
    check(logits, None, 8, G=8, KG=3, score=score, group="top2")
    check(logits, torch.zeros(96, device=DEV), 12, G=4, KG=2, score=score)
    check(torch.zeros(T, 96, device=DEV), None, 16, G=6, KG=2, score=score)
    check(torch.where(logits > 0, logits, logits * 0.0 * -1.0), None, 8, score=score)  # zeros of both signs are equal


@pytest.mark.parametrize("T", [5, 4100])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_experts_and_empty_rows(score, T):
    logits, bias = data(T, 64, 11)
    logits[0] = -math.inf                      # a row that its mask leaves empty
    logits[1, :62] = -math.inf                 # two experts left for eight slots
    logits[2, 5] = math.nan
    logits[3, ::2] = -math.inf
    logits[4, :] = torch.finfo(torch.float32).min   # a mask of the lowest value: ties, not holes
    bias[7] = -math.inf                        # an expert that is switched off
    bias[9] = math.nan
    for kw in (dict(), dict(G=8, KG=2), dict(G=8, KG=2, group="max"), dict(G=8, KG=8, renorm=False)):
        ids, w = check(logits, bias, 8, score=score, **kw)
        assert (ids[0] == -1).all() and (w[0] == 0).all()
        assert not ((ids == 7) | (ids == 9)).any()
        check(logits, None, 8, score=score, **kw)


def test_extreme_logits_and_biases():
    logits, bias = data(64, 32, 5)
    logits[0] = 3e38
    logits[1] = -3e38
    logits[2, 3] = 200.0
    logits[3] = -200.0
    logits[4, 1:] = -100.0
    check(logits, bias, 4, G=4, KG=2, score="sigmoid")
    check(logits, bias, 4, G=4, KG=2, score="softmax")
    check(logits, bias - 50.0, 4, G=4, KG=2, score="sigmoid")   # every choice score below zero
    big = bias.clone()
    big[3], big[5] = math.inf, math.inf
    ids, _ = umdk_amd.moe_route_grouped(logits, big, 3, score_func="sigmoid")
    assert (ids[:, 0] == 3).all() and (ids[:, 1] == 5).all()


def test_a_pick_leaves_the_mirrored_expert_below_zero():
    # 34 groups of 15 experts, 16 places each: those of (group 32, expert 1) and (group 31, expert 14) add up to 1023, the
    # places being turned over in keys below zero
    logits = torch.full((3, 510), -5.0, device=DEV)
    logits[:, 32 * 15 + 1] = 1.0
    logits[:, 31 * 15 + 14] = -1.0
    check(logits, None, 2, G=34, KG=34, renorm=False)
    # 40 groups of 12: groups 30 and 33, whose ids add up to 63
    logits = torch.full((3, 480), -5.0, device=DEV)
    logits[:, 30 * 12] = 1.0
    logits[:, 33 * 12] = -1.0
    check(logits, None, 2, G=40, KG=2, group="max", renorm=False)


def test_logits_of_infinity_count_as_the_largest_number():
    logits, bias = data(40, 64, 6)
    logits[0, 9] = math.inf
    logits[1, [50, 3]] = math.inf
    logits[2, :] = math.inf
    largest = torch.where(logits == math.inf, torch.full_like(logits, torch.finfo(torch.float32).max), logits)
    for b in (None, bias):
        for kw in (dict(), dict(group="max"), dict(renorm=False)):
            own = dict(n_group=8, topk_group=3, score_func="softmax", group_score=kw.get("group", "top2"),
                       renormalize=kw.get("renorm", True))
            ids, w = umdk_amd.moe_route_grouped(logits, b, 4, **own)
            rids, rw = reference(largest, b, 4, G=8, KG=3, **kw)
            assert torch.equal(ids.cpu(), rids)
            assert ((w.cpu().double() - rw).abs() <= 2 * U * rw.abs() + 2.0 ** -150).all()


def test_rows_with_a_stride_and_no_rows():
    logits, bias = data(50, 200, 8)
    part = logits[:, 20:148]
    check(part, bias[20:148], 8, G=8, KG=4, score="sigmoid")
    check(logits.t().contiguous().t()[:, :64], None, 4)
    check(logits[::3], None, 4)
    check(logits[:1].expand(7, 200), None, 4)
    ids, w = umdk_amd.moe_route_grouped(logits[:0], None, 4)
    assert ids.shape == (0, 4) and w.shape == (0, 4)


def test_offsets_past_32_bits():
    wide = torch.empty(40000, 30000, dtype=torch.float32, device=DEV)   # 4.8 GB
    part = wide[:, 29000:29064]
    fresh, bias = data(40000, 64, 9)
    part.copy_(fresh)
    ids, w = umdk_amd.moe_route_grouped(part, bias, 6, score_func="sigmoid")
    rids, rw = umdk_amd.moe_route_grouped(fresh, bias, 6, score_func="sigmoid")
    assert torch.equal(ids, rids) and torch.equal(w, rw)


def test_same_as_moe_route_where_they_agree():
    logits, _ = data(300, 128, 2)
    ids, w = umdk_amd.moe_route_grouped(logits, None, 6)
    rids, rw = umdk_amd.moe_route(logits, None, 6)
    assert torch.equal(ids, rids)
    assert ((w - rw).abs() <= 8 * U * rw.abs()).all()   # (moe_route: an fp32 exponential, sum and division)


def test_captured_on_a_side_stream_and_replayed():
    logits, bias = data(128, 256, 4)
    args = (bias, 8, 8, 4, "sigmoid", "top2", True, 2.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        umdk_amd.moe_route_grouped(logits, *args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, w = torch.ops.umdk_cam_op_lib.moe_route_grouped(logits, *args)
    for seed in range(3):
        fresh, _ = data(128, 256, 40 + seed)
        logits.copy_(fresh)
        graph.replay()
        eids, ew = umdk_amd.moe_route_grouped(logits, *args)
        torch.cuda.synchronize()
        assert torch.equal(ids, eids) and torch.equal(w, ew)
