"""moe_route_grouped where sums of different parts are equal.

The scores here are known without rounding: 1 / n for n equal logits (softmax), 1/2 and 1 for logits of 0 and 100 (sigmoid:
1 - 4e-44 is 1 in 64 bits).  Biases are small integers over 64, so s + b and the sum of two such are exact in 64 bits, and
two that are equal as real numbers are equal there: the lower group, the lower id is due."""
import math

import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def choice(c, K, G, KG, group):
    """ids by the definition, for scores c [T, E] that are exact; -inf: never picked."""
    T, E = c.shape
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
    return torch.where(top.values[:, :K] > -math.inf, top.indices[:, :K], torch.full((T, K), -1)).int()


def check(logits, bias, c, K, G, KG, group, score):
    ids, _ = umdk_amd.moe_route_grouped(logits.to(DEV), bias.float().to(DEV), K, G, KG, score, group, True, 1.0)
    want = choice(c, K, G, KG, group)
    assert torch.equal(ids.cpu(), want), (ids.cpu() != want).any(dim=1).nonzero().flatten()[:5].tolist()


@pytest.mark.parametrize("bias", [[-0.078125, 0.203125, 0.078125, -0.125, 0.15625, 0.0, 0.125, -0.171875],
                                  [3 * 2.0 ** 60, 3 * 2.0 ** 60, 0, 0, 4 * 2.0 ** 60, 2 * 2.0 ** 60, 0, 0],
                                  [2.0, -1.5, -4, -4, 1.5, -1.0, -4, -4],          # sums of parts that cancel
                                  [-2.125, -2.125, -4, -4, -2.0, -2.25, -4, -4]])
def test_equal_group_sums_of_different_parts(bias):
    b = torch.tensor(bias, dtype=torch.float64)
    for T in (1, 4100):
        for flip in (b, torch.cat([b[4:], b[:4]])):
            check(torch.zeros(T, 8), flip, (flip + 0.125).expand(T, 8), 2, 2, 1, "top2", "softmax")
            check(torch.zeros(T, 8), flip, (flip + 0.5).expand(T, 8), 2, 2, 1, "top2", "sigmoid")


def test_equal_group_sums_of_many_experts():
    b = torch.full((512,), -0.45, dtype=torch.float64).float().double()
    b[254], b[255], b[256], b[257] = -1 / 16, 1 / 16, 0.0, 0.0
    for shift in (0.0, -2.0):   # (scores above and below zero)
        c = (b + shift + 0.5).expand(3, 512)
        check(torch.zeros(3, 512), b + shift, c, 1, 2, 1, "top2", "sigmoid")


SIZES = [(1, 8, 2, 2, 1), (7, 96, 8, 8, 3), (9, 256, 8, 8, 4), (5, 512, 6, 16, 4), (6, 64, 4, 32, 3), (8, 60, 5, 5, 2), (9, 72, 3, 6, 2),
         (3, 384, 12, 4, 2), (4, 512, 16, 2, 1), (1030, 160, 6, 8, 3), (4099, 256, 8, 8, 4), (4100, 512, 12, 16, 4),
         (8195, 64, 8, 8, 4), (8193, 192, 6, 6, 2), (24577, 256, 8, 8, 4), (4097, 40, 4, 4, 2), (4097, 510, 9, 34, 3)]


@pytest.mark.parametrize("T,E,K,G,KG", SIZES)
@pytest.mark.parametrize("group", ["top2", "max"])
def test_random_ties_of_sigmoid_scores(T, E, K, G, KG, group):
    g = torch.Generator().manual_seed(T + E)
    for lo, hi in ((-16, 16), (-128, 128), (-256, -128)):
        b = torch.randint(lo, hi + 1, (E,), generator=g).double() / 64
        on = torch.randint(0, 2, (T, E), generator=g)
        there = torch.rand(T, E, generator=g) < 0.9
        logits = torch.where(there, 100.0 * on, torch.full((T, E), -math.inf))
        c = torch.where(there, 0.5 + 0.5 * on.double() + b, torch.full((T, E), -math.inf, dtype=torch.float64))
        check(logits, b, c, K, G, KG, group, "sigmoid")


@pytest.mark.parametrize("T,E,K,G,KG", SIZES)
@pytest.mark.parametrize("group", ["top2", "max"])
def test_random_ties_of_softmax_scores(T, E, K, G, KG, group):
    # n of a token's experts share its softmax, 1 / n each: the order is that of the biases, sums of two shift by 2 / n
    # (a second expert missing is the one case where they do not: no group is left with one)
    g = torch.Generator().manual_seed(T + E)
    for lo, hi in ((-16, 16), (-128, 128), (-256, -128)):
        b = torch.randint(lo, hi + 1, (E,), generator=g).double() / 64
        there = torch.rand(T, E, generator=g) < 0.9
        there.view(T, G, E // G)[:, :, :2] = True
        logits = torch.where(there, torch.randn(T, 1, generator=g), torch.full((T, E), -math.inf))
        c = torch.where(there, b, torch.full((T, E), -math.inf, dtype=torch.float64))
        check(logits, b, c, K, G, KG, group, "softmax")


def test_equal_scores_of_different_parts():
    # 1/2 + 1/2 and 1 + 0; 1/2 - 1/2 and 1 - 1; in both orders of the ids
    logits = torch.tensor([[0.0, 100.0, 100.0, 0.0], [100.0, 0.0, 0.0, 100.0]])
    for b in ([0.5, 0.0, 0.0, 0.5], [-0.5, -1.0, -1.0, -0.5], [0.0, -0.5, -0.5, 0.0]):
        b = torch.tensor(b, dtype=torch.float64)
        c = torch.where(logits > 0, 1.0, 0.5).double() + b
        for K in (1, 2, 4):
            check(logits, b, c, K, 1, 1, "max", "sigmoid")
