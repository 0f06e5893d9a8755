"""The numbers inside the operators of a decode step: sums whose terms cancel, so that what the operators hold in between
comes out at the end, unhidden by the output's rounding."""
import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def one_expert(x, w1, w2, dtype):
    """moe_decode_layer with one expert, whose gate is 1, of small whole weights, the same in every type."""
    H, I = x.shape[1], w2.shape[1]
    cast = lambda w: w.to(torch.float32).to(TYPES[dtype])[None].contiguous().to(DEV)  # noqa: E731
    ones = lambda n, k: None if dtype == "bf16" else torch.ones(  # noqa: E731
        (1, n) if dtype == "int8" else (1, n // 128, k // 128), device=DEV)
    router = torch.zeros(1, H, device=DEV)
    out, ids, gates = umdk_amd.moe_decode_layer(x.to(DEV), router, None, cast(w1), ones(2 * I, H), cast(w2), ones(H, I), 1)
    assert (ids == 0).all() and (gates == 1).all()
    return out.cpu().double()


def cancelling_pairs(I, H, pairs):
    """W1 and W2 by which out[n] = 3 silu(x[2 + n]) x[0] - silu(x[2 + n]) x[1] for n < pairs, 0 for the others."""
    w1, w2 = torch.zeros(2 * I, H), torch.zeros(H, I)
    for n in range(pairs):
        w1[2 * n, 2 + n] = w1[2 * n + 1, 2 + n] = 1
        w1[I + 2 * n, 0] = w1[I + 2 * n + 1, 1] = 1
        w2[n, 2 * n], w2[n, 2 * n + 1] = 3, -1
    return w1, w2


@pytest.mark.parametrize("dtype", ["bf16", "int8", "fp8"])
def test_h_reaches_the_second_product_with_all_its_bits(dtype):
    """With x[0] = 1 and x[1] = 3 every output is 3 s - 3 s = 0.  g and u are exact, s is the same number in both terms, 3 s is
    rounded once (2^-24 of it); the products' six parts are exact and each addition of theirs loses 2^-23 of 3 s at most, however a
    matrix instruction rounds: together less than 2^-20 of 3 s.  (With 16 bits of h the terms are up to 2^-18 of 3 s apart.)"""
    T, H, I, pairs = 5, 256, 128, 64
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(1)).bfloat16()
    x[:, 0], x[:, 1] = 1, 3
    g = x[:, 2:2 + pairs].double()
    out = one_expert(x, *cancelling_pairs(I, H, pairs), dtype)
    assert (out[:, :pairs].abs() <= 3 * (torch.sigmoid(g) * g).abs() * 2.0 ** -20).all()
    assert (out[:, pairs:] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "int8", "fp8"])
def test_an_infinite_h_stays_infinite(dtype):
    """h past the range of 32 bits is an infinity, and so are sums of it with weights of one sign."""
    H, I = 256, 128
    x = torch.zeros(3, H, dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = 1e30, torch.tensor([1e30, -1e30, 1e-30])
    w1, w2 = torch.zeros(2 * I, H), torch.ones(H, I)
    w1[:I, 0] = w1[I:, 1] = 1
    w2[1::2] = -1
    out = one_expert(x, w1, w2, dtype)
    sign = torch.tensor([1.0, -1.0]).repeat(H // 2)
    assert torch.equal(out[0], sign * float("inf")) and torch.equal(out[1], -sign * float("inf"))
    # (1e30 and 1e-30 to 2^-9 each, the sum of 128 products of 1, the output to 2^-8)
    assert ((out[2] - 128 * sign).abs() <= 128 * (2.0 ** -7 + 2.0 ** -8)).all()


@pytest.mark.parametrize("lo,hi", [(-4, 4), (-30, -4), (-80, -30)])
def test_silu_far_from_zero(lo, hi):
    """out[n] = h - 64 v - 64 w with v and w the leading 16 bits of h / 64, exact as products with a gate of 64, whose sigmoid
    is 1.  The exponential is within 2^-22 of itself, 1 + e and the quotient are rounded once each, u is a power of two, and five
    additions lose 2^-23 of h each at most: 2^-20 of h, and the output's rounding."""
    T, H, I, n = 4, 256, 256, 60
    g = torch.Generator().manual_seed(2)
    x = torch.zeros(T, H, dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = 64, 2.0 ** 40
    x[:, 2:2 + n] = (torch.rand(T, n, generator=g) * (hi - lo) + lo).bfloat16()
    gate = x[:, 2:2 + n].double()
    h = torch.sigmoid(gate) * gate * 2.0 ** 40
    x[:, 2 + n:2 + 2 * n] = (h / 64).bfloat16()
    x[:, 2 + 2 * n:2 + 3 * n] = (h / 64 - x[:, 2 + n:2 + 2 * n].double()).bfloat16()
    w1, w2 = torch.zeros(2 * I, H), torch.zeros(H, I)
    for i in range(n):
        w1[i, 2 + i] = w1[I + i, 1] = 1
        for k in (1, 2):
            w1[k * n + i, 0] = w1[I + k * n + i, 2 + k * n + i] = 1
        w2[i, i], w2[i, n + i], w2[i, 2 * n + i] = 1, -1, -1
    want = h - 64 * (x[:, 2 + n:2 + 2 * n].double() + x[:, 2 + 2 * n:2 + 3 * n].double())
    out = one_expert(x, w1, w2, "bf16")[:, :n]
    assert ((out - want).abs() <= h.abs() * 2.0 ** -20 + want.abs() * 2.0 ** -8).all()


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("T", [1, 6, 13])
def test_rows_that_are_not_finite_do_not_come_out_clean(T, shared):
    """A NaN, or infinities that cancel, leave a token without a logit and so without an expert: its results are NaN, with a shared
    expert beside the others or without, unless the token is not active; the tokens beside it keep their bits."""
    g = torch.Generator().manual_seed(3)
    H, E, I = 512, 16, 128
    x = torch.randn(T, H, generator=g).bfloat16().to(DEV)
    router = (torch.randn(E, H, generator=g) * H ** -0.5).to(DEV)
    router[:, 9] = router[:, 5]
    w1, w2 = (torch.randn(E, n, k, generator=g).mul_(k ** -0.5).bfloat16().to(DEV) for n, k in ((2 * I, H), (H, I)))
    kw = dict(share_gmm1_weight=w1[0], share_gmm2_weight=w2[0]) if shared else {}
    call = lambda x, m: umdk_amd.moe_decode_layer(x, router, None, w1, None, w2, None, 4, x_active_mask=m, **kw)  # noqa: E731
    want = call(x, None)
    bad = x.clone()
    bad[0, 7] = float("nan")
    bad[T - 1, 500] = float("-nan")
    if T > 4:
        bad[2, 5], bad[2, 9] = float("inf"), -float("inf")
    rows = sorted({0, T - 1} | ({2} if T > 4 else set()))
    keep = [t for t in range(T) if t not in rows]
    out, ids, gates = call(bad, None)
    assert (ids[rows] == -1).all() and (gates[rows] == 0).all() and out[rows].isnan().all()
    for a, b in zip((out, ids, gates), want):
        assert torch.equal(a[keep], b[keep])
    mask = torch.ones(T, dtype=torch.bool, device=DEV)
    mask[T - 1] = False
    out, ids, _ = call(bad, mask)
    assert (out[T - 1] == 0).all() and (T == 1 or out[0].isnan().all()) and torch.equal(out[keep], want[0][keep])


@pytest.mark.parametrize("T,shared", [(1, True), (9, False)])
def test_a_wait_that_gives_up_says_so(T, shared):
    """Forced by the host: with every target unreachable and a bound of 20 us each wait gives up, the launch ends normally, its rows
    are NaN, those of tokens that are not active 0, and the status is set; the next call is itself again."""
    from umdk_amd import _lib
    g = torch.Generator().manual_seed(4)
    H, E, I = 512, 16, 256
    x = torch.randn(T, H, generator=g).bfloat16().to(DEV)
    router = torch.randn(E, H, generator=g).to(DEV)
    w1, w2 = (torch.randn(E, n, k, generator=g).mul_(k ** -0.5).bfloat16().to(DEV) for n, k in ((2 * I, H), (H, I)))
    kw = dict(share_gmm1_weight=w1[0], share_gmm2_weight=w2[0]) if shared else {}
    mask = torch.arange(T, device=DEV) != 3
    call = lambda: umdk_amd.moe_decode_layer(x, router, None, w1, None, w2, None, 4, x_active_mask=mask, **kw)  # noqa: E731
    _lib.sync_status(clear=True)
    want = call()
    assert _lib.sync_status() == 0
    L = _lib.lib()
    print("layer, forced give-up", flush=True)
    L.camhipDebugSetSyncWait(2000, 1)
    try:
        out, ids, gates = call()
        torch.cuda.synchronize()
    finally:
        L.camhipDebugSetSyncWait(0, 0)
    assert _lib.sync_status() == 2 and _lib.sync_status(clear=True) == 2 and _lib.sync_status() == 0
    assert out[mask].isnan().all() and (out[~mask] == 0).all()
    assert torch.equal(ids, want[1]) and torch.equal(gates, want[2])
    assert all(torch.equal(a, b) for a, b in zip(call(), want)) and _lib.sync_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,base", [(1, 64, torch.float32), (70, 33, torch.float32), (300, 100, torch.float16),
                                      (2900, 4232, torch.bfloat16), (8300, 2600, torch.bfloat16)])
def test_z_reaches_the_second_product_with_all_its_bits(M, N, base, dtype):
    """Whole numbers: with A's row 9 three times its row 3 out[n] = 3 z - 1 (3 z) = 0, exactly: the magnitudes of no sum on the way
    come to 2^24 (32 products of up to 255 * 2^7 by up to 3 are below 2^22, the second product's two terms together below 2^23)."""
    g = torch.Generator().manual_seed(5)
    K, R, L = 32, 16, 2
    x = torch.randint(128, 256, (M, K), generator=g) * 2 ** torch.randint(0, 8, (M, K), generator=g)
    x = (x * (torch.randint(0, 2, (M, K), generator=g) * 2 - 1)).to(dtype).to(DEV)
    a = torch.zeros(L, R, K, dtype=dtype)
    a[:, 3] = torch.randint(-1, 2, (L, K), generator=g).to(dtype)
    a[:, 9] = 3 * a[:, 3]
    b = torch.zeros(L, N, R, dtype=dtype)
    b[:, :, 3], b[:, :, 9] = 3, -1
    ids = (torch.arange(M) % 2).int().to(DEV)
    out = umdk_amd.lora_add(torch.zeros(M, N, dtype=base, device=DEV), x, a.to(DEV), b.to(DEV), ids)
    assert not out.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(5, 64, 48), (40, 72, 208), (300, 100, 64), (2900, 4232, 80), (8300, 2600, 48)])
def test_an_infinite_z_stays_infinite(M, N, K, dtype):
    """Products of an infinity with ones are infinite, and so are their sums with finite terms, wherever in the row it stands."""
    R = 16
    x = torch.ones(M, K, dtype=dtype)
    x[0::3, K - 1] = float("inf")
    x[1::3, 0] = -float("inf")
    a, b = torch.ones(2, R, K, dtype=dtype), torch.ones(2, N, R, dtype=dtype)
    a[1] = -1
    b[:, 1::2] = -1
    ids = (torch.arange(M) // 7 % 2).int()
    base = torch.zeros(M, N, dtype=dtype)
    out = umdk_amd.lora_add(base.to(DEV), x.to(DEV), a.to(DEV), b.to(DEV), ids.to(DEV)).cpu()
    z = (x.float().sum(1) * (1 - 2 * ids.float()))[:, None] * R
    assert torch.equal(out.float(), (z * torch.tensor([1.0, -1.0]).repeat(N // 2)).to(dtype).float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_finite_numbers_beside_an_infinite_z_stay_finite(dtype):
    """One row of A is infinite: its z is, and the others', far past what fp16 holds, are not."""
    K, R, N = 32, 16, 40
    x = torch.full((3, K), 60000.0, dtype=dtype)
    a, b = torch.full((1, R, K), -30000.0, dtype=dtype), torch.ones(1, N, R, dtype=dtype)
    a[0, 4, 7] = float("inf")
    out = umdk_amd.lora_add(torch.zeros(3, N, dtype=dtype, device=DEV), x.to(DEV), a.to(DEV), b.to(DEV),
                            torch.zeros(3, dtype=torch.int32, device=DEV))
    assert (out == float("inf")).all()


def test_a_row_whose_logits_are_all_minus_infinity():
    """No expert, as the routing has it: NaN for a row that is not finite, an empty sum for one whose logits pass 32 bits."""
    H, E, I = 256, 4, 128
    x = torch.zeros(3, H, dtype=torch.bfloat16)
    x[0, 3], x[1, 3], x[2, 3] = float("inf"), 1e38, 1.0
    router = torch.full((E, H), -1.0)
    router[:, 3] = -1e30
    w1, w2 = torch.ones(E, 2 * I, H, dtype=torch.bfloat16), torch.ones(E, H, I, dtype=torch.bfloat16)
    out, ids, gates = umdk_amd.moe_decode_layer(x.to(DEV), router.to(DEV), None, w1.to(DEV), None, w2.to(DEV), None, 2)
    assert (ids[:2] == -1).all() and (gates[:2] == 0).all() and (ids[2] >= 0).all()
    assert out[0].isnan().all() and (out[1] == 0).all() and out[2].isfinite().all()
