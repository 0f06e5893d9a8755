"""add_rms_norm against its formula in 64 bits, and its codes against the recipe in fp32 bit for bit.

The fp32 part of an output: the sum of squares (8 + 4 + 6 + 16 additions at most in a row, halved by the root), the mean, eps,
the root, its reciprocal, v itself and two products: below 32 roundings of 2^-24.  The output's own rounding is half a step
of its type."""
import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 32 * 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rows(T, H, seed, dtype, stride=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, stride or H, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    return x.to(dtype).to(DEV)[:, :H]


def weights(H, dtype, seed=1):
    return (1.0 + 0.3 * torch.randn(H, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def check(x, residual, weight, quant, eps=1e-6):
    y, scale, new = umdk_amd.add_rms_norm(x, residual, weight, eps, quant)
    f = x.cpu().float() if residual is None else x.cpu().float() + residual.cpu().float()
    if residual is None:
        assert new.numel() == 0
    else:
        assert torch.equal(new.cpu(), f.to(x.dtype))
    v = x.cpu().double() if residual is None else x.cpu().double() + residual.cpu().double()
    r = torch.rsqrt(v.square().mean(dim=1, keepdim=True) + eps)
    w = weight.cpu().double()
    y, scale = y.cpu(), scale.cpu()
    if quant == 0:
        want = v * r * w
        small = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps  # a step of the subnormal range
        assert y.dtype == x.dtype and scale.numel() == 0
        assert ((y.double() - want).abs() <= (HALF[x.dtype] + U) * want.abs() + small).all()
        return
    t = f * weight.cpu().float()
    T, H = x.shape
    b = t.view(T, 1, H) if quant == 2 else t.view(T, H // 128, 128)
    a = b.abs().amax(dim=2, keepdim=True).clamp(min=2.0 ** -100)
    most = 127.0 if quant == 2 else 448.0
    codes = b * torch.div(torch.full_like(a, most), a)
    if quant == 2:
        assert y.dtype == torch.int8 and torch.equal(y, torch.round(codes).to(torch.int8).view(T, H))
        assert scale.shape == (T,)
    else:
        want = codes.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(T, H)
        assert y.dtype == torch.float8_e4m3fn and torch.equal(y.view(torch.uint8), want.view(torch.uint8))
        assert scale.shape == (T, H // 128)
    wants = (a.double() / most)[:, :, 0] * r
    err = (scale.double().view_as(wants) - wants).abs()
    assert (err <= U * wants).all(), float((err / wants).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quant", [0, 2, 3])
@pytest.mark.parametrize("T,H", [(1, 7168), (16, 7168), (5, 128), (1, 1), (3, 7), (9, 511), (130, 512), (4, 513), (7, 1024),
                                 (6, 1025), (2, 1536), (3, 2049), (300, 4096), (2, 8192), (3, 16383), (2, 16384),
                                 (1, 32768), (2, 20001), (1000, 384), (33, 5120)])
def test_against_the_formula(T, H, quant, dtype):
    if quant == 3 and H % 128:
        with pytest.raises(RuntimeError):
            umdk_amd.add_rms_norm(rows(T, H, 1, dtype), None, weights(H, dtype), 1e-6, 3)
        return
    check(rows(T, H, T + H, dtype), rows(T, H, T + H + 1, dtype), weights(H, dtype), quant)
    check(rows(T, H, T + H + 2, dtype), None, weights(H, torch.float32), quant)


@pytest.mark.parametrize("quant", [0, 2, 3])
def test_slices_strides_and_alignment(quant):
    bf = torch.bfloat16
    check(rows(40, 512, 3, bf, 576), None, weights(512, bf), quant)
    check(rows(40, 640, 3, bf, 651), rows(40, 640, 4, bf), weights(640, bf), quant)      # rows off every alignment
    flat = rows(1, 1 + 6 * 256, 5, bf)[0]
    check(flat[1:].view(6, 256), rows(6, 256, 6, bf), weights(257, bf)[1:], quant)       # bases off by one element
    check(rows(256, 12, 7, bf).t()[:, :128].contiguous().t().t(), None, weights(128, bf), quant)
    check(rows(128, 12, 7, bf).t(), rows(128, 12, 8, bf).t(), weights(128, bf), quant)   # columns first
    check(rows(1, 256, 9, bf).expand(5, 256), None, weights(256, bf), quant)
    w2 = weights(512, torch.float32)[::2]
    check(rows(3, 256, 9, bf), None, w2, quant)


@pytest.mark.parametrize("quant", [0, 2, 3])
def test_no_rows(quant):
    y, scale, new = umdk_amd.add_rms_norm(rows(0, 256, 1, torch.bfloat16), rows(0, 256, 1, torch.bfloat16),
                                          weights(256, torch.bfloat16), 1e-6, quant)
    assert y.shape == (0, 256) and new.shape == (0, 256)


@pytest.mark.parametrize("H", [512, 7168])
@pytest.mark.parametrize("quant", [0, 2, 3])
def test_zero_tiny_and_huge_rows(H, quant):
    x = rows(6, H, 3, torch.bfloat16)
    x[0] = 0
    x[1] *= 2.0 ** -110
    x[2] *= 2.0 ** 50
    x[3, 1:] = 0
    x[4] = 1e-20
    check(x, None, weights(H, torch.bfloat16), quant)
    check(x, None, weights(H, torch.bfloat16), quant, eps=1e-5)


@pytest.mark.parametrize("H", [256, 7168])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rows_with_infinities_and_nans_say_so(bad, H):
    x, res = rows(5, H, 3, torch.bfloat16), rows(5, H, 4, torch.bfloat16)
    x[2, H - 3] = bad
    w = weights(H, torch.bfloat16)
    good = [0, 1, 3, 4]
    for quant in (0, 2, 3):
        y, scale, new = umdk_amd.add_rms_norm(x, res, w, 1e-6, quant)
        yg, sg, ng = umdk_amd.add_rms_norm(x[good], res[good], w, 1e-6, quant)
        bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
        assert torch.equal(bits(y[good]), bits(yg)) and torch.equal(new[good], ng)   # the other rows do not notice
        if quant:
            assert torch.equal(scale[good], sg)
            assert torch.isnan(scale[2]).any() if quant == 2 else torch.isnan(scale[2, -1])
        else:
            assert torch.isnan(y[2, H - 3])


def test_offsets_past_32_bits():
    T, H = 262400, 8192   # 4.3 GB a tensor
    x = torch.zeros(T, H, dtype=torch.bfloat16, device=DEV)
    x[-3:] = rows(3, H, 3, torch.bfloat16)
    w = weights(H, torch.bfloat16)
    for quant in (0, 2, 3):
        y, scale, new = umdk_amd.add_rms_norm(x, x, w, 1e-6, quant)
        ys, ss, ns = umdk_amd.add_rms_norm(x[-3:], x[-3:], w, 1e-6, quant)
        bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
        assert torch.equal(bits(y[-3:]), bits(ys)) and torch.equal(new[-3:], ns)
        assert not quant or torch.equal(scale[-3:], ss)
        assert (y[T // 2].float() == 0).all()   # (zeros of both signs: a weight below zero turns them)
        del y, scale, new


def test_more_rows_than_a_launch_takes_threads_for():
    T, H = 2 ** 25 + 7, 3   # a wave of 64 threads a row
    x = torch.ones(T, H, dtype=torch.bfloat16, device=DEV)
    x[2 ** 25 - 4:] = rows(11, H, 3, torch.bfloat16)
    w = weights(H, torch.bfloat16)
    for quant in (0, 2):
        y, scale, new = umdk_amd.add_rms_norm(x, x, w, 1e-6, quant)
        ys, ss, ns = umdk_amd.add_rms_norm(x[-12:], x[-12:], w, 1e-6, quant)
        assert torch.equal(y[-12:], ys) and torch.equal(new[-12:], ns) and (not quant or torch.equal(scale[-12:], ss))
        assert torch.equal(y[:1], ys[:1]) and bool((y[:2 ** 25 - 4] == y[:1]).all())
        assert bool((new[:2 ** 25 - 4] == 2).all())


def test_results_do_not_hang_on_the_batch():
    x, res, w = rows(300, 7168, 3, torch.bfloat16), rows(300, 7168, 4, torch.bfloat16), weights(7168, torch.bfloat16)
    y, _, _ = umdk_amd.add_rms_norm(x, res, w)
    for i in (0, 1, 299):
        assert torch.equal(umdk_amd.add_rms_norm(x[i:i + 1], res[i:i + 1], w)[0], y[i:i + 1])


def test_captured_and_replayed():
    x, res, w = rows(64, 7168, 3, torch.bfloat16), rows(64, 7168, 4, torch.bfloat16), weights(7168, torch.bfloat16)
    umdk_amd.add_rms_norm(x, res, w, 1e-6, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.ops.umdk_cam_op_lib.add_rms_norm(x, res, w, 1e-6, 2)
    for seed in range(3):
        x.copy_(rows(64, 7168, 50 + seed, torch.bfloat16))
        graph.replay()
        for a, b in zip(held, umdk_amd.add_rms_norm(x, res, w, 1e-6, 2)):
            torch.cuda.synchronize()
            assert torch.equal(a, b)


@pytest.mark.parametrize("H", [256, 513, 7168])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinities_under_a_weight_of_zero_and_bad_weights_say_so(bad, H):
    x, res, w = rows(5, H, 3, torch.bfloat16), rows(5, H, 4, torch.bfloat16), weights(H, torch.bfloat16)
    w[7] = 0
    x[2, 7] = bad                     # 0 times it is NaN in the formula
    for quant in (0, 2, 3):
        if quant == 3 and H % 128:
            continue
        y, scale, _ = umdk_amd.add_rms_norm(x, res, w, 1e-6, quant)
        if quant == 0:
            assert torch.isnan(y[2, 7])
            continue
        by_row = torch.isnan(scale) if quant == 2 else torch.isnan(scale[:, 0])
        assert by_row.tolist() == [False, False, True, False, False]
    x[2, 7] = 1.0
    w[7] = bad                        # every row has it
    for quant in (0, 2, 3):
        if quant == 3 and H % 128:
            continue
        y, scale, _ = umdk_amd.add_rms_norm(x, res, w, 1e-6, quant)
        if quant == 0:
            assert not torch.isfinite(y[:, 7]).any() and torch.isfinite(y[:, 8:]).all()
        elif quant == 2:
            assert not torch.isfinite(scale).any()
        else:
            assert not torch.isfinite(scale[:, 0]).any() and torch.isfinite(scale[:, 1:]).all()
