"""quant_matmul against the exact integer product (in 64-bit floats, which hold every sum) and the epilogue's fp32 steps:
bit for bit, whatever the shape and however the kernel splits it."""
import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def operands(m, n, k, seed, full=False):
    g = torch.Generator().manual_seed(seed)
    lo = -128 if full else -127
    x = torch.randint(lo, 128, (m, k), generator=g).to(torch.int8)
    w = torch.randint(lo, 128, (n, k), generator=g).to(torch.int8)
    xs = torch.rand(m, generator=g) * 0.1 + 1e-3
    ws = torch.rand(n, generator=g) * 0.01 + 1e-4
    return x, xs, w, ws, torch.randn(n, generator=g)


def reference(x, xs, w, ws, bias, dtype):
    acc = x.double() @ w.double().t()
    y = (acc.float() * ws) * xs[:, None]
    return (y if bias is None else y + bias).to(dtype)


def check(m, n, k, seed=0, dtypes=(torch.bfloat16,), full=False):
    x, xs, w, ws, bias = operands(m, n, k, seed, full)
    on = [t.to(DEV) for t in (x, xs, w, ws)]
    for i, dtype in enumerate(dtypes):
        b = bias if (i + seed) % 2 else None
        y = umdk_amd.quant_matmul(*on, None if b is None else b.to(DEV), dtype)
        assert y.dtype == dtype and torch.equal(y.cpu(), reference(x, xs, w, ws, b, dtype)), (m, n, k, dtype)


ALL = (torch.bfloat16, torch.float16, torch.float32)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 7, 16), (1, 4096, 7168), (2, 33, 48), (5, 130, 144), (16, 64, 64), (17, 65, 80),
                                   (31, 576, 7168), (33, 129, 1536), (64, 256, 128), (65, 511, 272), (1, 1, 16384),
                                   (3, 5001, 512), (100, 100, 1008), (7, 16, 131056)])
def test_few_rows(m, n, k):
    check(m, n, k, m + n, ALL)


@pytest.mark.parametrize("m,n,k", [(127, 128, 128), (128, 2112, 7168), (129, 257, 400), (200, 1000, 1024), (256, 256, 256),
                                   (257, 513, 1040), (511, 1408, 2048), (1021, 1001, 512), (1500, 96, 64), (2049, 300, 16),
                                   (300, 2500, 4096), (4096, 512, 512)])
def test_many_rows(m, n, k):
    check(m, n, k, m + n, ALL[(m + n) % 3:] + ALL[:(m + n) % 3])


# (a size for each of the kernels' shapes, which the launcher takes by what a product costs with them; edges in m, n and k)
@pytest.mark.parametrize("m,n,k", [(7, 4093, 1040), (13, 4001, 1200), (27, 4093, 1232), (61, 4099, 400), (95, 4091, 848),
                                   (9, 4567, 144), (250, 4001, 6416), (9, 8697, 272), (70, 8235, 272), (131, 8361, 272),
                                   (389, 8711, 144), (769, 7021, 656), (1042, 7209, 144), (1, 28672, 272), (3071, 1, 144)])
def test_every_shape_of_block(m, n, k):
    check(m, n, k, m + n, ALL[(m + n) % 3:] + ALL[:(m + n) % 3], full=True)


def test_extreme_codes_fit_the_sum():
    # -128 in every place: the largest sum there is, 2^14 k
    k = 131056
    x = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((5, k), -128, dtype=torch.int8, device=DEV)
    one = torch.ones(5, device=DEV)
    assert (umdk_amd.quant_matmul(x, one[:3], w, one, None, torch.float32) == float(k << 14)).all()
    check(65, 70, 2048, 3, full=True)


def test_scales_that_are_zero_or_not_finite():
    x, xs, w, ws, _ = (t.to(DEV) for t in operands(70, 80, 256, 1))
    want = umdk_amd.quant_matmul(x, xs, w, ws)
    xs[3], xs[4], ws[5] = 0.0, float("nan"), float("inf")
    y = umdk_amd.quant_matmul(x, xs, w, ws)
    rows = [i for i in range(70) if i not in (3, 4)]
    cols = [i for i in range(80) if i != 5]
    assert torch.equal(y[rows][:, cols], want[rows][:, cols])
    assert (y[3, cols] == 0).all() and torch.isnan(y[4]).all() and not torch.isfinite(y[rows][:, 5]).any()


def test_no_rows():
    x, xs, w, ws, _ = (t.to(DEV) for t in operands(4, 80, 256, 1))
    assert umdk_amd.quant_matmul(x[:0], xs[:0], w, ws).shape == (0, 80)


def test_nothing_is_written_behind_the_output():
    from umdk_amd import _lib
    for m, n, k in ((3, 5, 32), (70, 131, 64), (300, 515, 512), (129, 127, 4096)):
        x, xs, w, ws, _ = (t.to(DEV) for t in operands(m, n, k, 1))
        room = torch.full((m * n + 64,), 7.0, dtype=torch.bfloat16, device=DEV)
        _lib.call("camhipQuantMatmul", x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, m, n, k, 0,
                  room.data_ptr() + 64, device=x.device)
        assert torch.equal(room[32:32 + m * n].view(m, n), umdk_amd.quant_matmul(x, xs, w, ws))
        assert (room[:32] == 7).all() and (room[32 + m * n:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(270000, 24, 16400), (70000, 33001, 48), (5, 270001, 16400)])
def test_offsets_past_32_bits(m, n, k):
    # x, the output and W past 4 GiB: the last rows and columns against a product of their own
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8, device=DEV)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8, device=DEV)
    xs, ws = torch.rand(m, generator=g, device=DEV), torch.rand(n, generator=g, device=DEV)
    y = umdk_amd.quant_matmul(x, xs, w, ws)
    for rows in (slice(0, 3), slice(m // 2, m // 2 + 3), slice(m - 3, m)):
        for cols in (slice(0, 19), slice(n - 19, n)):
            want = reference(x[rows].cpu(), xs[rows].cpu(), w[cols].cpu(), ws[cols].cpu(), None, torch.bfloat16)
            assert torch.equal(y[rows, cols].cpu(), want)


def test_agrees_with_the_grouped_product():
    x, xs, w, ws, _ = (t.to(DEV) for t in operands(77, 512, 1024, 9))
    groups = torch.tensor([77], device=DEV)
    assert torch.equal(umdk_amd.quant_matmul(x, xs, w, ws), umdk_amd.grouped_matmul(x, xs, groups, w[None], ws[None]))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_two_streams_at_once_and_graphs(m):
    a = [t.to(DEV) for t in operands(m, 512, 4096, 1)[:4]]
    b = [t.to(DEV) for t in operands(m, 512, 4096, 2)[:4]]
    wa, wb = umdk_amd.quant_matmul(*a), umdk_amd.quant_matmul(*b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            got.append((umdk_amd.quant_matmul(*a), wa))
        with torch.cuda.stream(s2):
            got.append((umdk_amd.quant_matmul(*b), wb))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y, want in got)
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        ya = torch.ops.umdk_cam_op_lib.quant_matmul(*a)
    with torch.cuda.graph(gb, pool=ga.pool()):   # (captured after, and replayed in the order of their captures)
        yb = torch.ops.umdk_cam_op_lib.quant_matmul(*b)
    for _ in range(3):
        ya.zero_(), yb.zero_()
        ga.replay()
        gb.replay()
        eager = umdk_amd.quant_matmul(*a)
        torch.cuda.synchronize()
        assert torch.equal(ya, wa) and torch.equal(yb, wb) and torch.equal(eager, wa)
