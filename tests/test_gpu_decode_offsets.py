"""The operators of a decode step where byte offsets pass 32 bits.

What lies past 4 GiB is compared with the same data in small tensors, bit for bit: an offset that loses its high bits reads
other data, which is there (every 4 GiB of the large tensors begin with other numbers)."""
import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GIB4 = 1 << 32


@pytest.fixture(autouse=True)
def memory_given_back():
    yield
    torch.cuda.empty_cache()


def test_experts_past_4_gib():
    """272 int8 experts of 4096 x 4096: 9.1 GB and 4.6 GB.  The last ones, picked by the bias, against the same among few."""
    g = torch.Generator(device=DEV).manual_seed(1)
    E, H, I = 272, 4096, 4096
    w1 = torch.randint(-100, 100, (E, 2 * I, H), generator=g, device=DEV, dtype=torch.int8)
    w2 = torch.randint(-100, 100, (E, H, I), generator=g, device=DEV, dtype=torch.int8)
    assert w1[:-1].numel() > 2 * GIB4 and w2[:-1].numel() > GIB4
    s1, s2 = (torch.rand(E, n, generator=g, device=DEV) * 1e-3 for n in (2 * I, H))
    x = torch.randn(2, H, generator=g, device=DEV).bfloat16()
    picks = [271, 0, 130, 260]  # (w1 past 8 GiB and w2 past 4 GiB, neither, w1 past 4 GiB, both again)
    bias = torch.zeros(E, device=DEV)
    bias[picks] = torch.tensor([4.0, 3.0, 2.0, 1.0], device=DEV)
    out, ids, gates = umdk_amd.moe_decode_layer(x, torch.zeros(E, H, device=DEV), bias, w1, s1, w2, s2, 4)
    assert ids.tolist() == [picks] * 2
    few = [t[picks].contiguous() for t in (w1, s1, w2, s2)]
    want, ids, wgates = umdk_amd.moe_decode_layer(x, torch.zeros(4, H, device=DEV), torch.tensor([4.0, 3.0, 2.0, 1.0], device=DEV), *few, 4)
    assert ids.tolist() == [[0, 1, 2, 3]] * 2 and torch.equal(gates, wgates) and torch.equal(out, want)
    assert out.isfinite().all() and out.any()


def test_block_scales_of_many_experts():
    """fp8 experts whose weights pass 4 GiB, with their scales."""
    g = torch.Generator(device=DEV).manual_seed(2)
    E, H, I = 512, 4096, 2176
    w1 = torch.randint(0, 0x78, (E, 2 * I, H), generator=g, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
    w2 = torch.randint(0, 0x78, (E, H, I), generator=g, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert (E - 1) * 2 * I * H > 2 * GIB4 and (E - 1) * I * H > GIB4
    s1 = torch.rand(E, 2 * I // 128, H // 128, generator=g, device=DEV) * 1e-3
    s2 = torch.rand(E, H // 128, I // 128, generator=g, device=DEV) * 1e-3
    x = torch.randn(3, H, generator=g, device=DEV).bfloat16()
    picks, order = [511, 3, 500], torch.tensor([3.0, 2.0, 1.0], device=DEV)
    bias = torch.zeros(E, device=DEV)
    bias[picks] = order
    out, ids, _ = umdk_amd.moe_decode_layer(x, torch.zeros(E, H, device=DEV), bias, w1, s1, w2, s2, 3)
    assert ids.tolist() == [picks] * 3
    few = [torch.stack([t[e].view(torch.uint8) for e in picks]).view(t.dtype) if t.dtype != torch.float32 else t[picks].contiguous()
           for t in (w1, s1, w2, s2)]
    want = umdk_amd.moe_decode_layer(x, torch.zeros(3, H, device=DEV), order, *few, 3)[0]
    assert torch.equal(out, want) and out.isfinite().all() and out.any()


def few_adapters(base, x, a, b, ids, picks, **kw):
    """The same call with the picked adapters alone."""
    few = torch.full_like(ids, -1)
    for i, p in enumerate(picks):
        few[ids == p] = i
    return umdk_amd.lora_add(base, x, a[picks].contiguous(), b[picks].contiguous(), few, **kw)


@pytest.mark.parametrize("M", [7, 300])
def test_first_matrices_past_4_gib(M):
    """130 adapters of rank 256 on 131056 columns: 8.7 GB.  (M = 300: chunks of 32 rows, ids in no order.)"""
    g = torch.Generator(device=DEV).manual_seed(3)
    L, R, K, N = 130, 256, 131056, 64
    a = torch.empty(L, R, K, device=DEV, dtype=torch.bfloat16)
    for i in range(L):
        a[i] = torch.randn(R, K, generator=g, device=DEV) * K ** -0.5
    assert (L - 1) * R * K * 2 > 2 * GIB4
    b = torch.randn(L, N, R, generator=g, device=DEV).bfloat16()
    picks = [129, 0, 65, 100]
    ids = torch.tensor(picks + [-1], dtype=torch.int32, device=DEV)[torch.randint(0, 5, (M,), generator=g, device=DEV)].contiguous()
    ids[:5] = torch.tensor(picks + [-1], dtype=torch.int32, device=DEV)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    base = torch.zeros(M, N, device=DEV, dtype=torch.bfloat16)
    out = umdk_amd.lora_add(base, x, a, b, ids)
    for p, t in zip(picks, range(4)):
        z = x[t].double() @ a[p].double().t().contiguous()
        want = z @ b[p].double().t().contiguous()
        # (K products of the row, each step of the sum within 2^-24, a few hundred steps a wave: far below the output's 2^-8)
        assert (out[t].double() - want).norm() <= 2.0 ** -8 * want.norm()
    if M > 256:  # (the split of K goes by M and the number of adapters: equal there)
        assert torch.equal(out, few_adapters(base, x, a, b, ids, picks))


@pytest.mark.parametrize("M,dtype", [(9, torch.bfloat16), (600, torch.float16), (2000, torch.bfloat16)])
def test_second_matrices_past_4_gib(M, dtype):
    """70 adapters of 2^18 columns and rank 128: 4.7 GB; base and out of 2000 rows 1 GB each."""
    g = torch.Generator(device=DEV).manual_seed(4)
    L, R, K, N = 70, 128, 64, 1 << 18
    b = torch.empty(L, N, R, device=DEV, dtype=dtype)
    for i in range(L):
        b[i] = torch.randn(N, R, generator=g, device=DEV)
    assert (L - 1) * N * R * 2 > GIB4
    a = (torch.randn(L, R, K, generator=g, device=DEV) * K ** -0.5).to(dtype)
    picks = [69, 0, 35, 64]
    ids = torch.tensor(picks, dtype=torch.int32, device=DEV)[torch.arange(M, device=DEV) * 4 // M].contiguous()
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    base = torch.zeros(M, N, device=DEV, dtype=dtype)
    out = umdk_amd.lora_add(base, x, a, b, ids)
    for t in (0, M // 3, M // 2, M - 1):
        p = int(ids[t])
        want = (x[t].double() @ a[p].double().t().contiguous()) @ b[p].double().t().contiguous()
        assert (out[t].double() - want).norm() <= 2.0 ** -8 * want.norm()


@pytest.mark.parametrize("rows,step,M,dtype", [("bf16", 1 << 24, 200, torch.bfloat16), ("int8", 1 << 25, 300, torch.bfloat16),
                                               ("bf16", 1 << 18, 9000, torch.bfloat16)])
def test_rows_past_4_gib(rows, step, M, dtype):
    """Rows of x far apart (and of base, where it fits): the last of them past 4 GiB."""
    g = torch.Generator(device=DEV).manual_seed(5)
    K, N, R, L = 80, 128, 16, 3
    x = (torch.randint(-127, 128, (M, K), generator=g, device=DEV, dtype=torch.int8) if rows == "int8"
         else torch.randn(M, K, generator=g, device=DEV).to(dtype))
    xs = torch.rand(M, generator=g, device=DEV) if rows == "int8" else None
    a = (torch.randn(L, R, K, generator=g, device=DEV) * K ** -0.5).to(dtype)
    b = torch.randn(L, N, R, generator=g, device=DEV).to(dtype)
    ids = torch.randint(-1, L, (M,), generator=g, device=DEV).int()
    base = torch.randn(M, N, generator=g, device=DEV).to(dtype)
    want = umdk_amd.lora_add(base, x, a, b, ids, None, xs)
    far = torch.zeros((M - 1) * step + K, device=DEV, dtype=x.dtype).as_strided((M, K), (step, 1))
    far.copy_(x)
    assert (M - 1) * step * x.element_size() > GIB4
    assert torch.equal(umdk_amd.lora_add(base, far, a, b, ids, None, xs), want)
    del far
    wide = torch.zeros((M - 1) * step + N, device=DEV, dtype=dtype).as_strided((M, N), (step, 1))
    wide.copy_(base)
    assert torch.equal(umdk_amd.lora_add(wide, x, a, b, ids, None, xs), want)
