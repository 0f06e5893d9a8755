"""lora_add on the rows of a batch in other orders."""
import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("M,K,N,L,R,dtype,rows,base", [
    (5, 64, 96, 2, 8, "bf16", "bf16", "bf16"), (64, 1024, 512, 32, 16, "bf16", "int8", "fp32"),
    (256, 512, 200, 20, 40, "fp16", "fp16", "fp16"), (257, 512, 96, 300, 24, "bf16", "bf16", "bf16"),
    (2900, 256, 4232, 40, 32, "bf16", "bf16", "bf16"), (3000, 256, 1031, 8, 64, "fp16", "int8", "fp16"),
    (8300, 144, 2600, 6, 64, "bf16", "bf16", "bf16"), (9000, 128, 264, 64, 16, "fp16", "fp16", "fp32"),
])
def test_a_row_has_the_same_bits_in_any_order(M, K, N, L, R, dtype, rows, base):
    """Of a batch of the same size and the same adapters: rows in other orders, sorted by adapter and back to front."""
    types = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
    g = torch.Generator().manual_seed(M)
    x = (torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8) if rows == "int8"
         else torch.randn(M, K, generator=g).to(types[rows])).to(DEV)
    xs = (torch.rand(M, generator=g) * 0.02).to(DEV) if rows == "int8" else None
    a = (torch.randn(L, R, K, generator=g) * K ** -0.5).to(types[dtype]).to(DEV)
    b = torch.randn(L, N, R, generator=g).to(types[dtype]).to(DEV)
    ids = torch.randint(-1, L, (M,), generator=g).int().to(DEV)
    y = torch.randn(M, N, generator=g).to(types[base]).to(DEV)
    scaling = torch.rand(L, generator=g).to(DEV)
    want = umdk_amd.lora_add(y, x, a, b, ids, scaling, xs)
    for p in (torch.randperm(M, generator=g).to(DEV), torch.argsort(ids, stable=True), torch.arange(M - 1, -1, -1, device=DEV)):
        got = umdk_amd.lora_add(y[p].contiguous(), x[p].contiguous(), a, b, ids[p].contiguous(), scaling,
                                None if xs is None else xs[p].contiguous())
        assert torch.equal(got, want[p])
