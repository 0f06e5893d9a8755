"""Where the operators around the expert layer write: in place where the C ABI allows it, and nothing beside their outputs."""
import pytest
import torch

import umdk_amd
from tests.test_gpu_norm import rows, weights
from umdk_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = 0


def norm(x, residual, w, quant, y, scale, new, eps=1e-6):
    T, H = x.shape
    _lib.launch("camhipAddRmsNorm", x.data_ptr(), None if residual is None else residual.data_ptr(), w.data_ptr(), T, H, H, BF16,
                BF16, 5 if quant == 3 else quant, eps, y.data_ptr(), scale.data_ptr(), None if new is None else new.data_ptr(),
                device=x.device)


def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("quant", [0, 2, 3])
@pytest.mark.parametrize("T,H", [(1, 7168), (9, 7), (5, 513), (33, 7168), (7, 512), (6, 1024), (3, 20001), (2, 32768)])
def test_the_sum_may_go_where_the_residual_is(T, H, quant):
    if quant == 3 and H % 128:
        return
    x, res, w = rows(T, H, 1, torch.bfloat16), rows(T, H, 2, torch.bfloat16), weights(H, torch.bfloat16)
    y, scale, new = umdk_amd.add_rms_norm(x, res, w, 1e-6, quant)
    held = res.clone()
    y2, scale2 = torch.empty_like(y), torch.empty_like(scale)
    norm(x, held, w, quant, y2, scale2, held)
    assert torch.equal(held, new) and torch.equal(bits(y2), bits(y)) and torch.equal(scale2, scale)


class Guarded:
    """`count` elements between two runs of 512 of a pattern, off elements further on."""

    def __init__(self, count, dtype, off=0):
        size = torch.empty(0, dtype=dtype).element_size()
        self.bytes = torch.full(((1024 + off + count) * size,), 0xA5, dtype=torch.uint8, device=DEV)
        self.lo, self.hi = (512 + off) * size, (512 + off + count) * size
        self.part = self.bytes[self.lo:self.hi].view(dtype)

    def untouched(self):
        return bool((self.bytes[:self.lo] == 0xA5).all() and (self.bytes[self.hi:] == 0xA5).all())


@pytest.mark.parametrize("quant", [0, 2, 3])
@pytest.mark.parametrize("T,H", [(1, 1), (5, 7), (3, 509), (6, 513), (5, 512), (9, 1024), (2, 1025), (3, 7161), (5, 7168), (1, 16383),
                                 (2, 16385), (1, 32768), (2, 640), (3, 32767)])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_the_norm_writes_its_rows_only(T, H, quant, off):
    if quant == 3 and H % 128:
        return
    x, res, w = rows(T, H, 1, torch.bfloat16), rows(T, H, 2, torch.bfloat16), weights(H, torch.bfloat16)
    want = umdk_amd.add_rms_norm(x, res, w, 1e-6, quant)
    y = Guarded(T * H, want[0].dtype, off)
    scale = Guarded(want[1].numel(), torch.float32, off)
    new = Guarded(T * H, torch.bfloat16, off)
    norm(x, res, w, quant, y.part, scale.part, new.part)
    assert y.untouched() and scale.untouched() and new.untouched()
    assert torch.equal(y.part.view(torch.uint8), bits(want[0]).flatten()) and torch.equal(new.part.view(T, H), want[2])
    assert torch.equal(scale.part, want[1].t().flatten() if quant == 3 else want[1].flatten())


@pytest.mark.parametrize("T,E,K,G,KG", [(1, 256, 8, 8, 4), (17, 64, 6, 1, 1), (33, 160, 6, 8, 3), (5, 512, 16, 8, 4), (3, 60, 3, 5, 2),
                                        (1025, 256, 8, 8, 4), (2049, 96, 5, 1, 1), (8193, 64, 8, 8, 4), (24577, 256, 7, 8, 4),
                                        (4097, 512, 9, 1, 1), (7, 1, 1, 1, 1)])
@pytest.mark.parametrize("off", [0, 1])
def test_the_routing_writes_its_slots_only(T, E, K, G, KG, off):
    g = torch.Generator().manual_seed(T + E)
    logits, bias = torch.randn(T, E, generator=g).to(DEV), (0.1 * torch.randn(E, generator=g)).to(DEV)
    want = umdk_amd.moe_route_grouped(logits, bias, K, G, KG, "sigmoid")
    ids, w, wide = Guarded(T * K, torch.int32, off), Guarded(T * K, torch.float32, off), Guarded(T * K, torch.int64, off)
    _lib.launch("camhipMoeRouteGrouped", logits.data_ptr(), bias.data_ptr(), T, E, K, 4, E, G, KG, 1, 2, 1, 1.0,
                ids.part.data_ptr(), w.part.data_ptr(), wide.part.data_ptr(), device=logits.device)
    assert ids.untouched() and w.untouched() and wide.untouched()
    assert torch.equal(ids.part, want[0].flatten()) and torch.equal(w.part, want[1].flatten())
    assert torch.equal(wide.part, want[0].flatten().long())
