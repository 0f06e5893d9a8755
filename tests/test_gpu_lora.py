"""lora_add against its definition in 64 bits.

Tolerances.  Products are exact in fp32 sums: a sum of n has at most n additions on its longest path, each within 2^-24 of
the sum of magnitudes; A x in between is held to 2^-16 of itself (bf16) or to 2^-21 of the row's
largest (fp16); scales and the roundings between them are 4 steps of 2^-24;
the output is rounded once, by 2^-8 (bf16) or 2^-11 (fp16) of it."""
import pytest
import torch

import umdk_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E32 = 2.0 ** -24
T16 = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(M, K, N, L, R, dtype="bf16", rows=None, base=None, none=0.2, seed=0, runs=False, scaling=True):
    g = torch.Generator().manual_seed(seed)
    rows, base = rows or dtype, base or dtype
    d = dict(a=(torch.randn(L, R, K, generator=g) * K ** -0.5).to(T16[dtype]),
             b=(torch.randn(L, N, R, generator=g) * R ** -0.5).to(T16[dtype]), base=torch.randn(M, N, generator=g).to(T16[base]),
             scaling=torch.rand(L, generator=g) * 2 if scaling else None, xs=None)
    if rows == "int8":
        d["x"] = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8)
        d["xs"] = torch.rand(M, generator=g) * 0.02 + 0.001
    else:
        d["x"] = torch.randn(M, K, generator=g).to(T16[rows])
    ids = torch.randint(0, L, (M,), generator=g)
    if runs:
        ids = ids[torch.sort(torch.randint(0, max(1, M // 50) + 1, (M,), generator=g)).values]
    ids[torch.rand(M, generator=g) < none] = -1
    d["ids"] = ids.int()
    return {k: None if v is None else v.to(DEV) for k, v in d.items()}


def call(d, out_dtype=None, **over):
    d = {**d, **over}
    return umdk_amd.lora_add(d["base"], d["x"], d["a"], d["b"], d["ids"], d["scaling"], d["xs"], out_dtype)


def check(d, got):
    bf16 = d["a"].dtype == torch.bfloat16
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    base, L = d["base"].double(), d["a"].shape[0]
    K, R = d["a"].shape[2], d["a"].shape[1]
    want, bound = base.clone(), torch.zeros_like(base)
    x = d["x"].double() if d["xs"] is None else d["x"].double() * d["xs"].double()[:, None]
    for a in range(L):
        t = torch.nonzero(d["ids"] == a)[:, 0]
        if not len(t):
            continue
        s = 1.0 if d["scaling"] is None else float(d["scaling"][a].double())
        A, B = d["a"][a].double().t().contiguous(), d["b"][a].double().t().contiguous()
        z, size = x[t] @ A * s, x[t].abs() @ A.abs() * abs(s)
        dz = size * (K * E32 + 4 * E32) + (z.abs() * 2.0 ** -16 if bf16 else z.abs().amax(1, keepdim=True) * 2.0 ** -21)
        want[t] += z @ B
        bound[t] += dz @ B.abs() + (R + 4) * E32 * ((z.abs() + dz) @ B.abs())
    bound += 4 * E32 * base.abs()
    assert got.isfinite().all()
    # (2^-25: half a step of fp16 where it has no normal numbers)
    assert ((got.double() - want).abs() <= want.abs() * half + bound * (1 + half) + (0 if half == 2.0 ** -8 else 2.0 ** -25)).all()
    keep = (d["ids"] < 0) | (d["ids"] >= L)
    assert torch.equal(got[keep], d["base"][keep].to(got.dtype))


@pytest.mark.parametrize("dtype,rows,base", [("bf16", "bf16", "bf16"), ("fp16", "fp16", "fp16"), ("bf16", "int8", "fp32"),
                                             ("fp16", "int8", "fp16"), ("bf16", "bf16", "fp32"), ("fp16", "fp16", "bf16")])
@pytest.mark.parametrize("M,K,N,L,R", [
    (1, 4096, 4096, 8, 16), (1, 16, 1, 1, 8), (3, 48, 17, 2, 8), (64, 1024, 512, 32, 16), (65, 1040, 513, 3, 24),
    (200, 640, 333, 20, 64), (257, 512, 96, 300, 40), (130, 2048, 1000, 2, 128), (37, 7168, 130, 5, 256), (20, 256, 4100, 20, 136),
])
def test_against_the_definition(dtype, rows, base, M, K, N, L, R):
    d = make(M, K, N, L, R, dtype, rows, base, seed=M)
    check(d, call(d))


@pytest.mark.parametrize("M,K,N,L,R,dtype,rows,base", [
    (1021, 1024, 640, 6, 32, "bf16", "bf16", "bf16"), (4099, 512, 264, 5, 16, "bf16", "int8", "fp32"),
    (3000, 256, 1031, 8, 64, "fp16", "fp16", "fp16"), (2500, 384, 300, 40, 72, "bf16", "bf16", "fp32"),
    (9000, 128, 128, 3, 8, "bf16", "bf16", "bf16"),
])
@pytest.mark.parametrize("runs", [True, False])
def test_prompts(M, K, N, L, R, dtype, rows, base, runs):
    d = make(M, K, N, L, R, dtype, rows, base, seed=M, runs=runs)
    check(d, call(d))


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513])
@pytest.mark.parametrize("how", ["one", "all different", "none", "two in turn"])
def test_row_counts_and_shares(M, how):
    d = make(M, 128, 80, max(M, 2), 16, seed=M, none=0.0)
    i = torch.arange(M, device=DEV, dtype=torch.int32)
    d["ids"] = {"one": i * 0 + 1, "all different": i.flip(0).contiguous(), "none": i * 0 - 1, "two in turn": i % 2}[how]
    check(d, call(d))


def test_no_rows():
    d = make(4, 64, 32, 2, 8)
    out = call(d, base=d["base"][:0], x=d["x"][:0], ids=d["ids"][:0])
    assert out.shape == (0, 32) and out.dtype == torch.bfloat16


def test_ids_outside_the_adapters():
    d = make(12, 64, 32, 3, 8, none=0.0)
    d["ids"] = torch.tensor([-1, 0, 1, 2, 3, -2 ** 31, 2 ** 31 - 1, 100, 0, -7, 2, 3], dtype=torch.int32, device=DEV)
    got = call(d)
    check(d, got)
    wide = d["ids"].long()
    wide[4], wide[0] = 2 ** 32, -2 ** 40   # (0 if cut to 32 bits)
    assert torch.equal(call(d, ids=wide), got)


def test_row_of_no_adapter_ignores_its_input():
    d = make(6, 64, 32, 3, 8, none=0.0)
    d["ids"][[1, 4]] = -1
    d["x"][[1, 4]] = float("nan")
    check(d, call(d))


def test_unused_adapters_are_not_read_into_the_sums():
    d = make(40, 256, 96, 8, 16, none=0.0)
    d["ids"] = (d["ids"] % 3 * 2).contiguous()
    want = call(d)
    for n in ("a", "b"):
        d[n][1::2] = float("nan")
    d["scaling"][1::2] = float("inf")
    assert torch.equal(call(d), want)


def test_infinities_and_nan_stay_in_their_rows():
    d = make(48, 256, 96, 4, 16, none=0.0)
    want = call(d)
    x = d["x"].clone()
    x[5, 9], x[20, 0] = float("nan"), float("inf")
    got = call(d, x=x)
    assert got[5].isnan().all() and not got[20].isfinite().any()
    others = torch.ones(48, dtype=torch.bool, device=DEV)
    others[[5, 20]] = False
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("dtype,rows", [("bf16", "bf16"), ("fp16", "int8")])
def test_strides_and_offsets(dtype, rows):
    d = make(70, 256, 100, 4, 16, dtype, rows, seed=3)
    want = call(d)
    wide = torch.zeros(70, 777, dtype=d["base"].dtype, device=DEV)
    wide[:, 13:113] = d["base"]
    xw = torch.zeros(70, 301, dtype=d["x"].dtype, device=DEV)
    xw[:, 3:259] = d["x"]
    assert torch.equal(call(d, base=wide[:, 13:113]), want)
    assert torch.equal(call(d, x=xw[:, 3:259]), want)
    assert torch.equal(call(d, base=d["base"].t().contiguous().t(), x=d["x"].t().contiguous().t()), want)
    assert torch.equal(call(d, ids=d["ids"].repeat_interleave(2)[::2], scaling=d["scaling"].repeat_interleave(3)[::3]), want)
    one = call(d, base=wide[2:3, 13:113], x=xw[2:3, 3:259], ids=d["ids"][2:3], xs=None if d["xs"] is None else d["xs"][2:3])
    assert one.shape == (1, 100)
    assert torch.equal(call(d, base=d["base"][:1].expand(70, 100)), call(d, base=d["base"][:1].expand(70, 100).contiguous()))


def test_without_scaling_and_other_output_types():
    d = make(33, 512, 200, 4, 32, "bf16", "bf16", "fp32", scaling=False)
    check(d, call(d))
    assert call(d).dtype == torch.bfloat16
    out = call(d, torch.float16)
    assert out.dtype == torch.float16
    check(d, out)
    f = make(33, 512, 200, 4, 32, "fp16", "fp16", "fp32")
    assert call(f).dtype == torch.float16


def test_the_same_bits_again_and_in_any_batch():
    d = make(300, 1024, 520, 6, 32, seed=8)
    want = call(d)
    for _ in range(3):
        assert torch.equal(call(d), want)


def test_captured_and_replayed():
    d = make(96, 1024, 512, 8, 16, "bf16", "int8", "fp32", seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(d)
        again = call(d, base=held.float())
    for seed in range(5):
        new = make(96, 1024, 512, 8, 16, "bf16", "int8", "fp32", seed=50 + seed, none=0.1 * seed)
        for n in ("x", "xs", "ids", "base", "scaling"):
            d[n].copy_(new[n])
        graph.replay()
        eager = call(d)
        second = call(d, base=eager.float())
        torch.cuda.synchronize()
        assert torch.equal(held, eager) and torch.equal(again, second), seed


def test_calls_on_several_streams_at_once():
    ds = [make(120 + i, 1024, 512, 8, 16, seed=i) for i in range(4)]
    want = [call(d) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    got = [[] for _ in ds]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(ds[i]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(o, w) for o in g)


def test_guard_bands_and_output_in_place_of_the_base():
    from umdk_amd import _lib
    d = make(67, 272, 131, 5, 24, none=0.2, seed=6)
    want = call(d)
    size = 67 * 131 * 2
    def args(base):
        return [base, d["x"].data_ptr(), None, d["a"].data_ptr(), d["b"].data_ptr(), d["ids"].data_ptr(),
                d["scaling"].data_ptr(), 67, 131, 272, 24, 5, 131, 272, 0, 0, 0, 0]
    need = _lib.workspace_size("camhipLoraAdd", *args(0x1000), 0x1000)
    ws = torch.full((need + 512,), 0xA5, dtype=torch.uint8, device=DEV)
    buf = torch.full((size + 512,), 0x5A, dtype=torch.uint8, device=DEV)
    buf[256:-256] = d["base"].view(torch.uint8).flatten()
    for _ in range(2):
        buf[256:-256] = d["base"].view(torch.uint8).flatten()
        _lib.launch("camhipLoraAdd", *args(buf.data_ptr() + 256), buf.data_ptr() + 256, workspace=ws[256:256 + need])
        torch.cuda.synchronize()
        assert (ws[:256] == 0xA5).all() and (ws[-256:] == 0xA5).all()
        assert (buf[:256] == 0x5A).all() and (buf[-256:] == 0x5A).all()
        assert torch.equal(buf[256:-256], want.view(torch.uint8).flatten())


def test_offsets_past_32_bits():
    """Outputs and rows past 4 GiB, adapters past 4 GiB."""
    M, N, K, L, R = 70000, 40000, 64, 2, 8
    g = torch.Generator(device=DEV).manual_seed(2)
    base = torch.zeros(M, N, device=DEV, dtype=torch.bfloat16)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    a = torch.randn(L, R, K, generator=g, device=DEV).bfloat16()
    b = torch.randn(L, N, R, generator=g, device=DEV).bfloat16()
    ids = torch.full((M,), -1, dtype=torch.int32, device=DEV)
    rows = torch.tensor([0, 1, 33333, 53688, 69998, 69999], device=DEV)
    ids[rows] = torch.tensor([0, 1, 0, 1, 1, 0], dtype=torch.int32, device=DEV)
    out = umdk_amd.lora_add(base, x, a, b, ids)
    part = dict(base=base[rows].contiguous(), x=x[rows].contiguous(), a=a, b=b, ids=ids[rows].contiguous(), scaling=None, xs=None)
    check(part, out[rows])
    assert int((out != 0).any(dim=1).sum()) == len(rows)


def test_adapters_past_4_gib():
    L, R, K, N = 40, 256, 131056, 16384
    g = torch.Generator(device=DEV).manual_seed(2)
    a = (torch.randn(L, R, K, generator=g, device=DEV) * K ** -0.5).bfloat16()
    assert a.numel() * 2 > 1 << 31
    b = torch.randn(L, N, R, generator=g, device=DEV).bfloat16()
    ids = torch.tensor([39, 0, 17, -1, 39], dtype=torch.int32, device=DEV)
    d = dict(base=torch.randn(5, N, generator=g, device=DEV).bfloat16(), x=torch.randn(5, K, generator=g, device=DEV).bfloat16(),
             a=a, b=b, ids=ids, scaling=None, xs=None)
    out = call(d)
    used = torch.tensor([0, 17, 39], device=DEV)
    small = dict(d, a=a[used].contiguous(), b=b[used].contiguous(), ids=torch.tensor([2, 0, 1, -1, 2], dtype=torch.int32, device=DEV))
    check(small, out)


def test_gradients_are_refused_not_dropped():
    d = make(4, 64, 32, 2, 8)
    for name in ("base", "x", "a", "b", "scaling"):
        with pytest.raises(RuntimeError, match="no backward"):
            call(d, **{name: d[name].detach().clone().requires_grad_()})
    with torch.no_grad():
        call(d, x=d["x"].detach().clone().requires_grad_())


@pytest.mark.parametrize("M,N,L,R,dtype,out", [
    (9000, 2568, 5, 32, "bf16", None), (9000, 2568, 5, 8, "fp16", None), (8200, 4160, 7, 64, "bf16", torch.float16),
    (8192, 4104, 3, 40, "fp16", torch.bfloat16), (3000, 4160, 4, 64, "fp16", None), (2900, 4232, 40, 32, "bf16", None),
    (8300, 2600, 6, 128, "bf16", None), (8195, 2632, 3, 200, "fp16", None), (4100, 4168, 1, 256, "bf16", None),
])
def test_prompts_by_whole_lines(M, N, L, R, dtype, out):
    """Aligned rows of 16 bits go by whole cache lines, others by a kernel that takes any: the same bits."""
    d = make(M, 144, N, L, R, dtype, seed=M + R, runs=R != 32)
    got = call(d, out)
    check(d, got)
    odd = torch.empty(M * N + 1, dtype=d["base"].dtype, device=DEV)[1:].view(M, N)
    odd.copy_(d["base"])
    assert torch.equal(call(d, out, base=odd), got)
    wide = torch.full((M, N + 24), float("nan"), dtype=d["base"].dtype, device=DEV)
    wide[:, 8:N + 8] = d["base"]
    assert torch.equal(call(d, out, base=wide[:, 8:N + 8]), got)


def test_prompts_in_place_of_the_base():
    from umdk_amd import _lib
    M, K, N, L, R = 8500, 64, 2696, 4, 16
    d = make(M, K, N, L, R, seed=12, runs=True)
    want = call(d)
    guard = torch.full((M + 2, N), 7.0, dtype=torch.bfloat16, device=DEV)
    guard[1:-1] = d["base"]
    args = (guard[1:-1].data_ptr(), d["x"].data_ptr(), None, d["a"].data_ptr(), d["b"].data_ptr(), d["ids"].data_ptr(),
            d["scaling"].data_ptr(), M, N, K, R, L, N, K, 0, 0, 0, 0, guard[1:-1].data_ptr())
    ws = torch.empty(_lib.workspace_size("camhipLoraAdd", *args), dtype=torch.uint8, device=DEV)
    _lib.launch("camhipLoraAdd", *args, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(guard[1:-1], want) and (guard[0] == 7).all() and (guard[-1] == 7).all()
