// Low-rank adapters of many requests beside a projection that they share:
//   out[t] = base[t] + scaling[a] * B_a (A_a x_t),  a = ids[t];  out[t] = base[t] where a is no adapter
// Products exact, sums fp32, one rounding at the end.
#include "cam_device.h"
#include "launchers.h"

namespace cam {

namespace {

__device__ __forceinline__ float half_value(uint32_t h, int dtype)
{
    return dtype == LORA_BF16 ? bf16_to_f32(h & 0xffffu) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
__device__ __forceinline__ float element(const void *p, int64_t at, int dtype)
{
    if (dtype == LORA_FP32)
        return reinterpret_cast<const float *>(p)[at];
    if (dtype == LORA_INT8)
        return (float)reinterpret_cast<const int8_t *>(p)[at];
    return half_value(reinterpret_cast<const uint16_t *>(p)[at], dtype);
}

// z[t, r] = scaling * xs[t] * A_a[r] . x_t, a wave each
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraArgs p, float *z)
{
    const int lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6);
    for (int64_t t = blockIdx.y; t < p.M; t += gridDim.y) {
        const int a = p.ids[t];
        if (a < 0 || a >= p.L || r >= p.R)
            continue;
        float sum = 0.0f;
        for (int k = lane; k < p.K; k += 64)
            sum = __builtin_fmaf(half_value(reinterpret_cast<const uint16_t *>(p.a)[((int64_t)a * p.R + r) * p.K + k], p.dtype),
                                 element(p.x, t * p.x_stride + k, p.x_dtype), sum);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            sum += __shfl_xor(sum, o, 64);
        if (lane == 0)
            z[t * p.R + r] = sum * (p.xs ? p.xs[t] : 1.0f) * (p.scaling ? p.scaling[a] : 1.0f);
    }
}

__global__ __launch_bounds__(256) void lora_expand_kernel(const LoraArgs p, const float *z)
{
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= p.N)
        return;
    for (int64_t t = blockIdx.y; t < p.M; t += gridDim.y) {
        const int a = p.ids[t];
        float sum = 0.0f;
        if (a >= 0 && a < p.L)
            for (int r = 0; r < p.R; ++r)
                sum = __builtin_fmaf(half_value(reinterpret_cast<const uint16_t *>(p.b)[((int64_t)a * p.N + n) * p.R + r], p.dtype),
                                     z[t * p.R + r], sum);
        const float v = element(p.base, t * p.base_stride + n, p.base_dtype) + sum;
        uint16_t *out = reinterpret_cast<uint16_t *>(p.out) + t * p.N + n;
        *out = p.out_dtype == LORA_BF16 ? (uint16_t)(f32x2_to_bf16x2(v, 0.0f) & 0xffffu)
                                        : __builtin_bit_cast(uint16_t, (_Float16)v);
    }
}

}  // namespace

size_t lora_workspace_bytes(const LoraArgs &a) { return (size_t)a.M * a.R * 4; }

hipError_t launch_lora_add(const LoraArgs &a, void *ws, hipStream_t s)
{
    if (a.M == 0)
        return hipSuccess;
    float *z = reinterpret_cast<float *>(ws);
    const int rows = (int)(a.M < 32768 ? a.M : 32768);
    hipLaunchKernelGGL(lora_shrink_kernel, dim3((a.R + 3) / 4, rows), dim3(256), 0, s, a, z);
    hipLaunchKernelGGL(lora_expand_kernel, dim3((a.N + 255) / 256, rows), dim3(256), 0, s, a, (const float *)z);
    return hipGetLastError();
}

}  // namespace cam
