// A whole expert layer for 1 to 16 tokens.  With x the tokens' rows, R the router, b the balance bias:
//   l = x R^T;  ids, gates = grouped routing of l (route_grouped.hip)
//   E_e(x) = W2_e (silu(g) * u),  (g, u) = halves of W1_e x
//   out[t] = sum_k gates[t, k] E_ids[t, k](x_t) + E_shared(x_t)
// Products of the weights' exact values, fp32 sums, one rounding at the end.
#include "cam_device.h"
#include "launchers.h"

namespace cam {

namespace {

// ---------------------------------------------------------------- the router product
// Logits in 64 bits, rounded to fp32: which expert is picked must not hang on the order of a sum.  A block per expert, its
// waves take turns at runs of 512 columns; products of 16-bit values (and of those with fp32) are exact in 64 bits.
constexpr int MD_ROUTER_WAVES = 4;

__global__ __launch_bounds__(MD_ROUTER_WAVES * 64) void moe_decode_router_kernel(const MoeDecodeArgs p, float *logits)
{
    const int e = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __shared__ double part[MD_ROUTER_WAVES][MD_MAX_TOKENS];
    for (int t = 0; t < p.T; ++t) {
        double sum = 0.0;
        for (int k = (w * 64 + lane) * 8; k < p.H; k += MD_ROUTER_WAVES * 512) {
            float xf[8], rf[8];
            unpack_bf16x8(*reinterpret_cast<const u32x4 *>(p.x + (size_t)t * p.H + k), xf);
            if (p.router_fp32) {
                const float *r = reinterpret_cast<const float *>(p.router) + (size_t)e * p.H + k;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    rf[j] = r[j];
            } else {
                unpack_bf16x8(*reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(p.router) + (size_t)e * p.H + k), rf);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                sum = __builtin_fma((double)xf[j], (double)rf[j], sum);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            sum += __shfl_xor(sum, o, 64);
        if (lane == 0)
            part[w][t] = sum;
    }
    __syncthreads();
    if (threadIdx.x < p.T) {
        double sum = 0.0;
        for (int v = 0; v < MD_ROUTER_WAVES; ++v)
            sum += part[v][threadIdx.x];
        const bool on = !p.active || p.active[threadIdx.x];
        logits[(size_t)threadIdx.x * p.E + e] = on ? (float)sum : __builtin_nanf("");
    }
}

// ---------------------------------------------------------------- the experts, one output at a time
template <int WT> __device__ __forceinline__ float weight(const void *w, size_t at)
{
    if constexpr (WT == MD_BF16)
        return bf16_to_f32(reinterpret_cast<const uint16_t *>(w)[at]);
    else if constexpr (WT == MD_INT8)
        return (float)reinterpret_cast<const int8_t *>(w)[at];
    else
        return __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t *>(w)[at], 0);
}
// row n of a matrix of rows of k: the dot product with v, in this wave
template <int WT, typename V>
__device__ __forceinline__ float row_dot(const void *w, const float *s, size_t n, int k, int blocks_k, V v)
{
    const int lane = threadIdx.x & 63;
    float sum = 0.0f;
    for (int j = lane; j < k; j += 64) {
        float q = weight<WT>(w, n * k + j);
        if constexpr (WT == MD_FP8)
            q *= s[n / 128 * blocks_k + j / 128];
        sum = __builtin_fmaf(q, v(j), sum);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o, 64);
    if constexpr (WT == MD_INT8)
        sum *= s[n];
    return sum;
}

template <int WT> __global__ __launch_bounds__(256) void moe_decode_gmm1_kernel(const MoeDecodeArgs p, float *h, int width)
{
    const int slots = p.K + (p.Is > 0), t = blockIdx.y / slots, k = blockIdx.y % slots;
    const bool shared = k == p.K;
    const int I = shared ? p.Is : p.I, i = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int e = shared ? 0 : p.topk_idx[t * p.K + k];
    if (i >= I || e < 0)
        return;
    const size_t per = (size_t)2 * I * p.H * (WT == MD_BF16 ? 2 : 1);
    const size_t per_s = WT == MD_INT8 ? 2 * I : (size_t)(2 * I / 128) * (p.H / 128);
    const void *w = shared ? p.sw1 : (const char *)p.w1 + e * per;
    const float *s = WT == MD_BF16 ? nullptr : shared ? p.ss1 : p.s1 + e * per_s;
    const auto x = [&](int j) { return bf16_to_f32(p.x[(size_t)t * p.H + j]); };
    const float g = row_dot<WT>(w, s, i, p.H, p.H / 128, x), u = row_dot<WT>(w, s, I + i, p.H, p.H / 128, x);
    if ((threadIdx.x & 63) == 0)
        h[(size_t)blockIdx.y * width + i] = g / (1.0f + __expf(-g)) * u;
}

template <int WT> __global__ __launch_bounds__(256) void moe_decode_gmm2_kernel(const MoeDecodeArgs p, const float *h, int width)
{
    const int slots = p.K + (p.Is > 0), t = blockIdx.y, n = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= p.H)
        return;
    float sum = 0.0f;
    for (int k = 0; k < slots; ++k) {
        const bool shared = k == p.K;
        const int I = shared ? p.Is : p.I, e = shared ? 0 : p.topk_idx[t * p.K + k];
        if (e < 0 || (shared && p.active && !p.active[t]))
            continue;
        const size_t per = (size_t)I * p.H * (WT == MD_BF16 ? 2 : 1);
        const size_t per_s = WT == MD_INT8 ? p.H : (size_t)(I / 128) * (p.H / 128);
        const void *w = shared ? p.sw2 : (const char *)p.w2 + e * per;
        const float *s = WT == MD_BF16 ? nullptr : shared ? p.ss2 : p.s2 + e * per_s;
        const float *row = h + (size_t)(t * slots + k) * width;
        const float y = row_dot<WT>(w, s, n, I, I / 128, [&](int j) { return row[j]; });
        sum = shared ? sum + y : __builtin_fmaf(p.topk_w[t * p.K + k], y, sum);
    }
    if ((threadIdx.x & 63) == 0)
        p.out[(size_t)t * p.H + n] = (uint16_t)(f32x2_to_bf16x2(sum, 0.0f) & 0xffffu);
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

template <int WT> hipError_t run(const MoeDecodeArgs &a, float *h, int width, hipStream_t s)
{
    const int slots = a.K + (a.Is > 0);
    hipLaunchKernelGGL(moe_decode_gmm1_kernel<WT>, dim3((width + 3) / 4, a.T * slots), dim3(256), 0, s, a, h, width);
    hipLaunchKernelGGL(moe_decode_gmm2_kernel<WT>, dim3((a.H + 3) / 4, a.T), dim3(256), 0, s, a, (const float *)h, width);
    return hipGetLastError();
}

}  // namespace

size_t moe_decode_workspace_bytes(const MoeDecodeArgs &a)
{
    const size_t width = a.I > a.Is ? a.I : a.Is;
    return align256((size_t)a.T * a.E * 4) + align256((size_t)a.T * (a.K + 1) * width * 4);
}

hipError_t launch_moe_decode(const MoeDecodeArgs &a, void *ws, hipStream_t s)
{
    if (a.T == 0)
        return hipSuccess;
    float *logits = reinterpret_cast<float *>(ws);
    float *h = reinterpret_cast<float *>((char *)ws + align256((size_t)a.T * a.E * 4));
    hipLaunchKernelGGL(moe_decode_router_kernel, dim3(a.E), dim3(MD_ROUTER_WAVES * 64), 0, s, a, logits);
    RouteGroupedArgs r{};
    r.logits = logits;
    r.row_bytes = (int64_t)a.E * 4;
    r.bias = a.bias;
    r.T = a.T;
    r.E = a.E;
    r.K = a.K;
    r.G = a.G;
    r.KG = a.KG;
    r.score = a.score;
    r.group_top2 = a.group_top2;
    r.renorm = a.renorm;
    r.dtype = ROUTE_FP32;
    r.scaling = a.scaling;
    r.topk_idx = a.topk_idx;
    r.topk_w = a.topk_w;
    hipError_t e = launch_route_grouped(r, s);
    if (e != hipSuccess)
        return e;
    const int width = a.I > a.Is ? a.I : a.Is;
    switch (a.wtype) {
    case MD_BF16:
        return run<MD_BF16>(a, h, width, s);
    case MD_INT8:
        return run<MD_INT8>(a, h, width, s);
    case MD_FP8:
        return run<MD_FP8>(a, h, width, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace cam
