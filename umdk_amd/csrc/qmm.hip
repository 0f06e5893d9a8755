// G4: int8 matrix product with one scale per row of x and one per row of W (output channel):
//   out[m, n] = ((float)sum_k x[m, k] w[n, k]) * ws[n] * xs[m] + bias[n], rounded once to the output's type
// The sum is exact in int32 (K <= 131056: 2^14 K stays below 2^31), so neither the order of its parts nor a split of K
// changes a bit of the result.
#include "cam_device.h"
#include "launchers.h"

namespace cam {

namespace {

typedef _Float16 cam_f16x4 __attribute__((ext_vector_type(4)));

// four consecutive outputs of one row, the first `n` of them stored
template <int OUT> __device__ __forceinline__ void store4(void *out, size_t at, const float *v, int n)
{
    if constexpr (OUT == QMM_FP32) {
        float *o = reinterpret_cast<float *>(out) + at;
        if (n >= 4) {
            __builtin_memcpy(o, v, 16);
        } else {
            for (int q = 0; q < n; ++q)
                o[q] = v[q];
        }
    } else {
        u32x2 b;
        if constexpr (OUT == QMM_BF16)
            b = u32x2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
        else
            b = __builtin_bit_cast(u32x2, cam_f16x4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]});
        uint16_t *o = reinterpret_cast<uint16_t *>(out) + at;
        if (n >= 4) {
            __builtin_memcpy(o, &b, 8);
        } else {
#pragma unroll
            for (int q = 0; q < 3; ++q)
                if (q < n)
                    o[q] = (uint16_t)(b[q >> 1] >> (16 * (q & 1)));
        }
    }
}

// The simple form: a wave computes 32 x 32 outputs, its fragments read straight from memory (a lane of
// v_mfma_i32_16x16x64_i8 holds 16 consecutive bytes of one row).  Operands (W, x): a lane's four results are four
// consecutive columns of one row.
template <int OUT> __global__ __launch_bounds__(256) void qmm_direct_kernel(const QmmArgs p)
{
#pragma clang fp contract(off)
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4, w = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)blockIdx.y * 64 + (w & 1) * 32;
    const int64_t n0 = (int64_t)blockIdx.x * 64 + (w >> 1) * 32;
    const int8_t *xp[2], *wp[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        xp[i] = p.x + min(m0 + 16 * i + l16, p.M - 1) * (int64_t)p.K + lg * 16;
        wp[i] = p.w + min(n0 + 16 * i + l16, (int64_t)p.N - 1) * p.K + lg * 16;
    }
    i32x4 acc[2][2] = {};
    for (int k = 0; k < p.K; k += 64) {
        const bool in = k + lg * 16 < p.K;  // K % 16 == 0: a lane's 16 bytes are whole or none
        i32x4 a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[i] = in ? *reinterpret_cast<const i32x4 *>(xp[i] + k) : i32x4{0, 0, 0, 0};
            b[i] = in ? *reinterpret_cast<const i32x4 *>(wp[i] + k) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[j], a[i], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t m = m0 + 16 * i + l16;
        if (m >= p.M)
            continue;
        const float xs = p.xs[m];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t n = n0 + 16 * j + 4 * lg;
            const int left = (int)min((int64_t)4, (int64_t)p.N - n);
            if (left <= 0)
                continue;
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t c = min(n + q, (int64_t)p.N - 1);
                v[q] = (float)acc[i][j][q] * p.ws[c] * xs;
                if (p.bias)
                    v[q] += p.bias[c];
            }
            store4<OUT>(p.out, (size_t)(m * p.N + n), v, left);
        }
    }
}

}  // namespace

size_t qmm_workspace_bytes(int64_t M, int N, int K) { return 0; }

hipError_t launch_quant_matmul(const QmmArgs &a, void *ws, hipStream_t s)
{
    if (a.M == 0)
        return hipSuccess;
    if (a.N < 1 || a.K < 16 || a.K % 16 || a.M > 65535 * 64)
        return hipErrorInvalidValue;
    const dim3 grid((uint32_t)((a.N + 63) / 64), (uint32_t)((a.M + 63) / 64));
    if (a.out_dtype == QMM_BF16)
        hipLaunchKernelGGL(qmm_direct_kernel<QMM_BF16>, grid, dim3(256), 0, s, a);
    else if (a.out_dtype == QMM_FP16)
        hipLaunchKernelGGL(qmm_direct_kernel<QMM_FP16>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(qmm_direct_kernel<QMM_FP32>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace cam
