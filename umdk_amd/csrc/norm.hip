// N1: residual addition, root-mean-square norm and the quantisation of its rows, in one pass.  Per row of H columns
//   v = x + residual (fp32);  residual_out = v in x's type
//   r = 1 / sqrt(mean(v^2) + eps);  y = v * r * w
// rows in x's type, in int8 with one scale per row, or in fp8 e4m3 with one scale per 128 columns:
//   int8: t = v * w, a = max |t|, code = rint(t * (127 / a)), scale = a / 127 * r
//   fp8:  per block of 128 columns code = e4m3(t * (448 / a)), scale = a / 448 * r
// r cancels out of the codes, so they hang on a sum, a product, a maximum and a division of fp32 and not on the order in
// which the squares are added up, and need not wait for that sum.  (a is taken as at least 2^-100: 127 / a stays finite,
// and a row of zeros gives codes 0 and scale 2^-100 / 127 * r.)  A row that holds an infinity or a NaN has NaN scales: a NaN
// is above all for a (an infinity under a weight of 0 is one), and other infinities meet r = 0.
//
// Bound by memory: x, the residual, its sum and the rows pass once, the row in registers from its load to its last store
// (T = 4096, H = 7168 with a residual, six sets of rows in turn: int8 36.9 us = 5.6 TB/s, fp8 39.8, bf16 41.6; three sets,
// part of which the last-level cache holds: fp8 37.6; T = 32768 bf16 305 us = 6.2 TB/s, where a large copy reaches 4.7; T = 1
// 3.9 us).  A block per row of 8 waves with 16 columns a thread (36.4 us int8 when this was chosen; 4 waves of 32 columns:
// 37.2, and 4.6 for one row; 16 waves of 8: 38.6 and 3.75); up to 1024 columns a wave per row.
//
// The norm reads v before it is rounded to 16 bits (the stored residual stream is the rounded one): one rounding per
// output.
#include "cam_device.h"
#include "launchers.h"

namespace cam {

namespace {

constexpr float NORM_TINY = 0x1p-100f;

// Global memory takes 16- and 8-byte accesses at any address: rows of odd strides and widths need no code of their own.
// Rows stream: read and written nontemporally (T = 4096, H = 7168: bf16 rows 48.6 -> 42.6 us, int8 43.7 -> 38.7, fp8 46.1
// -> 40.9; T = 32768 324 -> 311 us; the loads or the stores alone about half of that); the weight is cached.
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef u32x2 u32x2_u __attribute__((aligned(1)));
// the first n of 8 consecutive 16-bit elements, the others 0
template <bool STREAM> __device__ __forceinline__ u32x4 load8(const uint16_t *p, int n)
{
    if (n >= 8) {
        if constexpr (STREAM)
            return __builtin_nontemporal_load(reinterpret_cast<const u32x4_u *>(p));
        else
            return *reinterpret_cast<const u32x4_u *>(p);
    }
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n)
            v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return v;
}
__device__ __forceinline__ void store8(uint16_t *p, const u32x4 v, int n)
{
    if (n >= 8) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4_u *>(p));
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n)
            p[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
}
__device__ __forceinline__ void store8(uint8_t *p, const u32x2 v, int n)
{
    if (n >= 8) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x2_u *>(p));
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n)
            p[i] = (uint8_t)(v[i >> 2] >> (8 * (i & 3)));
}
template <bool FP16> __device__ __forceinline__ float unpack1(uint32_t h)
{
    return FP16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : bf16_to_f32(h);
}
template <bool FP16> __device__ __forceinline__ void unpack8(const u32x4 v, float *f)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = unpack1<FP16>(v[i] & 0xffffu);
        f[2 * i + 1] = unpack1<FP16>(v[i] >> 16);
    }
}
typedef _Float16 cam_f16x2 __attribute__((ext_vector_type(2)));
template <bool FP16> __device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (FP16)
        return __builtin_bit_cast(uint32_t, cam_f16x2{(_Float16)a, (_Float16)b});
    else
        return f32x2_to_bf16x2(a, b);
}
template <bool FP16> __device__ __forceinline__ u32x4 pack8(const float *f)
{
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = pack2<FP16>(f[2 * i], f[2 * i + 1]);
    return r;
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v += __shfl_xor(v, o, 64);
    return v;
}

// the larger one, NaN if either is
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
template <int WIDTH> __device__ __forceinline__ float nan_group_max(float v)
{
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1)
        v = nan_max(v, __shfl_xor(v, o, 64));
    return v;
}

__device__ __forceinline__ uint32_t int8x4(const float *t, float inv)
{
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r |= ((uint32_t)(int)__builtin_rintf(t[i] * inv) & 0xffu) << (8 * i);
    return r;
}

// One row per ROW_WAVES waves, ROWS rows per block; a thread holds NIT pieces of 8 columns, 8 ROW_THREADS apart.
template <bool FP16, int QUANT, int NIT, int ROW_WAVES, int ROWS>
__global__ __launch_bounds__(64 * ROW_WAVES *ROWS) void add_rms_norm_kernel(const NormArgs p)
{
#pragma clang fp contract(off)
    constexpr int RT = 64 * ROW_WAVES;
    static_assert(ROWS == 1 || ROW_WAVES == 1, "a block holds one row, or a row per wave");
    const int64_t row = p.row0 + (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? (int)(threadIdx.x >> 6) : 0);
    if (ROWS > 1 && row >= p.T)
        return;
    const int tid = ROWS > 1 ? threadIdx.x & 63 : threadIdx.x;
    const uint16_t *x = p.x + row * p.x_stride;
    const uint16_t *res = p.residual ? p.residual + row * p.H : nullptr;

    u32x4 xv[NIT], rv[NIT];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
        const int col = (i * RT + tid) * 8;
        xv[i] = load8<true>(x + col, p.H - col);
    }
    if (res) {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
            const int col = (i * RT + tid) * 8;
            rv[i] = load8<true>(res + col, p.H - col);
        }
    }
    // (the weight before the first store, which the compiler has to think it may overlap: int8 38.7 -> 36.4 us)
    u32x4 wv[NIT][2];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
        const int col = (i * RT + tid) * 8;
        if (p.weight_fp32) {
            const uint32_t *wp = reinterpret_cast<const uint32_t *>(p.weight) + col;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                wv[i][j >> 2][j & 3] = col + j < p.H ? wp[j] : 0;
        } else {
            wv[i][0] = load8<false>(reinterpret_cast<const uint16_t *>(p.weight) + col, p.H - col);
        }
    }
    float t[NIT][8];
    float ss = 0.0f, am = 0.0f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
        const int col = (i * RT + tid) * 8, n = p.H - col;
        unpack8<FP16>(xv[i], t[i]);
        if (res) {
            float r[8];
            unpack8<FP16>(rv[i], r);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                t[i][j] += r[j];
            store8(p.residual_out + row * p.H + col, pack8<FP16>(t[i]), n);
        }
        float s8 = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            s8 += t[i][j] * t[i][j];
        ss += s8;
        float w[8];
        if (p.weight_fp32) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = __uint_as_float(wv[i][j >> 2][j & 3]);
        } else {
            unpack8<FP16>(wv[i][0], w);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            t[i][j] *= w[j];
        if constexpr (QUANT == QUANT_INT8_TOKEN) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                am = nan_max(am, fabsf(t[i][j]));
        }
    }
    ss = wave_sum(ss);
    if constexpr (QUANT == QUANT_INT8_TOKEN)
        am = nan_group_max<64>(am);
    if constexpr (ROW_WAVES > 1) {
        __shared__ float red[2][ROW_WAVES];
        if ((tid & 63) == 0) {
            red[0][tid >> 6] = ss;
            red[1][tid >> 6] = am;
        }
        __syncthreads();
        ss = 0.0f;
        am = 0.0f;
#pragma unroll
        for (int w = 0; w < ROW_WAVES; ++w) {
            ss += red[0][w];
            am = nan_max(am, red[1][w]);
        }
    }
    const float rms = 1.0f / __builtin_sqrtf(ss / (float)p.H + p.eps);

    if constexpr (QUANT == QUANT_NONE) {
        uint16_t *y = reinterpret_cast<uint16_t *>(p.y) + row * p.H;
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
            const int col = (i * RT + tid) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                t[i][j] *= rms;
            store8(y + col, pack8<FP16>(t[i]), p.H - col);
        }
    } else if constexpr (QUANT == QUANT_INT8_TOKEN) {
        uint8_t *y = reinterpret_cast<uint8_t *>(p.y) + row * p.H;
        const float a = nan_max(am, NORM_TINY), inv = 127.0f / a;
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
            const int col = (i * RT + tid) * 8;
            store8(y + col, u32x2{int8x4(t[i], inv), int8x4(t[i] + 4, inv)}, p.H - col);
        }
        if (tid == 0)
            p.scales[row] = a / 127.0f * rms;
    } else {
        uint8_t *y = reinterpret_cast<uint8_t *>(p.y) + row * p.H;
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
            const int col = (i * RT + tid) * 8;  // H % 128 == 0: 16 lanes hold a block, whole or not at all
            float a = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                a = nan_max(a, fabsf(t[i][j]));
            a = nan_max(nan_group_max<16>(a), NORM_TINY);
            const float inv = 448.0f / a;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                t[i][j] *= inv;
            store8(y + col, u32x2{f32x4_to_e4m3(t[i][0], t[i][1], t[i][2], t[i][3]),
                                  f32x4_to_e4m3(t[i][4], t[i][5], t[i][6], t[i][7])}, p.H - col);
            if (col < p.H && (tid & 15) == 0)
                p.scales[(int64_t)(col / 128) * p.T + row] = a / 448.0f * rms;
        }
    }
}

template <bool FP16, int QUANT> hipError_t launch_quant(NormArgs a, hipStream_t s)
{
    // (a launch takes fewer than 2^32 threads: more rows go in several)
#define NORM_CASE(NIT, RW, ROWS)                                                                                    \
    if (a.H <= NIT * 512 * RW) {                                                                                    \
        constexpr int THREADS = 64 * RW * ROWS;                                                                     \
        constexpr int64_t MOST = ((int64_t)1 << 31) / THREADS * ROWS;                                               \
        for (; a.row0 < a.T; a.row0 += MOST) {                                                                      \
            const int64_t rows = a.T - a.row0 < MOST ? a.T - a.row0 : MOST;                                         \
            hipLaunchKernelGGL((add_rms_norm_kernel<FP16, QUANT, NIT, RW, ROWS>),                                   \
                               dim3((uint32_t)((rows + ROWS - 1) / ROWS)), dim3(THREADS), 0, s, a);                 \
            const hipError_t e = hipGetLastError();                                                                 \
            if (e != hipSuccess)                                                                                    \
                return e;                                                                                           \
        }                                                                                                           \
        return hipSuccess;                                                                                          \
    }
    NORM_CASE(1, 1, 4)
    NORM_CASE(2, 1, 4)
    NORM_CASE(1, 4, 1)
    NORM_CASE(2, 4, 1)
    NORM_CASE(2, 8, 1)
    NORM_CASE(2, 16, 1)
    NORM_CASE(4, 16, 1)
#undef NORM_CASE
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_add_rms_norm(const NormArgs &a, hipStream_t s)
{
    if (a.T == 0)
        return hipSuccess;
    if (a.H < 1 || a.T < 0 || a.T > 0x7fffffff || (a.quant == QUANT_FP8_BLOCK && a.H % 128))
        return hipErrorInvalidValue;
    if (a.quant == QUANT_NONE)
        return a.fp16 ? launch_quant<true, QUANT_NONE>(a, s) : launch_quant<false, QUANT_NONE>(a, s);
    if (a.quant == QUANT_INT8_TOKEN)
        return a.fp16 ? launch_quant<true, QUANT_INT8_TOKEN>(a, s) : launch_quant<false, QUANT_INT8_TOKEN>(a, s);
    if (a.quant == QUANT_FP8_BLOCK)
        return a.fp16 ? launch_quant<true, QUANT_FP8_BLOCK>(a, s) : launch_quant<false, QUANT_FP8_BLOCK>(a, s);
    return hipErrorInvalidValue;
}

}  // namespace cam
