// R1: routing over groups of experts.  With l the logits of a token, b the experts' balance bias:
//   s = sigmoid(l) or softmax(l);  c = s + b
//   a group's score: the sum of its two largest c, or its largest; the KG best groups are kept
//   the picks: the K largest c within the kept groups, in that order; equal ones go to the lower id
//   gates: s at the picks (without b), over their sum if renormalised, times a factor
// An expert whose logit or bias is -inf (or NaN) is never picked; slots left without one hold id -1 and gate 0,
// which the layout, the dispatch and the fused op skip.
//
// Which of two experts comes first may hang on the last bits of their scores, so c is computed in 64 bits (the
// vector unit runs 64-bit FMAs at the rate of single 32-bit ones) and its order does not depend on how an fp32
// exponential rounds.  The low 9 mantissa bits of c then hold the expert's id, so that one v_max_f64 reduction gives
// both the score and the id, with ties to the lower id; scores nearer than 2^-43 of their size count as equal.  Without
// a bias s orders as l does, and the keys are the logits themselves (exact: a float leaves 29 bits of a double free):
// no exponential then, but for the picks and the denominator.
//
// A token is handled by LANES (16 or 64) adjacent lanes, each holding PER consecutive experts of one group; a group
// has LANES / (number of groups, rounded up to a power of two) lanes.  So the best two of a group are found by a scan of
// the lane's own experts and log2 of those lanes' steps, all groups at once.
#include "cam_device.h"
#include "launchers.h"

namespace cam {

namespace {

constexpr int RG_WAVES = 4;
constexpr uint32_t RG_NONE_HI = 0xFFEFFFFFu;  // high word of -1.797e308: no expert, no group
constexpr double RG_NONE_MAX = -1.7e308;      // keys at or below it are none

// DPP moves within a row of 16 lanes: quad xor 1, quad xor 2, half-row mirror, row mirror.  In a reduction the mirrors act
// as xor 4 and xor 8, as the lanes that they pair hold their quad's (half row's) result already.
template <int CTRL> __device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int STEP> __device__ __forceinline__ double lane_step(double v)
{
    if constexpr (STEP == 1)
        return dpp_f64<0xB1>(v);
    else if constexpr (STEP == 2)
        return dpp_f64<0x4E>(v);
    else if constexpr (STEP == 4)
        return dpp_f64<0x141>(v);
    else if constexpr (STEP == 8)
        return dpp_f64<0x140>(v);
    else
        return __shfl_xor(v, STEP, 64);
}
template <int LANES> __device__ __forceinline__ double row_max(double v)
{
    v = fmax(v, lane_step<1>(v));
    v = fmax(v, lane_step<2>(v));
    v = fmax(v, lane_step<4>(v));
    v = fmax(v, lane_step<8>(v));
    if constexpr (LANES == 64) {
        v = fmax(v, lane_step<16>(v));
        v = fmax(v, lane_step<32>(v));
    }
    return v;
}
template <int LANES> __device__ __forceinline__ double row_sum(double v)
{
    v += lane_step<1>(v);
    v += lane_step<2>(v);
    v += lane_step<4>(v);
    v += lane_step<8>(v);
    if constexpr (LANES == 64) {
        v += lane_step<16>(v);
        v += lane_step<32>(v);
    }
    return v;
}
// the two largest of the sets behind two lanes
template <int STEP> __device__ __forceinline__ void top2_step(double &m1, double &m2)
{
    const double o1 = lane_step<STEP>(m1), o2 = lane_step<STEP>(m2);
    m2 = fmax(fmin(m1, o1), fmax(m2, o2));
    m1 = fmax(m1, o1);
}

// exp(x) in 64 bits for x in [-745, 700]: x = n ln 2 + r, |r| <= ln 2 / 2, and the polynomial of degree 9 that meets
// exp(r) in the ten Chebyshev nodes of that interval: within 1.9e-14 of it, below the 2^-43 that count as equal.  The
// coefficients sit in scalar registers (as literals each costs two moves to the FMA that uses it).
struct Exp64 {
    double c[10], log2e, ln2_hi, ln2_lo;
    __device__ __forceinline__ Exp64()
        : c{0x1.000000000003dp+0,  0x1.0000000000006p+0,  0x1.ffffffffe74f0p-2,  0x1.5555555550d87p-3,  0x1.55555588b8538p-5,
            0x1.11111123bf1c5p-7, 0x1.6c162bb7b3ef5p-10, 0x1.a01994c82e1c6p-13, 0x1.a17df105a3981p-16, 0x1.72e107e8d8eb6p-19},
          log2e(0x1.71547652b82fep+0), ln2_hi(-0x1.62e42fefa39efp-1), ln2_lo(-0x1.abc9e3b39803fp-56)
    {
#pragma unroll
        for (int i = 0; i < 10; ++i)
            asm("" : "+s"(c[i]));
        asm("" : "+s"(log2e));
        asm("" : "+s"(ln2_hi));
        asm("" : "+s"(ln2_lo));
    }
    __device__ __forceinline__ double operator()(double x) const
    {
        const double n = __builtin_rint(x * log2e);
        double r = __builtin_fma(n, ln2_hi, x);
        r = __builtin_fma(n, ln2_lo, r);
        double p = __builtin_fma(c[9], r, c[8]);
#pragma unroll
        for (int i = 7; i >= 0; --i)
            p = __builtin_fma(p, r, c[i]);
        return __builtin_ldexp(p, (int)n);
    }
};
// 1 / d for d in [1, 1e304]: the hardware's estimate (of single precision) and one step of third order
__device__ __forceinline__ double recip64(double d)
{
    const double y = __builtin_amdgcn_rcp(d), e = __builtin_fma(-d, y, 1.0);
    return __builtin_fma(y, __builtin_fma(e, e, e), y);
}
// (exp of less than -745 would be 0: nothing beside 1; a NaN gives some number, its expert is not eligible)
__device__ __forceinline__ double sigmoid64(const Exp64 &exp64, float l)
{
    return recip64(1.0 + exp64((double)fmaxf(fminf(-l, 700.0f), -745.0f)));
}
// exp(l - mx), 0 for an expert that has no logit (-inf or NaN)
__device__ __forceinline__ double exp_rel(const Exp64 &exp64, float l, float mx)
{
    const double e = exp64(fmin(fmax((double)l - (double)mx, -745.0), 0.0));
    return l > -INFINITY ? e : 0.0;
}

// c with `id` in its low BITS bits, the lower id the larger of two equal c
template <int BITS> __device__ __forceinline__ double tag(double c, int id)
{
    constexpr uint32_t M = (1u << BITS) - 1;
    const uint64_t u = __builtin_bit_cast(uint64_t, fmin(c, 0x1p1023));  // (an infinity would turn into a NaN)
    const uint32_t hi = (uint32_t)(u >> 32), low = (M ^ (uint32_t)id) ^ (uint32_t)((int32_t)hi >> 31);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | (((uint32_t)u & ~M) | (low & M)));
}
template <int BITS> __device__ __forceinline__ int untag(double key)
{
    constexpr uint32_t M = (1u << BITS) - 1;
    const uint64_t u = __builtin_bit_cast(uint64_t, key);
    return (int)(((uint32_t)u ^ M ^ (uint32_t)((int64_t)u >> 63)) & M);
}
// a key (a group) that is out: the value below RG_NONE_MAX, whatever its low word
__device__ __forceinline__ double none_if(bool out, double key)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, key);
    return __builtin_bit_cast(double, (uint64_t)(out ? RG_NONE_HI : (uint32_t)(u >> 32)) << 32 | (uint32_t)u);
}
__device__ __forceinline__ double none() { return __builtin_bit_cast(double, (uint64_t)RG_NONE_HI << 32); }
// whether two tagged keys are the same expert's (group's): their low words hold its id
__device__ __forceinline__ bool same_id(double a, double b)
{
    return (uint32_t)__builtin_bit_cast(uint64_t, a) == (uint32_t)__builtin_bit_cast(uint64_t, b);
}

__device__ __forceinline__ float half_to_f32(uint32_t h, bool bf16)
{
    return bf16 ? bf16_to_f32(h & 0xffffu) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
__device__ __forceinline__ float logit(const char *row, int dtype, int e)
{
    if (dtype == ROUTE_FP32)
        return reinterpret_cast<const float *>(row)[e];
    return half_to_f32(reinterpret_cast<const uint16_t *>(row)[e], dtype == ROUTE_BF16);
}
// the logits e0 ... e0 + PER - 1 of a row (past the last expert the last one again)
template <int PER> __device__ __forceinline__ void load_logits(const char *row, const RouteGroupedArgs &p, int e0, float *lg)
{
    if (PER % 4 == 0 && p.vec) {
        if (p.dtype == ROUTE_FP32) {
#pragma unroll
            for (int j = 0; j < PER / 4; ++j) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(row + (e0 + 4 * j) * 4);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    lg[4 * j + q] = v[q];
            }
            return;
        }
        u32x2 v[PER / 4 ? PER / 4 : 1];
#pragma unroll
        for (int j = 0; j < PER / 4; ++j)
            v[j] = *reinterpret_cast<const u32x2 *>(row + (e0 + 4 * j) * 2);
        const bool bf16 = p.dtype == ROUTE_BF16;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            lg[j] = half_to_f32(v[j / 4][(j >> 1) & 1] >> (16 * (j & 1)), bf16);
    } else if (p.dtype == ROUTE_FP32) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            lg[j] = reinterpret_cast<const float *>(row)[min(e0 + j, p.E - 1)];
    } else {
        uint32_t h[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j)
            h[j] = reinterpret_cast<const uint16_t *>(row)[min(e0 + j, p.E - 1)];
        const bool bf16 = p.dtype == ROUTE_BF16;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            lg[j] = half_to_f32(h[j], bf16);
    }
}

template <int LANES, int PER>
__global__ __launch_bounds__(RG_WAVES * 64) void route_grouped_kernel(const RouteGroupedArgs p)
{
    constexpr int TPW = 64 / LANES;  // tokens per wave
    const int lane = threadIdx.x & 63, rl = lane & (LANES - 1);
    const int t = ((int)blockIdx.x * RG_WAVES + (int)(threadIdx.x >> 6)) * TPW + lane / LANES;
    const bool live = t < p.T;  // dead rows run along (they read row 0)
    const char *row = reinterpret_cast<const char *>(p.logits) + (size_t)(live ? t : 0) * (size_t)p.row_bytes;
    // (lanes past the last group look at expert 0's, so that their loads stay inside the row, and hold none)
    const int g = rl / p.lpg, pos0 = (rl % p.lpg) * PER, e0 = g < p.G ? g * p.gs + pos0 : 0;
    const int have = g < p.G ? min(max(p.gs - pos0, 0), PER) : 0;

    float lg[PER], bs[PER];
    load_logits<PER>(row, p, e0, lg);
    if (p.bias) {
        if (PER % 4 == 0 && p.vec) {
#pragma unroll
            for (int j = 0; j < PER / 4; ++j) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(p.bias + e0 + 4 * j);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    bs[4 * j + q] = v[q];
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                bs[j] = p.bias[min(e0 + j, p.E - 1)];
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            bs[j] = 0.0f;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        lg[j] = j < have ? lg[j] : -INFINITY;
        mx = fmaxf(mx, lg[j]);
    }
    const Exp64 exp64;
    const bool softmax = p.score == ROUTE_SOFTMAX;
    const bool by_logit = p.by_logit != 0;
    double denom = 0.0;
    if (softmax)
        mx = (float)row_max<LANES>((double)mx);

    double key[PER];
    if (by_logit) {
        if (softmax && !p.renorm) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                denom += exp_rel(exp64, lg[j], mx);
            denom = row_sum<LANES>(denom);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j)  // (+ 0: the zeros of both signs are equal)
            key[j] = none_if(!(lg[j] > -INFINITY), tag<9>((double)lg[j] + 0.0, e0 + j));
    } else {
        if (softmax) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                key[j] = exp_rel(exp64, lg[j], mx);
                denom += key[j];
            }
            denom = row_sum<LANES>(denom);
            const double inv = recip64(denom);
#pragma unroll
            for (int j = 0; j < PER; ++j)
                key[j] *= inv;
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                key[j] = sigmoid64(exp64, lg[j]);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const double c = key[j] + (double)bs[j];
            key[j] = none_if(!(lg[j] > -INFINITY) | !(bs[j] > -INFINITY), tag<9>(c, e0 + j));
        }
    }

    if (p.KG < p.G) {
        double m1 = key[0], m2 = none();
#pragma unroll
        for (int j = 1; j < PER; ++j) {
            m2 = fmax(m2, fmin(m1, key[j]));
            m1 = fmax(m1, key[j]);
        }
        if (p.lpg > 1)
            top2_step<1>(m1, m2);
        if (p.lpg > 2)
            top2_step<2>(m1, m2);
        if (p.lpg > 4)
            top2_step<4>(m1, m2);
        if (p.lpg > 8)
            top2_step<8>(m1, m2);
        if constexpr (LANES == 64) {
            if (p.lpg > 16)
                top2_step<16>(m1, m2);
        }
        // (the ids in the low bits change a score by 2^-43 of itself at most)
        const double two = p.group_top2 && m2 > RG_NONE_MAX ? m1 + m2 : m1;
        double gk = none_if(!(m1 > RG_NONE_MAX), tag<6>(two, g));
        bool kept = false;
        for (int i = 0; i < p.KG; ++i) {
            const double win = row_max<LANES>(gk);
            const bool mine = same_id(gk, win) && win > RG_NONE_MAX;
            kept |= mine;
            gk = none_if(mine, gk);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j)
            key[j] = none_if(!kept, key[j]);
    }

    int my_idx = -1;
#pragma unroll 1
    for (int k = 0; k < p.K; ++k) {
        double best = key[0];
#pragma unroll
        for (int j = 1; j < PER; ++j)
            best = fmax(best, key[j]);
        best = row_max<LANES>(best);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            key[j] = none_if(same_id(key[j], best), key[j]);
        if (rl == k)
            my_idx = best > RG_NONE_MAX ? untag<9>(best) : -1;
    }

    double gate = 0.0;
    if (my_idx >= 0) {
        const float l = logit(row, p.dtype, my_idx);
        if (!softmax) {
            gate = sigmoid64(exp64, l);
        } else {
            gate = exp_rel(exp64, l, mx);
            if (denom > 0.0)
                gate *= recip64(denom);
        }
    }
    if (p.renorm)
        gate = gate / (row_sum<LANES>(gate) + 1e-20);
    if (live && rl < p.K) {
        p.topk_idx[(size_t)t * p.K + rl] = my_idx;
        p.topk_w[(size_t)t * p.K + rl] = (float)(gate * (double)p.scaling);
        if (p.topk_idx64)
            p.topk_idx64[(size_t)t * p.K + rl] = my_idx;
    }
}

int pow2_at_least(int v)
{
    int r = 1;
    while (r < v)
        r *= 2;
    return r;
}

}  // namespace

hipError_t launch_route_grouped(RouteGroupedArgs a, hipStream_t s)
{
    if (a.T == 0)
        return hipSuccess;
    if (a.E < 1 || a.E > 512 || a.K < 1 || a.K > 16 || a.G < 1 || a.G > 64 || a.E % a.G || a.KG < 1 || a.KG > a.G)
        return hipErrorInvalidValue;
    const int g2 = pow2_at_least(a.G);
    a.gs = a.E / a.G;
    // without a bias the scores order as the logits do, and so do the groups by their largest one
    a.by_logit = !a.bias && (a.KG == a.G || !a.group_top2);
    int lanes = 64;
    if (g2 <= 16 && (a.gs + 16 / g2 - 1) / (16 / g2) <= 32 && a.T > 4096)
        lanes = 16;
    a.lpg = lanes / g2;
    const int per = (a.gs + a.lpg - 1) / a.lpg;
    const uintptr_t bases = (uintptr_t)a.logits | (uintptr_t)a.bias | (uintptr_t)a.row_bytes;
    const int tokens = RG_WAVES * (64 / lanes);
    const dim3 grid((a.T + tokens - 1) / tokens), block(RG_WAVES * 64);
#define RG_CASE(L, P)                                                                                               \
    if (lanes == L && per <= P) {                                                                                   \
        a.vec = P % 4 == 0 && a.gs == a.lpg * P && bases % 16 == 0; /* every lane's experts in whole vectors */      \
        hipLaunchKernelGGL((route_grouped_kernel<L, P>), grid, block, 0, s, a);                                     \
        return hipGetLastError();                                                                                   \
    }
    RG_CASE(64, 1)
    RG_CASE(64, 2)
    RG_CASE(64, 4)
    RG_CASE(64, 8)
    RG_CASE(64, 16)
    RG_CASE(16, 1)
    RG_CASE(16, 2)
    RG_CASE(16, 4)
    RG_CASE(16, 8)
    RG_CASE(16, 10)
    RG_CASE(16, 12)
    RG_CASE(16, 16)
    RG_CASE(16, 24)
    RG_CASE(16, 32)
#undef RG_CASE
    return hipErrorInvalidValue;
}

}  // namespace cam
