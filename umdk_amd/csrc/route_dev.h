#pragma once
// Routing of one token over groups of experts, by some lanes of a wave: shared by route_grouped.hip, where the mathematics
// and the choices are explained, and moe_decode.hip.
#include "cam_device.h"
#include "launchers.h"

namespace cam {

namespace {

constexpr uint32_t RG_NONE_HI = 0xFFEFFFFFu;  // high word of -1.797e308: no expert, no group
constexpr double RG_NONE_MAX = -1.7e308;      // keys at or below it are none

// Larger and smaller of two keys.  (Keys are never NaN; the compiler cannot know, and puts a v_max of every operand with
// itself in front of a fmax of numbers that come out of bit operations: half of all instructions here.)
__device__ __forceinline__ double kmax(double a, double b)
{
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double kmin(double a, double b)
{
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
// A value on its way to other lanes: those moves need wait states behind the instruction that wrote it, which the
// compiler does not count for the two above.
__device__ __forceinline__ double settled(double v)
{
    asm("s_nop 3" : "+v"(v));
    return v;
}

// The values of this lane and of the lane STEP (1, 2, 4, ... 32) away, in an order that both share: what a reduction that
// does not mind the order needs.  Within a row of 16 lanes DPP moves: quad xor 1, quad xor 2, half-row mirror, row mirror
// (the mirrors act as xor 4 and 8, as the lanes that they pair hold their quad's or half row's result already); between
// rows the swaps of gfx950.
struct Pair {
    double a, b;
};
template <int CTRL> __device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int STEP> __device__ __forceinline__ Pair both(double v)
{
    if constexpr (STEP <= 8) {
        return {v, dpp_f64<STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140>(v)};
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t l = (uint32_t)u, h = (uint32_t)(u >> 32);
        if constexpr (STEP == 16) {
            const auto lo = __builtin_amdgcn_permlane16_swap(l, l, false, false);
            const auto hi = __builtin_amdgcn_permlane16_swap(h, h, false, false);
            return {__builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]),
                    __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1])};
        } else {
            const auto lo = __builtin_amdgcn_permlane32_swap(l, l, false, false);
            const auto hi = __builtin_amdgcn_permlane32_swap(h, h, false, false);
            return {__builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]),
                    __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1])};
        }
    }
}
template <int STEP> __device__ __forceinline__ double max_step(double v)
{
    const Pair p = both<STEP>(settled(v));
    return kmax(p.a, p.b);
}
template <int STEP> __device__ __forceinline__ double sum_step(double v)
{
    const Pair p = both<STEP>(v);
    return p.a + p.b;
}
template <int LANES> __device__ __forceinline__ double row_max(double v)
{
    v = max_step<4>(max_step<2>(max_step<1>(v)));
    if constexpr (LANES >= 16)
        v = max_step<8>(v);
    if constexpr (LANES == 64)
        v = max_step<32>(max_step<16>(v));
    return v;
}
template <int LANES> __device__ __forceinline__ double row_sum(double v)
{
    v = sum_step<4>(sum_step<2>(sum_step<1>(v)));
    if constexpr (LANES >= 16)
        v = sum_step<8>(v);
    if constexpr (LANES == 64)
        v = sum_step<32>(sum_step<16>(v));
    return v;
}
// the two largest of the sets behind two lanes
template <int STEP> __device__ __forceinline__ void top2_step(double &m1, double &m2)
{
    const Pair p = both<STEP>(settled(m1)), q = both<STEP>(settled(m2));
    m1 = kmax(p.a, p.b);
    m2 = kmax(kmin(p.a, p.b), kmax(q.a, q.b));
}

// Sorting networks, largest first.
__device__ __forceinline__ void order(double &a, double &b)
{
    const double x = kmax(a, b);
    b = kmin(a, b);
    a = x;
}
__device__ __forceinline__ void sort8(double *k)
{
    constexpr int NET[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
    for (int i = 0; i < 19; ++i)
        order(k[NET[i][0]], k[NET[i][1]]);
}
// k, rising and then falling (or a rotation of that): a merge of two sorted halves
__device__ __forceinline__ void sort_bitonic8(double *k)
{
#pragma unroll
    for (int d = 4; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(i & d))
                order(k[i], k[i + d]);
}
// the 8 largest of two sorted lists of 8, sorted
__device__ __forceinline__ void merge8(double *k, const double *o)
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
        k[i] = kmax(k[i], o[7 - i]);
    sort_bitonic8(k);
}
// k rising and then falling, sorted
__device__ __forceinline__ void sort_bitonic16(double *k)
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
        order(k[i], k[i + 8]);
    sort_bitonic8(k);
    sort_bitonic8(k + 8);
}
__device__ __forceinline__ void sort16(double *k)
{
    sort8(k);
    sort8(k + 8);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        order(k[i], k[15 - i]);
    sort_bitonic8(k);
    sort_bitonic8(k + 8);
}
template <int STEP> __device__ __forceinline__ void merge_step(double *k)
{
    double a[8], b[8];
    asm("s_nop 3" : "+v"(k[0]), "+v"(k[1]), "+v"(k[2]), "+v"(k[3]), "+v"(k[4]), "+v"(k[5]), "+v"(k[6]), "+v"(k[7]));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const Pair p = both<STEP>(k[i]);
        a[i] = p.a;
        b[i] = p.b;
    }
    merge8(a, b);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        k[i] = a[i];
}

// exp(x) in 64 bits for x in [-700, 700]: x log2 e = n + f, |f| <= 1/2, and the polynomial of degree 9 that meets 2^f in the
// ten Chebyshev nodes of that interval, within 1.9e-14 of it: a twelfth of the last of the 42 bits that count.  n comes out of the
// low bits of x log2 e + 1.5 2^52 and goes into the exponent by an integer addition (rounding, conversion and ldexp
// are slow in 64 bits).  The constants sit in scalar registers: as literals each costs two moves to the FMA that uses it.
struct Exp64 {
    double c[10], log2e, magic;
    __device__ __forceinline__ Exp64()
        : c{0x1.000000000003dp+0,  0x1.62e42fefa39f7p-1,  0x1.ebfbdff8149f1p-3,  0x1.c6b08d7044119p-5,  0x1.3b2ab72b1770bp-7,
            0x1.5d87fe908f91ap-10, 0x1.43088e255df70p-13, 0x1.ffcb767876e1dp-17, 0x1.63ef96c061bdep-20, 0x1.b6571e093a8b8p-24},
          log2e(0x1.71547652b82fep+0), magic(0x1.8p52)
    {
#pragma unroll
        for (int i = 0; i < 10; ++i)
            asm("" : "+s"(c[i]));
        asm("" : "+s"(log2e));
        asm("" : "+v"(magic));  // (an instruction reads one scalar)
    }
    __device__ __forceinline__ double operator()(double x) const
    {
        const double t = __builtin_fma(x, log2e, magic);
        const double f = __builtin_fma(x, log2e, magic - t);
        double p = __builtin_fma(c[9], f, c[8]);
#pragma unroll
        for (int i = 7; i >= 0; --i)
            p = __builtin_fma(p, f, c[i]);
        const uint64_t u = __builtin_bit_cast(uint64_t, p);
        uint32_t hi = (uint32_t)(u >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, t) << 20);
        asm("" : "+v"(hi));  // (one 32-bit shift-add, not five instructions of a 64-bit sum)
        return __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)u);
    }
};
// 1 / d for d in [1, 1e304]: the hardware's estimate (of single precision) and one step of third order
__device__ __forceinline__ double recip64(double d)
{
    const double y = __builtin_amdgcn_rcp(d), e = __builtin_fma(-d, y, 1.0);
    return __builtin_fma(y, __builtin_fma(e, e, e), y);
}
// (a NaN gives some number: its expert is not eligible)
__device__ __forceinline__ double sigmoid64(const Exp64 &exp64, float l)
{
    return recip64(1.0 + exp64((double)__builtin_amdgcn_fmed3f(-l, 700.0f, -700.0f)));
}
// exp(l - mx), 0 for an expert that has no logit (-inf or NaN)
__device__ __forceinline__ double exp_rel(const Exp64 &exp64, float l, float mx)
{
    const double e = exp64(fmin(fmax((double)l - (double)mx, -700.0), 0.0));
    return l > -INFINITY ? e : 0.0;
}

// s >= 0 to 42 fraction bits, the nearest.  (A carry goes on into the exponent, as it should.)
__device__ __forceinline__ double round42(double s)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, s) + 0x200;
    return __builtin_bit_cast(double, (u >> 32) << 32 | ((uint32_t)u & ~0x3FFu));
}

// c with `id` in its low BITS bits, the lower id the larger of two equal c.  flip ^ j: all ones of BITS bits ^ id
// FINITE: c is.  (Otherwise it is limited first: an infinity would turn into a NaN.)
template <int BITS, bool FINITE = false> __device__ __forceinline__ double tag(double c, uint32_t flip, int j = 0)
{
    constexpr uint32_t M = (1u << BITS) - 1;
    const uint64_t u = __builtin_bit_cast(uint64_t, FINITE ? c : fmin(c, 0x1p1023));
    const uint32_t hi = (uint32_t)(u >> 32);
    uint32_t sign = (uint32_t)((int32_t)hi >> 31);
    asm("" : "+v"(sign));  // (a comparison of 64 bits and a selection otherwise)
    const uint32_t id = __builtin_amdgcn_bitop3_b32(flip, sign, (uint32_t)j, 0x96);       // flip ^ sign ^ j
    const uint32_t low = __builtin_amdgcn_bitop3_b32(M, id, (uint32_t)u, 0xCA);  // (M & id) | (~M & u)
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | low);
}
template <int BITS> __device__ __forceinline__ int untag(double key)
{
    constexpr uint32_t M = (1u << BITS) - 1;
    const uint64_t u = __builtin_bit_cast(uint64_t, key);
    return (int)(((uint32_t)u ^ M ^ (uint32_t)((int64_t)u >> 63)) & M);
}
constexpr int RG_PLACE = 10;  // bits of an expert's place: its lane of the token, then its place in the lane
constexpr int place_bits(int per) { return per <= 1 ? 0 : 1 + place_bits((per + 1) / 2); }
// a key (a group) that is out: the value below RG_NONE_MAX, whatever its low word
__device__ __forceinline__ double none_if(bool out, double key)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, key);
    return __builtin_bit_cast(double, (uint64_t)(out ? RG_NONE_HI : (uint32_t)(u >> 32)) << 32 | (uint32_t)u);
}
__device__ __forceinline__ double none() { return __builtin_bit_cast(double, (uint64_t)RG_NONE_HI << 32); }
// whether two tagged keys are the same expert's (group's).  (The whole keys: a low word alone can be that of another
// expert's, as the ids in keys below zero are turned over.)
__device__ __forceinline__ bool same_id(double a, double b) { return a == b; }

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
// The logits e0 ... e0 + PER - 1 of a row, or the biases; past the last expert the last ones again.  vec: by fours (a
// group's size is a multiple of 4 then, and so is e0).  With every lane full nothing needs to be kept inside the row.  (By
// fours against one by one: 96 experts, 128 tokens 5.1 -> 4.0 us, 320 experts, 65536 tokens 77 -> 48.)
// Global memory takes such loads at any address: a slice that starts anywhere is as fast (256 experts, 65536 tokens 31.0 us on 16
// bytes and 31.2 off them).
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));
template <int PER, typename LOAD> __device__ __forceinline__ void fours(const RouteGroupedArgs &p, int e0, LOAD load)
{
    if (p.full) {
#pragma unroll
        for (int j = 0; j < PER / 4; ++j)
            load(j, e0 + 4 * j);
    } else {
#pragma unroll
        for (int j = 0; j < PER / 4; ++j)
            load(j, min(e0 + 4 * j, p.E - 4));
    }
}
template <int PER> __device__ __forceinline__ void load_f32(const float *row, const RouteGroupedArgs &p, int e0, float *v)
{
    if (PER % 4 == 0 && p.vec) {
        f32x4 q[PER / 4 ? PER / 4 : 1];
        fours<PER>(p, e0, [&](int j, int e) { q[j] = *reinterpret_cast<const f32x4_u *>(row + e); });
#pragma unroll
        for (int j = 0; j < PER; ++j)
            v[j] = q[j / 4][j & 3];
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            v[j] = row[min(e0 + j, p.E - 1)];
    }
}
template <int PER> __device__ __forceinline__ void load_logits(const char *row, const RouteGroupedArgs &p, int e0, float *lg)
{
    if (p.dtype == ROUTE_FP32) {
        load_f32<PER>(reinterpret_cast<const float *>(row), p, e0, lg);
        return;
    }
    const uint16_t *half = reinterpret_cast<const uint16_t *>(row);
    const bool bf16 = p.dtype == ROUTE_BF16;
    if (PER % 4 == 0 && p.vec) {
        u32x2 v[PER / 4 ? PER / 4 : 1];
        fours<PER>(p, e0, [&](int j, int e) { v[j] = *reinterpret_cast<const u32x2_u *>(half + e); });
#pragma unroll
        for (int j = 0; j < PER; ++j)
            lg[j] = half_to_f32(v[j / 4][(j >> 1) & 1] >> (16 * (j & 1)), bf16);
    } else {
        uint32_t h[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j)
            h[j] = half[min(e0 + j, p.E - 1)];
#pragma unroll
        for (int j = 0; j < PER; ++j)
            lg[j] = half_to_f32(h[j], bf16);
    }
}

// How the picks are found.  RG_EACH: each by a reduction over all of a lane's experts and the lanes.  RG_MERGE (K <= 8): the
// lanes sort their experts and merge their lists of 8.  RG_POP: the lanes sort their experts, each pick is the largest of the
// lists' heads, and its lane's list moves up.
enum { RG_EACH, RG_MERGE, RG_POP };
// Pick FROM and those behind it, K in all: lane k of a token gets the k-th.
template <int LANES, int LIST, int FROM> __device__ __forceinline__ void pop_picks(double *key, int K, int rl, double &pick)
{
    if constexpr (FROM < 16) {
        const double best = row_max<LANES>(key[0]);
        pick = rl == FROM ? best : pick;
        if (FROM + 1 == K)
            return;
        const bool mine = same_id(key[0], best);
        constexpr int MOVES = LIST - 1 < 15 - FROM ? LIST - 1 : 15 - FROM;  // (what the picks to come may need)
#pragma unroll
        for (int j = 0; j < MOVES; ++j)
            key[j] = mine ? key[j + 1] : key[j];
        if constexpr (LIST == 8)
            key[7] = none_if(mine, key[7]);
        pop_picks<LANES, LIST, FROM + 1>(key, K, rl, pick);
    }
}

// the two largest of a group, from those of its lanes
template <int LANES> __device__ __forceinline__ void best_two_of_group(int lpg, double &m1, double &m2)
{
    if (lpg > 1)
        top2_step<1>(m1, m2);
    if (lpg > 2)
        top2_step<2>(m1, m2);
    if (lpg > 4)
        top2_step<4>(m1, m2);
    if constexpr (LANES >= 16) {
        if (lpg > 8)
            top2_step<8>(m1, m2);
    }
    if constexpr (LANES == 64) {
        if (lpg > 16)
            top2_step<16>(m1, m2);
    }
}
// the two largest of a lane
template <int N> __device__ __forceinline__ void best_two(const double *k, double &m1, double &m2)
{
    m1 = k[0];
    m2 = none();
#pragma unroll
    for (int j = 1; j < N; ++j) {
        m2 = kmax(m2, kmin(m1, k[j]));
        m1 = kmax(m1, k[j]);
    }
}
// whether this lane's group g, of that score, is among the KG best (some: there is an expert to pick in it)
template <int LANES> __device__ __forceinline__ bool keep_group(int KG, int g, double score, bool some)
{
    double gk = none_if(!some, tag<6>(score, 63u ^ (uint32_t)g));
    bool kept = false;
    for (int i = 0; i < KG; ++i) {
        const double win = row_max<LANES>(gk);
        const bool mine = same_id(gk, win) && win > RG_NONE_MAX;
        kept |= mine;
        gk = none_if(mine, gk);
    }
    return kept;
}
// One token's picks, by LANES adjacent lanes of which this is the rl-th: lane k gets the k-th pick (-1: none) and its gate,
// not yet scaled.  row: the token's logits.
template <int LANES, int PER, int PICK>
__device__ __forceinline__ void route_token(const RouteGroupedArgs &p, const char *row, int rl, int &my_idx, double &gate)
{
    constexpr bool SORTED = PICK != RG_EACH;
    // (lanes past the last group look at expert 0's, so that their loads stay inside the row, and hold none)
    const int g = rl >> p.lpg_log, pos0 = (rl & (p.lpg - 1)) * PER, e0 = g < p.G ? g * p.gs + pos0 : 0;
    const int have = g < p.G ? min(max(p.gs - pos0, 0), PER) : 0;
    constexpr int LOG = place_bits(PER);
    static_assert((LANES << LOG) <= (1 << RG_PLACE), "places fit their bits");
    const uint32_t flip = ((1u << RG_PLACE) - 1) ^ (uint32_t)(rl << LOG);
    const auto expert_of = [&](double key) {
        const int at = untag<RG_PLACE>(key), l = at >> LOG;
        return (l >> p.lpg_log) * p.gs + (l & (p.lpg - 1)) * PER + (at & ((1 << LOG) - 1));
    };

    float lg[PER], bs[PER];
    load_logits<PER>(row, p, e0, lg);
    if (p.bias) {
        load_f32<PER>(p.bias, p, e0, bs);
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            bs[j] = 0.0f;
    }
    if (!p.full) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            lg[j] = j < have ? lg[j] : -INFINITY;
    }
    const Exp64 exp64;
    const bool softmax = p.score == ROUTE_SOFTMAX;
    const bool by_logit = p.by_logit != 0, choose = p.KG < p.G;
    bool kept = true;
    double denom = 0.0;
    float mx = -INFINITY;
    if (softmax) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            mx = fmaxf(mx, lg[j]);
        mx = fminf((float)row_max<LANES>((double)mx), 0x1.fffffep127f);  // (exact; +inf is taken as the largest number)
    }

    constexpr int LIST = PICK == RG_EACH ? PER : PICK == RG_POP && PER > 8 ? 16 : 8;
    double key[LIST > PER ? LIST : PER];
    if (by_logit) {
        if (softmax && !p.renorm) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                denom += exp_rel(exp64, lg[j], mx);
            denom = row_sum<LANES>(denom);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j)  // (+ 0: the zeros of both signs are equal)
            key[j] = none_if(!(lg[j] > -INFINITY), tag<RG_PLACE>((double)lg[j] + 0.0, flip, j));
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
        for (int j = 0; j < PER; ++j)
            key[j] = round42(key[j]) + (double)bs[j];
        // infinities and NaN among the wave's logits and biases: seldom, so that none is looked for one by one
        float far = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            far = __builtin_elementwise_maximum(__builtin_elementwise_maximum(far, fabsf(lg[j])), fabsf(bs[j]));
        if (__any(!(far < INFINITY))) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const bool out = !(lg[j] > -INFINITY) | !(bs[j] > -INFINITY);
                key[j] = out ? none() : fmin(key[j], 0x1p1023);
            }
        }
        // sums of whole scores: with the places in their low bits, which weigh by each one's exponent, those would decide
        // between equal sums of different parts.  (The sorted keys' two first would be free: 512 experts, 65536 tokens 61.5
        // us against 65.8; 256 36.8 and 36.0, one token 4.9 and 4.9.)
        if (choose && p.group_top2) {
            double m1, m2;
            best_two<PER>(key, m1, m2);
            best_two_of_group<LANES>(p.lpg, m1, m2);
            kept = keep_group<LANES>(p.KG, g, m2 > RG_NONE_MAX ? m1 + m2 : m1, m1 > RG_NONE_MAX);
        }
#pragma unroll
        for (int j = 0; j < PER; ++j)
            key[j] = tag<RG_PLACE, true>(key[j], flip, j);
    }

    // the lane's best, sorted
    if constexpr (SORTED) {
        constexpr int PADDED = (PER + 7) & ~7;
        double pad[PADDED];
#pragma unroll
        for (int j = 0; j < PADDED; ++j)
            pad[j] = j < PER ? key[j < PER ? j : 0] : none();
        if constexpr (LIST == 8) {
#pragma unroll
            for (int j = 0; j < PADDED; j += 8) {
                sort8(pad + j);
                if (j > 0)
                    merge8(pad, pad + j);
            }
        } else {
            sort16(pad);
            if constexpr (PADDED == 24)
                sort8(pad + 16);
            if constexpr (PADDED == 32)
                sort16(pad + 16);
            if constexpr (PADDED > 16) {
#pragma unroll
                for (int j = 16; j < PADDED; ++j)
                    pad[31 - j] = kmax(pad[31 - j], pad[j]);
                sort_bitonic16(pad);
            }
        }
#pragma unroll
        for (int j = 0; j < LIST; ++j)
            key[j] = pad[j];
    }

    if (choose) {
        if (!p.group_top2) {  // (the places give equal ones to the lower group, as its tag does)
            double m1 = key[0], m2 = none();
            if constexpr (!SORTED)
                best_two<PER>(key, m1, m2);
            best_two_of_group<LANES>(p.lpg, m1, m2);
            kept = keep_group<LANES>(p.KG, g, m1, m1 > RG_NONE_MAX);
        }
#pragma unroll
        for (int j = 0; j < LIST; ++j)
            key[j] = none_if(!kept, key[j]);
    }

    my_idx = -1;
    if constexpr (PICK == RG_POP) {
        double pick = none();
        pop_picks<LANES, LIST, 0>(key, p.K, rl, pick);
        if (pick > RG_NONE_MAX)
            my_idx = expert_of(pick);
    } else if constexpr (SORTED) {
        merge_step<1>(key);
        merge_step<2>(key);
        merge_step<4>(key);
        if constexpr (LANES >= 16)
            merge_step<8>(key);
        if constexpr (LANES == 64) {
            merge_step<16>(key);
            merge_step<32>(key);
        }
        double mine = key[0];
#pragma unroll
        for (int j = 1; j < 8; ++j)
            mine = rl == j ? key[j] : mine;
        if (rl < p.K && mine > RG_NONE_MAX)
            my_idx = expert_of(mine);
    } else {
#pragma unroll 1
        for (int k = 0; k < p.K; ++k) {
            double best = key[0];
#pragma unroll
            for (int j = 1; j < PER; ++j)
                best = kmax(best, key[j]);
            best = row_max<LANES>(best);
#pragma unroll
            for (int j = 0; j < PER; ++j)
                key[j] = none_if(same_id(key[j], best), key[j]);
            if (rl == k)
                my_idx = best > RG_NONE_MAX ? expert_of(best) : -1;
        }
    }

    gate = 0.0;
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
}

inline int route_pow2(int v)  // the power of two at or above
{
    int r = 1;
    while (r < v)
        r *= 2;
    return r;
}
// The lanes' shares of the experts, for `lanes` lanes a token: returns how many each holds at most.
inline int route_shares(RouteGroupedArgs &a, int lanes)
{
    a.gs = a.E / a.G;
    // without a bias the scores order as the logits do, and so do the groups by their largest one
    a.by_logit = !a.bias && (a.KG == a.G || !a.group_top2);
    a.lpg = lanes / route_pow2(a.G);
    a.lpg_log = __builtin_ctz((unsigned)a.lpg);
    return (a.gs + a.lpg - 1) / a.lpg;
}
// PER: the places for a lane's experts
inline void route_places(RouteGroupedArgs &a, int lanes, int per)
{
    a.full = a.gs == a.lpg * per && a.G * a.lpg == lanes;  // every lane holds PER experts
    a.vec = per % 4 == 0 && a.gs % 4 == 0;                 // a lane's experts by fours
}

}  // namespace

}  // namespace cam
