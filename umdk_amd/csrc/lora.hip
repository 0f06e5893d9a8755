// Low-rank adapters of many requests beside a projection that they share:
//   out[t] = base[t] + scaling[a] * B_a (A_a x_t),  a = ids[t];  out[t] = base[t] where a is no adapter
// Two launches: z = A x in fp32, then out = base + B z.
//
// Tokens come in any order, so every block sorts for itself: it looks at a window of 256 tokens, counts for each one the
// earlier ones with the same adapter, and takes up to CHUNK tokens of one adapter, a chunk.  A decode batch is one window, in which an
// adapter is read once for all of its tokens; in prompts a window holds a run or two.  No order is prepared in a launch of
// its own or kept, and no sum hangs on what other tokens are there: a token's bits are the same in any order of a batch of its size.
//
// What bounds it: for few tokens the adapters' stream and the latency of two launches, for many the streams of x, base and out.
// Measured (K x N): one row of 4096 x 4096 at rank 16 3.5 + 4.4 us; 64 int8 rows of 7168 x 4096 with 32 adapters 6.7 + 7.5; 1021
// rows of 4096 x 4096 6.3 + 9.4; 16384 rows of 4096 x 14336 at rank 64 33.6 (4.1 TB/s) + 202 (4.6 TB/s; B and z, 100 MB of
// them past L2, included 5.2).  Both in one launch, each block with a z of its own, took longer where it should have helped
// (one row 8.3 -> 10.8 us, 64 rows 13 -> 20).
// Matrix instructions take 16 tokens as their columns, rows of A or B as their rows.  z goes into the second product as 16-bit
// numbers, each what those before it leave out, with all the bits of the fp32 sums: three bf16 numbers, or two of fp16, which are
// within 2^-24 of it (2^-35 of the row's largest, brought to 2^10 first).  (Two bf16 numbers lost 2^-18: 16384 rows of rank 64 230 us,
// with three 236.)
#include <atomic>
#include <type_traits>

#include "cam_device.h"
#include "launchers.h"

namespace cam {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int LR_WINDOW = 256, LR_WAVES = 4, LR_THREADS = 64 * LR_WAVES;
constexpr int LR_MAX_SPLITS = 8;
static_assert(LR_THREADS == LR_WINDOW, "a thread per token of the window");

// two fp32 -> two 16-bit numbers, the nearest
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b)
{
    if constexpr (BF16)
        return f32x2_to_bf16x2(a, b);
    else
        return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}
template <bool BF16> __device__ __forceinline__ float unpack(uint32_t v, int i)
{
    if constexpr (BF16)
        return __uint_as_float(i ? v & 0xffff0000u : v << 16);
    else
        return (float)__builtin_bit_cast(f16x2, v)[i];
}
template <bool BF16> __device__ __forceinline__ f32x4 mfma(const u32x4 a, const u32x4 b, const f32x4 c)
{
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// four int8 -> four 16-bit numbers
template <bool BF16> __device__ __forceinline__ u32x2 bytes4(uint32_t d)
{
    return u32x2{pack2<BF16>((float)(int8_t)d, (float)(int8_t)(d >> 8)), pack2<BF16>((float)(int8_t)(d >> 16), (float)((int32_t)d >> 24))};
}

// ---------------------------------------------------------------- chunks
// The tokens of a window by chunks: chunk q holds up to SIZE tokens of one adapter, or of none (id -1).  A token's rank is the
// number of earlier ones with its adapter: those of its wave by ballots, an adapter of the wave at a time, those of earlier
// waves from a table (open addressing; where an adapter lies in it hangs on the order of the waves, but nothing else
// does: all blocks of a window, and both kernels, number its chunks alike).
constexpr int LR_TABLE = 2 * LR_WINDOW, LR_EMPTY = -2;
struct Chunks {
    int32_t key[LR_TABLE];
    uint8_t tokens[LR_TABLE][LR_WAVES];  // of an adapter, in each wave
    int32_t count[LR_WAVES];
    int32_t at, place;  // of the chunk asked for: its first rank, its adapter's place in the table
    int32_t list[LR_WINDOW];
};
// This thread's token: its adapter's place, its rank, the number of the chunk that it leads (-1: none)
struct Token {
    int place, rank, leads;
};
// returns the number of chunks
__device__ __forceinline__ int find_chunks(Chunks &c, const int32_t *ids, int64_t m0, int n, int L, int size, Token &tok)
{
    const int j = threadIdx.x, lane = j & 63, w = __builtin_amdgcn_readfirstlane(j >> 6);
    int a = LR_EMPTY;
    if (j < n)
        a = ids[m0 + j];
#pragma unroll
    for (int i = 0; i < LR_TABLE; i += LR_THREADS) {
        c.key[i + j] = LR_EMPTY;
        reinterpret_cast<uint32_t *>(c.tokens)[i + j] = 0;
    }
    if (j < n)
        a = a < 0 || a >= L ? -1 : a;
    // among the wave
    tok.rank = -1;
    int leader = lane, same = 0;
    for (uint64_t left = __ballot(j < n); left;) {
        const int first = __builtin_ctzll(left);
        const uint64_t m = __ballot(a == __builtin_amdgcn_readlane(a, first));
        if (m >> lane & 1) {
            leader = first;
            tok.rank = __popcll(m & lanemask_lt());
            same = __popcll(m);
        }
        left &= ~m;
    }
    __syncthreads();
    int place = 0;
    if (j < n && leader == lane) {
        place = (int)((uint32_t)a * 0x9E3779B1u >> 23);
        static_assert(LR_TABLE == 1 << 9, "the hash's bits");
        for (;;) {  // (at most 256 of the 512 places are taken)
            const int there = atomicCAS(&c.key[place], LR_EMPTY, a);
            if (there == LR_EMPTY || there == a)
                break;
            place = (place + 1) & (LR_TABLE - 1);
        }
        c.tokens[place][w] = (uint8_t)same;
    }
    tok.place = j < n ? __shfl(place, leader, 64) : -1;
    __syncthreads();
    if (j < n) {
#pragma unroll
        for (int v = 0; v < LR_WAVES; ++v)
            tok.rank += v < w ? c.tokens[tok.place][v] : 0;
    }
    const bool leads = j < n && (tok.rank & (size - 1)) == 0;
    const uint64_t mask = __ballot(leads);
    if (lane == 0)
        c.count[w] = __popcll(mask);
    __syncthreads();
    int total = 0;
    tok.leads = __popcll(mask & lanemask_lt());
#pragma unroll
    for (int v = 0; v < LR_WAVES; ++v) {
        tok.leads += v < w ? c.count[v] : 0;
        total += c.count[v];
    }
    if (!leads)
        tok.leads = -1;
    return __builtin_amdgcn_readfirstlane(total);
}
// chunk q's tokens into c.list; its adapter (-1: none) and how many they are
__device__ __forceinline__ int take_chunk(Chunks &c, int size, int q, const Token &tok, int &members)
{
    if (tok.leads == q) {
        c.place = tok.place;
        c.at = tok.rank;
    }
    __syncthreads();
    const int place = __builtin_amdgcn_readfirstlane(c.place), at = __builtin_amdgcn_readfirstlane(c.at);
    if (tok.place == place && tok.rank >= at && tok.rank < at + size)
        c.list[tok.rank - at] = threadIdx.x;
    int all = 0;
#pragma unroll
    for (int v = 0; v < LR_WAVES; ++v)
        all += c.tokens[place][v];
    members = __builtin_amdgcn_readfirstlane(min(size, all - at));
    const int adapter = __builtin_amdgcn_readfirstlane(c.key[place]);
    __syncthreads();
    return adapter;
}

// ---------------------------------------------------------------- A x
struct ShrinkArgs {
    const void *x, *a;
    const int32_t *ids;
    float *z;           // [splits, M, R]
    int64_t M, x_stride;
    int K, R, L, splits, slots, groups;  // slots: blocks that share a window's chunks; groups: of rows of A
};
// at most N of this wave's loads are in flight, and none of its LDS reads
template <int N> __device__ __forceinline__ void wait_loads()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}
template <int MOST, int LOADS> __device__ __forceinline__ void wait_steps(int left)
{
    if constexpr (MOST == 0) {
        wait_loads<0>();
    } else {
        if (left >= MOST)
            wait_loads<MOST * LOADS>();
        else
            wait_steps<MOST - 1, LOADS>(left);
    }
}
__device__ __forceinline__ void dma(const uint8_t *g, uint8_t *lds)
{
    __builtin_amdgcn_global_load_lds(g, (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// 16 MF tokens by 16 NF rows of A over a block's share of K.  The waves take turns at units of 128 bytes of x (64 values, of
// int8 128), each with a ring of SLOTS units of its own in LDS, so that no wave waits for another before the end.  A load
// instruction brings 8 rows by 128 bytes, whole cache lines; 16-byte pieces are turned by (row / 2) mod 8, so that the rows of
// a fragment fall on different banks.
template <bool BF16, bool INT8, int MF, int NF, int SLOTS>
__global__ __launch_bounds__(LR_THREADS) void lora_shrink_kernel(const ShrinkArgs p)
{
    constexpr int LINES = INT8 ? 2 : 1;                        // of A, to a line of x
    constexpr int A_BANDS = 2 * NF * LINES, BANDS = A_BANDS + 2 * MF, SLOT = BANDS * 1024, UNIT = INT8 ? 128 : 64;
    static_assert(MF * NF * 1024 <= SLOTS * SLOT && (SLOTS - 1) * BANDS < 64, "sums where the ring was; vmcnt range");
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    __shared__ Chunks c;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int group = id % p.groups;
    id /= p.groups;
    const int first = id % p.slots;
    const int64_t m0 = (int64_t)(id / p.slots) * LR_WINDOW;
    const int n = (int)min((int64_t)LR_WINDOW, p.M - m0);
    Token tok;
    const int chunks = find_chunks(c, p.ids, m0, n, p.L, 16 * MF, tok);

    const int K = p.K, x_bytes = INT8 ? K : 2 * K, a_bytes = 2 * K;
    const int units = (K + UNIT - 1) / UNIT, from = units * split / p.splits, to = units * (split + 1) / p.splits;
    const int mine = to - from > w ? (to - from - w + LR_WAVES - 1) / LR_WAVES : 0;
    uint8_t *ring = smem + w * SLOTS * SLOT;
    const int turned = (lane & 7) ^ (lane >> 4);  // in even bands of 8 rows; odd ones: ^ 4
    for (int q = first; q < chunks; q += p.slots) {
        int members;
        const int adapter = take_chunk(c, 16 * MF, q, tok, members);
        if (adapter < 0)
            continue;
        const uint8_t *xr[2 * MF], *ar[2 * NF];
#pragma unroll
        for (int b = 0; b < 2 * MF; ++b)
            xr[b] = reinterpret_cast<const uint8_t *>(p.x) +
                    (m0 + c.list[min(b * 8 + (lane >> 3), members - 1)]) * p.x_stride * (INT8 ? 1 : 2);
#pragma unroll
        for (int b = 0; b < 2 * NF; ++b)
            ar[b] = reinterpret_cast<const uint8_t *>(p.a) +
                    ((int64_t)adapter * p.R + min((group * 2 * NF + b) * 8 + (lane >> 3), p.R - 1)) * a_bytes;
        const auto load = [&](int t, int slot) {
            const int u = from + w + t * LR_WAVES;
            uint8_t *lds = ring + slot * SLOT;
#pragma unroll
            for (int b = 0; b < 2 * NF; ++b)
#pragma unroll
                for (int l = 0; l < LINES; ++l)
                    dma(ar[b] + min((u * LINES + l) * 128 + ((turned ^ (4 * (b & 1))) << 4), a_bytes - 16), lds + (l * 2 * NF + b) * 1024);
#pragma unroll
            for (int b = 0; b < 2 * MF; ++b)
                dma(xr[b] + min(u * 128 + ((turned ^ (4 * (b & 1))) << 4), x_bytes - 16), lds + (A_BANDS + b) * 1024);
        };
        f32x4 acc[MF][NF];
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if (s < mine)
                load(s, s);
        // 16-byte piece `piece` of row l16 of a fragment
        const auto piece_at = [&](int piece) { return l16 * 128 + ((piece ^ (l16 >> 1)) << 4); };
        int slot = 0;
#pragma unroll 1
        for (int t = 0; t < mine; ++t) {
            wait_steps<SLOTS - 1, BANDS>(mine - 1 - t);
            const uint8_t *at = ring + slot * SLOT;
            constexpr int STEPS = INT8 ? 4 : 2;  // of 32 values
            u32x4 xf[MF][STEPS], af[NF][STEPS];
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4 v = *reinterpret_cast<const u32x4 *>(at + (A_BANDS + 2 * i) * 1024 + piece_at(lq + 4 * h));
                    if constexpr (INT8) {
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            const u32x2 lo = bytes4<BF16>(v[2 * s]), hi = bytes4<BF16>(v[2 * s + 1]);
                            xf[i][2 * h + s] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                        }
                    } else {
                        xf[i][h] = v;
                    }
                }
            // the same columns of A: of int8 rows' piece lq + 4 h the 16 values from 64 h + 16 lq on
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
                    af[j][s] = *reinterpret_cast<const u32x4 *>(
                        at + (INT8 ? (s >> 1) * 2 * NF + 2 * j : 2 * j) * 1024 + piece_at(INT8 ? 2 * lq + (s & 1) : lq + 4 * s));
            wait_loads<63>();  // (the slot has been read)
            if (t + SLOTS < mine)
                load(t + SLOTS, slot);
            const int k = (from + w + t * LR_WAVES) * UNIT;
            if (k + UNIT > K) {
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
                    if (k + (INT8 ? (s >> 1) * 64 + lq * 16 + (s & 1) * 8 : s * 32 + lq * 8) >= K) {
#pragma unroll
                        for (int j = 0; j < NF; ++j)
                            af[j][s] = u32x4{0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < MF; ++i)
                            xf[i][s] = u32x4{0, 0, 0, 0};
                    }
            }
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int i = 0; i < MF; ++i)
#pragma unroll
                    for (int j = 0; j < NF; ++j)
                        acc[i][j] = mfma<BF16>(af[j][s], xf[i][s], acc[i][j]);
            slot = slot == SLOTS - 1 ? 0 : slot + 1;
        }
        // the waves' sums meet where their rings were
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                *reinterpret_cast<f32x4 *>(ring + (i * NF + j) * 1024 + lane * 16) = acc[i][j];
        __syncthreads();
        for (int f = w; f < MF * NF; f += LR_WAVES) {
            f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < LR_WAVES; ++v)
                sum += *reinterpret_cast<const f32x4 *>(smem + v * SLOTS * SLOT + f * 1024 + lane * 16);
            const int i = f / NF * 16 + l16, r = (group * NF + f % NF) * 16 + lq * 4;
            if (i < members && r < p.R)
                *reinterpret_cast<f32x4 *>(p.z + ((int64_t)split * p.M + m0 + c.list[i]) * p.R + r) = sum;
        }
    }
}

// ---------------------------------------------------------------- base + B z
struct ExpandArgs {
    const void *base, *b;
    const float *z, *xs, *scaling;
    const int32_t *ids;
    void *out;
    int64_t M, base_stride;
    int N, R, L;
    int16_t splits, slots, tiles;  // tiles: of 64 columns, that a wave does
    int8_t base_dtype, out_bf16;
};
// 8 consecutive numbers of base, of 16 or (WIDE) of 32 bits.  FULL: all of them are there, otherwise the first `left`.
template <bool WIDE> struct Raw8 {
    u32x4 v[WIDE ? 2 : 1];
};
typedef u32x4 u32x4_u __attribute__((aligned(2)));
template <bool WIDE, bool FULL> __device__ __forceinline__ Raw8<WIDE> load8(const void *p, int64_t at, int left)
{
    Raw8<WIDE> r;
    const uint8_t *b = reinterpret_cast<const uint8_t *>(p) + at * (WIDE ? 4 : 2);
#pragma unroll
    for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
        if constexpr (FULL) {
            r.v[h] = *reinterpret_cast<const u32x4_u *>(b + 16 * h);
        } else {
            r.v[h] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < (WIDE ? 4 : 8); ++i)
                if (i + 4 * h < left) {
                    if constexpr (WIDE)
                        r.v[h][i] = reinterpret_cast<const uint32_t *>(b)[i + 4 * h];
                    else
                        r.v[h][i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(b)[i] << (16 * (i & 1));
                }
        }
    }
    return r;
}
template <bool WIDE> __device__ __forceinline__ void to_fp32(const Raw8<WIDE> &r, bool bf16, float *v)
{
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = __uint_as_float(r.v[i >> 2][i & 3]);
    } else if (bf16) {
        unpack_bf16x8(r.v[0], v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = unpack<false>(r.v[0][i >> 1], i & 1);
    }
}
__device__ __forceinline__ u32x4 pack8(bool bf16, const float *v)
{
    u32x4 r;
    if (bf16) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = pack2<true>(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = pack2<false>(v[2 * i], v[2 * i + 1]);
    }
    return r;
}
template <bool FULL> __device__ __forceinline__ void store8(void *p, int64_t at, bool bf16, int left, const float *v)
{
    const u32x4 r = pack8(bf16, v);
    uint16_t *h = reinterpret_cast<uint16_t *>(p) + at;
    if constexpr (FULL) {
        *reinterpret_cast<u32x4_u *>(h) = r;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left)
                h[i] = (uint16_t)(r[i >> 1] >> (16 * (i & 1)));
    }
}

// z of a chunk into LDS as the instructions' second operand: [token fragment][step of 32][number][lane] 16 bytes, and each
// token's factor
template <bool BF16> constexpr int NUMBERS = BF16 ? 3 : 2;
template <bool BF16, int KS, int MF>
__device__ __forceinline__ void lay_out(const ExpandArgs &p, const Chunks &c, int64_t m0, int members, int adapter,
                                        u32x4 (&zs)[MF][KS][NUMBERS<BF16>][64], float (&factor)[16 * MF])
{
    // 4 KS threads a token, 8 values each
    for (int i = threadIdx.x; i < 16 * MF * 4 * KS; i += LR_THREADS) {
        const int t = i / (4 * KS), part = i % (4 * KS), r = part * 8;
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            z[e] = 0.0f;
        const int64_t m = m0 + c.list[min(t, members - 1)];
        if (r < p.R) {
            constexpr int AT_ONCE = MF == 4 ? 2 : LR_MAX_SPLITS;  // (many rows: few splits, and registers are waves)
            for (int s0 = 0; s0 < p.splits; s0 += AT_ONCE) {
                f32x4 v[AT_ONCE][2];
#pragma unroll
                for (int s = 0; s < AT_ONCE; ++s) {
                    const f32x4 *from = reinterpret_cast<const f32x4 *>(p.z + ((int64_t)min(s0 + s, p.splits - 1) * p.M + m) * p.R + r);
                    v[s][0] = from[0];
                    v[s][1] = from[1];
                }
#pragma unroll
                for (int s = 0; s < AT_ONCE; ++s)
                    if (s0 + s < p.splits) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            z[e] += v[s][e >> 2][e & 3];
                    }
            }
        }
        float f = p.scaling ? p.scaling[adapter] : 1.0f;
        if (p.xs)
            f *= p.xs[m];
        if constexpr (!BF16) {  // the row's largest finite one to 2^10 or a little less: what is left out then keeps its bits
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                most = fmaxf(most, fabsf(z[e]) < INFINITY ? fabsf(z[e]) : 0.0f);
            most = KS == 8 ? group_max<32>(most) : KS == 4 ? group_max<16>(most) : KS == 2 ? group_max<8>(most) : group_max<4>(most);
            const int e2 = most > 0.0f ? 10 - ilogbf(most) : 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                z[e] = ldexpf(z[e], e2);
            f = ldexpf(f, -e2);
        }
        // (Nothing is left of an infinity or a NaN, where the difference would make a NaN of both.  bf16 numbers are cut off, not
        // rounded: what is left out then has 8 bits less, and no finite number becomes an infinity.)
#pragma unroll
        for (int k = 0; k < NUMBERS<BF16>; ++k) {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (BF16)
                    v[e] = __float_as_uint(z[2 * e]) >> 16 | (__float_as_uint(z[2 * e + 1]) & 0xffff0000u);
                else
                    v[e] = pack2<BF16>(z[2 * e], z[2 * e + 1]);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    z[2 * e + i] = fabsf(z[2 * e + i]) < INFINITY ? z[2 * e + i] - unpack<BF16>(v[e], i) : 0.0f;
            }
            zs[t >> 4][part >> 2][k][(part & 3) * 16 + (t & 15)] = v;
        }
        if (part == 0)
            factor[t] = f;
    }
}
// B's rows of a tile of 64 columns from n0 on.  Row i of fragment f is column 32 (f / 2) + 8 (i / 4) + 4 (f mod 2) + i mod 4,
// so that a lane's results are twice 8 consecutive columns of one token.
template <int KS> struct Tile {
    u32x4 v[4][KS];
};
template <int KS> __device__ __forceinline__ Tile<KS> load_b(const ExpandArgs &p, int adapter, int n0, int l16, int lq)
{
    Tile<KS> t;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int col = min(n0 + 32 * (f >> 1) + 8 * (l16 >> 2) + 4 * (f & 1) + (l16 & 3), p.N - 1);
        const uint16_t *row = reinterpret_cast<const uint16_t *>(p.b) + ((int64_t)adapter * p.N + col) * p.R;
#pragma unroll
        for (int s = 0; s < KS; ++s)  // (past the rank: the last of it, for now)
            t.v[f][s] = *reinterpret_cast<const u32x4 *>(row + min(s * 32 + lq * 8, p.R - 8));
    }
    return t;
}
template <int KS> __device__ __forceinline__ void clear_past_rank(Tile<KS> &t, int R, int lq)
{
    if (32 * KS > R) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
            if (s * 32 + lq * 8 >= R) {
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    t.v[f][s] = u32x4{0, 0, 0, 0};
            }
    }
}
// a fragment of 16 tokens' z times a tile of B, scaled, added to v
template <bool BF16, int KS>
__device__ __forceinline__ void add_product(const Tile<KS> &b, const u32x4 (&z)[KS][NUMBERS<BF16>][64], float scale, int lane, float (&v)[2][8])
{
    f32x4 acc[4];
#pragma unroll
    for (int f = 0; f < 4; ++f)
        acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int part = 0; part < NUMBERS<BF16>; ++part) {
            const u32x4 zv = z[s][part][lane];
#pragma unroll
            for (int f = 0; f < 4; ++f)
                acc[f] = mfma<BF16>(b.v[f][s], zv, acc[f]);
        }
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[g][e] = __builtin_fmaf(scale, acc[2 * g + (e >> 2)][e & 3], v[g][e]);
}

// A chunk of up to 16 MF tokens by 64 columns a wave at a time, of base of any type and alignment.
template <bool BF16, bool WIDE, int KS, int MF> __global__ __launch_bounds__(LR_THREADS) void lora_expand_kernel(const ExpandArgs p)
{
    __shared__ Chunks c;
    __shared__ u32x4 zs[MF][KS][NUMBERS<BF16>][64];
    __shared__ float factor[16 * MF];
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int span = 64 * LR_WAVES * p.tiles, n_blocks = (p.N + span - 1) / span;
    int id = blockIdx.x;
    const int n_block = id % n_blocks;
    id /= n_blocks;
    const int first = id % p.slots;
    const int64_t m0 = (int64_t)(id / p.slots) * LR_WINDOW;
    const int n = (int)min((int64_t)LR_WINDOW, p.M - m0);
    Token tok;
    const int chunks = find_chunks(c, p.ids, m0, n, p.L, 16 * MF, tok);
    for (int q = first; q < chunks; q += p.slots) {
        int members;
        const int adapter = take_chunk(c, 16 * MF, q, tok, members);
        const auto column_of = [&](int tile) { return n_block * span + (tile * LR_WAVES + w) * 64; };
        Tile<KS> b;
        Raw8<WIDE> raw[MF][2];
        const auto load_tile = [&](int n0) {
            if (adapter >= 0)
                b = load_b<KS>(p, adapter, n0, l16, lq);
            // (all of base before any output: out may be base, so that no load would pass a store)
            const auto base = [&](auto all_there) {
#pragma unroll
                for (int i = 0; i < MF; ++i) {
                    const int64_t m = m0 + c.list[min(i * 16 + l16, members - 1)];
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                        raw[i][g] = load8<WIDE, decltype(all_there)::value>(p.base, m * p.base_stride + n0 + 32 * g + 8 * lq,
                                                                            p.N - (n0 + 32 * g + 8 * lq));
                }
            };
            if (n0 + 64 <= p.N)
                base(std::true_type{});
            else
                base(std::false_type{});
        };
        if (column_of(0) < p.N)  // (on its way while z is laid out)
            load_tile(column_of(0));
        if (adapter >= 0)
            lay_out<BF16, KS, MF>(p, c, m0, members, adapter, zs, factor);
        __syncthreads();
        for (int tile = 0; tile < p.tiles; ++tile) {
            const int n0 = column_of(tile);
            if (n0 >= p.N)
                break;
            if (tile > 0)
                load_tile(n0);
            clear_past_rank(b, p.R, lq);
#pragma unroll
            for (int i = 0; i < MF; ++i) {
                if (i * 16 >= members)
                    break;
                const int t = i * 16 + l16;
                float v[2][8];
#pragma unroll
                for (int g = 0; g < 2; ++g)
                    to_fp32<WIDE>(raw[i][g], p.base_dtype == LORA_BF16, v[g]);
                if (adapter >= 0)
                    add_product<BF16, KS>(b, zs[i], factor[t], lane, v);
                if (t < members) {
                    const int64_t m = m0 + c.list[t];
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const int col = n0 + 32 * g + 8 * lq;
                        if (n0 + 64 <= p.N)
                            store8<true>(p.out, m * p.N + col, p.out_bf16, 8, v[g]);
                        else
                            store8<false>(p.out, m * p.N + col, p.out_bf16, p.N - col, v[g]);
                    }
                }
            }
        }
    }
}

// The same of many tokens, where base and out are of 16 bits, their rows begin at 16-byte boundaries and a window's lie within
// 2 GiB: both go through LDS, so that they are read and written by whole cache lines.  A wave has a ring of units of its own,
// 32 tokens by 64 columns of base each; what comes out lies in the unit's place before it is stored.  What is not there is asked
// for past the buffers' ends, which costs no memory access: every unit has the same number of memory operations, so that
// a wait can name the ones that it does not need.
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr int LE_UNIT = 4096, LE_SLOTS = 3, LE_MAX_WIDTH = 1 << 20;  // (256 rows of 2^20 16-bit numbers are 2^29 bytes)
constexpr int LE_NT = 2;  // base and out pass once: the caches are B's and z's (16384 rows: 256 -> 239 us)
constexpr uint32_t LE_BYTES = 0x80000000u, LE_OUT = 0x80000000u;
__device__ __forceinline__ rsrc_t lines_of(const void *p)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, LE_BYTES, 0x00020000);
}
__device__ __forceinline__ void dma_line(rsrc_t r, uint32_t lane_off, uint32_t off, uint8_t *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16, lane_off, off, 0, LE_NT);
}
template <bool BF16, int KS, int MF> __global__ __launch_bounds__(LR_THREADS) void lora_expand_lines_kernel(const ExpandArgs p)
{
    static_assert(MF == 2 || MF == 4, "units of two fragments");
    constexpr int HALVES = MF / 2;  // units of a tile of 64 columns
    __shared__ Chunks c;
    __shared__ u32x4 zs[MF][KS][NUMBERS<BF16>][64];
    __shared__ float factor[16 * MF];
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];  // rings [wave][slot]
    uint8_t *const my_ring = smem + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * LE_SLOTS * LE_UNIT;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int span = 64 * LR_WAVES * p.tiles, n_blocks = (p.N + span - 1) / span;
    int id = blockIdx.x;
    const int n_block = id % n_blocks;
    id /= n_blocks;
    const int first = id % p.slots;
    const int64_t m0 = (int64_t)(id / p.slots) * LR_WINDOW;
    const int n = (int)min((int64_t)LR_WINDOW, p.M - m0);
    const int n_first = n_block * span + w * 64, n_end = min(n_block * span + span, p.N);
    const int turned = (lane & 7) ^ (lane >> 4);  // this lane's 16-byte piece of a row, in even bands of 8 rows; odd ones: ^ 4
    const rsrc_t base = lines_of(reinterpret_cast<const uint16_t *>(p.base) + m0 * p.base_stride);
    const rsrc_t out = lines_of(reinterpret_cast<const uint16_t *>(p.out) + m0 * p.N);
    Token tok;
    const int chunks = find_chunks(c, p.ids, m0, n, p.L, 16 * MF, tok);
    for (int q = first; q < chunks; q += p.slots) {
        int members;
        const int adapter = take_chunk(c, 16 * MF, q, tok, members);
        const rsrc_t rb = lines_of(reinterpret_cast<const uint16_t *>(p.b) + (int64_t)max(adapter, 0) * p.N * p.R);
        uint32_t from[2 * MF], to[2 * MF];  // this lane's row of each band of 8 rows
#pragma unroll
        for (int b = 0; b < 2 * MF; ++b) {
            const int t = b * 8 + (lane >> 3), row = c.list[min(t, members - 1)];
            from[b] = t < members ? (uint32_t)row * (uint32_t)p.base_stride * 2 : LE_OUT;
            to[b] = t < members ? (uint32_t)row * (uint32_t)p.N * 2 : LE_OUT;
        }
        const auto at = [&](uint32_t row, int b, int n0) {  // 8 columns of it, or nowhere
            const int piece = (turned ^ (4 * (b & 1))) * 8;
            return n0 + piece < n_end ? row + piece * 2 : LE_OUT;
        };
        const auto load = [&](int half, int n0, int slot) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
                dma_line(base, at(from[half * 4 + b], b, n0), (uint32_t)n0 * 2, my_ring + slot * LE_UNIT + b * 1024);
        };
        const auto load_next = [&](int n0) {
            Tile<KS> t;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const int col = n0 + 32 * (f >> 1) + 8 * (l16 >> 2) + 4 * (f & 1) + (l16 & 3);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int r = s * 32 + lq * 8;
                    t.v[f][s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                    rb, col < n_end && r < p.R && adapter >= 0 ? ((uint32_t)col * p.R + r) * 2 : LE_OUT, 0, 0));
                }
            }
            return t;
        };
        constexpr int STEP = 64 * LR_WAVES;
        // (unit u: half u mod HALVES of tile u / HALVES)
#pragma unroll
        for (int u = 0; u < LE_SLOTS; ++u)
            load(u % HALVES, n_first + u / HALVES * STEP, u);
        Tile<KS> next = load_next(n_first);
        if (adapter >= 0)
            lay_out<BF16, KS, MF>(p, c, m0, members, adapter, zs, factor);
        wait_loads<0>();
        __syncthreads();
        int slot = 0;
#pragma unroll 1
        for (int n0 = n_first; n0 < n_end; n0 += STEP) {
            const Tile<KS> b = next;
            next = load_next(n0 + STEP);  // (a tile ahead: loads are done in order)
#pragma unroll
            for (int half = 0; half < HALVES; ++half) {
                // since the loads of this unit: the stores of the unit before them, loads and stores of two units, and of B those
                // at the beginnings of tiles (the counter ends at 63, where a wait would wait for nothing)
                constexpr int B_LOADS = 4 * KS;
                constexpr auto most = [](int tiles) { return 20 + tiles * B_LOADS < 63 ? 20 + tiles * B_LOADS : 62; };
                if (HALVES == 1)
                    wait_loads<most(3)>();
                else if (half == 0)
                    wait_loads<most(2)>();
                else
                    wait_loads<most(1)>();
                uint8_t *ring = my_ring + slot * LE_UNIT;
                if (half * 32 < members) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float v[2][8];
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            Raw8<false> raw;
                            raw.v[0] = *reinterpret_cast<const u32x4 *>(ring + i * 2048 + l16 * 128 + (((4 * g + lq) ^ (l16 >> 1)) << 4));
                            to_fp32<false>(raw, p.base_dtype == LORA_BF16, v[g]);
                        }
                        if (adapter >= 0)
                            add_product<BF16, KS>(b, zs[half * 2 + i], factor[half * 32 + i * 16 + l16], lane, v);
#pragma unroll
                        for (int g = 0; g < 2; ++g)
                            *reinterpret_cast<u32x4 *>(ring + i * 2048 + l16 * 128 + (((4 * g + lq) ^ (l16 >> 1)) << 4)) = pack8(p.out_bf16, v[g]);
                    }
                }
                u32x4 o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o[k] = *reinterpret_cast<const u32x4 *>(ring + k * 1024 + lane * 16);
                wait_loads<63>();  // (the unit's place has been read)
                load((half + LE_SLOTS) % HALVES, n0 + (half + LE_SLOTS) / HALVES * STEP, slot);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    __builtin_amdgcn_raw_buffer_store_b128(o[k], out, at(to[half * 4 + k], k, n0), (uint32_t)n0 * 2, LE_NT);
                slot = slot == LE_SLOTS - 1 ? 0 : slot + 1;
            }
        }
    }
}

// ---------------------------------------------------------------- which kernels
// Tokens of a chunk: 16 in a decode batch, whose adapters have few each; 32 and 64 for prompts, where a chunk's share of A and B
// is read again for each.
int chunk_frags(int64_t M) { return M <= LR_WINDOW ? 1 : M < 8192 ? 2 : 4; }
// Blocks that share a window's chunks: of a decode batch as many as there can be; of prompts as many as there are of one adapter
// and two more, or, while they do not fill the chip twice, as many as there can be (441 rows, 41 adapters 41 -> 16 us; 2048 rows
// of 4096 columns and 16 adapters with 8 more 33 -> 39).
int chunk_slots(const LoraArgs &a, int mf)
{
    const int64_t alone = (a.M <= LR_WINDOW ? a.M : LR_WINDOW) / (16 * mf), most = alone + 1 + a.L;
    if (a.M <= LR_WINDOW)
        return (int)(a.M < most ? a.M : most);
    const int64_t fill = 2 * 256 / ((a.M + LR_WINDOW - 1) / LR_WINDOW * ((a.N + 255) / 256));
    return (int)(fill < alone + 2 ? alone + 2 : fill < most ? fill : most);
}
struct Plan {
    int mf, nf, groups, slots, splits;
    int64_t windows;
};
Plan lora_plan(const LoraArgs &a)
{
    Plan p;
    const bool int8 = a.x_dtype == LORA_INT8;
    p.windows = (a.M + LR_WINDOW - 1) / LR_WINDOW;
    p.mf = chunk_frags(a.M);
    const int frags = (a.R + 15) / 16, most = int8 ? 2 : 4;
    p.nf = frags >= most ? most : frags >= 2 ? 2 : 1;
    p.groups = (frags + p.nf - 1) / p.nf;
    // a window's chunks: all of a decode batch at once, of prompts a few more than if they had one adapter
    p.slots = chunk_slots(a, p.mf);
    // K is split until the chips' CUs have something to do, and no wave has less than a unit
    const int64_t chunks = a.M <= LR_WINDOW ? (a.M < a.L + a.M / 16 ? a.M : a.L + a.M / 16) : a.M / (16 * p.mf);
    const int64_t units = (a.K + (int8 ? 127 : 63)) / (int8 ? 128 : 64);
    int64_t s = 512 / (chunks * p.groups > 0 ? chunks * p.groups : 1);
    s = s < units / LR_WAVES ? s : units / LR_WAVES;
    p.splits = (int)(s < 1 ? 1 : s > LR_MAX_SPLITS ? LR_MAX_SPLITS : s);
    return p;
}

constexpr int LR_MAX_DEVICES = 64;
// a launch with LDS bytes of dynamic LDS, for which the kernel's limit is raised once per device
template <auto KERNEL, int LDS, typename Args> hipError_t launch_with_lds(const Args &a, uint32_t blocks, hipStream_t s)
{
    static std::atomic<bool> done[LR_MAX_DEVICES];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && !(dev < LR_MAX_DEVICES && done[dev].load(std::memory_order_acquire))) {
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e == hipSuccess && dev < LR_MAX_DEVICES)
            done[dev].store(true, std::memory_order_release);
    }
    if (e != hipSuccess)
        return e;
    hipLaunchKernelGGL(KERNEL, dim3(blocks), dim3(LR_THREADS), LDS, s, a);
    return hipGetLastError();
}
template <bool BF16, bool INT8, int MF, int NF> hipError_t shrink(const ShrinkArgs &a, int64_t blocks, hipStream_t s)
{
    constexpr int SLOT = (2 * NF * (INT8 ? 2 : 1) + 2 * MF) * 1024, SLOTS = SLOT <= 4096 ? 4 : SLOT <= 10240 ? 2 : 1, LDS = LR_WAVES * SLOTS * SLOT;
    return launch_with_lds<&lora_shrink_kernel<BF16, INT8, MF, NF, SLOTS>, LDS>(a, (uint32_t)blocks, s);
}
template <bool BF16, bool INT8, int MF> hipError_t shrink_nf(int nf, const ShrinkArgs &a, int64_t blocks, hipStream_t s)
{
    if (nf == 1)
        return shrink<BF16, INT8, MF, 1>(a, blocks, s);
    if (nf == 2)
        return shrink<BF16, INT8, MF, 2>(a, blocks, s);
    if constexpr (!INT8)
        return shrink<BF16, INT8, MF, 4>(a, blocks, s);
    return hipErrorInvalidValue;
}
template <bool BF16, bool INT8> hipError_t shrink_mf(int mf, int nf, const ShrinkArgs &a, int64_t blocks, hipStream_t s)
{
    return mf == 1 ? shrink_nf<BF16, INT8, 1>(nf, a, blocks, s) : mf == 2 ? shrink_nf<BF16, INT8, 2>(nf, a, blocks, s)
                                                                          : shrink_nf<BF16, INT8, 4>(nf, a, blocks, s);
}
template <bool BF16, int MF> hipError_t expand_lines(const ExpandArgs &a, uint32_t blocks, hipStream_t s)
{
    constexpr int LDS = LR_WAVES * LE_SLOTS * LE_UNIT;
    if (a.R <= 32)
        return launch_with_lds<&lora_expand_lines_kernel<BF16, 1, MF>, LDS>(a, blocks, s);
    if (a.R <= 64)
        return launch_with_lds<&lora_expand_lines_kernel<BF16, 2, MF>, LDS>(a, blocks, s);
    return launch_with_lds<&lora_expand_lines_kernel<BF16, 4, 2>, LDS>(a, blocks, s);
}
template <bool BF16, bool WIDE, int MF> hipError_t expand_ks(const ExpandArgs &a, uint32_t blocks, hipStream_t s)
{
    const dim3 grid(blocks), block(LR_THREADS);
    if (a.R <= 32)
        hipLaunchKernelGGL((lora_expand_kernel<BF16, WIDE, 1, MF>), grid, block, 0, s, a);
    else if (a.R <= 64)
        hipLaunchKernelGGL((lora_expand_kernel<BF16, WIDE, 2, MF>), grid, block, 0, s, a);
    else if (a.R <= 128)
        hipLaunchKernelGGL((lora_expand_kernel<BF16, WIDE, 4, MF>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((lora_expand_kernel<BF16, WIDE, 8, (MF < 4 ? MF : 2)>), grid, block, 0, s, a);
    return hipGetLastError();
}
template <bool BF16, bool WIDE> hipError_t expand(int mf, const ExpandArgs &a, uint32_t blocks, hipStream_t s)
{
    return mf == 1 ? expand_ks<BF16, WIDE, 1>(a, blocks, s) : mf == 2 ? expand_ks<BF16, WIDE, 2>(a, blocks, s)
                                                                      : expand_ks<BF16, WIDE, 4>(a, blocks, s);
}

}  // namespace

size_t lora_workspace_bytes(const LoraArgs &a)
{
    return a.M == 0 ? 0 : (size_t)lora_plan(a).splits * (size_t)a.M * (size_t)a.R * 4;
}

hipError_t launch_lora_add(const LoraArgs &a, void *ws, hipStream_t s)
{
    if (a.M == 0)
        return hipSuccess;
    const Plan p = lora_plan(a);
    const bool bf16 = a.dtype == LORA_BF16, int8 = a.x_dtype == LORA_INT8;
    const ShrinkArgs sa{a.x, a.a, a.ids, reinterpret_cast<float *>(ws), a.M, a.x_stride, a.K, a.R, a.L, p.splits, p.slots, p.groups};
    const int64_t blocks = p.windows * p.slots * p.groups * p.splits;
    if (blocks * LR_THREADS > 0xffffffffll)
        return hipErrorInvalidValue;
    hipError_t e = bf16 ? (int8 ? shrink_mf<true, true>(p.mf, p.nf, sa, blocks, s) : shrink_mf<true, false>(p.mf, p.nf, sa, blocks, s))
                        : (int8 ? shrink_mf<false, true>(p.mf, p.nf, sa, blocks, s) : shrink_mf<false, false>(p.mf, p.nf, sa, blocks, s));
    if (e != hipSuccess)
        return e;
    // base and out by whole lines, where they are of 16 bits and their rows aligned, and a wave has two tiles at least (16384 rows
    // of 14336 columns 299 -> 256 us; 1021 rows of 4096, with one tile a wave, 15.7 -> 18.2; ranks past 128 leave too few registers
    // for a tile of B ahead: 305 -> 309)
    const bool lines = p.mf > 1 && a.R <= 128 && a.base_dtype != LORA_FP32 && a.N % 8 == 0 && a.base_stride % 8 == 0 && a.N <= LE_MAX_WIDTH &&
                       a.base_stride <= LE_MAX_WIDTH &&
                       (reinterpret_cast<uintptr_t>(a.base) | reinterpret_cast<uintptr_t>(a.out)) % 16 == 0;
    const int mf = a.R > (lines ? 64 : 128) && p.mf > 2 ? 2 : p.mf, slots = chunk_slots(a, mf);
    ExpandArgs ea{a.base, a.b, reinterpret_cast<const float *>(ws), a.xs, a.scaling, a.ids, a.out, a.M, a.base_stride, a.N, a.R, a.L,
                  (int16_t)p.splits, (int16_t)slots, 1, a.base_dtype, (int8_t)(a.out_dtype == LORA_BF16)};
    // a block's columns: the more, the seldomer z is laid out
    while (ea.tiles < 4 && a.M > LR_WINDOW && p.windows * slots * ((a.N + 256 * 2 * ea.tiles - 1) / (256 * 2 * ea.tiles)) >= 1024)
        ea.tiles *= 2;
    const int64_t n_blocks = (a.N + 256 * ea.tiles - 1) / (256 * ea.tiles), eb = p.windows * slots * n_blocks;
    if (eb * LR_THREADS > 0xffffffffll)
        return hipErrorInvalidValue;
    if (lines && ea.tiles > 1 && mf == 4)
        return bf16 ? expand_lines<true, 4>(ea, (uint32_t)eb, s) : expand_lines<false, 4>(ea, (uint32_t)eb, s);
    if (lines && ea.tiles > 1)
        return bf16 ? expand_lines<true, 2>(ea, (uint32_t)eb, s) : expand_lines<false, 2>(ea, (uint32_t)eb, s);
    if (a.base_dtype == LORA_FP32)
        return bf16 ? expand<true, true>(mf, ea, (uint32_t)eb, s) : expand<false, true>(mf, ea, (uint32_t)eb, s);
    return bf16 ? expand<true, false>(mf, ea, (uint32_t)eb, s) : expand<false, false>(mf, ea, (uint32_t)eb, s);
}

}  // namespace cam
