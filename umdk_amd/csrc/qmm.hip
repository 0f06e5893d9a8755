// G4: int8 matrix product with one scale per row of x and one per row of W (output channel):
//   out[m, n] = ((float)sum_k x[m, k] w[n, k]) * ws[n] * xs[m] + bias[n], rounded once to the output's type
// The sum is exact in int32 (K <= 131056: 2^14 K stays below 2^31), so neither the order of its parts nor a split of K
// changes a bit of the result.
#include <atomic>
#include <type_traits>

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
#pragma unroll
            for (int q = 0; q < 3; ++q)
                if (q < n)
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

// 16 bytes of consecutive outputs of one row, the first `left` outputs of them stored
template <int OUT> __device__ __forceinline__ void store16b(void *out, size_t at, const u32x4 v, int left)
{
    constexpr int SIZE = OUT == QMM_FP32 ? 4 : 2, CNT = 16 / SIZE;
    uint8_t *o = reinterpret_cast<uint8_t *>(out) + at * SIZE;
    if (left >= CNT) {
        __builtin_memcpy(o, &v, 16);
        return;
    }
#pragma unroll
    for (int q = 0; q < CNT - 1; ++q)
        if (q < left) {
            if constexpr (SIZE == 4)
                reinterpret_cast<uint32_t *>(o)[q] = v[q];
            else
                reinterpret_cast<uint16_t *>(o)[q] = (uint16_t)(v[q >> 1] >> (16 * (q & 1)));
        }
}

// ---------------------------------------------------------------- tiles
// BM x BN output tiles of WAVES_M x WAVES_N waves, k-steps of 128 bytes (whole cache lines) through LDS.  Direct
// global->LDS loads bring a k-step's rows; 16-byte chunks are XOR-swizzled by (row >> 1) & 7, so the 16 rows of a fragment
// read fall on different banks.  Loads are counted with vmcnt and published with a bare s_barrier, so that those of later
// steps stay in flight.  Two rings:
//   RING > 0: RING slots of both operands, the loads of step ks + RING - 1 issued at the start of step ks.  Small tiles:
//     nearly all of a block's share of K is in flight at once.
//   RING == 0: three slots of x and two of W (256 x 256: all of a CU's LDS).  x of the step after next is loaded from a
//     step's start on (its slot was last read in the step before), W from the step's middle on, once every wave holds
//     its W fragments in registers: one and a half to two steps in flight.
constexpr int QKB = 128;

template <int BM_, int BN_, int WAVES_M_, int WAVES_N_, int RING_> struct QTile {
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, NW = WAVES_M * WAVES_N;
    static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, IF = WM / 16, JF = WN / 16;
    static constexpr int A_LOADS = BM * QKB / 1024 / NW, W_LOADS = BN * QKB / 1024 / NW, LOADS = A_LOADS + W_LOADS;
    static constexpr int RING = RING_, A_SLOTS = RING ? RING : 3, W_SLOTS = RING ? RING : 2;
    static constexpr int A_BYTES = BM * QKB, W_BYTES = BN * QKB;
    static constexpr int LDS = A_SLOTS * A_BYTES + W_SLOTS * W_BYTES;
    static_assert(NW % 2 == 0, "the chunk swizzle of a wave's bands is one and the same");
    static_assert(A_LOADS * 1024 * NW == A_BYTES && W_LOADS * 1024 * NW == W_BYTES, "whole bands for every wave");
    static_assert(RING == 0 || (RING >= 3 && (RING - 2) * LOADS < 64), "vmcnt range");
};

// at most N of this wave's loads are in flight, and none of its LDS reads
template <int N> __device__ __forceinline__ void q_wait()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (7 << 4));
}
// the same for N = LEFT * LOADS, LEFT <= MOST steps that are still to come
template <int MOST, int LOADS> __device__ __forceinline__ void q_wait_steps(int left)
{
    if constexpr (MOST == 0) {
        q_wait<0>();
    } else {
        if (left >= MOST)
            q_wait<MOST * LOADS>();
        else
            q_wait_steps<MOST - 1, LOADS>(left);
    }
}
__device__ __forceinline__ void q_bar()  // a barrier that leaves loads in flight
{
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void q_dma(__amdgpu_buffer_rsrc_t r, uint32_t off, void *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16, off, 0, 0, 0);
}
// the same past the caches: W where it is read once
__device__ __forceinline__ void q_dma_nt(__amdgpu_buffer_rsrc_t r, uint32_t off, void *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16, off, 0, 0, 2);
}

// The tile of a block: blocks go round the 8 XCDs, so logical tiles are handed out such that those of one XCD are a run
// of consecutive ones, whose rows of x and W meet in that XCD's L2.
__device__ __forceinline__ int xcd_run(int id, int total)
{
    const int per = total >> 3, rest = total & 7, xcd = id & 7;
    return xcd * per + min(xcd, rest) + (id >> 3);
}

// ---------------------------------------------------------------- few rows
// 16 MF rows (8 for MF = 0) by 16 NF rows of W per block, over the whole of K: the waves take turns at units of 128 bytes
// of K, each with a ring of SLOTS units of its own in LDS, so that no wave waits for another before the end, where their
// sums meet in LDS and no other block is waited for.  What it reads, (MF + NF) 2 KB a unit, is what takes its time; a
// CU takes in about 60 GB/s this way (whole lines per load instruction; 16 rows x 64 bytes straight into registers: 30 to
// 45 GB/s, 8.1 against 6.7 us for one row, K = 7168, N = 4096, and 21.5 against 12.5 us for 64).
template <int MF, int NF, int NWV, int SLOTS, bool NT, int OUT>
__global__ __launch_bounds__(64 * NWV) void qmm_waves_kernel(const QmmArgs p, int mt, int nt)
{
#pragma clang fp contract(off)
    constexpr int MR = MF ? 16 * MF : 8, IF = MF ? MF : 1, F = IF * NF;  // rows, fragments of x, fragments of a block
    constexpr int XB = MR / 8, BANDS = 2 * NF + XB, SLOT = BANDS * 1024;
    static_assert(F * 1024 <= SLOTS * SLOT && (SLOTS - 1) * BANDS < 64, "sums where the ring was; vmcnt range");
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int tile = xcd_run(blockIdx.x, mt * nt), n0 = (tile / mt) * 16 * NF, K = p.K;
    const int64_t m0 = (int64_t)(tile % mt) * MR;
    uint8_t *ring = smem + w * SLOTS * SLOT;
    const int last_m = (int)min((int64_t)MR - 1, p.M - 1 - m0), last_n = min(16 * NF - 1, p.N - 1 - n0);
    const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p.x + m0 * K), (short)0, -1, 0x00020000);
    const auto rw =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p.w + (int64_t)n0 * K), (short)0, -1, 0x00020000);
    // a load instruction fills a band of 8 rows x 128 bytes: lane l row l / 8, chunk slot l % 8.  W's bands, then x's; rows
    // past the last are the last one again.
    uint32_t rows[BANDS];
#pragma unroll
    for (int b = 0; b < BANDS; ++b)
        rows[b] = b < 2 * NF ? (uint32_t)min(b * 8 + (lane >> 3), last_n) * (uint32_t)K
                             : (uint32_t)min((b - 2 * NF) * 8 + (lane >> 3), last_m) * (uint32_t)K;
    const int ca = ((lane & 7) ^ (lane >> 4)) << 4, cb = ca ^ 64;  // the chunk swizzle in even and in odd bands
    const int units = (K + QKB - 1) / QKB, mine = units > w ? (units - w + NWV - 1) / NWV : 0;
    auto load = [&](int t, int slot) {
        const int k = (w + t * NWV) * QKB;
        const uint32_t ka = (uint32_t)min(k + ca, K - 16), kb = (uint32_t)min(k + cb, K - 16);
#pragma unroll
        for (int b = 0; b < BANDS; ++b) {
            uint8_t *lds = ring + slot * SLOT + b * 1024;
            if (b < 2 * NF && NT)
                q_dma_nt(rw, rows[b] + ((b & 1) ? kb : ka), lds);
            else
                q_dma(b < 2 * NF ? rw : rx, rows[b] + ((b & 1) ? kb : ka), lds);
        }
    };
    i32x4 acc[IF][NF];
#pragma unroll
    for (int i = 0; i < IF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
            acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
        if (s < mine)
            load(s, s);
    const int frag = l16 * QKB + ((lg ^ (l16 >> 1)) << 4);
    const int xfrag = MF ? frag : (l16 & 7) * QKB + ((lg ^ ((l16 & 7) >> 1)) << 4);  // (8 rows: twice the same)
    int slot = 0;
#pragma unroll 1
    for (int t = 0; t < mine; ++t) {
        q_wait_steps<SLOTS - 1, BANDS>(mine - 1 - t);
        asm volatile("" ::: "memory");
        const uint8_t *at = ring + slot * SLOT;
        i32x4 wf[NF][2], xf[IF][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NF; ++j)
                wf[j][h] = *reinterpret_cast<const i32x4 *>(at + j * 2048 + (frag ^ (h * 64)));
#pragma unroll
            for (int i = 0; i < IF; ++i)
                xf[i][h] = *reinterpret_cast<const i32x4 *>(at + (NF + i) * 2048 + (xfrag ^ (h * 64)));
        }
        q_wait<63>();  // (the slot has been read)
        asm volatile("" ::: "memory");
        if (t + SLOTS < mine)
            load(t + SLOTS, slot);
        const int k = (w + t * NWV) * QKB;
        if (k + QKB > K) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (k + h * 64 + lg * 16 >= K) {
#pragma unroll
                    for (int j = 0; j < NF; ++j)
                        wf[j][h] = i32x4{0, 0, 0, 0};
                }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < IF; ++i)
#pragma unroll
                for (int j = 0; j < NF; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j][h], xf[i][h], acc[i][j], 0, 0, 0);
        slot = slot == SLOTS - 1 ? 0 : slot + 1;
    }
    // the wave's sums go where its ring was; fragment f is added up and written by wave f mod NWV
#pragma unroll
    for (int i = 0; i < IF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
            *reinterpret_cast<i32x4 *>(ring + (i * NF + j) * 1024 + lane * 16) = acc[i][j];
    constexpr int MINE = (F + NWV - 1) / NWV;
    float ws[MINE][4], bias[MINE][4], xs[MINE];
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        const int f = min(r * NWV + w, F - 1), n = n0 + 16 * (f % NF) + 4 * lg;
        xs[r] = p.xs[min(m0 + 16 * (f / NF) + l16, p.M - 1)];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            ws[r][q] = p.ws[min(n + q, p.N - 1)];
            bias[r][q] = p.bias ? p.bias[min(n + q, p.N - 1)] : 0.0f;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MINE; ++r) {
        const int f = r * NWV + w;
        if (f >= F)
            return;
        i32x4 t = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < NWV; ++v)
            t += *reinterpret_cast<const i32x4 *>(smem + v * SLOTS * SLOT + f * 1024 + lane * 16);
        const int row = 16 * (f / NF) + l16, n = n0 + 16 * (f % NF) + 4 * lg, left = p.N - n;
        float o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            o[q] = (float)t[q] * ws[r][q] * xs[r];
            if (p.bias)
                o[q] += bias[r][q];
        }
        if (row <= last_m && left > 0)
            store4<OUT>(p.out, (size_t)((m0 + row) * p.N + n), o, left);
    }
}

template <typename TC, int OUT>
__global__ __launch_bounds__(64 * TC::NW) void qmm_tile_kernel(const QmmArgs p, int mt, int nt)
{
#pragma clang fp contract(off)
    constexpr int NW = TC::NW, IF = TC::IF, JF = TC::JF, A_LOADS = TC::A_LOADS, W_LOADS = TC::W_LOADS, RING = TC::RING;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = w / TC::WAVES_N, wn = w % TC::WAVES_N;

    // an XCD's run of tiles, 8 row tiles by as many column tiles as it takes
    const int tile = xcd_run(blockIdx.x, mt * nt);
    constexpr int GM = 8;
    const int grp = tile / (GM * nt), rem = tile - grp * GM * nt;
    const int gm = min(GM, mt - grp * GM);
    const int64_t m0 = (int64_t)(grp * GM + rem % gm) * TC::BM;
    const int n0 = (rem / gm) * TC::BN;

    const int K = p.K, nk = (K + QKB - 1) / QKB;
    const int last_m = (int)min((int64_t)TC::BM - 1, p.M - 1 - m0), last_n = min(TC::BN - 1, p.N - 1 - n0);
    const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p.x + m0 * K), (short)0, -1, 0x00020000);
    const auto rw =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p.w + (int64_t)n0 * K), (short)0, -1, 0x00020000);
    // a load instruction of a wave fills a band of 8 rows x 128 bytes: lane l row l / 8, slot l % 8.  Rows past the last
    // are the last one again.
    uint32_t arow[A_LOADS], wrow[W_LOADS];
#pragma unroll
    for (int i = 0; i < A_LOADS; ++i)
        arow[i] = (uint32_t)min((i * NW + w) * 8 + (lane >> 3), last_m) * (uint32_t)K;
#pragma unroll
    for (int i = 0; i < W_LOADS; ++i)
        wrow[i] = (uint32_t)min((i * NW + w) * 8 + (lane >> 3), last_n) * (uint32_t)K;
    const int c16 = ((lane & 7) ^ ((4 * (w & 1) + (lane >> 4)) & 7)) << 4;  // (row >> 1) & 7 of band w: 4 w + l / 16
    // bytes past K: the last chunk again (the fragments of the last step are cleared there)
    auto k_off = [&](int ks) { return (uint32_t)min(ks * QKB + c16, K - 16); };
    auto load_a = [&](int ks, int slot) {
        const uint32_t k = k_off(ks);
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i)
            q_dma(ra, arow[i] + k, smem + slot * TC::A_BYTES + (i * NW + w) * 1024);
    };
    auto load_w = [&](int ks, int slot) {
        const uint32_t k = k_off(ks);
#pragma unroll
        for (int i = 0; i < W_LOADS; ++i)
            q_dma(rw, wrow[i] + k, smem + TC::A_SLOTS * TC::A_BYTES + slot * TC::W_BYTES + (i * NW + w) * 1024);
    };

    i32x4 acc[IF][JF];
#pragma unroll
    for (int i = 0; i < IF; ++i)
#pragma unroll
        for (int j = 0; j < JF; ++j)
            acc[i][j] = i32x4{0, 0, 0, 0};

    // byte of this lane's 16 in row l16 of a slot, for the first 64 bytes of a step (the others: bit 6 turned)
    const int frag = l16 * QKB + ((lg ^ (l16 >> 1)) << 4);
    auto a_frag = [&](int slot, int i, int h) {
        return *reinterpret_cast<const i32x4 *>(smem + slot * TC::A_BYTES + (wm * TC::WM + i * 16) * QKB + (frag ^ (h * 64)));
    };
    auto w_frag = [&](int slot, int j, int h) {
        return *reinterpret_cast<const i32x4 *>(smem + TC::A_SLOTS * TC::A_BYTES + slot * TC::W_BYTES +
                                                (wn * TC::WN + j * 16) * QKB + (frag ^ (h * 64)));
    };
    // The products of a step from its slots; middle() runs behind fragment row MIDDLE.  (One row earlier: M = 1021, N =
    // 5001, K = 5120 in 128 x 192 tiles 35.9 against 32.0 us, M = 2048, N = 4096, K = 7168 in 256 x 128 58.7 against 56.4;
    // the 128 x 128 tile, whose rows have few products, is 2% better off with it.)
    constexpr int MIDDLE = JF <= 2 ? IF / 2 - 1 : IF / 2;
    auto multiply = [&](int ks, int sa, int sw, bool last, auto middle) {
        i32x4 wf[JF][2], af[2][2];
#pragma unroll
        for (int j = 0; j < JF; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                wf[j][h] = w_frag(sw, j, h);
#pragma unroll
        for (int h = 0; h < 2; ++h)
            af[0][h] = a_frag(sa, 0, h);
        if (last) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (ks * QKB + h * 64 + lg * 16 >= K) {
#pragma unroll
                    for (int j = 0; j < JF; ++j)
                        wf[j][h] = i32x4{0, 0, 0, 0};
                }
        }
#pragma unroll
        for (int i = 0; i < IF; ++i) {
            if (i + 1 < IF) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    af[(i + 1) & 1][h] = a_frag(sa, i + 1, h);
            }
#pragma unroll
            for (int j = 0; j < JF; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j][h], af[i & 1][h], acc[i][j], 0, 0, 0);
            if (i == MIDDLE)
                middle();
        }
    };
    auto nothing = [] {};
    if constexpr (RING > 0) {
#pragma unroll
        for (int r = 0; r < RING - 1; ++r)
            if (r < nk) {
                load_a(r, r);
                load_w(r, r);
            }
        int slot = 0;
#pragma unroll 1
        for (int ks = 0; ks < nk; ++ks) {
            q_wait_steps<RING - 2, TC::LOADS>(nk - 1 - ks);
            q_bar();
            const int free_slot = slot == 0 ? RING - 1 : slot - 1;  // (read in the step before)
            if (ks + RING - 1 < nk) {
                load_a(ks + RING - 1, free_slot);
                load_w(ks + RING - 1, free_slot);
            }
            multiply(ks, slot, slot, ks == nk - 1, nothing);
            slot = slot == RING - 1 ? 0 : slot + 1;
        }
    } else {
        load_a(0, 0);
        load_w(0, 0);
        if (nk > 1) {
            load_a(1, 1);
            load_w(1, 1);
        }
        int sa = 0;
#pragma unroll 1
        for (int ks = 0; ks < nk - 2; ++ks) {
            q_wait<TC::LOADS>();
            q_bar();
            load_a(ks + 2, sa == 0 ? 2 : sa - 1);
            multiply(ks, sa, ks & 1, false, [&] {
                q_wait<63>();  // (no LDS read of this wave is under way: its W slot may be written)
                q_bar();
                load_w(ks + 2, ks & 1);
            });
            sa = sa == 2 ? 0 : sa + 1;
        }
        if (nk > 1) {
            q_wait<TC::LOADS>();
            q_bar();
            multiply(nk - 2, sa, nk & 1, false, nothing);
            sa = sa == 2 ? 0 : sa + 1;
        }
        q_wait<0>();
        q_bar();
        multiply(nk - 1, sa, (nk - 1) & 1, true, nothing);
    }

    // A lane holds row 16 i + l16 and, per j, the four consecutive columns 16 j + 4 lg + q.
    // Stored like that, an instruction writes 32 bytes of each of 16 rows, and all blocks end together: 12.7 us a
    // 256 x 256 tile.  So the wave turns its part round in LDS (the ring is done with), half its rows at a time, and
    // writes whole runs of WN columns: 4.4 us.
    constexpr int SIZE = OUT == QMM_FP32 ? 4 : 2, HROWS = TC::WM / 2, ROWB = TC::WN * SIZE, PITCH = ROWB + 16;
    constexpr int LPR = ROWB / 16;  // 16-byte pieces of a row
    static_assert(HROWS * PITCH * NW <= TC::LDS && HROWS % 16 == 0 && HROWS * LPR % 64 == 0, "the exchange area");
    uint8_t *mine = smem + w * HROWS * PITCH;
    const int nw0 = n0 + wn * TC::WN;
    float ws[JF][4], bias[JF][4], xs[IF];
#pragma unroll
    for (int j = 0; j < JF; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = min(nw0 + 16 * j + 4 * lg + q, p.N - 1);
            ws[j][q] = p.ws[c];
            bias[j][q] = p.bias ? p.bias[c] : 0.0f;
        }
#pragma unroll
    for (int i = 0; i < IF; ++i)
        xs[i] = p.xs[m0 + min(wm * TC::WM + 16 * i + l16, last_m)];
    q_wait<63>();
    q_bar();
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
        for (int i = 0; i < HROWS / 16; ++i)
#pragma unroll
            for (int j = 0; j < JF; ++j) {
                float v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    v[q] = (float)acc[hh * IF / 2 + i][j][q] * ws[j][q] * xs[hh * IF / 2 + i];
                    if (p.bias)
                        v[q] += bias[j][q];
                }
                store4<OUT>(mine + (16 * i + l16) * PITCH + (16 * j + 4 * lg) * SIZE, 0, v, 4);
            }
#pragma unroll
        for (int c = 0; c < HROWS * LPR / 64; ++c) {
            const int at = c * 64 + lane, row = at / LPR, col = (at % LPR) * (16 / SIZE);
            const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + row * PITCH + col * SIZE);
            const int m = wm * TC::WM + hh * HROWS + row, left = p.N - nw0 - col;
            if (m <= last_m && left > 0)
                store16b<OUT>(p.out, (size_t)((m0 + m) * p.N + nw0 + col), v, left);
        }
    }
}

// the dynamic LDS limit of a kernel, raised once per device
constexpr int Q_MAX_DEVICES = 64;
template <auto KERNEL, int LDS> hipError_t allow_lds()
{
    static std::atomic<bool> done[Q_MAX_DEVICES];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess || (dev < Q_MAX_DEVICES && done[dev].load(std::memory_order_acquire)))
        return e;
    e = hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e == hipSuccess && dev < Q_MAX_DEVICES)
        done[dev].store(true, std::memory_order_release);
    return e;
}

// ---------------------------------------------------------------- which kernel
// Every shape gives the same bits; they differ in how evenly their blocks fill the 256 CUs and in what a k-step of 128
// bytes costs: alone on a CU, and where two blocks fit one, for the pair.  The shape with the least
//   rounds x (k-steps x cost + a block's own overhead)
// is taken.  Costs in ns, measured on whole products of one and of several rounds (gaussian codes, K = 4096 and 7168):
struct QShape {
    int bm, bn;
    int step, pair;  // pair: two blocks at once on a CU (2 * step: only one fits, or two are no faster than in turn)
    int block;       // start and end of a block
};
enum { Q_W81, Q_W11, Q_W21, Q_W22, Q_W32, Q_W42, Q_W44, Q_T64, Q_T128X64, Q_T128, Q_T128X192, Q_T256X128, Q_T256, Q_SHAPES };
constexpr QShape Q_SHAPE[Q_SHAPES] = {
    {8, 16, 49, 80, 600},        {16, 16, 66, 110, 800},      {32, 16, 98, 196, 1200},     {32, 32, 136, 272, 1500},
    {48, 32, 161, 322, 1500},    {64, 32, 193, 386, 1500},    {64, 64, 274, 600, 2800},    {64, 64, 290, 500, 2000},
    {128, 64, 450, 740, 2500},   {128, 128, 580, 1040, 2500}, {128, 192, 660, 1320, 4000}, {256, 128, 840, 1680, 6000},
    {256, 256, 1430, 2860, 7000},
};

int q_choose(int64_t M, int64_t N, int64_t K)
{
    int best = 0;
    int64_t least = INT64_MAX;
    const int64_t steps = (K + QKB - 1) / QKB;
    for (int i = 0; i < Q_SHAPES; ++i) {
        const QShape &q = Q_SHAPE[i];
        const int64_t blocks = ((M + q.bm - 1) / q.bm) * ((N + q.bn - 1) / q.bn), rounds = (blocks + 255) / 256;
        const int64_t cost = (rounds / 2) * (steps * q.pair + 2 * q.block) + (rounds & 1) * (steps * q.step + q.block);
        if (cost < least) {
            least = cost;
            best = i;
        }
    }
    return best;
}

template <auto KERNEL, int LDS> hipError_t q_launch(const QmmArgs &a, int bm, int bn, int threads, hipStream_t s)
{
    const int64_t mt = (a.M + bm - 1) / bm, nt = (a.N + bn - 1) / bn;
    if (mt * nt * threads > 0xffffffff)  // (no output of that size fits the memory)
        return hipErrorInvalidValue;
    const hipError_t e = allow_lds<KERNEL, LDS>();
    if (e != hipSuccess)
        return e;
    hipLaunchKernelGGL(KERNEL, dim3((uint32_t)(mt * nt)), dim3(threads), LDS, s, a, (int)mt, (int)nt);
    return hipGetLastError();
}

template <int OUT, int BM, int BN, int WAVES_M, int WAVES_N, int RING> hipError_t q_tile(const QmmArgs &a, hipStream_t s)
{
    using TC = QTile<BM, BN, WAVES_M, WAVES_N, RING>;
    return q_launch<qmm_tile_kernel<TC, OUT>, TC::LDS>(a, BM, BN, 64 * TC::NW, s);
}
template <int OUT, int MF, int NF, int NWV, int SLOTS> hipError_t q_waves(const QmmArgs &a, hipStream_t s)
{
    constexpr int MR = MF ? 16 * MF : 8, LDS = NWV * SLOTS * (2 * NF + MR / 8) * 1024;
    // W past the caches where one block alone reads it
    if (a.M <= MR)
        return q_launch<qmm_waves_kernel<MF, NF, NWV, SLOTS, true, OUT>, LDS>(a, MR, 16 * NF, 64 * NWV, s);
    return q_launch<qmm_waves_kernel<MF, NF, NWV, SLOTS, false, OUT>, LDS>(a, MR, 16 * NF, 64 * NWV, s);
}

template <int OUT> hipError_t q_run(int shape, const QmmArgs &a, hipStream_t s)
{
    switch (shape) {
    case Q_W81:
        return q_waves<OUT, 0, 1, 8, 2>(a, s);
    case Q_W11:
        return q_waves<OUT, 1, 1, 8, 2>(a, s);
    case Q_W21:
        return q_waves<OUT, 2, 1, 4, 3>(a, s);
    case Q_W22:
        return q_waves<OUT, 2, 2, 8, 2>(a, s);
    case Q_W32:
        return q_waves<OUT, 3, 2, 8, 2>(a, s);
    case Q_W42:
        return q_waves<OUT, 4, 2, 4, 2>(a, s);
    case Q_W44:
        return q_waves<OUT, 4, 4, 4, 2>(a, s);
    case Q_T64:
        return q_tile<OUT, 64, 64, 2, 2, 5>(a, s);
    case Q_T128X64:
        return q_tile<OUT, 128, 64, 2, 2, 3>(a, s);
    case Q_T128:
        return q_tile<OUT, 128, 128, 2, 4, 0>(a, s);
    case Q_T128X192:
        return q_tile<OUT, 128, 192, 2, 4, 0>(a, s);
    case Q_T256X128:
        return q_tile<OUT, 256, 128, 4, 2, 0>(a, s);
    case Q_T256:
        return q_tile<OUT, 256, 256, 2, 4, 0>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_quant_matmul(const QmmArgs &a, hipStream_t s)
{
    if (a.M == 0)
        return hipSuccess;
    if (a.N < 1 || a.K < 16 || a.K % 16 || a.K > 131056)
        return hipErrorInvalidValue;
    const int shape = q_choose(a.M, a.N, a.K);
    switch (a.out_dtype) {
    case QMM_BF16:
        return q_run<QMM_BF16>(shape, a, s);
    case QMM_FP16:
        return q_run<QMM_FP16>(shape, a, s);
    case QMM_FP32:
        return q_run<QMM_FP32>(shape, a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace cam
