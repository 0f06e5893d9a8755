// A whole expert layer for 1 to 16 tokens, in two launches.  With x the tokens' rows, R the router, b the balance bias:
//   l = x R^T;  ids, gates = grouped routing of l (route_grouped.hip)
//   E_e(x) = W2_e (silu(g) * u),  (g, u) = halves of W1_e x
//   out[t] = sum_k gates[t, k] E_ids[t, k](x_t) + E_shared(x_t)
// The first kernel computes the logits.  In the second every block routes all tokens for itself (16 tokens are two a wave),
// and then streams weights.
//
// What bounds it is the stream of the weights of the experts that any token picked, each read once.  So the layout serves
// that stream: a wave multiplies 16 weight rows by all tokens at once (the tokens are the 16 columns of one matrix
// instruction: no permutation, no gathered rows; columns of tokens that did not pick the expert are never looked at), and
// what it multiplies them by stays in registers: the wave's share of x for all experts, of h = silu(g) * u for one item.  The 8
// waves of a block share a sum's products by units of 128 bytes of a weight row.  Each has a ring of 7 units (16 rows by 128
// bytes, whole cache lines) of its own in LDS, that loads past the registers refill, unit by unit, as it is used, past the ends
// of tiles and work items.  So some 110 KB are in flight on a CU all the time, and no wave waits for another before its
// tiles' sums meet; matrix and vector instructions are a tenth of what they could be.  (The same ring in
// registers made the compiler spill.)
//
// Work items are numbered, those of the first product (16 gate rows and their 16 up rows) before those of the second (some
// 16-row tiles of one expert's chunk of W2), and blocks take them in that order from a counter, one ahead: the last wave, the
// clerk, takes the tickets and says what they are while the others stream.  An item of the second product waits until the
// expert's h is whole.  That cannot lock: what it waits for are items with lower numbers, taken by blocks that run and
// never wait themselves, however many blocks the GPU holds at once and whatever else it runs.
//
// Sums are fp32 in an order that hangs on the shapes alone: a token's results are the same bits in any batch, on any
// schedule.  Each (token, pick) gets its own row of partial results; whoever adds the last one to a tile of the output sums
// them up, picks ascending.  h is held as three bf16 numbers, each the leading bits of what those before it leave out, so that
// all 24 bits of it go into the second product: one number would add 2^-8 roundings of I values to the result's own, two leave
// an error ten times that of the fp32 sums.  The matrix instructions for the others are hidden; that a wave holds a shorter run
// of h costs up to 4%.
//
// Measured: one token on 8 of 64 fp8 experts and a shared one of 7168 x 2048 (398 MB of weights) 95 us, of which 4.5 are the
// logits, 6 the routing, 4 until the first weights are there and some 10 the blocks' not ending together; 16 such tokens (44 to
// 56 experts, 2.0 to 2.5 GB) 383-395 us, 7.0 TB/s in the first product and 5.2 in the second, whose items' h comes behind
// their own first weights; 7 tokens on 6 of 160 bf16 experts of 5120 x 1408 (1.67 GB) 279 us; one token on 2 of 8 bf16 experts of
// 1024 x 512 26 us, all of it latency: two launches, the routing, an expert's h on its way from block to block.  (With two numbers
// of h and a third longer chunks 92, 378 and 275 us.)
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gmm.h"
#include "route_dev.h"

namespace cam {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;

// ---------------------------------------------------------------- sizes
constexpr int MD_WAVES = 8, MD_RING = 7, MD_BLOCKS = 256;
constexpr int MD_SLOT = 2048;  // bytes of a slot of the ring: 16 rows by 128 bytes
constexpr int MD_BATCH = 4;    // tiles of a wave between two meetings of the waves
constexpr int MD_MAX_PICKS = 16, MD_MAX_EXPERTS = 512, MD_MAX_ENTRIES = MD_MAX_TOKENS * MD_MAX_PICKS + 1;
// The longest run of h that a work item of the second product multiplies by: what the waves hold of it in MD_NUMBERS numbers of
// MD_STEPS matrix instructions each, 144 registers.
constexpr int MD_NUMBERS = 3, MD_STEPS = 12, MD_CHUNK = MD_WAVES * MD_STEPS * 32;
// Counters in the workspace, 64 bytes apart: the queue, the experts' h (finished pairs of tiles), the output's tiles.
constexpr int MD_CTR = 16, MD_CTR_READY = 1, MD_CTR_DONE = MD_CTR_READY + MD_MAX_ENTRIES;
constexpr int MD_COUNTERS = MD_CTR_DONE + MD_MAX_HIDDEN / 16;
constexpr uint32_t MD_OUT = 0x80000000u;  // an offset past every buffer here: loads give 0, stores nothing
constexpr int AUX_NT = 2, AUX_AGENT = 16;

// nonzero once a wait for an expert's h has given up (sticky; read and cleared by the host, moe_decode_sync_status)
__device__ int g_decode_sync_status;

struct Ws {
    int *ctr;
    float *logits;           // [T, E]
    uint16_t *h;             // [MD_NUMBERS][T, K + 1, width]
    float *part;             // [T, K + 1, chunks, H]
    uint32_t h_bytes, part_bytes;
};
struct Layout {
    size_t logits, h, part, total;
    uint32_t h_bytes, part_bytes;
    int width, chunks;
};
int md_chunks(int I) { return (I + MD_CHUNK - 1) / MD_CHUNK; }
Layout md_layout(const MoeDecodeArgs &a)
{
    const auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    Layout l;
    l.width = a.I > a.Is ? a.I : a.Is;
    l.chunks = md_chunks(l.width);
    l.h_bytes = (uint32_t)((size_t)MD_NUMBERS * a.T * (a.K + 1) * l.width * 2);
    l.part_bytes = (uint32_t)((size_t)a.T * (a.K + 1) * l.chunks * a.H * 4);
    l.logits = up((size_t)MD_COUNTERS * MD_CTR * 4);
    l.h = l.logits + up((size_t)a.T * a.E * 4);
    l.part = l.h + up(l.h_bytes);
    l.total = l.part + up(l.part_bytes);
    return l;
}

// ---------------------------------------------------------------- the router product
// Logits in 64 bits, rounded to fp32: which expert is picked must not hang on the order of a sum.  A block per expert
// and 4 tokens, 16 columns a thread, so that all loads are on their way at once (16 tokens a block: 8.8 us where 4 take 4.6); products of 16-bit values (and of those with fp32) are
// exact in 64 bits.  The kernel also clears the counters of the next one.
constexpr int MD_ROUTER_WAVES = 8, MD_ROUTER_TOKENS = 4, MD_ROUTER_RUNS = MD_MAX_HIDDEN / (MD_ROUTER_WAVES * 512);

struct RouterArgs {
    const uint16_t *x;
    const void *router;
    const uint8_t *active;
    float *logits;
    int *ctr;
    int T, E, H, router_fp32;
};

__global__ __launch_bounds__(MD_ROUTER_WAVES * 64) void moe_decode_router_kernel(const RouterArgs p)
{
    const int e = blockIdx.x, t0 = blockIdx.y * MD_ROUTER_TOKENS, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __shared__ double part[MD_ROUTER_WAVES][MD_ROUTER_TOKENS];
    float r[MD_ROUTER_RUNS][8];
    const int k0 = threadIdx.x * 8;
#pragma unroll
    for (int i = 0; i < MD_ROUTER_RUNS; ++i) {
        const int k = k0 + i * MD_ROUTER_WAVES * 512;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            r[i][j] = 0.0f;
        if (k < p.H) {
            if (p.router_fp32) {
                const f32x4 *v = reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(p.router) + (size_t)e * p.H + k);
                const f32x4 a = v[0], b = v[1];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    r[i][j] = j < 4 ? a[j & 3] : b[j & 3];
            } else {
                unpack_bf16x8(*reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(p.router) + (size_t)e * p.H + k), r[i]);
            }
        }
    }
    for (int i = (blockIdx.y * p.E + e) * MD_ROUTER_WAVES * 64 + threadIdx.x; i < MD_COUNTERS; i += gridDim.y * p.E * MD_ROUTER_WAVES * 64)
        p.ctr[i * MD_CTR] = 0;
    u32x4 v[MD_ROUTER_TOKENS][MD_ROUTER_RUNS];
#pragma unroll
    for (int t = 0; t < MD_ROUTER_TOKENS; ++t)
#pragma unroll
        for (int i = 0; i < MD_ROUTER_RUNS; ++i) {
            const int k = k0 + i * MD_ROUTER_WAVES * 512;
            v[t][i] = u32x4{0, 0, 0, 0};
            if (t0 + t < p.T && k < p.H)
                v[t][i] = *reinterpret_cast<const u32x4 *>(p.x + (size_t)(t0 + t) * p.H + k);
        }
#pragma unroll
    for (int t = 0; t < MD_ROUTER_TOKENS; ++t) {
        if (t0 + t < p.T) {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < MD_ROUTER_RUNS; ++i) {
                float x[8];
                unpack_bf16x8(v[t][i], x);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    sum = __builtin_fma((double)x[j], (double)r[i][j], sum);
            }
            sum = row_sum<64>(sum);
            if (lane == 0)
                part[w][t] = sum;
        }
    }
    __syncthreads();
    if (const int t = t0 + (int)threadIdx.x; (int)threadIdx.x < MD_ROUTER_TOKENS && t < p.T) {
        double sum = 0.0;
#pragma unroll
        for (int v = 0; v < MD_ROUTER_WAVES; ++v)
            sum += part[v][threadIdx.x];
        const bool on = !p.active || p.active[t];  // (a token without a logit has no experts)
        p.logits[(size_t)t * p.E + e] = on ? (float)sum : __builtin_nanf("");
    }
}

// ---------------------------------------------------------------- the experts
// A weight type: bytes of a value, values of a unit, matrix instructions (32 values deep) of a unit.
template <int WT> struct Weight {
    static constexpr int SIZE = WT == MD_BF16 ? 2 : 1, UNIT = 128 / SIZE, STEPS = UNIT / 32;
};
// the s-th 8 values (s < STEPS / 2) of 16 bytes, as bf16: exact
template <int WT> __device__ __forceinline__ bf16x8 values(const u32x4 v, int s)
{
    if constexpr (WT == MD_BF16) {
        return __builtin_bit_cast(bf16x8, v);
    } else {
        u32x4 r;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t d = v[2 * s + q];
            if constexpr (WT == MD_FP8) {
                r[2 * q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, 1.0f, false));
                r[2 * q + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, 1.0f, true));
            } else {
                r[2 * q] = f32x2_to_bf16x2((float)(int8_t)d, (float)(int8_t)(d >> 8));
                r[2 * q + 1] = f32x2_to_bf16x2((float)(int8_t)(d >> 16), (float)(int8_t)(d >> 24));
            }
        }
        return __builtin_bit_cast(bf16x8, r);
    }
}

__device__ __forceinline__ rsrc_t rsrc(const void *p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)bytes, 0x00020000);
}
// 16 bytes for each lane from r + off + at, into LDS at lds + 16 lane, past the caches: weights are read once
__device__ __forceinline__ void dma(rsrc_t r, uint32_t off, uint32_t at, uint8_t *lds)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16, off, at, 0, AUX_NT);
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename T> __device__ __forceinline__ T *uniform(T *p)
{
    const uint64_t u = (uint64_t)p;
    return (T *)((uint64_t)(uint32_t)uniform((int)(u >> 32)) << 32 | (uint32_t)uniform((int)(uint32_t)u));
}
template <typename T> __device__ __forceinline__ __attribute__((address_space(1))) T *gp(T *p)
{
    return (__attribute__((address_space(1))) T *)p;
}
__device__ __forceinline__ int ctr_add(int *p, int v)
{
    return __hip_atomic_fetch_add(gp(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ int ctr_load(int *p)
{
    return __hip_atomic_load(gp(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void lds_barrier()  // a barrier that leaves loads in flight
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

struct DecodeArgs {
    MoeDecodeArgs p;
    RouteGroupedArgs r;  // one token's routing by a wave
    int route_per, width, chunks;
    Ws ws;
    uint32_t wait_ticks;  // the bound of a wait for h
    int unreachable;      // 1: a test makes every wait give up
};

// A work item.  phase 1: a pair of 16-row tiles (gate, up) of an entry's first matrix; 2: `count` tiles of a chunk of its
// second; 0: none.
struct Item {
    int phase, entry, tile, count;
    int lkw, k0, units, chunk;  // log2 of the waves that share a tile's sum; the chunk's first unit, its units
    uint32_t row_bytes, step;   // step: rows from a gate tile to its up tile, or from a wave's tile to its next one
    const char *w;
    const float *s;             // the matrix's scales
};

// How the tiles of the second product make up items: first the shared expert's parts (chunks of it), `run` tiles an item, then
// the other entries' parts, the last of them by fewer tiles.
struct Split {
    int run_s, runs_s, items_s;   // the shared expert's tiles an item, items a part, items
    int run, runs, big, items_b;  // the first `big` other parts' tiles an item, items a part, items
    int run_e, runs_e;            // the rest's tiles an item, items a part
};

// What the streams need of the arguments, in LDS: in scalar registers it would crowd out what they work with.
struct Late {
    const void *w1, *w2, *sw1, *sw2;
    const float *s1, *s2, *ss1, *ss2;
    uint16_t *out, *h;
    float *part;
    int *ctr;
    int I, Is, K, width, chunks;
    uint32_t h_bytes, part_bytes, wait_ticks;
    int unreachable;
};

// LDS.  red: what the waves have summed up of their tiles.
struct Shared {
    uint8_t ring[MD_WAVES][MD_RING][MD_SLOT];
    f32x4 red[MD_WAVES][MD_BATCH][64];
    uint32_t expert_mask[MD_MAX_EXPERTS];
    int16_t expert_entry[MD_MAX_EXPERTS];
    int16_t ids[MD_MAX_TOKENS][MD_MAX_PICKS];
    float gates[MD_MAX_TOKENS][MD_MAX_PICKS];
    uint8_t lost[MD_MAX_TOKENS];  // an active token without an expert whose row is not finite: its results are NaN, not empty sums
    int16_t entry_expert[MD_MAX_ENTRIES];
    uint16_t entry_mask[MD_MAX_ENTRIES];
    uint8_t entry_pick[MD_MAX_ENTRIES][MD_MAX_TOKENS];
    int wave_count[MD_WAVES], known;
    Item item[2];
    Split split;
    Late a;
};
static_assert(sizeof(Shared) <= 160 * 1024, "a CU's LDS");

// f(0), f(1), ... f(n - 1) with constants, n <= N.  (One jump past the rest: code that is only skipped costs its fetch.)
template <int N, int I = 0, typename F> __device__ __forceinline__ void upto(int n, F &&f)
{
    if constexpr (I < N) {
        if (I < n) {
            f(std::integral_constant<int, I>{});
            upto<N, I + 1>(n, f);
        }
    }
}

// at most N of this wave's memory operations are in flight
template <int N> __device__ __forceinline__ void wait_loads()
{
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | 0xF70);
    asm volatile("" ::: "memory");
}
// the oldest of `ahead` slots' loads, two each, has arrived
template <int MOST> __device__ __forceinline__ void wait_slot(int ahead)
{
    if constexpr (MOST <= 1) {
        wait_loads<0>();
    } else {
        if (ahead >= MOST)
            wait_loads<2 * (MOST - 1)>();
        else
            wait_slot<MOST - 1>(ahead);
    }
}

template <int WT> __global__ __launch_bounds__(MD_WAVES * 64) void moe_decode_kernel(const DecodeArgs args)
{
    using W = Weight<WT>;
    constexpr int PIECES = 16 / W::SIZE / 8;               // steps of 16 bytes
    constexpr int U1 = MD_MAX_HIDDEN / W::UNIT / MD_WAVES;  // a wave's units of a row of the first matrix at most
    constexpr int U2 = MD_STEPS / W::STEPS;                 // and of a chunk of the second
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    Shared &sh = *reinterpret_cast<Shared *>(smem);
    const Late &a = sh.a;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
    const int w = uniform((int)threadIdx.x >> 6);
    const int T = args.p.T, H = args.p.H;
    const bool nshared = args.p.Is > 0;

    // The last wave is the block's clerk: it takes the tickets and says what their items are.  (The first two are on their way
    // while the tokens are routed, by other waves where there are few; otherwise the second is not asked for before the clerk's
    // tokens' logits, which would come after it: 2 us of 44.)
    const bool clerk = w == MD_WAVES - 1;
    int ticket = 0, ticket2 = 0;
    if (clerk && lane == 0) {
        ticket = ctr_add(args.ws.ctr, 1);
        if (T < MD_WAVES)
            ticket2 = ctr_add(args.ws.ctr, 1);
    }
    int entries;
    uint32_t on;  // the tokens that are active
    {
        const MoeDecodeArgs &p = args.p;
        const int K = p.K;
        // ---- routing (picks by reductions, here not by the heads of sorted lists where there are many: 256 experts, 8 picks, one
        // token 32.2 us in all, by heads 30.6)
        for (int i = threadIdx.x; i < MD_MAX_EXPERTS; i += MD_WAVES * 64)
            sh.expert_mask[i] = 0;
        for (int t = w; t < T; t += MD_WAVES) {
            int idx = -1;
            double gate = 0.0;
            const char *row = reinterpret_cast<const char *>(args.ws.logits + (size_t)t * p.E);
            if (args.route_per == 1)
                route_token<64, 1, RG_EACH>(args.r, row, lane, idx, gate);
            else if (args.route_per == 4)
                route_token<64, 4, RG_EACH>(args.r, row, lane, idx, gate);
            else
                route_token<64, 16, RG_EACH>(args.r, row, lane, idx, gate);
            if (lane < K) {
                const float g = (float)(gate * (double)p.scaling);
                sh.ids[t][lane] = (int16_t)idx;
                sh.gates[t][lane] = g;
                if (blockIdx.x == 0) {
                    p.topk_idx[t * K + lane] = idx;
                    p.topk_w[t * K + lane] = g;
                }
            }
            bool lost = false;
            if (uniform(idx) < 0 && (!p.active || p.active[t])) {
                for (int k = lane * 8; k < H; k += 512) {
                    const u32x4 v = *reinterpret_cast<const u32x4 *>(p.x + (size_t)t * H + k);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        lost |= (v[q] & 0x7f80u) == 0x7f80u || (v[q] & 0x7f800000u) == 0x7f800000u;
                }
                lost = __ballot(lost) != 0;
            }
            if (lane == 0)
                sh.lost[t] = lost;
        }
        if (clerk && lane == 0 && T >= MD_WAVES)
            ticket2 = ctr_add(args.ws.ctr, 1);
        if (threadIdx.x == MD_WAVES * 64 - 1)
            sh.a = Late{p.w1,         p.w2,        p.sw1, p.sw2, p.s1, p.s2,       p.ss1,       p.ss2,           p.out,             args.ws.h,
                        args.ws.part, args.ws.ctr, p.I,   p.Is,  p.K,  args.width, args.chunks, args.ws.h_bytes, args.ws.part_bytes,
                        args.wait_ticks, args.unreachable};
        __syncthreads();
        if ((int)threadIdx.x < T * K) {
            const int t = threadIdx.x / K, e = sh.ids[t][threadIdx.x % K];
            if (e >= 0)
                atomicOr(&sh.expert_mask[e], 1u << t);
        }
        __syncthreads();
        // the entries: the shared expert, then the experts that any token picked, ascending
        const uint32_t mask = sh.expert_mask[threadIdx.x];  // (as many threads as experts at most)
        const uint64_t some = __ballot(mask != 0);
        if (lane == 0)
            sh.wave_count[w] = __popcll(some);
        __syncthreads();
        int before = nshared, all = nshared;
#pragma unroll
        for (int v = 0; v < MD_WAVES; ++v) {
            before += v < w ? sh.wave_count[v] : 0;
            all += sh.wave_count[v];
        }
        if (mask) {
            const int d = before + __popcll(some & lanemask_lt());
            sh.entry_expert[d] = (int16_t)threadIdx.x;
            sh.entry_mask[d] = (uint16_t)mask;
            sh.expert_entry[threadIdx.x] = (int16_t)d;
        }
        on = (1u << T) - 1;
        if (p.active)
            on = (uint32_t)__ballot(lane < T && p.active[min(lane, T - 1)]);
        if (nshared && threadIdx.x == 0)
            sh.entry_mask[0] = (uint16_t)on;
        __syncthreads();
        if ((int)threadIdx.x < T * K) {
            const int t = threadIdx.x / K, k = threadIdx.x % K, e = sh.ids[t][k];
            if (e >= 0)
                sh.entry_pick[sh.expert_entry[e]][t] = (uint8_t)k;
        }
        if (nshared && (int)threadIdx.x < T)
            sh.entry_pick[0][threadIdx.x] = (uint8_t)K;
        entries = uniform(all);
        if (entries == 0) {  // nobody has an expert
            for (int i = blockIdx.x * MD_WAVES * 64 + threadIdx.x; i < T * H / 4; i += gridDim.x * MD_WAVES * 64)
                reinterpret_cast<u32x2 *>(p.out)[i] = sh.lost[i / (H / 4)] ? u32x2{0x7fc07fc0u, 0x7fc07fc0u} : u32x2{0, 0};
            return;
        }
    }

    // ---- the items
    const uint32_t row1 = (uint32_t)(H * W::SIZE);  // bytes of a row of the first matrix
    const auto chunks_of = [](int I) { return (I + MD_CHUNK - 1) / MD_CHUNK; };
    const auto log_waves = [](int units) {  // that share a tile of so many units: the fewer, the more tiles are done at once
        return units > 4 * U2 ? 3 : units > 2 * U2 ? 2 : units > U2 ? 1 : 0;
    };
    const auto first_items = [&] {  // how many items the first product has
        return (nshared ? uniform(a.Is) / 16 : 0) + (entries - nshared) * (uniform(a.I) / 16);
    };
    if (w == MD_WAVES - 2 || (clerk && uniform(ticket) >= first_items())) {  // (the clerk where it needs it at once: the same numbers)
        // An item costs about what 100 KB more of weights would (4 us: h, a meeting of the waves, the parts' way to memory).  Of
        // 1 to 32 tiles an item and 1 to 8 of the shared expert's the cheapest, a lane each: what the blocks' share of all items
        // costs, and half of the largest for their not ending together.  (A wave's four tiles between two meetings at most, but 8 in
        // any case.)
        constexpr int ITEM_COST = 100;  // KB
        const int I0 = uniform(a.I), Is = uniform(a.Is), tiles = H / 16;
        const int C0 = chunks_of(I0), Cs = nshared ? chunks_of(Is) : 0, parts = (entries - nshared) * C0;
        const auto most = [&](int I, int C) {
            const int units = (I * W::SIZE + 127) / 128;
            return max(8, 32 >> log_waves((units + C - 1) / C));
        };
        const int kb = parts ? 16 * I0 * W::SIZE / C0 >> 10 : 0, kb_s = Cs ? 16 * Is * W::SIZE / Cs >> 10 : 0;  // a tile's
        const int log = min(lane & 7, 5), log_s = Cs ? lane >> 3 & 3 : 0, run = 1 << log, run_s = 1 << log_s;
        const int runs_s = (tiles + run_s - 1) >> log_s, runs = (tiles + run - 1) >> log;
        const int items_s = Cs * runs_s, items_0 = parts * runs, items = items_s + items_0;
        const int one_s = ITEM_COST + run_s * kb_s, one = ITEM_COST + run * kb;
        int cost = items <= MD_BLOCKS ? max(one, one_s) : (items_s * one_s + items_0 * one) / MD_BLOCKS + max(one, one_s) / 2;
        if (run > (parts ? most(I0, C0) : 1))
            cost = 0x3ffffff;
        int least = cost << 5 | (lane & 31);
#pragma unroll
        for (int d = 1; d < 32; d *= 2)
            least = min(least, __shfl_xor(least, d, 64));
        if (lane == (least & 31)) {
            Split v;
            v.run_s = run_s;
            v.runs_s = runs_s;
            v.items_s = items_s;
            v.run = run;
            v.runs = runs;
            v.big = items > MD_BLOCKS && run > 1 ? parts - parts / 4 : parts;  // (so that the blocks end together)
            v.items_b = v.big * v.runs;
            v.run_e = max(run / 2, 1);
            v.runs_e = (tiles + v.run_e - 1) >> max(log - 1, 0);
            sh.split = v;
        }
    }
    // the item of the clerk's ticket, for all to read
    const auto describe = [&](int slot) {
        const int q = uniform(ticket), I0 = uniform(a.I), Is = uniform(a.Is);
        const int per1 = I0 / 16, per1s = nshared ? Is / 16 : 0, N1 = per1s + (entries - nshared) * per1;
        Item it{};
        if (q < N1) {
            const bool shared = q < per1s;
            const int I = shared ? Is : I0, at = q - per1s, d = shared ? 0 : nshared + at / per1;
            const int e = shared ? 0 : uniform(sh.entry_expert[d]);
            it.phase = 1;
            it.entry = d;
            it.tile = shared ? q : at % per1;
            it.count = 2;
            it.lkw = 3;
            it.units = ((int)row1 + 127) / 128;
            it.row_bytes = row1;
            it.step = (uint32_t)I;
            it.w = reinterpret_cast<const char *>(shared ? a.sw1 : a.w1) + (size_t)e * (size_t)(2 * I) * row1;
            if constexpr (WT == MD_FP8)
                it.s = (shared ? a.ss1 : a.s1) + (size_t)e * (2 * I / 128) * (H / 128);
            if constexpr (WT == MD_INT8)
                it.s = (shared ? a.ss1 : a.s1) + (size_t)e * 2 * I;
        } else {
            const int C0 = chunks_of(I0), Cs = nshared ? chunks_of(Is) : 0, parts = Cs + (entries - nshared) * C0;
            const Split &v = sh.split;
            const int items_s = uniform(v.items_s), items_b = uniform(v.items_b);
            int at = q - N1, c = 0, run, runs;
            if (at < items_s) {
                run = uniform(v.run_s);
                runs = uniform(v.runs_s);
            } else if (at -= items_s; at < items_b) {
                run = uniform(v.run);
                runs = uniform(v.runs);
                c = Cs;
            } else {
                at -= items_b;
                run = uniform(v.run_e);
                runs = uniform(v.runs_e);
                c = Cs + uniform(v.big);
            }
            c += at / runs;
            at %= runs;
            if (c < parts) {
                const bool shared = c < Cs;
                const int I = shared ? Is : I0, C = shared ? Cs : C0, d = shared ? 0 : nshared + (c - Cs) / C0;
                const int e = shared ? 0 : uniform(sh.entry_expert[d]);
                const int units = (I * W::SIZE + 127) / 128, cu = (units + C - 1) / C;
                it.phase = 2;
                it.entry = d;
                it.chunk = shared ? c : (c - Cs) % C0;
                it.tile = at * run;
                it.count = min(run, H / 16 - it.tile);
                it.lkw = log_waves(cu);
                it.k0 = it.chunk * cu;
                it.units = min(cu, units - it.k0);
                it.row_bytes = (uint32_t)(I * W::SIZE);
                it.step = 128u >> it.lkw;
                it.w = reinterpret_cast<const char *>(shared ? a.sw2 : a.w2) + (size_t)e * (size_t)H * it.row_bytes;
                if constexpr (WT == MD_FP8)
                    it.s = (shared ? a.ss2 : a.s2) + (size_t)e * (H / 128) * (I / 128);
                if constexpr (WT == MD_INT8)
                    it.s = (shared ? a.ss2 : a.s2) + (size_t)e * H;
            }
        }
        if (lane == 0)
            sh.item[slot] = it;
    };
    const auto read_item = [&](int slot) -> Item {
        const Item &v = sh.item[slot];
        Item it;
        it.phase = uniform(v.phase);
        it.entry = uniform(v.entry);
        it.tile = uniform(v.tile);
        it.count = uniform(v.count);
        it.lkw = uniform(v.lkw);
        it.k0 = uniform(v.k0);
        it.units = uniform(v.units);
        it.chunk = uniform(v.chunk);
        it.row_bytes = (uint32_t)uniform((int)v.row_bytes);
        it.step = (uint32_t)uniform((int)v.step);
        it.w = uniform(v.w);
        it.s = uniform(v.s);
        return it;
    };
    const auto take = [&] {
        if (clerk && lane == 0)
            ticket = ctr_add(a.ctr, 1);
    };
    // this wave's share of an item: units of a tile, tiles
    const auto units_of = [&](const Item &it) { return (it.units - (w & ((1 << it.lkw) - 1)) + (1 << it.lkw) - 1) >> it.lkw; };
    const auto tiles_of = [&](const Item &it) {
        const int wr = w >> it.lkw, at_once = 8 >> it.lkw;
        return it.phase == 0 ? 0 : (it.count - wr + at_once - 1) >> (3 - it.lkw);
    };

    // ---- the ring.  A load instruction brings 8 rows by 128 bytes (whole cache lines): lane l 16 bytes of row l / 8, into
    // the l-th 16 bytes of half a slot.  Which 16 of the row's 128: l mod 8, turned by (row / 2) mod 8, so that the 16 rows of
    // an operand fall on different banks.
    uint8_t *const my_ring = sh.ring[w][0];
    const int turned = (lane & 7) ^ (lane >> 4), frag = l16 * 128 + ((lq ^ (l16 >> 1)) << 4);
    int ahead = 0, in_slot = 0, out_slot = 0;  // slots filled or being filled; the next to fill, to use
    struct {                                   // what the next slot to fill holds
        const char *w;
        uint32_t off, first, tile_step, unit_step, row_bytes;
        int units, unit, tiles;                // tiles: left, with this one
        uint32_t lane_off;
        int which;                             // 0: of the current item, 1: of the next, 2: of one not yet known
    } in;
    const auto stream = [&](const Item &it) {
        in.units = units_of(it);
        in.tiles = in.units > 0 ? tiles_of(it) : 0;
        in.unit = 0;
        in.row_bytes = it.row_bytes;
        in.w = it.w;
        in.unit_step = 128u << it.lkw;
        in.first = (uint32_t)(it.k0 + (w & ((1 << it.lkw) - 1))) * 128u;
        in.off = (uint32_t)(it.tile * 16 + (it.phase == 2 ? (w >> it.lkw) * 16 : 0)) * it.row_bytes + in.first;
        in.tile_step = it.step * it.row_bytes;
        in.lane_off = (uint32_t)(lane >> 3) * it.row_bytes;
    };
    Item cur, nxt;
    const auto fill = [&] {  // (in.tiles > 0, ahead < MD_RING)
        const rsrc_t r = rsrc(in.w, 0xffffffffu);
        uint8_t *lds = my_ring + in_slot * MD_SLOT;
        int c0 = turned, c1 = turned ^ 4;
        if (WT == MD_INT8 && in.first + in.unit * in.unit_step + 64 >= in.row_bytes) {  // (a row may end within a unit)
            c0 &= 3;
            c1 &= 3;
        }
        const uint32_t at = in.off + in.unit * in.unit_step;
        dma(r, in.lane_off + c0 * 16, at, lds);
        dma(r, in.lane_off + 8 * in.row_bytes + c1 * 16, at, lds + 1024);
        in_slot = in_slot == MD_RING - 1 ? 0 : in_slot + 1;
        ++ahead;
        if (++in.unit == in.units) {
            in.unit = 0;
            in.off += in.tile_step;
            if (--in.tiles == 0 && in.which == 0) {
                in.which = 1;
                stream(nxt);
            }
        }
    };
    const auto top_up = [&] {
        while (ahead < MD_RING && in.tiles > 0)
            fill();
    };
    // the next slot's products with x, or with the numbers of h (step by step), added to acc; the slot is filled again
    const auto use = [&](const u32x4 *x, auto numbers, float s, bool half, f32x4 &acc) {
        constexpr int NUMBERS = decltype(numbers)::value;
        wait_slot<MD_RING>(ahead);
        const uint8_t *at = my_ring + out_slot * MD_SLOT;
        u32x4 v[2];
        v[0] = *reinterpret_cast<const u32x4 *>(at + frag);
        v[1] = *reinterpret_cast<const u32x4 *>(at + (frag ^ 64));
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v[0]), "+v"(v[1])::"memory");  // (the slot has been read)
        out_slot = out_slot == MD_RING - 1 ? 0 : out_slot + 1;
        --ahead;
        if (in.tiles > 0)
            fill();
        if (WT == MD_INT8 && half)
            v[1] = u32x4{0, 0, 0, 0};
        f32x4 sum = WT == MD_FP8 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc;
#pragma unroll
        for (int i = 0; i < W::STEPS; ++i) {
            const bf16x8 b = values<WT>(v[i / PIECES], i % PIECES);
#pragma unroll
            for (int k = 0; k < NUMBERS; ++k)
                sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, __builtin_bit_cast(bf16x8, x[i * NUMBERS + k]), sum, 0, 0, 0);
        }
        if constexpr (WT == MD_FP8) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                acc[q] = __builtin_fmaf(s, sum[q], acc[q]);
        } else {
            acc = sum;
        }
    };
    const auto scale = [&](const float *s, int at) {  // (by a scalar load)
        return reinterpret_cast<const __attribute__((address_space(4))) float *>((uintptr_t)s)[at];
    };

    if (clerk)
        describe(0);
    __syncthreads();
    cur = read_item(0);
    int turn = 0;  // the place of the current item, where the one after the next goes
    in.which = 0;
    stream(cur);
    nxt.phase = 0;
    nxt.w = cur.w;
    nxt.s = cur.s;
    nxt.entry = nxt.tile = nxt.count = nxt.lkw = nxt.k0 = nxt.units = nxt.chunk = 0;
    nxt.row_bytes = nxt.step = 0;
    top_up();  // (all there is of it: the next item is not known yet)
    if (clerk) {
        ticket = ticket2;
        describe(1);
    }
    lds_barrier();
    nxt = read_item(1);
    if (in.tiles == 0) {
        in.which = 1;
        stream(nxt);
    }
    const auto advance = [&] {
        cur = nxt;
        nxt = read_item(turn);
        turn ^= 1;
        in.which = in.which == 0 ? 0 : in.which - 1;
        if (in.tiles == 0) {  // (all of the item that is now the current one has been asked for)
            in.which = 1;
            stream(nxt);
        }
        top_up();
    };

    // ---- the first product
    if (cur.phase == 1) {
        const int units = units_of(cur);  // the same for all of these items
        // the wave's share of x: 32 columns each
        u32x4 x[U1 * W::STEPS];
        {
            const rsrc_t rx = rsrc(args.p.x, (uint32_t)(T * H * 2));
#pragma unroll
            for (int i = 0; i < U1 * W::STEPS; ++i)
                x[i] = u32x4{0, 0, 0, 0};
            if (l16 < T) {  // (lanes that ask for nothing cost nothing)
                upto<U1>(units, [&](auto c) {
                    constexpr int u = decltype(c)::value;
#pragma unroll
                    for (int st = 0; st < W::STEPS; ++st) {
                        const int col = (w + u * 8) * W::UNIT + (16 / W::SIZE) * (4 * (st / PIECES) + lq) + 8 * (st % PIECES);
                        x[u * W::STEPS + st] = __builtin_amdgcn_raw_buffer_load_b128(rx, col < H ? (l16 * H + col) * 2 : MD_OUT, 0, 0);
                    }
                });
            }
        }
        wait_loads<0>();
        while (cur.phase == 1) {
            take();
            float s[2][U1];  // the scales of the gate rows and of the up rows
            if constexpr (WT == MD_FP8) {
#pragma unroll
                for (int u = 0; u < U1; ++u) {
                    const int at = min(w + 8 * u, H / 128 - 1);
                    s[0][u] = scale(cur.s, (cur.tile >> 3) * (H / 128) + at);
                    s[1][u] = scale(cur.s, ((cur.tile + (int)cur.step / 16) >> 3) * (H / 128) + at);
                }
            }
            f32x4 acc[2];  // (the loops' code is kept short: what runs for the first time comes from memory)
#pragma unroll 1
            for (int j = 0; j < 2; ++j) {
                acc[0] = acc[1];
                acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
                upto<U1>(units, [&](auto c) {
                    constexpr int u = decltype(c)::value;
                    use(x + u * W::STEPS, std::integral_constant<int, 1>{}, WT == MD_FP8 ? s[0][u] : 0.f, (uint32_t)(w + 8 * u) * 128 + 64 >= row1, acc[1]);
                });
                if constexpr (WT == MD_FP8) {
#pragma unroll
                    for (int u = 0; u < U1; ++u)
                        s[0][u] = s[1][u];
                }
            }
            if (clerk)
                describe(turn);
            lds_barrier();  // (the last sums have been read)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                sh.red[w][j][lane] = acc[j];
            lds_barrier();
            if (w == (cur.tile & 7)) {  // another one each time
                f32x4 g = f32x4{0.f, 0.f, 0.f, 0.f}, u = g;
#pragma unroll
                for (int v = 0; v < MD_WAVES; ++v) {
                    g += sh.red[v][0][lane];
                    u += sh.red[v][1][lane];
                }
                const int i0 = cur.tile * 16 + lq * 4;
                if constexpr (WT == MD_INT8) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        g[q] *= cur.s[i0 + q];
                        u[q] *= cur.s[cur.step + i0 + q];
                    }
                }
                f32x4 h;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    h[q] = g[q] / (1.0f + expf(-g[q])) * u[q];  // (the quick exponential is off by |g| 2^-24)
                const bool mine = l16 < T && (sh.entry_mask[cur.entry] >> l16 & 1);
                const size_t plane = (size_t)T * (a.K + 1) * a.width;
                uint16_t *to = a.h + (size_t)(mine ? l16 * (a.K + 1) + sh.entry_pick[cur.entry][l16] : 0) * a.width + i0;
                // (cut off, not rounded: what is left out then has 8 bits less, and nothing is left of 24 bits after three; nothing is
                // left of an infinity or a NaN either, where the difference would make a NaN of both)
#pragma unroll
                for (int k = 0; k < MD_NUMBERS; ++k) {
                    uint32_t v[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        v[q] = __float_as_uint(h[q]) & 0xffff0000u;
                        h[q] = __builtin_fabsf(h[q]) < INFINITY ? h[q] - __uint_as_float(v[q]) : 0.0f;
                    }
                    if (mine)
                        __hip_atomic_store(gp(reinterpret_cast<uint64_t *>(to + k * plane)),
                                           (uint64_t)(v[2] >> 16 | v[3]) << 32 | (v[0] >> 16 | v[1]), __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
                }
                wait_loads<0>();
                if (lane == 0)
                    ctr_add(a.ctr + (MD_CTR_READY + cur.entry) * MD_CTR, 1);
            }
            advance();
        }
    }

    // ---- the second product
    top_up();
    bool gave_up = false;
    int known = 0;  // the entries below have their h
    while (cur.phase == 2) {
        take();
        const int slots = uniform(a.K) + 1, per_tile = 8 >> cur.lkw;  // tiles at once, by the waves' shares
        const int units = units_of(cur), wk = w & ((1 << cur.lkw) - 1);
        const uint32_t mask = sh.entry_mask[cur.entry];
        const int pick = sh.entry_pick[cur.entry][l16];
        const bool mine = mask >> l16 & 1;  // this lane's token has the expert
        float s[U2];
        const auto scales_of = [&](int tile) {
            if constexpr (WT == MD_FP8) {
#pragma unroll
                for (int u = 0; u < U2; ++u)
                    s[u] = scale(cur.s, (tile >> 3) * (int)(cur.row_bytes / 128) + min(cur.k0 + wk + (u << cur.lkw), (int)(cur.row_bytes / 128) - 1));
            }
        };
        scales_of(cur.tile);
        // h of the entry, once all of it has been written.  One wave looks, at this entry and the 63 after it, and then, while it
        // waits, at this one alone: all blocks' looks at many counters slow down the streams that they wait for.
        if (cur.entry >= known) {
            if (w == 0) {
                uint32_t last = (uint32_t)wall_clock64(), waited = 0;
                const int d = min(cur.entry + lane, entries - 1), want = (nshared && d == 0 ? a.Is : a.I) / 16 + a.unreachable;
                int *const counter = a.ctr + (MD_CTR_READY + d) * MD_CTR;
                const uint64_t not_yet = __ballot(ctr_load(counter) < want);
                int to = cur.entry + (not_yet ? __builtin_ctzll(not_yet) : 64);
                while (to == cur.entry) {
                    __builtin_amdgcn_s_sleep(8);
                    if (__ballot(lane == 0 && ctr_load(counter) >= want)) {
                        to = cur.entry + 1;
                        break;
                    }
                    const uint32_t now = (uint32_t)wall_clock64();
                    waited += min(now - last, 100000u);  // (1 ms: what else passes between two looks, this wave did not run in)
                    last = now;
                    if (waited > a.wait_ticks) {
                        to = -1;
                        if (lane == 0)
                            __hip_atomic_fetch_or(gp(&g_decode_sync_status), 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
                }
                if (lane == 0)
                    sh.known = to;
            }
            lds_barrier();
            known = uniform(sh.known);
            if (known < 0) {
                gave_up = true;
                known = MD_MAX_ENTRIES + 64;
            }
        }
        asm volatile("" ::: "memory");
        u32x4 h[U2 * W::STEPS * MD_NUMBERS];
        {
            const rsrc_t rh = rsrc(uniform(a.h), uniform((int)a.h_bytes));
            const uint32_t row = (uint32_t)((l16 * slots + pick) * a.width), plane = uniform((int)a.h_bytes) / MD_NUMBERS;
            const int limit = (int)(cur.row_bytes / W::SIZE);
#pragma unroll
            for (int i = 0; i < U2 * W::STEPS * MD_NUMBERS; ++i)
                h[i] = u32x4{0, 0, 0, 0};
            upto<U2>(units, [&](auto c) {
                constexpr int u = decltype(c)::value;
                if (mine) {
#pragma unroll
                    for (int st = 0; st < W::STEPS; ++st) {
                        const int col = (cur.k0 + wk + (u << cur.lkw)) * W::UNIT + (16 / W::SIZE) * (4 * (st / PIECES) + lq) + 8 * (st % PIECES);
                        const uint32_t off = col < limit ? (row + col) * 2 : MD_OUT;
#pragma unroll
                        for (int k = 0; k < MD_NUMBERS; ++k)
                            h[(u * W::STEPS + st) * MD_NUMBERS + k] = __builtin_amdgcn_raw_buffer_load_b128(rh, off, k * plane, AUX_AGENT);
                    }
                }
            });
            wait_loads<0>();  // (once here, not for every use below)
        }
        const rsrc_t rp = rsrc(uniform(a.part), uniform((int)a.part_bytes));
        const int chunks = uniform(a.chunks), C0 = chunks_of(uniform(a.I)), Cs = nshared ? chunks_of(uniform(a.Is)) : 0;
        const int tiles = units > 0 ? tiles_of(cur) : 0;
        for (int t0 = 0; t0 < cur.count; t0 += MD_BATCH * per_tile) {  // t0: the batch's first tile
            const int j0 = t0 >> (3 - cur.lkw);
            const bool last_batch = t0 + MD_BATCH * per_tile >= cur.count;
            f32x4 acc[MD_BATCH];
#pragma unroll 1
            for (int j = 0; j < MD_BATCH; ++j) {
#pragma unroll
                for (int i = 1; i < MD_BATCH; ++i)
                    acc[i - 1] = acc[i];
                acc[MD_BATCH - 1] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (j0 + j < tiles) {
                    if (WT == MD_FP8 && cur.count > 8)  // (otherwise all of one block of rows)
                        scales_of(cur.tile + (w >> cur.lkw) + (j0 + j) * per_tile);
                    upto<U2>(units, [&](auto c) {
                        constexpr int u = decltype(c)::value;
                        use(h + u * W::STEPS * MD_NUMBERS, std::integral_constant<int, MD_NUMBERS>{}, WT == MD_FP8 ? s[u] : 0.f,
                            (uint32_t)(cur.k0 + wk + (u << cur.lkw)) * 128 + 64 >= cur.row_bytes, acc[MD_BATCH - 1]);
                    });
                }
            }
            lds_barrier();  // (the last sums have been read)
#pragma unroll
            for (int j = 0; j < MD_BATCH; ++j)
                sh.red[w][j][lane] = acc[j];
            if (clerk && last_batch)
                describe(turn);
            lds_barrier();
            // tile v of the batch is the (v / per_tile)-th of the 2^lkw waves from (v mod per_tile) 2^lkw on; another wave each
            // time adds them up, and up to four at once
            const int v0 = (w + cur.tile) & 7, here = min(MD_BATCH * per_tile, cur.count - t0);
#pragma unroll 1
            for (int v = v0; v < here; v += MD_WAVES) {
                const int from = (v & (per_tile - 1)) << cur.lkw, j = v >> (3 - cur.lkw);
                f32x4 y = f32x4{0.f, 0.f, 0.f, 0.f};
                for (int k = 0; k < min(1 << cur.lkw, cur.units); ++k)
                    y += sh.red[from + k][j][lane];
                const int n = (cur.tile + t0 + v) * 16 + lq * 4;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if constexpr (WT == MD_INT8)
                        y[q] *= cur.s[n + q];
                    if (gave_up)
                        y[q] = __builtin_nanf("");
                }
                const uint32_t at = (uint32_t)(((l16 * slots + pick) * chunks + cur.chunk) * H + n) * 4u;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), rp, mine ? at : MD_OUT, 0, AUX_AGENT);
            }
            if (v0 < here) {
                wait_loads<0>();
                const int v = v0 + MD_WAVES * lane;
                int before = -1;
                if (v < here)
                    before = ctr_add(a.ctr + (MD_CTR_DONE + cur.tile + t0 + v) * MD_CTR, 1);
                uint64_t last = __ballot(before + 1 == Cs + (entries - nshared) * C0);  // every part of this tile of the output is there
                asm volatile("" ::: "memory");
                for (; last; last &= last - 1) {
                    const int n = (cur.tile + t0 + v0 + MD_WAVES * __builtin_ctzll(last)) * 16 + lq * 4;
                    const int t = min(l16, T - 1), routed = (slots - 1) * C0, n_parts = routed + Cs;
                    const float none = sh.lost[t] ? __builtin_nanf("") : 0.0f;
                    f32x4 o = f32x4{none, none, none, none};
                    constexpr int AT_ONCE = 8;
#pragma unroll 1
                    for (int i0 = 0; i0 < n_parts; i0 += AT_ONCE) {  // picks ascending, the shared expert last
                        f32x4 v[AT_ONCE];
                        float gate[AT_ONCE];
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i) {
                            const int k = i0 + i < routed ? (i0 + i) / C0 : slots - 1, c = i0 + i < routed ? (i0 + i) % C0 : i0 + i - routed;
                            const bool have = i0 + i < routed ? sh.ids[t][k] >= 0 : i0 + i < n_parts && (on >> t & 1);
                            gate[i] = !have ? 0.0f : i0 + i < routed ? sh.gates[t][k] : 1.0f;
                            v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                       rp, have ? (uint32_t)(((t * slots + k) * chunks + c) * H + n) * 4u : MD_OUT, 0, AUX_AGENT));
                        }
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                o[q] = __builtin_fmaf(gate[i], v[i][q], o[q]);  // (what is not there is 0 times 0)
                    }
                    if (l16 < T)
                        *reinterpret_cast<u32x2 *>(a.out + (size_t)t * H + n) =
                            u32x2{f32x2_to_bf16x2(o[0], o[1]), f32x2_to_bf16x2(o[2], o[3])};
                }
            }
        }
        advance();
    }
}

constexpr int MD_MAX_DEVICES = 64;

template <int WT> hipError_t run(const DecodeArgs &a, hipStream_t s)
{
    static std::atomic<bool> done[MD_MAX_DEVICES];  // the kernel's dynamic LDS limit is raised once per device
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && !(dev < MD_MAX_DEVICES && done[dev].load(std::memory_order_acquire))) {
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(&moe_decode_kernel<WT>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)sizeof(Shared));
        if (e == hipSuccess && dev < MD_MAX_DEVICES)
            done[dev].store(true, std::memory_order_release);
    }
    if (e != hipSuccess)
        return e;
    hipLaunchKernelGGL(moe_decode_kernel<WT>, dim3(MD_BLOCKS), dim3(MD_WAVES * 64), sizeof(Shared), s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t moe_decode_sync_status(int *status, bool clear) { return sync_word_read(&g_decode_sync_status, status, clear); }

size_t moe_decode_workspace_bytes(const MoeDecodeArgs &a) { return md_layout(a).total; }

hipError_t launch_moe_decode(const MoeDecodeArgs &a, void *ws, hipStream_t s)
{
    if (a.T == 0)
        return hipSuccess;
    const Layout l = md_layout(a);
    DecodeArgs d{};
    d.p = a;
    d.width = l.width;
    d.chunks = l.chunks;
    d.ws.ctr = reinterpret_cast<int *>(ws);
    d.ws.logits = reinterpret_cast<float *>((char *)ws + l.logits);
    d.ws.h = reinterpret_cast<uint16_t *>((char *)ws + l.h);
    d.ws.part = reinterpret_cast<float *>((char *)ws + l.part);
    d.ws.h_bytes = l.h_bytes;
    d.ws.part_bytes = l.part_bytes;
    const SyncWait wait = sync_wait();
    d.wait_ticks = (uint32_t)std::min(wait.ticks, 0x7fffffffll);
    d.unreachable = wait.unreachable;
    RouteGroupedArgs &r = d.r;
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
    const int per = route_shares(r, 64);
    d.route_per = per <= 1 ? 1 : per <= 4 ? 4 : 16;
    if (per > 16)
        return hipErrorInvalidValue;
    route_places(r, 64, d.route_per);
    const RouterArgs ra{a.x, a.router, a.active, d.ws.logits, d.ws.ctr, a.T, a.E, a.H, a.router_fp32};
    hipLaunchKernelGGL(moe_decode_router_kernel, dim3(a.E, (a.T + MD_ROUTER_TOKENS - 1) / MD_ROUTER_TOKENS), dim3(MD_ROUTER_WAVES * 64), 0, s, ra);
    switch (a.wtype) {
    case MD_BF16:
        return run<MD_BF16>(d, s);
    case MD_INT8:
        return run<MD_INT8>(d, s);
    case MD_FP8:
        return run<MD_FP8>(d, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace cam
