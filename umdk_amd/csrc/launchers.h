// Internal host launchers, one per kernel family.  Not exported: the public
// surface is the two-phase C ABI in include/camhip.h (implemented in api.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cam {

// QUANT_INT8_FUSED: the fused decode op's int8 recipe (no epsilon, optional smooth scales); internal only
enum QuantMode { QUANT_NONE = 0, QUANT_INT8_TOKEN = 2, QUANT_FP8_BLOCK = 3, QUANT_INT8_FUSED = 4 };

// ---- routing (route.hip)
// topk_idx64 (optional): the same ids as int64, the layout op's input type
hipError_t launch_route(const float *logits, const float *bias, int T, int E, int K, int32_t *topk_idx,
                        float *topk_w, hipStream_t s, int64_t *topk_idx64 = nullptr);

// routing that also writes per-chunk histograms of the ids below Ec: chunks of route_tokens_per_block() tokens,
// chunk_counts[e * nc + c], each chunk's exclusive prefix of its histogram over the experts, chunk_pref[e * nc +
// c], and each such pick's rank among its chunk's picks of the same expert, chunk_rank[t * K + k] (the prefill
// step)
int route_tokens_per_block();
hipError_t launch_route_hist(const float *logits, const float *bias, int T, int E, int K, int Ec, int32_t *topk_idx,
                             float *topk_w, int32_t *chunk_counts, int32_t *chunk_pref, int32_t *chunk_rank,
                             hipStream_t s);

// A launch of up to 112 bytes of arguments takes the host 2.75 us, from 120 bytes on 3.5 us.
constexpr size_t LAUNCH_ARGS = 112;

// ---- routing over groups of experts (route_grouped.hip)
enum RouteScore { ROUTE_SOFTMAX = 0, ROUTE_SIGMOID = 1 };
enum RouteDtype { ROUTE_BF16 = 0, ROUTE_FP16 = 1, ROUTE_FP32 = 4 };  // the CAMHIP_DTYPE_* codes
struct RouteGroupedArgs {
    const void *logits;
    int64_t row_bytes;  // between two tokens' logits
    const float *bias;  // or nullptr
    int T, E, K, G, KG;
    int score, group_top2, renorm, dtype;
    float scaling;
    int32_t *topk_idx;
    float *topk_w;
    int64_t *topk_idx64;  // or nullptr
    // set by the launcher: experts per group, lanes per group and their logarithm, whether the keys are the logits, whether
    // every lane holds as many experts as it can, vector loads
    int gs, lpg, lpg_log, by_logit, full, vec;
};
static_assert(sizeof(RouteGroupedArgs) <= LAUNCH_ARGS, "a cheap launch");
hipError_t launch_route_grouped(RouteGroupedArgs a, hipStream_t s);

// ---- residual addition + root-mean-square norm (+ quantisation) (norm.hip)
struct NormArgs {
    const uint16_t *x;
    int64_t x_stride;          // elements between two rows of x
    const uint16_t *residual;  // or nullptr; rows of H
    const void *weight;        // [H], x's type or fp32 (weight_fp32)
    int64_t T;
    int64_t row0;  // the launcher's: the first row of a launch
    int H;
    float eps;
    int fp16, weight_fp32, quant;  // quant: QUANT_NONE, QUANT_INT8_TOKEN, QUANT_FP8_BLOCK (k-major scales)
    void *y;                       // [T, H]
    float *scales;                 // [T] (int8), [H/128, T] (fp8)
    uint16_t *residual_out;        // [T, H], with a residual only
};
static_assert(sizeof(NormArgs) <= LAUNCH_ARGS, "a cheap launch");
hipError_t launch_add_rms_norm(const NormArgs &a, hipStream_t s);

// ---- int8 matrix product (qmm.hip)
enum QmmOut { QMM_BF16 = 0, QMM_FP16 = 1, QMM_FP32 = 4 };  // the CAMHIP_DTYPE_* codes
struct QmmArgs {
    const int8_t *x, *w;     // [M, K], [N, K]
    const float *xs, *ws;    // [M], [N]
    const float *bias;       // [N] or nullptr
    int64_t M;
    int N, K, out_dtype;
    void *out;               // [M, N]
};
static_assert(sizeof(QmmArgs) + 2 * sizeof(int) <= LAUNCH_ARGS, "a cheap launch");
hipError_t launch_quant_matmul(const QmmArgs &a, hipStream_t s);

// ---- a whole expert layer for a few tokens (moe_decode.hip)
enum MoeDecodeWeight { MD_BF16 = 0, MD_INT8 = 2, MD_FP8 = 3 };  // the CAMHIP_DTYPE_* codes
constexpr int MD_MAX_TOKENS = 16, MD_MAX_HIDDEN = 8192, MD_MAX_INTER = 32768;
struct MoeDecodeArgs {
    const uint16_t *x;          // [T, H] bf16
    const void *router;         // [E, H] bf16, or fp32 (router_fp32)
    const float *bias;          // [E] or nullptr
    const uint8_t *active;      // [T] or nullptr
    const void *w1, *w2;        // [E, 2 I, H], [E, H, I]
    const float *s1, *s2;       // int8: [E, 2 I], [E, H]; fp8: [E, 2 I / 128, H / 128], [E, H / 128, I / 128]
    const void *sw1, *sw2;      // the shared expert's, or nullptr
    const float *ss1, *ss2;
    uint16_t *out;              // [T, H] bf16
    int32_t *topk_idx;          // [T, K]
    float *topk_w;
    int T, H, E, I, Is, K;      // Is: 0 without a shared expert
    int G, KG, score, group_top2, renorm, router_fp32, wtype;
    float scaling;
};
// The layer's sync status (as gmm.h's): nonzero once a wait for an expert's h has given up.
hipError_t moe_decode_sync_status(int *status, bool clear);
size_t moe_decode_workspace_bytes(const MoeDecodeArgs &a);
hipError_t launch_moe_decode(const MoeDecodeArgs &a, void *ws, hipStream_t s);

// ---- low-rank adapters beside a projection (lora.hip)
enum LoraDtype { LORA_BF16 = 0, LORA_FP16 = 1, LORA_INT8 = 2, LORA_FP32 = 4 };  // the CAMHIP_DTYPE_* codes
struct LoraArgs {
    const void *base;           // [M, N], rows base_stride elements apart
    const void *x;              // [M, K], rows x_stride elements apart
    const float *xs;            // [M], int8 rows only
    const void *a, *b;          // [L, R, K], [L, N, R]
    const int32_t *ids;         // [M]
    const float *scaling;       // [L] or nullptr
    void *out;                  // [M, N]
    int64_t M, base_stride, x_stride;
    int N, K, R, L;
    int8_t base_dtype, x_dtype, dtype, out_dtype;
};
size_t lora_workspace_bytes(const LoraArgs &a);
hipError_t launch_lora_add(const LoraArgs &a, void *ws, hipStream_t s);

// ---- dispatch layout (layout.hip)
struct LayoutPlan {
    int tokens_per_chunk;
    int n_chunks;
};
LayoutPlan layout_plan(int T, int K);
size_t layout_workspace_bytes(int T, int K, int E, int R);
hipError_t launch_layout(const int64_t *topk_idx, int T, int K, int E, int R, int32_t *ntok_per_rank,
                         int32_t *ntok_per_expert, int32_t *is_token_in_rank, int32_t *send_token_idx,
                         void *ws, hipStream_t s);
// the prefill step: chunk counts [E][nc] -> exclusive chunk bases in place, and the one-rank count exchange from
// the row totals and the summed chunk prefixes [E][nc] of launch_route_hist
hipError_t launch_scan_notify(int E, int nc, int32_t *counts, const int32_t *pref, int32_t *send_offset,
                              int32_t *recv_count, int64_t *tokens_per_expert, hipStream_t s);
// int32 topk ids, used by the fused path
hipError_t launch_layout_i32(const int32_t *topk_idx, int T, int K, int E, int32_t *ntok_per_expert,
                             int32_t *send_token_idx, void *ws, hipStream_t s);

// decode-sized layout + count exchange in one launch (T*K <= 8192; ids masked by `active`); it also zeroes
// zero[0, nzero) (a later launch's counters) and, for a shared expert that the GEMMs run as group E, writes their group
// list groups[0, E] (tokens_per_expert, then T)
hipError_t launch_layout_small(const int32_t *ids, const uint8_t *active, int T, int K, int E, int32_t *ids_eff,
                               int32_t *counts, int32_t *sti, int32_t *send_offset, int32_t *recv_count,
                               int32_t *total, int64_t *tokens_per_expert, hipStream_t s, int32_t *zero = nullptr,
                               int nzero = 0, int64_t *groups = nullptr);

// ---- small utilities (notify.hip)
hipError_t launch_fill_i32(int32_t *p, int32_t v, long n, hipStream_t s);

// ---- count exchange for one rank (notify.hip)
hipError_t launch_notify(const int32_t *counts, int E, int T, int32_t *send_offset, int32_t *total_recv,
                         int32_t *recv_count, int32_t *recv_offset, int32_t *max_bs,
                         int64_t *recv_tokens_per_expert, int local_experts, hipStream_t s);

// ---- permute + quantise (dispatch.hip); topk_idx == nullptr: identity rows (K must be 1)
hipError_t launch_dispatch(const uint16_t *x, const int32_t *topk_idx, const int32_t *send_offset,
                           const int32_t *send_token_idx, int T, int H, int K, int E, int rank, int cap, int quant_mode,
                           void *expand_x, float *scales, int32_t *expand_idx, hipStream_t s,
                           int32_t *inv_out = nullptr, const float *smooth = nullptr, bool kmajor_scales = false,
                           const int32_t *chunk_base = nullptr, int tpc = 0, const int32_t *chunk_rank = nullptr,
                           bool skip_unrouted = false, const int32_t *share = nullptr,
                           const float *share_smooth = nullptr);
// decode sizes (dispatch_decode_fits: T*K <= 2048, E <= 512; bf16 or fp8 rows): layout + count exchange +
// dispatch as one launch (the arguments of launch_layout_small and launch_dispatch; the ranks and effective ids
// stay in LDS)
hipError_t launch_dispatch_decode(const int32_t *ids, const uint8_t *active, const uint16_t *x, int T, int H, int K,
                                  int E, int cap, int quant_mode, void *expand_x, float *scales, int32_t *expand_idx,
                                  int32_t *inv_out, bool kmajor_scales, int32_t *counts, int32_t *send_offset,
                                  int32_t *recv_count, int32_t *total, int64_t *tokens_per_expert, hipStream_t s,
                                  int32_t *zero, int nzero, int64_t *groups = nullptr);
// (groups: as for launch_layout_small; every token then also goes to row total + t.  share: the same from a layout's
// total; share_smooth: the int8 smooth scales of those rows)
bool dispatch_decode_fits(int T, int K, int E);
// (send_token_idx == nullptr: the rank within the expert is chunk_base[e * nc + t / tpc] plus chunk_rank[t * K + k],
// the rank inside the token's chunk of tpc tokens; skip_unrouted: tokens with no pick in [0, E) read nothing, for a
// rank that holds only some of the experts)
// (fp8: kmajor_scales writes the block scales as [H/128, cap], the layout the grouped GEMMs read)
// combine without the scatter launch, for callers whose dispatch already wrote inv
hipError_t launch_combine_gather(const uint16_t *y, const int32_t *expand_idx, int N, const int32_t *recv_count_last,
                                 const float *topk_w, int T, int K, int H, uint16_t *out, const int32_t *inv,
                                 hipStream_t s);

// ---- diagnose outputs (diag.hip): stats[idx] += microseconds between the two stream points
hipError_t launch_phase_begin(uint64_t *stamp, hipStream_t s);
hipError_t launch_phase_end(const uint64_t *stamp, int32_t *stats, int idx, hipStream_t s);

// ---- fused decode helpers (fused.hip)
hipError_t launch_prepare_ids(const int32_t *ids, const uint8_t *active, int T, int K, int first_local, int L,
                              int32_t *out, hipStream_t s);
hipError_t launch_fill_i64(int64_t *p, int64_t v, long n, hipStream_t s);

// ---- weighted unpermute (combine.hip)
hipError_t launch_combine(const uint16_t *y, const int32_t *expand_idx, int N, const int32_t *recv_count_last,
                          const float *topk_w, int T, int K, int H, uint16_t *out, int32_t *inv_ws,
                          hipStream_t s);
// the same combine with its row map (and diagnose stamp) in the library's static per-device scratch:
// no workspace, no allocation; T*K <= COMBINE_NOALLOC_MAX_SLOTS
constexpr long COMBINE_NOALLOC_MAX_SLOTS = 1L << 18;
hipError_t launch_combine_noalloc(const uint16_t *y, const int32_t *expand_idx, int N, const int32_t *recv_count_last,
                                  const float *topk_w, int T, int K, int H, uint16_t *out, int32_t *cost_stats,
                                  int stats_idx, hipStream_t s);

}  // namespace cam
