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
// exponential rounds.  For the choice s is rounded to 42 fraction bits: what is left of the exponential's error goes (1/2
// is 1/2), and s + b and the sum of two such are exact in 64 bits for most biases, so that sums of different parts that
// are equal are found equal.  The low 10 mantissa bits of c then give way to the expert's place among the lanes (which
// rises with its id), so that one v_max_f64 reduction gives both the score and the expert, with ties to the lower id; a
// group's sum is taken before that, of the whole c.  Without a bias s orders as l does, and the keys are the logits
// themselves (exact: a float leaves 29 bits of a double free): no exponential then, but for the picks and the denominator.
//
// A token is handled by LANES (8, 16 or 64) adjacent lanes, each holding PER consecutive experts of one group; a group
// has LANES / (number of groups, rounded up to a power of two) lanes.  So the best two of a group are found by a scan of
// the lane's own experts and log2 of those lanes' steps, all groups at once.
//
// Bound by vector instructions where there are many tokens, 50 an expert (65536 tokens, 256 experts, 8 picks in 4 of 8
// groups: 33 us, where the logits' stream takes 15), and by one token's chain of steps and the launch where there are few
// (one token 4.1 us).  Figures of two sides, below, are those that a choice was made on; the scores' rounding and the group
// sums of whole scores came after most of them and cost both sides up to 0.3 us at few tokens and -4 to 10% at
// 65536.
#include "route_dev.h"

namespace cam {

namespace {

constexpr int RG_WAVES = 4;

// (PER = 32: 156 registers with merges, 164 with heads, three waves of a SIMD; held to 128 they spill: 64 against 33 us at
// 65536 tokens.)
template <int LANES, int PER, int PICK>
__global__ __launch_bounds__(RG_WAVES * 64) void route_grouped_kernel(const RouteGroupedArgs p)
{
    constexpr int TPW = 64 / LANES;  // tokens per wave
    const int lane = threadIdx.x & 63, rl = lane & (LANES - 1);
    const int t = ((int)blockIdx.x * RG_WAVES + (int)(threadIdx.x >> 6)) * TPW + lane / LANES;
    const bool live = t < p.T;  // dead rows run along (they read row 0)
    const char *row = reinterpret_cast<const char *>(p.logits) + (size_t)(live ? t : 0) * (size_t)p.row_bytes;
    int my_idx;
    double gate;
    route_token<LANES, PER, PICK>(p, row, rl, my_idx, gate);
    if (live && rl < p.K) {
        p.topk_idx[(size_t)t * p.K + rl] = my_idx;
        p.topk_w[(size_t)t * p.K + rl] = (float)(gate * (double)p.scaling);
        if (p.topk_idx64)
            p.topk_idx64[(size_t)t * p.K + rl] = my_idx;
    }
}

}  // namespace

hipError_t launch_route_grouped(RouteGroupedArgs a, hipStream_t s)
{
    if (a.T == 0)
        return hipSuccess;
    if (a.E < 1 || a.E > 512 || a.K < 1 || a.K > 16 || a.G < 1 || a.G > 64 || a.E % a.G || a.KG < 1 || a.KG > a.G)
        return hipErrorInvalidValue;
    const int g2 = route_pow2(a.G);
    a.gs = a.E / a.G;
    // How many lanes a token gets.  More lanes hold fewer experts each (shorter chains: one token), fewer have fewer steps
    // between lanes to pay for (many tokens); from 64 lanes to 16 a grid has a quarter of the waves.  In us, sigmoid with a
    // bias, the lanes chosen first:
    //   5 to 8 picks, 8 lanes:
    //     5 to 8 experts in one of 8 lanes: 64 experts, 128 tokens 3.7 against 3.9 in 16 lanes, 65536 tokens 12.0 against 15.2.
    //     up to 24, from 8192 tokens on: 128 experts 4.7 against 5.1, 160 (8 groups) 5.4 against 6.8, 192 5.4 against 5.7
    //     (below: 128 experts, 128 tokens 4.4 against 3.8).
    //     up to 32, from 24576 tokens on: 256 experts (8 groups) 14.6 against 15.1, 65536 tokens 34.7 against 37.3 (16384 both
    //     11.8; 8192 7.7 against 7.0).
    //   64 lanes while there are few tokens, 16 otherwise:
    //     25 to 32 experts in one of 16 lanes: 512 experts, 8 picks, 2048 tokens 5.5 against 6.8, 3000 6.4 against 6.8, 4096 7.4
    //     against 6.8; 16 picks 3000 8.5 and 8.5; 4 picks 4096 7.2 against 8.2, 8192 12.0 against 12.2.
    //     17 to 24, 5 to 8 picks: 384 experts, 1024 tokens 4.9 against 5.1, 2048 6.0 against 5.1.  (256, one token: 4.9 against 4.6.)
    //     9 to 24, more picks: 256 experts, 16 picks, 1024 tokens 5.6 against 5.9, 2048 6.5 against 5.9.  (128, 10 picks, one
    //     token 4.6 against 4.0.)
    //     5 to 24, fewer picks: 128 experts, 4 picks, 128 tokens 3.7 against 4.1, 2048 both 4.1; 256, 2 picks, 2048 4.0 against 4.5.
    //     groups that are not read by fours: 150 (5 groups), 6 picks, 128 tokens 4.8 against 6.3, 2048 5.7 against 6.5.
    const int per16 = g2 <= 16 ? (a.gs + 16 / g2 - 1) / (16 / g2) : 64;
    const int per8 = g2 <= 8 ? (a.gs + 8 / g2 - 1) / (8 / g2) : 64;
    const bool merged = a.K > 4 && a.K <= 8;
    int few = 0;
    if (per16 > 24)
        few = a.K > 4 ? 3000 : 4096;
    else if (per16 > 4 && (a.K <= 4 || a.gs % 4))
        few = 2048;
    else if (per16 > (merged ? 16 : 8))
        few = 1024;
    int lanes = per16 > 32 || a.T <= few ? 64 : 16;
    if (merged && ((per8 > 4 && per8 <= 8) || (per8 <= 24 && a.T >= 8192) || (per8 <= 32 && a.T >= 24576)))
        lanes = 8;
    const int per = route_shares(a, lanes);
    const int tokens = RG_WAVES * (64 / lanes);
    const dim3 grid((a.T + tokens - 1) / tokens), block(RG_WAVES * 64);
    // A pick by a reduction over everything takes about 3 PER + 25 instructions, of a sorted list's heads 45 to 15 (fewer as
    // fewer are left to move up), a merge of two lists 90; sorting 16 experts 140 (8 of them kept: 100).  So: up to 4 picks by
    // reductions, 5 to 8 by merges (16 lanes, PER = 16, K = 8: 460 against 520), more from the heads (256 experts, 12 picks,
    // 4096 tokens 7.5 -> 6.2 us, 512 experts, 16 picks, 65536 tokens 101 -> 78), and from the heads too where 64 lanes would
    // need six merges (512 experts, 8 picks, one token 5.0 -> 4.2).
#define RG_LAUNCH(L, P, S)                                                                                          \
    do {                                                                                                            \
        route_places(a, lanes, P);                                                                                  \
        hipLaunchKernelGGL((route_grouped_kernel<L, P, S>), grid, block, 0, s, a);                                  \
        return hipGetLastError();                                                                                   \
    } while (0)
#define RG_CASE(L, P)                                                                                               \
    if (lanes == L && per <= P)                                                                                     \
    RG_LAUNCH(L, P, RG_EACH)
#define RG_SORT(L, P)                                                                                               \
    if (lanes == L && per <= P && a.K > 4 && a.K <= 8)                                                              \
    RG_LAUNCH(L, P, RG_MERGE)
#define RG_POPS(L, P)                                                                                               \
    if (lanes == L && per <= P && a.K > (L == 64 ? 4 : 8))                                                          \
    RG_LAUNCH(L, P, RG_POP)
    RG_SORT(8, 8);
    RG_SORT(8, 16);
    RG_SORT(8, 20);
    RG_SORT(8, 24);
    RG_SORT(8, 32);
    RG_CASE(64, 1);
    RG_CASE(64, 2);
    RG_POPS(64, 4);
    RG_CASE(64, 4);
    RG_POPS(64, 8);
    RG_CASE(64, 8);
    RG_POPS(64, 16);
    RG_CASE(64, 16);
    RG_CASE(16, 1);
    RG_CASE(16, 2);
    RG_POPS(16, 4);
    RG_CASE(16, 4);
    RG_POPS(16, 8);
    RG_POPS(16, 12);
    RG_POPS(16, 16);
    RG_POPS(16, 24);
    RG_POPS(16, 32);
    RG_SORT(16, 8);
    RG_CASE(16, 8);
    if (a.by_logit || a.gs % 4)  // (with scores to compute, 12 by fours are ahead of 10: 160 experts, one token 4.8 against 5.0 us)
        RG_SORT(16, 10);
    RG_SORT(16, 12);
    RG_CASE(16, 10);
    RG_CASE(16, 12);
    RG_SORT(16, 16);
    RG_CASE(16, 16);
    RG_SORT(16, 24);
    RG_CASE(16, 24);
    RG_SORT(16, 32);
    RG_CASE(16, 32);
#undef RG_SORT
#undef RG_POPS
#undef RG_LAUNCH
#undef RG_CASE
    return hipErrorInvalidValue;
}

}  // namespace cam
