// Two-phase C ABI of the operators of a decode step of a few requests (include/camhip.h): the whole expert layer of a few
// tokens, low-rank adapters.  Argument checks and executors; nothing thrown inside leaves a C entry point.
#include <hip/hip_runtime.h>

#include <exception>
#include <functional>

#include "../../include/camhip.h"
#include "launchers.h"

namespace cam {
camhipStatus api_fail(camhipStatus code, const char *fmt, ...);  // api.cpp
camhipStatus api_make_executor(uint64_t ws_bytes, std::function<hipError_t(void *, hipStream_t)> fn,
                               uint64_t *workspaceSize, camhipExecutor **executor);
camhipStatus api_run_executor(const char *op, void *workspace, uint64_t workspaceSize, camhipExecutor *ex,
                              void *stream);
}  // namespace cam

using cam::api_fail;

static_assert(CAMHIP_DTYPE_BF16 == (int)cam::MD_BF16 && CAMHIP_DTYPE_INT8 == (int)cam::MD_INT8 &&
                  CAMHIP_DTYPE_FP8 == (int)cam::MD_FP8,
              "type codes of the header");
static_assert(CAMHIP_DTYPE_BF16 == (int)cam::LORA_BF16 && CAMHIP_DTYPE_FP16 == (int)cam::LORA_FP16 &&
                  CAMHIP_DTYPE_INT8 == (int)cam::LORA_INT8 && CAMHIP_DTYPE_FP32 == (int)cam::LORA_FP32,
              "type codes of the header");

namespace {

#define CHECK_PARAM(cond, ...)                                                                                      \
    do {                                                                                                            \
        if (!(cond))                                                                                                \
            return api_fail(CAMHIP_ERROR_INVALID_PARAM, __VA_ARGS__);                                               \
    } while (0)
#define CHECK_PTR(op, p)                                                                                            \
    do {                                                                                                            \
        if ((p) == nullptr)                                                                                         \
            return api_fail(CAMHIP_ERROR_NULLPTR, "%s: %s must not be NULL", op, #p);                               \
    } while (0)
#define CHECK_ALIGN(op, p, n)                                                                                       \
    CHECK_PARAM((reinterpret_cast<uintptr_t>(p) & ((n)-1)) == 0, "%s: %s must be %d-byte aligned", op, #p, (int)(n))

typedef long long ll;

template <typename F> camhipStatus guarded(const char *op, F &&f)
{
    try {
        return f();
    } catch (const std::exception &e) {
        return api_fail(CAMHIP_ERROR_RUNTIME, "%s: %s", op, e.what());
    } catch (...) {
        return api_fail(CAMHIP_ERROR_RUNTIME, "%s: unknown error", op);
    }
}

bool is_16_bit(int64_t dtype) { return dtype == CAMHIP_DTYPE_BF16 || dtype == CAMHIP_DTYPE_FP16; }
int dtype_bytes(int64_t dtype) { return dtype == CAMHIP_DTYPE_FP32 ? 4 : dtype == CAMHIP_DTYPE_INT8 ? 1 : 2; }

}  // namespace

extern "C" {

// ---------------------------------------------------------------- a whole expert layer for a few tokens
camhipStatus camhipMoeDecodeLayerGetWorkspaceSize(
    const uint16_t *x, const void *router, const float *bias, const void *gmm1Weight, const float *gmm1WeightScale,
    const void *gmm2Weight, const float *gmm2WeightScale, const void *shareGmm1Weight,
    const float *shareGmm1WeightScale, const void *shareGmm2Weight, const float *shareGmm2WeightScale,
    const uint8_t *xActiveMask, int64_t numTokens, int64_t hidden, int64_t numExperts, int64_t gmm1HiddenSize,
    int64_t shareGmm1HiddenSize, int64_t topK, int64_t weightDtype, int64_t routerDtype, int64_t numGroups,
    int64_t topkGroups, int64_t scoreFunc, int64_t groupScore, int64_t renormalize, double routedScaling, uint16_t *out,
    int32_t *topkIdx, float *topkWeights, uint64_t *workspaceSize, camhipExecutor **executor)
{
    static const char op[] = "moe_decode_layer";
    const bool shared = shareGmm1HiddenSize != 0;
    CHECK_PARAM(weightDtype == CAMHIP_DTYPE_BF16 || weightDtype == CAMHIP_DTYPE_INT8 || weightDtype == CAMHIP_DTYPE_FP8,
                "%s: weightDtype %lld is not bf16, int8 or fp8", op, (ll)weightDtype);
    CHECK_PARAM(routerDtype == CAMHIP_DTYPE_BF16 || routerDtype == CAMHIP_DTYPE_FP32,
                "%s: routerDtype %lld is neither bf16 nor fp32", op, (ll)routerDtype);
    const int64_t unit = weightDtype == CAMHIP_DTYPE_FP8 ? 128 : 64;
    CHECK_PARAM(numTokens >= 0 && numTokens <= cam::MD_MAX_TOKENS, "%s: numTokens %lld out of [0,%d]", op, (ll)numTokens,
                cam::MD_MAX_TOKENS);
    CHECK_PARAM(hidden >= unit && hidden <= cam::MD_MAX_HIDDEN && hidden % unit == 0,
                "%s: hidden %lld must be a multiple of %lld up to %d", op, (ll)hidden, (ll)unit, cam::MD_MAX_HIDDEN);
    CHECK_PARAM(gmm1HiddenSize >= 2 * unit && gmm1HiddenSize <= 2 * cam::MD_MAX_INTER && gmm1HiddenSize % (2 * unit) == 0,
                "%s: gmm1HiddenSize %lld must be a multiple of %lld up to %d", op, (ll)gmm1HiddenSize, (ll)(2 * unit),
                2 * cam::MD_MAX_INTER);
    CHECK_PARAM(!shared || (shareGmm1HiddenSize >= 2 * unit && shareGmm1HiddenSize <= 2 * cam::MD_MAX_INTER &&
                            shareGmm1HiddenSize % (2 * unit) == 0),
                "%s: shareGmm1HiddenSize %lld must be 0 or a multiple of %lld up to %d", op, (ll)shareGmm1HiddenSize,
                (ll)(2 * unit), 2 * cam::MD_MAX_INTER);
    CHECK_PARAM(numExperts >= 1 && numExperts <= 512, "%s: numExperts %lld out of [1,512]", op, (ll)numExperts);
    CHECK_PARAM(topK >= 1 && topK <= 16 && topK <= numExperts, "%s: topK %lld out of [1,min(16,numExperts)]", op, (ll)topK);
    CHECK_PARAM(numGroups >= 1 && numGroups <= 64 && numExperts % numGroups == 0,
                "%s: numGroups %lld must be in [1,64] and divide numExperts %lld", op, (ll)numGroups, (ll)numExperts);
    CHECK_PARAM(topkGroups >= 1 && topkGroups <= numGroups, "%s: topkGroups %lld out of [1,%lld]", op, (ll)topkGroups,
                (ll)numGroups);
    CHECK_PARAM(topK <= topkGroups * (numExperts / numGroups),
                "%s: topK %lld exceeds the %lld experts of topkGroups %lld groups", op, (ll)topK,
                (ll)(topkGroups * (numExperts / numGroups)), (ll)topkGroups);
    CHECK_PARAM(scoreFunc == CAMHIP_ROUTE_SOFTMAX || scoreFunc == CAMHIP_ROUTE_SIGMOID,
                "%s: scoreFunc %lld is neither softmax nor sigmoid", op, (ll)scoreFunc);
    CHECK_PARAM(groupScore == CAMHIP_ROUTE_GROUP_MAX || groupScore == CAMHIP_ROUTE_GROUP_TOP2,
                "%s: groupScore %lld is neither max nor top2", op, (ll)groupScore);
    CHECK_PARAM(renormalize == 0 || renormalize == 1, "%s: renormalize must be 0 or 1", op);
    if (numTokens > 0) {
        CHECK_PTR(op, x);
        CHECK_PTR(op, router);
        CHECK_PTR(op, gmm1Weight);
        CHECK_PTR(op, gmm2Weight);
        CHECK_PTR(op, out);
        CHECK_PTR(op, topkIdx);
        CHECK_PTR(op, topkWeights);
        if (weightDtype != CAMHIP_DTYPE_BF16) {
            CHECK_PTR(op, gmm1WeightScale);
            CHECK_PTR(op, gmm2WeightScale);
        }
        if (shared) {
            CHECK_PTR(op, shareGmm1Weight);
            CHECK_PTR(op, shareGmm2Weight);
            if (weightDtype != CAMHIP_DTYPE_BF16) {
                CHECK_PTR(op, shareGmm1WeightScale);
                CHECK_PTR(op, shareGmm2WeightScale);
            }
        }
    }
    CHECK_ALIGN(op, x, 16);
    CHECK_ALIGN(op, router, 16);
    CHECK_ALIGN(op, gmm1Weight, 16);
    CHECK_ALIGN(op, gmm2Weight, 16);
    CHECK_ALIGN(op, shareGmm1Weight, 16);
    CHECK_ALIGN(op, shareGmm2Weight, 16);
    CHECK_ALIGN(op, bias, 4);
    CHECK_ALIGN(op, gmm1WeightScale, 4);
    CHECK_ALIGN(op, gmm2WeightScale, 4);
    CHECK_ALIGN(op, shareGmm1WeightScale, 4);
    CHECK_ALIGN(op, shareGmm2WeightScale, 4);
    CHECK_ALIGN(op, out, 8);
    CHECK_ALIGN(op, topkIdx, 4);
    CHECK_ALIGN(op, topkWeights, 4);
    cam::MoeDecodeArgs a{};
    a.x = x;
    a.router = router;
    a.bias = bias;
    a.active = xActiveMask;
    a.w1 = gmm1Weight;
    a.w2 = gmm2Weight;
    a.s1 = gmm1WeightScale;
    a.s2 = gmm2WeightScale;
    a.sw1 = shareGmm1Weight;
    a.sw2 = shareGmm2Weight;
    a.ss1 = shareGmm1WeightScale;
    a.ss2 = shareGmm2WeightScale;
    a.out = out;
    a.topk_idx = topkIdx;
    a.topk_w = topkWeights;
    a.T = (int)numTokens;
    a.H = (int)hidden;
    a.E = (int)numExperts;
    a.I = (int)(gmm1HiddenSize / 2);
    a.Is = (int)(shareGmm1HiddenSize / 2);
    a.K = (int)topK;
    a.G = (int)numGroups;
    a.KG = (int)topkGroups;
    a.score = (int)scoreFunc;
    a.group_top2 = groupScore == CAMHIP_ROUTE_GROUP_TOP2;
    a.renorm = (int)renormalize;
    a.router_fp32 = routerDtype == CAMHIP_DTYPE_FP32;
    a.wtype = (int)weightDtype;
    a.scaling = (float)routedScaling;
    return guarded(op, [&] {
        return cam::api_make_executor(
            cam::moe_decode_workspace_bytes(a),
            [a](void *ws, hipStream_t s) { return cam::launch_moe_decode(a, ws, s); }, workspaceSize, executor);
    });
}

camhipStatus camhipMoeDecodeLayer(void *workspace, uint64_t workspaceSize, camhipExecutor *executor, void *stream)
{
    return guarded("moe_decode_layer", [&] {
        return cam::api_run_executor("moe_decode_layer", workspace, workspaceSize, executor, stream);
    });
}

// ---------------------------------------------------------------- low-rank adapters
camhipStatus camhipLoraAddGetWorkspaceSize(const void *base, const void *x, const float *xScale, const void *loraA,
                                           const void *loraB, const int32_t *adapterIds, const float *scaling,
                                           int64_t m, int64_t n, int64_t k, int64_t rank, int64_t numAdapters,
                                           int64_t baseRowStride, int64_t xRowStride, int64_t baseDtype, int64_t xDtype,
                                           int64_t loraDtype, int64_t outDtype, void *out, uint64_t *workspaceSize,
                                           camhipExecutor **executor)
{
    static const char op[] = "lora_add";
    CHECK_PARAM(m >= 0 && m <= (int64_t)1 << 20, "%s: m %lld out of [0,2^20]", op, (ll)m);
    CHECK_PARAM(n >= 1 && n <= (int64_t)1 << 20, "%s: n %lld out of [1,2^20]", op, (ll)n);
    CHECK_PARAM(k >= 16 && k <= 131056 && k % 16 == 0, "%s: k %lld must be a multiple of 16 in [16,131056]", op, (ll)k);
    CHECK_PARAM(rank >= 8 && rank <= 256 && rank % 8 == 0, "%s: rank %lld must be a multiple of 8 in [8,256]", op, (ll)rank);
    CHECK_PARAM(numAdapters >= 1 && numAdapters <= 65536, "%s: numAdapters %lld out of [1,65536]", op, (ll)numAdapters);
    CHECK_PARAM(is_16_bit(baseDtype) || baseDtype == CAMHIP_DTYPE_FP32, "%s: baseDtype %lld is not bf16, fp16 or fp32", op,
                (ll)baseDtype);
    CHECK_PARAM(is_16_bit(loraDtype), "%s: loraDtype %lld is neither bf16 nor fp16", op, (ll)loraDtype);
    CHECK_PARAM(xDtype == loraDtype || xDtype == CAMHIP_DTYPE_INT8, "%s: xDtype %lld must be loraDtype or int8", op,
                (ll)xDtype);
    CHECK_PARAM(is_16_bit(outDtype), "%s: outDtype %lld is neither bf16 nor fp16", op, (ll)outDtype);
    CHECK_PARAM(baseRowStride >= n && baseRowStride <= (int64_t)1 << 31, "%s: baseRowStride %lld out of [n %lld,2^31]", op,
                (ll)baseRowStride, (ll)n);
    CHECK_PARAM(xRowStride >= k && xRowStride <= (int64_t)1 << 31, "%s: xRowStride %lld out of [k %lld,2^31]", op,
                (ll)xRowStride, (ll)k);
    if (m > 0) {
        CHECK_PTR(op, base);
        CHECK_PTR(op, x);
        CHECK_PTR(op, loraA);
        CHECK_PTR(op, loraB);
        CHECK_PTR(op, adapterIds);
        CHECK_PTR(op, out);
        if (xDtype == CAMHIP_DTYPE_INT8)
            CHECK_PTR(op, xScale);
    }
    CHECK_ALIGN(op, base, dtype_bytes(baseDtype));
    CHECK_ALIGN(op, x, 16);
    CHECK_PARAM(xRowStride * dtype_bytes(xDtype) % 16 == 0, "%s: xRowStride %lld: rows must be 16-byte aligned", op, (ll)xRowStride);
    CHECK_ALIGN(op, loraA, 16);
    CHECK_ALIGN(op, loraB, 16);
    CHECK_ALIGN(op, adapterIds, 4);
    CHECK_ALIGN(op, scaling, 4);
    CHECK_ALIGN(op, xScale, 4);
    CHECK_ALIGN(op, out, 2);
    cam::LoraArgs a{};
    a.base = base;
    a.x = x;
    a.xs = xDtype == CAMHIP_DTYPE_INT8 ? xScale : nullptr;
    a.a = loraA;
    a.b = loraB;
    a.ids = adapterIds;
    a.scaling = scaling;
    a.out = out;
    a.M = m;
    a.base_stride = baseRowStride;
    a.x_stride = xRowStride;
    a.N = (int)n;
    a.K = (int)k;
    a.R = (int)rank;
    a.L = (int)numAdapters;
    a.base_dtype = (int8_t)baseDtype;
    a.x_dtype = (int8_t)xDtype;
    a.dtype = (int8_t)loraDtype;
    a.out_dtype = (int8_t)outDtype;
    return guarded(op, [&] {
        return cam::api_make_executor(
            cam::lora_workspace_bytes(a), [a](void *ws, hipStream_t s) { return cam::launch_lora_add(a, ws, s); },
            workspaceSize, executor);
    });
}

camhipStatus camhipLoraAdd(void *workspace, uint64_t workspaceSize, camhipExecutor *executor, void *stream)
{
    return guarded("lora_add", [&] {
        return cam::api_run_executor("lora_add", workspace, workspaceSize, executor, stream);
    });
}

}  // extern "C"
