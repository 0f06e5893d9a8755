// Two-phase C ABI of the operators around the expert layer (include/camhip.h): grouped routing, residual norm, int8
// product.  Argument checks and executors; nothing thrown inside leaves a C entry point.
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

static_assert(CAMHIP_DTYPE_BF16 == (int)cam::ROUTE_BF16 && CAMHIP_DTYPE_FP16 == (int)cam::ROUTE_FP16 &&
                  CAMHIP_DTYPE_FP32 == (int)cam::ROUTE_FP32,
              "type codes of the header");
static_assert(CAMHIP_DTYPE_BF16 == (int)cam::QMM_BF16 && CAMHIP_DTYPE_FP16 == (int)cam::QMM_FP16 &&
                  CAMHIP_DTYPE_FP32 == (int)cam::QMM_FP32,
              "type codes of the header");
static_assert(CAMHIP_ROUTE_SOFTMAX == (int)cam::ROUTE_SOFTMAX && CAMHIP_ROUTE_SIGMOID == (int)cam::ROUTE_SIGMOID,
              "score codes of the header");

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
// element alignment (a misaligned base would be a misaligned access of every element)
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

size_t dtype_bytes(int64_t dtype) { return dtype == CAMHIP_DTYPE_FP32 ? 4 : 2; }

}  // namespace

extern "C" {

// ---------------------------------------------------------------- routing over groups of experts
camhipStatus camhipMoeRouteGroupedGetWorkspaceSize(const void *logits, const float *bias, int64_t numTokens,
                                                   int64_t numExperts, int64_t topK, int64_t logitsDtype,
                                                   int64_t logitsRowStride, int64_t numGroups, int64_t topkGroups,
                                                   int64_t scoreFunc, int64_t groupScore, int64_t renormalize,
                                                   double routedScaling, int32_t *topkIdx, float *topkWeights,
                                                   int64_t *topkIdxInt64, uint64_t *workspaceSize,
                                                   camhipExecutor **executor)
{
    static const char op[] = "moe_route_grouped";
    CHECK_PARAM(numTokens >= 0 && numTokens <= 65536, "%s: numTokens %lld out of [0,65536]", op, (ll)numTokens);
    CHECK_PARAM(numExperts >= 1 && numExperts <= 512, "%s: numExperts %lld out of [1,512]", op, (ll)numExperts);
    CHECK_PARAM(topK >= 1 && topK <= 16 && topK <= numExperts, "%s: topK %lld out of [1,min(16,numExperts)]", op,
                (ll)topK);
    CHECK_PARAM(logitsDtype == CAMHIP_DTYPE_BF16 || logitsDtype == CAMHIP_DTYPE_FP16 ||
                    logitsDtype == CAMHIP_DTYPE_FP32,
                "%s: logitsDtype %lld is not bf16, fp16 or fp32", op, (ll)logitsDtype);
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
    CHECK_PARAM(logitsRowStride >= numExperts, "%s: logitsRowStride %lld is below numExperts %lld", op,
                (ll)logitsRowStride, (ll)numExperts);
    CHECK_PARAM(logitsRowStride <= (int64_t)1 << 31, "%s: logitsRowStride %lld is out of range", op,
                (ll)logitsRowStride);
    if (numTokens > 0) {
        CHECK_PTR(op, logits);
        CHECK_PTR(op, topkIdx);
        CHECK_PTR(op, topkWeights);
    }
    CHECK_ALIGN(op, logits, dtype_bytes(logitsDtype));
    CHECK_ALIGN(op, bias, 4);
    CHECK_ALIGN(op, topkIdx, 4);
    CHECK_ALIGN(op, topkWeights, 4);
    CHECK_ALIGN(op, topkIdxInt64, 8);
    cam::RouteGroupedArgs a{};
    a.logits = logits;
    a.row_bytes = logitsRowStride * (int64_t)dtype_bytes(logitsDtype);
    a.bias = bias;
    a.T = (int)numTokens;
    a.E = (int)numExperts;
    a.K = (int)topK;
    a.G = (int)numGroups;
    a.KG = (int)topkGroups;
    a.score = (int)scoreFunc;
    a.group_top2 = groupScore == CAMHIP_ROUTE_GROUP_TOP2;
    a.renorm = (int)renormalize;
    a.dtype = (int)logitsDtype;
    a.scaling = (float)routedScaling;
    a.topk_idx = topkIdx;
    a.topk_w = topkWeights;
    a.topk_idx64 = topkIdxInt64;
    return guarded(op, [&] {
        return cam::api_make_executor(
            0, [a](void *, hipStream_t s) { return cam::launch_route_grouped(a, s); }, workspaceSize, executor);
    });
}

camhipStatus camhipMoeRouteGrouped(void *workspace, uint64_t workspaceSize, camhipExecutor *executor, void *stream)
{
    return guarded("moe_route_grouped", [&] {
        return cam::api_run_executor("moe_route_grouped", workspace, workspaceSize, executor, stream);
    });
}

// ---------------------------------------------------------------- residual addition + norm
camhipStatus camhipAddRmsNormGetWorkspaceSize(const void *x, const void *residual, const void *weight,
                                              int64_t numTokens, int64_t hidden, int64_t xRowStride, int64_t dtype,
                                              int64_t weightDtype, int64_t outQuant, double eps, void *y,
                                              float *yScales, void *residualOut, uint64_t *workspaceSize,
                                              camhipExecutor **executor)
{
    static const char op[] = "add_rms_norm";
    CHECK_PARAM(numTokens >= 0 && numTokens <= 0x7fffffff, "%s: numTokens %lld out of [0,2^31)", op, (ll)numTokens);
    CHECK_PARAM(hidden >= 1 && hidden <= 32768, "%s: hidden %lld out of [1,32768]", op, (ll)hidden);
    CHECK_PARAM(dtype == CAMHIP_DTYPE_BF16 || dtype == CAMHIP_DTYPE_FP16, "%s: dtype %lld is neither bf16 nor fp16", op,
                (ll)dtype);
    CHECK_PARAM(weightDtype == dtype || weightDtype == CAMHIP_DTYPE_FP32,
                "%s: weightDtype %lld must be dtype or fp32", op, (ll)weightDtype);
    CHECK_PARAM(outQuant == CAMHIP_QUANT_NONE || outQuant == CAMHIP_QUANT_INT8_TOKEN ||
                    outQuant == CAMHIP_QUANT_FP8_BLOCK_KMAJOR,
                "%s: outQuant %lld not supported (0, 2 or 5)", op, (ll)outQuant);
    CHECK_PARAM(outQuant != CAMHIP_QUANT_FP8_BLOCK_KMAJOR || hidden % 128 == 0,
                "%s: fp8 rows need hidden to be a multiple of 128 (got %lld)", op, (ll)hidden);
    CHECK_PARAM(xRowStride >= hidden && xRowStride <= (int64_t)1 << 31, "%s: xRowStride %lld out of [hidden %lld,2^31]", op,
                (ll)xRowStride, (ll)hidden);
    CHECK_PARAM(eps >= 0.0 && eps <= 1.0, "%s: eps %g out of [0,1]", op, eps);
    if (numTokens > 0) {
        CHECK_PTR(op, x);
        CHECK_PTR(op, weight);
        CHECK_PTR(op, y);
        if (outQuant != CAMHIP_QUANT_NONE)
            CHECK_PTR(op, yScales);
        if (residual)
            CHECK_PTR(op, residualOut);
    }
    CHECK_ALIGN(op, x, 2);
    CHECK_ALIGN(op, residual, 2);
    CHECK_ALIGN(op, weight, dtype_bytes(weightDtype));
    CHECK_ALIGN(op, residualOut, 2);
    CHECK_ALIGN(op, y, outQuant == CAMHIP_QUANT_NONE ? 2 : 1);
    CHECK_ALIGN(op, yScales, 4);
    cam::NormArgs a{};
    a.x = static_cast<const uint16_t *>(x);
    a.x_stride = xRowStride;
    a.residual = static_cast<const uint16_t *>(residual);
    a.weight = weight;
    a.T = numTokens;
    a.H = (int)hidden;
    a.eps = (float)eps;
    a.fp16 = dtype == CAMHIP_DTYPE_FP16;
    a.weight_fp32 = weightDtype == CAMHIP_DTYPE_FP32;
    a.quant = outQuant == CAMHIP_QUANT_FP8_BLOCK_KMAJOR ? cam::QUANT_FP8_BLOCK : (int)outQuant;
    a.y = y;
    a.scales = yScales;
    a.residual_out = static_cast<uint16_t *>(residualOut);
    return guarded(op, [&] {
        return cam::api_make_executor(
            0, [a](void *, hipStream_t s) { return cam::launch_add_rms_norm(a, s); }, workspaceSize, executor);
    });
}

camhipStatus camhipAddRmsNorm(void *workspace, uint64_t workspaceSize, camhipExecutor *executor, void *stream)
{
    return guarded("add_rms_norm", [&] {
        return cam::api_run_executor("add_rms_norm", workspace, workspaceSize, executor, stream);
    });
}

// ---------------------------------------------------------------- int8 product
camhipStatus camhipQuantMatmulGetWorkspaceSize(const void *x, const float *xScale, const void *weight,
                                               const float *weightScale, const float *bias, int64_t m, int64_t n,
                                               int64_t k, int64_t outDtype, void *out, uint64_t *workspaceSize,
                                               camhipExecutor **executor)
{
    static const char op[] = "quant_matmul";
    CHECK_PARAM(m >= 0 && m <= (int64_t)1 << 20, "%s: m %lld out of [0,2^20]", op, (ll)m);
    CHECK_PARAM(n >= 1 && n <= (int64_t)1 << 20, "%s: n %lld out of [1,2^20]", op, (ll)n);
    CHECK_PARAM(k >= 16 && k <= 131056 && k % 16 == 0, "%s: k %lld must be a multiple of 16 in [16,131056]", op, (ll)k);
    CHECK_PARAM(outDtype == CAMHIP_DTYPE_BF16 || outDtype == CAMHIP_DTYPE_FP16 || outDtype == CAMHIP_DTYPE_FP32,
                "%s: outDtype %lld is not bf16, fp16 or fp32", op, (ll)outDtype);
    if (m > 0) {
        CHECK_PTR(op, x);
        CHECK_PTR(op, xScale);
        CHECK_PTR(op, weight);
        CHECK_PTR(op, weightScale);
        CHECK_PTR(op, out);
    }
    CHECK_ALIGN(op, x, 16);
    CHECK_ALIGN(op, weight, 16);
    CHECK_ALIGN(op, xScale, 4);
    CHECK_ALIGN(op, weightScale, 4);
    CHECK_ALIGN(op, bias, 4);
    CHECK_ALIGN(op, out, dtype_bytes(outDtype));
    cam::QmmArgs a{};
    a.x = static_cast<const int8_t *>(x);
    a.w = static_cast<const int8_t *>(weight);
    a.xs = xScale;
    a.ws = weightScale;
    a.bias = bias;
    a.M = m;
    a.N = (int)n;
    a.K = (int)k;
    a.out_dtype = (int)outDtype;
    a.out = out;
    return guarded(op, [&] {
        return cam::api_make_executor(
            0, [a](void *, hipStream_t s) { return cam::launch_quant_matmul(a, s); }, workspaceSize, executor);
    });
}

camhipStatus camhipQuantMatmul(void *workspace, uint64_t workspaceSize, camhipExecutor *executor, void *stream)
{
    return guarded("quant_matmul", [&] {
        return cam::api_run_executor("quant_matmul", workspace, workspaceSize, executor, stream);
    });
}

}  // extern "C"
