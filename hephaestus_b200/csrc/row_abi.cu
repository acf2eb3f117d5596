// row_abi.cu — the C ABI of the language-model row operators: every check of
// their arguments, the device they run on, and the launch.  A refused call
// touches no device.
#include <cfloat>
#include <cmath>
#include <exception>

#include "row_ops.h"

namespace heph {

namespace {

constexpr uint64_t kMaxRows = 0x7fffffff;   // blocks of a grid, 32-bit row numbers
constexpr uint64_t kMaxCols = 1u << 24;
constexpr uint64_t kMaxScales = 8192;       // group maxima of a row in 32 KiB of shared memory
constexpr uint64_t kMaxVocab = (1u << 22) - (1u << 16);  // sums of the limbs of masses in 32 bits (sample.cu)

size_t row_dtype_size(heph_row_dtype dt) {
    switch (dt) {
        case HEPH_ROW_F32: return 4;
        case HEPH_ROW_BF16: case HEPH_ROW_F16: return 2;
        default: return 0;
    }
}

heph_status refuse(const std::string &msg) { return fail(HEPH_INVALID_CONFIGURATION, msg); }

// Bytes [begin, end) of a matrix.
struct Span {
    uintptr_t begin = 0, end = 0;
    Span(const void *p, uint64_t rows, uint64_t cols, int64_t stride, size_t es) {
        if (!p || !rows || !cols) return;
        begin = reinterpret_cast<uintptr_t>(p);
        end = begin + ((rows - 1) * (uint64_t)stride + cols) * es;
    }
    Span(const void *p, uint64_t count, size_t es) : Span(p, 1, count, 0, es) {}
    bool overlaps(const Span &o) const { return begin < o.end && o.begin < end; }
};

// Outputs share no byte with an input or with one another.
heph_status check_apart(const char *op, std::initializer_list<Span> inputs, std::initializer_list<Span> outputs) {
    for (const Span *o = outputs.begin(); o != outputs.end(); ++o) {
        for (const Span &i : inputs)
            if (o->overlaps(i)) return refuse(std::string(op) + " outputs must not alias its inputs");
        for (const Span *q = outputs.begin(); q != o; ++q)
            if (o->overlaps(*q)) return refuse(std::string(op) + " outputs must not alias one another");
    }
    return HEPH_OK;
}

heph_status check_matrix(const char *name, const void *p, uint64_t rows, uint64_t cols, int64_t stride, size_t es) {
    if (!rows || !cols) return HEPH_OK;
    if (!p) return refuse(std::string(name) + " is null");
    if (reinterpret_cast<uintptr_t>(p) % es) return refuse(std::string(name) + " is not aligned to its element type");
    if (stride < 0) return refuse(std::string(name) + " has a negative row stride");
    if ((uint64_t)stride > (uint64_t)INT64_MAX / 16 / rows) return refuse(std::string(name) + " has a row stride out of range");
    return HEPH_OK;
}

#define HEPH_TRY(expr)                        \
    do {                                      \
        const heph_status st_ = (expr);       \
        if (st_ != HEPH_OK) return st_;       \
    } while (0)

// Makes a device current for the call and restores the caller's.
class OnDevice {
public:
    heph_status enter(int ordinal) {
        HEPH_CUDA_TRY(cudaGetDevice(&before_), HEPH_DEVICE_UNAVAILABLE, "current device query");
        if (ordinal != before_) {
            HEPH_CUDA_TRY(cudaSetDevice(ordinal), HEPH_DEVICE_UNAVAILABLE, "cudaSetDevice");
            moved_ = true;
        }
        return HEPH_OK;
    }
    ~OnDevice() {
        if (moved_) cudaSetDevice(before_);
    }

private:
    int before_ = 0;
    bool moved_ = false;
};

heph_status sm_count(int ordinal, int *out) {
    HEPH_CUDA_TRY(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, ordinal), HEPH_DEVICE_UNAVAILABLE,
                  "device query");
    return HEPH_OK;
}

// No C++ exception leaves a C entry point.
template <typename F> heph_status guarded(F &&f) noexcept {
    try {
        return f();
    } catch (...) {
        return HEPH_ALLOCATION_FAILED;  // the only source is a failed host allocation
    }
}

heph_status check_norm(const char *op, heph_row_dtype dtype, heph_row_dtype weight_dtype, const void *weight, double eps,
                       uint64_t rows, uint64_t cols) {
    if (!row_dtype_size(dtype)) return refuse(std::string(op) + " takes f32, bf16 or f16 rows");
    if (weight && weight_dtype != dtype && weight_dtype != HEPH_ROW_F32)
        return refuse(std::string(op) + " takes a weight of the rows' type or f32");
    if (!(eps >= 0.0) || std::isinf(eps)) return refuse(std::string(op) + " takes a finite eps of 0 or more");
    // The kernels have it in 32 bits, where a smaller one is 0 (and a row of zeros 0 / 0) and a larger one infinite.
    if (eps > FLT_MAX || (eps > 0.0 && eps < FLT_MIN)) return refuse(std::string(op) + " takes an eps of 0 or within the normal f32 numbers");
    if (cols == 0) return refuse(std::string(op) + " is undefined for rows of no columns");
    if (rows > kMaxRows || cols > kMaxCols) return refuse(std::string(op) + " rows or columns out of range");
    return check_matrix("weight", weight, weight ? 1 : 0, cols, 0, row_dtype_size(weight_dtype));
}

heph_status check_experts(const char *op, heph_row_dtype dtype, uint64_t rows, uint64_t experts, uint64_t k) {
    if (!row_dtype_size(dtype)) return refuse(std::string(op) + " takes f32, bf16 or f16 logits");
    if (rows > kMaxRows) return refuse(std::string(op) + " rows out of range");
    if (experts < 1 || experts > kMaxExperts)
        return refuse(std::string(op) + " takes 1 to " + std::to_string(kMaxExperts) + " experts");
    if (k < 1 || k > kMaxChoices || k > experts)
        return refuse(std::string(op) + " chooses 1 to " + std::to_string(kMaxChoices) + " of the experts");
    return HEPH_OK;
}

}  // namespace
}  // namespace heph

using namespace heph;

extern "C" heph_status heph_rms_norm(int ordinal, heph_row_dtype dtype, const void *x, int64_t x_stride, const void *residual,
                                     int64_t residual_stride, const void *weight, heph_row_dtype weight_dtype, double eps,
                                     uint64_t rows, uint64_t cols, void *y, void *sum, heph_stream stream) {
    return guarded([&]() -> heph_status {
        HEPH_TRY(check_norm("rms_norm", dtype, weight_dtype, weight, eps, rows, cols));
        const size_t es = row_dtype_size(dtype);
        HEPH_TRY(check_matrix("x", x, rows, cols, x_stride, es));
        if (!residual != !sum && rows) return refuse("rms_norm writes the sum with, and only with, a residual");
        if (residual) HEPH_TRY(check_matrix("residual", residual, rows, cols, residual_stride, es));
        HEPH_TRY(check_matrix("y", y, rows, cols, (int64_t)cols, es));
        if (sum) HEPH_TRY(check_matrix("sum", sum, rows, cols, (int64_t)cols, es));
        HEPH_TRY(check_apart("rms_norm",
                             {Span(x, rows, cols, x_stride, es), Span(residual, rows, cols, residual_stride, es),
                              Span(weight, cols, row_dtype_size(weight_dtype))},
                             {Span(y, rows * cols, es), Span(sum, rows * cols, es)}));
        if (!rows) return HEPH_OK;
        OnDevice on;
        HEPH_TRY(on.enter(ordinal));
        return launch_rms_norm({dtype, {x, x_stride}, {residual, residual_stride}, weight, weight_dtype != dtype, (float)eps,
                                (uint32_t)rows, (uint32_t)cols, y, sum, nullptr, 0},
                               static_cast<cudaStream_t>(stream));
    });
}

extern "C" heph_status heph_rms_norm_fp8(int ordinal, heph_row_dtype dtype, const void *x, int64_t x_stride,
                                         const void *residual, int64_t residual_stride, const void *weight,
                                         heph_row_dtype weight_dtype, double eps, uint64_t rows, uint64_t cols, uint32_t group,
                                         uint8_t *q, float *scales, void *sum, heph_stream stream) {
    return guarded([&]() -> heph_status {
        HEPH_TRY(check_norm("rms_norm_fp8", dtype, weight_dtype, weight, eps, rows, cols));
        if (group && (group < 16 || (group & (group - 1))))
            return refuse("rms_norm_fp8 takes groups of a power of two of 16 or more columns");
        const uint64_t scales_per_row = group && group < cols ? (cols + group - 1) / group : 1;
        if (scales_per_row > kMaxScales)
            return refuse("rms_norm_fp8 takes at most " + std::to_string(kMaxScales) + " groups a row");
        const size_t es = row_dtype_size(dtype);
        HEPH_TRY(check_matrix("x", x, rows, cols, x_stride, es));
        if (!residual != !sum && rows) return refuse("rms_norm_fp8 writes the sum with, and only with, a residual");
        if (residual) HEPH_TRY(check_matrix("residual", residual, rows, cols, residual_stride, es));
        HEPH_TRY(check_matrix("q", q, rows, cols, (int64_t)cols, 1));
        HEPH_TRY(check_matrix("scales", scales, rows, scales_per_row, (int64_t)scales_per_row, 4));
        if (sum) HEPH_TRY(check_matrix("sum", sum, rows, cols, (int64_t)cols, es));
        HEPH_TRY(check_apart("rms_norm_fp8",
                             {Span(x, rows, cols, x_stride, es), Span(residual, rows, cols, residual_stride, es),
                              Span(weight, cols, row_dtype_size(weight_dtype))},
                             {Span(q, rows * cols, 1), Span(scales, rows * scales_per_row, 4), Span(sum, rows * cols, es)}));
        if (!rows) return HEPH_OK;
        OnDevice on;
        HEPH_TRY(on.enter(ordinal));
        return launch_rms_norm({dtype, {x, x_stride}, {residual, residual_stride}, weight, weight_dtype != dtype, (float)eps,
                                (uint32_t)rows, (uint32_t)cols, q, sum, scales, group},
                               static_cast<cudaStream_t>(stream));
    });
}

extern "C" heph_status heph_rms_norm_backward_workspace(int ordinal, uint64_t rows, uint64_t cols, uint64_t *out_bytes) {
    return guarded([&]() -> heph_status {
        if (!out_bytes) return refuse("null output");
        if (rows > kMaxRows || cols > kMaxCols) return refuse("rms_norm_backward rows or columns out of range");
        int sms = 0;
        HEPH_TRY(sm_count(ordinal, &sms));
        *out_bytes = (uint64_t)norm_grad_partials((uint32_t)rows, (uint32_t)cols, sms) * cols * sizeof(float);
        return HEPH_OK;
    });
}

extern "C" heph_status heph_rms_norm_backward(int ordinal, heph_row_dtype dtype, const void *dy, int64_t dy_stride,
                                              const void *x, int64_t x_stride, const void *dsum, int64_t dsum_stride,
                                              const void *weight, heph_row_dtype weight_dtype, double eps, uint64_t rows,
                                              uint64_t cols, void *dx, void *dweight, void *workspace,
                                              uint64_t workspace_bytes, heph_stream stream) {
    return guarded([&]() -> heph_status {
        HEPH_TRY(check_norm("rms_norm_backward", dtype, weight_dtype, weight, eps, rows, cols));
        const size_t es = row_dtype_size(dtype), ws = row_dtype_size(weight_dtype);
        HEPH_TRY(check_matrix("dy", dy, rows, cols, dy_stride, es));
        HEPH_TRY(check_matrix("x", x, rows, cols, x_stride, es));
        if (dsum) HEPH_TRY(check_matrix("dsum", dsum, rows, cols, dsum_stride, es));
        HEPH_TRY(check_matrix("dx", dx, rows, cols, (int64_t)cols, es));
        if (dweight && !weight) return refuse("rms_norm_backward has no weight to differentiate by");
        if (dweight) HEPH_TRY(check_matrix("dweight", dweight, 1, cols, 0, ws));
        HEPH_TRY(check_apart("rms_norm_backward",
                             {Span(dy, rows, cols, dy_stride, es), Span(x, rows, cols, x_stride, es),
                              Span(dsum, rows, cols, dsum_stride, es), Span(weight, cols, ws)},
                             {Span(dx, rows * cols, es), Span(dweight, cols, ws), Span(workspace, workspace_bytes, 1)}));
        if (!rows && !dweight) return HEPH_OK;
        if (reinterpret_cast<uintptr_t>(workspace) % 16) return refuse("rms_norm_backward workspace is not aligned to 16 bytes");
        OnDevice on;
        HEPH_TRY(on.enter(ordinal));
        int sms = 0;
        HEPH_TRY(sm_count(ordinal, &sms));
        const uint64_t need = dweight ? (uint64_t)norm_grad_partials((uint32_t)rows, (uint32_t)cols, sms) * cols * sizeof(float) : 0;
        if (need && (!workspace || workspace_bytes < need))
            return refuse("rms_norm_backward needs a workspace of " + std::to_string(need) + " bytes");
        return launch_rms_norm_backward({dtype, {dy, dy_stride}, {x, x_stride}, {dsum, dsum_stride}, weight,
                                         weight_dtype != dtype, (float)eps, (uint32_t)rows, (uint32_t)cols, dx, dweight,
                                         static_cast<float *>(workspace)},
                                        sms, static_cast<cudaStream_t>(stream));
    });
}

extern "C" heph_status heph_route_experts(int ordinal, heph_row_dtype dtype, const void *logits, int64_t stride,
                                          const float *bias, uint64_t rows, uint32_t experts, uint32_t k,
                                          heph_route_score score, uint32_t groups, uint32_t groups_kept, uint32_t group_top,
                                          int renormalize, float scale, float *weights, int32_t *picks, heph_stream stream) {
    return guarded([&]() -> heph_status {
        HEPH_TRY(check_experts("route_experts", dtype, rows, experts, k));
        if (score != HEPH_ROUTE_SOFTMAX && score != HEPH_ROUTE_SIGMOID) return refuse("unknown routing score");
        if (groups < 1 || groups > kMaxGroups || experts % groups)
            return refuse("route_experts takes 1 to " + std::to_string(kMaxGroups) + " groups of equal size");
        if (groups_kept < 1 || groups_kept > groups) return refuse("route_experts keeps 1 to all of the groups");
        if (group_top != 1 && group_top != 2) return refuse("route_experts values a group by its one or two best experts");
        if ((uint64_t)k > (uint64_t)groups_kept * (experts / groups))
            return refuse("route_experts cannot choose " + std::to_string(k) + " experts from the groups it keeps");
        const size_t es = row_dtype_size(dtype);
        HEPH_TRY(check_matrix("logits", logits, rows, experts, stride, es));
        if (bias) HEPH_TRY(check_matrix("bias", bias, 1, experts, 0, 4));
        HEPH_TRY(check_matrix("weights", weights, rows, k, k, 4));
        HEPH_TRY(check_matrix("picks", picks, rows, k, k, 4));
        HEPH_TRY(check_apart("route_experts", {Span(logits, rows, experts, stride, es), Span(bias, experts, 4)},
                             {Span(weights, rows * k, 4), Span(picks, rows * k, 4)}));
        if (!rows) return HEPH_OK;
        OnDevice on;
        HEPH_TRY(on.enter(ordinal));
        return launch_route({dtype, {logits, stride}, bias, (uint32_t)rows, experts, k, groups, groups_kept, group_top,
                             score == HEPH_ROUTE_SIGMOID, renormalize != 0, scale, weights, picks},
                            static_cast<cudaStream_t>(stream));
    });
}

extern "C" heph_status heph_route_experts_backward(int ordinal, heph_row_dtype dtype, const float *dweights,
                                                   int64_t dweights_stride, const void *logits, int64_t stride,
                                                   const int32_t *picks, int64_t picks_stride, uint64_t rows, uint32_t experts,
                                                   uint32_t k, heph_route_score score, int renormalize, float scale,
                                                   void *dlogits, heph_stream stream) {
    return guarded([&]() -> heph_status {
        HEPH_TRY(check_experts("route_experts_backward", dtype, rows, experts, k));
        if (score != HEPH_ROUTE_SOFTMAX && score != HEPH_ROUTE_SIGMOID) return refuse("unknown routing score");
        const size_t es = row_dtype_size(dtype);
        HEPH_TRY(check_matrix("dweights", dweights, rows, k, dweights_stride, 4));
        HEPH_TRY(check_matrix("logits", logits, rows, experts, stride, es));
        HEPH_TRY(check_matrix("picks", picks, rows, k, picks_stride, 4));
        HEPH_TRY(check_matrix("dlogits", dlogits, rows, experts, experts, es));
        HEPH_TRY(check_apart("route_experts_backward",
                             {Span(dweights, rows, k, dweights_stride, 4), Span(logits, rows, experts, stride, es),
                              Span(picks, rows, k, picks_stride, 4)},
                             {Span(dlogits, rows * experts, es)}));
        if (!rows) return HEPH_OK;
        OnDevice on;
        HEPH_TRY(on.enter(ordinal));
        return launch_route_backward({dtype, {logits, stride}, {dweights, dweights_stride}, {picks, picks_stride},
                                      (uint32_t)rows, experts, k, score == HEPH_ROUTE_SIGMOID, renormalize != 0, scale, dlogits},
                                     static_cast<cudaStream_t>(stream));
    });
}

extern "C" heph_status heph_expert_order_workspace(uint64_t count, uint32_t experts, uint64_t *out_bytes) {
    return guarded([&]() -> heph_status {
        if (!out_bytes) return refuse("null output");
        if (count > kMaxRows || experts > kMaxExperts) return refuse("expert_order pairs or experts out of range");
        *out_bytes = expert_order_workspace((uint32_t)count, experts);
        return HEPH_OK;
    });
}

extern "C" heph_status heph_expert_order(int ordinal, const int32_t *picks, uint64_t count, uint32_t experts,
                                         int32_t *offsets, int32_t *order, int32_t *slot, void *workspace,
                                         uint64_t workspace_bytes, heph_stream stream) {
    return guarded([&]() -> heph_status {
        if (experts < 1 || experts > kMaxExperts)
            return refuse("expert_order takes 1 to " + std::to_string(kMaxExperts) + " experts");
        if (count > kMaxRows) return refuse("expert_order pairs out of range");
        HEPH_TRY(check_matrix("picks", picks, 1, count, 0, 4));
        HEPH_TRY(check_matrix("offsets", offsets, 1, experts + 1, 0, 4));
        HEPH_TRY(check_matrix("order", order, 1, count, 0, 4));
        HEPH_TRY(check_matrix("slot", slot, 1, count, 0, 4));
        HEPH_TRY(check_apart("expert_order", {Span(picks, count, 4)},
                             {Span(offsets, experts + 1, 4), Span(order, count, 4), Span(slot, count, 4),
                              Span(workspace, workspace_bytes, 1)}));
        const uint64_t need = expert_order_workspace((uint32_t)count, experts);
        if (need && (!workspace || workspace_bytes < need))
            return refuse("expert_order needs a workspace of " + std::to_string(need) + " bytes");
        if (reinterpret_cast<uintptr_t>(workspace) % 16) return refuse("expert_order workspace is not aligned to 16 bytes");
        OnDevice on;
        HEPH_TRY(on.enter(ordinal));
        return launch_expert_order(picks, (uint32_t)count, experts, offsets, order, slot, static_cast<uint32_t *>(workspace),
                                   static_cast<cudaStream_t>(stream));
    });
}

extern "C" heph_status heph_sample_tokens(int ordinal, heph_row_dtype dtype, const void *logits, int64_t stride, uint64_t rows,
                                          uint32_t vocab, const float *uniform, const float *temperature,
                                          double temperature_all, const int32_t *top_k, int32_t top_k_all, const float *top_p,
                                          double top_p_all, const float *min_p, double min_p_all, int64_t *tokens, float *probs,
                                          heph_stream stream) {
    return guarded([&]() -> heph_status {
        if (!row_dtype_size(dtype)) return refuse("sample_tokens takes f32, bf16 or f16 logits");
        if (vocab < 1 || vocab > kMaxVocab) return refuse("sample_tokens vocabulary out of range");
        if (rows > kMaxRows / 8) return refuse("sample_tokens rows out of range");
        if (!temperature && !(temperature_all >= 0.0 && std::isfinite(temperature_all)))
            return refuse("sample_tokens takes a finite temperature of 0 or more");
        if (!top_k && top_k_all < 0) return refuse("sample_tokens takes a top_k of 0 (off) or more");
        if (!top_p && !(top_p_all >= 0.0 && top_p_all <= 1.0)) return refuse("sample_tokens takes a top_p in [0, 1]");
        if (!min_p && !(min_p_all >= 0.0 && min_p_all <= 1.0)) return refuse("sample_tokens takes a min_p in [0, 1]");
        const size_t es = row_dtype_size(dtype);
        HEPH_TRY(check_matrix("logits", logits, rows, vocab, stride, es));
        HEPH_TRY(check_matrix("uniform", uniform, 1, rows, 0, 4));
        if (temperature) HEPH_TRY(check_matrix("temperature", temperature, 1, rows, 0, 4));
        if (top_k) HEPH_TRY(check_matrix("top_k", top_k, 1, rows, 0, 4));
        if (top_p) HEPH_TRY(check_matrix("top_p", top_p, 1, rows, 0, 4));
        if (min_p) HEPH_TRY(check_matrix("min_p", min_p, 1, rows, 0, 4));
        HEPH_TRY(check_matrix("tokens", tokens, 1, rows, 0, 8));
        HEPH_TRY(check_matrix("probs", probs, 1, rows, 0, 4));
        HEPH_TRY(check_apart("sample_tokens",
                             {Span(logits, rows, vocab, stride, es), Span(uniform, rows, 4), Span(temperature, rows, 4),
                              Span(top_k, rows, 4), Span(top_p, rows, 4), Span(min_p, rows, 4)},
                             {Span(tokens, rows, 8), Span(probs, rows, 4)}));
        if (!rows) return HEPH_OK;
        OnDevice on;
        HEPH_TRY(on.enter(ordinal));
        int sms = 0;
        HEPH_TRY(sm_count(ordinal, &sms));
        return launch_sample({dtype, {logits, stride}, uniform, temperature, top_p, min_p, top_k, temperature_all, top_p_all,
                              min_p_all, top_k_all, (uint32_t)rows, vocab, tokens, probs},
                             sms, static_cast<cudaStream_t>(stream));
    });
}
