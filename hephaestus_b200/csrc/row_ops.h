// row_ops.h — host launchers of the language-model row operators (norm, expert
// routing, expert order, token sampling).  They work on caller-owned device
// memory, allocate nothing and validate nothing (row_abi.cu has).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"

namespace heph {

constexpr uint32_t kMaxExperts = 1024;  // 32 a lane in expert_route
constexpr uint32_t kMaxChoices = 32;    // a lane each in expert_route
constexpr uint32_t kMaxGroups = 32;

// A matrix of adjacent columns: row r starts `stride` elements after row r-1.
struct Rows {
    const void *ptr;
    int64_t stride;
};

struct NormArgs {
    heph_row_dtype dtype;
    Rows x, residual;  // residual.ptr may be null
    const void *weight;  // may be null
    bool weight_f32;     // weight is f32 (else of dtype)
    float eps;
    uint32_t rows, cols;
    void *y;    // of dtype, or e4m3 when scales is set
    void *sum;  // x + residual, of dtype; null without residual
    float *scales;
    uint32_t group;  // columns per scale; 0 = the whole row
};
heph_status launch_rms_norm(const NormArgs &a, cudaStream_t stream);

struct NormGradArgs {
    heph_row_dtype dtype;
    Rows dy, x, dsum;  // dsum.ptr may be null
    const void *weight;
    bool weight_f32;
    float eps;
    uint32_t rows, cols;
    void *dx;
    void *dweight;      // of the weight's type; null with it
    float *partials;    // norm_grad_partials() x cols
};
uint32_t norm_grad_partials(uint32_t rows, uint32_t cols, int sm_count);
heph_status launch_rms_norm_backward(const NormGradArgs &a, int sm_count, cudaStream_t stream);

struct RouteArgs {
    heph_row_dtype dtype;
    Rows logits;
    const float *bias;  // may be null
    uint32_t rows, experts, k, groups, groups_kept, group_top;
    bool sigmoid, renormalize;
    float scale;
    float *weights;
    int32_t *picks;
};
heph_status launch_route(const RouteArgs &a, cudaStream_t stream);

struct RouteGradArgs {
    heph_row_dtype dtype;
    Rows logits, dweights, picks;
    uint32_t rows, experts, k;
    bool sigmoid, renormalize;
    float scale;
    void *dlogits;
};
heph_status launch_route_backward(const RouteGradArgs &a, cudaStream_t stream);

size_t expert_order_workspace(uint32_t count, uint32_t experts);
heph_status launch_expert_order(const int32_t *picks, uint32_t count, uint32_t experts, int32_t *offsets,
                                int32_t *order, int32_t *slot, uint32_t *workspace, cudaStream_t stream);

struct SampleArgs {
    heph_row_dtype dtype;
    Rows logits;
    const float *uniform;
    const float *temperature, *top_p, *min_p;  // one per row, or null: the scalar
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int32_t top_k_all;
    uint32_t rows, vocab;
    int64_t *tokens;
    float *probs;
};
heph_status launch_sample(const SampleArgs &a, int sm_count, cudaStream_t stream);

}  // namespace heph
