// Serving rows: one step of a server over a paged cache (page plan, rotary
// positions with the cache write, tree attention, logit rules). All launch on
// the device's stream and return without synchronising. The host side has
// checked the geometry (capi_serving.cu); values that live on the device are
// checked by the kernels.
#pragma once

#include "../../include/nert_b200.h"
#include "ops.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace nb2 {

struct PagePlanArgs {
    nb2_page_plan_geom g;
    const int32_t* seq_lens;
    const int32_t* new_lens;
    const int32_t* free_blocks;
    const int32_t* free_head;
    const int32_t* parents;
    int32_t* table;
    int32_t* new_total;
    int32_t* offsets;
    int32_t* free_head_out;
    int32_t* slots;
    int32_t* positions;
    uint32_t* mask;
    int* err;
};
constexpr int64_t kPlanMaxBatch = 8192;
constexpr int64_t kPlanMaxWords = 32;
void page_plan(nb2_device* dev, PagePlanArgs a);

struct RopeArgs {
    nb2_rope_geom g;
    const void* q;
    const void* k;
    const void* v;
    const float* table;
    const int32_t* positions;
    const int32_t* slots;
    void* q_out;
    void* k_out;
    void* k_cache;
    void* v_cache;
    int* err;
};
void rope_append(nb2_device* dev, RopeArgs a);

struct TreeAttnArgs {
    nb2_tree_attn_geom g;
    const void* q;
    const void* kc;
    const void* vc;
    const int32_t* table;
    const int32_t* total;
    const int32_t* offsets;
    const uint32_t* mask; // null: a chain
    void* out;
    float* lse; // may be null
    int* err;
};
void tree_attention(nb2_device* dev, TreeAttnArgs a);

struct LogitsArgs {
    nb2_logits_geom g;
    const void* logits;
    void* out;
    const int32_t* row_request;
    const int32_t* prompt_ids;
    const int32_t* prompt_offsets;
    const int32_t* output_ids;
    const int32_t* output_offsets;
    const float* repetition;
    const float* presence;
    const float* frequency;
    const int32_t* bias_ids;
    const float* bias_values;
    const int32_t* bias_offsets;
    const uint32_t* grammar;
    const int32_t* grammar_rows;
    int* err;
};
void logits_process(nb2_device* dev, LogitsArgs a);

// ---- element access -------------------------------------------------------

inline int64_t dtype_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// V elements of T moved as one access when aligned to their size.
template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
    T e[V];
};

__device__ __forceinline__ void record_error(int* err, int code) { atomicExch(err, code); }

} // namespace nb2
