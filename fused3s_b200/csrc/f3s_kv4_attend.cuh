// f3s_kv4_attend.cuh -- what the kernels of attention over request pages share.
#pragma once
#include "f3s_kv4_math.cuh"
#include "f3s_kv4_plan.cuh"

namespace f3s {

struct AttendParams {
    const void* q;
    int64_t q_token, q_head;  // strides in elements
    int q_bf16;
    const uint8_t* pages;
    int num_pages;
    int kv_heads, heads, group;
    float scale;   // times log2(e)
    void* o;       // contiguous [rows, heads, D] of o_dtype
    int o_dtype;
    int* status;
    float* partials;  // (rows of a tile) x (D + 2) floats per slot and K/V head
    const Kv4PlanHeader* plan;
    const int* tables;
    int64_t table_stride;
};

// Tiles of 128 query rows on tcgen05 (f3s_kv4_prefill.cu); units: an upper bound.
int attend_tiles128(const AttendParams& p, int head_dim, int64_t units, cudaStream_t stream);

}  // namespace f3s
