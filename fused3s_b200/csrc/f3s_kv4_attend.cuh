// f3s_kv4_attend.cuh -- what the kernels of attention over request pages share.
#pragma once
#include "f3s_kv4_math.cuh"
#include "f3s_kv4_plan.cuh"

namespace f3s {

// The kernel of 128-row tiles sits at its register limit (72, a few of them spilled), so
// its time moves by some percent with small changes anywhere, these fields among them.
struct AttendParams {
    const void* q;
    int64_t q_token, q_head;  // strides in elements
    int q_bf16;
    int items_cap;
    const uint8_t* pages;
    int num_pages;
    int kv_heads, heads, group;
    float scale;   // times log2(e)
    int num_requests;
    void* o;       // contiguous [rows, heads, D] of o_dtype
    int o_dtype;
    int num_tokens;
    int* status;
    float* partials;  // (rows of a tile) x (D + 2) floats per slot and K/V head; before it the places of runs
    const Kv4PlanHeader* plan;
    const int* tables;
    int64_t table_stride;
};

// True for a plan made with this call's sizes; any other's items would reach past
// this call's arrays.
__device__ __forceinline__ bool plan_fits(const AttendParams& p, const int4& counts, const int4& made_with) {
    return counts.z == p.items_cap && made_with.x == p.heads && made_with.y == p.kv_heads &&
           made_with.z == p.num_requests && made_with.w == p.num_tokens;
}

// The plan's work items; 0 if it is not this call's (which the merge reports).
__device__ __forceinline__ int plan_items(const AttendParams& p) {
    const int4* h = reinterpret_cast<const int4*>(&p.plan->num_items);
    const int4 counts = h[0], made_with = h[1];
    return plan_fits(p, counts, made_with) ? counts.x : 0;
}

// Tiles of 128 query rows on tcgen05 (f3s_kv4_prefill.cu); units: an upper bound.
int attend_tiles128(const AttendParams& p, int head_dim, int64_t units, cudaStream_t stream);

}  // namespace f3s
