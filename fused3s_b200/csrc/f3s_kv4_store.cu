// f3s_kv4_store.cu -- rows of K and V into 4-bit pages by a slot map, and back.
//
// Store, per row x of D channels (one token, one K/V head):
//   lo = min(0, min x), hi = max(0, max x)
//   s  = fp16((hi - lo) / 15), at least 2^-24, at most 65504
//   z  = clamp(rint(-lo / s), 0, 15)
//   u_c = clamp(rint(x_c / s) + z, 0, 15),  standing for s * (u_c - z)
// rint rounds halves to even.  x and s have 11 significant bits or fewer, so a
// quotient next to a half-integer differs from it by 2^-12 of its value or is
// it exactly: a correctly rounded fp32 division puts every value on the right
// side.  A row with a NaN stands for NaN (its scale is NaN).
//
// Both kernels are bound by HBM: 2 bytes per value on the wide side, (D + 8) / 2D
// on the other.  A group of D / 8 lanes owns a row and each lane 8 channels, so
// the wide side moves 16 bytes per lane and the K codes 4.
#include <cuda_bf16.h>
#include "f3s_internal.cuh"
#include "f3s_kv4.cuh"

namespace f3s {

struct Kv4RowsParams {
    const void* k;  // [num_tokens, kv_heads, D] with strides in elements (store: input)
    const void* v;
    int64_t k_token, k_head, v_token, v_head;
    void* k_out;  // load: output, contiguous
    void* v_out;
    const int* slots;
    uint8_t* pages;
    int64_t num_slots;  // num_pages * 16
    int64_t rows;       // num_tokens * kv_heads
    int kv_heads;
    int* status;
};

template <class T>
__device__ __forceinline__ void unpack8(const uint4 w, float (&x)[8]);
template <>
__device__ __forceinline__ void unpack8<__half>(const uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

// Codes of a row's 8 channels (in this lane) and its scale and zero (in every
// lane of the row's group of LANES).
template <int LANES>
__device__ __forceinline__ void quantise8(const float (&x)[8], uint32_t (&u)[8], __half& scale, float& zero) {
    float lo = 0.f, hi = 0.f;
    int nan = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        nan |= x[i] != x[i];
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        nan |= __shfl_xor_sync(0xffffffffu, nan, o);
    }
    const float raw = __half2float(__float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
    const float s = fminf(fmaxf(raw, kKv4MinScale), kKv4MaxScale);
    const float inv = __frcp_rn(s);
    // x / s, correctly rounded where it is a half-integer and to 1 ulp
    // elsewhere: the residual of the first quotient is exact
    auto divide = [&](float a) {
        const float q = a * inv;
        const float r = fmaf(fmaf(-q, s, a), inv, q);
        return fabsf(a) <= 3.0e38f ? r : q;  // an infinity has no residual
    };
    zero = nan ? 0.f : fminf(rintf(divide(-lo)), 15.f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        u[i] = nan ? 0u : (uint32_t)fminf(fmaxf(rintf(divide(x[i])) + zero, 0.f), 15.f);
    scale = nan ? __ushort_as_half(0x7fffu) : __float2half_rn(s);
}

__device__ __forceinline__ uint32_t half2_bits(__half a, __half b) {
    return (uint32_t)__half_as_ushort(a) | ((uint32_t)__half_as_ushort(b) << 16);
}

template <int D, class T>
__global__ void __launch_bounds__(256) k_kv4_store(const Kv4RowsParams p) {
    constexpr int LANES = D / 8;  // lanes per row
    const int sub = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool live = row < p.rows;
    const int64_t token = live ? row / p.kv_heads : 0;
    const int head = live ? (int)(row - token * p.kv_heads) : 0;
    const int64_t slot = live ? p.slots[token] : -1;
    const bool ok = slot >= 0 && slot < p.num_slots;
    if (live && !ok && slot != -1 && sub == 0) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
    uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
    if (ok) {
        kw = __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(p.k) + token * p.k_token + head * p.k_head) + sub);
        vw = __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + token * p.v_token + head * p.v_head) + sub);
    }
    float x[8];
    uint32_t uk[8], uv[8];
    __half ks, vs;
    float kz, vz;
    unpack8<T>(kw, x);
    quantise8<LANES>(x, uk, ks, kz);
    unpack8<T>(vw, x);
    quantise8<LANES>(x, uv, vs, vz);
    if (!ok) return;
    const int tok = (int)(slot & 15);
    uint8_t* rec = p.pages + ((slot >> 4) * p.kv_heads + head) * kv4_record_bytes(D);
    uint32_t word = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) word |= uk[2 * n] << (4 * n) | uk[2 * n + 1] << (4 * n + 16);
    *reinterpret_cast<uint32_t*>(rec + kv4_k_off(D, tok, sub)) = word;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t h = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) h |= uv[4 * i + n] << (4 * n);
        const int c = 8 * sub + 4 * i;
        *reinterpret_cast<uint16_t*>(rec + kv4_v_off(D, tok, c / (D / 8), c % (D / 8) / 4)) = (uint16_t)h;
    }
    if (sub == 0)
        *reinterpret_cast<uint2*>(rec + kv4_scale_off(D, tok)) =
            make_uint2(half2_bits(ks, __float2half_rn(kz)), half2_bits(vs, __float2half_rn(vz)));
}

template <class T>
__device__ __forceinline__ void store8(T* dst, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* dst, const float (&x)[8]) {
    __stcs(reinterpret_cast<float4*>(dst), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4*>(dst) + 1, make_float4(x[4], x[5], x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<__half>(__half* dst, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_half2(x[2 * i], x[2 * i + 1]);
    __stcs(reinterpret_cast<uint4*>(dst), make_uint4(w[0], w[1], w[2], w[3]));
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* dst, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    __stcs(reinterpret_cast<uint4*>(dst), make_uint4(w[0], w[1], w[2], w[3]));
}

template <int D, class T>
__global__ void __launch_bounds__(256) k_kv4_load(const Kv4RowsParams p) {
    constexpr int LANES = D / 8;
    const int sub = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (row >= p.rows) return;
    const int64_t token = row / p.kv_heads;
    const int head = (int)(row - token * p.kv_heads);
    const int64_t slot = p.slots[token];
    const bool ok = slot >= 0 && slot < p.num_slots;
    if (!ok && slot != -1 && sub == 0) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
    float k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.f;
    if (ok) {
        const int tok = (int)(slot & 15);
        const uint8_t* rec = p.pages + ((slot >> 4) * p.kv_heads + head) * kv4_record_bytes(D);
        const uint32_t word = *reinterpret_cast<const uint32_t*>(rec + kv4_k_off(D, tok, sub));
        uint32_t h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = 8 * sub + 4 * i;
            h[i] = *reinterpret_cast<const uint16_t*>(rec + kv4_v_off(D, tok, c / (D / 8), c % (D / 8) / 4));
        }
        const uint2 sc = *reinterpret_cast<const uint2*>(rec + kv4_scale_off(D, tok));
        const float2 ks = __half22float2(*reinterpret_cast<const __half2*>(&sc.x));
        const float2 vs = __half22float2(*reinterpret_cast<const __half2*>(&sc.y));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            k[2 * n] = ks.x * ((float)((word >> (4 * n)) & 15u) - ks.y);
            k[2 * n + 1] = ks.x * ((float)((word >> (4 * n + 16)) & 15u) - ks.y);
            v[n] = vs.x * ((float)((h[0] >> (4 * n)) & 15u) - vs.y);
            v[4 + n] = vs.x * ((float)((h[1] >> (4 * n)) & 15u) - vs.y);
        }
    }
    store8<T>(static_cast<T*>(p.k_out) + row * D + sub * 8, k);
    store8<T>(static_cast<T*>(p.v_out) + row * D + sub * 8, v);
}

// Arguments that store and load share.
static int check_rows(const int* slots, int64_t num_tokens, const void* pages, int32_t num_pages, int32_t kv_heads,
                      int32_t head_dim, const void* ws, size_t ws_bytes) {
    if (num_tokens < 0 || num_pages < 0 || kv_heads <= 0) return F3S_ERR_INVALID_VALUE;
    if (head_dim != 64 && head_dim != 128) return F3S_ERR_UNSUPPORTED;
    if ((int64_t)num_pages * 16 > INT32_MAX) return F3S_ERR_TOO_LARGE;
    if (num_tokens * kv_heads > (int64_t)INT32_MAX * 8) return F3S_ERR_TOO_LARGE;  // blocks of 16 rows or more
    if (!ws) return F3S_ERR_INVALID_VALUE;
    if (ws_bytes < kWsHeaderBytes) return F3S_ERR_WORKSPACE;
    if (num_tokens == 0) return F3S_SUCCESS;
    if (!slots || !pages || (reinterpret_cast<uintptr_t>(pages) & 15)) return F3S_ERR_INVALID_VALUE;
    return F3S_SUCCESS;
}


}  // namespace f3s

extern "C" {

size_t f3s_kv4_record_bytes(int32_t head_dim) {
    return head_dim == 64 || head_dim == 128 ? (size_t)f3s::kv4_record_bytes(head_dim) : 0;
}

int f3s_kv4_store(const void* d_K, const void* d_V, int32_t dtype, int64_t k_token_stride, int64_t k_head_stride,
                  int64_t v_token_stride, int64_t v_head_stride, const int32_t* d_slots, int64_t num_tokens,
                  void* d_pages, int32_t num_pages, int32_t kv_heads, int32_t head_dim, void* d_workspace,
                  size_t workspace_bytes, f3s_stream_t stream) {
    f3s::NvtxRange nvtx_("f3s_kv4_store");
    if (dtype != F3S_OUT_F16 && dtype != F3S_OUT_BF16) return F3S_ERR_INVALID_VALUE;
    const int rc = f3s::check_rows(d_slots, num_tokens, d_pages, num_pages, kv_heads, head_dim, d_workspace,
                                   workspace_bytes);
    if (rc != F3S_SUCCESS || num_tokens == 0) return rc;
    auto bad = [](const void* x) { return !x || (reinterpret_cast<uintptr_t>(x) & 15) != 0; };
    if (bad(d_K) || bad(d_V) || ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7))
        return F3S_ERR_INVALID_VALUE;
    f3s::Kv4RowsParams p{};
    p.k = d_K;
    p.v = d_V;
    p.k_token = k_token_stride;
    p.k_head = k_head_stride;
    p.v_token = v_token_stride;
    p.v_head = v_head_stride;
    p.slots = d_slots;
    p.pages = static_cast<uint8_t*>(d_pages);
    p.num_slots = (int64_t)num_pages * 16;
    p.rows = num_tokens * kv_heads;
    p.kv_heads = kv_heads;
    p.status = &static_cast<f3s::WsHeader*>(d_workspace)->status;
    const int per = 256 / (head_dim / 8);
    const unsigned grid = (unsigned)((p.rows + per - 1) / per);
    cudaStream_t s = (cudaStream_t)stream;
    const bool half = dtype == F3S_OUT_F16;
    if (head_dim == 64 && half) f3s::k_kv4_store<64, __half><<<grid, 256, 0, s>>>(p);
    else if (head_dim == 64) f3s::k_kv4_store<64, __nv_bfloat16><<<grid, 256, 0, s>>>(p);
    else if (half) f3s::k_kv4_store<128, __half><<<grid, 256, 0, s>>>(p);
    else f3s::k_kv4_store<128, __nv_bfloat16><<<grid, 256, 0, s>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

int f3s_kv4_load(const void* d_pages, int32_t num_pages, int32_t kv_heads, int32_t head_dim, const int32_t* d_slots,
                 int64_t num_tokens, void* d_K, void* d_V, int32_t dtype, void* d_workspace, size_t workspace_bytes,
                 f3s_stream_t stream) {
    f3s::NvtxRange nvtx_("f3s_kv4_load");
    if (dtype != F3S_OUT_F32 && dtype != F3S_OUT_F16 && dtype != F3S_OUT_BF16) return F3S_ERR_INVALID_VALUE;
    const int rc = f3s::check_rows(d_slots, num_tokens, d_pages, num_pages, kv_heads, head_dim, d_workspace,
                                   workspace_bytes);
    if (rc != F3S_SUCCESS || num_tokens == 0) return rc;
    auto bad = [](const void* x) { return !x || (reinterpret_cast<uintptr_t>(x) & 15) != 0; };
    if (bad(d_K) || bad(d_V)) return F3S_ERR_INVALID_VALUE;
    f3s::Kv4RowsParams p{};
    p.k_out = d_K;
    p.v_out = d_V;
    p.slots = d_slots;
    p.pages = const_cast<uint8_t*>(static_cast<const uint8_t*>(d_pages));
    p.num_slots = (int64_t)num_pages * 16;
    p.rows = num_tokens * kv_heads;
    p.kv_heads = kv_heads;
    p.status = &static_cast<f3s::WsHeader*>(d_workspace)->status;
    const int per = 256 / (head_dim / 8);
    const unsigned grid = (unsigned)((p.rows + per - 1) / per);
    cudaStream_t s = (cudaStream_t)stream;
    if (head_dim == 64) {
        if (dtype == F3S_OUT_F16) f3s::k_kv4_load<64, __half><<<grid, 256, 0, s>>>(p);
        else if (dtype == F3S_OUT_BF16) f3s::k_kv4_load<64, __nv_bfloat16><<<grid, 256, 0, s>>>(p);
        else f3s::k_kv4_load<64, float><<<grid, 256, 0, s>>>(p);
    } else {
        if (dtype == F3S_OUT_F16) f3s::k_kv4_load<128, __half><<<grid, 256, 0, s>>>(p);
        else if (dtype == F3S_OUT_BF16) f3s::k_kv4_load<128, __nv_bfloat16><<<grid, 256, 0, s>>>(p);
        else f3s::k_kv4_load<128, float><<<grid, 256, 0, s>>>(p);
    }
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

}  // extern "C"
