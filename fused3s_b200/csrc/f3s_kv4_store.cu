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
// What they cannot do without is HBM traffic: 2 bytes per value on the wide side,
// (D + 8) / 2D on the other.  16,381 tokens of 8 heads, D = 128, bf16 (85 MB each way):
// store 21.8 us, load 19 us, 3.9 and 4.5 TB/s, 61 and 70 % of a copy's rate; what keeps
// them from more has not been found.
#include <type_traits>
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
    int64_t num_tokens;
    int kv_heads;
    int* status;
};

// Two 16-bit values as fp32, in one 64-bit register.
template <class T>
__device__ __forceinline__ uint64_t unpack2(uint32_t u) {
    float2 f;
    if constexpr (std::is_same_v<T, __half>) f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    else f = make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(f.x), "f"(f.y));
    return d;
}

// The larger (smaller) of two values each, NaN if one is.
template <class T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (std::is_same_v<T, __half>) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <class T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (std::is_same_v<T, __half>) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t twice(float a) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %1};" : "=l"(d) : "f"(a));
    return d;
}

// 2^23 + 2^22: added to a number of few bits, it leaves the nearest whole
// number (halves to even) in the low bits.
constexpr float kWhole = 12582912.f;

// The CH channels of a row that this lane holds, as pairs of codes: channel 2i
// in the low half of code[i], 2i + 1 in the high one.  Scale and zero are the
// row's, in each of its 8 lanes.
//
// x / s is computed as q + (x - q s) / s with q = x * (1 / s), a quotient corrected by
// its residual (P. Markstein, Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990): the residual is exact in a fused multiply-add, so
// the result is exact where it is a half-integer and off by 1 ulp at most elsewhere,
// and rounding it to a whole number is right.
template <class T, int CH>
__device__ __forceinline__ void quantise(const uint32_t (&raw)[CH / 2], uint32_t (&code)[CH / 2], __half& scale, float& zero) {
    uint32_t lo2 = 0, hi2 = 0;
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
        lo2 = min2<T>(lo2, raw[i]);
        hi2 = max2<T>(hi2, raw[i]);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        lo2 = min2<T>(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
        hi2 = max2<T>(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
    }
    lo2 = min2<T>(lo2, lo2 >> 16 | lo2 << 16);
    hi2 = max2<T>(hi2, hi2 >> 16 | hi2 << 16);
    float lo, hi;
    if constexpr (std::is_same_v<T, __half>) {
        lo = __half22float2(*reinterpret_cast<const __half2*>(&lo2)).x;
        hi = __half22float2(*reinterpret_cast<const __half2*>(&hi2)).x;
    } else {
        lo = __uint_as_float(lo2 << 16);
        hi = __uint_as_float(hi2 << 16);
    }
    const bool nan = hi != hi;
    const float span = __fsub_rn(hi, lo);
    const float scaled = __half2float(__float2half_rn(__fdiv_rn(span, 15.f)));
    const float s = nan ? 1.f : fminf(fmaxf(scaled, kKv4MinScale), kKv4MaxScale);
    const float inv = __frcp_rn(s);
    {
        const float low = nan ? 0.f : fmaxf(lo, -3.0e38f), q = -low * inv;
        zero = fminf(rintf(fmaf(fmaf(-q, s, -low), inv, q)), 15.f);
    }
    const uint64_t inv2 = twice(inv), minus_s = twice(-s), whole = twice(kWhole), z2 = twice(zero);
    if (span < 15.f * kKv4MaxScale) {  // the codes are the clamp's by a step or less
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
            const uint64_t x = unpack2<T>(raw[i]), q = mul2(x, inv2);
            const uint64_t t = add2(add2(fma2(fma2(q, minus_s, x), inv2, q), whole), z2);
            uint32_t a, b, pair;
            asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(t));
            asm("prmt.b32 %0, %1, %2, 0x5410;" : "=r"(pair) : "r"(a), "r"(b));
            asm("min.relu.s16x2 %0, %1, %2;" : "=r"(code[i]) : "r"(pair), "r"(0x000f000fu));
        }
    } else {  // rare: an infinity counts as a large number, the codes of a NaN row are 0
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
            float x[2];
            uint32_t u[2];
            asm("mov.b64 {%0, %1}, %2;" : "=f"(x[0]), "=f"(x[1]) : "l"(unpack2<T>(raw[i])));
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float y = nan ? 0.f : fminf(fmaxf(x[k], -3.0e38f), 3.0e38f), q = y * inv;
                u[k] = (uint32_t)fminf(fmaxf(rintf(fmaf(fmaf(-q, s, y), inv, q)) + zero, 0.f), 15.f);
            }
            code[i] = u[0] | u[1] << 16;
        }
    }
    scale = nan ? __ushort_as_half(0x7fffu) : __float2half_rn(s);
}

__device__ __forceinline__ uint32_t half2_bits(__half a, __half b) {
    return (uint32_t)__half_as_ushort(a) | ((uint32_t)__half_as_ushort(b) << 16);
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* src, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 y = *reinterpret_cast<const uint4*>(src);
        w[0] = y.x;
        w[1] = y.y;
        w[2] = y.z;
        w[3] = y.w;
    } else if constexpr (N == 2) {
        const uint2 y = *reinterpret_cast<const uint2*>(src);
        w[0] = y.x;
        w[1] = y.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(src);
    }
}

template <int N>
__device__ __forceinline__ void store_words(uint8_t* dst, const uint32_t (&w)[N]) {
    static_assert(N == 1 || N == 2 || N == 4, "4, 8 or 16 bytes");
    if constexpr (N == 4) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (N == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
}

// Eight lanes per row, lane g with the D / 8 channels g * D / 8 ... -- the V codes
// that lie together -- and TOK consecutive tokens of one head per lane, so four
// times TOK tokens per warp.  Two consecutive tokens in an even and the
// following odd slot (most of a prompt's, wherever it starts) write their V codes
// together, 2 W words at once; others write 16-bit halves.
template <int D, class T, int TOK>
__global__ void __launch_bounds__(128) k_kv4_store(const Kv4RowsParams p) {
    constexpr int CH = D / 8, W = D / 32;  // channels per lane; V halves per lane and token
    const int lane = threadIdx.x & 31, g = lane & 7, quad = lane >> 3;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);  // (4 TOK tokens, head)
    const int64_t group = unit / p.kv_heads;
    const int head = (int)(unit - group * p.kv_heads);
    const int64_t token0 = group * 4 * TOK + quad * TOK;
    int slot[TOK];
    uint4 kw[TOK][CH / 8], vw[TOK][CH / 8];
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        const int64_t token = token0 + i;
        slot[i] = token < p.num_tokens ? p.slots[token] : -1;
        if (slot[i] < -1 || slot[i] >= p.num_slots) {
            if (g == 0) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
            slot[i] = -1;
        }
        const uint4* ks = reinterpret_cast<const uint4*>(static_cast<const T*>(p.k) + token * p.k_token + head * p.k_head + g * CH);
        const uint4* vs = reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + token * p.v_token + head * p.v_head + g * CH);
#pragma unroll
        for (int c = 0; c < CH / 8; ++c) {
            kw[i][c] = token < p.num_tokens ? __ldcs(ks + c) : make_uint4(0, 0, 0, 0);
            vw[i][c] = token < p.num_tokens ? __ldcs(vs + c) : make_uint4(0, 0, 0, 0);
        }
    }
    uint32_t half[TOK][W];  // V codes of four channels each
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        uint32_t raw[CH / 2], code[CH / 2], word[CH / 8];
        __half ks, vs;
        float kz, vz;
#pragma unroll
        for (int c = 0; c < CH / 8; ++c) {
            raw[4 * c] = kw[i][c].x;
            raw[4 * c + 1] = kw[i][c].y;
            raw[4 * c + 2] = kw[i][c].z;
            raw[4 * c + 3] = kw[i][c].w;
        }
        quantise<T, CH>(raw, code, ks, kz);
#pragma unroll
        for (int c = 0; c < CH / 8; ++c)
            word[c] = code[4 * c] + (code[4 * c + 1] << 4) + (code[4 * c + 2] << 8) + (code[4 * c + 3] << 12);
#pragma unroll
        for (int c = 0; c < CH / 8; ++c) {
            raw[4 * c] = vw[i][c].x;
            raw[4 * c + 1] = vw[i][c].y;
            raw[4 * c + 2] = vw[i][c].z;
            raw[4 * c + 3] = vw[i][c].w;
        }
        quantise<T, CH>(raw, code, vs, vz);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint32_t y = code[2 * w] + (code[2 * w + 1] << 8);  // channels 0 and 2, 1 and 3
            half[i][w] = (y + (y >> 12)) & 0xffffu;
        }
        if (slot[i] >= 0) {
            const int tok = slot[i] & 15;
            uint8_t* rec = p.pages + ((int64_t)(slot[i] >> 4) * p.kv_heads + head) * kv4_record_bytes(D);
            store_words<CH / 8>(rec + kv4_k_off(D, tok, g * (CH / 8)), word);
            if (g == 0)
                *reinterpret_cast<uint2*>(rec + kv4_scale_off(D, tok)) =
                    make_uint2(half2_bits(ks, __float2half_rn(kz)), half2_bits(vs, __float2half_rn(vz)));
        }
    }
    // the first token of the next eight lanes follows this lane's last
    const int slot_next = __shfl_down_sync(0xffffffffu, slot[0], 8);
    const int slot_prev = __shfl_up_sync(0xffffffffu, slot[TOK - 1], 8);
    uint32_t half_next[W];
#pragma unroll
    for (int w = 0; w < W; ++w) half_next[w] = __shfl_down_sync(0xffffffffu, half[0][w], 8);
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        if (slot[i] < 0) continue;
        const int after = i + 1 < TOK ? slot[i + 1 < TOK ? i + 1 : i] : quad < 3 ? slot_next : -1;
        const int before = i > 0 ? slot[i > 0 ? i - 1 : 0] : quad > 0 ? slot_prev : -1;
        uint8_t* dst = p.pages + ((int64_t)(slot[i] >> 4) * p.kv_heads + head) * kv4_record_bytes(D) +
                       kv4_v_off(D, slot[i] & 14, g, 0);
        if (slot[i] & 1) {
            if (before == slot[i] - 1) continue;  // written with the token before
        } else if (after == slot[i] + 1) {
            uint32_t both[W];
#pragma unroll
            for (int w = 0; w < W; ++w) both[w] = half[i][w] | (i + 1 < TOK ? half[i + 1 < TOK ? i + 1 : i][w] : half_next[w]) << 16;
            store_words<W>(dst, both);
            continue;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) *reinterpret_cast<uint16_t*>(dst + 4 * w + 2 * (slot[i] & 1)) = (uint16_t)half[i][w];
    }
}

template <class T, int CH>
__device__ __forceinline__ void store_row(T* dst, const float (&x)[CH]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int i = 0; i < CH / 4; ++i)
            __stcs(reinterpret_cast<float4*>(dst) + i, make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
    } else {
        uint32_t w[CH / 2];
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                w[i] = pack_half2(x[2 * i], x[2 * i + 1]);
            } else {
                const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
        }
#pragma unroll
        for (int i = 0; i < CH / 8; ++i)
            __stcs(reinterpret_cast<uint4*>(dst) + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
    }
}

// Eight lanes per row, as in the store; a lane reads the V words of its token's
// pair and takes its own half.
template <int D, class T>
__global__ void __launch_bounds__(256) k_kv4_load(const Kv4RowsParams p) {
    constexpr int CH = D / 8, W = D / 32;
    const int g = threadIdx.x & 7;
    const int64_t row = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3), token = row / p.kv_heads;
    if (token >= p.num_tokens) return;
    const int head = (int)(row - token * p.kv_heads);
    int slot = p.slots[token];
    if (slot < -1 || slot >= p.num_slots) {
        if (g == 0) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
        slot = -1;
    }
    uint32_t kw[CH / 8] = {}, vw[W] = {};
    uint2 sc = make_uint2(0, 0);
    if (slot >= 0) {
        const int tok = slot & 15;
        const uint8_t* rec = p.pages + ((int64_t)(slot >> 4) * p.kv_heads + head) * kv4_record_bytes(D);
        load_words<CH / 8>(rec + kv4_k_off(D, tok, g * (CH / 8)), kw);
        load_words<W>(rec + kv4_v_off(D, tok & 14, g, 0), vw);
        sc = *reinterpret_cast<const uint2*>(rec + kv4_scale_off(D, tok));
    }
    const float2 ks = __half22float2(*reinterpret_cast<const __half2*>(&sc.x));
    const float2 vs = __half22float2(*reinterpret_cast<const __half2*>(&sc.y));
    // 2^23 | code as a number, less 2^23 + zero, is code - zero, exactly
    const float kz = 8388608.f + ks.y, vz = 8388608.f + vs.y;
    auto value = [](uint32_t code, float z, float s) { return (__uint_as_float(0x4b000000u | code) - z) * s; };
    float x[CH];
#pragma unroll
    for (int c = 0; c < CH / 8; ++c)
#pragma unroll
        for (int n = 0; n < 8; ++n) x[8 * c + n] = value(kw[c] >> (4 * (n / 2) + 16 * (n & 1)) & 15u, kz, ks.x);
    store_row<T, CH>(static_cast<T*>(p.k_out) + row * D + g * CH, x);
    const int shift = 16 * (slot & 1);
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int n = 0; n < 4; ++n) x[4 * w + n] = value(vw[w] >> (shift + 4 * n) & 15u, vz, vs.x);
    store_row<T, CH>(static_cast<T*>(p.v_out) + row * D + g * CH, x);
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


// Two tokens per lane once that still fills the SMs (16 warps each), one where
// a step's few tokens are spread over the warps instead.  16,381 tokens of 8 heads,
// d = 128: 22 us with two, 24 with one, 26 with four (fewer blocks fit an SM).
template <int D, class T>
static void store_launch_t(const Kv4RowsParams& p, cudaStream_t s) {
    const bool many = p.num_tokens * p.kv_heads >= 8ll * 16 * num_sms_of_current_device();
    const int64_t tokens = many ? 8 : 4;  // per warp
    const int64_t units = (p.num_tokens + tokens - 1) / tokens * p.kv_heads;
    const unsigned grid = (unsigned)((units + 3) / 4);
    if (many) k_kv4_store<D, T, 2><<<grid, 128, 0, s>>>(p);
    else k_kv4_store<D, T, 1><<<grid, 128, 0, s>>>(p);
}

template <int D>
static void store_launch(const Kv4RowsParams& p, bool half, cudaStream_t s) {
    if (half) store_launch_t<D, __half>(p, s);
    else store_launch_t<D, __nv_bfloat16>(p, s);
}

template <int D>
static void load_launch(const Kv4RowsParams& p, int dtype, cudaStream_t s) {
    const int64_t rows = p.num_tokens * p.kv_heads;
    const unsigned grid = (unsigned)((rows + 31) / 32);
    if (dtype == F3S_OUT_F16) k_kv4_load<D, __half><<<grid, 256, 0, s>>>(p);
    else if (dtype == F3S_OUT_BF16) k_kv4_load<D, __nv_bfloat16><<<grid, 256, 0, s>>>(p);
    else k_kv4_load<D, float><<<grid, 256, 0, s>>>(p);
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
    p.num_tokens = num_tokens;
    p.kv_heads = kv_heads;
    p.status = &static_cast<f3s::WsHeader*>(d_workspace)->status;
    cudaStream_t s = (cudaStream_t)stream;
    if (head_dim == 64) f3s::store_launch<64>(p, dtype == F3S_OUT_F16, s);
    else f3s::store_launch<128>(p, dtype == F3S_OUT_F16, s);
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
    p.num_tokens = num_tokens;
    p.kv_heads = kv_heads;
    p.status = &static_cast<f3s::WsHeader*>(d_workspace)->status;
    cudaStream_t s = (cudaStream_t)stream;
    if (head_dim == 64) f3s::load_launch<64>(p, dtype, s);
    else f3s::load_launch<128>(p, dtype, s);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

}  // extern "C"
