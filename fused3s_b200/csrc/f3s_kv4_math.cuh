// f3s_kv4_math.cuh -- pieces that the two 4-bit attention kernels share:
// requests' pages (f3s_kv4_attend.cu) and graph windows (f3s_kv4_forward.cu).
//
// With k_t = s_t (u_t - z_t) and v_t = r_t (w_t - y_t) (scales s, r, zeros z, y, codes u, w):
//   x_t = scale log2(e) s_t (q . u_t - z_t sum(q))                 the score, in powers of two
//   a_t = 2^(x_t + log2 r_t - R),  R >= x_t + log2 r_t - 15         the weight times V's scale
//   O   = (sum a_t w_t - sum a_t y_t) / sum a_t / r_t
// so the two matrix products read whole numbers 0 ... 15 and every scale is
// applied to a score, not to a value.  R is a running reference per query row:
// it moves (and the sums are rescaled) only when a weight would pass 2^15, which
// one vote per step decides, and then leaves the largest weight at 2^7: of the
// fp16 numbers that P is held in, those with full precision reach from 2^-14 to
// 2^16, and what a weight loses below that is 2^-25, 2^-32 of the largest.  (With
// the largest at 1 a thousand tokens that weigh 2^-20 each moved fp32 results by 3e-5.)
#pragma once
#include <cuda_bf16.h>
#include "f3s_internal.cuh"
#include "f3s_kv4.cuh"

namespace f3s {

constexpr uint64_t kAttendTimeoutNs = 5ull * 1000 * 1000 * 1000;
constexpr uint64_t kDrainNs = 100ull * 1000 * 1000;
constexpr float kNoReference = -3.0e38f;  // finite: a weight against it is 0, not NaN
// The tensor cores truncate when they add a product to an accumulator, and sums of codes
// never cancel: n pages in a row lose about n 2^-25 of V's span (twice that with a
// second product: 1.5e-2 for 250,000 pages).  After so many pages an accumulator is
// added to a sum in fp32, rounded to nearest, and begins anew.
constexpr int kRunPages = 256;
constexpr float kRescaleAt = 15.f;  // log2 of the largest weight that a reference is kept for, below fp16's end
constexpr float kTopWeight = 7.f;   // and of the largest weight when a reference is set

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float log2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Pairs of fp32 numbers in one 64-bit register: one instruction for two.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ float2 half2_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// Two 16-bit numbers of Q's type as fp32.
__device__ __forceinline__ float2 q_floats(uint32_t u, int bf16) {
    return bf16 ? make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)) : half2_floats(u);
}

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[N]) {
    static_assert(N == 2 || N == 4, "8 or 16 bytes");
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x;
        w[1] = v.y;
    }
}

// Waits for a phase of an mbarrier, by a whole warp; bounded.  False: give up, which
// `status` reports and `stop` tells the waits that come after (the launch's own word,
// or a plan's status: an error that an earlier launch left elsewhere stops nothing).
static __device__ __noinline__ bool phase_wait_slow(uint32_t bar, uint32_t parity, int* status, int* stop) {
    const uint64_t t0 = global_timer_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (load_volatile(stop) == F3S_ERR_TIMEOUT) return false;
        if (global_timer_ns() - t0 > kAttendTimeoutNs) {
            atomicExch(status, F3S_ERR_TIMEOUT);
            atomicExch(stop, F3S_ERR_TIMEOUT);
            return false;
        }
    }
}
__device__ __forceinline__ bool phase_wait(uint32_t bar, uint32_t parity, int* status, int* stop) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, phase_wait_slow(bar, parity, status, stop));
}

// Lets the copies of ring steps first ... end - 1 land (stages bars apart 8 bytes), for
// a limited time: shared memory is neither reused nor given up while they are in flight.
static __device__ __noinline__ void ring_drain(uint32_t bars, uint32_t stages, uint32_t first, uint32_t end) {
    for (uint32_t l = first; l < end; ++l)
        if (!mbar_try_wait(bars + 8 * (l % stages), l / stages & 1))
            mbar_drain(bars + 8 * (l % stages), l / stages & 1, kDrainNs);
}

// CH consecutive channels of a query row in O's type.
template <int CH>
__device__ __forceinline__ void store_channels(void* o, int64_t idx, const float (&v)[CH], int dtype) {
    if (dtype == F3S_OUT_F32) {
        float* dst = static_cast<float*>(o) + idx;
        if constexpr (CH == 2) {
            __stcs(reinterpret_cast<float2*>(dst), make_float2(v[0], v[1]));
        } else {
#pragma unroll
            for (int i = 0; i < CH / 4; ++i)
                __stcs(reinterpret_cast<float4*>(dst) + i, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
        }
        return;
    }
    uint32_t w[CH / 2];
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
        if (dtype == F3S_OUT_F16) {
            w[i] = pack_half2(v[2 * i], v[2 * i + 1]);
        } else {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
    }
    uint16_t* dst = static_cast<uint16_t*>(o) + idx;
    if constexpr (CH == 2) {
        __stcs(reinterpret_cast<unsigned int*>(dst), w[0]);
    } else if constexpr (CH == 4) {
        __stcs(reinterpret_cast<uint2*>(dst), make_uint2(w[0], w[1]));
    } else {
#pragma unroll
        for (int i = 0; i < CH / 8; ++i)
            __stcs(reinterpret_cast<uint4*>(dst) + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
    }
}

// Adds the pieces of split tiles (or windows): for `count` splits x `subs` heads x
// `tq` rows, the partial sums of the row's pieces in order, by one warp, or by a
// block's four warps (each every fourth piece, then the four in order) where there
// are too few rows (`live` of a tile, usually) to fill the blocks' warps.  Which
// of the two follows from counts, so the result repeats.  find(split, sub, row,
// &slot, &parts) gives the first slot, the pieces and the row of O, or -1 for none.
// A slot holds, per head, tq x D sums and then tq pairs (R, sum a / r).
template <int D, class Find>
__device__ __forceinline__ void merge_rows(int count, int subs, int tq, int live, const float* partials, void* o,
                                           int o_dtype, Find find) {
    constexpr int E = D / 32;  // channels per lane
    constexpr int AHEAD = 8;   // pieces read at a time
    __shared__ float s_o[4][D], s_l[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t units = (int64_t)count * subs * tq;
    const bool team = (int64_t)count * subs * live <= 4ll * gridDim.x;
    const int64_t stride = (int64_t)subs * tq * (D + 2);  // from piece to piece
    const int64_t first = team ? blockIdx.x : (int64_t)blockIdx.x * 4 + warp, step = (int64_t)gridDim.x * (team ? 1 : 4);
    for (int64_t u = first; u < units; u += step) {
        const int r = (int)(u % tq), sub = (int)(u / tq % subs), split = (int)(u / tq / subs);
        int slot, parts;
        const int64_t dst = find(split, sub, r, slot, parts);
        if (dst < 0) continue;  // for the whole team
        const float* part = partials + (int64_t)slot * stride + (int64_t)sub * tq * (D + 2);
        const float2* ml = reinterpret_cast<const float2*>(part + tq * D + 2 * r);
        const float* src = part + r * D + lane * E;
        float top = kNoReference;
        for (int k = lane; k < parts; k += 32) top = fmaxf(top, ml[k * (stride / 2)].x);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        float v[E], l = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = 0.f;
        const int k0 = team ? warp : 0, dk = team ? 4 : 1;
        for (int k = k0; k < parts; k += dk * AHEAD) {
            float2 m[AHEAD];
            float x[AHEAD][E];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (k + a * dk >= parts) break;
                const int64_t at = (int64_t)(k + a * dk) * stride;
                m[a] = ml[at / 2];
                if constexpr (E == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(src + at);
                    x[a][0] = y.x;
                    x[a][1] = y.y;
                    x[a][2] = y.z;
                    x[a][3] = y.w;
                } else {
                    const float2 y = *reinterpret_cast<const float2*>(src + at);
                    x[a][0] = y.x;
                    x[a][1] = y.y;
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (k + a * dk < parts) {
                    const float c = exp2_approx(m[a].x - top);
                    l = fmaf(c, m[a].y, l);
#pragma unroll
                    for (int i = 0; i < E; ++i) v[i] = fmaf(c, x[a][i], v[i]);
                }
            }
        }
        if (team) {
#pragma unroll
            for (int i = 0; i < E; ++i) s_o[warp][lane * E + i] = v[i];
            if (lane == 0) s_l[warp] = l;
            __syncthreads();
            if (warp == 0) {
                l = 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    l += s_l[w];
#pragma unroll
                    for (int i = 0; i < E; ++i) v[i] += s_o[w][lane * E + i];
                }
            }
            __syncthreads();
            if (warp != 0) continue;
        }
        const float inv = l != 0.f ? __frcp_rn(l) : 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] *= inv;
        store_channels<E>(o, dst * D + lane * E, v, o_dtype);
    }
}

// Whether the weights are multiplied in full (fp16 and what its rounding drops) or
// rounded to fp16.  Rounded weights go into all three sums: then a result is the
// average that these weights make, and a rounding moves it by at most 2^-11 of the
// values' distance from it.  (With unrounded weights in the sums of zeros and of
// weights, a rounding would act on codes, 0 ... 15, whose sums are far larger than
// their difference, the result: 3e-4 of V's size for 3,000 tokens of +1 and -1 that
// weigh alike, where the result is 2e-2.)  Rounded, a result's error doubles
// where it is written in fp16 (4.0e-4 against 2.1e-4 of the result, 131,057 nodes).
inline bool weights_in_full(int o_dtype) { return o_dtype != F3S_OUT_BF16; }

// Arguments that the attentions share.
inline int check_attend_args(const void* Q, int q_dtype, int64_t qt, int64_t qh, const void* pages, int num_pages, int heads,
                        int kv_heads, int head_dim, const void* O, int o_dtype) {
    auto bad = [](const void* x) { return !x || (reinterpret_cast<uintptr_t>(x) & 15) != 0; };
    if (q_dtype != F3S_OUT_F16 && q_dtype != F3S_OUT_BF16) return F3S_ERR_INVALID_VALUE;
    if (o_dtype != F3S_OUT_F32 && o_dtype != F3S_OUT_F16 && o_dtype != F3S_OUT_BF16) return F3S_ERR_INVALID_VALUE;
    if (head_dim != 64 && head_dim != 128) return F3S_ERR_UNSUPPORTED;
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || num_pages < 0) return F3S_ERR_INVALID_VALUE;
    if (bad(Q) || bad(O) || ((qt | qh) & 7)) return F3S_ERR_INVALID_VALUE;
    if (num_pages == 0 || bad(pages)) return F3S_ERR_INVALID_VALUE;
    return F3S_SUCCESS;
}

}  // namespace f3s
