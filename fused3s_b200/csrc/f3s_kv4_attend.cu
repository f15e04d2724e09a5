// f3s_kv4_attend.cu -- softmax(scale Q K^T) V over K and V held in 4 bits: over
// the pages of a request (block tables; causal; grouped heads) and over the
// active blocks of a row window (the block-sparse format; columns >= N masked).
//
// With k_t = s_t (u_t - z_t) and v_t = r_t (w_t - y_t) (scales s, r, zeros z, y, codes u, w):
//   x_t = scale log2(e) s_t (q . u_t - z_t sum(q))                 the score, in powers of two
//   a_t = 2^(x_t + log2 r_t - R),  R >= x_t + log2 r_t - 8          the weight times V's scale
//   O   = (sum a_t w_t - sum a_t y_t) / sum a_t / r_t
// so the two matrix products read whole numbers 0 ... 15 and every scale is
// applied to a score, not to a value.  R is a running reference per query row:
// it moves (and the sums are rescaled) only when a weight would pass 2^8, which
// one vote per page decides.
//
// Per warp: pages stream through a ring of shared-memory stages, one bulk copy
// of 16 D + 128 bytes per page, issued by one lane as soon as the stage has been
// read.  S^T = K Q^T and O^T = V^T P^T run on mma.m16n8k16 with the cache as
// the 16-row operand (unpacked in registers, one AND per two values; see
// f3s_kv4.cuh) and 8 NT query rows as columns; P goes from accumulator to
// operand layout through movmatrix.  tcgen05's M = 64 / 128 rows would stand
// mostly empty here: 8 to 32 query rows share a page.
//
// Bound: HBM where few query rows read a page (decoding: D + 8 bytes per token
// and K/V head); the mma.sync rate and the unpacking where many do.
#include <algorithm>
#include <cuda_bf16.h>
#include "f3s_internal.cuh"
#include "f3s_kv4.cuh"
#include "f3s_kv4_plan.cuh"

namespace f3s {

constexpr int kAttendWarps = 4;
constexpr uint64_t kAttendTimeoutNs = 5ull * 1000 * 1000 * 1000;
constexpr float kNoReference = -3.0e38f;  // finite: a weight against it is 0, not NaN
constexpr float kRescaleAt = 8.f;

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
    // paged
    const Kv4PlanHeader* plan;
    const int* tables;
    int64_t table_stride;
    // windows
    const int* offsets;
    const int* cols;
    const int* order;
    int num_items;
    int num_nodes, windows, q_window_base, q_rows;
    int warps_per_unit;  // 4, or 1: one warp per window and head
};

template <int D, int NT>
struct AttendCfg {
    static constexpr int RB = kv4_record_bytes(D);
    static constexpr int STAGES = D == 64 ? 8 : 4;
    static constexpr int RING = kAttendWarps * STAGES * RB;
    static constexpr bool Q_SMEM = NT == 4;  // four warps per unit only: they share it
    static constexpr int Q_BYTES = Q_SMEM ? 8 * NT * D * 2 : 0;
    static constexpr int OPITCH = D + 4;
    static constexpr int MERGE = kAttendWarps * 8 * NT * (OPITCH + 2) * 4;
    static constexpr int DATA = RING + Q_BYTES > MERGE ? RING + Q_BYTES : (MERGE + 127) / 128 * 128;
    static constexpr int BARS = DATA;
    static constexpr int SINK = BARS + kAttendWarps * STAGES * 8;  // one word per warp, written, never read
    static constexpr int SMEM = SINK + kAttendWarps * 4;
    static constexpr int MIN_CTAS = NT == 4 ? 2 : NT == 2 && D == 128 ? 3 : 4;
};

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

// Waits for a stage of this warp's own ring; bounded.  False: give up.
static __device__ __noinline__ bool stage_wait_slow(uint32_t bar, uint32_t parity, int* status) {
    const uint64_t t0 = global_timer_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (load_volatile(status) == F3S_ERR_TIMEOUT) return false;
        if (global_timer_ns() - t0 > kAttendTimeoutNs) {
            atomicExch(status, F3S_ERR_TIMEOUT);
            return false;
        }
    }
}

// 8 NT values of one query row in O's type: CH consecutive channels.
template <int CH>
__device__ __forceinline__ void store_channels(void* o, int64_t idx, const float (&v)[CH], int dtype) {
    if (dtype == F3S_OUT_F32) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(o) + idx);
#pragma unroll
        for (int i = 0; i < CH / 4; ++i) __stcs(dst + i, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
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
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(o) + idx);
#pragma unroll
    for (int i = 0; i < CH / 8; ++i) __stcs(dst + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
}

// PAGED: a unit is (work item of the plan, K/V head) and the CTA's four warps
// take its pages in turn.  Otherwise a unit is (window, head): four warps in
// turn, or one warp.  PRECISE adds the part of P that rounding to fp16 drops
// with a second product, which makes the result as exact as fp32 arithmetic.
template <int D, int NT, bool PAGED, bool PRECISE>
__global__ void __launch_bounds__(kAttendWarps * 32, AttendCfg<D, NT>::MIN_CTAS) k_attend4(const AttendParams p) {
    using C = AttendCfg<D, NT>;
    constexpr int RB = C::RB, STAGES = C::STAGES;
    constexpr int W = D / 32;    // words of a token's K (and of a token pair's V) per lane
    constexpr int CH = D / 8;    // output channels per lane
    constexpr int TQ = 8 * NT;   // query rows of a tile
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wpu = PAGED ? kAttendWarps : p.warps_per_unit;
    const int wq = wpu == 1 ? 0 : warp;
    uint8_t* ring = smem + warp * STAGES * RB;
    const uint32_t ring_a = smem_addr(ring);
    const uint32_t bars = smem_addr(smem + C::BARS) + warp * STAGES * 8;
    const uint32_t sink = smem_addr(smem + C::SINK) + warp * 4;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) mbar_init(bars + 8 * i, 1);
        fence_mbar_init();
    }
    __syncwarp();
    bool dead = false;  // a wait ran out: no more pages for this warp
    uint32_t used = 0;  // pages this warp has streamed: stage and parity of the next

    const int per_cta = kAttendWarps / wpu;
    const int kv_units = PAGED ? p.kv_heads : p.heads;
    const int64_t units = (int64_t)(PAGED ? p.plan->num_items : p.num_items) * kv_units;
    const int64_t page_bytes = (int64_t)p.kv_heads * RB;

    for (int64_t base = (int64_t)blockIdx.x * per_cta; base < units; base += (int64_t)gridDim.x * per_cta) {
        const int64_t unit = base + (wpu == 1 ? warp : 0);
        if (unit >= units) break;  // one warp per unit: nothing is shared
        const int item = (int)(unit / kv_units), sub = (int)(unit - (int64_t)item * kv_units);
        const int hk = PAGED ? sub : sub / p.group;
        Kv4Item it{};
        const int* list;
        int first, count;  // blocks of the unit
        int window = 0;
        if constexpr (PAGED) {
            const int4* src = reinterpret_cast<const int4*>(reinterpret_cast<const Kv4Item*>(p.plan + 1) + item);
            const int4 a = __ldg(src), b = __ldg(src + 1);
            it.request = a.x;
            it.q_token = a.y;
            it.row0 = a.z;
            it.rows = a.w;
            it.context = b.x;
            it.page0 = b.y;
            it.page1 = b.z;
            it.slot = b.w;
            list = p.tables + (int64_t)it.request * p.table_stride;
            first = it.page0;
            count = max(it.page1 - it.page0, 0);
        } else {
            window = p.order[item];
            const bool ok = window >= p.q_window_base && window < p.windows &&
                            (int64_t)(window - p.q_window_base) * 16 < p.q_rows;
            if (!ok) {
                if (lane == 0) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
                continue;  // the whole unit: every warp of it sees the same window
            }
            list = p.cols;
            first = p.offsets[window];
            count = max(p.offsets[window + 1] - first, 0);
        }
        const int own = !dead && count > wq ? (count - wq + wpu - 1) / wpu : 0;
        const int limit_id = PAGED ? p.num_pages : p.windows;

        // ---- page ids, 32 at a time (one per lane), the next 32 ahead
        auto load_ids = [&](int batch) {
            const int i = batch * 32 + lane;
            int id = 0;
            if (i < own) {
                id = __ldg(list + first + wq + (int64_t)i * wpu);
                if (id < 0 || id >= limit_id) {
                    if (!(PAGED && id == -1)) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
                    id = -1;
                }
            }
            return id;
        };
        int ids = load_ids(0), ids_next = 0;
        uint32_t skip = 0, tail = 0;  // of the pages in flight, bit (page index % 32)
        auto issue = [&](int i) {
            if ((i & 31) == 0) {
                if (i > 0) ids = ids_next;
                if (i + 32 < own) ids_next = load_ids(i / 32 + 1);
            }
            const int id = __shfl_sync(0xffffffffu, ids, i & 31);
            const uint32_t bit = 1u << (i & 31);
            skip = id < 0 ? skip | bit : skip & ~bit;
            if constexpr (!PAGED) tail = id == p.windows - 1 ? tail | bit : tail & ~bit;
            const uint32_t n = used + i, st = n % STAGES;
            if (lane == 0) {
                mbar_arrive_expect_tx(bars + 8 * st, RB);
                bulk_load(ring_a + st * RB, p.pages + (int64_t)max(id, 0) * page_bytes + (int64_t)hk * RB, RB,
                          bars + 8 * st);
            }
        };
        for (int i = 0; i < min(own, STAGES); ++i) issue(i);

        // ---- Q: rows g of each n-tile, channels t * D / 4 ..., as fp16 times a
        // power of two that brings the tile's largest to [2^9, 2^10); channels
        // whose codes come in units of 2^-24 another 2^4
        uint32_t qf[C::Q_SMEM ? 1 : NT][C::Q_SMEM ? 1 : W][4];
        float qs[NT][2];  // sum of q (in the scores' unit) of rows 2t, 2t + 1
        float unit_scale;
        uint4* qsm = reinterpret_cast<uint4*>(smem + C::RING);
        {
            float amax = 0.f;
            uint4 raw[NT][W];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int r = nt * 8 + g;
                int64_t off = -1;
                if constexpr (PAGED) {
                    const int row = it.row0 + r;
                    if (row < it.rows) {
                        const int tok = row / p.group;
                        off = (int64_t)(it.q_token + tok) * p.q_token +
                              (int64_t)(hk * p.group + row - tok * p.group) * p.q_head;
                    }
                } else {
                    const int64_t row = (int64_t)(window - p.q_window_base) * 16 + r;
                    if (row < p.q_rows) off = row * p.q_token + (int64_t)sub * p.q_head;
                }
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + off + t * (D / 4));
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    raw[nt][w] = off >= 0 ? __ldg(src + w) : make_uint4(0, 0, 0, 0);
                    const uint32_t u[4] = {raw[nt][w].x, raw[nt][w].y, raw[nt][w].z, raw[nt][w].w};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        float a, b;
                        if (p.q_bf16) {
                            a = __uint_as_float(u[n] << 16);
                            b = __uint_as_float(u[n] & 0xffff0000u);
                        } else {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[n]));
                            a = f.x;
                            b = f.y;
                        }
                        a = fabsf(a);
                        b = fabsf(b);
                        if (a < INFINITY) amax = fmaxf(amax, a);  // NaN and infinities stay what they are
                        if (b < INFINITY) amax = fmaxf(amax, b);
                    }
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            // 2^(9 - floor(log2 amax)), kept within fp32's normal range
            const int e = amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 : 9;
            const int up = min(max(9 - e, -120), 120);
            const float f = __uint_as_float((uint32_t)(up + 127) << 23);
            unit_scale = p.scale * __uint_as_float((uint32_t)(127 - up) << 23);
            float sums[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t u[4] = {raw[nt][w].x, raw[nt][w].y, raw[nt][w].z, raw[nt][w].w};
                    uint32_t h[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        float a, b;
                        if (p.q_bf16) {
                            a = __uint_as_float(u[n] << 16);
                            b = __uint_as_float(u[n] & 0xffff0000u);
                        } else {
                            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u[n]));
                            a = x.x;
                            b = x.y;
                        }
                        const float m = n & 1 ? f : f * 16.f;
                        h[n] = pack_half2(a * m, b * m);
                        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[n]));
                        sum += (x.x + x.y) * (n & 1 ? 1.f : 0.0625f);
                    }
                    if constexpr (C::Q_SMEM) {
                        if (warp == nt) qsm[(nt * W + w) * 32 + lane] = make_uint4(h[0], h[1], h[2], h[3]);
                    } else {
#pragma unroll
                        for (int n = 0; n < 4; ++n) qf[nt][w][n] = h[n];
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sums[nt] = sum * 9.5367431640625e-7f;  // 2^-20
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                qs[nt][0] = __shfl_sync(0xffffffffu, sums[nt], 8 * t);      // row 2t is summed in lanes 4 * 2t ...
                qs[nt][1] = __shfl_sync(0xffffffffu, sums[nt], 8 * t + 4);  // row 2t + 1
            }
            if constexpr (C::Q_SMEM) __syncthreads();
        }

        float acc[NT][D / 16][4];
        float ref[NT][2], den[NT][2], off[NT][2];  // R, sum a / r, sum a y (this lane's tokens)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[nt][m][i] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ref[nt][i] = kNoReference;
                den[nt][i] = off[nt][i] = 0.f;
            }
        }
        // first token that some row of the tile must not see
        const int open = PAGED ? it.context + it.row0 / p.group + 1 : 0;

        for (int i = 0; i < own; ++i) {
            const uint32_t n = used + i, st = n % STAGES, parity = (n / STAGES) & 1;
            bool ready = mbar_try_wait(bars + 8 * st, parity);
            if (!__all_sync(0xffffffffu, ready)) {
                ready = stage_wait_slow(bars + 8 * st, parity, p.status);
                if (!__all_sync(0xffffffffu, ready)) {
                    dead = true;
                    break;
                }
            }
            const uint8_t* rec = ring + st * RB;
            // ---- S^T = K Q^T
            uint32_t kg[W], kh[W], v0[W], v1[W];
            lds_words<W>(rec + g * (D / 2) + t * (D / 8), kg);
            lds_words<W>(rec + (g + 8) * (D / 2) + t * (D / 8), kh);
            const uint4 sc = *reinterpret_cast<const uint4*>(rec + 16 * D + g * 16);
            lds_words<W>(rec + 8 * D + lane * (D / 8), v0);
            lds_words<W>(rec + 12 * D + lane * (D / 8), v1);
            float s[NT][2][4];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const uint32_t a8 = kg[w] >> 8, b8 = kh[w] >> 8;
                const uint32_t a0[4] = {kg[w] & kNib0, kh[w] & kNib0, kg[w] & kNib1, kh[w] & kNib1};
                const uint32_t a1[4] = {a8 & kNib0, b8 & kNib0, a8 & kNib1, b8 & kNib1};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t b[4];
                    if constexpr (C::Q_SMEM) {
                        const uint4 x = qsm[(nt * W + w) * 32 + lane];
                        b[0] = x.x;
                        b[1] = x.y;
                        b[2] = x.z;
                        b[3] = x.w;
                    } else {
#pragma unroll
                        for (int n = 0; n < 4; ++n) b[n] = qf[nt][w][n];
                    }
                    constexpr int odd = NT == 1 ? 1 : 0;  // one n-tile: two chains
                    if (w == 0) {
                        mma_16816_zero(s[nt][0], a0, b[0], b[1]);
                        if (odd) mma_16816_zero(s[nt][1], a1, b[2], b[3]);
                        else mma_16816(s[nt][0], a1, b[2], b[3]);
                    } else {
                        mma_16816(s[nt][0], a0, b[0], b[1]);
                        mma_16816(s[nt][odd], a1, b[2], b[3]);
                    }
                }
            }
            // ---- scores to weights
            const float2 ka = __half22float2(*reinterpret_cast<const __half2*>(&sc.x));
            const float2 va = __half22float2(*reinterpret_cast<const __half2*>(&sc.y));
            const float2 kb = __half22float2(*reinterpret_cast<const __half2*>(&sc.z));
            const float2 vb = __half22float2(*reinterpret_cast<const __half2*>(&sc.w));
            const float fa = ka.x * 1048576.f * unit_scale, fb = kb.x * 1048576.f * unit_scale;  // 2^20: the codes' unit
            const float ra = va.x < kKv4MinScale ? kKv4MinScale : va.x;  // keeps a NaN
            const float rb = vb.x < kKv4MinScale ? kKv4MinScale : vb.x;
            const float la = log2_approx(ra), lb = log2_approx(rb);
            const float ia = __frcp_rn(ra), ib = __frcp_rn(rb);
            const int tok0 = PAGED ? (it.page0 + wq + i * wpu) * 16 : 0;
            const bool skipped = (skip >> (i & 31)) & 1;
            bool masked;
            if constexpr (PAGED) masked = skipped || tok0 + 16 > open;
            else masked = skipped || ((tail >> (i & 31)) & 1);
            float x[NT][4];
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float d = s[nt][0][c];
                    if (NT == 1) d += s[nt][1][c];
                    const float z = c < 2 ? ka.y : kb.y;
                    x[nt][c] = fmaf(fmaf(-z, qs[nt][c & 1], d), c < 2 ? fa : fb, c < 2 ? la : lb);
                }
            if (masked) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int tk = g + (c < 2 ? 0 : 8);
                        bool hide;
                        if constexpr (PAGED) {
                            // a tile's rows past its last see what the last sees
                            const int row = min(it.row0 + nt * 8 + 2 * t + (c & 1), it.rows - 1);
                            hide = tok0 + tk > it.context + row / p.group;
                        } else {
                            hide = (p.windows - 1) * 16 + tk >= p.num_nodes;
                        }
                        if (hide || skipped) x[nt][c] = -INFINITY;
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) over |= x[nt][c] > ref[nt][c & 1] + kRescaleAt;
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float m = fmaxf(x[nt][j], x[nt][j + 2]);
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                        m = fmaxf(m, ref[nt][j]);
                        const float c = exp2_approx(ref[nt][j] - m);
                        ref[nt][j] = m;
                        den[nt][j] *= c;
                        off[nt][j] *= c;
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            acc[nt][k][j] *= c;
                            acc[nt][k][j + 2] *= c;
                        }
                    }
            }
            uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float a[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) a[c] = exp2_approx(x[nt][c] - ref[nt][c & 1]);
                const uint32_t h0 = pack_half2(a[0], a[1]), h1 = pack_half2(a[2], a[3]);
                const float2 r0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                const float2 r1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                pb[nt][0] = movmatrix_t(h0);
                pb[nt][1] = movmatrix_t(h1);
                if constexpr (PRECISE) {
                    pl[nt][0] = movmatrix_t(pack_half2(a[0] - r0.x, a[1] - r0.y));
                    pl[nt][1] = movmatrix_t(pack_half2(a[2] - r1.x, a[3] - r1.y));
                } else {
                    // the sums take the weights that the product takes
                    a[0] = r0.x;
                    a[1] = r0.y;
                    a[2] = r1.x;
                    a[3] = r1.y;
                }
                if (masked) {
                    // a masked token's scale and zero may be anything, NaN too
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const bool on = x[nt][c] != -INFINITY;
                        den[nt][c & 1] += on ? a[c] * (c < 2 ? ia : ib) : 0.f;
                        off[nt][c & 1] += on ? a[c] * (c < 2 ? va.y : vb.y) : 0.f;
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        den[nt][c & 1] = fmaf(a[c], c < 2 ? ia : ib, den[nt][c & 1]);
                        off[nt][c & 1] = fmaf(a[c], c < 2 ? va.y : vb.y, off[nt][c & 1]);
                    }
                }
            }
            // ---- O^T += V^T P^T
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const uint32_t a8 = v0[w] >> 8, b8 = v1[w] >> 8;
                const uint32_t a0[4] = {v0[w] & kNib0, v0[w] & kNib1, v1[w] & kNib0, v1[w] & kNib1};
                const uint32_t a1[4] = {a8 & kNib0, a8 & kNib1, b8 & kNib0, b8 & kNib1};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_16816(acc[nt][2 * w], a0, pb[nt][0], pb[nt][1]);
                    mma_16816(acc[nt][2 * w + 1], a1, pb[nt][0], pb[nt][1]);
                    if constexpr (PRECISE) {
                        mma_16816(acc[nt][2 * w], a0, pl[nt][0], pl[nt][1]);
                        mma_16816(acc[nt][2 * w + 1], a1, pl[nt][0], pl[nt][1]);
                    }
                }
            }
            // refill the stage once the loads from it have landed in every lane:
            // the store needs a word of each load, and comes before the copy
            if (i + STAGES < own) {
                const uint32_t dep = kg[0] ^ kh[0] ^ v0[0] ^ v1[0] ^ sc.x;
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(sink), "r"(dep) : "memory");
                __syncwarp();
                issue(i + STAGES);
            }
        }
        used += own;

        // ---- sums over the tokens of the other lanes; units of the accumulators
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    den[nt][j] += __shfl_xor_sync(0xffffffffu, den[nt][j], o);
                    off[nt][j] += __shfl_xor_sync(0xffffffffu, off[nt][j], o);
                }
        // channel g * CH + 4 w + n of row 2t + j:  acc[2 w + n / 2][2 (n % 2) + j]
        auto channel = [&](int nt, int j, int c) {
            const int w = c / 4, n = c % 4;
            return fmaf(acc[nt][2 * w + n / 2][2 * (n & 1) + j], n & 1 ? 1048576.f : 16777216.f, -off[nt][j]);
        };

        if (wpu == 1) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int64_t row = (int64_t)(window - p.q_window_base) * 16 + nt * 8 + 2 * t + j;
                    const int64_t node = (int64_t)window * 16 + nt * 8 + 2 * t + j;
                    if (row >= p.q_rows || node >= p.num_nodes) continue;
                    const float inv = den[nt][j] != 0.f ? __frcp_rn(den[nt][j]) : 0.f;
                    float v[CH];
#pragma unroll
                    for (int c = 0; c < CH; ++c) v[c] = channel(nt, j, c) * inv;
                    store_channels<CH>(p.o, (row * p.heads + sub) * D + g * CH, v, p.o_dtype);
                }
            continue;
        }

        // ---- the four warps' sums, through shared memory
        __syncthreads();  // every warp's stages have been read
        float* mo = reinterpret_cast<float*>(smem);
        float* ml = mo + kAttendWarps * TQ * C::OPITCH;  // (R, den) per warp and row
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = nt * 8 + 2 * t + j;
                float4* dst = reinterpret_cast<float4*>(mo + (warp * TQ + r) * C::OPITCH + g * CH);
#pragma unroll
                for (int c = 0; c < CH; c += 4)
                    dst[c / 4] = make_float4(channel(nt, j, c), channel(nt, j, c + 1), channel(nt, j, c + 2),
                                             channel(nt, j, c + 3));
                if (g == 0) {
                    ml[2 * (warp * TQ + r)] = ref[nt][j];
                    ml[2 * (warp * TQ + r) + 1] = den[nt][j];
                }
            }
        __syncthreads();
        for (int e = threadIdx.x; e < TQ * (D / 8); e += kAttendWarps * 32) {
            const int r = e / (D / 8), c0 = (e % (D / 8)) * 8;
            int64_t dst = -1;
            bool valid;
            if constexpr (PAGED) {
                const int row = it.row0 + r;
                valid = row < it.rows;
                const int tok = row / p.group;
                dst = ((int64_t)(it.q_token + tok) * p.heads + hk * p.group + row - tok * p.group) * D + c0;
            } else {
                const int64_t row = (int64_t)(window - p.q_window_base) * 16 + r;
                valid = row < p.q_rows && (int64_t)window * 16 + r < p.num_nodes;
                dst = (row * p.heads + sub) * D + c0;
            }
            if (!valid) continue;
            float top = kNoReference;
#pragma unroll
            for (int w = 0; w < kAttendWarps; ++w) top = fmaxf(top, ml[2 * (w * TQ + r)]);
            float den_all = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kAttendWarps; ++w) {
                const float c = exp2_approx(ml[2 * (w * TQ + r)] - top);
                den_all = fmaf(c, ml[2 * (w * TQ + r) + 1], den_all);
                const float* src = mo + (w * TQ + r) * C::OPITCH + c0;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = fmaf(c, src[k], v[k]);
            }
            if (PAGED && it.slot >= 0) {
                float* part = p.partials + ((int64_t)it.slot * p.kv_heads + hk) * TQ * (D + 2);
                float4* po = reinterpret_cast<float4*>(part + r * D + c0);
                po[0] = make_float4(v[0], v[1], v[2], v[3]);
                po[1] = make_float4(v[4], v[5], v[6], v[7]);
                if (c0 == 0) *reinterpret_cast<float2*>(part + TQ * D + 2 * r) = make_float2(top, den_all);
            } else {
                const float inv = den_all != 0.f ? __frcp_rn(den_all) : 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] *= inv;
                store_channels<8>(p.o, dst, v, p.o_dtype);
            }
        }
        // the ring is written by the copies of the next unit
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
}

// One block per (split tile, K/V head, query row): the pieces' sums, in piece
// order within each warp and the four warps in order (the result repeats).
template <int D>
__global__ void __launch_bounds__(128) k_attend4_merge(const AttendParams p) {
    constexpr int E = D / 32;  // channels per lane
    __shared__ float s_o[4][D], s_l[4];
    const Kv4PlanHeader* plan = p.plan;
    const int tq = plan->tile_rows, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Kv4Split* splits =
        reinterpret_cast<const Kv4Split*>(reinterpret_cast<const char*>(plan + 1) + (int64_t)plan->items_cap * sizeof(Kv4Item));
    const int64_t units = (int64_t)plan->num_splits * p.kv_heads * tq;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int r = (int)(u % tq);
        const int64_t rest = u / tq;
        const int hk = (int)(rest % p.kv_heads);
        const Kv4Split s = splits[rest / p.kv_heads];
        const int row = s.row0 + r;
        if (row >= s.rows) continue;
        const int64_t stride = (int64_t)p.kv_heads * tq * (D + 2);
        const float* part = p.partials + ((int64_t)s.slot * p.kv_heads + hk) * tq * (D + 2);
        const float2* ml = reinterpret_cast<const float2*>(part + tq * D + 2 * r);
        float top = kNoReference;
        for (int k = lane; k < s.parts; k += 32) top = fmaxf(top, ml[k * (stride / 2)].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float v[E], l = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = 0.f;
        const float* src = part + r * D + lane * E;
#pragma unroll 8
        for (int k = warp; k < s.parts; k += 4) {
            const float2 m = ml[k * (stride / 2)];
            const float c = exp2_approx(m.x - top);
            l = fmaf(c, m.y, l);
            if constexpr (E == 4) {
                const float4 x = *reinterpret_cast<const float4*>(src + k * stride);
                v[0] = fmaf(c, x.x, v[0]);
                v[1] = fmaf(c, x.y, v[1]);
                v[2] = fmaf(c, x.z, v[2]);
                v[3] = fmaf(c, x.w, v[3]);
            } else {
                const float2 x = *reinterpret_cast<const float2*>(src + k * stride);
                v[0] = fmaf(c, x.x, v[0]);
                v[1] = fmaf(c, x.y, v[1]);
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) s_o[warp][lane * E + i] = v[i];
        if (lane == 0) s_l[warp] = l;
        __syncthreads();
        if (threadIdx.x < D / 8) {
            float den = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                den += s_l[w];
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] += s_o[w][threadIdx.x * 8 + k];
            }
            const float inv = den != 0.f ? __frcp_rn(den) : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] *= inv;
            const int tok = row / p.group;
            store_channels<8>(p.o, ((int64_t)(s.q_token + tok) * p.heads + hk * p.group + row - tok * p.group) * D + threadIdx.x * 8,
                              o, p.o_dtype);
        }
        __syncthreads();
    }
}

template <int D, int NT, bool PAGED, bool PRECISE>
static int attend_variant(const AttendParams& p, int64_t units, cudaStream_t stream) {
    using C = AttendCfg<D, NT>;
    static PerContext<int> attr;
    const int rc = attr.get(nullptr, [](int* v) -> int {
        *v = 1;
        F3S_CUDA_TRY(cudaFuncSetAttribute(k_attend4<D, NT, PAGED, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::SMEM));
        return F3S_SUCCESS;
    });
    if (rc != F3S_SUCCESS) return rc;
    const int per_cta = PAGED ? 1 : kAttendWarps / p.warps_per_unit;
    const int64_t grid = std::min<int64_t>((units + per_cta - 1) / per_cta, INT32_MAX);
    if (grid == 0) return F3S_SUCCESS;
    k_attend4<D, NT, PAGED, PRECISE><<<(unsigned)grid, kAttendWarps * 32, C::SMEM, stream>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

template <int NT, bool PAGED>
static int attend_launch(const AttendParams& p, int head_dim, int64_t units, cudaStream_t stream) {
    // fp16 and fp32 results take the exact form of P: fp16's rounding of P
    // would be as large as that of an fp16 result
    const bool precise = p.o_dtype != F3S_OUT_BF16;
    if (head_dim == 64)
        return precise ? attend_variant<64, NT, PAGED, true>(p, units, stream)
                       : attend_variant<64, NT, PAGED, false>(p, units, stream);
    return precise ? attend_variant<128, NT, PAGED, true>(p, units, stream)
                   : attend_variant<128, NT, PAGED, false>(p, units, stream);
}

static int check_attend(const void* Q, int q_dtype, int64_t qt, int64_t qh, const void* pages, int num_pages, int heads,
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

extern "C" {

size_t f3s_kv4_attention_workspace_size(int32_t num_requests, int64_t num_tokens, int32_t heads, int32_t kv_heads,
                                        int32_t head_dim) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || num_requests < 0 || num_tokens < 0) return 0;
    if (head_dim != 64 && head_dim != 128) return 0;
    const f3s::Kv4PlanLayout L = f3s::kv4_plan_layout(num_requests, num_tokens, heads, kv_heads,
                                                      f3s::num_sms_of_current_device());
    return (size_t)L.slots_cap * kv_heads * L.tile_rows * (head_dim + 2) * 4;
}

int f3s_kv4_attention(const void* d_Q, int32_t q_dtype, int64_t q_token_stride, int64_t q_head_stride,
                      const void* d_pages, int32_t num_pages, const int32_t* d_tables, int64_t table_stride,
                      void* d_plan, int32_t num_requests, int64_t num_tokens, int32_t heads,
                      int32_t kv_heads, int32_t head_dim, float scale, void* d_O, int32_t o_dtype, void* d_workspace,
                      size_t workspace_bytes, f3s_stream_t stream) {
    f3s::NvtxRange nvtx_("f3s_kv4_attention");
    if (num_requests < 0 || num_tokens < 0) return F3S_ERR_INVALID_VALUE;
    if (head_dim != 64 && head_dim != 128) return F3S_ERR_UNSUPPORTED;
    if (num_requests == 0 || num_tokens == 0) return F3S_SUCCESS;
    const int rc = f3s::check_attend(d_Q, q_dtype, q_token_stride, q_head_stride, d_pages, num_pages, heads, kv_heads,
                                     head_dim, d_O, o_dtype);
    if (rc != F3S_SUCCESS) return rc;
    if (num_tokens * (heads / kv_heads) > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
    if (!d_tables || !d_plan || (reinterpret_cast<uintptr_t>(d_plan) & 15)) return F3S_ERR_INVALID_VALUE;
    if (!d_workspace || (reinterpret_cast<uintptr_t>(d_workspace) & 15)) return F3S_ERR_INVALID_VALUE;
    const f3s::Kv4PlanLayout L = f3s::kv4_plan_layout(num_requests, num_tokens, heads, kv_heads,
                                                      f3s::num_sms_of_current_device());
    if (L.items_cap > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
    if (workspace_bytes < (size_t)L.slots_cap * kv_heads * L.tile_rows * (head_dim + 2) * 4) return F3S_ERR_WORKSPACE;
    f3s::AttendParams p{};
    p.q = d_Q;
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.q_bf16 = q_dtype == F3S_OUT_BF16;
    p.pages = static_cast<const uint8_t*>(d_pages);
    p.num_pages = num_pages;
    p.kv_heads = kv_heads;
    p.heads = heads;
    p.group = heads / kv_heads;
    p.scale = scale * 1.4426950408889634f;
    p.o = d_O;
    p.o_dtype = o_dtype;
    p.plan = static_cast<const f3s::Kv4PlanHeader*>(d_plan);
    p.status = &static_cast<f3s::WsHeader*>(d_plan)->status;
    p.partials = static_cast<float*>(d_workspace);
    p.tables = d_tables;
    p.table_stride = table_stride;
    p.warps_per_unit = f3s::kAttendWarps;
    cudaStream_t s = (cudaStream_t)stream;
    const int64_t units = L.items_cap * kv_heads;
    int st;
    if (L.tile_rows == 8) st = f3s::attend_launch<1, true>(p, head_dim, units, s);
    else if (L.tile_rows == 16) st = f3s::attend_launch<2, true>(p, head_dim, units, s);
    else st = f3s::attend_launch<4, true>(p, head_dim, units, s);
    if (st != F3S_SUCCESS) return st;
    const int64_t blocks = std::min<int64_t>((int64_t)L.splits_cap * kv_heads * L.tile_rows,
                                             8ll * f3s::num_sms_of_current_device());
    if (head_dim == 64) f3s::k_attend4_merge<64><<<(unsigned)blocks, 128, 0, s>>>(p);
    else f3s::k_attend4_merge<128><<<(unsigned)blocks, 128, 0, s>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

int f3s_kv4_forward(const void* d_Q, int32_t q_dtype, const void* d_pages, int32_t num_pages, void* d_O,
                    int32_t o_dtype, const int32_t* d_window_offsets, const int32_t* d_block_cols,
                    const int32_t* d_order, int32_t num_items, int32_t num_nodes, int32_t heads, int32_t kv_heads,
                    int32_t head_dim, float scale, int32_t q_window_base, int32_t q_rows, void* d_workspace,
                    size_t workspace_bytes, f3s_stream_t stream) {
    f3s::NvtxRange nvtx_("f3s_kv4_forward");
    if (num_items < 0 || num_nodes < 0 || q_window_base < 0 || q_rows < 0) return F3S_ERR_INVALID_VALUE;
    if (head_dim != 64 && head_dim != 128) return F3S_ERR_UNSUPPORTED;
    if (!d_workspace) return F3S_ERR_INVALID_VALUE;
    if (workspace_bytes < f3s::kWsHeaderBytes) return F3S_ERR_WORKSPACE;
    if (num_items == 0 || num_nodes == 0 || q_rows == 0) return F3S_SUCCESS;
    const int rc = f3s::check_attend(d_Q, q_dtype, (int64_t)heads * head_dim, head_dim, d_pages, num_pages, heads,
                                     kv_heads, head_dim, d_O, o_dtype);
    if (rc != F3S_SUCCESS) return rc;
    if (!d_window_offsets || !d_block_cols || !d_order) return F3S_ERR_INVALID_VALUE;
    const int windows = (int)(((int64_t)num_nodes + 15) / 16);
    if (num_pages < windows) return F3S_ERR_INVALID_VALUE;
    f3s::AttendParams p{};
    p.q = d_Q;
    p.q_token = (int64_t)heads * head_dim;
    p.q_head = head_dim;
    p.q_bf16 = q_dtype == F3S_OUT_BF16;
    p.pages = static_cast<const uint8_t*>(d_pages);
    p.num_pages = num_pages;
    p.kv_heads = kv_heads;
    p.heads = heads;
    p.group = heads / kv_heads;
    p.scale = scale * 1.4426950408889634f;
    p.o = d_O;
    p.o_dtype = o_dtype;
    p.status = &static_cast<f3s::WsHeader*>(d_workspace)->status;
    p.offsets = d_window_offsets;
    p.cols = d_block_cols;
    p.order = d_order;
    p.num_items = num_items;
    p.num_nodes = num_nodes;
    p.windows = windows;
    p.q_window_base = q_window_base;
    p.q_rows = q_rows;
    const int64_t units = (int64_t)num_items * heads;
    // one warp per window and head once that fills the SMs' warps
    p.warps_per_unit = units >= 16ll * f3s::num_sms_of_current_device() ? 1 : f3s::kAttendWarps;
    return f3s::attend_launch<2, false>(p, head_dim, units, (cudaStream_t)stream);
}

}  // extern "C"
