// f3s_kv4_prefill.cu -- causal attention over request pages for many new tokens:
// tiles of 128 query rows on tcgen05, K and V held in 4 bits.  (f3s_kv4_math.cuh
// has the formulas.)
//
// A block takes one work item (128 rows of a request and K/V head, a run of its
// pages) in steps of 64 tokens:
//   warps 0-7   two threads per query row, 32 tokens of the step each: scores,
//               weights; P (fp16) takes the place of S.  The two agree on the row's
//               reference by a barrier that also votes.
//   warps 8-11  unpack one page each: codes become fp16 (one AND per two values) in
//               shared memory, K as [token][channel], V as [channel][token], both in
//               the 128-byte swizzle; the scales go into arrays per token
//   warp 12     issues S = Q K^T into one of two S buffers in tensor memory, and
//               O += P V with P read from tensor memory
// S of a step runs while the weights of the one before are worked out, and two
// blocks share an SM.  A row's reference moves when a weight passes 2^15; then the
// rows' warps rescale O in tensor memory themselves, once the products before are
// done.
//
// V's rows are ordered so that unpacking does not collide in shared memory's
// banks: row r holds channel (r % 8) * D / 8 + r / 8.
//
// Accumulators are emptied every kRunPages pages (f3s_kv4_math.cuh) into sums in
// scratch, in a place that a block with more pages than that takes for its run.
//
// Bound: a chain of short waits (scores, vote, weights, product) with neither unit
// full: issue slots 44 % busy, most of it the weights (15 instructions and 2.5 loads from
// shared memory per two scores), tensor pipe 16 %.  Five prompts of up to 3,200 tokens,
// 32 / 8 heads, D = 128, 81 GFLOP, in a CUDA graph: 245 us with bf16 results, 332 TFLOP/s;
// 267 with fp16 and 273 with fp32 ones.  When it was first built, one thread per row
// with 64 tokens each took 316 us against 255, mma.sync with 32 rows 506.
#include <algorithm>
#include <type_traits>
#include "f3s_kv4_attend.cuh"
#include "f3s_tcgen05.cuh"

namespace f3s {

constexpr int kTileRows = 128;
constexpr int kStepTokens = 64;
constexpr int kRowWarps = 8;   // two halves of a step's tokens x 4 x 32 rows
constexpr int kCodeWarps = 4;  // a page each
constexpr int kTileThreads = (kRowWarps + kCodeWarps + 1) * 32;

template <int D>
struct TileCfg {
    static constexpr int RB = kv4_record_bytes(D);
    static constexpr int ATOMS = D / 64;             // 128-byte column blocks of Q and K
    static constexpr int Q_BYTES = ATOMS * kTileRows * 128;
    static constexpr int K_BYTES = ATOMS * kStepTokens * 128;
    static constexpr int V_BYTES = D * 128;
    static constexpr int Q = 0;
    static constexpr int K = Q + Q_BYTES;            // two buffers
    static constexpr int V = K + 2 * K_BYTES;        // two buffers
    static constexpr int TOKENS = V + 2 * V_BYTES;   // two buffers of [f, z, l, ri, y][64]
    static constexpr int TOKEN_BYTES = 5 * kStepTokens * 4;
    static constexpr int ROWS = TOKENS + 2 * TOKEN_BYTES;  // [unit scale, sum q][128], [largest, den, off][half][128]
    static constexpr int BARS = ROWS + 8 * kTileRows * 4;
    static constexpr int NBARS = 9;
    static constexpr int TMEM_SLOT = BARS + (NBARS * 8 + 15) / 16 * 16;
    static constexpr int SMEM = TMEM_SLOT + 16 + 1024;  // and room to align the base
    static constexpr int TMEM_COLUMNS = 256;         // S 2 x 64, O D
};

// A place for the sums of a block's runs, and its return; by one thread.  -1: none is
// free, which two blocks per SM leave no room for; the accumulators then run on.
__device__ __noinline__ int take_run_place(const Kv4PlanHeader* plan) {
    uint32_t* taken = const_cast<uint32_t*>(plan->run_taken);
    const int places = min(plan->run_places, 10 * 32), words = (places + 31) / 32;
    for (int i = 0; i < 64 * words; ++i) {
        const int w = (int)((blockIdx.x + i) % words);
        const uint32_t all = places - 32 * w >= 32 ? 0xffffffffu : (1u << (places - 32 * w)) - 1;
        const uint32_t free = ~(uint32_t)load_volatile(reinterpret_cast<int*>(taken + w)) & all;
        if (free == 0) continue;
        const uint32_t bit = free & (0u - free);
        if (atomicOr(taken + w, bit) & bit) continue;
        __threadfence();  // what its last owner wrote there comes first
        return 32 * w + __ffs((int)bit) - 1;
    }
    return -1;
}
__device__ __forceinline__ void return_run_place(const Kv4PlanHeader* plan, int place) {
    __threadfence();
    atomicAnd(const_cast<uint32_t*>(plan->run_taken) + place / 32, ~(1u << (place % 32)));
}

// Adds half of a row's columns of O to the sums of the runs before (row stride
// kTileRows, its reference behind them) and zeroes them, by a whole warp.
template <int D>
__device__ __noinline__ void end_run(float* runs, uint32_t tmem_row, int half, float minus_ref, bool first) {
    const float by = first ? 0.f : exp2_approx(fminf(minus_ref - runs[(D + half) * kTileRows], 0.f));
    runs[(D + half) * kTileRows] = minus_ref;
#pragma unroll 1
    for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
        uint32_t o[32];
        tmem_load32(tmem_row + c, o);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float* sum = runs + (c + i) * kTileRows;
            const float before = first ? 0.f : *sum;
            *sum = fmaf(before, by, __uint_as_float(o[i]));
            o[i] = 0;
        }
        __syncwarp();
        tmem_store32(tmem_row + c, o);
    }
    tc_wait_st();
}

template <int D, bool PRECISE>
__global__ void __launch_bounds__(kTileThreads, 2) k_attend4_tiles(const AttendParams p) {
    using C = TileCfg<D>;
    constexpr int RB = C::RB, W = D / 32;
    extern __shared__ __align__(1024) uint8_t raw_smem[];
    uint8_t* smem = raw_smem + ((1024u - (smem_addr(raw_smem) & 1023u)) & 1023u);
    const uint32_t base = smem_addr(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t kv_full = base + C::BARS, kv_empty = kv_full + 16, s_full = kv_empty + 16, p_full = s_full + 16,
                   q_full = p_full + 16;
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(kv_full + 8 * i, 128);
            mbar_init(kv_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, kRowWarps * 32);
        }
        mbar_init(q_full, 128);
        fence_mbar_init();
    }
    if (warp == kRowWarps + kCodeWarps) tmem_alloc(base + C::TMEM_SLOT, C::TMEM_COLUMNS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<const uint32_t*>(smem + C::TMEM_SLOT);
    const uint32_t tmem_o = tmem + 128;
    launch_dependents();
    wait_for_primary();  // the plan
    const int item = blockIdx.x / p.kv_heads, hk = blockIdx.x - item * p.kv_heads;
    const bool live = item < plan_items(p);
    Kv4Item it{};
    if (live) {
        const int4* src = reinterpret_cast<const int4*>(reinterpret_cast<const Kv4Item*>(p.plan + 1) + item);
        const int4 a = src[0], b = src[1];
        it.request = a.x;
        it.q_token = a.y;
        it.row0 = a.z;
        it.rows = a.w;
        it.context = b.x;
        it.page0 = b.y;
        it.page1 = b.z;
        it.slot = b.w;
    }
    const int steps = live ? (max(it.page1 - it.page0, 0) + 3) / 4 : 0;
    constexpr int RUN = kRunPages / 4;  // steps in a row
    volatile int* run_place = reinterpret_cast<int*>(smem + C::TMEM_SLOT) + 1;
    if (steps > RUN) {
        if (threadIdx.x == 0) *run_place = take_run_place(p.plan);
        __syncthreads();
    }
    const int last_row = min(it.row0 + kTileRows, it.rows) - 1;
    bool ok = true;  // false: a wait ran out; the warp stops waiting

    if (warp < kRowWarps && live) {
        // ------------------------------------------------------------ rows
        const int half = warp >> 2, quad = warp & 3;  // tokens 32 half ... of a step; rows 32 quad ...
        const int r = quad * 32 + lane, row = it.row0 + r;
        const bool valid = row < it.rows;
        const int at = min(row, last_row), tok = at / p.group;
        const int limit = it.context + tok;  // the last token this row sees
        const int64_t out_row = (int64_t)(it.q_token + tok) * p.heads + hk * p.group + at - tok * p.group;
        float* rows = reinterpret_cast<float*>(smem + C::ROWS);
        auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory"); };
        auto pair_any = [&](bool x) {
            uint32_t any;
            asm volatile(
                "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %2, 0;\n\tbar.red.or.pred b, %1, 64, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
                : "=r"(any)
                : "r"(1 + quad), "r"((uint32_t)x)
                : "memory");
            return any != 0;
        };
        // Q as fp16 times a power of two that brings the row's largest to [2^9, 2^10);
        // channels whose codes come in units of 2^-24 another 2^4
        if (half == 0) {
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) +
                                                              (int64_t)(it.q_token + tok) * p.q_token +
                                                              (int64_t)(hk * p.group + at - tok * p.group) * p.q_head);
            float amax = 0.f, sum = 0.f;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = valid ? src[c] : make_uint4(0, 0, 0, 0);
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float2 x = q_floats(u[n], p.q_bf16);
                    if (fabsf(x.x) < INFINITY) amax = fmaxf(amax, fabsf(x.x));  // NaN and infinities stay what they are
                    if (fabsf(x.y) < INFINITY) amax = fmaxf(amax, fabsf(x.y));
                }
            }
            const int e = amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 : 9;
            const int up = min(max(9 - e, -120), 120);  // 2^(9 - floor(log2 amax)), within fp32's normal range
            const float f = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = valid ? src[c] : make_uint4(0, 0, 0, 0);
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
                uint32_t h[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float2 x = q_floats(u[n], p.q_bf16);
                    const float m = n & 1 ? f : f * 16.f;
                    h[n] = pack_half2(x.x * m, x.y * m);
                    const float2 y = half2_floats(h[n]);
                    sum += (y.x + y.y) * (n & 1 ? 1.f : 0.0625f);
                }
                *reinterpret_cast<uint4*>(smem + C::Q + (c / 8) * (kTileRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                    make_uint4(h[0], h[1], h[2], h[3]);
            }
            rows[r] = p.scale * __uint_as_float((uint32_t)(127 - up) << 23);
            rows[kTileRows + r] = sum * 9.5367431640625e-7f;  // 2^-20: the codes' unit
            fence_proxy_async_shared();
            mbar_arrive(q_full);
        }
        pair_sync();
        const float unit_scale = rows[r], qs = rows[kTileRows + r];
        float* largest = rows + 2 * kTileRows;
        float* sums = rows + 4 * kTileRows;
        const uint32_t mine = tmem + ((uint32_t)quad << 21);  // lanes 32 quad ...
        const uint64_t scale2 = pair(unit_scale, unit_scale), qs2 = pair(qs, qs);
        float minus_ref = 0.f;
        uint64_t den = 0, off = 0;  // of this half's tokens
        bool unset = true;
        for (int j = 0; j < steps; ++j) {
            const int b = j & 1;
            ok = ok && phase_wait(s_full + 8 * b, j >> 1 & 1, p.status, p.status);
            if (pair_any(!ok)) {  // both halves leave together
                ok = false;
                break;
            }
            tc_fence_after();
            if (j > 0 && j % RUN == 0 && *run_place >= 0) {  // the run ends: O, once its products are in it, goes to the sums
                ok = phase_wait(kv_empty + 8 * (b ^ 1), (j - 1) >> 1 & 1, p.status, p.status) && ok;
                tc_fence_after();
                end_run<D>(p.partials - (*run_place + 1) * kv4_run_floats(D) + r, mine + 128, half, minus_ref, j == RUN);
            }
            const float* tokens = reinterpret_cast<const float*>(smem + C::TOKENS + b * C::TOKEN_BYTES) + 32 * half;
            const int tok0 = (it.page0 + 4 * j) * 16 + 32 * half;
            uint32_t hi[16], lo[PRECISE ? 16 : 1];  // P, two tokens each, and what its rounding drops
            // Weights and sums against the reference as it stands; the largest score.  A score
            // is rounded before the reference is taken off, so that no weight passes
            // 2^8 once the reference is the largest score less 7, however large that is.
            auto weigh_row = [&](auto hides, uint64_t& den_out, uint64_t& off_out) {
                constexpr bool HIDES = decltype(hides)::value;
                float most = -INFINITY;
                uint64_t d = den, o = off;
                const uint64_t mref2 = pair(minus_ref, minus_ref);
                uint32_t s[32];
                tmem_load32(mine + 64 * b + 32 * half, s);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const ulonglong2 f = reinterpret_cast<const ulonglong2*>(tokens)[c];
                    const ulonglong2 z = reinterpret_cast<const ulonglong2*>(tokens + 64)[c];
                    const ulonglong2 l = reinterpret_cast<const ulonglong2*>(tokens + 128)[c];
                    ulonglong2 ri = reinterpret_cast<const ulonglong2*>(tokens + 192)[c];
                    ulonglong2 y = reinterpret_cast<const ulonglong2*>(tokens + 256)[c];
                    // scale s (q . u - z sum(q)) + log2 r
                    uint64_t x[2] = {pair(__uint_as_float(s[4 * c]), __uint_as_float(s[4 * c + 1])),
                                     pair(__uint_as_float(s[4 * c + 2]), __uint_as_float(s[4 * c + 3]))};
                    x[0] = fma2(mul2(f.x, fma2(z.x, qs2, x[0])), scale2, l.x);
                    x[1] = fma2(mul2(f.y, fma2(z.y, qs2, x[1])), scale2, l.y);
                    if constexpr (HIDES) {
                        // a hidden token's scale and zero may be anything, NaN too
                        const int left = limit - (tok0 + 4 * c);  // tokens up to this one are seen
                        auto keep = [](uint64_t v, bool a, bool c2, float other) {
                            const float2 w = unpair(v);
                            return pair(a ? w.x : other, c2 ? w.y : other);
                        };
                        x[0] = keep(x[0], left >= 0, left >= 1, -INFINITY);
                        x[1] = keep(x[1], left >= 2, left >= 3, -INFINITY);
                        ri.x = keep(ri.x, left >= 0, left >= 1, 0.f);
                        ri.y = keep(ri.y, left >= 2, left >= 3, 0.f);
                        y.x = keep(y.x, left >= 0, left >= 1, 0.f);
                        y.y = keep(y.y, left >= 2, left >= 3, 0.f);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 v = unpair(x[i]), w = unpair(add2(x[i], mref2));
                        most = fmaxf(most, fmaxf(v.x, v.y));
                        const float2 a = make_float2(exp2_approx(w.x), exp2_approx(w.y));
                        hi[2 * c + i] = pack_half2(a.x, a.y);
                        const float2 h = half2_floats(hi[2 * c + i]);
                        if constexpr (PRECISE) lo[2 * c + i] = pack_half2(a.x - h.x, a.y - h.y);
                        const uint64_t a2 = PRECISE ? pair(a.x, a.y) : pair(h.x, h.y);  // the same weights in every sum
                        d = fma2(a2, i ? ri.y : ri.x, d);
                        o = fma2(a2, i ? y.y : y.x, o);
                    }
                }
                den_out = d;
                off_out = o;
                return most;
            };
            // the warp's first row sees the least
            const bool hides = tok0 + 32 > it.context + (it.row0 + 32 * quad) / p.group + 1;
            uint64_t den_new, off_new;
#pragma unroll 1
            for (bool again = false;; again = true) {  // twice at most
                const float most = hides ? weigh_row(std::true_type{}, den_new, off_new)
                                         : weigh_row(std::false_type{}, den_new, off_new);
                // Past these barriers both halves have read their scores.
                if (again) {
                    pair_sync();
                    break;
                }
                // a row that has seen nothing takes its first largest score as the reference
                if (!pair_any(unset ? most > -INFINITY : most + minus_ref > kRescaleAt)) break;
                largest[half * kTileRows + r] = most;
                pair_sync();
                const float m = fmaxf(most, largest[(half ^ 1) * kTileRows + r]);
                const float before = minus_ref;
                if (m > -INFINITY) minus_ref = unset ? kTopWeight - m : fminf(minus_ref, kTopWeight - m);
                const float down = unset ? 1.f : exp2_approx(minus_ref - before);
                unset = unset && !(m > -INFINITY);
                den = mul2(den, pair(down, down));
                off = mul2(off, pair(down, down));
                if (j > 0) {  // O, once the products so far are in it: half of its columns each
                    ok = phase_wait(kv_empty + 8 * (b ^ 1), (j - 1) >> 1 & 1, p.status, p.status) && ok;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
                        uint32_t o[32];
                        tmem_load32(mine + 128 + c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
                        tmem_store32(mine + 128 + c, o);
                    }
                    tc_wait_st();
                }
            }
            den = den_new;
            off = off_new;
            __syncwarp();
            tmem_store16(mine + 64 * b + 16 * half, hi);
            if constexpr (PRECISE) tmem_store16(mine + 64 * b + 32 + 16 * half, lo);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(p_full + 8 * b);
        }
        // ---- the result
        if (ok && steps > 0) {
            ok = phase_wait(kv_empty + 8 * ((steps - 1) & 1), (steps - 1) >> 1 & 1, p.status, p.status);
            tc_fence_after();
        }
        {
            const float2 d2 = unpair(den), o2 = unpair(off);
            sums[half * kTileRows + r] = d2.x + d2.y;
            sums[(2 + half) * kTileRows + r] = o2.x + o2.y;
        }
        pair_sync();
        const float row_den = sums[r] + sums[kTileRows + r], row_off = sums[2 * kTileRows + r] + sums[3 * kTileRows + r];
        const float inv = it.slot >= 0 ? 1.f : row_den != 0.f ? __frcp_rn(row_den) : 0.f;
        float* part = it.slot >= 0 ? p.partials + ((int64_t)it.slot * p.kv_heads + hk) * kTileRows * (D + 2) : nullptr;
#pragma unroll 1
        for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            uint32_t o[32] = {};
            __syncwarp();
            if (steps > 0) {
                tmem_load32(mine + 128 + c, o);
                tc_wait_ld();
            }
            if (!valid) continue;
            if (steps > RUN && *run_place >= 0) {  // and the runs that ended
                const float* runs = p.partials - (*run_place + 1) * kv4_run_floats(D) + r;
                const float by = exp2_approx(fminf(minus_ref - runs[(D + half) * kTileRows], 0.f));
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(runs[(c + i) * kTileRows], by, __uint_as_float(o[i])));
            }
            // column c + 8 i + g holds channel g * D / 8 + c / 8 + i, its codes in units of
            // 2^-24 (even i) and 2^-20
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = fmaf(__uint_as_float(o[8 * i + g]), i & 1 ? 1048576.f : 16777216.f, -row_off) * inv;
                if (part) *reinterpret_cast<float4*>(part + r * D + g * (D / 8) + c / 8) = make_float4(v[0], v[1], v[2], v[3]);
                else store_channels<4>(p.o, out_row * D + g * (D / 8) + c / 8, v, p.o_dtype);
            }
        }
        if (part && valid && half == 0)
            *reinterpret_cast<float2*>(part + kTileRows * D + 2 * r) = make_float2(unset ? kNoReference : -minus_ref, row_den);
        tc_fence_before();
    } else if (warp < kRowWarps + kCodeWarps && live) {
        // ------------------------------------------------------------ codes
        const int dw = warp - kRowWarps, g = lane >> 2, t = lane & 3;
        const int64_t page_bytes = (int64_t)p.kv_heads * RB;
        const int* list = p.tables + (int64_t)it.request * p.table_stride;
        const int last_seen = it.context + last_row / p.group;
        auto id_of = [&](int j) {
            const int page = it.page0 + 4 * j + dw;
            int id = page < it.page1 ? list[page] : -1;
            if (id < -1 || id >= p.num_pages) {
                atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
                id = -1;
            }
            return id;
        };
        uint32_t kg[W], kh[W], v0[W], v1[W];
        uint2 sc;
        auto load = [&](int id) {
            const uint8_t* rec = p.pages + (int64_t)max(id, 0) * page_bytes + (int64_t)hk * RB;
            lds_words<W>(rec + g * (D / 2) + t * (D / 8), kg);
            lds_words<W>(rec + (g + 8) * (D / 2) + t * (D / 8), kh);
            lds_words<W>(rec + 8 * D + lane * (D / 8), v0);
            lds_words<W>(rec + 12 * D + lane * (D / 8), v1);
            sc = *reinterpret_cast<const uint2*>(rec + kv4_scale_off(D, lane & 15));
        };
        int id = steps > 0 ? id_of(0) : -1, id_next = steps > 1 ? id_of(1) : -1;
        if (steps > 0) load(id);
        for (int j = 0; j < steps && ok; ++j) {
            const int b = j & 1;
            ok = phase_wait(kv_empty + 8 * b, (j >> 1 & 1) ^ 1, p.status, p.status);
            if (!ok) break;
            uint8_t* ks = smem + C::K + b * C::K_BYTES;
            uint8_t* vs = smem + C::V + b * C::V_BYTES;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int chunk = t * W + w;  // of 8 channels
                const uint32_t g8 = kg[w] >> 8, h8 = kh[w] >> 8;
                uint8_t* dst = ks + (chunk / 8) * (kStepTokens * 128) + (dw * 16 + g) * 128 + (((chunk & 7) ^ g) << 4);
                *reinterpret_cast<uint4*>(dst) = make_uint4(kg[w] & kNib0, kg[w] & kNib1, g8 & kNib0, g8 & kNib1);
                *reinterpret_cast<uint4*>(dst + 8 * 128) = make_uint4(kh[w] & kNib0, kh[w] & kNib1, h8 & kNib0, h8 & kNib1);
                const uint32_t a8 = v0[w] >> 8, b8 = v1[w] >> 8;
                const uint32_t an[4] = {v0[w] & kNib0, v0[w] & kNib1, a8 & kNib0, a8 & kNib1};
                const uint32_t bn[4] = {v1[w] & kNib0, v1[w] & kNib1, b8 & kNib0, b8 & kNib1};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    uint8_t* to = vs + ((4 * w + n) * 8 + g) * 128 + 4 * t;
                    *reinterpret_cast<uint32_t*>(to + (((2 * dw) ^ g) << 4)) = an[n];
                    *reinterpret_cast<uint32_t*>(to + (((2 * dw + 1) ^ g) << 4)) = bn[n];
                }
            }
            if (lane < 16) {
                float* tokens = reinterpret_cast<float*>(smem + C::TOKENS + b * C::TOKEN_BYTES) + dw * 16 + lane;
                const float2 k2 = half2_floats(sc.x), v2 = half2_floats(sc.y);
                const float r = v2.x < kKv4MinScale ? kKv4MinScale : v2.x;  // keeps a NaN
                // tokens that no row of the tile sees weigh nothing, whatever is there
                const bool hidden = id < 0 || (it.page0 + 4 * j + dw) * 16 + lane > last_seen;
                tokens[0] = hidden ? 0.f : k2.x * 1048576.f;  // 2^20
                tokens[64] = hidden ? 0.f : -k2.y;
                tokens[128] = hidden ? -INFINITY : log2_approx(r);
                tokens[192] = hidden ? 0.f : rcp_approx(r);
                tokens[256] = hidden ? 0.f : v2.y;
            }
            id = id_next;
            if (j + 1 < steps) load(id);
            if (j + 2 < steps) id_next = id_of(j + 2);
            fence_proxy_async_shared();
            mbar_arrive(kv_full + 8 * b);
        }
    } else if (warp == kRowWarps + kCodeWarps && live && steps > 0) {
        // ------------------------------------------------------------ products
        uint32_t last = 0, last_parity = 0;  // what the last products issued arrive on
        ok = phase_wait(q_full, 0, p.status, p.status);
        auto weigh = [&](int j) {  // O += P V of step j
            const int b = j & 1;
            ok = phase_wait(p_full + 8 * b, j >> 1 & 1, p.status, p.status);
            if (!ok) return;
            tc_fence_after();
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < kStepTokens / 16; ++k) {
                    const uint64_t v = smem_operand(base + C::V + b * C::V_BYTES + 32 * k);
                    mma_ts(tmem_o, tmem + 64 * b + 8 * k, v, mma_f16_shape(kTileRows, D), j > 0 || k > 0);
                    if constexpr (PRECISE) mma_ts(tmem_o, tmem + 64 * b + 32 + 8 * k, v, mma_f16_shape(kTileRows, D), true);
                }
                mma_commit(kv_empty + 8 * b);  // K, V, the tokens' numbers and P are free, O is the step's
            }
            last = kv_empty + 8 * b;
            last_parity = j >> 1 & 1;
            __syncwarp();
        };
        for (int j = 0; j < steps && ok; ++j) {
            const int b = j & 1;
            ok = phase_wait(kv_full + 8 * b, j >> 1 & 1, p.status, p.status);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_ss(tmem + 64 * b, smem_operand(base + C::Q + (k / 4) * (kTileRows * 128) + 32 * (k % 4)),
                           smem_operand(base + C::K + b * C::K_BYTES + (k / 4) * (kStepTokens * 128) + 32 * (k % 4)),
                           mma_f16_shape(kTileRows, kStepTokens), k > 0);
                mma_commit(s_full + 8 * b);
            }
            last = s_full + 8 * b;
            last_parity = j >> 1 & 1;
            __syncwarp();
            if (j > 0) weigh(j - 1);
        }
        if (ok) weigh(steps - 1);
        // tensor and shared memory are given up after the products
        if (last) mbar_drain(last, last_parity, kDrainNs);
    }
    __syncthreads();
    if (steps > RUN && threadIdx.x == 0 && *run_place >= 0) return_run_place(p.plan, *run_place);
    if (warp == kRowWarps + kCodeWarps) {
        tc_fence_after();
        tmem_free(tmem, C::TMEM_COLUMNS);
    }
}

template <int D, bool PRECISE>
static int tiles_variant(const AttendParams& p, int64_t units, cudaStream_t stream) {
    using C = TileCfg<D>;
    static PerContext<int> attr;
    const int rc = attr.get(nullptr, [](int* v) -> int {
        *v = 1;
        F3S_CUDA_TRY(cudaFuncSetAttribute(k_attend4_tiles<D, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        return F3S_SUCCESS;
    });
    if (rc != F3S_SUCCESS) return rc;
    if (units > INT32_MAX) return F3S_ERR_TOO_LARGE;
    if (units == 0) return F3S_SUCCESS;
    return launch_after(k_attend4_tiles<D, PRECISE>, (unsigned)units, kTileThreads, C::SMEM, stream, p);
}

int attend_tiles128(const AttendParams& p, int head_dim, int64_t units, cudaStream_t stream) {
    const bool precise = weights_in_full(p.o_dtype);
    if (head_dim == 64) return precise ? tiles_variant<64, true>(p, units, stream) : tiles_variant<64, false>(p, units, stream);
    return precise ? tiles_variant<128, true>(p, units, stream) : tiles_variant<128, false>(p, units, stream);
}

}  // namespace f3s
