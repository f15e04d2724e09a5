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
// one vote per step decides.
//
// A block has four consumer warps and one producer warp.  The producer walks
// the page lists and copies one or two pages per step, the records of up to four
// K/V heads in one bulk copy per page (they lie together), into a ring of
// stages; it runs ahead over the ends of the units.  A consumer warp has a head
// of its own; with fewer than four heads to a block, warps share a head and
// take its steps in turn (their sums are added at the end).
//
// The codes are unpacked in registers, one AND per two values (f3s_kv4.cuh), and
// multiplied with mma.m16n8k16:
//   8 query rows per tile (decoding): the cache is the 16-row operand, S^T = K Q^T
//     and O^T = V^T P^T; P turns from accumulator to operand through movmatrix.
//   16 and 32 rows: Q and P are the 16-row operands, P's accumulators being its
//     operand registers already.
// What a token multiplies by (scale, zero, log2 r, 1 / r, y) is worked out by one
// lane per token, put down in shared memory and read as pairs; the arithmetic on
// scores runs on pairs of fp32 numbers.  tcgen05's M = 64 / 128 rows would stand
// mostly empty: 8 to 32 query rows share a page.
//
// Bound: HBM where few query rows read a page (decoding: D + 8 bytes per token
// and K/V head); the rate of instructions where many do.
#include <algorithm>
#include <cuda_bf16.h>
#include "f3s_internal.cuh"
#include "f3s_kv4.cuh"
#include "f3s_kv4_plan.cuh"

namespace f3s {

constexpr int kConsumers = 4;
constexpr int kAttendThreads = (kConsumers + 1) * 32;
constexpr int kRingHeadSteps = 16;  // stages times K/V heads per stage
constexpr uint64_t kAttendTimeoutNs = 5ull * 1000 * 1000 * 1000;
constexpr float kNoReference = -3.0e38f;  // finite: a weight against it is 0, not NaN
constexpr float kRescaleAt = 8.f;

// The windows of a graph as work (k_window_pieces): item i is the i-th listed
// window or its first piece, the other pieces of cut windows follow behind the
// listed ones.
struct WindowPieces {
    int extra, splits, slots, ticket;
    int pad[60];
};
static_assert(sizeof(WindowPieces) == 256, "piece header is 256 bytes");

struct AttendParams {
    const void* q;
    int64_t q_token, q_head;  // strides in elements
    int q_bf16;
    const uint8_t* pages;
    int num_pages;
    int kv_heads, heads, group;
    int hg;        // heads per unit, one per consumer warp (times 4 / hg warps)
    int kvs;       // K/V heads per stage
    int stages;    // kRingHeadSteps / kvs
    float scale;   // times log2(e)
    void* o;       // contiguous [rows, heads, D] of o_dtype
    int o_dtype;
    int* status;
    float* partials;  // (rows of a tile) x (D + 2) floats per slot and head
    // paged
    const Kv4PlanHeader* plan;
    const int* tables;
    int64_t table_stride;
    // windows
    WindowPieces* pieces;
    const int4* items;  // window (-1: none), first block, end block, slot or -1
    const int4* window_splits;
    int num_items, extra_cap, splits_cap;
    const int* cols;
    int num_nodes, windows, q_window_base, q_rows;
};

// Pieces of at most `piece` blocks: a quarter of a block's even share of the
// work (3 blocks per SM), and 16 per warp that takes them in any case.
struct WindowPieceLayout {
    int piece;
    int64_t extra_cap, splits_cap, slots_cap;
    size_t items, splits, partials, total;
};

static int window_head_group(int heads, int group) {
    for (int hg = 4; hg > 1; hg >>= 1)
        if (heads % hg == 0 && (group % hg == 0 || hg % group == 0)) return hg;
    return 1;
}

static WindowPieceLayout window_piece_layout(int num_items, int64_t num_blocks, int heads, int group, int head_dim, int sms) {
    WindowPieceLayout L{};
    const int hg = window_head_group(heads, group);
    const int64_t blocks = 4 * 3ll * sms;
    const int64_t share = (num_blocks * (heads / hg) + blocks - 1) / blocks;
    L.piece = (int)std::min<int64_t>(std::max<int64_t>(share, 16 * (4 / hg)), 1 << 28);
    const int64_t cut = num_blocks / L.piece;
    L.extra_cap = cut;
    L.splits_cap = std::min<int64_t>(num_items, cut);
    L.slots_cap = 2 * cut;
    size_t off = sizeof(WindowPieces);
    L.items = off;
    off += (size_t)(num_items + L.extra_cap) * 16;
    L.splits = off;
    off += (size_t)L.splits_cap * 16;
    L.partials = off;
    off += (size_t)L.slots_cap * heads * 16 * (head_dim + 2) * 4;
    L.total = off;
    return L;
}

struct WindowPieceParams {
    const int* offsets;
    const int* order;
    int num_items, windows, q_window_base, q_rows;
    int piece, extra_cap, splits_cap, slots_cap;
    WindowPieces* pieces;
    int4* items;
    int4* splits;  // window, first slot, pieces, -
    int* status;
};

// One thread per listed window.  A block reserves its share of the extra items
// and slots with atomics, so their places vary; a window's cuts and the order in
// which its pieces are summed do not.
__global__ void __launch_bounds__(256) k_window_pieces(const WindowPieceParams p) {
    __shared__ int s_scan[256 / 32 + 1], s_base[3];
    const int i = blockIdx.x * 256 + threadIdx.x;
    int window = 0, b0 = 0, nb = 0;
    bool live = i < p.num_items;
    if (live) {
        window = p.order[i];
        live = window >= p.q_window_base && window < p.windows && (int64_t)(window - p.q_window_base) * 16 < p.q_rows;
        if (!live) {
            atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
            p.items[i] = make_int4(-1, 0, 0, -1);
        }
    }
    if (live) {
        b0 = p.offsets[window];
        nb = max(p.offsets[window + 1] - b0, 0);
    }
    const int parts = live && nb > p.piece ? (int)(((int64_t)nb + p.piece - 1) / p.piece) : 1;
    const bool split = parts > 1;
    int total[3], at[3];
    at[0] = block_exclusive_scan<256>(parts - 1, total[0], s_scan);
    at[1] = block_exclusive_scan<256>(split, total[1], s_scan);
    at[2] = block_exclusive_scan<256>(split ? parts : 0, total[2], s_scan);
    if (threadIdx.x < 3 && total[threadIdx.x] > 0) {
        int* counters[3] = {&p.pieces->extra, &p.pieces->splits, &p.pieces->slots};
        s_base[threadIdx.x] = atomicAdd(counters[threadIdx.x], total[threadIdx.x]);
    }
    __syncthreads();
    if (!live) return;
    if (split) {
        at[0] += s_base[0];
        at[1] += s_base[1];
        at[2] += s_base[2];
        if (at[0] + parts - 1 <= p.extra_cap && at[1] < p.splits_cap && at[2] + parts <= p.slots_cap) {
            for (int k = 0; k < parts; ++k) {
                const int lo = (int)((int64_t)nb * k / parts), hi = (int)((int64_t)nb * (k + 1) / parts);
                p.items[k == 0 ? i : p.num_items + at[0] + k - 1] = make_int4(window, b0 + lo, b0 + hi, at[2] + k);
            }
            p.splits[at[1]] = make_int4(window, at[2], parts, 0);
            return;
        }
        // more blocks than the caller said (a heavy window listed many times): one piece
        for (int k = 0; k < parts - 1 && at[0] + k < p.extra_cap; ++k)
            p.items[p.num_items + at[0] + k] = make_int4(-1, 0, 0, -1);
        if (at[1] < p.splits_cap) p.splits[at[1]] = make_int4(-1, 0, 0, 0);
    }
    p.items[i] = make_int4(window, b0, b0 + nb, -1);
}

// ROWS query rows per tile: 8 (the cache is the 16-row operand) or 16, 32.
template <int D, int ROWS>
struct AttendCfg {
    static constexpr int RB = kv4_record_bytes(D);
    static constexpr bool QM = ROWS > 8;        // Q is the 16-row operand
    static constexpr int PP = ROWS == 32 ? 1 : 2;  // pages per step
    static constexpr int MT = QM ? ROWS / 16 : 1;
    static constexpr int LANE_ROWS = 2 * MT;    // query rows whose sums a lane holds
    static constexpr int ACC = QM ? MT * D / 8 * 4 : D / 16 * 4;
    static constexpr bool Q_SMEM = ROWS * D > 16 * 64;
    static constexpr int RING = kRingHeadSteps * PP * RB;
    static constexpr int TOKENS = RING;         // per warp: what the tokens of a step multiply by
    static constexpr int TOKEN_BYTES = (QM ? 5 * 16 * 4 : 48 * 16) * PP;
    static constexpr int Q = TOKENS + kConsumers * TOKEN_BYTES;
    static constexpr int Q_BYTES = Q_SMEM ? ROWS * D * 2 : 0;  // per warp
    static constexpr int BARS = Q + kConsumers * Q_BYTES;
    static constexpr int NBARS = 2 * kRingHeadSteps + 4;
    static constexpr int UNITS = BARS + NBARS * 8;      // two unit records
    static constexpr int FLAGS = UNITS + 2 * 32;        // per stage
    static constexpr int SINK = FLAGS + kRingHeadSteps * 4;
    static constexpr int MERGE = (SINK + kConsumers * 4 + 127) / 128 * 128;  // two warps' sums, where warps share a head
    static constexpr int MERGE_WORDS = ACC + (3 * LANE_ROWS + 3) / 4 * 4;     // per lane
    static constexpr int SMEM = MERGE;
    static constexpr int SMEM_SHARED = MERGE + 2 * 32 * MERGE_WORDS * 4;
    static constexpr int MIN_CTAS = ACC >= 128 ? 2 : 3;
};

struct Unit {  // as the producer hands it to the consumers (graph)
    int live, window, slot, steps, head0;
    int pad[3];
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

// Waits for a phase of an mbarrier, by a whole warp; bounded.  False: give up.
static __device__ __noinline__ bool phase_wait_slow(uint32_t bar, uint32_t parity, int* status) {
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
__device__ __forceinline__ bool phase_wait(uint32_t bar, uint32_t parity, int* status) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, phase_wait_slow(bar, parity, status));
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

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

// The producer warp: units, their page lists, the copies.
template <int D, int PP, bool PAGED>
__device__ __forceinline__ void attend_produce(const AttendParams& p, uint32_t ring, uint32_t full, uint32_t empty,
                                               uint32_t unit_full, uint32_t unit_empty, Unit* unit_out, int* flags_out,
                                               int64_t units, int groups) {
    constexpr int RB = kv4_record_bytes(D);
    const int lane = threadIdx.x & 31;
    const int stages = p.stages, stage_bytes = PP * p.kvs * RB, copy_bytes = p.kvs * RB;
    const int64_t page_bytes = (int64_t)p.kv_heads * RB;
    const int limit = PAGED ? p.num_pages : p.windows;
    uint32_t n = 0;  // steps issued
    int ticket = 0;
    if (!PAGED && lane == 0) ticket = atomicAdd(&p.pieces->ticket, 1);
    for (int k = 0;; ++k) {
        const int* list;
        int count, head0;
        if constexpr (PAGED) {
            const int64_t unit = blockIdx.x + (int64_t)k * gridDim.x;
            if (unit >= units) return;
            const int item = (int)(unit / groups);
            const int4* src = reinterpret_cast<const int4*>(reinterpret_cast<const Kv4Item*>(p.plan + 1) + item);
            const int4 a = __ldg(src), b = __ldg(src + 1);
            list = p.tables + (int64_t)a.x * p.table_stride + b.y;
            count = max(b.z - b.y, 0);
            head0 = (int)(unit - (int64_t)item * groups) * p.hg;
        } else {
            const int unit = __shfl_sync(0xffffffffu, ticket, 0);
            const bool live = unit < units;
            int4 piece = make_int4(-1, 0, 0, -1);
            if (live) {
                if (lane == 0) ticket = atomicAdd(&p.pieces->ticket, 1);
                const int item = unit / groups, extra = min(p.pieces->extra, p.extra_cap);
                piece = __ldcg(p.items + (item < extra ? p.num_items + item : item - extra));
            }
            count = piece.x >= 0 ? piece.z - piece.y : 0;
            head0 = live ? unit % groups * p.hg : 0;
            list = p.cols + piece.y;
            if (!phase_wait(unit_empty + 8 * (k & 1), (k >> 1 & 1) ^ 1, p.status)) return;
            if (lane == 0) {
                unit_out[k & 1] = Unit{live, piece.x, piece.w, (count + PP - 1) / PP, head0};
                mbar_arrive(unit_full + 8 * (k & 1));
            }
            if (!live) return;
            if (piece.x >= 0) {  // the unit's Q rows, a line or more each, on their way to L2
                const int64_t row = (int64_t)(piece.x - p.q_window_base) * 16 + (lane & 15);
                if (row < p.q_rows) {
                    const char* at = static_cast<const char*>(p.q) + 2 * (row * p.q_token + (int64_t)head0 * p.q_head);
                    for (int off = (lane >> 4) * 128; off < p.hg * D * 2; off += 256)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(at + off));
                }
            }
        }
        const uint8_t* src = p.pages + (int64_t)(PAGED ? head0 : head0 / p.group) * RB;
        auto load_ids = [&](int i0) {
            int id = -1;
            if (i0 + lane < count) {
                id = __ldg(list + i0 + lane);
                if (id < 0 || id >= limit) {
                    if (!(PAGED && id == -1)) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
                    id = -1;
                }
            }
            return id;
        };
        int ids = load_ids(0), ids_next = 0;
        for (int i = 0; i < count; i += PP, ++n) {
            if ((i & 31) == 0) {
                if (i > 0) ids = ids_next;
                if (i + 32 < count) ids_next = load_ids(i + 32);
            }
            // lane k of the first PP copies page k
            const int id = __shfl_sync(0xffffffffu, ids, (i + lane) & 31);
            const bool mine = lane < PP, have = mine && i + lane < count;
            const uint32_t skip = __ballot_sync(0xffffffffu, mine && (!have || id < 0));
            const uint32_t tail = __ballot_sync(0xffffffffu, !PAGED && have && id == p.windows - 1);
            const uint32_t st = n & (stages - 1);
            if (!phase_wait(empty + 8 * st, (n / stages & 1) ^ 1, p.status)) return;
            if (lane == 0) {
                flags_out[st] = (int)(skip | tail << 8);
                mbar_arrive_expect_tx(full + 8 * st, min(PP, count - i) * copy_bytes);
            }
            if (have)
                bulk_load(ring + st * stage_bytes + lane * copy_bytes, src + (int64_t)max(id, 0) * page_bytes, copy_bytes,
                          full + 8 * st);
        }
    }
}

// PAGED: a unit is (work item of the plan, hg K/V heads), one or more per block.
// Otherwise persistent blocks take units (window or piece, hg query heads) by
// ticket.  PRECISE adds the part of P that rounding to fp16 drops with a second
// product, which makes the result as exact as fp32 arithmetic.
template <int D, int ROWS, bool PAGED, bool PRECISE>
__global__ void __launch_bounds__(kAttendThreads, AttendCfg<D, ROWS>::MIN_CTAS) k_attend4(const AttendParams p) {
    using C = AttendCfg<D, ROWS>;
    constexpr int RB = C::RB, MT = C::MT, PP = C::PP;
    constexpr bool QM = C::QM;
    constexpr int W = D / 32;             // words of a token's K (and of a token pair's V) per lane
    constexpr int CH = QM ? D / 4 : D / 8;  // output channels per lane and row
    constexpr int NR = C::LANE_ROWS;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t base = smem_addr(smem), full = base + C::BARS, empty = full + 8 * kRingHeadSteps;
    const uint32_t unit_full = empty + 8 * kRingHeadSteps, unit_empty = unit_full + 16;
    Unit* unit_records = reinterpret_cast<Unit*>(smem + C::UNITS);
    int* stage_flags = reinterpret_cast<int*>(smem + C::FLAGS);
    const int hg = p.hg, turns = kConsumers / hg;  // warps that share a head take its steps in turn
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, hg);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(unit_full + 8 * i, 1);
            mbar_init(unit_empty + 8 * i, kConsumers);
        }
        fence_mbar_init();
    }
    __syncthreads();
    const int unit_heads = PAGED ? p.kv_heads : p.heads, groups = unit_heads / hg;
    const int64_t units = (int64_t)(PAGED ? p.plan->num_items : p.num_items + min(p.pieces->extra, p.extra_cap)) * groups;
    if (warp == kConsumers) {
        attend_produce<D, C::PP, PAGED>(p, base, full, empty, unit_full, unit_empty, unit_records, stage_flags, units, groups);
        return;
    }

    const int hh = warp % hg, turn = warp / hg;
    const uint32_t sink = base + C::SINK + warp * 4;
    uint8_t* tokens = smem + C::TOKENS + warp * C::TOKEN_BYTES;
    uint4* qsm = reinterpret_cast<uint4*>(smem + C::Q + warp * C::Q_BYTES);
    const int stage_bytes = PP * p.kvs * RB;
    bool dead = false;  // a wait ran out: nothing more is read
    uint32_t done = 0;  // steps of the units before this one

    for (int k = 0;; ++k) {
        Kv4Item it{};
        int steps, head, slot, window = 0;
        if constexpr (PAGED) {
            const int64_t unit = blockIdx.x + (int64_t)k * gridDim.x;
            if (unit >= units) break;
            const int item = (int)(unit / groups);
            head = (int)(unit - (int64_t)item * groups) * hg + hh;
            const int4* src = reinterpret_cast<const int4*>(reinterpret_cast<const Kv4Item*>(p.plan + 1) + item);
            const int4 a = __ldg(src), b = __ldg(src + 1);
            it.q_token = a.y;
            it.row0 = a.z;
            it.rows = a.w;
            it.context = b.x;
            it.page0 = b.y;
            slot = b.w;
            steps = (max(b.z - b.y, 0) + PP - 1) / PP;
        } else {
            if (!phase_wait(unit_full + 8 * (k & 1), k >> 1 & 1, p.status)) break;
            const Unit u = unit_records[k & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(unit_empty + 8 * (k & 1));
            if (!u.live) break;
            if (u.window < 0) continue;  // no steps either
            window = u.window;
            slot = u.slot;
            steps = u.steps;
            head = u.head0 + hh;
        }
        const int kv_off = (PAGED ? hh : head / p.group - (head - hh) / p.group) * RB;  // in a page of a stage

        // ---- Q as fp16 times a power of two that brings the tile's largest to
        // [2^9, 2^10); channels whose codes come in units of 2^-24 another 2^4.
        // Lane (g, t): rows g (and g + 8, ...), channels t * D / 4 ...
        uint32_t qf[C::Q_SMEM ? 1 : QM ? 2 * MT : 1][C::Q_SMEM ? 1 : W][4];
        uint64_t qs[QM ? NR : 1];  // sum of q in the scores' unit: (row, row), or rows (2t, 2t + 1)
        float unit_scale;
        {
            constexpr int R = QM ? 2 * MT : 1;
            float amax = 0.f, sums[R];
            uint4 raw[R][W];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                int64_t off = -1;
                if constexpr (PAGED) {
                    const int row = it.row0 + 8 * r + g;
                    if (row < it.rows) {
                        const int tok = row / p.group;
                        off = (int64_t)(it.q_token + tok) * p.q_token + (int64_t)(head * p.group + row - tok * p.group) * p.q_head;
                    }
                } else {
                    const int64_t row = (int64_t)(window - p.q_window_base) * 16 + 8 * r + g;
                    if (row < p.q_rows) off = row * p.q_token + (int64_t)head * p.q_head;
                }
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + off + t * (D / 4));
#pragma unroll
                for (int w = 0; w < W; ++w) raw[r][w] = off >= 0 ? __ldg(src + w) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t u[4] = {raw[r][w].x, raw[r][w].y, raw[r][w].z, raw[r][w].w};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float2 x = q_floats(u[n], p.q_bf16);
                        const float a = fabsf(x.x), b = fabsf(x.y);
                        if (a < INFINITY) amax = fmaxf(amax, a);  // NaN and infinities stay what they are
                        if (b < INFINITY) amax = fmaxf(amax, b);
                    }
                }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            // 2^(9 - floor(log2 amax)), kept within fp32's normal range
            const int e = amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 : 9;
            const int up = min(max(9 - e, -120), 120);
            const float f = __uint_as_float((uint32_t)(up + 127) << 23);
            unit_scale = p.scale * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t u[4] = {raw[r][w].x, raw[r][w].y, raw[r][w].z, raw[r][w].w};
                    uint32_t h[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float2 x = q_floats(u[n], p.q_bf16);
                        const float m = n & 1 ? f : f * 16.f;
                        h[n] = pack_half2(x.x * m, x.y * m);
                        const float2 y = half2_floats(h[n]);
                        sum += (y.x + y.y) * (n & 1 ? 1.f : 0.0625f);
                    }
                    if constexpr (C::Q_SMEM) {
                        qsm[(r * W + w) * 32 + lane] = make_uint4(h[0], h[1], h[2], h[3]);
                    } else {
#pragma unroll
                        for (int n = 0; n < 4; ++n) qf[r][w][n] = h[n];
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sums[r] = sum * 9.5367431640625e-7f;  // 2^-20
            }
            if constexpr (QM) {
#pragma unroll
                for (int r = 0; r < NR; ++r) qs[r] = pair(sums[r], sums[r]);
            } else {
                // row 2t is summed in lanes 4 * 2t ..., row 2t + 1 in the next four
                qs[0] = pair(__shfl_sync(0xffffffffu, sums[0], 8 * t), __shfl_sync(0xffffffffu, sums[0], 8 * t + 4));
            }
            // each lane reads back what it wrote itself: no barrier
        }

        float acc[C::ACC / 4][4];
        // -R, sum a / r, sum a y.  16 and 32 rows: a row's, over this lane's even and
        // odd tokens (R twice); 8 rows: rows (2t, 2t + 1)
        uint64_t minus_ref[QM ? NR : 1], den[QM ? NR : 1], off[QM ? NR : 1];
#pragma unroll
        for (int m = 0; m < C::ACC / 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
#pragma unroll
        for (int r = 0; r < (QM ? NR : 1); ++r) minus_ref[r] = den[r] = off[r] = 0;
        uint32_t unset = (1u << NR) - 1;  // rows that have no reference yet (a bit each)
        // first token that some row of the tile must not see
        const int open = PAGED ? it.context + it.row0 / p.group + 1 : 0;

        for (int j = turn; j < steps && !dead; j += turns) {
            const uint32_t n = done + j, st = n & (p.stages - 1);
            if (!phase_wait(full + 8 * st, n / p.stages & 1, p.status)) {
                dead = true;
                break;
            }
            const uint8_t* rec0 = smem + st * stage_bytes + kv_off;
            const int flags = stage_flags[st];
            uint32_t dep;
            // ---- what each token multiplies by, one lane per token: f = scale s, -z f,
            // log2 r, 1 / r, y
            {
                const int tk = lane & 15, pg = PP == 2 ? lane >> 4 : 0;  // one page: both halves of the warp do the same
                const uint2 sc = *reinterpret_cast<const uint2*>(rec0 + pg * p.kvs * RB + kv4_scale_off(D, tk));
                dep = sc.x;
                const float2 ks = half2_floats(sc.x), vs = half2_floats(sc.y);
                const float f = ks.x * 1048576.f * unit_scale;  // 2^20: the codes' unit
                const float r = vs.x < kKv4MinScale ? kKv4MinScale : vs.x;  // keeps a NaN
                const float z = -ks.y * f, l = log2_approx(r), ri = rcp_approx(r);
                if constexpr (QM) {  // [page][f, z, l, ri, y][t][token 2t, 2t + 1, 2t + 8, 2t + 9]
                    float* dst = reinterpret_cast<float*>(tokens) + pg * 80 + ((tk & 7) >> 1) * 4 + (tk >> 3) * 2 + (tk & 1);
                    dst[0] = f;
                    dst[16] = z;
                    dst[32] = l;
                    dst[48] = ri;
                    dst[64] = vs.y;
                } else {  // [token][f, f, z, z][ri, ri, y, y][l, l, -, -]
                    float4* dst = reinterpret_cast<float4*>(tokens + (pg * 16 + tk) * 48);
                    dst[0] = make_float4(f, f, z, z);
                    dst[1] = make_float4(ri, ri, vs.y, vs.y);
                    *reinterpret_cast<float2*>(dst + 2) = make_float2(l, l);
                }
            }
            __syncwarp();
            // scores less the reference.  16 and 32 rows: row r, tokens (2t, 2t + 1) and (2t + 8,
            // 2t + 9); 8 rows: rows (2t, 2t + 1), tokens g and g + 8
            uint64_t x[PP][QM ? NR : 1][2];
#pragma unroll
            for (int k2 = 0; k2 < PP; ++k2) {
                const uint8_t* rec = rec0 + k2 * p.kvs * RB;
                uint32_t kg[W], kh[W];
                lds_words<W>(rec + g * (D / 2) + t * (D / 8), kg);
                lds_words<W>(rec + (g + 8) * (D / 2) + t * (D / 8), kh);
                dep ^= kg[0] ^ kh[0];
                float s[QM ? 2 * MT : 1][4];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t g8 = kg[w] >> 8, h8 = kh[w] >> 8;
                    const uint32_t gn[4] = {kg[w] & kNib0, kg[w] & kNib1, g8 & kNib0, g8 & kNib1};
                    const uint32_t hn[4] = {kh[w] & kNib0, kh[w] & kNib1, h8 & kNib0, h8 & kNib1};
                    if constexpr (QM) {
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            uint32_t lo[4], hi[4];  // rows g and g + 8
                            if constexpr (C::Q_SMEM) {
                                const uint4 a = qsm[(2 * m * W + w) * 32 + lane], b = qsm[((2 * m + 1) * W + w) * 32 + lane];
                                lo[0] = a.x, lo[1] = a.y, lo[2] = a.z, lo[3] = a.w;
                                hi[0] = b.x, hi[1] = b.y, hi[2] = b.z, hi[3] = b.w;
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) lo[i] = qf[2 * m][w][i], hi[i] = qf[2 * m + 1][w][i];
                            }
                            const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
                            if (w == 0) {
                                mma_16816_zero(s[2 * m], a0, gn[0], gn[1]);
                                mma_16816_zero(s[2 * m + 1], a0, hn[0], hn[1]);
                            } else {
                                mma_16816(s[2 * m], a0, gn[0], gn[1]);
                                mma_16816(s[2 * m + 1], a0, hn[0], hn[1]);
                            }
                            mma_16816(s[2 * m], a1, gn[2], gn[3]);
                            mma_16816(s[2 * m + 1], a1, hn[2], hn[3]);
                        }
                    } else {
                        const uint32_t a0[4] = {gn[0], hn[0], gn[1], hn[1]}, a1[4] = {gn[2], hn[2], gn[3], hn[3]};
                        uint32_t b[4];
                        if constexpr (C::Q_SMEM) {
                            const uint4 y = qsm[w * 32 + lane];
                            b[0] = y.x, b[1] = y.y, b[2] = y.z, b[3] = y.w;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) b[i] = qf[0][w][i];
                        }
                        if (w == 0) mma_16816_zero(s[0], a0, b[0], b[1]);
                        else mma_16816(s[0], a0, b[0], b[1]);
                        mma_16816(s[0], a1, b[2], b[3]);
                    }
                }
                if constexpr (QM) {
                    const float* tok = reinterpret_cast<const float*>(tokens) + k2 * 80 + 4 * t;
                    const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(tok);
                    const ulonglong2 z = *reinterpret_cast<const ulonglong2*>(tok + 16);
                    const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(tok + 32);
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const float* a = s[r & ~1] + 2 * (r & 1);
                        const float* b = s[r | 1] + 2 * (r & 1);
                        x[k2][r][0] = fma2(pair(a[0], a[1]), f.x, fma2(z.x, qs[r], add2(l.x, minus_ref[r])));
                        x[k2][r][1] = fma2(pair(b[0], b[1]), f.y, fma2(z.y, qs[r], add2(l.y, minus_ref[r])));
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const ulonglong2* tok = reinterpret_cast<const ulonglong2*>(tokens + (k2 * 16 + g + 8 * c) * 48);
                        const ulonglong2 fz = tok[0];
                        const uint64_t l = *reinterpret_cast<const uint64_t*>(tok + 2);
                        x[k2][0][c] = fma2(pair(s[0][2 * c], s[0][2 * c + 1]), fz.x, fma2(fz.y, qs[0], add2(l, minus_ref[0])));
                    }
                }
            }
            // ---- masks: only where a page has tokens that some row must not see
            const int tok0 = PAGED ? (it.page0 + j * PP) * 16 : 0;
            if (flags || (PAGED && tok0 + 16 * PP > open)) {
                __syncwarp();
#pragma unroll
                for (int k2 = 0; k2 < PP; ++k2) {
                    const bool skipped = flags >> k2 & 1, last = flags >> (8 + k2) & 1;
#pragma unroll
                    for (int r = 0; r < (QM ? NR : 1); ++r)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float2 y = unpair(x[k2][r][c]);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const int tk = QM ? 2 * t + 8 * c + i : g + 8 * c;
                                bool hide = skipped;
                                if constexpr (PAGED) {
                                    // a tile's rows past its last see what the last sees
                                    const int row = min(it.row0 + (QM ? 8 * r + g : 2 * t + i), it.rows - 1);
                                    hide = hide || tok0 + 16 * k2 + tk > it.context + row / p.group;
                                } else {
                                    hide = hide || (last && (p.windows - 1) * 16 + tk >= p.num_nodes);
                                }
                                if (hide) (i ? y.y : y.x) = -INFINITY;
                            }
                            x[k2][r][c] = pair(y.x, y.y);
                        }
                }
                // a hidden token's scale and zero may be anything: its weight of 0
                // must stay 0 (where it is seen, a NaN is in the weight already)
                if (PP == 1 && lane >= 16) {
                } else if constexpr (QM) {
                    float* own = reinterpret_cast<float*>(tokens) + (lane >> 4) * 80 + (lane & 15);
                    if (!(fabsf(own[48]) < INFINITY)) own[48] = 0.f;
                    if (!(fabsf(own[64]) < INFINITY)) own[64] = 0.f;
                } else {
                    float4* own = reinterpret_cast<float4*>(tokens + lane * 48) + 1;
                    float4 y = *own;
                    if (!(fabsf(y.x) < INFINITY)) y.x = y.y = 0.f;
                    if (!(fabsf(y.z) < INFINITY)) y.z = y.w = 0.f;
                    *own = y;
                }
                __syncwarp();
            }
            // ---- weights
            bool over = unset != 0;
#pragma unroll
            for (int k2 = 0; k2 < PP; ++k2)
#pragma unroll
                for (int r = 0; r < (QM ? NR : 1); ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float2 y = unpair(x[k2][r][c]);
                        over = over || y.x > kRescaleAt || y.y > kRescaleAt;
                    }
            if (__any_sync(0xffffffffu, over)) {
                float up[NR], down[NR];  // the reference moves up by `up`
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float m = -INFINITY;
#pragma unroll
                    for (int k2 = 0; k2 < PP; ++k2)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float2 y = unpair(x[k2][QM ? r : 0][c]);
                            m = fmaxf(m, QM ? fmaxf(y.x, y.y) : r ? y.y : y.x);
                        }
#pragma unroll
                    for (int o = QM ? 1 : 4; o < (QM ? 4 : 32); o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    if (unset >> r & 1) {  // nothing seen so far: the sums are 0, whatever they are scaled by
                        up[r] = m > -INFINITY ? m : 0.f;
                        down[r] = 1.f;
                        if (m > -INFINITY) unset &= ~(1u << r);
                    } else {
                        up[r] = fmaxf(m, 0.f);
                        down[r] = exp2_approx(-up[r]);
                    }
                }
#pragma unroll
                for (int r = 0; r < (QM ? NR : 1); ++r) {
                    const uint64_t minus = QM ? pair(-up[r], -up[r]) : pair(-up[0], -up[NR - 1]);
                    const uint64_t by = QM ? pair(down[r], down[r]) : pair(down[0], down[NR - 1]);
                    minus_ref[r] = add2(minus_ref[r], minus);
                    den[r] = fma2(den[r], by, 0);
                    off[r] = fma2(off[r], by, 0);
#pragma unroll
                    for (int k2 = 0; k2 < PP; ++k2)
#pragma unroll
                        for (int c = 0; c < 2; ++c) x[k2][r][c] = add2(x[k2][r][c], minus);
                }
                if constexpr (QM) {
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int e = 0; e < D / 8; ++e)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[m * (D / 8) + e][i] *= down[2 * m + i / 2];
                } else {
#pragma unroll
                    for (int e = 0; e < D / 16; ++e)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[e][i] *= down[i & 1];
                }
            }
#pragma unroll
            for (int k2 = 0; k2 < PP; ++k2) {
                uint32_t pb[MT][4], pl[MT][4];  // P: a 16-row operand, or (first two) an 8-column one
                ulonglong2 ri, vz;              // 1 / r and y
                if constexpr (QM) {
                    const float* tok = reinterpret_cast<const float*>(tokens) + k2 * 80 + 4 * t;
                    ri = *reinterpret_cast<const ulonglong2*>(tok + 48);
                    vz = *reinterpret_cast<const ulonglong2*>(tok + 64);
                } else {
                    const ulonglong2 a = reinterpret_cast<const ulonglong2*>(tokens + (k2 * 16 + g) * 48)[1];
                    const ulonglong2 b = reinterpret_cast<const ulonglong2*>(tokens + (k2 * 16 + g + 8) * 48)[1];
                    ri.x = a.x, vz.x = a.y, ri.y = b.x, vz.y = b.y;
                }
#pragma unroll
                for (int r = 0; r < (QM ? NR : 1); ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float2 y = unpair(x[k2][r][c]);
                        const float2 a = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                        const uint64_t a2 = pair(a.x, a.y);
                        const uint32_t h = pack_half2(a.x, a.y);
                        uint32_t low = 0;
                        if constexpr (PRECISE) {
                            const float2 b = half2_floats(h);
                            const float2 d = unpair(fma2(pair(b.x, b.y), pair(-1.f, -1.f), a2));
                            low = pack_half2(d.x, d.y);
                        }
                        if constexpr (QM) {
                            pb[r / 2][2 * c + (r & 1)] = h;
                            pl[r / 2][2 * c + (r & 1)] = low;
                        } else {
                            pb[0][c] = movmatrix_t(h);
                            if constexpr (PRECISE) pl[0][c] = movmatrix_t(low);
                        }
                        den[r] = fma2(a2, c ? ri.y : ri.x, den[r]);
                        off[r] = fma2(a2, c ? vz.y : vz.x, off[r]);
                    }
                // ---- O += P V, or O^T += V^T P^T
                const uint8_t* rec = rec0 + k2 * p.kvs * RB;
                uint32_t v0[W], v1[W];
                lds_words<W>(rec + 8 * D + lane * (D / 8), v0);
                lds_words<W>(rec + 12 * D + lane * (D / 8), v1);
                dep ^= v0[0] ^ v1[0];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t a8 = v0[w] >> 8, b8 = v1[w] >> 8;
                    const uint32_t an[4] = {v0[w] & kNib0, v0[w] & kNib1, a8 & kNib0, a8 & kNib1};
                    const uint32_t bn[4] = {v1[w] & kNib0, v1[w] & kNib1, b8 & kNib0, b8 & kNib1};
                    if constexpr (QM) {
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                mma_16816(acc[m * (D / 8) + 4 * w + i], pb[m], an[i], bn[i]);
                                if constexpr (PRECISE) mma_16816(acc[m * (D / 8) + 4 * w + i], pl[m], an[i], bn[i]);
                            }
                    } else {
                        const uint32_t a0[4] = {an[0], an[1], bn[0], bn[1]}, a1[4] = {an[2], an[3], bn[2], bn[3]};
                        mma_16816(acc[2 * w], a0, pb[0][0], pb[0][1]);
                        mma_16816(acc[2 * w + 1], a1, pb[0][0], pb[0][1]);
                        if constexpr (PRECISE) {
                            mma_16816(acc[2 * w], a0, pl[0][0], pl[0][1]);
                            mma_16816(acc[2 * w + 1], a1, pl[0][0], pl[0][1]);
                        }
                    }
                }
            }
            // the stage is free once the loads from it have landed in every lane: the
            // store needs a word of each load, and comes before the arrival.  The
            // tokens' numbers have been read by then, too.
            __syncwarp();
            if (lane == 0) mbar_arrive_after(empty + 8 * st, sink, dep);
        }
        done += steps;

        // ---- per row of this lane: R, and the sums over its tokens
        float ref[NR], row_den[NR], row_off[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float2 m = unpair(minus_ref[QM ? r : 0]), d = unpair(den[QM ? r : 0]), o = unpair(off[QM ? r : 0]);
            ref[r] = unset >> r & 1 ? kNoReference : QM ? -m.x : r ? -m.y : -m.x;
            row_den[r] = QM ? d.x + d.y : r ? d.y : d.x;
            row_off[r] = QM ? o.x + o.y : r ? o.y : o.x;
        }
        // row of acc[m][i]
        auto row_of = [](int m, int i) { return QM ? 2 * (m / (D / 8)) + i / 2 : i & 1; };

        if (turns > 1) {  // the sums of the warps that shared a head, by halves
            float4* area = reinterpret_cast<float4*>(smem + C::MERGE);
            for (int half = turns / 2; half > 0; half >>= 1) {
                float4* mine = area + ((turn & (half - 1)) * hg + hh) * 32 * (C::MERGE_WORDS / 4) + lane;
                if (turn >= half && turn < 2 * half) {
#pragma unroll
                    for (int m = 0; m < C::ACC / 4; ++m) mine[32 * m] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
                    float rest[C::MERGE_WORDS - C::ACC] = {};
#pragma unroll
                    for (int r = 0; r < NR; ++r) rest[3 * r] = ref[r], rest[3 * r + 1] = row_den[r], rest[3 * r + 2] = row_off[r];
#pragma unroll
                    for (int m = 0; m < (C::MERGE_WORDS - C::ACC) / 4; ++m)
                        mine[32 * (C::ACC / 4 + m)] = make_float4(rest[4 * m], rest[4 * m + 1], rest[4 * m + 2], rest[4 * m + 3]);
                }
                consumers_sync();
                if (turn < half) {
                    float rest[C::MERGE_WORDS - C::ACC], a[NR], b[NR];
#pragma unroll
                    for (int m = 0; m < (C::MERGE_WORDS - C::ACC) / 4; ++m) {
                        const float4 y = mine[32 * (C::ACC / 4 + m)];
                        rest[4 * m] = y.x, rest[4 * m + 1] = y.y, rest[4 * m + 2] = y.z, rest[4 * m + 3] = y.w;
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const float top = fmaxf(ref[r], rest[3 * r]);
                        a[r] = exp2_approx(ref[r] - top);
                        b[r] = exp2_approx(rest[3 * r] - top);
                        ref[r] = top;
                        row_den[r] = a[r] * row_den[r] + b[r] * rest[3 * r + 1];
                        row_off[r] = a[r] * row_off[r] + b[r] * rest[3 * r + 2];
                    }
#pragma unroll
                    for (int m = 0; m < C::ACC / 4; ++m) {
                        const float4 y = mine[32 * m];
                        const float other[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[m][i] = a[row_of(m, i)] * acc[m][i] + b[row_of(m, i)] * other[i];
                    }
                }
                consumers_sync();
            }
            if (turn > 0) continue;
        }
        // ---- the other lanes' tokens; the result
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int o = QM ? 1 : 4; o < (QM ? 4 : 32); o <<= 1) {
                row_den[r] += __shfl_xor_sync(0xffffffffu, row_den[r], o);
                row_off[r] += __shfl_xor_sync(0xffffffffu, row_off[r], o);
            }
            const int row = QM ? 8 * r + g : 2 * t + r;
            int64_t dst;
            bool valid;
            if constexpr (PAGED) {
                const int at = it.row0 + row, tok = at / p.group;
                valid = at < it.rows;
                dst = (int64_t)(it.q_token + tok) * p.heads + head * p.group + at - tok * p.group;
            } else {
                const int64_t at = (int64_t)(window - p.q_window_base) * 16 + row;
                valid = at < p.q_rows && (int64_t)window * 16 + row < p.num_nodes;
                dst = at * p.heads + head;
            }
            if (!valid) continue;
            // channel c0 + c: 16 and 32 rows, acc[c % (D / 8)][c / (D / 8)]; 8 rows, acc[c / 2][2 (c % 2)]; codes in
            // units of 2^-24 and 2^-20 in turn
            const int c0 = QM ? t * CH : g * CH;
            float v[CH];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const float a = QM ? acc[(r / 2) * (D / 8) + c % (D / 8)][2 * (r & 1) + c / (D / 8)] : acc[c / 2][2 * (c & 1) + r];
                v[c] = fmaf(a, c & 1 ? 1048576.f : 16777216.f, -row_off[r]);
            }
            if (slot >= 0) {
                float* part = p.partials + ((int64_t)slot * unit_heads + head) * ROWS * (D + 2);
                float4* po = reinterpret_cast<float4*>(part + row * D + c0);
#pragma unroll
                for (int c = 0; c < CH; c += 4) po[c / 4] = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                if (c0 == 0) *reinterpret_cast<float2*>(part + ROWS * D + 2 * row) = make_float2(ref[r], row_den[r]);
            } else {
                const float inv = row_den[r] != 0.f ? __frcp_rn(row_den[r]) : 0.f;
#pragma unroll
                for (int c = 0; c < CH; ++c) v[c] *= inv;
                store_channels<CH>(p.o, dst * D + c0, v, p.o_dtype);
            }
        }
    }
}

// The sums of split tiles and windows: per (split, head, query row) the pieces
// in order, by one warp, or by a block's four warps (each every fourth piece,
// then the four in order) where there are too few rows to fill the blocks'
// warps.  Which of the two follows from counts, so the result repeats.
template <int D, bool PAGED>
__global__ void __launch_bounds__(128) k_attend4_merge(const AttendParams p) {
    constexpr int E = D / 32;  // channels per lane
    constexpr int AHEAD = 8;   // pieces read at a time
    __shared__ float s_o[4][D], s_l[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tq = PAGED ? p.plan->tile_rows : 16, subs = PAGED ? p.kv_heads : p.heads;
    const int count = PAGED ? p.plan->num_splits : min(p.pieces->splits, p.splits_cap);
    const int live_rows = PAGED ? min(tq, max(p.group, 1)) : tq;  // of a tile of one token
    const int64_t units = (int64_t)count * subs * tq;
    const bool team = (int64_t)count * subs * live_rows <= 4ll * gridDim.x;
    const int64_t stride = (int64_t)subs * tq * (D + 2);  // from piece to piece
    const int64_t first = team ? blockIdx.x : (int64_t)blockIdx.x * 4 + warp, step = (int64_t)gridDim.x * (team ? 1 : 4);
    for (int64_t u = first; u < units; u += step) {
        const int r = (int)(u % tq);
        const int sub = (int)(u / tq % subs), split = (int)(u / tq / subs);
        int slot, parts;
        int64_t dst;  // row of O, or -1
        if constexpr (PAGED) {
            const Kv4Split* splits = reinterpret_cast<const Kv4Split*>(reinterpret_cast<const char*>(p.plan + 1) +
                                                                       (int64_t)p.plan->items_cap * sizeof(Kv4Item));
            const Kv4Split s = splits[split];
            const int row = s.row0 + r, tok = row / p.group;
            slot = s.slot;
            parts = s.parts;
            dst = row < s.rows ? ((int64_t)(s.q_token + tok) * p.heads + sub * p.group + row - tok * p.group) : -1;
        } else {
            const int4 s = p.window_splits[split];
            const int64_t row = (int64_t)(s.x - p.q_window_base) * 16 + r;
            slot = s.y;
            parts = s.z;
            dst = s.x >= 0 && row < p.q_rows && (int64_t)s.x * 16 + r < p.num_nodes ? row * p.heads + sub : -1;
        }
        if (dst < 0) continue;  // for the whole team
        const float* part = p.partials + (int64_t)slot * stride + (int64_t)sub * tq * (D + 2);
        const float2* ml = reinterpret_cast<const float2*>(part + tq * D + 2 * r);
        const float* src = part + r * D + lane * E;
        float top = kNoReference;
        for (int k = lane; k < parts; k += 32) top = fmaxf(top, ml[k * (stride / 2)].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float v[E], l = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = 0.f;
        const int k0 = team ? warp : 0, dk = team ? 4 : 1;
        for (int k = k0; k < parts; k += dk * AHEAD) {
            float2 m[AHEAD];
            float x[AHEAD][E];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int64_t at = (int64_t)min(k + a * dk, parts - 1) * stride;
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
        store_channels<E>(p.o, dst * D + lane * E, v, p.o_dtype);
    }
}

template <int D, int ROWS, bool PAGED, bool PRECISE>
static int attend_variant(const AttendParams& p, int64_t units, cudaStream_t stream) {  // units: an upper bound
    using C = AttendCfg<D, ROWS>;
    static PerContext<int> attr;
    const int rc = attr.get(nullptr, [](int* v) -> int {
        *v = 1;
        F3S_CUDA_TRY(cudaFuncSetAttribute(k_attend4<D, ROWS, PAGED, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::SMEM_SHARED));
        return F3S_SUCCESS;
    });
    if (rc != F3S_SUCCESS) return rc;
    // a block per item of a plan; by ticket, as many as run at the same time
    const int64_t grid = std::min<int64_t>(units, PAGED ? INT32_MAX : C::MIN_CTAS * num_sms_of_current_device());
    if (grid == 0) return F3S_SUCCESS;
    k_attend4<D, ROWS, PAGED, PRECISE>
        <<<(unsigned)grid, kAttendThreads, p.hg < kConsumers ? C::SMEM_SHARED : C::SMEM, stream>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

template <int ROWS, bool PAGED>
static int attend_launch(const AttendParams& p, int head_dim, int64_t units, cudaStream_t stream) {
    // fp32 results take the exact form of P; fp16 and bf16 ones round it to fp16,
    // as much as an fp16 result is rounded
    const bool precise = p.o_dtype == F3S_OUT_F32;
    if (head_dim == 64)
        return precise ? attend_variant<64, ROWS, PAGED, true>(p, units, stream)
                       : attend_variant<64, ROWS, PAGED, false>(p, units, stream);
    return precise ? attend_variant<128, ROWS, PAGED, true>(p, units, stream)
                   : attend_variant<128, ROWS, PAGED, false>(p, units, stream);
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

size_t f3s_kv4_attention_scratch_size(int32_t num_requests, int64_t num_tokens, int32_t heads, int32_t kv_heads,
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
                      int32_t kv_heads, int32_t head_dim, float scale, void* d_O, int32_t o_dtype, void* d_scratch,
                      size_t scratch_bytes, f3s_stream_t stream) {
    f3s::NvtxRange nvtx_("f3s_kv4_attention");
    if (num_requests < 0 || num_tokens < 0) return F3S_ERR_INVALID_VALUE;
    if (head_dim != 64 && head_dim != 128) return F3S_ERR_UNSUPPORTED;
    if (num_requests == 0 || num_tokens == 0) return F3S_SUCCESS;
    const int rc = f3s::check_attend(d_Q, q_dtype, q_token_stride, q_head_stride, d_pages, num_pages, heads, kv_heads,
                                     head_dim, d_O, o_dtype);
    if (rc != F3S_SUCCESS) return rc;
    if (num_tokens * (heads / kv_heads) > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
    if (!d_tables || !d_plan || (reinterpret_cast<uintptr_t>(d_plan) & 15)) return F3S_ERR_INVALID_VALUE;
    if (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15)) return F3S_ERR_INVALID_VALUE;
    const f3s::Kv4PlanLayout L = f3s::kv4_plan_layout(num_requests, num_tokens, heads, kv_heads,
                                                      f3s::num_sms_of_current_device());
    if (L.items_cap > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
    if (scratch_bytes < (size_t)L.slots_cap * kv_heads * L.tile_rows * (head_dim + 2) * 4) return F3S_ERR_WORKSPACE;
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
    p.partials = static_cast<float*>(d_scratch);
    p.tables = d_tables;
    p.table_stride = table_stride;
    cudaStream_t s = (cudaStream_t)stream;
    p.hg = kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1;
    p.kvs = p.hg;
    p.stages = f3s::kRingHeadSteps / p.kvs;
    const int64_t units = L.items_cap * (kv_heads / p.hg);
    int st;
    if (L.tile_rows == 8) st = f3s::attend_launch<8, true>(p, head_dim, units, s);
    else if (L.tile_rows == 16) st = f3s::attend_launch<16, true>(p, head_dim, units, s);
    else st = f3s::attend_launch<32, true>(p, head_dim, units, s);
    if (st != F3S_SUCCESS) return st;
    const int64_t blocks = std::min<int64_t>((int64_t)L.splits_cap * kv_heads * L.tile_rows,
                                             8ll * f3s::num_sms_of_current_device());
    if (head_dim == 64) f3s::k_attend4_merge<64, true><<<(unsigned)blocks, 128, 0, s>>>(p);
    else f3s::k_attend4_merge<128, true><<<(unsigned)blocks, 128, 0, s>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

size_t f3s_kv4_forward_scratch_size(int32_t num_items, int64_t num_blocks, int32_t heads, int32_t kv_heads,
                                    int32_t head_dim) {
    if (num_items < 0 || num_blocks < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
    if (head_dim != 64 && head_dim != 128) return 0;
    return f3s::window_piece_layout(num_items, num_blocks, heads, heads / kv_heads, head_dim,
                                    f3s::num_sms_of_current_device()).total;
}

int f3s_kv4_forward(const void* d_Q, int32_t q_dtype, const void* d_pages, int32_t num_pages, void* d_O,
                    int32_t o_dtype, const int32_t* d_window_offsets, const int32_t* d_block_cols,
                    const int32_t* d_order, int32_t num_items, int64_t num_blocks, int32_t num_nodes, int32_t heads,
                    int32_t kv_heads, int32_t head_dim, float scale, int32_t q_window_base, int32_t q_rows,
                    void* d_workspace, size_t workspace_bytes, void* d_scratch, size_t scratch_bytes,
                    f3s_stream_t stream) {
    f3s::NvtxRange nvtx_("f3s_kv4_forward");
    if (num_items < 0 || num_blocks < 0 || num_nodes < 0 || q_window_base < 0 || q_rows < 0) return F3S_ERR_INVALID_VALUE;
    if (head_dim != 64 && head_dim != 128) return F3S_ERR_UNSUPPORTED;
    if (heads <= 0) return F3S_ERR_INVALID_VALUE;
    if (!d_workspace) return F3S_ERR_INVALID_VALUE;
    if (workspace_bytes < f3s::kWsHeaderBytes) return F3S_ERR_WORKSPACE;
    if (num_items == 0 || num_nodes == 0 || q_rows == 0) return F3S_SUCCESS;
    const int rc = f3s::check_attend(d_Q, q_dtype, (int64_t)heads * head_dim, head_dim, d_pages, num_pages, heads,
                                     kv_heads, head_dim, d_O, o_dtype);
    if (rc != F3S_SUCCESS) return rc;
    if (!d_window_offsets || !d_block_cols || !d_order) return F3S_ERR_INVALID_VALUE;
    const int windows = (int)(((int64_t)num_nodes + 15) / 16);
    if (num_pages < windows) return F3S_ERR_INVALID_VALUE;
    if (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15)) return F3S_ERR_INVALID_VALUE;
    if (scratch_bytes < f3s_kv4_forward_scratch_size(num_items, num_blocks, heads, kv_heads, head_dim)) return F3S_ERR_WORKSPACE;
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
    p.cols = d_block_cols;
    p.num_nodes = num_nodes;
    p.windows = windows;
    p.q_window_base = q_window_base;
    p.q_rows = q_rows;
    p.hg = f3s::window_head_group(heads, p.group);
    p.kvs = p.hg > p.group ? p.hg / p.group : 1;
    p.stages = f3s::kRingHeadSteps / p.kvs;
    const int sms = f3s::num_sms_of_current_device();
    const f3s::WindowPieceLayout L = f3s::window_piece_layout(num_items, num_blocks, heads, p.group, head_dim, sms);
    const int64_t units = ((int64_t)num_items + L.extra_cap) * (heads / p.hg);
    if (units > INT32_MAX / 2) return F3S_ERR_TOO_LARGE;
    char* base = static_cast<char*>(d_scratch);
    f3s::WindowPieceParams w{};
    w.offsets = d_window_offsets;
    w.order = d_order;
    w.num_items = num_items;
    w.windows = windows;
    w.q_window_base = q_window_base;
    w.q_rows = q_rows;
    w.piece = windows <= L.piece ? INT32_MAX : L.piece;  // no window has more blocks than there are columns
    w.extra_cap = (int)L.extra_cap;
    w.splits_cap = (int)L.splits_cap;
    w.slots_cap = (int)L.slots_cap;
    w.pieces = reinterpret_cast<f3s::WindowPieces*>(base);
    w.items = reinterpret_cast<int4*>(base + L.items);
    w.splits = reinterpret_cast<int4*>(base + L.splits);
    w.status = p.status;
    p.pieces = w.pieces;
    p.items = w.items;
    p.window_splits = w.splits;
    p.num_items = num_items;
    p.extra_cap = w.extra_cap;
    p.splits_cap = w.splits_cap;
    p.partials = reinterpret_cast<float*>(base + L.partials);
    cudaStream_t s = (cudaStream_t)stream;
    F3S_CUDA_TRY(cudaMemsetAsync(base, 0, sizeof(f3s::WindowPieces), s));
    f3s::k_window_pieces<<<(unsigned)((num_items + 255) / 256), 256, 0, s>>>(w);
    F3S_LAUNCH_CHECK();
    const int st = f3s::attend_launch<16, false>(p, head_dim, units, s);
    if (st != F3S_SUCCESS || L.splits_cap == 0 || w.piece == INT32_MAX) return st;  // no window is split
    const int64_t blocks = std::min<int64_t>(L.splits_cap * heads * 16, 8ll * sms);
    if (head_dim == 64) f3s::k_attend4_merge<64, false><<<(unsigned)blocks, 128, 0, s>>>(p);
    else f3s::k_attend4_merge<128, false><<<(unsigned)blocks, 128, 0, s>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

}  // extern "C"
