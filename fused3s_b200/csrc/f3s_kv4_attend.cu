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

struct WindowPieces;

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
    WindowPieces* pieces;
    const int4* heavy_items;
    const int* light_items;
    const int4* window_splits;
    int heavy_cap, splits_cap;
    const int* offsets;
    const int* cols;
    int num_nodes, windows, q_window_base, q_rows;
};

// The windows of a graph as work for warps and blocks (k_window_pieces).
// A window of at most `light` blocks is one warp's, per head; a heavier one
// is cut into pieces of at most `heavy` blocks, each a block's of four warps,
// and a window of several pieces has their sums merged.
struct WindowPieces {
    int heavy_items, light_items, splits, slots;
    int heavy_ticket, light_ticket;
    int pad[58];
};
static_assert(sizeof(WindowPieces) == 256, "piece header is 256 bytes");

struct WindowPieceLayout {
    int light, heavy;
    int64_t heavy_cap, splits_cap, slots_cap;
    size_t heavy_items, light_items, splits, partials, total;
};

// A light window holds at most a quarter of a warp's even share of the work
// (and 8 blocks are one warp's in any case), a piece at most four times that.
static WindowPieceLayout window_piece_layout(int num_items, int64_t num_blocks, int heads, int head_dim, int sms) {
    WindowPieceLayout L{};
    const int64_t warps = (int64_t)sms * 16;
    const int64_t share = (num_blocks * heads + 4 * warps - 1) / (4 * warps);
    L.light = (int)std::min<int64_t>(std::max<int64_t>(share, 8), 1 << 28);
    L.heavy = 4 * L.light;
    const int64_t cut = num_blocks / L.heavy;
    L.heavy_cap = std::min<int64_t>(num_items, num_blocks / L.light) + cut;
    L.splits_cap = std::min<int64_t>(num_items, cut);
    L.slots_cap = 2 * cut;
    size_t off = sizeof(WindowPieces);
    L.heavy_items = off;
    off += (size_t)L.heavy_cap * 16;
    L.splits = off;
    off += (size_t)L.splits_cap * 16;
    L.light_items = off;
    off = align_up(off + (size_t)num_items * 4, 16);
    L.partials = off;
    off += (size_t)L.slots_cap * heads * 16 * (head_dim + 2) * 4;
    L.total = off;
    return L;
}

struct WindowPieceParams {
    const int* offsets;
    const int* order;
    int num_items, windows, q_window_base, q_rows;
    int light, heavy, heavy_cap, splits_cap, slots_cap;
    WindowPieces* pieces;
    int4* heavy_items;  // window, first block, end block, slot or -1
    int* light_items;
    int4* splits;       // window, first slot, pieces, -
    int* status;
};

// One thread per listed window.  Blocks reserve their share of the lists with
// atomics, so the lists' order varies; a window's cuts and the order in which
// its pieces are summed do not.
__global__ void __launch_bounds__(256) k_window_pieces(const WindowPieceParams p) {
    __shared__ int s_scan[256 / 32 + 1], s_base[4];
    const int i = blockIdx.x * 256 + threadIdx.x;
    int window = 0, b0 = 0, nb = 0;
    bool live = i < p.num_items;
    if (live) {
        window = p.order[i];
        live = window >= p.q_window_base && window < p.windows && (int64_t)(window - p.q_window_base) * 16 < p.q_rows;
        if (!live) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
    }
    if (live) {
        b0 = p.offsets[window];
        nb = max(p.offsets[window + 1] - b0, 0);
    }
    const bool heavy = live && nb > p.light;
    const int parts = heavy ? (int)(((int64_t)nb + p.heavy - 1) / p.heavy) : 0;
    const bool split = parts > 1;
    int total[4], at[4];
    at[0] = block_exclusive_scan<256>(parts, total[0], s_scan);
    at[1] = block_exclusive_scan<256>(live && !heavy, total[1], s_scan);
    at[2] = block_exclusive_scan<256>(split, total[2], s_scan);
    at[3] = block_exclusive_scan<256>(split ? parts : 0, total[3], s_scan);
    if (threadIdx.x < 4) {
        int* counters[4] = {&p.pieces->heavy_items, &p.pieces->light_items, &p.pieces->splits, &p.pieces->slots};
        s_base[threadIdx.x] = atomicAdd(counters[threadIdx.x], total[threadIdx.x]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) at[k] += s_base[k];
    if (live && !heavy) p.light_items[at[1]] = window;
    // more blocks than the caller said (a heavy window listed many times): one
    // warp takes what the lists have no room for
    if (heavy && (at[0] + parts > p.heavy_cap || (split && (at[2] >= p.splits_cap || at[3] + parts > p.slots_cap)))) {
        for (int k = 0; k < parts && at[0] + k < p.heavy_cap; ++k) p.heavy_items[at[0] + k] = make_int4(-1, 0, 0, -1);
        if (split && at[2] < p.splits_cap) p.splits[at[2]] = make_int4(-1, 0, 0, 0);
        p.light_items[atomicAdd(&p.pieces->light_items, 1)] = window;
        return;
    }
    for (int k = 0; k < parts; ++k) {
        const int lo = (int)((int64_t)nb * k / parts), hi = (int)((int64_t)nb * (k + 1) / parts);
        p.heavy_items[at[0] + k] = make_int4(window, b0 + lo, b0 + hi, split ? at[3] + k : -1);
    }
    if (split) p.splits[at[2]] = make_int4(window, at[3], parts, 0);
}

template <int D, int NT>
struct AttendCfg {
    static constexpr int RB = kv4_record_bytes(D);
    static constexpr int PP = NT == 4 ? 1 : 2;  // pages per step and stage
    static constexpr int STAGES = (D == 64 ? 8 : 4) / PP;
    static constexpr int STAGE_BYTES = PP * RB;
    static constexpr int RING = kAttendWarps * STAGES * STAGE_BYTES;
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

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// 2 or 4 values, as above.
template <int E>
__device__ __forceinline__ void store_few(void* o, int64_t idx, const float (&v)[E], int dtype) {
    if (dtype == F3S_OUT_F32) {
        float* dst = static_cast<float*>(o) + idx;
        if constexpr (E == 4) __stcs(reinterpret_cast<float4*>(dst), make_float4(v[0], v[1], v[2], v[3]));
        else __stcs(reinterpret_cast<float2*>(dst), make_float2(v[0], v[1]));
        return;
    }
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = dtype == F3S_OUT_F16 ? pack_half2(v[2 * i], v[2 * i + 1]) : *reinterpret_cast<const uint32_t*>(&b);
    }
    uint16_t* dst = static_cast<uint16_t*>(o) + idx;
    if constexpr (E == 4) __stcs(reinterpret_cast<uint2*>(dst), make_uint2(w[0], w[1]));
    else __stcs(reinterpret_cast<unsigned int*>(dst), w[0]);
}

// PAGED: a unit is (work item of the plan, K/V head) and the CTA's four warps
// take its pages in turn.  Otherwise persistent CTAs take units by ticket: first
// (piece, head), four warps in turn, then each warp (light window, head) by
// itself; the next ticket is drawn while a unit runs.  PRECISE adds the part of P that rounding to fp16 drops
// with a second product, which makes the result as exact as fp32 arithmetic.
template <int D, int NT, bool PAGED, bool PRECISE>
__global__ void __launch_bounds__(kAttendWarps * 32, AttendCfg<D, NT>::MIN_CTAS) k_attend4(const AttendParams p) {
    using C = AttendCfg<D, NT>;
    constexpr int RB = C::RB, STAGES = C::STAGES, PP = C::PP;
    constexpr int W = D / 32;    // words of a token's K (and of a token pair's V) per lane
    constexpr int CH = D / 8;    // output channels per lane
    constexpr int TQ = 8 * NT;   // query rows of a tile
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * STAGES * C::STAGE_BYTES;
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
    uint32_t used = 0;  // steps this warp has streamed: stage and parity of the next

    const int kv_units = PAGED ? p.kv_heads : p.heads;
    const int64_t page_bytes = (int64_t)p.kv_heads * RB;
    int wpu = kAttendWarps, wq = warp;  // warps per unit, this one among them
    int64_t units, light_units = 0;
    int ticket = 0;
    __shared__ int s_ticket;
    if constexpr (PAGED) {
        units = (int64_t)p.plan->num_items * kv_units;
    } else {
        units = (int64_t)min(p.pieces->heavy_items, p.heavy_cap) * kv_units;
        light_units = (int64_t)p.pieces->light_items * kv_units;
        if (threadIdx.x == 0) ticket = atomicAdd(&p.pieces->heavy_ticket, 1);
    }

    for (int64_t unit = blockIdx.x;; unit += gridDim.x) {
        if constexpr (PAGED) {
            if (unit >= units) break;
        } else {
            if (wpu == kAttendWarps) {
                if (threadIdx.x == 0) s_ticket = ticket;
                __syncthreads();
                unit = s_ticket;
                if (unit >= units) {  // for every warp of the CTA
                    wpu = 1;
                    wq = 0;
                    if (lane == 0) ticket = atomicAdd(&p.pieces->light_ticket, 1);
                } else if (threadIdx.x == 0) {
                    ticket = atomicAdd(&p.pieces->heavy_ticket, 1);
                }
            }
            if (wpu == 1) {
                unit = __shfl_sync(0xffffffffu, ticket, 0);
                if (unit >= light_units) break;
                if (lane == 0) ticket = atomicAdd(&p.pieces->light_ticket, 1);
            }
        }
        const int item = (int)(unit / kv_units), sub = (int)(unit - (int64_t)item * kv_units);
        const int hk = PAGED ? sub : sub / p.group;
        Kv4Item it{};
        it.slot = -1;
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
            list = p.cols;
            if (wpu == 1) {
                window = p.light_items[item];
                first = p.offsets[window];
                count = max(p.offsets[window + 1] - first, 0);
            } else {
                const int4 piece = __ldcg(p.heavy_items + item);
                window = piece.x;
                first = piece.y;
                count = piece.z - piece.y;
                it.slot = piece.w;
                if (window < 0) {  // did not fit the lists
                    __syncthreads();
                    continue;
                }
            }
        }
        // this warp's pages: PP in a row of every PP * wpu
        const int mine = dead ? 0 : count - wq * PP;
        const int steps = mine > 0 ? (mine + PP * wpu - 1) / (PP * wpu) : 0;
        const int own = steps ? (steps - 1) * PP + min(PP, mine - (steps - 1) * PP * wpu) : 0;
        const int limit_id = PAGED ? p.num_pages : p.windows;

        // ---- page ids, 32 at a time (one per lane), the next 32 ahead; `flags`
        // marks those that need a look before their scores count: no page, or
        // the graph's last block column
        const int* mine_at = list + first + wq * PP;
        auto id_at = [&](int i) { return __ldg(mine_at + (int64_t)(i / PP) * PP * wpu + i % PP); };
        auto load_ids = [&](int batch) {
            const int i = batch * 32 + lane;
            int id = -1;
            if (i < own) {
                id = id_at(i);
                if (id < 0 || id >= limit_id) {
                    if (!(PAGED && id == -1)) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
                    id = -1;
                }
            }
            return id;
        };
        auto flags_of = [&](int id) {
            return __ballot_sync(0xffffffffu, id < 0 || (!PAGED && id == p.windows - 1));
        };
        int ids = load_ids(0), ids_next = 0;
        uint32_t flags = flags_of(ids), flags_now = 0;  // of the batch last issued, of the one at work
        const uint8_t* head_pages = p.pages + (int64_t)hk * RB;
        auto issue = [&](int step) {
            const int i = step * PP;
            if ((i & 31) == 0) {
                if (i > 0) {
                    ids = ids_next;
                    flags = flags_of(ids);
                }
                if (i + 32 < own) ids_next = load_ids(i / 32 + 1);
            }
            int id[PP];
#pragma unroll
            for (int k = 0; k < PP; ++k) id[k] = __shfl_sync(0xffffffffu, ids, (i + k) & 31);
            const uint32_t n = used + step, st = n % STAGES;
            if (lane == 0) {
                const int have = min(PP, own - i);
                mbar_arrive_expect_tx(bars + 8 * st, have * RB);
#pragma unroll
                for (int k = 0; k < PP; ++k)
                    if (k < have)
                        bulk_load(ring_a + st * C::STAGE_BYTES + k * RB, head_pages + (int64_t)max(id[k], 0) * page_bytes,
                                  RB, bars + 8 * st);
            }
        };
        for (int i = 0; i < min(steps, STAGES); ++i) issue(i);

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

        for (int i = 0; i < steps; ++i) {
            const uint32_t n = used + i, st = n % STAGES, parity = (n / STAGES) & 1;
            bool ready = mbar_try_wait(bars + 8 * st, parity);
            if (!__all_sync(0xffffffffu, ready)) {
                ready = stage_wait_slow(bars + 8 * st, parity, p.status);
                if (!__all_sync(0xffffffffu, ready)) {
                    dead = true;
                    break;
                }
            }
            uint32_t dep = 0;
            float x[PP][NT][4];
            float ri[PP][2], vz[PP][2];  // 1 / r and y of tokens g, g + 8
            const uint8_t* rec0 = ring + st * C::STAGE_BYTES;
#pragma unroll
            for (int k = 0; k < PP; ++k) {
                // ---- S^T = K Q^T
                const uint8_t* rec = rec0 + k * RB;
                uint32_t kg[W], kh[W];
                lds_words<W>(rec + g * (D / 2) + t * (D / 8), kg);
                lds_words<W>(rec + (g + 8) * (D / 2) + t * (D / 8), kh);
                const uint4 sc = *reinterpret_cast<const uint4*>(rec + 16 * D + g * 16);
                dep ^= kg[0] ^ kh[0] ^ sc.x;
                float s[NT][4];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t a8 = kg[w] >> 8, b8 = kh[w] >> 8;
                    const uint32_t a0[4] = {kg[w] & kNib0, kh[w] & kNib0, kg[w] & kNib1, kh[w] & kNib1};
                    const uint32_t a1[4] = {a8 & kNib0, b8 & kNib0, a8 & kNib1, b8 & kNib1};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint32_t b[4];
                        if constexpr (C::Q_SMEM) {
                            const uint4 y = qsm[(nt * W + w) * 32 + lane];
                            b[0] = y.x;
                            b[1] = y.y;
                            b[2] = y.z;
                            b[3] = y.w;
                        } else {
#pragma unroll
                            for (int m = 0; m < 4; ++m) b[m] = qf[nt][w][m];
                        }
                        if (w == 0) mma_16816_zero(s[nt], a0, b[0], b[1]);
                        else mma_16816(s[nt], a0, b[0], b[1]);
                        mma_16816(s[nt], a1, b[2], b[3]);
                    }
                }
                // ---- scores
                const float2 ka = __half22float2(*reinterpret_cast<const __half2*>(&sc.x));
                const float2 va = __half22float2(*reinterpret_cast<const __half2*>(&sc.y));
                const float2 kb = __half22float2(*reinterpret_cast<const __half2*>(&sc.z));
                const float2 vb = __half22float2(*reinterpret_cast<const __half2*>(&sc.w));
                const float fa = ka.x * 1048576.f * unit_scale, fb = kb.x * 1048576.f * unit_scale;  // 2^20: the codes' unit
                const float ra = va.x < kKv4MinScale ? kKv4MinScale : va.x;  // keeps a NaN
                const float rb = vb.x < kKv4MinScale ? kKv4MinScale : vb.x;
                const float la = log2_approx(ra), lb = log2_approx(rb);
                ri[k][0] = rcp_approx(ra);
                ri[k][1] = rcp_approx(rb);
                vz[k][0] = va.y;
                vz[k][1] = vb.y;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float z = c < 2 ? ka.y : kb.y;
                        x[k][nt][c] = fmaf(fmaf(-z, qs[nt][c & 1], s[nt][c]), c < 2 ? fa : fb, c < 2 ? la : lb);
                    }
            }
            // ---- masks: only where a page has tokens that some row must not see
            const int tok0 = PAGED ? (it.page0 + wq * PP + i * PP * wpu) * 16 : 0;
            if ((i * PP & 31) == 0) flags_now = flags;  // no later batch has been issued yet
            if ((PAGED && tok0 + 16 * PP > open) || (flags_now >> (i * PP & 31) & (PP == 2 ? 3u : 1u))) {
                __syncwarp();
#pragma unroll
                for (int k = 0; k < PP; ++k) {
                    const int id = i * PP + k < own ? id_at(i * PP + k) : -1;
                    const bool skipped = id < 0 || id >= limit_id;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int tk = g + (c < 2 ? 0 : 8);
                            bool hide;
                            if constexpr (PAGED) {
                                // a tile's rows past its last see what the last sees
                                const int row = min(it.row0 + nt * 8 + 2 * t + (c & 1), it.rows - 1);
                                hide = tok0 + 16 * k + tk > it.context + row / p.group;
                            } else {
                                hide = id == p.windows - 1 && id * 16 + tk >= p.num_nodes;
                            }
                            if (hide || skipped) x[k][nt][c] = -INFINITY;
                        }
                    // a hidden token's scale and zero may be anything: its weight of 0
                    // must stay 0 (where it is seen, a NaN is in the weight already)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (!(fabsf(ri[k][c]) < INFINITY)) ri[k][c] = 0.f;
                        if (!(fabsf(vz[k][c]) < INFINITY)) vz[k][c] = 0.f;
                    }
                }
            }
            // ---- weights
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float most = ref[nt][j] + kRescaleAt;
#pragma unroll
                    for (int k = 0; k < PP; ++k) over = over || x[k][nt][j] > most || x[k][nt][j + 2] > most;
                }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float m = fmaxf(x[0][nt][j], x[0][nt][j + 2]);
                        if (PP == 2) m = fmaxf(m, fmaxf(x[PP - 1][nt][j], x[PP - 1][nt][j + 2]));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                        m = fmaxf(m, ref[nt][j]);
                        const float c = exp2_approx(ref[nt][j] - m);
                        ref[nt][j] = m;
                        den[nt][j] *= c;
                        off[nt][j] *= c;
#pragma unroll
                        for (int e = 0; e < D / 16; ++e) {
                            acc[nt][e][j] *= c;
                            acc[nt][e][j + 2] *= c;
                        }
                    }
            }
#pragma unroll
            for (int k = 0; k < PP; ++k) {
                uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float a[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) a[c] = exp2_approx(x[k][nt][c] - ref[nt][c & 1]);
                    const uint32_t h0 = pack_half2(a[0], a[1]), h1 = pack_half2(a[2], a[3]);
                    pb[nt][0] = movmatrix_t(h0);
                    pb[nt][1] = movmatrix_t(h1);
                    if constexpr (PRECISE) {
                        const float2 r0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                        const float2 r1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                        pl[nt][0] = movmatrix_t(pack_half2(a[0] - r0.x, a[1] - r0.y));
                        pl[nt][1] = movmatrix_t(pack_half2(a[2] - r1.x, a[3] - r1.y));
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        den[nt][c & 1] = fmaf(a[c], ri[k][c / 2], den[nt][c & 1]);
                        off[nt][c & 1] = fmaf(a[c], vz[k][c / 2], off[nt][c & 1]);
                    }
                }
                // ---- O^T += V^T P^T
                const uint8_t* rec = rec0 + k * RB;
                uint32_t v0[W], v1[W];
                lds_words<W>(rec + 8 * D + lane * (D / 8), v0);
                lds_words<W>(rec + 12 * D + lane * (D / 8), v1);
                dep ^= v0[0] ^ v1[0];
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
            }
            // refill the stage once the loads from it have landed in every lane:
            // the store needs a word of each load, and comes before the copy
            if (i + STAGES < steps) {
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(sink), "r"(dep) : "memory");
                __syncwarp();
                issue(i + STAGES);
            }
        }
        used += steps;

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
            if (it.slot >= 0) {
                float* part = p.partials + ((int64_t)it.slot * kv_units + sub) * TQ * (D + 2);
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
        store_few<E>(p.o, dst * D + lane * E, v, p.o_dtype);
    }
}

template <int D, int NT, bool PAGED, bool PRECISE>
static int attend_variant(const AttendParams& p, int64_t units, cudaStream_t stream) {  // units: an upper bound
    using C = AttendCfg<D, NT>;
    static PerContext<int> attr;
    const int rc = attr.get(nullptr, [](int* v) -> int {
        *v = 1;
        F3S_CUDA_TRY(cudaFuncSetAttribute(k_attend4<D, NT, PAGED, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::SMEM));
        return F3S_SUCCESS;
    });
    if (rc != F3S_SUCCESS) return rc;
    // a CTA per item of a plan; by ticket, as many as run at the same time
    const int64_t grid = std::min<int64_t>(units, PAGED ? INT32_MAX : C::MIN_CTAS * num_sms_of_current_device());
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
    const int64_t units = L.items_cap * kv_heads;
    int st;
    if (L.tile_rows == 8) st = f3s::attend_launch<1, true>(p, head_dim, units, s);
    else if (L.tile_rows == 16) st = f3s::attend_launch<2, true>(p, head_dim, units, s);
    else st = f3s::attend_launch<4, true>(p, head_dim, units, s);
    if (st != F3S_SUCCESS) return st;
    const int64_t blocks = std::min<int64_t>((int64_t)L.splits_cap * kv_heads * L.tile_rows,
                                             8ll * f3s::num_sms_of_current_device());
    if (head_dim == 64) f3s::k_attend4_merge<64, true><<<(unsigned)blocks, 128, 0, s>>>(p);
    else f3s::k_attend4_merge<128, true><<<(unsigned)blocks, 128, 0, s>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

size_t f3s_kv4_forward_scratch_size(int32_t num_items, int64_t num_blocks, int32_t heads, int32_t head_dim) {
    if (num_items < 0 || num_blocks < 0 || heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
    return f3s::window_piece_layout(num_items, num_blocks, heads, head_dim, f3s::num_sms_of_current_device()).total;
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
    if (scratch_bytes < f3s_kv4_forward_scratch_size(num_items, num_blocks, heads, head_dim)) return F3S_ERR_WORKSPACE;
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
    p.num_nodes = num_nodes;
    p.windows = windows;
    p.q_window_base = q_window_base;
    p.q_rows = q_rows;
    const int sms = f3s::num_sms_of_current_device();
    const f3s::WindowPieceLayout L = f3s::window_piece_layout(num_items, num_blocks, heads, head_dim, sms);
    const int64_t units = ((int64_t)num_items + L.heavy_cap) * heads;
    if (units > INT32_MAX / 2) return F3S_ERR_TOO_LARGE;
    char* base = static_cast<char*>(d_scratch);
    f3s::WindowPieceParams w{};
    w.offsets = d_window_offsets;
    w.order = d_order;
    w.num_items = num_items;
    w.windows = windows;
    w.q_window_base = q_window_base;
    w.q_rows = q_rows;
    w.light = L.light;
    w.heavy = windows <= L.heavy ? INT32_MAX : L.heavy;  // no window has more blocks than there are columns
    w.heavy_cap = (int)L.heavy_cap;
    w.splits_cap = (int)L.splits_cap;
    w.slots_cap = (int)L.slots_cap;
    w.pieces = reinterpret_cast<f3s::WindowPieces*>(base);
    w.heavy_items = reinterpret_cast<int4*>(base + L.heavy_items);
    w.light_items = reinterpret_cast<int*>(base + L.light_items);
    w.splits = reinterpret_cast<int4*>(base + L.splits);
    w.status = p.status;
    p.pieces = w.pieces;
    p.heavy_items = w.heavy_items;
    p.light_items = w.light_items;
    p.window_splits = w.splits;
    p.heavy_cap = w.heavy_cap;
    p.splits_cap = w.splits_cap;
    p.partials = reinterpret_cast<float*>(base + L.partials);
    cudaStream_t s = (cudaStream_t)stream;
    F3S_CUDA_TRY(cudaMemsetAsync(base, 0, sizeof(f3s::WindowPieces), s));
    f3s::k_window_pieces<<<(unsigned)((num_items + 255) / 256), 256, 0, s>>>(w);
    F3S_LAUNCH_CHECK();
    const int st = f3s::attend_launch<2, false>(p, head_dim, units, s);
    if (st != F3S_SUCCESS || L.splits_cap == 0 || w.heavy == INT32_MAX) return st;  // no window is split
    const int64_t blocks = std::min<int64_t>(L.splits_cap * heads * 16, 8ll * sms);
    if (head_dim == 64) f3s::k_attend4_merge<64, false><<<(unsigned)blocks, 128, 0, s>>>(p);
    else f3s::k_attend4_merge<128, false><<<(unsigned)blocks, 128, 0, s>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

}  // extern "C"
