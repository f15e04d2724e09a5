// f3s_kv4_forward.cu -- the block-sparse forward with K and V held in 4 bits: the
// 16 query rows of a window against the pages of its active blocks, columns >= N
// masked.  (f3s_kv4_math.cuh has the formulas.)
//
// Windows with many blocks are cut into pieces (k_window_pieces); persistent
// blocks take (window or piece, up to four query heads) by ticket.  A block has
// four consumer warps and one producer warp.  The producer walks the block lists
// and copies two pages per step, the records of the K/V heads in one bulk copy
// per page (they lie together), into a ring of stages; it runs ahead over the
// ends of the units.  A consumer warp has a head of its own; with fewer than four
// heads to a block, warps share a head and take its steps in turn.
//
// The codes are unpacked in registers, one AND per two values (f3s_kv4.cuh), and
// multiplied with mma.m16n8k16, Q and P as the 16-row operands: the accumulators
// of S are the operand registers of P.  What a token multiplies by (scale, zero,
// log2 r, 1 / r, y) is worked out by one lane per token, put down in shared memory
// and read as pairs; the arithmetic on scores runs on pairs of fp32 numbers.
// (tcgen05 with the queries as rows would be an eighth full; with eight pages as its 128
// rows it would need the codes unpacked into shared memory, which has not been built or
// measured here.)
//
// Accumulators are emptied every kRunPages pages (f3s_kv4_math.cuh) into sums in scratch,
// a place per consumer warp of the grid.
//
// 131,057 nodes of 8 heads, D = 64, 22 blocks per window (94 GFLOP, 516 MB from HBM, fp16
// O): 666 us; the copies alone took 219 us, and the products, half as many again for fp16
// O, need 267 us at the 530 TFLOP/s that mma.sync reaches.  40,009 nodes of 4 / 2 heads, D = 128, 80
// blocks per window (105 GFLOP, 85 % of the pages from L2, bf16 O): 454 us.  No unit is
// full: issue slots 56 and 51 % busy, mma.sync 40 and 45 %.  Each warp goes through score, vote,
// weight and product one after another, unpacks its pages and works out the tokens'
// numbers for itself, and spills (64 to 164 bytes a thread).
//
#include <algorithm>
#include "f3s_kv4_math.cuh"

namespace f3s {

constexpr int kConsumers = 4;
constexpr int kAttendThreads = (kConsumers + 1) * 32;

// The windows of a graph as work (k_window_pieces): item i is the i-th listed
// window or its first piece, the other pieces of cut windows follow behind the
// listed ones.
struct WindowPieces {
    int extra, splits, slots, ticket;
    int stop;  // F3S_ERR_TIMEOUT once a wait of this launch ran out
    int pad[59];
};
static_assert(sizeof(WindowPieces) == 256, "piece header is 256 bytes");

struct WindowParams {
    const void* q;
    int64_t q_token, q_head;  // strides in elements
    int q_bf16;
    const uint8_t* pages;
    int num_pages;
    int kv_heads, heads, group;
    int hg;        // heads per unit, one per consumer warp (times 4 / hg warps)
    int kvs;       // K/V heads per stage
    int stages;    // of the ring: RING_STEPS / kvs
    float scale;   // times log2(e)
    void* o;       // contiguous [rows, heads, D] of o_dtype
    int o_dtype;
    int* status;
    float* partials;  // (rows of a tile) x (D + 2) floats per slot and head
    WindowPieces* pieces;
    const int4* items;  // window (-1: none), first block, end block, slot or -1
    const int4* window_splits;
    int num_items, extra_cap, splits_cap;
    const int* cols;
    int num_nodes, windows, q_window_base, q_rows;
    float4* runs;  // (D / 8 + 1) x 32 per consumer warp of the grid: sums of the runs that ended, references
};

// Pieces of at most `piece` blocks: half of a thread block's even share of the
// work (3 of them per SM; a quarter costs more in sums to add, all of it leaves a
// tail: 470 + 9, 468 + 25 and 545 + 8 us for 40,009 nodes, d = 128), and 8 per warp
// that takes them in any case (2,708 nodes of one head, as measured then: 24.7 us; with 4 per
// warp 30.8, with 16 28.8).
struct WindowPieceLayout {
    int piece;
    int64_t extra_cap, splits_cap, slots_cap;
    int64_t ctas;  // most blocks of a launch
    size_t items, splits, partials, runs, total;
};

// Query heads to a block: 4, 2 or 1, as the counts divide.  With at most 1, 2 and 4 of
// 8 heads 1,164, 866 and 657 us (131,057 nodes, d = 64), of 4 / 2 heads 552, 482 and 447 (40,009
// nodes, d = 128); 2,708 nodes of 8 heads, d = 64, 58, 54 and 62.
static int window_head_group(int heads, int group) {
    for (int hg = 4; hg > 1; hg >>= 1)
        if (heads % hg == 0 && (group % hg == 0 || hg % group == 0)) return hg;
    return 1;
}

// Blocks that fit an SM; by head_dim (WindowCfg).
constexpr int window_ctas(int d) { return d == 64 ? 4 : 3; }

static WindowPieceLayout window_piece_layout(int num_items, int64_t num_blocks, int heads, int group, int head_dim, int sms) {
    WindowPieceLayout L{};
    const int hg = window_head_group(heads, group);
    const int64_t blocks = 2 * 3ll * sms;
    const int64_t share = (num_blocks * (heads / hg) + blocks - 1) / blocks;
    L.piece = (int)std::min<int64_t>(std::max<int64_t>(share, 8 * (4 / hg)), 1 << 28);
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
    L.ctas = std::min<int64_t>((num_items + L.extra_cap) * (heads / hg), (int64_t)window_ctas(head_dim) * sms);
    L.runs = off;
    off += (size_t)L.ctas * kConsumers * (head_dim / 8 + 1) * 32 * 16;
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
    launch_dependents();
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

template <int D>
struct WindowCfg {
    static constexpr int RB = kv4_record_bytes(D);
    static constexpr int PP = 2;                // pages per step
    static constexpr int ACC = D / 8 * 4;       // accumulators per lane
    static constexpr int RING_STEPS = D == 64 ? 16 : 8;  // stages times K/V heads per stage
    static constexpr int RING = RING_STEPS * PP * RB;
    static constexpr int TOKENS = RING;         // per warp: what the tokens of a step multiply by
    static constexpr int TOKEN_BYTES = 5 * 16 * 4 * PP;
    static constexpr int Q = TOKENS + kConsumers * TOKEN_BYTES;
    static constexpr int Q_BYTES = 16 * D * 2;  // per warp
    static constexpr int BARS = Q + kConsumers * Q_BYTES;
    static constexpr int NBARS = 2 * RING_STEPS + 4;
    static constexpr int UNITS = BARS + NBARS * 8;      // two unit records
    static constexpr int FLAGS = UNITS + 2 * 32;        // per stage
    static constexpr int SINK = FLAGS + RING_STEPS * 4;
    static constexpr int MERGE = (SINK + kConsumers * 4 + 127) / 128 * 128;  // two warps' sums, where warps share a head
    static constexpr int MERGE_WORDS = ACC + 8;         // per lane
    static constexpr int SMEM = MERGE;
    static constexpr int SMEM_SHARED = MERGE + 2 * 32 * MERGE_WORDS * 4;
    static constexpr int MIN_CTAS = window_ctas(D);
};

struct Unit {  // as the producer hands it to the consumers
    int live, window, slot, steps, head0;
    int pad[3];
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }
// True if x is, in every consumer.
__device__ __forceinline__ bool consumers_all(bool x) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\tbar.red.and.pred b, 1, %2, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)x), "n"(kConsumers * 32)
        : "memory");
    return all != 0;
}

// The producer warp: units, their block lists, the copies.
template <int D>
__device__ __forceinline__ void window_produce(const WindowParams& p, uint32_t ring, uint32_t full, uint32_t empty,
                                               uint32_t unit_full, uint32_t unit_empty, Unit* unit_out, int* flags_out,
                                               int units, int groups) {
    constexpr int RB = kv4_record_bytes(D), PP = WindowCfg<D>::PP;
    const int lane = threadIdx.x & 31;
    const int stages = p.stages, stage_bytes = PP * p.kvs * RB, copy_bytes = p.kvs * RB;
    const int64_t page_bytes = (int64_t)p.kv_heads * RB;
    const int extra = min(p.pieces->extra, p.extra_cap);
    int* stop = &p.pieces->stop;
    uint32_t n = 0;  // steps issued
    auto end = [&] { ring_drain(full, stages, n > (uint32_t)stages ? n - stages : 0, n); };
    int ticket = 0;
    if (lane == 0) ticket = atomicAdd(&p.pieces->ticket, 1);
    for (int k = 0;; ++k) {
        const int unit = __shfl_sync(0xffffffffu, ticket, 0);
        const bool live = unit < units;
        int4 piece = make_int4(-1, 0, 0, -1);
        int head0 = 0;
        if (live) {
            if (lane == 0) ticket = atomicAdd(&p.pieces->ticket, 1);
            const int item = unit / groups;
            piece = __ldcg(p.items + (item < extra ? p.num_items + item : item - extra));
            head0 = (unit - item * groups) * p.hg;
        }
        const int count = piece.x >= 0 ? piece.z - piece.y : 0;
        const int* list = p.cols + piece.y;
        if (!phase_wait(unit_empty + 8 * (k & 1), (k >> 1 & 1) ^ 1, p.status, stop)) return end();
        if (lane == 0) {
            unit_out[k & 1] = Unit{live, piece.x, piece.w, (count + PP - 1) / PP, head0};
            mbar_arrive(unit_full + 8 * (k & 1));
        }
        if (!live) return end();
        if (piece.x >= 0) {  // the unit's Q rows, a line or more each, on their way to L2
            const int64_t row = (int64_t)(piece.x - p.q_window_base) * 16 + (lane & 15);
            if (row < p.q_rows) {
                const char* at = static_cast<const char*>(p.q) + 2 * (row * p.q_token + (int64_t)head0 * p.q_head);
                for (int off = (lane >> 4) * 128; off < p.hg * D * 2; off += 256)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(at + off));
            }
        }
        const uint8_t* src = p.pages + (int64_t)(head0 / p.group) * RB;
        auto load_ids = [&](int i0) {
            int id = -1;
            if (i0 + lane < count) {
                id = list[i0 + lane];
                if (id < 0 || id >= p.windows) {
                    atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
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
            const uint32_t tail = __ballot_sync(0xffffffffu, have && id == p.windows - 1);
            const uint32_t st = n & (stages - 1);
            if (!phase_wait(empty + 8 * st, (n / stages & 1) ^ 1, p.status, stop)) return end();
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

// The largest of two 16-bit numbers each, whichever of Q's types they are of.
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b, int bf16) {
    uint32_t d;
    if (bf16) asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// PRECISE adds the part of P that rounding to fp16 drops with a second product,
// which makes the result as exact as fp32 arithmetic.
template <int D, bool PRECISE>
__global__ void __launch_bounds__(kAttendThreads, WindowCfg<D>::MIN_CTAS) k_window_attend4(const WindowParams p) {
    using C = WindowCfg<D>;
    constexpr int RB = C::RB, PP = C::PP;
    constexpr int W = D / 32;    // words of a token's K (and of a token pair's V) per lane
    constexpr int N = D / 8;     // products' column blocks: output channels t * D / 4 + c and + D / 8 + c, c < N
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t base = smem_addr(smem), full = base + C::BARS, empty = full + 8 * C::RING_STEPS;
    const uint32_t unit_full = empty + 8 * C::RING_STEPS, unit_empty = unit_full + 16;
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
    launch_dependents();
    wait_for_primary();  // the pieces
    if (warp == kConsumers) {
        const int groups = p.heads / hg;
        window_produce<D>(p, base, full, empty, unit_full, unit_empty, unit_records, stage_flags,
                          (p.num_items + min(p.pieces->extra, p.extra_cap)) * groups, groups);
        return;
    }

    const int hh = warp % hg, turn = warp / hg;
    const uint32_t sink = base + C::SINK + warp * 4;
    float* tokens = reinterpret_cast<float*>(smem + C::TOKENS + warp * C::TOKEN_BYTES);
    uint4* qsm = reinterpret_cast<uint4*>(smem + C::Q + warp * C::Q_BYTES);
    const int page_stride = p.kvs * RB, stage_bytes = PP * page_stride;
    int* stop = &p.pieces->stop;
    bool dead = false;  // a wait ran out: nothing more is read
    uint32_t done = 0;  // steps of the units before this one

    for (int k = 0;; ++k) {
        bool ready = phase_wait(unit_full + 8 * (k & 1), k >> 1 & 1, p.status, stop);
        if (turns > 1) ready = consumers_all(ready);  // warps that meet at barriers leave together
        if (!ready) break;
        const Unit u = unit_records[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(unit_empty + 8 * (k & 1));
        if (!u.live) break;
        if (u.window < 0) continue;  // no steps either
        const int head = u.head0 + hh;
        const int kv_off = (head / p.group - u.head0 / p.group) * RB;  // in a page of a stage
        const int64_t row0 = (int64_t)(u.window - p.q_window_base) * 16 + g;  // lane (g, t): rows g and g + 8

        // ---- Q as fp16 times a power of two that brings the row's largest to
        // [2^9, 2^10); channels whose codes come in units of 2^-24 another 2^4.
        // Lane (g, t): channels t * D / 4 ... of its rows
        uint64_t qs[2], qu[2];  // per row, twice: the sum of q, scaled; what a score's unit stands for
        {
            uint4 raw[2][W];
            uint32_t top[2] = {0, 0};
            uint64_t by[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t row = row0 + 8 * r;
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + row * p.q_token +
                                                                  (int64_t)head * p.q_head + t * (D / 4));
#pragma unroll
                for (int w = 0; w < W; ++w) raw[r][w] = row < p.q_rows ? src[w] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t x[4] = {raw[r][w].x, raw[r][w].y, raw[r][w].z, raw[r][w].w};
#pragma unroll
                    for (int n = 0; n < 4; ++n) top[r] = max_pair(top[r], x[n] & 0x7fff7fffu, p.q_bf16);
                }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = max_pair(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1), p.q_bf16);
                top[r] = max_pair(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2), p.q_bf16);
                const float2 two = q_floats(top[r], p.q_bf16);
                float amax = fmaxf(two.x, two.y);
                if (__any_sync(0xffffffffu, !(amax < INFINITY))) {  // an infinity: the largest of the others; it stays what it is
                    amax = 0.f;
                    const int64_t row = row0 + 8 * r;
                    const uint32_t* at = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + row * p.q_token +
                                                                           (int64_t)head * p.q_head + t * (D / 4));
#pragma unroll 1
                    for (int i = 0; i < W * 4; ++i) {
                        const float2 y = q_floats(row < p.q_rows ? at[i] : 0, p.q_bf16);
                        if (fabsf(y.x) < INFINITY) amax = fmaxf(amax, fabsf(y.x));
                        if (fabsf(y.y) < INFINITY) amax = fmaxf(amax, fabsf(y.y));
                    }
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                }
                // 2^(9 - floor(log2 amax)), kept within fp32's normal range
                const int e = amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 : 9;
                const int up = min(max(9 - e, -120), 120);
                const float f = __uint_as_float((uint32_t)(up + 127) << 23);
                const float unit = p.scale * __uint_as_float((uint32_t)(127 - up) << 23);
                qu[r] = pair(unit, unit);
                by[r][0] = pair(f * 16.f, f * 16.f);
                by[r][1] = pair(f, f);
            }
            float sum[4];  // the rows' sums, as a product with 1 (and 2^-4)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                uint32_t h[8];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t x[4] = {raw[r][w].x, raw[r][w].y, raw[r][w].z, raw[r][w].w};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float2 y = q_floats(x[n], p.q_bf16), z = unpair(mul2(pair(y.x, y.y), by[r][n & 1]));
                        h[4 * r + n] = pack_half2(z.x, z.y);
                    }
                }
                const uint32_t a0[4] = {h[0], h[4], h[1], h[5]}, a1[4] = {h[2], h[6], h[3], h[7]};
                if (w == 0) mma_16816_zero(sum, a0, 0x2c002c00u, 0x3c003c00u);
                else mma_16816(sum, a0, 0x2c002c00u, 0x3c003c00u);
                mma_16816(sum, a1, 0x2c002c00u, 0x3c003c00u);
                // each lane reads back what it wrote itself
                qsm[2 * w * 32 + lane] = make_uint4(h[0], h[4], h[1], h[5]);
                qsm[(2 * w + 1) * 32 + lane] = make_uint4(h[2], h[6], h[3], h[7]);
            }
            qs[0] = pair(sum[0], sum[0]);
            qs[1] = pair(sum[2], sum[2]);
        }

        float acc[N][4];
        uint64_t minus_ref[2], den[2], off[2];  // -R twice; sum a / r, sum a y over this lane's even and odd tokens
#pragma unroll
        for (int m = 0; m < N; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) minus_ref[r] = den[r] = off[r] = 0;
        uint32_t unset = 3;  // rows that have no reference yet (a bit each)
        // The sums of the runs of steps that ended, in the references as they stand; `first`: none has yet
        auto add_runs = [&](bool first, bool keep) {
            float4* runs = p.runs + ((int64_t)blockIdx.x * kConsumers + warp) * ((N + 1) * 32) + lane;
            const float now[2] = {unpair(minus_ref[0]).x, unpair(minus_ref[1]).x};
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!first) y = runs[32 * N];
            // references only rise; a row that had none has nothing to scale
            const float by[2] = {exp2_approx(fminf(now[0] - y.x, 0.f)), exp2_approx(fminf(now[1] - y.y, 0.f))};
            if (keep) runs[32 * N] = make_float4(now[0], now[1], 0.f, 0.f);
#pragma unroll
            for (int m = 0; m < N; ++m) {
                y = make_float4(0.f, 0.f, 0.f, 0.f);
                if (!first) y = runs[32 * m];
                acc[m][0] = fmaf(y.x, by[0], acc[m][0]);
                acc[m][1] = fmaf(y.y, by[0], acc[m][1]);
                acc[m][2] = fmaf(y.z, by[1], acc[m][2]);
                acc[m][3] = fmaf(y.w, by[1], acc[m][3]);
                if (keep) {
                    runs[32 * m] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
                    acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
                }
            }
        };
        constexpr int RUN = kRunPages / PP;  // steps of a warp in a row

        for (int j = turn; j < u.steps && !dead; j += turns) {
            const int mine = j >> (turns >> 1);  // steps of this warp so far
            if (mine > 0 && mine % RUN == 0) add_runs(mine == RUN, true);
            const uint32_t n = done + j, st = n & (p.stages - 1);
            if (!phase_wait(full + 8 * st, n / p.stages & 1, p.status, stop)) {
                dead = true;
                break;
            }
            const uint8_t* rec0 = smem + st * stage_bytes + kv_off;
            const int flags = stage_flags[st];
            uint32_t dep;
            // ---- what each token multiplies by, one lane per token: s (in the codes' unit),
            // -z s, log2 r, 1 / r, y as [page][f, z, l, ri, y][t][token 2t, 2t + 1, 2t + 8, 2t + 9]
            {
                const int tk = lane & 15;
                const uint2 sc = *reinterpret_cast<const uint2*>(rec0 + (lane >> 4) * page_stride + kv4_scale_off(D, tk));
                dep = sc.x;
                const float2 ks = half2_floats(sc.x), vs = half2_floats(sc.y);
                const float r = vs.x < kKv4MinScale ? kKv4MinScale : vs.x;  // keeps a NaN
                float* dst = tokens + (lane >> 4) * 80 + ((tk & 7) >> 1) * 4 + (tk >> 3) * 2 + (tk & 1);
                dst[0] = ks.x * 1048576.f;  // 2^20
                dst[16] = -ks.y * ks.x;
                dst[32] = log2_approx(r);
                dst[48] = rcp_approx(r);
                dst[64] = vs.y;
            }
            __syncwarp();
            // scores less the reference: row r, tokens (2t, 2t + 1) and (2t + 8, 2t + 9)
            uint64_t x[PP][2][2];
#pragma unroll
            for (int k2 = 0; k2 < PP; ++k2) {
                const uint8_t* rec = rec0 + k2 * page_stride;
                uint32_t kg[W], kh[W];
                lds_words<W>(rec + g * (D / 2) + t * (D / 8), kg);
                lds_words<W>(rec + (g + 8) * (D / 2) + t * (D / 8), kh);
                dep ^= kg[0] ^ kh[0];
                float s[2][4];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t g8 = kg[w] >> 8, h8 = kh[w] >> 8;
                    const uint4 a = qsm[2 * w * 32 + lane], b = qsm[(2 * w + 1) * 32 + lane];
                    const uint32_t a0[4] = {a.x, a.y, a.z, a.w}, a1[4] = {b.x, b.y, b.z, b.w};
                    if (w == 0) {
                        mma_16816_zero(s[0], a0, kg[w] & kNib0, kg[w] & kNib1);
                        mma_16816_zero(s[1], a0, kh[w] & kNib0, kh[w] & kNib1);
                    } else {
                        mma_16816(s[0], a0, kg[w] & kNib0, kg[w] & kNib1);
                        mma_16816(s[1], a0, kh[w] & kNib0, kh[w] & kNib1);
                    }
                    mma_16816(s[0], a1, g8 & kNib0, g8 & kNib1);
                    mma_16816(s[1], a1, h8 & kNib0, h8 & kNib1);
                }
                const float* tok = tokens + k2 * 80 + 4 * t;
                const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(tok);
                const ulonglong2 z = *reinterpret_cast<const ulonglong2*>(tok + 16);
                const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(tok + 32);
#pragma unroll
                for (int r = 0; r < 2; ++r) {  // a score is rounded before the reference is taken off: large ones stay in order
                    x[k2][r][0] = fma2(fma2(pair(s[0][2 * r], s[0][2 * r + 1]), f.x, mul2(z.x, qs[r])), qu[r], l.x);
                    x[k2][r][1] = fma2(fma2(pair(s[1][2 * r], s[1][2 * r + 1]), f.y, mul2(z.y, qs[r])), qu[r], l.y);
                    x[k2][r][0] = add2(x[k2][r][0], minus_ref[r]);
                    x[k2][r][1] = add2(x[k2][r][1], minus_ref[r]);
                }
            }
            // ---- masks: a missing page, or the columns past N of the last one
            if (flags) {
                __syncwarp();
#pragma unroll
                for (int k2 = 0; k2 < PP; ++k2) {
                    const bool skipped = flags >> k2 & 1, last = flags >> (8 + k2) & 1;
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int node = (p.windows - 1) * 16 + 2 * t + 8 * c;
                            float2 y = unpair(x[k2][r][c]);
                            if (skipped || (last && node >= p.num_nodes)) y.x = -INFINITY;
                            if (skipped || (last && node + 1 >= p.num_nodes)) y.y = -INFINITY;
                            x[k2][r][c] = pair(y.x, y.y);
                        }
                }
                // a hidden token's scale and zero may be anything: its weight of 0
                // must stay 0 (where it is seen, a NaN is in the weight already)
                float* own = tokens + (lane >> 4) * 80 + (lane & 15);
                if (!(fabsf(own[48]) < INFINITY)) own[48] = 0.f;
                if (!(fabsf(own[64]) < INFINITY)) own[64] = 0.f;
                __syncwarp();
            }
            // ---- weights
            bool over = unset != 0;
#pragma unroll
            for (int k2 = 0; k2 < PP; ++k2)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float2 y = unpair(x[k2][r][c]);
                        over = over || y.x > kRescaleAt || y.y > kRescaleAt;
                    }
            if (__any_sync(0xffffffffu, over)) {
                float down[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float m = -INFINITY;
#pragma unroll
                    for (int k2 = 0; k2 < PP; ++k2)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float2 y = unpair(x[k2][r][c]);
                            m = fmaxf(m, fmaxf(y.x, y.y));
                        }
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    float up;  // the reference moves up by this
                    if (unset >> r & 1) {  // nothing seen so far: the sums are 0, whatever they are scaled by
                        up = m > -INFINITY ? m - kTopWeight : 0.f;
                        down[r] = 1.f;
                        if (m > -INFINITY) unset &= ~(1u << r);
                    } else {
                        up = fmaxf(m - kTopWeight, 0.f);
                        down[r] = exp2_approx(-up);
                    }
                    const uint64_t minus = pair(-up, -up), by = pair(down[r], down[r]);
                    minus_ref[r] = add2(minus_ref[r], minus);
                    den[r] = mul2(den[r], by);
                    off[r] = mul2(off[r], by);
#pragma unroll
                    for (int k2 = 0; k2 < PP; ++k2)
#pragma unroll
                        for (int c = 0; c < 2; ++c) x[k2][r][c] = add2(x[k2][r][c], minus);
                }
#pragma unroll
                for (int e = 0; e < N; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[e][i] *= down[i / 2];
            }
#pragma unroll
            for (int k2 = 0; k2 < PP; ++k2) {
                uint32_t pa[4], pl[4];  // P as an operand, and what its rounding drops
                const float* tok = tokens + k2 * 80 + 4 * t;
                const ulonglong2 ri = *reinterpret_cast<const ulonglong2*>(tok + 48);
                const ulonglong2 vz = *reinterpret_cast<const ulonglong2*>(tok + 64);
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float2 y = unpair(x[k2][r][c]);
                        const float2 a = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                        uint64_t a2 = pair(a.x, a.y);
                        pa[2 * c + r] = pack_half2(a.x, a.y);
                        const float2 b = half2_floats(pa[2 * c + r]);
                        if constexpr (PRECISE) {
                            const float2 d = unpair(fma2(pair(b.x, b.y), pair(-1.f, -1.f), a2));
                            pl[2 * c + r] = pack_half2(d.x, d.y);
                        } else {  // the same weights in every sum
                            a2 = pair(b.x, b.y);
                        }
                        den[r] = fma2(a2, c ? ri.y : ri.x, den[r]);
                        off[r] = fma2(a2, c ? vz.y : vz.x, off[r]);
                    }
                // ---- O += P V
                const uint8_t* rec = rec0 + k2 * page_stride;
                uint32_t v0[W], v1[W];
                lds_words<W>(rec + 8 * D + lane * (D / 8), v0);
                lds_words<W>(rec + 12 * D + lane * (D / 8), v1);
                dep ^= v0[0] ^ v1[0];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t a8 = v0[w] >> 8, b8 = v1[w] >> 8;
                    const uint32_t an[4] = {v0[w] & kNib0, v0[w] & kNib1, a8 & kNib0, a8 & kNib1};
                    const uint32_t bn[4] = {v1[w] & kNib0, v1[w] & kNib1, b8 & kNib0, b8 & kNib1};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mma_16816(acc[4 * w + i], pa, an[i], bn[i]);
                        if constexpr (PRECISE) mma_16816(acc[4 * w + i], pl, an[i], bn[i]);
                    }
                }
            }
            // the stage is free once the loads from it have landed in every lane: the
            // store needs a word of each load, and comes before the arrival.  The
            // tokens' numbers have been read by then, too.
            __syncwarp();
            if (lane == 0) mbar_arrive_after(empty + 8 * st, sink, dep);
        }
        done += u.steps;
        if (u.steps - turn > RUN * turns) add_runs(false, false);

        // ---- per row of this lane: R, and the sums over its tokens
        float ref[2], row_den[2], row_off[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float2 d = unpair(den[r]), o = unpair(off[r]);
            ref[r] = unset >> r & 1 ? kNoReference : -unpair(minus_ref[r]).x;
            row_den[r] = d.x + d.y;
            row_off[r] = o.x + o.y;
        }
        if (turns > 1) {  // the sums of the warps that shared a head, by halves
            float4* area = reinterpret_cast<float4*>(smem + C::MERGE);
            for (int half = turns / 2; half > 0; half >>= 1) {
                float4* mine = area + ((turn & (half - 1)) * hg + hh) * 32 * (C::MERGE_WORDS / 4) + lane;
                if (turn >= half && turn < 2 * half) {
#pragma unroll
                    for (int m = 0; m < N; ++m) mine[32 * m] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
                    mine[32 * N] = make_float4(ref[0], row_den[0], row_off[0], 0.f);
                    mine[32 * (N + 1)] = make_float4(ref[1], row_den[1], row_off[1], 0.f);
                }
                consumers_sync();
                if (turn < half) {
                    float a[2], b[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float4 y = mine[32 * (N + r)];
                        const float top = fmaxf(ref[r], y.x);
                        a[r] = exp2_approx(ref[r] - top);
                        b[r] = exp2_approx(y.x - top);
                        ref[r] = top;
                        row_den[r] = a[r] * row_den[r] + b[r] * y.y;
                        row_off[r] = a[r] * row_off[r] + b[r] * y.z;
                    }
#pragma unroll
                    for (int m = 0; m < N; ++m) {
                        const float4 y = mine[32 * m];
                        acc[m][0] = a[0] * acc[m][0] + b[0] * y.x;
                        acc[m][1] = a[0] * acc[m][1] + b[0] * y.y;
                        acc[m][2] = a[1] * acc[m][2] + b[1] * y.z;
                        acc[m][3] = a[1] * acc[m][3] + b[1] * y.w;
                    }
                }
                consumers_sync();
            }
            if (turn > 0) continue;
        }
        // ---- the other lanes' tokens; the result
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                row_den[r] += __shfl_xor_sync(0xffffffffu, row_den[r], o);
                row_off[r] += __shfl_xor_sync(0xffffffffu, row_off[r], o);
            }
            const int64_t row = row0 + 8 * r;
            if (row >= p.q_rows || (int64_t)u.window * 16 + g + 8 * r >= p.num_nodes) continue;
            const float inv = u.slot >= 0 ? 1.f : row_den[r] != 0.f ? __frcp_rn(row_den[r]) : 0.f;
            const float even = 16777216.f * inv, odd = 1048576.f * inv, less = -row_off[r] * inv;  // codes' units in turn
            float v[2 * N];
#pragma unroll
            for (int c = 0; c < N; ++c) {
                v[c] = fmaf(acc[c][2 * r], c & 1 ? odd : even, less);
                v[N + c] = fmaf(acc[c][2 * r + 1], c & 1 ? odd : even, less);
            }
            if (u.slot >= 0) {
                float* part = p.partials + ((int64_t)u.slot * p.heads + head) * 16 * (D + 2);
                float4* po = reinterpret_cast<float4*>(part + (g + 8 * r) * D + t * (D / 4));
#pragma unroll
                for (int c = 0; c < 2 * N; c += 4) po[c / 4] = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                if (t == 0) *reinterpret_cast<float2*>(part + 16 * D + 2 * (g + 8 * r)) = make_float2(ref[r], row_den[r]);
            } else {
                store_channels<2 * N>(p.o, (row * p.heads + head) * D + t * (D / 4), v, p.o_dtype);
            }
        }
    }
}

// The sums of cut windows: see merge_rows.
template <int D>
__global__ void __launch_bounds__(128) k_window_merge(const WindowParams p) {
    wait_for_primary();  // the sums
    merge_rows<D>(min(p.pieces->splits, p.splits_cap), p.heads, 16, 16, p.partials, p.o, p.o_dtype,
                  [&](int split, int head, int r, int& slot, int& parts) -> int64_t {
                      const int4 s = p.window_splits[split];
                      const int64_t row = (int64_t)(s.x - p.q_window_base) * 16 + r;
                      slot = s.y;
                      parts = s.z;
                      return s.x >= 0 && row < p.q_rows && (int64_t)s.x * 16 + r < p.num_nodes ? row * p.heads + head : -1;
                  });
}

template <int D, bool PRECISE>
static int window_launch(const WindowParams& p, int64_t units, cudaStream_t stream) {  // units: an upper bound
    using C = WindowCfg<D>;
    static PerContext<int> attr;
    const int rc = attr.get(nullptr, [](int* v) -> int {
        *v = 1;
        F3S_CUDA_TRY(cudaFuncSetAttribute(k_window_attend4<D, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::SMEM_SHARED));
        return F3S_SUCCESS;
    });
    if (rc != F3S_SUCCESS) return rc;
    // f3s_set_forward_sm_limit counts blocks: a few of them, spread over the SMs, leave room on each
    const int sms = num_sms_of_current_device(), limit = forward_grid_limit();  // at most the layout's ctas
    const int64_t grid = std::min<int64_t>(units, limit < sms ? limit : C::MIN_CTAS * sms);
    return launch_after(k_window_attend4<D, PRECISE>, (unsigned)grid, kAttendThreads,
                        p.hg < kConsumers ? C::SMEM_SHARED : C::SMEM, stream, p);
}

}  // namespace f3s

extern "C" {

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
    const int rc = f3s::check_attend_args(d_Q, q_dtype, (int64_t)heads * head_dim, head_dim, d_pages, num_pages, heads,
                                     kv_heads, head_dim, d_O, o_dtype);
    if (rc != F3S_SUCCESS) return rc;
    if (!d_window_offsets || !d_block_cols || !d_order) return F3S_ERR_INVALID_VALUE;
    const int windows = (int)(((int64_t)num_nodes + 15) / 16);
    if (num_pages < windows) return F3S_ERR_INVALID_VALUE;
    if (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15)) return F3S_ERR_INVALID_VALUE;
    if (scratch_bytes < f3s_kv4_forward_scratch_size(num_items, num_blocks, heads, kv_heads, head_dim)) return F3S_ERR_WORKSPACE;
    f3s::WindowParams p{};
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
    p.stages = (head_dim == 64 ? f3s::WindowCfg<64>::RING_STEPS : f3s::WindowCfg<128>::RING_STEPS) / p.kvs;
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
    p.runs = reinterpret_cast<float4*>(base + L.runs);
    cudaStream_t s = (cudaStream_t)stream;
    F3S_CUDA_TRY(cudaMemsetAsync(base, 0, sizeof(f3s::WindowPieces), s));
    f3s::k_window_pieces<<<(unsigned)((num_items + 255) / 256), 256, 0, s>>>(w);
    F3S_LAUNCH_CHECK();
    const bool precise = f3s::weights_in_full(o_dtype);
    const int st = head_dim == 64 ? (precise ? f3s::window_launch<64, true>(p, units, s) : f3s::window_launch<64, false>(p, units, s))
                                  : (precise ? f3s::window_launch<128, true>(p, units, s) : f3s::window_launch<128, false>(p, units, s));
    if (st != F3S_SUCCESS || L.splits_cap == 0 || w.piece == INT32_MAX) return st;  // no window is split
    const int64_t blocks = std::min<int64_t>(L.splits_cap * heads * 16, 8ll * sms);
    return f3s::launch_after(head_dim == 64 ? f3s::k_window_merge<64> : f3s::k_window_merge<128>, (unsigned)blocks, 128, 0, s, p);
}

}  // extern "C"
