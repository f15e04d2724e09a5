// f3s_kv4_attend.cu -- causal attention over a request's pages, K and V held in
// 4 bits: one to many new tokens per request, grouped heads, block tables.
// (f3s_kv4_math.cuh has the formulas.)
//
// A block of four warps takes one work item of the plan (a piece of the pages
// of a tile of query rows) for one K/V head.  Each warp streams its share of
// the pages, two in a row, through a ring of its own in shared memory: one bulk
// copy of 16 D + 128 bytes per page, issued by a lane as soon as the stage has been
// read, so no warp waits for another before the sums are added at the end.
//
// S^T = K Q^T and O^T = V^T P^T run on mma.m16n8k16 with the cache as the 16-row
// operand (unpacked in registers, one AND per two values, f3s_kv4.cuh) and 8 NT
// query rows as columns; P goes from accumulator to operand layout through
// movmatrix.  (With eight pages as the 128 rows of a tcgen05 product the queries would
// fill its columns just as well, but the codes would have to be unpacked into shared
// memory first; that form has not been built or measured for so few query rows.)
//
// Accumulators are emptied every kRunPages pages (f3s_kv4_math.cuh) into sums that lie
// in shared memory beside the ring.
//
// Bound: HBM and instruction issue together.  64 requests of up to 8,191 tokens, one
// new token each, 32 / 8 heads, D = 128, bf16: 351 MB in 79 us, 4.4 TB/s (issue slots
// 57 % busy, most of it unpacking and weights; the copies alone took 59 us).
//
#include <algorithm>
#include "f3s_kv4_attend.cuh"

namespace f3s {

constexpr int kAttendWarps = 4;

template <int D, int NT>
struct AttendCfg {
    static constexpr int RB = kv4_record_bytes(D);
    static constexpr int PP = 2;  // pages per step and stage
    static constexpr int STAGES = (D == 64 ? 8 : 4) / PP;
    static constexpr int STAGE_BYTES = PP * RB;
    static constexpr int RING = kAttendWarps * STAGES * STAGE_BYTES;
    static constexpr int OPITCH = D + 4;
    static constexpr int MERGE = kAttendWarps * 8 * NT * (OPITCH + 2) * 4;
    static constexpr int DATA = RING > MERGE ? RING : (MERGE + 127) / 128 * 128;
    static constexpr int BARS = DATA;
    static constexpr int SINK = BARS + kAttendWarps * STAGES * 8;  // one word per warp, written, never read
    // sums of the runs that ended, [nt][D / 16][lane] x 4, and their references, [nt][lane] x 2, per warp
    static constexpr int RUNS = (SINK + kAttendWarps * 4 + 15) / 16 * 16;
    static constexpr int RUN_BYTES = NT * (D / 16) * 32 * 16 + NT * 32 * 8;
    static constexpr int SMEM = RUNS + kAttendWarps * RUN_BYTES;
    static constexpr int MIN_CTAS = NT == 2 && D == 128 ? 3 : 4;
};

// PRECISE adds the part of P that rounding to fp16 drops with a second product,
// which makes the result as exact as fp32 arithmetic.
template <int D, int NT, bool PRECISE>
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
    launch_dependents();
    wait_for_primary();  // the plan
    const int item = blockIdx.x / p.kv_heads, hk = blockIdx.x - item * p.kv_heads;
    if (item >= plan_items(p)) return;
    Kv4Item it;
    {
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
    const int count = max(it.page1 - it.page0, 0);
    const int64_t page_bytes = (int64_t)p.kv_heads * RB;
    // this warp's pages: PP in a row of every PP * kAttendWarps
    const int mine = count - warp * PP;
    const int steps = mine > 0 ? (mine + PP * kAttendWarps - 1) / (PP * kAttendWarps) : 0;
    const int own = steps ? (steps - 1) * PP + min(PP, mine - (steps - 1) * PP * kAttendWarps) : 0;

    // ---- page ids, 32 at a time (one per lane), the next 32 ahead; `flags`
    // marks entries without a page
    const int* mine_at = p.tables + (int64_t)it.request * p.table_stride + it.page0 + warp * PP;
    auto id_at = [&](int i) { return mine_at[(int64_t)(i / PP) * PP * kAttendWarps + i % PP]; };
    auto load_ids = [&](int batch) {
        const int i = batch * 32 + lane;
        int id = -1;
        if (i < own) {
            id = id_at(i);
            if (id < 0 || id >= p.num_pages) {
                if (id != -1) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
                id = -1;
            }
        }
        return id;
    };
    int ids = load_ids(0), ids_next = 0;
    uint32_t flags = __ballot_sync(0xffffffffu, ids < 0), flags_now = 0;  // of the batch last issued, of the one at work
    const uint8_t* head_pages = p.pages + (int64_t)hk * RB;
    auto issue = [&](int step) {
        const int i = step * PP;
        if ((i & 31) == 0) {
            if (i > 0) {
                ids = ids_next;
                flags = __ballot_sync(0xffffffffu, ids < 0);
            }
            if (i + 32 < own) ids_next = load_ids(i / 32 + 1);
        }
        int id[PP];
#pragma unroll
        for (int k = 0; k < PP; ++k) id[k] = __shfl_sync(0xffffffffu, ids, (i + k) & 31);
        const uint32_t st = step % STAGES;
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
    // power of two that brings the row's largest to [2^9, 2^10); channels
    // whose codes come in units of 2^-24 another 2^4
    uint32_t qf[NT][W][4];
    float qs[NT][2], qu[NT][2];  // rows 2t, 2t + 1: sum of q, and what a score's unit stands for
    {
        float amax[NT], up2[NT], sums[NT];  // up2: what the power of two divides by
        uint4 raw[NT][W];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g;
            amax[nt] = 0.f;
            int64_t off = -1;
            const int row = it.row0 + r;
            if (row < it.rows) {
                const int tok = row / p.group;
                off = (int64_t)(it.q_token + tok) * p.q_token + (int64_t)(hk * p.group + row - tok * p.group) * p.q_head;
            }
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + off + t * (D / 4));
#pragma unroll
            for (int w = 0; w < W; ++w) {
                raw[nt][w] = off >= 0 ? src[w] : make_uint4(0, 0, 0, 0);
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
                    if (a < INFINITY) amax[nt] = fmaxf(amax[nt], a);  // NaN and infinities stay what they are
                    if (b < INFINITY) amax[nt] = fmaxf(amax[nt], b);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            amax[nt] = fmaxf(amax[nt], __shfl_xor_sync(0xffffffffu, amax[nt], 1));
            amax[nt] = fmaxf(amax[nt], __shfl_xor_sync(0xffffffffu, amax[nt], 2));
            // 2^(9 - floor(log2 amax)), kept within fp32's normal range
            const int e = amax[nt] > 0.f ? (int)(__float_as_uint(amax[nt]) >> 23) - 127 : 9;
            const int up = min(max(9 - e, -120), 120);
            const float f = __uint_as_float((uint32_t)(up + 127) << 23);
            up2[nt] = __uint_as_float((uint32_t)(127 - up) << 23);
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
#pragma unroll
                for (int n = 0; n < 4; ++n) qf[nt][w][n] = h[n];
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sums[nt] = sum * 9.5367431640625e-7f;  // 2^-20
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            qs[nt][0] = __shfl_sync(0xffffffffu, sums[nt], 8 * t);      // row 2t is summed in lanes 4 * 2t ...
            qs[nt][1] = __shfl_sync(0xffffffffu, sums[nt], 8 * t + 4);  // row 2t + 1
            qu[nt][0] = p.scale * __shfl_sync(0xffffffffu, up2[nt], 8 * t);
            qu[nt][1] = p.scale * __shfl_sync(0xffffffffu, up2[nt], 8 * t + 4);
        }
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
    // The sums of the runs of steps that ended, in the references as they stand; `first`: none has yet
    auto add_runs = [&](bool first, bool keep) {
        float4* runs = reinterpret_cast<float4*>(smem + C::RUNS + warp * C::RUN_BYTES) + lane;
        float2* refs = reinterpret_cast<float2*>(smem + C::RUNS + warp * C::RUN_BYTES + NT * (D / 16) * 32 * 16) + lane;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float2 by = make_float2(0.f, 0.f);
            if (!first) by = refs[32 * nt];
            by.x = exp2_approx(by.x - ref[nt][0]);
            by.y = exp2_approx(by.y - ref[nt][1]);
            if (keep) refs[32 * nt] = make_float2(ref[nt][0], ref[nt][1]);
#pragma unroll
            for (int e = 0; e < D / 16; ++e) {
                float(&a)[4] = acc[nt][e];
                if (!first) {
                    const float4 y = runs[32 * (nt * (D / 16) + e)];
                    a[0] = fmaf(y.x, by.x, a[0]);
                    a[1] = fmaf(y.y, by.y, a[1]);
                    a[2] = fmaf(y.z, by.x, a[2]);
                    a[3] = fmaf(y.w, by.y, a[3]);
                }
                if (keep) {
                    runs[32 * (nt * (D / 16) + e)] = make_float4(a[0], a[1], a[2], a[3]);
                    a[0] = a[1] = a[2] = a[3] = 0.f;
                }
            }
        }
    };
    constexpr int RUN = kRunPages / PP;
    // first token that some row of the tile must not see
    const int open = it.context + it.row0 / p.group + 1;

    for (int i = 0; i < steps; ++i) {
        if (i > 0 && i % RUN == 0) add_runs(i == RUN, true);
        const uint32_t st = i % STAGES, parity = i / STAGES & 1;
        bool ready = mbar_try_wait(bars + 8 * st, parity);
        if (!__all_sync(0xffffffffu, ready)) {
            ready = phase_wait_slow(bars + 8 * st, parity, p.status, p.status);
            if (!__all_sync(0xffffffffu, ready)) {  // the wait ran out
                ring_drain(bars, STAGES, i, min(i + STAGES, steps));
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
                    const uint32_t(&b)[4] = qf[nt][w];
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
            const float fa = ka.x * 1048576.f, fb = kb.x * 1048576.f;  // 2^20: the codes' unit
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
                    x[k][nt][c] = fmaf(fmaf(-z, qs[nt][c & 1], s[nt][c]) * (c < 2 ? fa : fb), qu[nt][c & 1], c < 2 ? la : lb);
                }
        }
        // ---- masks: only where a page has tokens that some row must not see
        const int tok0 = (it.page0 + warp * PP + i * PP * kAttendWarps) * 16;
        if ((i * PP & 31) == 0) flags_now = flags;  // no later batch has been issued yet
        if (tok0 + 16 * PP > open || (flags_now >> (i * PP & 31) & 3u)) {
            __syncwarp();
#pragma unroll
            for (int k = 0; k < PP; ++k) {
                const int id = i * PP + k < own ? id_at(i * PP + k) : -1;
                const bool skipped = id < 0 || id >= p.num_pages;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int tk = g + (c < 2 ? 0 : 8);
                        // a tile's rows past its last see what the last sees
                        const int row = min(it.row0 + nt * 8 + 2 * t + (c & 1), it.rows - 1);
                        const bool hide = tok0 + 16 * k + tk > it.context + row / p.group;
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
                    m = fmaxf(m - kTopWeight, ref[nt][j]);
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
                const float2 r0 = half2_floats(h0), r1 = half2_floats(h1);
                if constexpr (PRECISE) {
                    pl[nt][0] = movmatrix_t(pack_half2(a[0] - r0.x, a[1] - r0.y));
                    pl[nt][1] = movmatrix_t(pack_half2(a[2] - r1.x, a[3] - r1.y));
                } else {  // the same weights in every sum (f3s_kv4_math.cuh)
                    a[0] = r0.x;
                    a[1] = r0.y;
                    a[2] = r1.x;
                    a[3] = r1.y;
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

    if (steps > RUN) add_runs(false, false);

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
        const int row = it.row0 + r, tok = row / p.group;
        if (row >= it.rows) continue;
        const int64_t dst = ((int64_t)(it.q_token + tok) * p.heads + hk * p.group + row - tok * p.group) * D + c0;
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
}

// The sums of split tiles: see merge_rows.
template <int D>
__global__ void __launch_bounds__(128) k_attend4_merge(const AttendParams p, const int tq, const int live) {
    wait_for_primary();  // the sums
    const int4* h = reinterpret_cast<const int4*>(&p.plan->num_items);
    const int4 counts = h[0], made_with = h[1];
    const bool fits = plan_fits(p, counts, made_with);
    if (!fits && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(p.status, 0, F3S_ERR_BAD_FORMAT);
    const int num_splits = fits ? counts.y : 0;
    const int group = p.group;
    const Kv4Split* splits =
        reinterpret_cast<const Kv4Split*>(reinterpret_cast<const char*>(p.plan + 1) + (int64_t)p.items_cap * sizeof(Kv4Item));
    merge_rows<D>(num_splits, p.kv_heads, tq, live, p.partials, p.o, p.o_dtype,
                  [&](int split, int hk, int r, int& slot, int& parts) -> int64_t {
                      const Kv4Split s = splits[split];
                      const int row = s.row0 + r, tok = row / group;
                      slot = s.slot;
                      parts = s.parts;
                      return row < s.rows ? (int64_t)(s.q_token + tok) * p.heads + hk * group + row - tok * group : -1;
                  });
}

template <int D, int NT, bool PRECISE>
static int attend_variant(const AttendParams& p, int64_t units, cudaStream_t stream) {
    using C = AttendCfg<D, NT>;
    static PerContext<int> attr;
    const int rc = attr.get(nullptr, [](int* v) -> int {
        *v = 1;
        F3S_CUDA_TRY(cudaFuncSetAttribute(k_attend4<D, NT, PRECISE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::SMEM));
        return F3S_SUCCESS;
    });
    if (rc != F3S_SUCCESS) return rc;
    if (units > INT32_MAX) return F3S_ERR_TOO_LARGE;
    if (units == 0) return F3S_SUCCESS;
    return launch_after(k_attend4<D, NT, PRECISE>, (unsigned)units, kAttendWarps * 32, C::SMEM, stream, p);
}

template <int NT>
static int attend_launch(const AttendParams& p, int head_dim, int64_t units, cudaStream_t stream) {
    const bool precise = weights_in_full(p.o_dtype);
    if (head_dim == 64)
        return precise ? attend_variant<64, NT, true>(p, units, stream) : attend_variant<64, NT, false>(p, units, stream);
    return precise ? attend_variant<128, NT, true>(p, units, stream) : attend_variant<128, NT, false>(p, units, stream);
}

}  // namespace f3s

namespace f3s {

// Scratch: the places of 128-row tiles' runs, then the sums of split tiles.
static size_t run_bytes(const Kv4PlanLayout& L, int head_dim) {
    return L.tile_rows == 128 ? (size_t)kv4_run_places(num_sms_of_current_device()) * kv4_run_floats(head_dim) * 4 : 0;
}
static size_t attend_scratch(const Kv4PlanLayout& L, int kv_heads, int head_dim) {
    return run_bytes(L, head_dim) + (size_t)L.slots_cap * kv_heads * L.tile_rows * (head_dim + 2) * 4;
}

}  // namespace f3s

extern "C" {

size_t f3s_kv4_attention_scratch_size(int32_t num_requests, int64_t num_tokens, int32_t heads, int32_t kv_heads,
                                        int32_t head_dim) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || num_requests < 0 || num_tokens < 0) return 0;
    if (head_dim != 64 && head_dim != 128) return 0;
    const f3s::Kv4PlanLayout L = f3s::kv4_plan_layout(num_requests, num_tokens, heads, kv_heads,
                                                      f3s::num_sms_of_current_device());
    return f3s::attend_scratch(L, kv_heads, head_dim);
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
    const int rc = f3s::check_attend_args(d_Q, q_dtype, q_token_stride, q_head_stride, d_pages, num_pages, heads, kv_heads,
                                     head_dim, d_O, o_dtype);
    if (rc != F3S_SUCCESS) return rc;
    if (num_tokens * (heads / kv_heads) > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
    if (!d_tables || !d_plan || (reinterpret_cast<uintptr_t>(d_plan) & 15)) return F3S_ERR_INVALID_VALUE;
    if (!d_scratch || (reinterpret_cast<uintptr_t>(d_scratch) & 15)) return F3S_ERR_INVALID_VALUE;
    const f3s::Kv4PlanLayout L = f3s::kv4_plan_layout(num_requests, num_tokens, heads, kv_heads,
                                                      f3s::num_sms_of_current_device());
    if (L.items_cap > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
    if (scratch_bytes < f3s::attend_scratch(L, kv_heads, head_dim)) return F3S_ERR_WORKSPACE;
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
    p.partials = reinterpret_cast<float*>(static_cast<char*>(d_scratch) + f3s::run_bytes(L, head_dim));
    p.items_cap = (int)L.items_cap;
    p.num_requests = num_requests;
    p.num_tokens = (int)num_tokens;
    p.tables = d_tables;
    p.table_stride = table_stride;
    cudaStream_t s = (cudaStream_t)stream;
    const int64_t units = L.items_cap * kv_heads;
    int st;
    if (L.tile_rows == 8) st = f3s::attend_launch<1>(p, head_dim, units, s);
    else if (L.tile_rows == 16) st = f3s::attend_launch<2>(p, head_dim, units, s);
    else st = f3s::attend_tiles128(p, head_dim, units, s);
    if (st != F3S_SUCCESS) return st;
    // rows of a tile, on average
    const int live = (int)std::min<int64_t>(L.tile_rows, (num_tokens * p.group + num_requests - 1) / num_requests);
    const int64_t blocks = std::min<int64_t>((int64_t)L.splits_cap * kv_heads * L.tile_rows,
                                             8ll * f3s::num_sms_of_current_device());
    return f3s::launch_after(head_dim == 64 ? f3s::k_attend4_merge<64> : f3s::k_attend4_merge<128>, (unsigned)blocks, 128, 0, s, p,
                             L.tile_rows, live);
}

}  // extern "C"
