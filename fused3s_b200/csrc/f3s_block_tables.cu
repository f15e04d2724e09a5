// f3s_block_tables.cu -- block tables, slot maps and the attention plan from
// request lengths, in one launch.
//
// A request with c cached and n new tokens holds ceil((c + n) / 16) pages; the
// first ceil(c / 16) entries of its table row are filled already and the rest
// come from the free list in request order:
//   query_offsets = exclusive sum of n,   page base = begin + exclusive sum of
//   ceil((c + n) / 16) - ceil(c / 16),   slot(j) = page((c + j) / 16) * 16 + (c + j) % 16
// Every block scans the lengths for itself, 512 requests at a time in shared
// memory, and then writes its share of the tokens, pages and work items of
// those requests, each found by a binary search in the scanned offsets.  No
// block waits for another: one launch, bound by latency (the lengths, the table
// look-up and the free-list look-up follow one another).  256 requests, one new
// token each: 3.8 us; 41 prompts of up to 1,777 new tokens: 5.7 us (in a CUDA graph).
#include <algorithm>
#include "f3s_internal.cuh"
#include "f3s_kv4_plan.cuh"

namespace f3s {

constexpr int kBtThreads = 512;

struct BlockTablesParams {
    const int* context;
    const int* fresh;  // new tokens per request
    int requests;
    int* tables;
    int64_t stride;
    int width;
    const int* free_pages;
    int num_free;
    const int* begin;
    int64_t num_tokens;
    int heads, kv_heads, group, tile_rows;
    int target;  // 0: no plan
    int items_cap, splits_cap, slots_cap, run_places;
    int* query_offsets;
    int* positions;
    int* slots;
    int* begin_out;
    WsHeader* ws;
    Kv4PlanHeader* plan;
    Kv4Item* items;
    Kv4Split* splits;
};

// Sums stop here: what lies past it does not fit any array (num_tokens and the
// plan's arrays are shorter), and two of them still add up in 32 bits.
constexpr uint32_t kBtMost = 1u << 30;
__device__ __forceinline__ uint32_t bt_add(uint32_t a, uint32_t b) { return min(a + b, kBtMost); }

struct BtRequest {
    int context, count;    // cached tokens, new tokens that have room
    int old_pages, pages;  // table entries filled before, and after
    int tiles;
    int error;
};

// What fits of a request whose new tokens start at `first` among all.
__device__ __forceinline__ BtRequest bt_request(const BlockTablesParams& p, int c, int n, uint32_t first) {
    BtRequest q;
    q.error = c < 0 || n < 0 ? F3S_ERR_INVALID_VALUE : 0;
    c = max(c, 0);
    n = max(n, 0);
    const int room_rows = max((int)p.num_tokens - (int)first, 0), room_table = p.width * 16 - c;
    const int fit = min(min(n, room_rows), max(room_table, 0));
    if (fit < n || room_table < 0) q.error = q.error ? q.error : F3S_ERR_TOO_LARGE;
    q.context = min(c, p.width * 16);
    q.count = fit;
    q.old_pages = (q.context + 15) >> 4;
    q.pages = (q.context + fit + 15) >> 4;
    q.tiles = (fit * p.group + p.tile_rows - 1) / p.tile_rows;
    return q;
}

// Exclusive sums of N values per thread over the block; total receives the
// block's.  Two barriers, whatever N is.
template <int N>
__device__ __forceinline__ void bt_scan(uint32_t (&v)[N], uint32_t (&total)[N], uint32_t (*scratch)[kBtThreads / 32]) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    uint32_t inc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        inc[k] = v[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t n = __shfl_up_sync(0xffffffffu, inc[k], o);
            if (lane >= o) inc[k] = bt_add(inc[k], n);
        }
        if (lane == 31) scratch[k][wid] = inc[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        // the warps' totals, scanned by every warp for itself
        uint32_t w = lane < kBtThreads / 32 ? scratch[k][lane] : 0;
#pragma unroll
        for (int o = 1; o < kBtThreads / 32; o <<= 1) {
            const uint32_t n = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w = bt_add(w, n);
        }
        total[k] = __shfl_sync(0xffffffffu, w, kBtThreads / 32 - 1);
        uint32_t before = __shfl_up_sync(0xffffffffu, w, 1);
        if (lane == 0) before = 0;
        v[k] = bt_add(__shfl_sync(0xffffffffu, before, wid), __shfl_up_sync(0xffffffffu, inc[k], 1) * (lane > 0));
    }
    __syncthreads();
}

// Index of the request (0 ... n - 1) whose range [s[i], s[i + 1]) holds x.
__device__ __forceinline__ int bt_find(const uint32_t* s, int n, uint32_t x) {
    int lo = 0, hi = n;  // s[lo] <= x < s[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void bt_error(const BlockTablesParams& p, int code) {
    // every block sees every error; the first block reports it
    if (blockIdx.x == 0) atomicCAS(&p.ws->status, 0, code);
}

__global__ void __launch_bounds__(kBtThreads) k_block_tables(const BlockTablesParams p) {
    __shared__ uint32_t s_first[kBtThreads + 1];  // first new token of each request of the chunk
    __shared__ uint32_t s_page[kBtThreads + 1];   // first new page
    __shared__ uint32_t s_item[kBtThreads + 1];   // first work item
    __shared__ uint32_t s_split[kBtThreads + 1];  // first split tile
    __shared__ uint32_t s_slot[kBtThreads + 1];   // first piece of a split tile
    __shared__ BtRequest s_req[kBtThreads];
    __shared__ uint32_t s_scratch[3][kBtThreads / 32];
    __shared__ unsigned long long s_work;
    launch_dependents();
    const int tid = threadIdx.x;
    const int chunks = (p.requests + kBtThreads - 1) / kBtThreads;
    // half of the threads write slots, a quarter table entries, a quarter work items
    const int role = tid / (kBtThreads / 4), at4 = tid % (kBtThreads / 4);
    const uint32_t token_at = blockIdx.x * (kBtThreads / 2) + tid % (kBtThreads / 2), token_step = gridDim.x * (kBtThreads / 2);
    const uint32_t other_at = blockIdx.x * (kBtThreads / 4) + at4, other_step = gridDim.x * (kBtThreads / 4);
    int c0 = 0, n0 = 0;  // this thread's request of the first chunk
    if (tid < p.requests) {
        c0 = p.context[tid];
        n0 = p.fresh[tid];
    }
    const int begin = p.begin ? max(p.begin[0], 0) : 0;
    const uint32_t avail = (uint32_t)max(p.num_free - begin, 0);
    if (tid == 0) s_work = 0;
    if (blockIdx.x == 0 && tid == 0) {
        p.ws->status = 0;
        p.ws->abort = 0;
    }
    __syncthreads();

    // pages that all tiles see together, which sets the size of a piece
    uint32_t v1[1], total1[1];
    uint32_t first_base = 0, first0 = 0, tokens0 = 0;
    unsigned long long work = 0;
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const int r = chunk * kBtThreads + tid;
        const int c = chunk == 0 ? c0 : r < p.requests ? p.context[r] : 0;
        const int n = chunk == 0 ? n0 : r < p.requests ? p.fresh[r] : 0;
        v1[0] = min((uint32_t)max(n, 0), kBtMost);
        bt_scan<1>(v1, total1, s_scratch);
        if (chunk == 0) {
            first0 = v1[0];
            tokens0 = total1[0];
        }
        if (p.target == 0) break;  // no plan: the first chunk's sums are all that is kept
        if (r < p.requests) {
            const BtRequest q = bt_request(p, c, n, bt_add(first_base, v1[0]));
            work += (unsigned long long)q.tiles * q.pages;
        }
        first_base = bt_add(first_base, total1[0]);
    }
    int piece = kKv4MinPiecePages;
    if (p.target) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
        if ((tid & 31) == 0 && work) atomicAdd(&s_work, work);
        __syncthreads();
        const unsigned long long share = (s_work + p.target - 1) / p.target;
        piece = (int)min(max(share, min(2 * share, (unsigned long long)kKv4LongPiecePages)), 1ull << 28);
        piece = max(piece, kKv4MinPiecePages);
    }

    first_base = 0;
    uint32_t page_base = 0, item_base = 0, split_base = 0, slot_base = 0;
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const int r0 = chunk * kBtThreads, r = r0 + tid, here = min(kBtThreads, p.requests - r0);
        int c = c0, n = n0;
        uint32_t first = first0, tokens = tokens0;
        if (chunk) {
            c = r < p.requests ? p.context[r] : 0;
            n = r < p.requests ? p.fresh[r] : 0;
            v1[0] = min((uint32_t)max(n, 0), kBtMost);
            bt_scan<1>(v1, total1, s_scratch);
            first = bt_add(first_base, v1[0]);
            tokens = total1[0];
        }
        BtRequest q = bt_request(p, c, n, first);
        if (r >= p.requests) q = BtRequest{};
        const int parts = q.tiles ? kv4_parts(q.pages, piece) : 0;
        // new pages, items, and tiles cut in several (their slots are parts times as many)
        uint32_t v[3] = {(uint32_t)(q.pages - q.old_pages), min((uint32_t)q.tiles * (uint32_t)parts, kBtMost),
                         parts > 1 ? (uint32_t)q.tiles : 0u};
        uint32_t total[3];
        bt_scan<3>(v, total, s_scratch);
        v1[0] = parts > 1 ? min((uint32_t)q.tiles * (uint32_t)parts, kBtMost) : 0u;
        total1[0] = 0;
        if (total[2]) bt_scan<1>(v1, total1, s_scratch);  // for the whole block
        if (q.error) bt_error(p, q.error);
        if (tid < here) {
            s_first[tid] = first;
            s_page[tid] = bt_add(page_base, v[0]);
            s_item[tid] = bt_add(item_base, v[1]);
            s_split[tid] = bt_add(split_base, v[2]);
            s_slot[tid] = bt_add(slot_base, v1[0]);
            s_req[tid] = q;
            if (blockIdx.x == 0) p.query_offsets[r] = (int)first;
        }
        const uint32_t token_end = bt_add(first_base, tokens), page_end = bt_add(page_base, total[0]),
                       item_end = bt_add(item_base, total[1]);
        if (tid == 0) {
            s_first[here] = token_end;
            s_page[here] = page_end;
            s_item[here] = item_end;
        }
        __syncthreads();
        if (role < 2) {  // slots and positions of the chunk's tokens
            const uint32_t end = min(token_end, (uint32_t)p.num_tokens);
            for (uint32_t t = first_base + token_at; t < end; t += token_step) {
                const int i = bt_find(s_first, here, t);
                const BtRequest& w = s_req[i];
                const int k = (int)(t - s_first[i]);
                const int64_t pos = (int64_t)w.context + k;
                int slot = -1;
                if (k < w.count) {
                    const int page = (int)(pos >> 4);
                    int id = -1;
                    if (page < w.old_pages) {
                        id = p.tables[(int64_t)(r0 + i) * p.stride + page];
                    } else {
                        const uint32_t f = s_page[i] + (page - w.old_pages);
                        if (f < avail) id = p.free_pages[begin + f];
                    }
                    // an entry that no cache can hold stays out of range, for the
                    // store to report
                    slot = id < 0 ? id : id < INT32_MAX / 16 ? id * 16 + (int)(pos & 15) : INT32_MAX;
                }
                p.slots[t] = slot;
                p.positions[t] = (int)min(pos, (int64_t)INT32_MAX);
            }
        } else if (role == 2) {  // the new entries of the chunk's table rows
            for (uint32_t f = page_base + other_at; f < page_end; f += other_step) {
                const int i = bt_find(s_page, here, f);
                const int k = s_req[i].old_pages + (int)(f - s_page[i]);
                p.tables[(int64_t)(r0 + i) * p.stride + k] = f < avail ? p.free_pages[begin + f] : -1;
            }
        } else {  // work items and split tiles
            for (uint32_t it = item_base + other_at; it < min(item_end, (uint32_t)p.items_cap); it += other_step) {
                const int i = bt_find(s_item, here, it);
                const BtRequest& w = s_req[i];
                const int m = kv4_parts(w.pages, piece);
                const int local = (int)(it - s_item[i]);
                const int nth = local / m, part = local - nth * m;
                // a request's last rows see the most: their tiles begin first
                const int row0 = (w.tiles - 1 - nth) * p.tile_rows, rows = w.count * p.group;
                const int last = min(row0 + p.tile_rows, rows) - 1;  // the tile's last row sees the most
                const int seen = (w.context + last / p.group) / 16 + 1;
                Kv4Item d;
                d.request = r0 + i;
                d.q_token = (int)s_first[i];
                d.row0 = row0;
                d.rows = rows;
                d.context = w.context;
                d.page0 = m == 1 ? 0 : (int)((int64_t)seen * part / m);
                d.page1 = m == 1 ? seen : (int)((int64_t)seen * (part + 1) / m);
                const uint32_t slot = s_slot[i] + local;
                d.slot = m > 1 && slot < (uint32_t)p.slots_cap ? (int)slot : -1;
                p.items[it] = d;
                if (part == 0 && m > 1) {
                    const uint32_t sp = s_split[i] + nth;
                    if (sp < (uint32_t)p.splits_cap) {
                        Kv4Split s{};
                        s.slot = (int)slot;
                        s.parts = m;
                        s.q_token = d.q_token;
                        s.row0 = row0;
                        s.rows = rows;
                        p.splits[sp] = s;
                    }
                }
            }
        }
        first_base = token_end;
        page_base = page_end;
        item_base = item_end;
        split_base = bt_add(split_base, total[2]);
        slot_base = bt_add(slot_base, total1[0]);
        if (chunk + 1 < chunks) __syncthreads();  // the chunk's arrays are read no more
    }
    // slots behind the last token
    for (uint32_t t = first_base + blockIdx.x * kBtThreads + tid; t < (uint32_t)p.num_tokens; t += gridDim.x * kBtThreads) {
        p.slots[t] = -1;
        p.positions[t] = 0;
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.query_offsets[p.requests] = (int)first_base;
        p.begin_out[0] = begin + (int)min(page_base, avail);
        if (first_base > (uint32_t)p.num_tokens) bt_error(p, F3S_ERR_TOO_LARGE);
        if (page_base > avail) bt_error(p, F3S_ERR_NO_PAGES);
        p.plan->num_items = (int)min(item_base, (uint32_t)p.items_cap);
        p.plan->num_splits = (int)min(split_base, (uint32_t)p.splits_cap);
        p.plan->items_cap = p.items_cap;
        p.plan->tile_rows = p.tile_rows;
        p.plan->heads = p.heads;
        p.plan->kv_heads = p.kv_heads;
        p.plan->num_requests = p.requests;
        p.plan->num_tokens = (int)p.num_tokens;
        p.plan->run_places = p.run_places;
        for (uint32_t& w : p.plan->run_taken) w = 0;
    }
}

static int check_tables(int num_requests, int64_t num_tokens, int heads, int kv_heads) {
    if (num_requests < 0 || num_tokens < 0 || heads < 0 || kv_heads < 0) return F3S_ERR_INVALID_VALUE;
    if ((heads == 0) != (kv_heads == 0) || (kv_heads && heads % kv_heads)) return F3S_ERR_INVALID_VALUE;
    const int64_t group = kv_heads ? heads / kv_heads : 1;
    if (num_tokens > INT32_MAX / 4 || num_tokens * group > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
    return F3S_SUCCESS;
}

}  // namespace f3s

extern "C" {

size_t f3s_block_tables_workspace_size(int32_t num_requests, int64_t num_tokens, int32_t heads, int32_t kv_heads) {
    if (f3s::check_tables(num_requests, num_tokens, heads, kv_heads) != F3S_SUCCESS) return 0;
    if (heads == 0) return sizeof(f3s::Kv4PlanHeader);
    const f3s::Kv4PlanLayout L = f3s::kv4_plan_layout(num_requests, num_tokens, heads, kv_heads,
                                                      f3s::num_sms_of_current_device());
    if (L.items_cap > INT32_MAX / 4) return 0;
    return L.total;
}

int f3s_block_tables(const int32_t* d_context_lens, const int32_t* d_new_lens, int32_t num_requests, int32_t* d_tables,
                     int64_t table_stride, int32_t table_width, const int32_t* d_free_pages, int32_t num_free,
                     const int32_t* d_free_begin, int64_t num_tokens, int32_t heads, int32_t kv_heads,
                     int32_t* d_query_offsets, int32_t* d_positions, int32_t* d_slots, int32_t* d_free_begin_out,
                     void* d_plan, size_t plan_bytes, f3s_stream_t stream) {
    f3s::NvtxRange nvtx_("f3s_block_tables");
    const int rc = f3s::check_tables(num_requests, num_tokens, heads, kv_heads);
    if (rc != F3S_SUCCESS) return rc;
    if (table_width < 0 || num_free < 0 || (num_requests > 1 && table_stride < table_width)) return F3S_ERR_INVALID_VALUE;
    if ((int64_t)table_width * 16 > INT32_MAX) return F3S_ERR_TOO_LARGE;
    if (num_requests > 0 && (!d_context_lens || !d_new_lens)) return F3S_ERR_INVALID_VALUE;
    if (num_requests > 0 && table_width > 0 && !d_tables) return F3S_ERR_INVALID_VALUE;
    if (num_free > 0 && !d_free_pages) return F3S_ERR_INVALID_VALUE;
    if (!d_query_offsets || !d_free_begin_out || (num_tokens > 0 && (!d_positions || !d_slots)))
        return F3S_ERR_INVALID_VALUE;
    if (!d_plan || (reinterpret_cast<uintptr_t>(d_plan) & 15)) return F3S_ERR_INVALID_VALUE;
    if (plan_bytes < sizeof(f3s::Kv4PlanHeader)) return F3S_ERR_WORKSPACE;
    f3s::BlockTablesParams p{};
    p.context = d_context_lens;
    p.fresh = d_new_lens;
    p.requests = num_requests;
    p.tables = d_tables;
    p.stride = table_stride;
    p.width = table_width;
    p.free_pages = d_free_pages;
    p.num_free = num_free;
    p.begin = d_free_begin;
    p.num_tokens = num_tokens;
    p.query_offsets = d_query_offsets;
    p.positions = d_positions;
    p.slots = d_slots;
    p.begin_out = d_free_begin_out;
    char* base = static_cast<char*>(d_plan);
    p.ws = static_cast<f3s::WsHeader*>(d_plan);
    p.plan = static_cast<f3s::Kv4PlanHeader*>(d_plan);
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.group = p.tile_rows = 1;
    int64_t units = std::max<int64_t>(num_tokens, 1);
    if (heads > 0) {
        const f3s::Kv4PlanLayout L = f3s::kv4_plan_layout(num_requests, num_tokens, heads, kv_heads,
                                                          f3s::num_sms_of_current_device());
        if (L.items_cap > INT32_MAX / 4) return F3S_ERR_TOO_LARGE;
        if (plan_bytes < L.total) return F3S_ERR_WORKSPACE;
        p.group = heads / kv_heads;
        p.tile_rows = L.tile_rows;
        p.target = L.target;
        p.items_cap = (int)L.items_cap;
        p.splits_cap = (int)L.splits_cap;
        p.slots_cap = (int)L.slots_cap;
        p.run_places = f3s::kv4_run_places(f3s::num_sms_of_current_device());
        p.items = reinterpret_cast<f3s::Kv4Item*>(base + L.items);
        p.splits = reinterpret_cast<f3s::Kv4Split*>(base + L.splits);
        units = std::max(units, L.items_cap);
    }
    // One block per 1024 tokens or items, a block per SM at most.  Every block reads
    // where the free list begins and the first one writes where it goes on: one block
    // where that is the same word, since blocks do not wait for each other (41 prompts,
    // 47,677 tokens: 79 us in place, 6.1 apart).
    const int64_t blocks = d_free_begin_out == d_free_begin
                               ? 1
                               : std::min<int64_t>((units + 1023) / 1024, f3s::num_sms_of_current_device());
    f3s::k_block_tables<<<(unsigned)blocks, f3s::kBtThreads, 0, (cudaStream_t)stream>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

}  // extern "C"
