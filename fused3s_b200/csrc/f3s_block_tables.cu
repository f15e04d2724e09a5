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
// block waits for another: one launch, a few microseconds, bound by latency
// (the lengths, the table look-up and the free-list look-up follow one another).
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
    int group;  // 0: no plan
    int tile_rows, target;
    int items_cap, splits_cap, slots_cap;
    int* query_offsets;
    int* positions;
    int* slots;
    int* begin_out;
    WsHeader* ws;
    Kv4PlanHeader* plan;
    Kv4Item* items;
    Kv4Split* splits;
};

struct BtRequest {
    int context, count;      // cached tokens, new tokens that have room
    int old_pages, pages;    // table entries filled before, and after
    int tiles;
    int error;
};

// What fits of request r, whose new tokens start at `first` among all.
__device__ __forceinline__ BtRequest bt_request(const BlockTablesParams& p, int c, int n, int64_t first) {
    BtRequest q;
    q.error = c < 0 || n < 0 ? F3S_ERR_INVALID_VALUE : 0;
    c = max(c, 0);
    n = max(n, 0);
    const int64_t room_rows = p.num_tokens - first, room_table = (int64_t)p.width * 16 - c;
    int64_t fit = n;
    if (fit > room_rows) fit = max(room_rows, (int64_t)0);
    if (fit > room_table) fit = max(room_table, (int64_t)0);
    if (fit < n || room_table < 0) q.error = q.error ? q.error : F3S_ERR_TOO_LARGE;
    q.context = (int)min((int64_t)c, (int64_t)p.width * 16);
    q.count = (int)fit;
    q.old_pages = (q.context + 15) / 16;
    q.pages = (int)(((int64_t)q.context + fit + 15) / 16);
    q.tiles = p.group ? (int)((fit * p.group + p.tile_rows - 1) / p.tile_rows) : 0;
    return q;
}

__device__ __forceinline__ int64_t bt_scan(int64_t v, int64_t& total, int64_t* scratch) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
    }
    if (lane == 31) scratch[wid] = inc;
    __syncthreads();
    int64_t base = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kBtThreads / 32; ++i) {
        const int64_t s = scratch[i];
        if (i < wid) base += s;
        total += s;
    }
    __syncthreads();
    return base + inc - v;
}

// Index of the request (0 ... n - 1) whose range [s[i], s[i + 1]) holds x.
__device__ __forceinline__ int bt_find(const int64_t* s, int n, int64_t x) {
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
    __shared__ int64_t s_first[kBtThreads + 1];  // first new token of each request of the chunk
    __shared__ int64_t s_page[kBtThreads + 1];   // first new page
    __shared__ int64_t s_item[kBtThreads + 1];   // first work item
    __shared__ int64_t s_split[kBtThreads + 1];  // first split tile
    __shared__ int64_t s_slot[kBtThreads + 1];   // first piece of a split tile
    __shared__ BtRequest s_req[kBtThreads];
    __shared__ int64_t s_scratch[kBtThreads / 32];
    const int tid = threadIdx.x;
    const int64_t at = (int64_t)blockIdx.x * kBtThreads + tid, step = (int64_t)gridDim.x * kBtThreads;
    const int chunks = (p.requests + kBtThreads - 1) / kBtThreads;
    if (blockIdx.x == 0 && tid == 0) {
        p.ws->status = 0;
        p.ws->abort = 0;
    }
    __syncthreads();

    // pages that all tiles see together, which sets the size of a piece
    int64_t piece = kKv4MinPiecePages;
    int c0 = 0, n0 = 0;  // this thread's request of the first chunk
    if (tid < p.requests) {
        c0 = p.context[tid];
        n0 = p.fresh[tid];
    }
    const int64_t begin = p.begin ? max(p.begin[0], 0) : 0;
    const int64_t avail = max((int64_t)p.num_free - begin, (int64_t)0);
    if (p.group) {
        int64_t work = 0, base = 0;
        for (int chunk = 0; chunk < chunks; ++chunk) {
            const int r = chunk * kBtThreads + tid;
            int c = c0, n = n0;
            if (chunk) {
                c = r < p.requests ? p.context[r] : 0;
                n = r < p.requests ? p.fresh[r] : 0;
            }
            int64_t total, sum;
            const int64_t first = base + bt_scan(max(n, 0), total, s_scratch);
            base += total;
            const BtRequest q = bt_request(p, c, n, first);
            bt_scan(r < p.requests ? (int64_t)q.tiles * q.pages : 0, sum, s_scratch);
            work += sum;
        }
        piece = max((work + p.target - 1) / p.target, (int64_t)kKv4MinPiecePages);
    }

    int64_t first_base = 0, page_base = 0, item_base = 0, split_base = 0, slot_base = 0;
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const int r0 = chunk * kBtThreads, r = r0 + tid, here = min(kBtThreads, p.requests - r0);
        int c = c0, n = n0;
        if (chunk) {
            c = r < p.requests ? p.context[r] : 0;
            n = r < p.requests ? p.fresh[r] : 0;
        }
        int64_t tokens, pages, items, splits, slots;
        const int64_t first = first_base + bt_scan(max(n, 0), tokens, s_scratch);
        BtRequest q = bt_request(p, c, n, first);
        if (r >= p.requests) q = BtRequest{};
        const int parts = q.tiles ? (int)((q.pages + piece - 1) / piece) : 0;
        const int64_t page = page_base + bt_scan(q.pages - q.old_pages, pages, s_scratch);
        const int64_t item = item_base + bt_scan((int64_t)q.tiles * parts, items, s_scratch);
        const int64_t split = split_base + bt_scan(parts > 1 ? q.tiles : 0, splits, s_scratch);
        const int64_t slot0 = slot_base + bt_scan(parts > 1 ? (int64_t)q.tiles * parts : 0, slots, s_scratch);
        if (q.error) bt_error(p, q.error);
        if (tid < here) {
            s_first[tid] = first;
            s_page[tid] = page;
            s_item[tid] = item;
            s_split[tid] = split;
            s_slot[tid] = slot0;
            s_req[tid] = q;
            if (blockIdx.x == 0 && p.query_offsets) p.query_offsets[r] = (int)min(first, (int64_t)INT32_MAX);
        }
        if (tid == 0) {
            s_first[here] = first_base + tokens;
            s_page[here] = page_base + pages;
            s_item[here] = item_base + items;
            s_split[here] = split_base + splits;
            s_slot[here] = slot_base + slots;
        }
        __syncthreads();
        // slots and positions of the chunk's tokens
        const int64_t token_end = min(first_base + tokens, p.num_tokens);
        for (int64_t t = first_base + at; t < token_end; t += step) {
            const int i = bt_find(s_first, here, t);
            const BtRequest& w = s_req[i];
            const int64_t pos = (int64_t)w.context + (t - s_first[i]);
            int slot = -1;
            if (t - s_first[i] < w.count) {
                const int k = (int)(pos >> 4);
                int id = -1;
                if (k < w.old_pages) {
                    id = p.tables[(int64_t)(r0 + i) * p.stride + k];
                } else {
                    const int64_t f = s_page[i] + (k - w.old_pages);
                    if (f < avail) id = p.free_pages[begin + f];
                }
                // an entry that no cache can hold stays out of range, for the
                // store to report
                slot = id < 0 ? id : id < INT32_MAX / 16 ? id * 16 + (int)(pos & 15) : INT32_MAX;
            }
            p.slots[t] = slot;
            p.positions[t] = (int)min(pos, (int64_t)INT32_MAX);
        }
        // the new entries of the chunk's table rows
        for (int64_t f = page_base + at; f < page_base + pages; f += step) {
            const int i = bt_find(s_page, here, f);
            const int k = s_req[i].old_pages + (int)(f - s_page[i]);
            p.tables[(int64_t)(r0 + i) * p.stride + k] = f < avail ? p.free_pages[begin + f] : -1;
        }
        // work items and split tiles
        for (int64_t it = item_base + at; it < item_base + items; it += step) {
            if (it >= p.items_cap) break;
            const int i = bt_find(s_item, here, it);
            const BtRequest& w = s_req[i];
            const int m = (int)((w.pages + piece - 1) / piece);
            const int local = (int)(it - s_item[i]);
            const int tile = local / m, part = local - tile * m;
            const int row0 = tile * p.tile_rows, rows = w.count * p.group;
            const int last = min(row0 + p.tile_rows, rows) - 1;  // the tile's last row sees the most
            const int64_t seen = ((int64_t)w.context + last / p.group) / 16 + 1;
            Kv4Item d;
            d.request = r0 + i;
            d.q_token = (int)s_first[i];
            d.row0 = row0;
            d.rows = rows;
            d.context = w.context;
            d.page0 = (int)(seen * part / m);
            d.page1 = (int)(seen * (part + 1) / m);
            const int64_t slot = s_slot[i] + local;
            d.slot = m > 1 && slot < p.slots_cap ? (int)slot : -1;
            p.items[it] = d;
            if (part == 0 && m > 1) {
                const int64_t sp = s_split[i] + tile;
                if (sp < p.splits_cap) {
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
        first_base += tokens;
        page_base += pages;
        item_base += items;
        split_base += splits;
        slot_base += slots;
        __syncthreads();  // the chunk's arrays are read no more
    }
    // slots behind the last token
    for (int64_t t = first_base + at; t < p.num_tokens; t += step) {
        p.slots[t] = -1;
        p.positions[t] = 0;
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.query_offsets[p.requests] = (int)min(first_base, (int64_t)INT32_MAX);
        p.begin_out[0] = (int)(begin + min(page_base, avail));
        if (first_base > p.num_tokens) bt_error(p, F3S_ERR_TOO_LARGE);
        if (page_base > avail) bt_error(p, F3S_ERR_NO_PAGES);
        if (p.plan) {
            p.plan->num_items = (int)min(item_base, (int64_t)p.items_cap);
            p.plan->num_splits = (int)min(split_base, (int64_t)p.splits_cap);
            p.plan->items_cap = p.items_cap;
            p.plan->splits_cap = p.splits_cap;
            p.plan->tile_rows = p.tile_rows;
            p.plan->group = p.group;
            p.plan->num_requests = p.requests;
            p.plan->num_tokens = (int)p.num_tokens;
        }
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
        p.items = reinterpret_cast<f3s::Kv4Item*>(base + L.items);
        p.splits = reinterpret_cast<f3s::Kv4Split*>(base + L.splits);
        units = std::max(units, L.items_cap);
    }
    // one block per 1024 tokens (two per thread), a block per SM at most
    const int64_t blocks = std::min<int64_t>((units + 1023) / 1024, f3s::num_sms_of_current_device());
    f3s::k_block_tables<<<(unsigned)blocks, f3s::kBtThreads, 0, (cudaStream_t)stream>>>(p);
    F3S_LAUNCH_CHECK();
    return F3S_SUCCESS;
}

}  // extern "C"
