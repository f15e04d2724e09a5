// f3s_kv4_plan.cuh -- the attention plan that f3s_block_tables writes and
// f3s_kv4_attention reads.
#pragma once
#include <algorithm>
#include <cstdint>
#include "f3s_internal.cuh"

namespace f3s {

// Query rows of one request and one K/V head are numbered row = token * group
// + head within the group; a tile is tile_rows of them (8, 16 or 128), a piece
// a run of the pages that the tile sees.  A work item is one piece of one
// tile, for every K/V head.
struct Kv4PlanHeader {
    WsHeader ws;  // first: a plan is a workspace to f3s_workspace_status
    int num_items, num_splits;
    int items_cap, tile_rows;
    int heads, kv_heads, num_requests, num_tokens;  // what the plan was made with
    // Places in an attention's scratch for the runs of 128-row tiles, one bit each while a
    // block of whichever attention has it; as many as blocks can run at a time.
    int run_places;
    uint32_t run_taken[10];
    int pad[45];
};
static_assert(sizeof(Kv4PlanHeader) == 512, "plan header is 512 bytes");

struct Kv4Item {
    int request;  // row of the block tables
    int q_token;  // the request's first row of Q
    int row0;     // first query row of the tile
    int rows;     // query rows of the request
    int context;  // tokens cached before the request's first new one
    int page0, page1;  // logical pages of the piece
    int slot;     // where the piece's sums go; -1: the tile is one piece and writes O itself
};
static_assert(sizeof(Kv4Item) == 32, "two 16-byte loads");

struct Kv4Split {
    int slot;   // of the tile's first piece; the others follow it
    int parts;
    int q_token, row0, rows;
    int pad[3];
};
static_assert(sizeof(Kv4Split) == 32, "two 16-byte loads");

// A piece is share = W / target pages (W and target: kv4_plan_layout), two shares as
// long as those are at most kKv4LongPiecePages, and kKv4MinPiecePages in any case.  A
// block costs some 30 pages' time to begin and end, so shorter pieces lose more than
// an even load gains.  Attention and merge, 32 / 8 heads, D = 128, one new token:
//   64 requests of 65 pages      20.9 us with 64 (one piece each), 34.7 with 40 (two)
//   4 requests of 1,000 pages    20.3 us with 64, 23.9 with 40
//   64 of up to 512 pages        90.8 us with one share (with tables), 94.0 with two
//   4 requests of 250 pages      11.6 us with 16 at least, 14.6 with 8
//   1 request of 63 pages        8.0 us with 16 at least, 7.4 with 8
constexpr int kKv4MinPiecePages = 16;
constexpr int kKv4LongPiecePages = 64;

// Pieces of a tile that sees so many pages: the nearest number, since a tile a little
// longer than a piece costs less whole than in two; all that fit at the least size.
__device__ __forceinline__ int kv4_parts(int pages, int piece) {
    return max((pages + (piece == kKv4MinPiecePages ? piece - 1 : piece / 2)) / piece, 1);
}

// Two blocks of 128-row tiles per SM, each with half of the tensor memory.
inline int kv4_run_places(int sms) { return std::min(2 * sms, 10 * 32); }
__host__ __device__ constexpr int64_t kv4_run_floats(int head_dim) { return 128 * (head_dim + 2); }

struct Kv4PlanLayout {
    int tile_rows;
    int target;  // pieces to cut the work into
    int64_t items_cap, splits_cap, slots_cap;
    size_t items, splits, total;
};

// What a host can know before the lengths are read; num_tokens bounds the new
// tokens.  With W = sum over tiles of the pages they see and pieces of
// P >= W / target pages, the tiles have at most tiles + W / P pieces; those of
// tiles cut in two or more hold more than P / 2 pages each.  (A share is W / target.)
inline Kv4PlanLayout kv4_plan_layout(int num_requests, int64_t num_tokens, int heads, int kv_heads, int sms) {
    Kv4PlanLayout L{};
    const int64_t group = heads / kv_heads;
    const int64_t rows = num_tokens * group;
    const int64_t mean = num_requests > 0 ? (rows + num_requests - 1) / num_requests : 0;
    // Rows per request -> us with tiles of 8, 16, 128 rows (64 requests of 1,024 tokens,
    // 8 K/V heads, D = 128; 64 requests, 2 K/V heads, D = 64; 8 requests, 8 heads, D = 128):
    //   24:  51, 60,  94   16, 27, 46   17, 25, 45
    //   32:  64, 59,  96   16, 28, 47   21, 26, 46
    //   48:  92, 85,  99   23, 21, 34   21, 32, 52
    //   64: 120, 106, 101  26, 22, 37   21, 37, 54
    //   96: 176, 153, 108  37, 32, 39   30, 36, 49
    //  128: 232, 202, 116  46, 36, 41   34, 38, 53
    //  256: 458, 393, 223  87, 66, 42   63, 58, 52
    // The rule looks at the mean alone: where few requests leave SMs idle, lower tiles are
    // faster than what it takes (8 requests of 64 rows: 21 against 37 us), and a batch
    // of unequal requests gets one height for all (63 decoding requests and a prompt of
    // 2,000 tokens: 178 us, 21 and 95 apart), as does one with spare capacity (64 decoding
    // requests in a batch for 2,048 tokens: 93 us).
    // Tiles of 32 rows on mma.sync were never faster than the best of these.
    L.tile_rows = mean <= 32 ? 8 : mean <= 96 ? 16 : 128;
    const int64_t tiles = rows / L.tile_rows + num_requests;
    // twice as many pieces as blocks run at a time (4 per SM, 2 of 128 rows, one K/V head each),
    // so that blocks of unequal work even out
    L.target = (int)std::max<int64_t>(1, (int64_t)sms * (L.tile_rows == 128 ? 4 : 8) / kv_heads);
    L.items_cap = tiles + L.target;
    L.slots_cap = 2 * (int64_t)L.target;
    L.splits_cap = L.target;
    L.items = sizeof(Kv4PlanHeader);
    L.splits = L.items + (size_t)L.items_cap * sizeof(Kv4Item);
    L.total = L.splits + (size_t)L.splits_cap * sizeof(Kv4Split);
    return L;
}

}  // namespace f3s
