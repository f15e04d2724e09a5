// f3s_kv4_plan.cuh -- the attention plan that f3s_block_tables writes and
// f3s_kv4_attention reads.
#pragma once
#include <cstdint>
#include "f3s_internal.cuh"

namespace f3s {

// Query rows of one request and one K/V head are numbered row = token * group
// + head within the group; a tile is tile_rows of them (8, 16, 32 or 128), a piece
// a run of the pages that the tile sees.  A work item is one piece of one
// tile, for every K/V head.
struct Kv4PlanHeader {
    WsHeader ws;  // first: a plan is a workspace to f3s_workspace_status
    int num_items, num_splits;
    int items_cap, tile_rows;
    int heads, kv_heads, num_requests, num_tokens;  // what the plan was made with
    int pad[56];
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

// A piece holds at least this many pages of a tile that is split.
constexpr int kKv4MinPiecePages = 8;

struct Kv4PlanLayout {
    int tile_rows;
    int target;  // pieces to cut the work into
    int64_t items_cap, splits_cap, slots_cap;
    size_t items, splits, total;
};

// What a host can know before the lengths are read; num_tokens bounds the new
// tokens.  With W = sum over tiles of the pages they see and pieces of
// P >= W / target pages, the tiles have at most tiles + W / P pieces; those of
// tiles cut in two or more hold more than P / 2 pages each.
inline Kv4PlanLayout kv4_plan_layout(int num_requests, int64_t num_tokens, int heads, int kv_heads, int sms) {
    Kv4PlanLayout L{};
    const int64_t group = heads / kv_heads;
    const int64_t rows = num_tokens * group;
    const int64_t mean = num_requests > 0 ? (rows + num_requests - 1) / num_requests : 0;
    L.tile_rows = mean <= 8 ? 8 : mean <= 16 ? 16 : mean <= 96 ? 32 : 128;
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
