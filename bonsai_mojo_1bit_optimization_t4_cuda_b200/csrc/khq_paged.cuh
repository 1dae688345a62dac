// khq_paged.cuh -- what the plan of a step over the paged cache and the attention kernels that run from it agree on.
#pragma once
#include <stdint.h>

namespace khq_paged {

// The schedule in device memory: a header of 16 ints, the items (one per request and query tile, request by request), and the
// items' first key blocks counted through (cum[n_items] = the total).  The attention runs over H_kv copies of that list, one kv
// head after the other.
constexpr int SCHED_HEADER = 16;  // ints: [0] items, [1] key blocks of one kv head
struct alignas(16) Item {
    int b, n_blocks, ntok, kv;  // request; key blocks (causal: up to the tile's last token); new tokens of the tile; the request's tokens
    int row0, pos0, pad[2];     // the tile's first row in the ragged tensors, that row's position
};
constexpr int ITEM_INTS = sizeof(Item) / 4;

// Query rows are (new token, query head of the kv head) pairs, token-major.  Up to 16 rows a request: the decode kernel, whose tile is
// a request's rows.  Above: tiles of 2 x 128 rows on a CTA pair.
constexpr int MAX_REP = 128;  // query heads of a kv head
constexpr int DECODE_ROWS = 16, DECODE_KEYS = 64, TILE_ROWS = 128, TILE_KEYS = 128;
struct Tile {
    int tokens, keys;  // new tokens of a query tile, keys of a block
    bool decode;
};
inline Tile tile_of(int H_q, int H_kv, int max_new) {
    const int n_rep = H_q / H_kv;
    if ((long long)max_new * n_rep <= DECODE_ROWS) return Tile{DECODE_ROWS / n_rep, DECODE_KEYS, true};
    return Tile{2 * (TILE_ROWS / n_rep), TILE_KEYS, false};
}
inline long long max_items(int requests, int max_tokens, int tile_tokens) { return (long long)max_tokens / tile_tokens + requests; }
inline long long schedule_ints(long long items) { return SCHED_HEADER + ITEM_INTS * items + items + 1; }

}  // namespace khq_paged
