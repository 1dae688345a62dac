// khq_paged.cuh -- what the plan of a step over the paged cache and the attention kernels that run from it agree on.
#pragma once
#include <stdint.h>

namespace khq_paged {

// The schedule in device memory: a header of 16 ints, the items (one per request and query tile, request by request), and the
// items' first key blocks counted through (cum[n_items] = the total).  The attention runs over H_kv copies of that list, one kv
// head after the other.
constexpr int SCHED_HEADER = 16;  // ints: [0] items, [1] key blocks of one kv head
struct Item {
    int b, q0, ntok, n_blocks;  // request; first of its new tokens; new tokens of the tile; key blocks (causal)
};

// Query rows are (new token, query head of the kv head) pairs, token-major.  A tile of the decode kernel has up to 16 rows, one
// of the prompt kernel two times up to 128.
constexpr int MAX_REP = 16;   // query heads of a kv head
constexpr int DECODE_ROWS = 16, DECODE_KEYS = 64;
struct Tile {
    int tokens, keys;  // new tokens of a query tile, keys of a block
    bool decode;
};
inline Tile tile_of(int H_q, int H_kv, int max_new) {
    (void)max_new;
    const int n_rep = H_q / H_kv;
    return Tile{DECODE_ROWS / n_rep, DECODE_KEYS, true};
}
inline long long max_items(int requests, int max_tokens, int tile_tokens) { return (long long)max_tokens / tile_tokens + requests; }
inline long long schedule_ints(long long items) { return SCHED_HEADER + 4 * items + items + 1; }

}  // namespace khq_paged
