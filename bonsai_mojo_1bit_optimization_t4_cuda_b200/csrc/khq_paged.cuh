// khq_paged.cuh -- what the plan of a step over the paged cache and the attention kernels that run from it agree on.
#pragma once
#include <stdint.h>

namespace khq_paged {

// The schedule in device memory: for the chunk kernel and for the decode kernel where each worker begins, then a list of items (in the order
// of the requests); the attention runs over H_kv copies of a list, one kv head after the other.  Behind them the items' first key blocks
// counted through, where the plan has no room for them in shared memory.
struct alignas(16) Item {
    int b, n_blocks, ntok, kv;  // request; key blocks (causal: up to the tile's last token); new tokens of the tile; the request's tokens
    int row0, pos0, pad[2];     // the tile's first row in the ragged tensors, that row's position
};
constexpr int ITEM_INTS = sizeof(Item) / 4;
// Where a worker (a CTA of the decode kernel, a pair of the chunk kernel) begins its stretch: everything that its first loads need.
struct alignas(16) Start {
    Item it;
    int item, h, blk, n_items;  // blk: the item's first block in the stretch
    int length, share;          // from the item's begin to the stretch's end (0: nothing to do); the workers from this one on that share the item it ends in
    int pad[2];
};
constexpr int START_INTS = sizeof(Start) / 4, MAX_WORKERS = 256;
static_assert(START_INTS == 16, "four 16-byte loads");

// Query rows are (new token, query head of the kv head) pairs, token-major.  A request with up to 16 rows goes to the decode kernel, whose
// tile is the request's rows (the cache's bytes bound those, and a pair's 256 rows would be all but empty); one with more is cut
// into tiles of 2 x 128 rows, each for a CTA pair.
constexpr int MAX_REP = 128;  // query heads of a kv head
constexpr int DECODE_ROWS = 16, TILE_ROWS = 128, TILE_KEYS = 128;
constexpr int decode_keys(int d) { return 64 * 256 / d; }  // keys of a block of the decode kernel: 64 KB of K and V
// What an item costs beside its key blocks, in blocks: its queries, gates and outputs, and the pipe's run-in; the joining of the warps.  And how
// near to an item's ends its blocks are not divided between two pairs: 264 KB of partial rows from each of them would have to be written
// and read again.
// (4 x 8192 tokens: 2.79 ms with 3 blocks of a chunk's tile, 2.65 with 6; 40 single tokens over 2600 on average: 92 us with 0 of a decode
// item, 84 with 2.)
constexpr int CHUNK_OVER = 6, DECODE_OVER = 2, CHUNK_SNAP = 4;
struct Schedule {
    bool chunks, decodes;             // the lists that the step can have
    int tile_tokens, decode_tokens;   // new tokens of a tile; the most of a request for the decode kernel (0: none)
    int decode_keys;                  // keys of its blocks
    long long chunk_cap, decode_cap;  // items at most
    long long chunk_starts, decode_starts, chunk_items, chunk_cum, decode_items, decode_cum, ints;  // offsets in ints
};
inline Schedule schedule_of(int requests, int max_tokens, int max_new, int H_q, int H_kv, int d) {
    const int n_rep = H_q / H_kv;
    Schedule s;
    s.tile_tokens = 2 * (TILE_ROWS / n_rep);
    s.decode_tokens = DECODE_ROWS / n_rep;
    s.decode_keys = decode_keys(d);
    s.chunks = max_new > s.decode_tokens;
    s.decodes = s.decode_tokens > 0;
    s.chunk_cap = s.chunks ? (long long)max_tokens / s.tile_tokens + requests : 0;
    s.decode_cap = s.decodes ? requests : 0;
    s.chunk_starts = 0;
    s.decode_starts = s.chunk_starts + START_INTS * MAX_WORKERS;
    s.chunk_items = s.decode_starts + START_INTS * MAX_WORKERS;
    s.decode_items = s.chunk_items + ITEM_INTS * s.chunk_cap;
    s.chunk_cum = s.decode_items + ITEM_INTS * s.decode_cap;
    s.decode_cum = s.chunk_cum + s.chunk_cap + 1;
    s.ints = s.decode_cum + s.decode_cap + 1;
    return s;
}

}  // namespace khq_paged
