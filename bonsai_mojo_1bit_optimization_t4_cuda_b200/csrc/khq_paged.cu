// khq_paged.cu -- the plan of a step over a raw paged K/V cache, and the pre-step that fills the cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "khq_b200.h"
#include "khq_common.cuh"
#include "khq_launch.cuh"
#include "khq_paged.cuh"

namespace khq_paged {

// ---- the plan of a step --------------------------------------------------------------------------
// One cluster.  Every CTA sums up the lengths of all requests for itself (8 bytes a request) and keeps three running sums in shared
// memory: tokens, pages taken, pages given back.  From those any moved page is found by bisection: the pages of ended requests are
// read where they stand in their table rows, on top of the free ones.  The row of a request whose pages ran out once may have any mixture of
// pages and none.  Whoever meets an entry that is no page tells the cluster, and behind the barrier the ended rows' pages are
// counted, a warp per row, and moved once more (3172 requests, 100 ended rows of some 200 entries: counting them in every step cost 6 of 32 us).  Behind one barrier (the table is complete, the number of free pages has
// been read and may be overwritten) two CTAs cut the step into the attention's items and its workers' stretches, and the others write
// positions and slots.  Latency bounds it: a chain of some ten loads, scans and bisections (a bisection step in shared memory is 30 cycles,
// in global memory some 500).  256 requests with a token each: 7.5 us; 3172 requests with 130 355 tokens: 25.
constexpr int PLAN_THREADS = 1024, PLAN_CTAS = 8, PLAN_MAX_REQUESTS = 16384, PLAN_MAX_TOKENS = 1 << 20;

struct PlanArgs {
    const int *ctx_lens, *new_lens;
    int* table;
    long long table_stride;
    int* free_list;
    const int* free_count;
    int *free_count_out, *cu_new, *kv_lens, *positions;
    long long* slots;
    int *info, *schedule;
    int requests, max_pages, n_pages, page_shift, max_tokens, max_new, H_kv, workers, cum_in_smem;
    Schedule sched;
};

// An end of a worker's stretch: position `off` of the item, which has n blocks (off 0: where it begins).
struct Cut {
    int item, h, off, n, at;
};

// Inclusive sums of two ints over the block.  `part`: 2 x 32 ints.
__device__ __forceinline__ void block_scan2(int& a, int& b, int* part, int& total_a, int& total_b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xFFFFFFFFu, a, o), y = __shfl_up_sync(0xFFFFFFFFu, b, o);
        if (lane >= o) {
            a += x;
            b += y;
        }
    }
    __syncthreads();  // the last use of `part`
    if (lane == 31) {
        part[warp] = a;
        part[32 + warp] = b;
    }
    __syncthreads();
    int wa = part[lane], wb = part[32 + lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xFFFFFFFFu, wa, o), y = __shfl_up_sync(0xFFFFFFFFu, wb, o);
        if (lane >= o) {
            wa += x;
            wb += y;
        }
    }
    total_a = __shfl_sync(0xFFFFFFFFu, wa, 31);
    total_b = __shfl_sync(0xFFFFFFFFu, wb, 31);
    const int before_a = __shfl_sync(0xFFFFFFFFu, wa, (warp + 31) & 31), before_b = __shfl_sync(0xFFFFFFFFu, wb, (warp + 31) & 31);
    if (warp > 0) {
        a += before_a;
        b += before_b;
    }
}

// The page behind `skip` others in a table row that has more of them, eight entries at a time.
__device__ __forceinline__ int page_behind(const int* row, int held, int n_pages, int skip) {
    int found = -1;
    for (int i0 = 0; i0 < held && found < 0; i0 += 8) {
        int e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i0 + i < held ? row[i0 + i] : -1;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((unsigned)e[i] < (unsigned)n_pages && skip-- == 0) found = e[i];
    }
    return found;
}

// The last i in [0, n) with cum[i] <= x; cum[0] = 0 <= x < cum[n].
__device__ __forceinline__ int find(const int* cum, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __cluster_dims__(PLAN_CTAS, 1, 1) __launch_bounds__(PLAN_THREADS, 1) khq_paged_plan_kernel(const PlanArgs a) {
    extern __shared__ int sums[];  // tokens, pages taken, pages given back: requests + 1 running sums each
    __shared__ int part[64];
    __shared__ Cut cuts[MAX_WORKERS + 1];
    __shared__ int holes;                               // this CTA has met an entry that is no page in an ended request's row
    __shared__ unsigned mixed[PLAN_MAX_REQUESTS / 32];  // bit by request: it has ended, and its pages are not its row's first entries
    int *const cu = sums, *const taken = cu + a.requests + 1, *const back = taken + a.requests + 1;
    const int tid = threadIdx.x, rank = blockIdx.x, B = a.requests, page = 1 << a.page_shift;
    if (tid == 0) holes = 0;
    khq::pdl_wait();
    khq::pdl_trigger();
    const bool pool = a.free_list != nullptr;
    const int count = pool ? min(max(*a.free_count, 0), a.n_pages) : 0;
    // table pages that `tokens` tokens lie in
    const int row_tokens = a.max_pages << a.page_shift;  // 2^30 at most
    const auto pages = [&](int tokens) { return (tokens + page - 1) >> a.page_shift; };
    const auto ctx_of = [&](int b) { return min(max(a.ctx_lens[b], 0), row_tokens); };
    int sum_tok = 0, sum_taken = 0, sum_back = 0;
    long long dropped = 0;
    int ctx_next = tid < B ? ctx_of(tid) : 0, asked_next = tid < B ? a.new_lens[tid] : 0;
    for (int b0 = 0; b0 < B; b0 += PLAN_THREADS) {
        const int b = b0 + tid, ctx = ctx_next, asked = asked_next, n = min(min(max(asked, 0), a.max_new), row_tokens - ctx);
        if (b + PLAN_THREADS < B) {  // the next round's lengths are on their way
            ctx_next = ctx_of(b + PLAN_THREADS);
            asked_next = a.new_lens[b + PLAN_THREADS];
        } else {
            ctx_next = asked_next = 0;
        }
        int incl = min(n, a.max_tokens), unused = 0, total, u;  // sums of up to 2^10 terms of up to 2^20
        block_scan2(incl, unused, part, total, u);
        const int first = min(sum_tok + incl - min(n, a.max_tokens), a.max_tokens), end = min(sum_tok + incl, a.max_tokens);
        sum_tok = min(sum_tok + total, a.max_tokens);
        const int kept = end - first, held = pages(ctx);
        int t = b < B && pool && asked >= 0 ? pages(ctx + kept) - held : 0, r = b < B && pool && asked < 0 ? held : 0;
        const int mine_t = t, mine_r = r;
        int total_t, total_r;
        block_scan2(t, r, part, total_t, total_r);
        if (b < B) {
            cu[b] = first;
            taken[b] = sum_taken + t - mine_t;
            back[b] = sum_back + r - mine_r;
            if (rank == 0) {
                a.cu_new[b] = first;
                a.kv_lens[b] = asked < 0 ? 0 : ctx + kept;
                dropped += max(asked, 0) - kept;
            }
        }
        sum_taken += total_t;
        sum_back += total_r;
    }
    if (tid == 0) {
        cu[B] = sum_tok;
        taken[B] = sum_taken;
        back[B] = sum_back;
    }
    __syncthreads();
    // ---- table entries and the free list: the free pages with the ones given back on top; pages are taken from the top ----
    const bool some_back = sum_back > 0;
    bool counted = false;  // `back` counts pages; at first the entries of the rows
#pragma unroll 1
    for (;;) {
        const int stack = count + sum_back, at = rank * PLAN_THREADS + tid, step = PLAN_CTAS * PLAN_THREADS;
        const auto given_back = [&](int r) {
            const int b = find(back, B, r), nth = r - back[b];
            const int* row = a.table + b * a.table_stride;
            return counted && (mixed[b >> 5] >> (b & 31)) & 1u ? page_behind(row, pages(ctx_of(b)), a.n_pages, nth) : row[nth];
        };
        bool none = false;
        for (int j = at; j < sum_taken; j += step) {
            const int b = find(taken, B, j), i = stack - 1 - j;
            a.table[b * a.table_stride + pages(ctx_of(b)) + (j - taken[b])] = i < 0 ? -1 : i < count ? a.free_list[i] : given_back(i - count);
        }
        for (int r = at; r < sum_back; r += step) {
            const int page_no = given_back(r);
            none |= (unsigned)page_no >= (unsigned)a.n_pages;
            if (count + r < a.n_pages) a.free_list[count + r] = page_no;
        }
        if (none) holes = 1;
        __syncwarp();  // the cluster's barrier wants whole warps, and the loops above end lane by lane
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (rank == 0 && !counted) {
            // the sum of 2^10 x 16 counts below 2^31, in words of 21 bits
            int low = (int)(dropped & 0x1FFFFF), high = (int)(dropped >> 21), total_low, total_high;
            block_scan2(low, high, part, total_low, total_high);
            if (tid == 0) {
                a.cu_new[B] = sum_tok;
                a.info[0] = sum_tok;
                a.info[4] = (int)min(((long long)total_high << 21) + total_low, 0x7FFFFFFFLL);
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (counted || !some_back) break;
        int met = 0;
        if ((tid & 31) < PLAN_CTAS)
            asm volatile("{.reg .b32 p; mapa.shared::cluster.u32 p, %1, %2; ld.shared::cluster.u32 %0, [p];}" : "=r"(met) : "r"(khq::smem_u32(&holes)), "r"(tid & 31) : "memory");
        counted = __any_sync(0xFFFFFFFFu, met);
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // nobody's shared memory goes before it has been read
        if (!counted) break;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        sum_back = 0;
        for (int b0 = 0; b0 < B; b0 += PLAN_THREADS) {
            const int b = b0 + tid, held = b < B && a.new_lens[b] < 0 ? pages(ctx_of(b)) : 0;
            int r = 0, unused = 0, total, u;
            unsigned mix = 0;
            for (unsigned ended = __ballot_sync(0xFFFFFFFFu, held > 0); ended != 0; ended &= ended - 1) {
                const int who = __ffs(ended) - 1, n_held = __shfl_sync(0xFFFFFFFFu, held, who);
                const int* row = a.table + (b - (tid & 31) + who) * a.table_stride;
                int n = 0, last = -1;  // this lane's pages, the last one's place
#pragma unroll 8
                for (int i = tid & 31; i < n_held; i += 32)
                    if ((unsigned)row[i] < (unsigned)a.n_pages) {
                        ++n;
                        last = i;
                    }
                n = __reduce_add_sync(0xFFFFFFFFu, n);
                last = __reduce_max_sync(0xFFFFFFFFu, last);
                if ((tid & 31) == who) r = n;
                if (last >= n) mix |= 1u << who;
            }
            if ((tid & 31) == 0 && b < B) mixed[b >> 5] = mix;
            const int mine = r;
            block_scan2(r, unused, part, total, u);
            if (b < B) back[b] = sum_back + r - mine;
            sum_back += total;
        }
        if (tid == 0) back[B] = sum_back;
        __syncthreads();
    }
    // the pages' sums have done their work: in their place the requests' lengths, and the items' sums
    int *const ctx_lens = back, *const first_item = taken;
    for (int b = tid; b < B; b += PLAN_THREADS) ctx_lens[b] = ctx_of(b);
    if (rank < 2) {
        // ---- the items of the attention: the first CTA the chunks', the second the decodes' ----------------
        if (rank == 0 && tid == 0) {
            const int stack = count + sum_back;  // 0 without a pool
            const int left = pool ? min(max(stack - sum_taken, 0), a.n_pages) : 0;  // (a page that was free already makes one too many)
            a.info[1] = min(sum_taken, stack);
            a.info[2] = sum_back;
            a.info[3] = max(sum_taken - stack, 0);
            a.info[5] = left;
            a.info[6] = a.info[7] = 0;
            if (pool) *a.free_count_out = left;
        }
        const bool decodes = rank == 1;
        const int tile_tokens = decodes ? a.sched.decode_tokens : a.sched.tile_tokens, tile_keys = decodes ? a.sched.decode_keys : TILE_KEYS;
        int items = 0, u;
        for (int b0 = 0; b0 < B; b0 += PLAN_THREADS) {
            const int b = b0 + tid;
            int n = 0, z = 0, total;
            if (b < B) {
                const int kept = cu[b + 1] - cu[b];
                if (kept > 0 && (kept <= a.sched.decode_tokens) == decodes) n = (kept + tile_tokens - 1) / tile_tokens;
            }
            const int mine = n;
            block_scan2(n, z, part, total, u);
            if (b < B) first_item[b] = items + n - mine;
            items += total;
        }
        if (tid == 0) first_item[B] = items;
        __syncthreads();
        Item* const list = reinterpret_cast<Item*>(a.schedule + (decodes ? a.sched.decode_items : a.sched.chunk_items));
        int* const cum = a.cum_in_smem ? back + B + 1 : a.schedule + (decodes ? a.sched.decode_cum : a.sched.chunk_cum);
        int blocks = 0;
        for (int i0 = 0; i0 < items; i0 += PLAN_THREADS) {
            const int i = i0 + tid;
            Item it = {};
            if (i < items) {
                it.b = find(first_item, B, i);
                const int q0 = (i - first_item[it.b]) * tile_tokens, kept = cu[it.b + 1] - cu[it.b], ctx = ctx_lens[it.b];
                it.ntok = min(tile_tokens, kept - q0);
                it.n_blocks = (ctx + q0 + it.ntok + tile_keys - 1) / tile_keys;
                it.kv = ctx + kept;
                it.row0 = cu[it.b] + q0;
                it.pos0 = ctx + q0;
            }
            int n = it.n_blocks, z = 0, total;
            block_scan2(n, z, part, total, u);
            if (i < items) {
                list[i] = it;
                cum[i] = blocks + n - it.n_blocks;
            }
            blocks += total;
        }
        __syncthreads();
        // Each worker's stretch of the blocks of all kv heads: equal ones, but that an end which falls into an item's first or last `snap` blocks
        // goes to the item's.  No more workers than blocks, so that every worker between an item's first and last has some of it.
        const int over = decodes ? DECODE_OVER : CHUNK_OVER, snap = decodes ? 0 : CHUNK_SNAP;
        const int per_head = blocks + items * over, total = per_head * a.H_kv;  // (all in 32 bits: the launcher refuses what would not fit)
        const int most = decodes ? a.workers : a.workers / 2, workers = min(most, total);
        const int share = workers > 0 ? total / workers : 0, larger = total - share * workers;
        const auto end_of = [&](int k) { return k * share + k * larger / workers; };  // of the first k workers: k total / workers, rounded down
        Start* const starts = reinterpret_cast<Start*>(a.schedule + (decodes ? a.sched.decode_starts : a.sched.chunk_starts));
        if (tid <= workers) {
            const int v = workers > 0 ? end_of(tid) : 0;
            Cut c = {0, 0, 0, 0, v};
            if (v < total) {
                c.h = v / per_head;
                const int r = v - c.h * per_head;
                int lo = 0, up = items;  // the last item that begins at r or in front
                while (up - lo > 1) {
                    const int mid = (lo + up) >> 1;
                    if (cum[mid] + mid * over <= r) lo = mid;
                    else up = mid;
                }
                c.item = lo;
                c.n = (lo + 1 < items ? cum[lo + 1] : blocks) - cum[lo];
                c.off = r - cum[lo] - lo * over;
                const int blk = max(c.off - over, 0), rest = c.n - blk;
                if (blk == 0 || (blk < snap && blk <= rest)) {
                    c.at -= c.off;
                    c.off = 0;
                } else if (rest < snap) {
                    c.at += rest;
                    c.off = 0;
                    if (++c.item == items) {
                        c.item = 0;
                        ++c.h;
                    }
                }
            }
            cuts[tid] = c;
        }
        __syncthreads();
        if (tid < most) {
            Start st = {};
            if (tid < workers) {
                const Cut from = cuts[tid], to = cuts[tid + 1];
                if (from.at < to.at) {
                    st.it = list[from.item];
                    st.item = from.item;
                    st.h = from.h;
                    st.blk = max(from.off - over, 0);
                    st.n_items = items;
                    st.length = to.at - (from.at - from.off);
                    if (to.off > 0) {  // the first cut behind the item's last undivided block ends it
                        const int end = to.at - to.off + over + (snap > 0 ? to.n - snap + 1 : to.n);
                        int k = min(max((int)((float)end / (float)total * (float)workers) - 1, tid + 1), workers);
                        while (end_of(k) < end) ++k;
                        while (end_of(k - 1) >= end) --k;
                        st.share = k - tid;
                    }
                }
            }
            starts[tid] = st;
        }
    } else {
        // ---- positions and slots: four tokens a thread, one bisection, and four table entries on their way at once ----
        __syncthreads();
        const int at = (rank - 2) * PLAN_THREADS + tid, step = (PLAN_CTAS - 2) * PLAN_THREADS;
        for (int t0 = 4 * at; t0 < a.max_tokens; t0 += 4 * step) {
            int b = t0 < sum_tok ? find(cu, B, t0) : B - 1;
            int pos[4], page_of[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + i;
                while (t < sum_tok && cu[b + 1] <= t) ++b;
                pos[i] = t < sum_tok ? ctx_lens[b] + (t - cu[b]) : -1;
                const int col = pos[i] >> a.page_shift;
                page_of[i] = t < sum_tok ? a.table[b * a.table_stride + col] : -1;
            }
            long long slot[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) slot[i] = page_of[i] >= 0 ? ((long long)page_of[i] << a.page_shift) + (pos[i] & (page - 1)) : -1;
            if (t0 + 4 <= a.max_tokens) {
                *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
                *reinterpret_cast<longlong2*>(a.slots + t0) = make_longlong2(slot[0], slot[1]);
                *reinterpret_cast<longlong2*>(a.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    if (t0 + i >= a.max_tokens) break;
                    a.positions[t0 + i] = pos[i];
                    a.slots[t0 + i] = slot[i];
                }
            }
        }
    }
    if (some_back && !counted) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// ---- the pre-step ------------------------------------------------------------------------------------
// Per head: x / sqrt(mean(x^2) + eps) * w, then the rotation of the pairs (i, i + r/2), i < r/2, by pos * theta^(-2i/r).  In fp32, one
// rounding to 16 bits where a value is stored (the rotated K is not made from the rounded un-rotated one).  The angle is
// formed in fp64 and reduced there: at position 2^18 an fp32 product would be off by 2^-7.
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
}

constexpr int PRE_WARPS = 8, MAX_PAIRS = 128;
struct PrestepArgs {
    khq_paged_prestep_args a;
    double freq[MAX_PAIRS];  // theta^(-2i/r) / 2 pi: turns per position
    int page_shift;
};

// Packed pairs of fp32, one instruction each.
__device__ __forceinline__ void mul2(float (&x)[8], int e, float a, float b) {
    asm("{.reg .b64 p, q; mov.b64 p, {%0, %1}; mov.b64 q, {%2, %3}; mul.rn.f32x2 p, p, q; mov.b64 {%0, %1}, p;}" : "+f"(x[e]), "+f"(x[e + 1]) : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1) {  // d += a b
    asm("{.reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 d, {%0, %1}; fma.rn.f32x2 d, a, b, d; mov.b64 {%0, %1}, d;}"
        : "+f"(d0), "+f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// A CTA takes a token, or a part of its heads; the heads of q, then of k, then of v, 8 values (16 bytes) a lane, so d / 8 lanes a head.  The
// token's bytes bound it: all of a warp's HEADS heads are on their way while the first threads form the cosines and sines.  With a pass
// over scalars for every head, v's too, it was instructions (190 a head: 8192 tokens
// 77 us, now 62, 4.6 TB/s).
template <int D, bool BF16, int HEADS>
__global__ void __launch_bounds__(PRE_WARPS * 32, 4) khq_paged_prestep_kernel(const __grid_constant__ PrestepArgs p) {
    constexpr int LANES = D / 8, PER = PRE_WARPS * 32 / LANES;
    __shared__ float2 turn[MAX_PAIRS];
    const khq_paged_prestep_args& a = p.a;
    const int lane = threadIdx.x % LANES, first = blockIdx.y * (PER * HEADS) + threadIdx.x / LANES, heads = a.H_q + 2 * a.H_kv;
    const long long t = blockIdx.x;
    const int n_pairs = a.rotary_dim / 2, half_lanes = a.rotary_dim / 16;
    khq::pdl_wait();
    khq::pdl_trigger();
    const int pos = static_cast<const int*>(a.positions)[t];
    long long slot = static_cast<const long long*>(a.slots)[t];
    const uint16_t* const q = static_cast<const uint16_t*>(a.q) + t * a.q_stride[0] + lane * 8;
    const uint16_t* const k = static_cast<const uint16_t*>(a.k) + t * a.k_stride[0] + lane * 8;
    const uint16_t* const v = static_cast<const uint16_t*>(a.v) + t * a.v_stride[0] + lane * 8;
    uint4 raw[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = first + i * PER, hk = h - a.H_q, hv = hk - a.H_kv;
        const uint16_t* src = hk < 0 ? q + h * a.q_stride[1] : hv < 0 ? k + hk * a.k_stride[1] : v + hv * a.v_stride[1];
        raw[i] = h < heads ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
    }
    if (pos < 0) return;  // behind the last token
    if (slot >= (long long)a.n_pages << p.page_shift) slot = -1;
    if (threadIdx.x < n_pairs) {
        double turns = (double)pos * p.freq[threadIdx.x];
        turns -= rint(turns);
        float s, c;
        sincospif((float)(2.0 * turns), &s, &c);
        turn[threadIdx.x] = make_float2(c, s);
    }
    __syncthreads();
    // the rotary pair of value e of lane l is value e of lane l +- half_lanes; x cos + y sin with the sign on the lower lane's sine, and cosine 1,
    // sine 0 where nothing is rotated
    const bool low = lane < half_lanes, turned = lane < 2 * half_lanes;
    const int partner = low ? lane + half_lanes : turned ? lane - half_lanes : lane;
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float2 f = turned ? turn[(low ? lane : partner) * 8 + e] : make_float2(1.0f, 0.0f);
        cs[e] = f.x;
        sn[e] = low ? -f.y : f.y;
    }
    const long long pg = slot >> p.page_shift, at = slot & (a.page_size - 1);
    const auto cache_row = [&](void* base, const int64_t (&st)[3], int h) {
        return reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + pg * st[0] + at * st[1] + h * st[2] + lane * 8);
    };
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = first + i * PER, hk = h - a.H_q, hv = hk - a.H_kv;
        if (__all_sync(0xFFFFFFFFu, hv >= 0)) {  // whole warps: at d 128 one has two heads
            if (h < heads && slot >= 0) *cache_row(a.v_cache, a.v_cache_stride, hv) = raw[i];
            continue;
        }
        const uint32_t rw[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        float x[8], sq[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2<BF16>(rw[e]);
            x[2 * e] = f.x;
            x[2 * e + 1] = f.y;
            fma2(sq[0], sq[1], f.x, f.y, f.x, f.y);
        }
        float sum = sq[0] + sq[1];
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o, LANES);
        const float inv = rsqrtf(sum * (1.0f / D) + a.rms_eps);
        const float* w = static_cast<const float*>(hk < 0 ? a.q_norm_w : a.k_norm_w);
#pragma unroll
        for (int e = 0; e < 8; e += 2) mul2(x, e, inv, inv);
        if (w) {
            const float4 w0 = __ldg(reinterpret_cast<const float4*>(w + lane * 8)), w1 = __ldg(reinterpret_cast<const float4*>(w + lane * 8) + 1);
            mul2(x, 0, w0.x, w0.y);
            mul2(x, 2, w0.z, w0.w);
            mul2(x, 4, w1.x, w1.y);
            mul2(x, 6, w1.z, w1.w);
        }
        if (hk >= 0 && hv < 0 && slot >= 0 && a.u_cache) *cache_row(a.u_cache, a.u_cache_stride, hk) = pack8<BF16>(x);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xFFFFFFFFu, x[e], partner, LANES);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            mul2(x, e, cs[e], cs[e + 1]);
            fma2(x[e], x[e + 1], y[e], y[e + 1], sn[e], sn[e + 1]);
        }
        const uint4 res = pack8<BF16>(x);
        if (hk < 0) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.q_out) + t * a.q_out_stride[0] + h * a.q_out_stride[1] + lane * 8) = res;
        else if (hv < 0 && slot >= 0) *cache_row(a.k_cache, a.k_cache_stride, hk) = res;
        else if (h < heads && slot >= 0) *cache_row(a.v_cache, a.v_cache_stride, hv) = raw[i];
    }
}

int log2_page(int page_size) {
    return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : -1;
}

int launch_prestep(const khq_paged_prestep_args* args, bool bf16, cudaStream_t stream) {
    if (!args) return -100;
    const khq_paged_prestep_args& a = *args;
    if (a.tokens <= 0 || a.H_q <= 0 || a.H_kv <= 0 || a.n_pages <= 0 || !a.q || !a.k || !a.v || !a.q_out || !a.k_cache || !a.v_cache || !a.slots || !a.positions)
        return -100;
    if (!(a.rope_theta > 0.0f) || !(a.rms_eps >= 0.0f)) return -100;
    if ((a.d != 128 && a.d != 256) || a.rotary_dim < 0 || a.rotary_dim > a.d || a.rotary_dim % 16 != 0 || log2_page(a.page_size) < 0) return -103;
    const void* ptrs[] = {a.q, a.k, a.v, a.q_out, a.k_cache, a.v_cache, a.u_cache, a.q_norm_w, a.k_norm_w};
    for (const void* q : ptrs)
        if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return -104;
    if ((reinterpret_cast<uintptr_t>(a.slots) & 7) != 0 || (reinterpret_cast<uintptr_t>(a.positions) & 3) != 0) return -104;
    for (int i = 0; i < 2; ++i)
        if (((a.q_stride[i] | a.k_stride[i] | a.v_stride[i] | a.q_out_stride[i]) & 7) != 0) return -104;
    for (int i = 0; i < 3; ++i)
        if (((a.k_cache_stride[i] | a.v_cache_stride[i] | (a.u_cache ? a.u_cache_stride[i] : 0)) & 7) != 0) return -104;
    PrestepArgs p;
    p.a = a;
    p.page_shift = log2_page(a.page_size);
    for (int i = 0; i < MAX_PAIRS; ++i)
        p.freq[i] = i < a.rotary_dim / 2 ? pow((double)a.rope_theta, -2.0 * i / a.rotary_dim) / 6.283185307179586476925 : 0.0;
    const auto launch = [&](auto kernel, int per_cta) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)a.tokens, (unsigned)((a.H_q + 2 * a.H_kv + per_cta - 1) / per_cta), 1);
        cfg.blockDim = dim3(PRE_WARPS * 32, 1, 1);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
    };
    // Few tokens: a head per warp, so that a token's heads are spread over more SMs.  Many: four, so that its angles are formed once or
    // twice and more bytes are in flight.
    const int per_warp = a.d == 256 ? 1 : 2, wide = a.tokens >= 2 * khq::sm_count() ? 4 : 1;
    const int per_cta = PRE_WARPS * per_warp * wide;
    if (a.d == 256) {
        if (wide == 4) return bf16 ? launch(khq_paged_prestep_kernel<256, true, 4>, per_cta) : launch(khq_paged_prestep_kernel<256, false, 4>, per_cta);
        return bf16 ? launch(khq_paged_prestep_kernel<256, true, 1>, per_cta) : launch(khq_paged_prestep_kernel<256, false, 1>, per_cta);
    }
    if (wide == 4) return bf16 ? launch(khq_paged_prestep_kernel<128, true, 4>, per_cta) : launch(khq_paged_prestep_kernel<128, false, 4>, per_cta);
    return bf16 ? launch(khq_paged_prestep_kernel<128, true, 1>, per_cta) : launch(khq_paged_prestep_kernel<128, false, 1>, per_cta);
}

}  // namespace khq_paged

extern "C" size_t khq_b200_paged_schedule_bytes(int requests, int max_tokens, int max_new, int H_q, int H_kv, int d) {
    using namespace khq_paged;
    if (requests <= 0 || max_tokens <= 0 || max_new <= 0 || H_q <= 0 || H_kv <= 0 || H_q % H_kv != 0 || H_q / H_kv > MAX_REP || (d != 128 && d != 256)) return 0;
    return (size_t)schedule_of(requests, max_tokens, max_new, H_q, H_kv, d).ints * 4;
}

extern "C" int launch_khq_paged_plan(const khq_paged_plan_args* args, khq_stream_t stream) {
    using namespace khq_paged;
    if (!args) return -100;
    const khq_paged_plan_args& p = *args;
    if (p.requests <= 0 || p.max_tokens <= 0 || p.max_new <= 0 || p.max_pages <= 0 || p.H_q <= 0 || p.H_kv <= 0 || !p.ctx_lens || !p.new_lens || !p.block_table ||
        !p.cu_new || !p.kv_lens || !p.positions || !p.slots || !p.info || !p.schedule)
        return -100;
    if (p.free_list ? (p.n_pages <= 0 || !p.free_count || !p.free_count_out) : (p.free_count || p.free_count_out)) return -100;
    const int shift = log2_page(p.page_size);
    if (shift < 0 || (p.d != 128 && p.d != 256) || p.H_q % p.H_kv != 0 || p.H_q / p.H_kv > MAX_REP || p.requests > PLAN_MAX_REQUESTS || p.max_tokens > PLAN_MAX_TOKENS ||
        (long long)p.requests * p.max_pages > 0x7FFFFFFFLL || p.table_stride < p.max_pages || (long long)p.max_pages << shift > (1LL << 30))
        return -103;
    const void* ptrs[] = {p.ctx_lens, p.new_lens, p.block_table, p.free_list, p.free_count, p.free_count_out, p.cu_new, p.kv_lens, p.positions, p.info};
    for (const void* q : ptrs)
        if ((reinterpret_cast<uintptr_t>(q) & 3) != 0) return -104;
    for (const void* q : {static_cast<const void*>(p.positions), static_cast<const void*>(p.slots), static_cast<const void*>(p.schedule)})
        if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return -104;
    const Schedule sched = schedule_of(p.requests, p.max_tokens, p.max_new, p.H_q, p.H_kv, p.d);
    if (p.schedule_bytes < (size_t)sched.ints * 4) return -105;
    // the key blocks of all items and kv heads are counted in 32 bits
    const long long row = ((long long)p.max_pages << shift) + p.max_tokens;
    if (sched.chunk_cap * (row / TILE_KEYS + 1 + CHUNK_OVER) > 0x7FFFFFFFLL / p.H_kv || sched.decode_cap * (row / sched.decode_keys + 1 + DECODE_OVER) > 0x7FFFFFFFLL / p.H_kv) return -103;
    PlanArgs a;
    a.ctx_lens = static_cast<const int*>(p.ctx_lens);
    a.new_lens = static_cast<const int*>(p.new_lens);
    a.table = static_cast<int*>(p.block_table);
    a.table_stride = p.table_stride;
    a.free_list = static_cast<int*>(p.free_list);
    a.free_count = static_cast<const int*>(p.free_count);
    a.free_count_out = static_cast<int*>(p.free_count_out);
    a.cu_new = static_cast<int*>(p.cu_new);
    a.kv_lens = static_cast<int*>(p.kv_lens);
    a.positions = static_cast<int*>(p.positions);
    a.slots = static_cast<long long*>(p.slots);
    a.info = static_cast<int*>(p.info);
    a.schedule = static_cast<int*>(p.schedule);
    a.requests = p.requests;
    a.max_pages = p.max_pages;
    a.n_pages = p.n_pages;
    a.page_shift = shift;
    a.max_tokens = p.max_tokens;
    a.max_new = p.max_new;
    a.H_kv = p.H_kv;
    a.workers = khq::sm_count() < MAX_WORKERS ? khq::sm_count() : MAX_WORKERS;
    a.sched = sched;
    // the items' sums in shared memory too, where there is room
    constexpr size_t room = (size_t)3 * (PLAN_MAX_REQUESTS + 1) * 4;
    size_t smem = (size_t)3 * (p.requests + 1) * 4;
    const size_t cum = (size_t)(sched.chunk_cap > sched.decode_cap ? sched.chunk_cap : sched.decode_cap) * 4;
    a.cum_in_smem = smem + cum <= room;
    if (a.cum_in_smem) smem += cum;
    static bool attr_done[64] = {};
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return static_cast<int>(err);
    if (dev < 0 || dev >= 64) return -100;
    if (!attr_done[dev]) {
        err = cudaFuncSetAttribute((const void*)khq_paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room);
        if (err != cudaSuccess) return static_cast<int>(err);
        attr_done[dev] = true;
    }
    err = khq::launch_pdl(khq_paged_plan_kernel, (unsigned)PLAN_CTAS, 0, smem, stream, (unsigned)PLAN_THREADS, a);
    return static_cast<int>(err);
}

extern "C" int launch_khq_paged_prestep_fp16(const khq_paged_prestep_args* args, khq_stream_t stream) {
    return khq_paged::launch_prestep(args, false, stream);
}

extern "C" int launch_khq_paged_prestep_bf16(const khq_paged_prestep_args* args, khq_stream_t stream) {
    return khq_paged::launch_prestep(args, true, stream);
}
