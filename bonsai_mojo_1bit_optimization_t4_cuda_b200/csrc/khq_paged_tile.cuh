// khq_paged_tile.cuh -- attention over the paged cache for chunks of new tokens, on CTA pairs (tcgen05 cta_group::2).  Included by
// khq_paged_attn.cu.
//
// A tile is up to 2 x 128 query rows of one kv head: the (new token, query head) pairs of 2 x (128 / n_rep) tokens, token-major, 128 rows
// a CTA.  So a chunk of 21 tokens with six heads per kv head fills a CTA's rows instead of 1/6 of six tiles, and a tile's rows attend almost the same keys.
// Per block of 128 keys the pair computes S = Q K^T (M 256) and O += P V, each CTA keeping half of the K block (64 keys) and half of
// the V block (d / 2 head dims).  As in khq_prefill_pair.cuh, whose comments give the reasons: two groups of four softmax warps take the blocks in turn, a
// thread per row; P goes back over S in tensor memory in two halves; O is rescaled only when a maximum has grown by 2^8.  P is of
// 16 bits, V's type in the instruction, as everywhere in the prompt kernels (half a step of it of sum w |v|); the weights' sum is of the fp32 values.
//
// Work: the key blocks of all (kv head, item) pairs stand in one row and each CTA pair takes an equal stretch of it, so any mix of chunks and
// single tokens is even.  A segment that begins or ends inside a pair's stretch leaves records, which khq_paged_merge_kernel
// joins in a fixed order.  (One item per pair instead leaves a chunk of 2048 tokens, 196 items, 2.65 rounds of 74 pairs.)
//
// Pages: the tensor map of a cache is {64 values, token of a page, column group, head, page}; a page's piece of a block is one
// box (all column groups) when it fills the block, else one per column group.  The 128-byte swizzle depends on the address only,
// so pieces of 16 rows and more stand together as one operand.  Rows of V behind a request's last token may hold anything, and a
// weight of 0 does not undo a NaN: in the one block per request that has some, the V producer waits for its rows and overwrites them
// with zeros before it hands them on.
#pragma once

namespace khq_paged {
namespace tile {

constexpr int BR = 128, BC = 128;            // query rows of a CTA, keys of a block
constexpr int NSOFT = 256, NTHREADS = NSOFT + 128;  // warp 11 has no work: registers are split by groups of four warps
constexpr uint32_t TM_COLS = 512;            // O from column 0, the S buffers behind it
constexpr float RESCALE_LOG2 = 8.0f;
constexpr int STG_BYTES = 32 * 64;           // per softmax warp: 32 rows x 32 columns
constexpr int MAX_STAGES = 4;
enum Bar {  // K and V by stage, S by buffer, P V by block parity
    B_KFULL = 0, B_KFREE = 4, B_VFULL = 8, B_VFREE = 12, B_SFULL = 16, B_PVDONE = 19, B_PREADY = 21 /* [buffer][half of the keys] */, B_QFULL = 27, B_QFREE = 28,
    B_PEER = 29, B_MREF = 30 /* [group][lane quarter] */, B_LSUM = 38 /* [lane quarter] */, B_OFREE = 42, B_VLAND = 43, B_COUNT = 44
};
template <int D> struct Shape {
    static constexpr int G = D / 64;               // column groups
    // K and V blocks in flight: what fits.  Few query rows leave the cache's latency and bytes as the bound.
    static constexpr int STAGES = D == 256 ? 2 : 4;
    // Score buffers: what tensor memory has room for.  With three, Q K^T runs two blocks ahead of P V, and a softmax group has its next block's scores
    // when it is done with one (at d 128 the softmax is the longer part of a block).
    static constexpr int BUFFERS = D == 256 ? 2 : 3, AHEAD = BUFFERS - 1;
    static constexpr uint32_t TM_S = D;
    static_assert(TM_S + BUFFERS * BC <= TM_COLS, "tensor memory");
    static constexpr int Q_BYTES = BR * D * 2, TILE_BYTES = 64 * D * 2;  // a CTA's rows; its share of a K or V block
    static constexpr int OFF_Q = 0, OFF_K = OFF_Q + Q_BYTES, OFF_V = OFF_K + STAGES * TILE_BYTES, OFF_STG = OFF_V + STAGES * TILE_BYTES;
    static constexpr int OFF_MREF = OFF_STG + 8 * STG_BYTES;  // float [2 groups][128 rows]: the reference behind the group's last block
    static constexpr int OFF_LSUM = OFF_MREF + 2 * 128 * 4;   // float [segment parity][2 groups][128 rows]
    static constexpr int OFF_BARS = OFF_LSUM + 4 * 128 * 4, OFF_SLOT = OFF_BARS + B_COUNT * 8, SMEM = OFF_SLOT + 16;
    static_assert(STAGES <= MAX_STAGES && SMEM <= 227 * 1024, "shared memory");
    // A CTA's record: its rows [4 columns][128 rows][4 floats], so that a thread per row writes whole lines, then (maximum, sum) by row.
    static constexpr int RECORD = BR * D + 2 * BR;
};

// Wait at cluster scope: what the other CTA wrote with ordinary stores before it arrived is visible.
__device__ __forceinline__ bool warp_wait_cluster(uint64_t* bar, uint32_t parity, int* status) {
    return bounded([&] {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        return ok != 0;
    }, [](bool x) { return __any_sync(0xFFFFFFFFu, x) != 0; }, status);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {  // all lanes go on together
    return bounded([&] { return khq::mbar_try_wait(bar, parity); }, [](bool x) { return __any_sync(0xFFFFFFFFu, x) != 0; }, status);
}
__device__ __forceinline__ void arrive_leader_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.release.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(in_leader(bar)), "r"(bytes) : "memory");
}
// What this warp stored before is visible to who waits at cluster scope.  (An arrival says nothing of that beyond its own CTA otherwise.)
__device__ __forceinline__ void release_to_leader(uint64_t* bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(bar)) : "memory");
}
// The page numbers of a segment's blocks, 32 / per_block blocks in the lanes and as many on their way.  A block has `per_block` pages
// (pages of 128 tokens and less).  n_pages stands for a page that is not there: a copy from it fills in zeros.
struct Pages {
    int now, next, at;
    __device__ __forceinline__ int fetch(const Params& p, const Segment& s, int blk, int log_per) const {
        const int lane = threadIdx.x & 31, col = (blk << log_per) + lane;
        int pg = p.n_pages;
        if (((long long)col << p.page_shift) < s.kv && col < p.max_pages) {
            pg = __ldg(p.table + s.b * p.table_stride + col);
            if ((unsigned)pg >= (unsigned)p.n_pages) pg = p.n_pages;
        }
        return pg;
    }
    __device__ __forceinline__ void begin(const Params& p, const Segment& s, int blk, int log_per) {
        at = blk;
        now = fetch(p, s, blk, log_per);
        next = fetch(p, s, blk + (32 >> log_per), log_per);
    }
    // lane offset of the block's first page
    __device__ __forceinline__ int seek(const Params& p, const Segment& s, int blk, int log_per) {
        if (blk - at >= (32 >> log_per)) {
            at += 32 >> log_per;
            now = next;
            next = fetch(p, s, at + (32 >> log_per), log_per);
        }
        return (blk - at) << log_per;
    }
};

// The pair's segments one after the other, as every role walks them.  Positions count the CHUNK_OVER blocks in front of every item.
struct Walk {
    int left, share;  // from where the segment's item begins to the stretch's end; the pairs that share the item there
    int n;            // its blocks in this stretch
    Segment s;
    __device__ __forceinline__ bool begin(const Params& p, int& n_items) {
        if (!first_segment(p, blockIdx.x >> 1, s, n_items, left, share)) return false;
        count();
        return n > 0;
    }
    __device__ __forceinline__ void count() { n = min(s.n_blocks, left - CHUNK_OVER) - s.blk; }
    __device__ __forceinline__ bool more() const { return s.n_blocks + 2 * CHUNK_OVER < left; }
    __device__ __forceinline__ void step_to(const Segment& next) {
        left -= s.n_blocks + CHUNK_OVER;
        s = next;
        count();
    }
    __device__ __forceinline__ bool step(const Params& p, int n_items) {
        if (!more()) return false;
        Segment next = s;
        next_segment(p, n_items, next);
        step_to(next);
        return true;
    }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(NTHREADS, 1)
khq_paged_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ Params p) {
    using S = Shape<D>;
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BARS);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + S::OFF_SLOT);
    float* const mref = reinterpret_cast<float*>(smem + S::OFF_MREF);
    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const int rank = (int)(blockIdx.x & 1);  // the pair's first CTA has the MMA warp
    int* const status = &g_paged_status;
    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled layouts need a 1024-byte aligned base; the same in both CTAs
        khq::pdl_wait();
        if (tid == 0) {
            atomicExch(status, 2);
            p.meta[blockIdx.x >> 1].n = 0;
        }
        return;
    }
    const int tok = BR / p.n_rep, rows = tok * p.n_rep;  // new tokens and query rows of a CTA
    if (tid == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            khq::mbar_init(&bars[B_KFULL + s], 1);
            khq::mbar_init(&bars[B_KFREE + s], 1);
            khq::mbar_init(&bars[B_VFULL + s], 2);  // the V producers of both CTAs
            khq::mbar_init(&bars[B_VFREE + s], 1);
        }
        for (int s = 0; s < 2; ++s) khq::mbar_init(&bars[B_PVDONE + s], 1);
        for (int s = 0; s < S::BUFFERS; ++s) khq::mbar_init(&bars[B_SFULL + s], 1);
        khq::mbar_init(&bars[B_QFULL], 1);
        khq::mbar_init(&bars[B_QFREE], 1);
        khq::mbar_init(&bars[B_PEER], 1);
        khq::mbar_init(&bars[B_VLAND], 1);
        khq::mbar_init(&bars[B_OFREE], 2 * NSOFT / 32);
        // one elected arrival per softmax warp of both CTAs: separate arrivals on one barrier serialise
        for (int q = 0; q < 2 * S::BUFFERS; ++q) khq::mbar_init(&bars[B_PREADY + q], 2 * NSOFT / 64);
        for (int q = 0; q < 4; ++q) khq::mbar_init(&bars[B_LSUM + q], 2);  // the two warps of a lane quarter
        for (int q = 0; q < 8; ++q) khq::mbar_init(&bars[B_MREF + q], 1);
        khq::fence_barrier_init();
    } else if (warp == 8 && lane < 3) {
        prefetch_map(lane == 0 ? &tm_q : lane == 1 ? &tm_k : &tm_v);
    }
    // query rows that no token has (128 is not a multiple of n_rep): zero, or their scores would ask for rescaling
    for (int i = tid; i < S::G * (BR - rows) * 8; i += NTHREADS) {
        const int g = i / ((BR - rows) * 8), j = i % ((BR - rows) * 8);
        *reinterpret_cast<uint4*>(smem + S::OFF_Q + (g * BR + rows) * 128 + j * 16) = make_uint4(0, 0, 0, 0);
    }
    khq::fence_proxy_async();
    __syncwarp();
    cluster_arrive();
    cluster_wait();  // the barriers of both CTAs are there
    // Everything above overlaps the kernel before; tensor memory is only taken once that kernel has finished (it may still have
    // to allocate its own on this SM).
    khq::pdl_wait();
    khq::pdl_trigger();
    const uint32_t sbase = smem_u32(smem);
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(TM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    // tensor memory is there; the loads do not wait for that
    if (warp == 8 || warp >= 10) asm volatile("bar.arrive 1, %0;" ::"n"(NTHREADS) : "memory");
    else asm volatile("bar.sync 1, %0;" ::"n"(NTHREADS) : "memory");
    tc_fence_after();

    int n_items = 0;
    const int log_per = 7 - p.page_shift;  // pages of a block
    Walk walk;
    // 384 threads start with 168 registers each; the softmax threads, who hold 128 scores, take 208 and leave the others 88: together
    // the same 64512.  (Behind a point where both come together the compiler counts on the smaller number.)
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            // ================================ producer of Q and K: the CTA's 64 keys of a block as [group][64 keys][128 B] =============
            // boxes: 64 keys x all groups, or page x one group
            const int per_half = p.page_shift >= 6 ? 1 : 1 << (6 - p.page_shift), boxes = p.page_shift >= 6 ? 1 : per_half * S::G;
            int g = 0, i = 0;
            bool ok = true;
            Pages pages;
            for (bool more = walk.begin(p, n_items); ok && more; more = walk.step(p, n_items), ++i) {
                if (i > 0 && !(ok = tile::warp_wait(&bars[B_QFREE], (uint32_t)((i - 1) & 1), status))) break;
                if (lane == 0) {
                    if (rank == 0) khq::mbar_arrive_expect_tx(&bars[B_QFULL], 2u * (uint32_t)(rows * 128 * S::G));
#pragma unroll
                    for (int c = 0; c < S::G; ++c)
                        asm volatile(
                            "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
                                sbase + S::OFF_Q + c * (BR * 128)),
                            "l"(reinterpret_cast<uint64_t>(&tm_q)), "r"(in_leader(&bars[B_QFULL])), "r"(0), "r"(walk.s.h * p.n_rep), "r"(walk.s.row0 + rank * tok),
                            "r"(c)
                            : "memory");
                }
                pages.begin(p, walk.s, walk.s.blk, log_per);
                const bool ahead = walk.more();  // the next segment's queries to L2: their load waits for this one's last Q K^T
                Segment next = walk.s;
                if (ahead) next_segment(p, n_items, next);
                for (int j = 0; j < walk.n; ++j, ++g) {
                    if (j == 0 && ahead && lane < S::G)
                        asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(reinterpret_cast<uint64_t>(&tm_q)), "r"(0),
                                     "r"(next.h * p.n_rep), "r"(next.row0 + rank * tok), "r"(lane)
                                     : "memory");
                    const int s = g % S::STAGES, blk = walk.s.blk + j;
                    const int at = pages.seek(p, walk.s, blk, log_per);
                    // the page of this lane's box: keys rank * 64 + (lane / groups) pages further
                    const int mine = p.page_shift >= 6 ? at + ((rank * 64) >> p.page_shift) : at + rank * per_half + lane / S::G;
                    const int page = __shfl_sync(0xFFFFFFFFu, pages.now, mine & 31);
                    if (g >= S::STAGES && !(ok = tile::warp_wait(&bars[B_KFREE + s], (uint32_t)((g / S::STAGES - 1) & 1), status))) break;
                    if (rank == 0 && lane == 0) khq::mbar_arrive_expect_tx(&bars[B_KFULL + s], 2 * S::TILE_BYTES);
                    __syncwarp();
                    if (lane < boxes) {
                        const int piece = lane / S::G, c = p.page_shift >= 6 ? 0 : lane % S::G;
                        load_for_pair(sbase + S::OFF_K + s * S::TILE_BYTES + (p.page_shift >= 6 ? 0 : c * (64 * 128) + (piece << p.page_shift) * 128), &tm_k,
                                      in_leader(&bars[B_KFULL + s]), p.page_shift == 7 ? rank * 64 : 0, c, walk.s.h, page);
                    }
                    __syncwarp();
                }
            }
            // nothing may still be in flight when the pair leaves: the first CTA waits for the loads of both
            if (!ok && rank == 0 && lane == 0)
                for (int k = max(0, g - S::STAGES); k < g; ++k) wait_for(&bars[B_KFULL + k % S::STAGES], (uint32_t)((k / S::STAGES) & 1), status);
        } else if (warp == 10) {
            // ================================ producer of V: the CTA's d / 2 head dims as [group][128 keys][128 B] ======================
            constexpr int VG = S::G / 2;
            const int pieces = 1 << log_per, boxes = log_per == 0 ? 1 : pieces * VG;
            int g = 0, lands = 0;
            bool ok = true;
            Pages pages;
            for (bool more = walk.begin(p, n_items); ok && more; more = walk.step(p, n_items)) {
                pages.begin(p, walk.s, walk.s.blk, log_per);
                for (int j = 0; j < walk.n; ++j, ++g) {
                    const int s = g % S::STAGES, blk = walk.s.blk + j, key0 = blk * BC;
                    const int at = pages.seek(p, walk.s, blk, log_per);
                    const int page = __shfl_sync(0xFFFFFFFFu, pages.now, (log_per == 0 ? at : at + lane / VG) & 31);
                    if (g >= S::STAGES && !(ok = tile::warp_wait(&bars[B_VFREE + s], (uint32_t)((g / S::STAGES - 1) & 1), status))) break;
                    const bool tail = key0 + BC > walk.s.kv && (walk.s.kv & p.page_mask) != 0;
                    if (lane == 0) {
                        if (tail) khq::mbar_arrive_expect_tx(&bars[B_VLAND], S::TILE_BYTES);
                        else arrive_leader_expect(&bars[B_VFULL + s], S::TILE_BYTES);
                    }
                    __syncwarp();
                    const uint32_t dst = sbase + S::OFF_V + s * S::TILE_BYTES;
                    if (lane < boxes) {
                        const int piece = log_per == 0 ? 0 : lane / VG, c = log_per == 0 ? 0 : lane % VG;
                        const uint32_t to = dst + c * (BC * 128) + (piece << p.page_shift) * 128;
                        if (tail) tma_load_5d(to, &tm_v, &bars[B_VLAND], 0, rank * VG + c, walk.s.h, page);
                        else load_for_pair(to, &tm_v, in_leader(&bars[B_VFULL + s]), 0, rank * VG + c, walk.s.h, page);
                    }
                    __syncwarp();
                    if (tail) {
                        if (!(ok = tile::warp_wait(&bars[B_VLAND], (uint32_t)(lands++ & 1), status))) break;
                        // the rest of the request's last page
                        const int r0 = walk.s.kv - key0, n = ((p.page_mask + 1) - (walk.s.kv & p.page_mask)) * 8;
#pragma unroll
                        for (int c = 0; c < VG; ++c)
                            for (int k = lane; k < n; k += 32)
                                *reinterpret_cast<uint4*>(smem + S::OFF_V + s * S::TILE_BYTES + c * (BC * 128) + r0 * 128 + k * 16) = make_uint4(0, 0, 0, 0);
                        khq::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) release_to_leader(&bars[B_VFULL + s]);
                    }
                }
            }
        } else if (warp == 9) {
            // ================================ MMA issuer ==============================================
            const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
            if (rank == 1 && lane == 0) arrive_leader(&bars[B_PEER]);
            if (rank == 0) {
                const uint32_t one = elect_one();
                constexpr uint32_t IDESC_S = instr_desc(2 * BR, BC, false, BF16), IDESC_O = instr_desc(2 * BR, D, true, BF16);
                constexpr uint32_t HI = desc_hi(1024);  // Q, K (K-major) and V (MN-major): 1024 bytes between 8-row groups
                const uint32_t q_lo = desc_lo(sbase + S::OFF_Q, 16), k_lo = desc_lo(sbase + S::OFF_K, 16);
                const uint32_t v_lo = desc_lo(sbase + S::OFF_V, 128 * 128);  // leading offset: the next 64-column group
                bool ok = true;
                // A wait costs some 300 cycles even when its barrier completed long ago: a barrier is tested in front of the last instructions
                // before its use, and waited for only if that came out negative.
                uint32_t k_there = 0, p_there = 0, v_there = 0;
                int k_of = -1;  // the block that k_there is about
                const auto need = [&](uint32_t there, uint64_t* bar, uint32_t parity) {
                    if (ok && !__any_sync(0xFFFFFFFFu, there)) ok = warp_wait(bar, parity, status);
                };
                // S = Q K^T of block g; the tests are of the weights and V of the block that is multiplied next
                const auto issue_qk = [&](int g, bool test) {
                    const uint32_t s_tmem = tmem + S::TM_S + (uint32_t)(g % S::BUFFERS) * BC;
                    const int ks_at = g % S::STAGES;
                    need(k_of == g ? k_there : 0u, &bars[B_KFULL + ks_at], (uint32_t)((g / S::STAGES) & 1));
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t k_at = k_lo + (uint32_t)ks_at * (S::TILE_BYTES >> 4);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        // byte offsets / 16: next 64-dim group = rows * 128 bytes, next K step = 32 bytes
                        const uint32_t oa = (uint32_t)((ks >> 2) * (BR * 128) + (ks & 3) * 32) >> 4;
                        const uint32_t ob = (uint32_t)((ks >> 2) * (64 * 128) + (ks & 3) * 32) >> 4;
                        if (ks == 0) umma2_ss<0>(one, s_tmem, q_lo + oa, HI, k_at + ob, HI, IDESC_S);
                        else umma2_ss<1>(one, s_tmem, q_lo + oa, HI, k_at + ob, HI, IDESC_S);
                        if (ks == D / 16 - 5 && test) {
                            const int n = g - S::AHEAD;
                            p_there = mbar_test(&bars[B_PREADY + 2 * (n % S::BUFFERS)], (uint32_t)((n / S::BUFFERS) & 1));
                            v_there = mbar_test(&bars[B_VFULL + n % S::STAGES], (uint32_t)((n / S::STAGES) & 1));
                        }
                    }
                    umma2_commit(one, &bars[B_SFULL + g % S::BUFFERS]);
                    umma2_commit(one, &bars[B_KFREE + ks_at]);
                };
                int g = 0, i = 0;
                bool more = walk.begin(p, n_items);
                if (more) ok = tile::warp_wait(&bars[B_PEER], 0u, status);
                for (; ok && more; more = walk.step(p, n_items), ++i) {
                    ok = tile::warp_wait(&bars[B_QFULL], (uint32_t)(i & 1), status);
                    if (!ok) break;
                    for (int j = 0; ok && j < min(S::AHEAD, walk.n); ++j) issue_qk(g + j, false);
                    if (!ok) break;
                    if (walk.n <= S::AHEAD) umma2_commit(one, &bars[B_QFREE]);
                    for (int j = 0; j < walk.n; ++j, ++g) {
                        const int s = g % S::BUFFERS, vs = g % S::STAGES;
                        const uint32_t par = (uint32_t)((g / S::BUFFERS) & 1), v_par = (uint32_t)((g / S::STAGES) & 1);
                        p_there = v_there = 0;
                        if (j + S::AHEAD < walk.n) {
                            issue_qk(g + S::AHEAD, true);
                            if (!ok) break;
                            if (j + S::AHEAD + 1 == walk.n) umma2_commit(one, &bars[B_QFREE]);
                        }
                        need(p_there, &bars[B_PREADY + 2 * s], par);
                        if ((walk.s.blk + j + 1) * BC > walk.s.kv) {
                            // zeros that the other CTA's V producer may have stored
                            if (ok) ok = warp_wait_cluster(&bars[B_VFULL + vs], v_par, status);
                        } else {
                            need(v_there, &bars[B_VFULL + vs], v_par);
                        }
                        // the first P V of a segment overwrites O: the one before has been read
                        if (j == 0 && i > 0 && ok) ok = tile::warp_wait(&bars[B_OFREE], (uint32_t)((i - 1) & 1), status);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t v_at = v_lo + (uint32_t)vs * (S::TILE_BYTES >> 4), p_tmem = tmem + S::TM_S + (uint32_t)s * BC;
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk) {
                            if (kk == 4) {  // the other half of the keys: its weights come while the first half is multiplied
                                need(p_there, &bars[B_PREADY + 2 * s + 1], par);
                                if (!ok) break;
                                tc_fence_after();
                            }
                            umma2_ts(one, tmem, p_tmem + kk * 8, v_at + ((uint32_t)(kk * 2048) >> 4), HI, IDESC_O, kk > 0 ? 1u : (uint32_t)(j > 0));  // 16 keys = 2048 bytes
                            if (kk == 1) p_there = mbar_test(&bars[B_PREADY + 2 * s + 1], par);
                            if (kk == 5) {
                                k_of = g + 1 + S::AHEAD;
                                k_there = mbar_test(&bars[B_KFULL + k_of % S::STAGES], (uint32_t)((k_of / S::STAGES) & 1));
                            }
                        }
                        if (!ok) break;
                        umma2_commit(one, &bars[B_PVDONE + (g & 1)]);
                        umma2_commit(one, &bars[B_VFREE + vs]);
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ================================ softmax + epilogue ======================================
        // Group 0 (warps 0-3) has the even blocks, group 1 (warps 4-7) the odd ones; a thread owns a row (all 128 keys of its blocks, and
        // half the columns of O in the epilogue).  The groups' reference maxima follow one another through shared memory, warp by
        // warp: the two warps of a lane quarter have the same rows.
        const uint32_t tmem = *tmem_slot;
        const int grp = warp >> 2, quarter = warp & 3, r = tid & 127, t_row = (r * p.rep_mul) >> 16;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
        unsigned char* const stage = smem + S::OFF_STG + warp * STG_BYTES;
        bool ok = true;
        int g0 = 0, i = 0;  // running index of the segment's first block; segments
        if (tid == 0 && rank == 0) p.meta[blockIdx.x >> 1].n = 0;  // overwritten below if a segment goes on in the next pair
        // pages that are not there, of block `blk` of a segment: bit by page
        const auto fetch_holes = [&](const Segment& sg, int blk) {
            const int col = (blk << log_per) + lane;
            int hole = 0;
            if (lane < (1 << log_per) && (long long)col << p.page_shift < sg.kv)
                hole = col >= p.max_pages || (unsigned)__ldg(p.table + sg.b * p.table_stride + (col < p.max_pages ? col : 0)) >= (unsigned)p.n_pages;
            return hole;
        };
        bool more = walk.begin(p, n_items);
        int hole_next = more && walk.n > grp ? fetch_holes(walk.s, walk.s.blk + grp) : 0;
        for (; ok && more; ++i) {
            const Segment& sg = walk.s;
            const int pos = min(sg.pos0 + rank * tok + t_row, sg.kv - 1);  // keys 0..pos
            const int pos_min = sg.pos0 + rank * tok + (quarter * 32) / p.n_rep;
            const int last = g0 + walk.n - 1;
            const bool whole = sg.blk == 0 && walk.n == sg.n_blocks, gated = whole && p.gate;
            const int n_tok = min(sg.ntok - rank * tok, tok);  // of this CTA, may be 0 or less
            const int row0 = sg.row0 + rank * tok;
            if (gated && t_row < n_tok && row0 + t_row < p.tokens) {  // this row's gates to L2, until the epilogue
                const uint16_t* at = p.gate + (row0 + t_row) * p.g_ts + (sg.h * p.n_rep + r - t_row * p.n_rep) * p.g_hs + grp * (D / 2);
#pragma unroll
                for (int c = 0; c < D / 2; c += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + c));
            }
            float m_l = -INFINITY, l_run = 0.0f;  // the sum of this group's blocks and the reference that it is against
            for (int g = g0 + ((g0 ^ grp) & 1); g <= last; g += 2) {
                const uint32_t holes = __ballot_sync(0xFFFFFFFFu, hole_next);
                if (g + 2 <= last) hole_next = fetch_holes(sg, sg.blk + g + 2 - g0);
                // the reference behind the block before, mostly there by now: ahead of the scores
                float before = 0.0f;
                if (g > g0) {
                    ok = __all_sync(0xFFFFFFFFu, wait_for(&bars[B_MREF + 4 * (grp ^ 1) + quarter], (uint32_t)(((g - 1) >> 1) & 1), status));
                    if (!ok) break;
                    before = mref[(grp ^ 1) * 128 + r];
                }
                const int buf = g % S::BUFFERS;
                ok = __all_sync(0xFFFFFFFFu, wait_for(&bars[B_SFULL + buf], (uint32_t)((g / S::BUFFERS) & 1), status));
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_addr = lane_base + S::TM_S + (uint32_t)buf * BC;
                uint32_t sr[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, sr[c]);
                tmem_ld_wait();
                const int k0 = (sg.blk + g - g0) * BC;
                if (k0 + BC - 1 > pos_min) {  // keys behind the row's position
#pragma unroll
                    for (int c = 0; c < BC; ++c)
                        if (k0 + c > pos) sr[c >> 5][c & 31] = 0xFF800000u;
                }
                if (holes) {
#pragma unroll
                    for (int c = 0; c < BC; ++c)
                        if ((holes >> (c >> p.page_shift)) & 1u) sr[c >> 5][c & 31] = 0xFF800000u;
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < BC; c += 2)
                    mx4[(c >> 1) & 3] = max3(mx4[(c >> 1) & 3], __uint_as_float(sr[c >> 5][c & 31]), __uint_as_float(sr[(c + 1) >> 5][(c + 1) & 31]));
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2e;  // scale > 0
                // the reference follows the maximum only when that has grown by more than 2^8
                const bool grow = g > g0 && mx > before + RESCALE_LOG2;
                const float m_used = g > g0 && !grow ? before : mx, factor = grow ? exp2f(before - mx) : 1.0f;
                mref[grp * 128 + r] = m_used;
                __syncwarp();
                if (lane == 0) khq::mbar_arrive(&bars[B_MREF + 4 * grp + quarter]);
                if (__any_sync(0xFFFFFFFFu, grow)) {
                    // O may only be touched between P V of the previous block and P V of this one.  The completion barriers alternate
                    // between two mbarriers so that a thread may skip phases: barrier (g-1)&1 last completed for block g-3 (certainly, since
                    // Q K^T of this block was issued behind P V of block g-2, or g-3 with three buffers) and cannot complete for block g+1 before this
                    // thread's own arrival for block g.
                    ok = __all_sync(0xFFFFFFFFu, wait_for(&bars[B_PVDONE + ((g - 1) & 1)], (uint32_t)(((g - 1) >> 1) & 1), status));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 16) {
                        uint32_t orr[16];
                        tmem_ld16(lane_base + c0, orr);
                        tmem_ld_wait();
#pragma unroll
                        for (int q = 0; q < 16; ++q) orr[q] = __float_as_uint(__uint_as_float(orr[q]) * factor);
                        tmem_st16(lane_base + c0, orr);
                    }
                }
                // p = 2^(s*scale - m): one fused multiply-add and one ex2 per score; P (16-bit pairs) over the S buffer it came from, in
                // two halves of 64 keys that the MMA warp takes as they come.  A row that has seen no key yet: all p 0.
                float rs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const float neg_m = m_used == -INFINITY ? 0.0f : -m_used;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t pk[32];
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        const uint32_t* sc = &sr[2 * h + (c >> 5)][c & 31];
                        float x0, x1;
                        fma2(x0, x1, __uint_as_float(sc[0]), __uint_as_float(sc[1]), p.scale_log2e, neg_m);
                        const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                        add2(rs[c & 2], rs[(c & 2) + 1], p0, p1);
                        pk[c >> 1] = pack2<BF16>(p0, p1);
                    }
                    tmem_st32(s_addr + h * 32, pk);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_leader(&bars[B_PREADY + 2 * buf + h]);
                    __syncwarp();  // the next access to tensor memory wants the whole warp
                }
                l_run = (m_l == m_used ? l_run : l_run * exp2f(m_l - m_used)) + ((rs[0] + rs[1]) + (rs[2] + rs[3]));
                m_l = m_used;
            }
            if (!ok) break;
            // ---- epilogue of the segment ----------------------------------------------------------------
            // the next segment is on its way meanwhile
            more = walk.more();
            Segment next = sg;
            if (more) next_segment(p, n_items, next);
            // Gates and outputs, 32 columns at a time, pass through the warp's own piece of shared memory: a thread owns a row, so its global
            // accesses would take a line each; this way four lanes take a row's 64 bytes.
            long long q_row[4];  // of the four rows that this lane moves: offset of its 8 columns of the first piece in the gates, -1: none
            long long o_row[4];  // and in the outputs
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int R = quarter * 32 + e * 8 + (lane >> 2), t = (R * p.rep_mul) >> 16, head = sg.h * p.n_rep + R - t * p.n_rep, c = grp * (D / 2) + (lane & 3) * 8;
                const bool live = whole && t < n_tok && row0 + t < p.tokens;
                q_row[e] = live && gated ? (row0 + t) * p.g_ts + head * p.g_hs + c : -1;
                o_row[e] = live ? (row0 + t) * p.o_ts + head * p.o_hs + c : -1;
            }
            const auto gate_at = [&](int e, int c) {
                return q_row[e] < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(p.gate + q_row[e] + c * 32));
            };
            uint4 gates[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) gates[e] = gate_at(e, 0);
            // the last block's reference, then both groups' sums against it
            if (grp != (last & 1))
                ok = wait_for(&bars[B_MREF + 4 * (last & 1) + quarter], (uint32_t)((last >> 1) & 1), status);
            const float m_end = mref[(last & 1) * 128 + r];
            l_run = m_l == m_end ? l_run : l_run * exp2f(m_l - m_end);
            // by segment parity: a group may be a segment ahead of the other's read
            float* const lsum = reinterpret_cast<float*>(smem + S::OFF_LSUM) + (i & 1) * 256;
            lsum[grp * 128 + r] = l_run;
            __syncwarp();
            if (lane == 0) khq::mbar_arrive(&bars[B_LSUM + quarter]);
            if (ok) ok = wait_for(&bars[B_LSUM + quarter], (uint32_t)(i & 1), status);
            if (ok) l_run += lsum[(grp ^ 1) * 128 + r];
            // With three buffers the last scores only say that P V of block last - 3 is complete; the barrier of block last would still show the phase of
            // last - 4 as long as last - 2 runs.  Behind block last - 1, last - 2 is complete too.
            if (S::AHEAD == 2 && ok && last > 0) ok = wait_for(&bars[B_PVDONE + ((last - 1) & 1)], (uint32_t)(((last - 1) >> 1) & 1), status);
            if (ok) ok = wait_for(&bars[B_PVDONE + (last & 1)], (uint32_t)((last >> 1) & 1), status);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            if (more) hole_next = fetch_holes(next, ((last + 1) ^ grp) & 1);  // (a block past the segment's end: no key, no hole)
            __syncwarp();
            if (whole) {
                const float inv = l_run > 0.0f ? 1.0f / l_run : l_run == 0.0f ? 0.0f : l_run;  // a NaN stays one
                const auto spot = [&](int row, int chunk) { return reinterpret_cast<uint4*>(stage + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4)); };
                // one copy of this code: the instructions come from far, once a segment
#pragma unroll 1
                for (int c = 0; c < D / 64; ++c) {
                    uint32_t o[32];
                    tmem_ld32(lane_base + grp * (D / 2) + c * 32, o);
                    if (gated) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            *spot(e * 8 + (lane >> 2), lane & 3) = gates[e];
                            if (c + 1 < D / 64) gates[e] = gate_at(e, c + 1);
                        }
                        __syncwarp();
                    }
                    tmem_ld_wait();
                    if (c == D / 64 - 1) {  // O has been read: the next segment's first P V may overwrite it
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_leader(&bars[B_OFREE]);
                    }
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint4* const at = spot(lane, q);
                        uint32_t w[4];
                        if (gated) {
                            const uint4 gv = *at;
                            const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 f = unpack2<BF16>(gw[e]);
                                w[e] = pack2<BF16>(__uint_as_float(o[8 * q + 2 * e]) * inv * sigmoid(f.x), __uint_as_float(o[8 * q + 2 * e + 1]) * inv * sigmoid(f.y));
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = pack2<BF16>(__uint_as_float(o[8 * q + 2 * e]) * inv, __uint_as_float(o[8 * q + 2 * e + 1]) * inv);
                        }
                        *at = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (o_row[e] >= 0) *reinterpret_cast<uint4*>(p.out + o_row[e] + c * 32) = *spot(e * 8 + (lane >> 2), lane & 3);
                    }
                    __syncwarp();
                }
                if (p.lse && grp == 0 && t_row < n_tok && row0 + t_row < p.tokens)
                    p.lse[(long long)(row0 + t_row) * p.H_q + sg.h * p.n_rep + (r - t_row * p.n_rep)] = (m_end + log2f(l_run)) * 0.6931471805599453f;
            } else {
                // record 1: of the segment that begins in this stretch, record 0: of one that began before
                float* const rec = p.records + (2LL * blockIdx.x + (sg.blk == 0 ? 1 : 0)) * S::RECORD;
#pragma unroll 1
                for (int c0 = grp * (D / 2); c0 < (grp + 1) * (D / 2); c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(lane_base + c0, o);  // whole warps, also where some rows have no token
                    tmem_ld_wait();
                    if (t_row < n_tok) {
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            reinterpret_cast<uint4*>(rec)[(c0 / 4 + q) * BR + r] = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
                    }
                    __syncwarp();
                }
                if (grp == 0 && t_row < n_tok) *reinterpret_cast<float2*>(rec + BR * D + 2 * r) = make_float2(m_end, l_run);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_leader(&bars[B_OFREE]);
                if (tid == 0 && rank == 0 && sg.blk == 0)  // it goes on in the next pairs
                    *reinterpret_cast<int4*>(p.meta + (blockIdx.x >> 1)) = make_int4(walk.share, sg.h, sg.row0, sg.ntok);
            }
            g0 = last + 1;
            if (more) walk.step_to(next);
        }
    }
    // ---- teardown: every thread arrives here, with or without a failed wait ----------------------
    tc_fence_before();
    __syncwarp();
    cluster_arrive();
    cluster_wait();  // no CTA leaves while the other's loads, products or arrivals concern it
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "n"(TM_COLS) : "memory");
}

// Joins the records of the segment that begins in pair `pair` of the chunk kernel and goes on in the next ones.  Two threads take a row of a CTA's 128
// and 16 of its columns each; `part`: the CTA of the pair and the columns.
constexpr int MERGE_CTAS = 16;
template <int D, bool BF16>
__device__ __forceinline__ void merge_chunk(const Params& p, int pair, int part) {
    using S = Shape<D>;
    constexpr int COLS = D / 4 / MERGE_CTAS;
    static_assert(MERGE_THREADS == 2 * BR, "two threads a row");
    const int4 meta = *reinterpret_cast<const int4*>(p.meta + pair);
    const int rank = part & 1, r = threadIdx.x & 127, n = meta.x;
    part = (part >> 1) * 2 + (threadIdx.x >> 7);
    if (n == 0) return;
    const int tok = BR / p.n_rep, t = (r * p.rep_mul) >> 16, n_tok = min(meta.w - rank * tok, tok), row = meta.z + rank * tok + t;
    if (t >= n_tok || row >= p.tokens) return;
    const auto record = [&](int i) { return p.records + (2LL * (2 * (pair + i) + rank) + (i == 0)) * S::RECORD; };
    float M = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < n; ++i) M = fmaxf(M, record(i)[BR * D + 2 * r]);
    float4 acc[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float L = 0.0f;
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
        const float* rec = record(i);
        const float2 ml = *reinterpret_cast<const float2*>(rec + BR * D + 2 * r);
        float4 a[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) a[c] = reinterpret_cast<const float4*>(rec)[(part * COLS + c) * BR + r];
        const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
        L += ml.y * f;
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            acc[c].x += a[c].x * f;
            acc[c].y += a[c].y * f;
            acc[c].z += a[c].z * f;
            acc[c].w += a[c].w * f;
        }
    }
    const int head = meta.y * p.n_rep + (r - t * p.n_rep);
    const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
#pragma unroll
    for (int c = 0; c < COLS; ++c) store_out<BF16>(p, row, head, (part * COLS + c) * 4, acc[c], inv);
    if (p.lse && part == 0) p.lse[(long long)row * p.H_q + head] = (M + log2f(L)) * 0.6931471805599453f;
}

}  // namespace tile
}  // namespace khq_paged
