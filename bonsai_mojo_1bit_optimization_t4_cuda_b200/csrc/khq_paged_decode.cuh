// khq_paged_decode.cuh -- attention over the paged cache for tiles of up to 16 query rows (a decode step: one or a few new tokens a
// request).  Included by khq_paged_attn.cu.
//
// Every K and V byte is used by 16 rows at most, so the cache's bytes bound it.  The key blocks (64 keys, 128 at d 128) of all (kv head,
// item) pairs stand in one row, and each CTA takes an equal stretch of it (one CTA per SM): any mix of lengths is even, and a CTA ends up with at most two
// segments that it shares with others.  Those leave records (unnormalised rows, maximum, sum) that khq_paged_merge_kernel joins
// in a fixed order; the others are finished here.
//
// A warp takes a unit of each block, 16 keys (32 at d 128), and runs alone: its first lanes bring their rows of K and V in by TMA three units
// ahead, into a ring that no other warp touches; S = Q K^T and O += P V are mma.sync m16n8k16 with the query rows as M and all of O in
// registers.  Only at a segment's end the four warps join their maxima, sums and rows through shared memory.
// One warp a scheduler, so a unit's chain of latencies counts (2100 cycles for 16 keys at d 128): 16 KB a unit and one wait for both halves
// of it keep the chain below the time that memory takes.  64 sequences of 4200 tokens, d 256: 185 us; with eight warps and half the
// ring for each 235; with K and V waited for one after the other, and one chain of products instead of two, 251.
//
// The weights enter the product with V as 16-bit values, the instruction's type and what the chunk kernel does: half a step of it (2^-11, bf16 2^-8) of sum w |v|,
// about what the output's own rounding takes.  Their sum is of the fp32 values.  A second product with what the rounding left out would add to the chain of
// a unit, which is just below memory's time.
#pragma once

namespace khq_paged {
namespace decode {

constexpr int WARPS = 4;
constexpr int JOIN_ROWS = 8;  // rows that are joined at a time
template <int D> struct Shape {
    static constexpr int KEYS = 64 * 256 / D, UNIT = KEYS / WARPS;   // of a block, of a warp's share of it
    static constexpr int G = D / 64, PIECE = UNIT * D * 2, STAGES = 3;  // column groups; K or V of a unit; units in a warp's ring
    static constexpr int NT = UNIT / 8;  // tiles of 8 keys
    static constexpr int ROW = D + 8;  // floats of a row in the join buffer: rows 8 banks apart
    static constexpr int OFF_JOIN = WARPS * STAGES * 2 * PIECE, OFF_ML = OFF_JOIN + WARPS * JOIN_ROWS * ROW * 4;
    static constexpr int OFF_BARS = OFF_ML + WARPS * DECODE_ROWS * 8, SMEM = OFF_BARS + WARPS * STAGES * 8;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static constexpr int RECORD = DECODE_ROWS * D + 2 * DECODE_ROWS;  // floats
};
// A piece is one box where a page holds the unit; else (32 keys, pages of 16) one per page and column group.
template <int D> int box_tokens(int page_size) { return page_size < Shape<D>::UNIT ? page_size : Shape<D>::UNIT; }
template <int D> int box_groups(int page_size) { return page_size < Shape<D>::UNIT ? 1 : Shape<D>::G; }

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <int D, bool BF16>
__global__ void __launch_bounds__(WARPS * 32, 1)
khq_paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
    using S = Shape<D>;
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BARS);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* const status = &g_paged_status;
    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled layout needs a 1024-byte aligned base
        khq::pdl_wait();
        if (tid == 0) {
            atomicExch(status, 2);
            p.meta[blockIdx.x].n = 0;
        }
        return;
    }
    if (lane == 0) {
        for (int s = 0; s < S::STAGES; ++s) khq::mbar_init(&bars[warp * S::STAGES + s], 1);
        khq::fence_barrier_init();
        prefetch_map(warp & 1 ? &tm_k : &tm_v);
    }
    __syncthreads();
    khq::pdl_wait();
    khq::pdl_trigger();

    // ---- this CTA's stretch of the key blocks ------------------------------------------------------
    Segment in, cur;  // where the loads and where the products are
    int n_items, length, share;
    const bool work = first_segment(p, blockIdx.x, in, n_items, length, share);
    if (tid == 0) p.meta[blockIdx.x].n = 0;  // overwritten below if a segment goes on in the next CTA
    if (!work) return;
    // what is left of the stretch from the item's begin on, and the item's blocks in it
    const auto of_stretch = [](const Segment& s, int left) { return min(s.n_blocks, left - DECODE_OVER) - s.blk; };
    int left_in = length, n_in = of_stretch(in, length), left = length, n_seg = n_in;
    cur = in;
    uint64_t* const bar = bars + warp * S::STAGES;
    const uint32_t ring = smem_u32(smem) + warp * S::STAGES * 2 * S::PIECE;

    // ---- loads ---------------------------------------------------------------------------------------
    // The lanes hold the pages of the units of 32 blocks (16, where a unit has two), the next ones are on their way; n_pages: none (the
    // copy then fills in zeros, and the keys are masked).
    constexpr int UNIT = S::UNIT;
    const int log_per = UNIT == 32 && p.page_shift == 4 ? 1 : 0, groups = log_per ? S::G : 1;
    int pages = 0, pages_next = 0, pages_at = -1;
    int s_in = 0;
    uint32_t missing = 0;  // two bits by unit of the ring: its first, second page is not there
    bool ok = true;        // no wait has run out
    const auto fetch_pages = [&](int blk) {
        const int key = (blk + (lane >> log_per)) * S::KEYS + warp * UNIT + ((lane & log_per) << 4), col = key >> p.page_shift;
        int pg = p.n_pages;
        if (key < in.kv && col < p.max_pages) {
            pg = __ldg(p.table + in.b * p.table_stride + col);
            if ((unsigned)pg >= (unsigned)p.n_pages) pg = p.n_pages;
        }
        return pg;
    };
    const auto issue = [&]() {
        if (n_in == 0) return;
        if (pages_at < 0 || in.blk - pages_at >= (32 >> log_per)) {
            pages = pages_at < 0 ? fetch_pages(in.blk) : pages_next;
            pages_at = in.blk;
            pages_next = fetch_pages(in.blk + (32 >> log_per));
        }
        const int page = __shfl_sync(0xFFFFFFFFu, pages, ((in.blk - pages_at) << log_per) + ((lane >> 3) & log_per));  // of this lane's box
        const uint32_t holes = __ballot_sync(0xFFFFFFFFu, page == p.n_pages);  // lane 0: the first page, lane 8: the second
        missing = (missing & ~(3u << (2 * s_in))) | (((holes & 1u) | ((holes >> 7) & 2u)) << (2 * s_in));
        if (ok) {
            if (lane == 0) khq::mbar_arrive_expect_tx(&bar[s_in], 2 * S::PIECE);
            __syncwarp();
            // boxes: one each of K and V, by lanes 0 and 4; or one by page (lane / 8), K or V (lane / 4 % 2) and group (lane % 4)
            const int c = lane & 3;
            if (lane < 8 << log_per && c < groups)
                tma_load_5d(ring + (2 * s_in + ((lane >> 2) & 1)) * S::PIECE + c * (UNIT * 128) + (lane >> 3) * (16 * 128), lane & 4 ? &tm_v : &tm_k, &bar[s_in],
                            (in.blk * S::KEYS + warp * UNIT) & p.page_mask, c, in.h, page);
        }
        s_in = s_in + 1 == S::STAGES ? 0 : s_in + 1;
        ++in.blk;
        if (--n_in == 0 && (left_in -= in.n_blocks + DECODE_OVER) > DECODE_OVER) {
            next_segment(p, n_items, in);
            n_in = of_stretch(in, left_in);
            pages_at = -1;
        }
    };
#pragma unroll 1
    for (int s = 0; s < S::STAGES; ++s) issue();

    // ---- products ------------------------------------------------------------------------------------
    const int g = lane >> 2, t2 = (lane & 3) * 2;  // rows g and g + 8, columns t2 and t2 + 1 of a fragment
    uint32_t qf[D / 16][4];
    float o[D / 8][4], m[2], l[2];
    // addresses of this lane's rows for ldmatrix; chunk c of key k is at (c ^ (k & 7)) << 4
    const int k_key = (lane & 7) + ((lane >> 4) & 1) * 8, k_chunk = (lane >> 3) & 1;
    const int v_key = (lane & 7) + ((lane >> 3) & 1) * 8, v_chunk = lane >> 4;
    const uint32_t k_row = k_key * 128, v_row = S::PIECE + v_key * 128, sw = (lane & 7);
    int s = 0;
    uint32_t phase = 0;
    bool fresh = true, begins = false;  // a segment's first block; the segment is the item's begin
#pragma unroll 1
    for (;;) {
        const int R = cur.ntok * p.n_rep;
        if (fresh) {
            fresh = false;
            begins = cur.blk == 0;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = g + 8 * half, t = (r * p.rep_mul) >> 16, row = cur.row0 + t;
                const bool live = r < R && row < p.tokens;
                const uint16_t* q = p.q + (live ? row * p.q_ts + (long long)(cur.h * p.n_rep + r - t * p.n_rep) * p.q_hs : 0) + t2;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    qf[kk][half] = live ? __ldg(reinterpret_cast<const uint32_t*>(q + kk * 16)) : 0u;
                    qf[kk][2 + half] = live ? __ldg(reinterpret_cast<const uint32_t*>(q + kk * 16 + 8)) : 0u;
                }
                m[half] = -INFINITY;
                l[half] = 0.0f;
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        }
        // (after a wait that ran out the warp goes on without data, so that the others are not left at a barrier; the status word tells)
        if (ok && !(ok = __all_sync(0xFFFFFFFFu, wait_for(&bar[s], phase, status))))
            for (int i = 1; i < S::STAGES; ++i) wait_for(&bar[(s + i) % S::STAGES], phase ^ (uint32_t)(s + i >= S::STAGES), status);  // what is still in flight
        const int key0 = cur.blk * S::KEYS + warp * UNIT;
        const uint32_t holes = (missing >> (2 * s)) & 3u;
        constexpr int NT = S::NT;
        if (ok && holes != 3u) {
            const uint32_t base = ring + 2 * s * S::PIECE;
            float x[NT][4] = {}, y[NT][4] = {};  // two chains each
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b[4];
                    ldsm4(base + (kk >> 2) * (UNIT * 128) + n * (8 * 128) + k_row + (((uint32_t)((kk & 3) * 2 + k_chunk) ^ sw) << 4), b);
                    mma16816<BF16>(kk & 1 ? y[n] : x[n], qf[kk], b[0], b[1]);
                    mma16816<BF16>(kk & 1 ? y[n + 1] : x[n + 1], qf[kk], b[2], b[3]);
                }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = (x[n][e] + y[n][e]) * p.scale_log2e;
            if (key0 + UNIT - 1 > cur.pos0) {  // some row's position lies in front of the unit's last key
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int at = cur.pos0 + (((g + 8 * half) * p.rep_mul) >> 16);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (key0 + n * 8 + t2 + e > at) x[n][half * 2 + e] = -INFINITY;
                }
            }
            if (NT > 2 && holes) {  // one of the unit's two pages
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((holes >> (n >> 1)) & 1u) x[n][e] = -INFINITY;
            }
            uint32_t pf[NT / 2][4];
            float factor[2];
            bool grow = false;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float mx = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(x[n][half * 2], x[n][half * 2 + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                factor[half] = 1.0f;
                // the reference follows the maximum only when that has grown by more than 2^8: fewer passes over O, and nothing leaves fp32's or
                // the 16-bit weights' range
                if (mx > m[half] + 8.0f) {
                    factor[half] = exp2f(m[half] - mx);
                    m[half] = mx;
                    grow = true;
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float ref = m[half] == -INFINITY ? 0.0f : m[half];
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float p0 = ex2_approx(x[n][half * 2] - ref), p1 = ex2_approx(x[n][half * 2 + 1] - ref);
                    sum += p0 + p1;
                    pf[n >> 1][(n & 1) * 2 + half] = pack2<BF16>(p0, p1);
                }
                l[half] = l[half] * factor[half] + sum;
            }
            if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
                for (int n = 0; n < D / 8; ++n) {
                    o[n][0] *= factor[0];
                    o[n][1] *= factor[0];
                    o[n][2] *= factor[1];
                    o[n][3] *= factor[1];
                }
            }
            // rows of V behind the request's last token may hold anything: a weight of 0 does not undo that
            uint32_t keep[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) keep[n] = 0xFFFFFFFFu;
            if (key0 + UNIT > cur.kv) {
                const int left = cur.kv - key0;  // keys that exist; this lane's are t2 and t2 + 1 of each 8
#pragma unroll
                for (int n = 0; n < NT; ++n) keep[n] = (n * 8 + t2 < left ? 0x0000FFFFu : 0u) | (n * 8 + t2 + 1 < left ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
#pragma unroll
                for (int k = 0; k < NT / 2; ++k) {
                    uint32_t b[4];
                    ldsm4_trans(base + (n >> 2) * (UNIT * 128) + k * (16 * 128) + v_row + (((uint32_t)((n & 3) * 2 + v_chunk) ^ sw) << 4), b);
                    mma16816<BF16>(o[2 * n], pf[k], b[0] & keep[2 * k], b[1] & keep[2 * k + 1]);
                    mma16816<BF16>(o[2 * n + 1], pf[k], b[2] & keep[2 * k], b[3] & keep[2 * k + 1]);
                }
        }
        __syncwarp();  // all lanes have read the stage
        s = s + 1 == S::STAGES ? 0 : s + 1;
        phase ^= (uint32_t)(s == 0);
        issue();
        const bool ends = cur.blk + 1 == cur.n_blocks;
        if (--n_seg == 0) {
            // ---- join the warps ----------------------------------------------------------------------
            const bool whole = begins && ends;
            float* const join = reinterpret_cast<float*>(smem + S::OFF_JOIN);
            float2* const ml = reinterpret_cast<float2*>(smem + S::OFF_ML);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 1);
                l[half] += __shfl_xor_sync(0xFFFFFFFFu, l[half], 2);
                if ((lane & 3) == 0) ml[warp * DECODE_ROWS + half * 8 + g] = make_float2(m[half], l[half]);
            }
            __syncthreads();
            const auto top = [&](int r) {
                float M = ml[r].x;
#pragma unroll
                for (int v = 1; v < WARPS; ++v) M = fmaxf(M, ml[v * DECODE_ROWS + r].x);
                return M;
            };
            float* const rec = p.records + (2LL * blockIdx.x + (begins ? 1 : 0)) * S::RECORD;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                if (half * 8 >= R) break;
                const float M = top(half * 8 + g), f = m[half] == -INFINITY ? 0.0f : ex2_approx(m[half] - M);
                float* const mine = join + (warp * JOIN_ROWS + g) * S::ROW + t2;
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<float2*>(mine + n * 8) = half == 0 ? make_float2(o[n][0] * f, o[n][1] * f) : make_float2(o[n][2] * f, o[n][3] * f);
                __syncthreads();
                const int rr = tid >> 4, r = rr + 8 * half;  // 16 threads a row
                if (r < R) {
                    const float Mr = top(r);
                    float L = 0.0f;
#pragma unroll
                    for (int v = 0; v < WARPS; ++v) {
                        const float2 a = ml[v * DECODE_ROWS + r];
                        L += a.x == -INFINITY ? a.y : a.y * ex2_approx(a.x - Mr);  // no maximum: 0, or NaN where every score was one
                    }
                    const int t = (r * p.rep_mul) >> 16, row = cur.row0 + t, head = cur.h * p.n_rep + (r - t * p.n_rep);
                    const bool live = row < p.tokens;
                    const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;  // a NaN stays one
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {
                        const int c = j * 64 + (tid & 15) * 4;
                        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                        for (int v = 0; v < WARPS; ++v) {
                            const float4 a = *reinterpret_cast<const float4*>(join + (v * JOIN_ROWS + rr) * S::ROW + c);
                            acc.x += a.x;
                            acc.y += a.y;
                            acc.z += a.z;
                            acc.w += a.w;
                        }
                        if (!whole) *reinterpret_cast<float4*>(rec + r * D + c) = acc;
                        else if (live) store_out<BF16>(p, row, head, c, acc, inv);
                    }
                    if ((tid & 15) == 0) {
                        if (!whole) *reinterpret_cast<float2*>(rec + DECODE_ROWS * D + 2 * r) = make_float2(Mr, L);
                        else if (live && p.lse) p.lse[(long long)row * p.H_q + head] = (Mr + log2f(L)) * 0.6931471805599453f;
                    }
                }
                __syncthreads();
            }
            if (tid == 0 && begins && !ends) *reinterpret_cast<int4*>(p.meta + blockIdx.x) = make_int4(share, cur.h, cur.row0, cur.ntok);
            if ((left -= cur.n_blocks + DECODE_OVER) <= DECODE_OVER) break;
            next_segment(p, n_items, cur);
            n_seg = of_stretch(cur, left);
            fresh = true;
        } else {
            ++cur.blk;
        }
    }
}

}  // namespace decode
}  // namespace khq_paged
