// khq_paged_attn.cu -- attention of a step's new tokens over a raw paged K/V cache: the kernels' common part, the joining of shared
// segments and the host side.  The kernels: khq_paged_decode.cuh (few rows a request), khq_paged_tile.cuh (chunks).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "khq_b200.h"
#include "khq_common.cuh"
#include "khq_launch.cuh"
#include "khq_paged.cuh"
#include "khq_tc5.cuh"

namespace khq_paged {

using khq::smem_u32;
using namespace khq_tc5;

__device__ int g_paged_status = 0;

// Waits give up after two seconds, record that in the status word and return false.  (A count of polls says little: a poll may
// park the thread for a while.)  `any` joins the lanes that wait together: their tests and their clocks have to agree.
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
template <class Test, class Any>
__device__ __forceinline__ bool bounded(Test test, Any any, int* status) {
    unsigned long long begin = 0;
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 32; ++i)
            if (any(test())) return true;
        const unsigned long long now = now_ns();
        if (begin == 0) begin = now;
        if (any(now - begin > 2000000000ull)) break;
    }
    atomicExch(status, 1);
    return false;
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* status) {
    return bounded([&] { return khq::mbar_try_wait(bar, parity); }, [](bool x) { return x; }, status);
}

// By worker: how many records there are of the segment which begins in it and goes on in the next ones (0: none), and what joining them needs.
// Record 1 of a worker is of the segment that begins in it, record 0 of one that it took over.
struct alignas(16) Meta {
    int n, h, row0, ntok;
};

struct Params {
    const uint16_t *q, *gate;
    uint16_t* out;
    float* lse;
    long long q_ts, q_hs, g_ts, g_hs, o_ts, o_hs, table_stride;
    const int* table;
    const Item* items;
    const Start* starts;
    float* records;
    Meta* meta;
    int tokens, max_pages, n_pages, page_shift, page_mask, H_q, H_kv, n_rep, rep_mul;  // x / n_rep = x * rep_mul >> 16 for x < 128
    float scale_log2e;
};

// An item of one kv head, and how far its key blocks have been walked.
struct Segment {
    int item, h, b, n_blocks, blk, ntok, kv, row0, pos0;  // row0: its first row in the ragged tensors, pos0: that row's position
};
__device__ __forceinline__ void load_segment(const Params& p, Segment& s) {
    const int4* it = reinterpret_cast<const int4*>(p.items + s.item);
    const int4 x = __ldg(it), y = __ldg(it + 1);
    s.b = x.x;
    s.n_blocks = x.y;
    s.ntok = x.z;
    s.kv = x.w;
    s.row0 = y.x;
    s.pos0 = y.y;
}
// The worker's first segment; false: none.
__device__ __forceinline__ bool first_segment(const Params& p, int worker, Segment& s, int& n_items, int& length, int& share) {
    const int4* at = reinterpret_cast<const int4*>(p.starts + worker);
    const int4 x = at[0], y = at[1], z = at[2];
    const int2 w = *reinterpret_cast<const int2*>(at + 3);  // (ordinary loads: nothing else keeps them behind the wait for the plan)
    s.b = x.x;
    s.n_blocks = x.y;
    s.ntok = x.z;
    s.kv = x.w;
    s.row0 = y.x;
    s.pos0 = y.y;
    s.item = z.x;
    s.h = z.y;
    s.blk = z.z;
    n_items = z.w;
    length = w.x;
    share = w.y;
    return length > 0;
}
// Every item has a key block at least (its own tokens).
__device__ __forceinline__ void next_segment(const Params& p, int n_items, Segment& s) {
    if (++s.item == n_items) {
        s.item = 0;
        ++s.h;
    }
    s.blk = 0;
    load_segment(p, s);
}

template <bool BF16>
__device__ __forceinline__ void store_out(const Params& p, int row, int head, int c, float4 acc, float inv) {
    acc.x *= inv;
    acc.y *= inv;
    acc.z *= inv;
    acc.w *= inv;
    if (p.gate) {
        const uint2 g = __ldg(reinterpret_cast<const uint2*>(p.gate + row * p.g_ts + head * p.g_hs + c));
        const float2 g0 = unpack2<BF16>(g.x), g1 = unpack2<BF16>(g.y);
        acc.x *= sigmoid(g0.x);
        acc.y *= sigmoid(g0.y);
        acc.z *= sigmoid(g1.x);
        acc.w *= sigmoid(g1.y);
    }
    *reinterpret_cast<uint2*>(p.out + row * p.o_ts + head * p.o_hs + c) = make_uint2(pack2<BF16>(acc.x, acc.y), pack2<BF16>(acc.z, acc.w));
}

// Joins row r of the records of the segment that begins in CTA `worker` of the decode kernel and goes on in the next ones.  Groups of D / 4 threads take the
// records in turn, 4 columns a thread.  Latency bounds it (one token over 4001: 37 records a row): a row per CTA, and the first records are on
// their way while their factors are formed.
constexpr int MERGE_THREADS = 256;
template <int D, bool BF16>
__device__ __forceinline__ void merge_decode(const Params& p, int record_floats, int worker, int r) {
    constexpr int PER_ROW = D / 4, GROUPS = MERGE_THREADS / PER_ROW, AHEAD = 6;
    __shared__ float factor[MAX_WORKERS];
    __shared__ float4 sums[GROUPS][PER_ROW];
    const int4 meta = *reinterpret_cast<const int4*>(p.meta + worker);
    const int n = meta.x, tid = threadIdx.x, lane = tid & 31;
    if (n == 0 || r >= meta.w * p.n_rep) return;
    const auto record = [&](int i) { return p.records + (2LL * (worker + i) + (i == 0)) * record_floats; };
    const int col = tid % PER_ROW, group = tid / PER_ROW;
    float4 a[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (group + k * GROUPS < n) a[k] = *reinterpret_cast<const float4*>(record(group + k * GROUPS) + r * D + col * 4);
    // every warp for itself: the row's maximum, its sum, and each record's factor
    float2 ml[MAX_WORKERS / 32];
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int k = 0; k < MAX_WORKERS / 32; ++k) {
        const int i = k * 32 + lane;
        ml[k] = i < n ? *reinterpret_cast<const float2*>(record(i) + DECODE_ROWS * D + 2 * r) : make_float2(-INFINITY, 0.0f);
        M = fmaxf(M, ml[k].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
#pragma unroll
    for (int k = 0; k < MAX_WORKERS / 32; ++k) {
        const int i = k * 32 + lane;
        const float f = ml[k].x == -INFINITY ? 0.0f : ex2_approx(ml[k].x - M);
        L += ml[k].y * f;
        if (tid < 32 && i < n) factor[i] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, o);
    __syncthreads();
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&](const float4& x, float f) {
        acc.x += x.x * f;
        acc.y += x.y * f;
        acc.z += x.z * f;
        acc.w += x.w * f;
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (group + k * GROUPS < n) add(a[k], factor[group + k * GROUPS]);
#pragma unroll 8
    for (int i = group + AHEAD * GROUPS; i < n; i += GROUPS) add(*reinterpret_cast<const float4*>(record(i) + r * D + col * 4), factor[i]);
    sums[group][col] = acc;
    __syncthreads();
    const int t = (r * p.rep_mul) >> 16, row = meta.z + t, head = meta.y * p.n_rep + (r - t * p.n_rep);
    if (group != 0 || row >= p.tokens) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) add(sums[g][col], 1.0f);
    store_out<BF16>(p, row, head, col * 4, acc, L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L);
    if (p.lse && col == 0) p.lse[(long long)row * p.H_q + head] = (M + log2f(L)) * 0.6931471805599453f;
}

}  // namespace khq_paged

#include "khq_paged_decode.cuh"
#include "khq_paged_tile.cuh"

namespace khq_paged {

// The records of both kernels: the first `chunk_ctas` CTAs those of the chunk kernel, the others the decode kernel's.
template <int D, bool BF16>
__global__ void __launch_bounds__(MERGE_THREADS)
khq_paged_merge_kernel(const __grid_constant__ Params chunk, const __grid_constant__ Params dec, int chunk_ctas, int rows) {
    khq::pdl_wait();
    khq::pdl_trigger();
    const int cta = blockIdx.x;
    if (cta < chunk_ctas) tile::merge_chunk<D, BF16>(chunk, cta / tile::MERGE_CTAS, cta % tile::MERGE_CTAS);
    else merge_decode<D, BF16>(dec, decode::Shape<D>::RECORD, (cta - chunk_ctas) / rows, (cta - chunk_ctas) % rows);
}

}  // namespace khq_paged

// ---- host side -----------------------------------------------------------------------------------
namespace {

using namespace khq_paged;

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = nullptr;
    static bool tried = false;
    if (!tried) {
        void* q = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(q);
        tried = true;
    }
    return fn;
}

// A cache (n_pages, page_size, heads, d) as {64 values, token of a page, 64-column group, head, page}; a box is `box_tokens` tokens
// x `box_groups` groups.
int cache_map(CUtensorMap* map, const void* base, const int64_t (&stride)[3], int page_size, int heads, int d, int n_pages, int box_tokens, int box_groups,
              bool bf16) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return -107;
    const cuuint64_t dims[5] = {64, (cuuint64_t)page_size, (cuuint64_t)(d / 64), (cuuint64_t)heads, (cuuint64_t)n_pages};
    // a dimension of one has any stride
    const auto bytes = [](int64_t s, int n) { return n == 1 ? (cuuint64_t)16 : (cuuint64_t)s * 2; };
    const cuuint64_t strides[4] = {(cuuint64_t)stride[1] * 2, 128, bytes(stride[2], heads), bytes(stride[0], n_pages)};
    const cuuint32_t box[5] = {64, (cuuint32_t)box_tokens, (cuuint32_t)box_groups, 1, 1};
    const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : -108;
}

// Queries (tokens, heads, d) as {64 values, head, token, column group}; a box is a column group of one kv head's heads of `box_tokens` tokens.
int query_map(CUtensorMap* map, const void* base, const int64_t (&stride)[2], int tokens, int heads, int d, int box_heads, int box_tokens, bool bf16) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return -107;
    const cuuint64_t dims[4] = {64, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)(d / 64)};
    const auto bytes = [](int64_t s, int n) { return n == 1 ? (cuuint64_t)16 : (cuuint64_t)s * 2; };
    const cuuint64_t strides[3] = {bytes(stride[1], heads), bytes(stride[0], tokens), 128};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : -108;
}

// The workspace: for each kernel that the step can have a line of `meta` and two records per CTA.
struct Work {
    int ctas, pairs;
    size_t decode_meta, decode_records, chunk_meta, chunk_records, bytes;
};
Work work_of(const Schedule& sched, int d) {
    Work w;
    w.ctas = khq::sm_count() < MAX_WORKERS ? khq::sm_count() : MAX_WORKERS;  // one per SM
    w.pairs = w.ctas / 2;
    w.decode_meta = 0;
    w.decode_records = w.decode_meta + (size_t)w.ctas * sizeof(Meta);
    w.chunk_meta = w.decode_records + (sched.decodes ? (size_t)2 * w.ctas * (d == 256 ? decode::Shape<256>::RECORD : decode::Shape<128>::RECORD) * 4 : 0);
    w.chunk_records = w.chunk_meta + (sched.chunks ? (size_t)w.pairs * sizeof(Meta) : 0);
    w.bytes = w.chunk_records + (sched.chunks ? (size_t)4 * w.pairs * (d == 256 ? tile::Shape<256>::RECORD : tile::Shape<128>::RECORD) * 4 : 0);
    return w;
}

// Both kernels' shared memory, once per device.
template <int D, bool BF16>
int prepare_kernels() {
    static bool attr_done[64] = {};
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return static_cast<int>(err);
    if (dev < 0 || dev >= 64) return -100;
    if (attr_done[dev]) return 0;
    err = cudaFuncSetAttribute((const void*)decode::khq_paged_decode_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, decode::Shape<D>::SMEM);
    if (err == cudaSuccess)
        err = cudaFuncSetAttribute((const void*)tile::khq_paged_tile_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, tile::Shape<D>::SMEM);
    if (err != cudaSuccess) return static_cast<int>(err);
    attr_done[dev] = true;
    return 0;
}

template <int D, bool BF16>
int launch_kernels(const khq_paged_attn_args& a, Params p, const Schedule& sched, const Work& w, cudaStream_t stream) {
    int rc = prepare_kernels<D, BF16>();
    unsigned char* const ws = static_cast<unsigned char*>(a.workspace);
    const auto of_kernel = [&](long long starts, long long items, size_t meta, size_t records) {
        p.starts = reinterpret_cast<const Start*>(static_cast<const int*>(a.schedule) + starts);
        p.items = reinterpret_cast<const Item*>(static_cast<const int*>(a.schedule) + items);
        p.meta = reinterpret_cast<Meta*>(ws + meta);
        p.records = reinterpret_cast<float*>(ws + records);
    };
    cudaError_t err;
    if (sched.chunks) {
        using S = tile::Shape<D>;
        of_kernel(sched.chunk_starts, sched.chunk_items, w.chunk_meta, w.chunk_records);
        CUtensorMap mq, mk, mv;
        if (rc == 0) rc = query_map(&mq, a.q, a.q_stride, a.tokens, a.H_q, D, p.n_rep, tile::BR / p.n_rep, BF16);
        if (rc == 0)
            rc = cache_map(&mk, a.k_cache, a.k_cache_stride, a.page_size, a.H_kv, D, a.n_pages, a.page_size < 64 ? a.page_size : 64, a.page_size < 64 ? 1 : S::G, BF16);
        if (rc == 0) rc = cache_map(&mv, a.v_cache, a.v_cache_stride, a.page_size, a.H_kv, D, a.n_pages, a.page_size, a.page_size < 128 ? 1 : S::G / 2, BF16);
        if (rc != 0) return rc;
        err = khq::launch_pdl(tile::khq_paged_tile_kernel<D, BF16>, (unsigned)(2 * w.pairs), 2u, (size_t)S::SMEM, stream, (unsigned)tile::NTHREADS, mq, mk, mv, p);
        if (err != cudaSuccess) return static_cast<int>(err);
    }
    const Params chunk = p;
    if (sched.decodes) {
        of_kernel(sched.decode_starts, sched.decode_items, w.decode_meta, w.decode_records);
        CUtensorMap mk, mv;
        if (rc == 0) rc = cache_map(&mk, a.k_cache, a.k_cache_stride, a.page_size, a.H_kv, D, a.n_pages, decode::box_tokens<D>(a.page_size), decode::box_groups<D>(a.page_size), BF16);
        if (rc == 0) rc = cache_map(&mv, a.v_cache, a.v_cache_stride, a.page_size, a.H_kv, D, a.n_pages, decode::box_tokens<D>(a.page_size), decode::box_groups<D>(a.page_size), BF16);
        if (rc != 0) return rc;
        err = khq::launch_pdl(decode::khq_paged_decode_kernel<D, BF16>, (unsigned)w.ctas, 0, (size_t)decode::Shape<D>::SMEM, stream,
                              (unsigned)(decode::WARPS * 32), mk, mv, p);
        if (err != cudaSuccess) return static_cast<int>(err);
    }
    // rows of a request for the decode kernel, at most
    const int rows = (a.max_new < sched.decode_tokens ? a.max_new : sched.decode_tokens) * p.n_rep;
    const int chunk_ctas = sched.chunks ? w.pairs * tile::MERGE_CTAS : 0, decode_ctas = sched.decodes ? w.ctas * rows : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(chunk_ctas + decode_ctas), 1, 1);
    cfg.blockDim = dim3(MERGE_THREADS, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    err = cudaLaunchKernelEx(&cfg, khq_paged_merge_kernel<D, BF16>, chunk, p, chunk_ctas, rows);
    if (err != cudaSuccess) return static_cast<int>(err);
    return 0;
}

bool heads_ok(int H_q, int H_kv) { return H_q > 0 && H_kv > 0 && H_q % H_kv == 0 && H_q / H_kv <= MAX_REP; }

int launch_attn(const khq_paged_attn_args* args, bool bf16, cudaStream_t stream) {
    if (!args) return -100;
    const khq_paged_attn_args& a = *args;
    if (a.tokens <= 0 || a.max_tokens <= 0 || a.max_new <= 0 || a.requests <= 0 || a.max_pages <= 0 || a.n_pages <= 0 || a.H_q <= 0 || a.H_kv <= 0 || !a.q ||
        !a.k_cache || !a.v_cache || !a.block_table || !a.schedule || !a.out || !a.workspace)
        return -100;
    const float scale_log2e = a.scale * 1.4426950408889634f;
    if (!(a.scale > 0.0f) || !(scale_log2e <= 3.0e38f)) return -100;
    const int shift = a.page_size == 16 ? 4 : a.page_size == 32 ? 5 : a.page_size == 64 ? 6 : a.page_size == 128 ? 7 : -1;
    if (shift < 0 || (a.d != 128 && a.d != 256) || !heads_ok(a.H_q, a.H_kv) || a.table_stride < a.max_pages) return -103;
    const void* ptrs[] = {a.q, a.gate, a.k_cache, a.v_cache, a.out, a.schedule};
    for (const void* x : ptrs)
        if ((reinterpret_cast<uintptr_t>(x) & 15) != 0) return -104;
    const void* ints[] = {a.block_table, a.lse};
    for (const void* x : ints)
        if ((reinterpret_cast<uintptr_t>(x) & 3) != 0) return -104;
    if ((reinterpret_cast<uintptr_t>(a.workspace) & 255) != 0) return -104;
    for (int i = 0; i < 2; ++i)
        if (((a.q_stride[i] | (a.gate ? a.gate_stride[i] : 0) | a.out_stride[i]) & 7) != 0) return -104;
    for (int i = 0; i < 3; ++i)
        if (((a.k_cache_stride[i] | a.v_cache_stride[i]) & 7) != 0 || a.k_cache_stride[i] < 0 || a.v_cache_stride[i] < 0) return -104;
    const Schedule sched = schedule_of(a.requests, a.max_tokens, a.max_new, a.H_q, a.H_kv, a.d);
    const Work w = work_of(sched, a.d);
    if (a.schedule_bytes < (size_t)sched.ints * 4 || a.workspace_bytes < w.bytes) return -105;
    Params p;
    p.q = static_cast<const uint16_t*>(a.q);
    p.gate = static_cast<const uint16_t*>(a.gate);
    p.out = static_cast<uint16_t*>(a.out);
    p.lse = static_cast<float*>(a.lse);
    p.q_ts = a.q_stride[0];
    p.q_hs = a.q_stride[1];
    p.g_ts = a.gate_stride[0];
    p.g_hs = a.gate_stride[1];
    p.o_ts = a.out_stride[0];
    p.o_hs = a.out_stride[1];
    p.table_stride = a.table_stride;
    p.table = static_cast<const int*>(a.block_table);
    p.tokens = a.tokens;
    p.max_pages = a.max_pages;
    p.n_pages = a.n_pages;
    p.page_shift = shift;
    p.page_mask = a.page_size - 1;
    p.H_q = a.H_q;
    p.H_kv = a.H_kv;
    p.n_rep = a.H_q / a.H_kv;
    p.rep_mul = 65536 / p.n_rep + 1;
    p.scale_log2e = scale_log2e;
    if (a.d == 256) return bf16 ? launch_kernels<256, true>(a, p, sched, w, stream) : launch_kernels<256, false>(a, p, sched, w, stream);
    return bf16 ? launch_kernels<128, true>(a, p, sched, w, stream) : launch_kernels<128, false>(a, p, sched, w, stream);
}

}  // namespace

extern "C" size_t khq_b200_paged_workspace_bytes(int max_new, int H_q, int H_kv, int d) {
    if (max_new <= 0 || !heads_ok(H_q, H_kv) || (d != 128 && d != 256)) return 0;
    return (work_of(schedule_of(1, 1, max_new, H_q, H_kv, d), d).bytes + 255) / 256 * 256;
}

extern "C" int launch_khq_paged_attn_fp16(const khq_paged_attn_args* args, khq_stream_t stream) { return launch_attn(args, false, stream); }

extern "C" int launch_khq_paged_attn_bf16(const khq_paged_attn_args* args, khq_stream_t stream) { return launch_attn(args, true, stream); }

extern "C" int khq_b200_paged_status(void) {
    int st = 0;
    if (cudaMemcpyFromSymbol(&st, khq_paged::g_paged_status, sizeof(int)) != cudaSuccess) return -1;
    if (st != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(khq_paged::g_paged_status, &zero, sizeof(int));
    }
    return st;
}
