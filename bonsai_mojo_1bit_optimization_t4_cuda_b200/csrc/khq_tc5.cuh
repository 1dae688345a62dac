// khq_tc5.cuh -- tcgen05, tensor-memory, TMA and barrier wrappers of the prompt kernels (khq_prefill_tc5.cu, khq_prefill_pair.cuh,
// khq_paged_attn.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "khq_common.cuh"

namespace khq_tc5 {

using khq::smem_u32;

// ---- descriptors ---------------------------------------------------------------------------------
// Shared-memory matrix descriptor (64 bits): start address, leading and stride byte offsets (all in
// 16-byte units; bits 0-13, 16-29, 32-45), descriptor version 1 in bits 46-47, layout type 2
// (128-byte swizzle) in bits 61-63.  It is assembled from a low and a high word, see desc_lo/desc_hi.
// Instruction descriptor for kind::f16: fp32 accumulate, fp16 A and B, A K-major, M = 128 (256: a CTA pair).
// (A/B format field: 0 = fp16, 1 = bf16, bits 7-9 and 10-12.)
__host__ __device__ constexpr uint32_t instr_desc(int m, int n, bool b_mn_major, bool bf16) {
    return (1u << 4) | (bf16 ? ((1u << 7) | (1u << 10)) : 0u) | (b_mn_major ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
// Two floats -> one 32-bit word of the 16-bit storage type (round to nearest even), and back.
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
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// ---- tcgen05 / TMA wrappers ----------------------------------------------------------------------
// The issuing warp is on the critical path: the 64-bit descriptors are assembled from a
// precomputed low word (start address and leading offset; the caller adds the K-step offset, which
// never carries out of the 14-bit address field) and a constant high word.  umma_ss: A and B from
// shared memory; umma_ts: A from tensor memory (row = lane, fp16 pairs, 8 columns per K step of 16).
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
    return ((addr & 0x3FFFFu) >> 4) | (((lbo >> 4) & 0x3FFFu) << 16);
}
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo) {
    return ((sbo >> 4) & 0x3FFFu) | (1u << 14) | (2u << 29);  // version 1 (bit 46), 128-byte swizzle (bits 61-63)
}
// All lanes of the MMA warp call these and one of them issues (`one`): the operands are then values of the whole warp, which the
// compiler keeps and steps in uniform registers (see khq_prefill_pair.cuh).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r));
    return r;
}
template <int ACC>
__device__ __forceinline__ void umma_ss(uint32_t one, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .b64 da, db;\n\t.reg .pred p, q;\n\t"
        "mov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
        "setp.ne.u32 p, %6, 0;\n\tsetp.ne.u32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(ACC), "r"(one)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .b64 db;\n\t.reg .pred p, q;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.u32 p, %5, 0;\n\tsetp.ne.u32 q, %6, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(one)
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / (1 + e^-x): four instructions, two of them approximations of 2^-22 relative error; subnormal terms are below the sum's rounding
// (and below 2^-126 of the result).
__device__ __forceinline__ float sigmoid(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + ex2_approx(x * -1.4426950408889634f)));
    return y;
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A piece of the gates to L2; a piece of the outputs from shared memory.
__device__ __forceinline__ void tma_prefetch_5d(const CUtensorMap* map, int c1, int c2, int c3, int c4) {
    asm volatile("cp.async.bulk.prefetch.tensor.5d.L2.global.tile [%0, {%1, %2, %3, %4, %5}];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
                 : "memory");
}
__device__ __forceinline__ void tma_store_5d(const CUtensorMap* map, uint32_t src, int c1, int c2, int c3, int c4) {
    asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// One 5-D tiled TMA load of a single CTA; coordinate 0 is always 0, so the 16-byte rule holds.
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c1, int c2,
                                            int c3, int c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, "
        "%6, %7}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

// Bounded wait on up to three barriers at once.  A satisfied mbarrier wait still costs a ~250-cycle
// round trip, so the MMA warp polls the barriers of a step together (the polls overlap) instead
// of one after the other; a barrier found complete stays "done" (its next phase cannot complete
// before this thread moves on).
__device__ __forceinline__ uint32_t mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok;
}
// Waits of a whole warp: all lanes go on together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {
    for (uint32_t it = 0; it < (1u << 22); ++it)
        if (__any_sync(0xFFFFFFFFu, khq::mbar_try_wait(bar, parity))) return true;
    atomicExch(status, 1);
    return false;
}
template <int N>
__device__ __forceinline__ bool mbar_wait_all_bounded(uint64_t* const (&bar)[N], const uint32_t (&parity)[N], int* status) {
    uint32_t done = 0;
    for (uint32_t it = 0; it < (1u << 22); ++it) {
        uint32_t got[N];
#pragma unroll
        for (int i = 0; i < N; ++i) got[i] = mbar_test(bar[i], parity[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) done |= (uint32_t)__any_sync(0xFFFFFFFFu, got[i]) << i;
        if (done == (1u << N) - 1u) return true;
        bool parked = false;  // park (a blocking try_wait) on the first barrier that is still open
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!parked && !((done >> i) & 1u)) {
                if (__any_sync(0xFFFFFFFFu, khq::mbar_try_wait(bar[i], parity[i]))) done |= 1u << i;
                parked = true;
            }
        if (done == (1u << N) - 1u) return true;
    }
    atomicExch(status, 1);
    return false;
}

// ---- CTA pairs (cta_group::2) and packed arithmetic ------------------------------------------------
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// (d0, d1) = (a0, a1) m + c and (s0, s1) += (a0, a1), one packed instruction each
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float m, float c) {
    asm("{.reg .b64 a, m, c, d; mov.b64 a, {%2, %3}; mov.b64 m, {%4, %4}; mov.b64 c, {%5, %5}; fma.rn.f32x2 d, a, m, c; mov.b64 {%0, %1}, d;}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(m), "f"(c));
}
__device__ __forceinline__ void add2(float& s0, float& s1, float a0, float a1) {
    asm("{.reg .b64 a, s; mov.b64 a, {%2, %3}; mov.b64 s, {%0, %1}; add.rn.f32x2 s, s, a; mov.b64 {%0, %1}, s;}" : "+f"(s0), "+f"(s1) : "f"(a0), "f"(a1));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
// The MMA warp stays together and one lane issues (`one`): its descriptors are then values of the whole warp, kept and stepped in uniform
// registers.  With one lane alone inside a branch each instruction's operands had to be moved there one by one, which took about as
// long as the pipe takes for the instruction, or longer by the luck of the code's placement (4 x 8192: 2.42 ms, 2.49 to 2.95).
template <int ACC>
__device__ __forceinline__ void umma2_ss(uint32_t one, uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .b64 da, db;\n\t.reg .pred p, q;\n\t"
        "mov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
        "setp.ne.u32 p, %6, 0;\n\tsetp.ne.u32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(ACC), "r"(one)
        : "memory");
}
__device__ __forceinline__ void umma2_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .b64 db;\n\t.reg .pred p, q;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.u32 p, %5, 0;\n\tsetp.ne.u32 q, %6, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
// Arrives at this barrier of both CTAs once the instructions issued so far have completed.
__device__ __forceinline__ void umma2_commit(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3), "r"(one)
        : "memory");
}
// The address of `bar` in the pair's first CTA.
__device__ __forceinline__ uint32_t in_leader(uint64_t* bar) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(bar)));
    return r;
}
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_leader(bar)) : "memory");
}
// A load into this CTA's shared memory whose bytes count at a barrier of the pair's first CTA.
__device__ __forceinline__ void load_for_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c1, int c2, int c3, int c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5, "
        "%6, %7}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}
// Of the MMA warp's barriers too: the other CTA's arrivals announce tensor-memory contents and asynchronous copies, which the tcgen05
// fences and the copies' byte counts order, not ordinary memory.  Acquiring at cluster scope cost 4 to 8 %.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

}  // namespace khq_tc5
