// Device helpers of the 8-bit kernels: quantising a group of 128 values, tensor-core products of e4m3 tiles, waits that end.
#pragma once

#include "t3_common.cuh"
#include "t3_tcgen05.cuh"

namespace t3 {

// The scale of a group whose largest magnitude has the bits `most` (as an f32 without its sign): the smallest power of two s with
// most / s <= 448 = 1.75 * 2^8, at least 2^-126; a NaN for a group that holds an infinity or a NaN. A power of two, so that x / s
// is exact and a value's rounding to e4m3 is the only one: the format floats, so nothing but its smallest values would gain from
// a scale that fills its range.
__device__ __forceinline__ float fp8_scale(uint32_t most) {
    if (most >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const int e = (int)(most >> 23) - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return __uint_as_float((uint32_t)(e < 1 ? 1 : e) << 23);
}
// 1 / s of a scale of fp8_scale (exponent field 1 .. 247, so the inverse is a normal number too)
__device__ __forceinline__ float fp8_inverse(float s) { return __uint_as_float(0x7F000000u - __float_as_uint(s)); }

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// two values to e4m3, to nearest even (a NaN to the format's): a in the low byte
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t to_e4m3x4(const float (&v)[4], float s) {
    // the inverse of a NaN scale is not looked at: every value becomes the NaN
    const float i = isnan(s) ? s : fp8_inverse(s);
    return to_e4m3x2(v[0] * i, v[1] * i) | (to_e4m3x2(v[2] * i, v[3] * i) << 16);
}

// D[tmem] (+)= A[smem] x B[smem]^T, e4m3 x e4m3 -> f32, K = 32 (32 bytes of both K-major tiles); the instruction descriptor is
// idesc_m128's: format 0 is e4m3 in this kind
__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t accumulate, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 tensor-memory lanes x 16 f32 columns on their way, r[j] column j of the thread's lane; tmem_ld_wait before their use
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// (c.x, c.y) += (a0 b0, a1 b1): two f32 multiply-adds in one instruction
__device__ __forceinline__ void fma2(float2& c, uint32_t a0, uint32_t a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
        : "+f"(c.x), "+f"(c.y)
        : "r"(a0), "r"(a1), "f"(b0), "f"(b1));
}

// load_act past L1
__device__ __forceinline__ float load_act_cg(const void* p, int dt, size_t i) {
    if (dt == kF32) return __ldcg(static_cast<const float*>(p) + i);
    const uint16_t b = __ldcg(static_cast<const unsigned short*>(p) + i);
    return dt == kF16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
}

// Waits for a barrier phase; gives up after a while, or at once when any wait of the CTA has given up (`dead`): every role then
// still walks to its end, on values nobody will use, and the error word says so. CLUSTER: what other CTAs of the cluster wrote
// before their arrivals is visible after it. The loop is a call: these kernels' code comes from memory again for every launch, behind the
// weights that have passed through L2, and what it does not hold it does not wait for. (fp8_wait_here: the loop in place, for a caller
// with so many registers in use that keeping them ready for a call costs more.)
// LAST: the wait that has run out takes some 50 us more, in which what the warp has issued (copies into this CTA's shared memory or out of it,
// products into its tensor memory) ends. A warp that issues has one behind its last issue, so nothing is under way when the CTA gives its memory
// back. (A look at `dead` at the CTA's end, or ahead of every issue, cost each call 0.2 to 0.4 us.)
constexpr uint32_t kFp8Tries = 1u << 20;  // of 1.5 us each
template <bool CLUSTER = false>
__device__ __forceinline__ bool fp8_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    if (CLUSTER)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
    else
        done = mbar_try(bar, parity);
    return done != 0u;
}
template <bool CLUSTER, bool LAST>
__device__ __forceinline__ void fp8_wait_here(uint32_t bar, uint32_t parity, volatile uint32_t* dead, uint32_t* err, uint32_t bit) {
    uint32_t i = 0;
#pragma unroll 1
    for (; i < kFp8Tries; ++i) {
        if (fp8_try<CLUSTER>(bar, parity)) return;
        if (*dead) break;
    }
    if (i == kFp8Tries) {
        *dead = 1u;
        if (err) atomicOr(err, bit);
    }
    if (LAST)
#pragma unroll 1
        for (i = 0; i < 50u; ++i) __nanosleep(1000);
}
template <bool CLUSTER>
__device__ __noinline__ void fp8_wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* dead, uint32_t* err, uint32_t bit) {
    fp8_wait_here<CLUSTER, true>(bar, parity, dead, err, bit);
}
template <bool CLUSTER = false>
__device__ __forceinline__ void fp8_wait(uint32_t bar, uint32_t parity, volatile uint32_t* dead, uint32_t* err, uint32_t bit) {
    if (!fp8_try<CLUSTER>(bar, parity)) fp8_wait_slow<CLUSTER>(bar, parity, dead, err, bit);
    __syncwarp();  // (whole warps wait)
}

// `bytes` (4 or 16) from global to shared memory, in this thread's copy group
template <uint32_t BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if (BYTES == 16u) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits until all but this thread's last N copy groups are in place
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- thread-block clusters ----
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// a shared-memory address of this CTA as the same place in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// v to another CTA's shared memory; its four bytes count on the barrier there (both addresses of peer_addr). No fence: a release at cluster
// scope waits for every earlier store of the thread, those to global memory too (4 us a task under a full load of copies). Only in a
// launch with a cluster: without one the instruction is illegal.
__device__ __forceinline__ void peer_store(uint32_t addr, float v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr), "r"(__float_as_uint(v)), "r"(bar) : "memory");
}
// `bytes` (a multiple of 16, both ends on 16 bytes) of this CTA's shared memory to another's, counted on the barrier there. What the copy reads was
// written ahead of a proxy_fence. For more than a value or two a thread: a peer_store is a transaction a lane (64 KB of them took 3 to 5 us).
__device__ __forceinline__ void peer_copy(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void peer_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// a box on its way into L2 only: harmless ahead of a wait for the stream's previous kernel, whatever that one writes
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y)
                 : "memory");
}

}  // namespace t3
