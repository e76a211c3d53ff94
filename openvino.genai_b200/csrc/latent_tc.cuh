// Device helpers of the tensor-core kernels of latent attention: tensor-map copies, bounded waits, tensor-memory accesses
// for 64-row accumulators.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "latent_kernels.h"
#include "tc05.cuh"

namespace latent {


__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(pa::smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(pa::smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                     pa::smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(pa::smem_u32(bar))
                 : "memory");
}
// Loads of what is read once or twice in short order: its lines are the first to leave the L2 cache, so that a long cache that streams through
// does not take weights, scratch and the kernels' own code with it.
__device__ __forceinline__ uint64_t evict_first() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(
                     pa::smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(pa::smem_u32(bar)), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void tma_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(
                     pa::smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(pa::smem_u32(bar)), "l"(policy)
                 : "memory");
}
// The same boxes into the L2 cache only.
__device__ __forceinline__ void prefetch_3d(const CUtensorMap* map, int x, int y, int z) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(map), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void prefetch_3d(const CUtensorMap* map, int x, int y, int z, uint64_t policy) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile.L2::cache_hint [%0, {%1, %2, %3}], %4;" ::"l"(map), "r"(x), "r"(y), "r"(z), "l"(policy) : "memory");
}
__device__ __forceinline__ void prefetch_4d(const CUtensorMap* map, int x, int y, int z, int w, uint64_t policy) {
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile.L2::cache_hint [%0, {%1, %2, %3, %4}], %5;" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "l"(policy) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pa::smem_u32(bar)) : "memory");
}
// One arrival for the whole warp, after every lane's preceding writes.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Whether the barrier's phase is complete, without the suspension that try_wait may take: for a warp that watches two barriers.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(pa::smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}

// Waits of a CTA's roles on one another are bounded: one that runs out raises `abort`, which all others poll, and sets the status bit.  The CTA's roles
// then end where they are; once all have, what they had under way is waited for (drain, drain_products) before its memory goes back.
struct Waiter {
    volatile int* abort;
    uint32_t* status;
    uint32_t polls;
    __device__ __forceinline__ bool give_up() const {
        *abort = 1;
        atomicOr(status, PA_DEV_WAIT_TIMEOUT_LATENT);
        return false;
    }
    __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) const {
        for (uint32_t i = 0; i < polls; ++i) {
            if (pa::mbar_try_wait(bar, parity)) return true;
            if ((i & 255u) == 255u && *abort) return false;
        }
        return give_up();
    }
    __device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) const { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; }
    // The same without the suspension: for the warps that hand the tensor core its work, whose every wait is on everybody's way (the attention of
    // 1100 - 2048 new tokens by 32 heads 431 -> 357 us).
    __device__ __forceinline__ bool spin_warp(uint64_t* bar, uint32_t parity) const {
        bool ok = false;
        for (uint32_t i = 0; i < polls << 4; ++i) {
            if (mbar_test(bar, parity)) { ok = true; break; }
            if ((i & 1023u) == 1023u && *abort) break;
        }
        if (__all_sync(0xffffffffu, ok)) return true;
        return give_up();
    }
};

// After an abort: until what was issued on `bar` has arrived, or a millisecond or two, which no copy takes
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    for (int k = 0; k < 4096 && !mbar_test(bar, parity); ++k) __nanosleep(400);
}
// The same for the products of this warp's elected lane; `idle` has had no arrival yet.
__device__ __forceinline__ void drain_products(uint64_t* idle) {
    if (tc05::elect_one()) tc05::commit(idle);
    __syncwarp();
    drain(idle, 0);
}

// Operand descriptors of 128-byte-swizzled tiles whose 8-row groups are GROUP bytes apart.  Their high words are constants, so only the low
// word (address and, for operands whose rows run along M or N, the distance of 64-element atoms) is carried along; a step is an addition.
__host__ __device__ constexpr uint32_t desc_high(uint32_t group_bytes) { return (group_bytes >> 4) | (1u << 14) | (2u << 29); }
__device__ __forceinline__ uint32_t desc_low(const void* smem, uint32_t atom_bytes = 16) {
    return ((pa::smem_u32(smem) >> 4) & 0x3fffu) | ((atom_bytes >> 4) & 0x3fffu) << 16;
}
// D[tmem] (+)= A[smem] * B[smem], issued by one thread; ACC == 0 overwrites D.
template <int ACC, uint32_t AGROUP = 1024, uint32_t BGROUP = 1024>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %6};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "n"(ACC), "n"(desc_high(AGROUP)), "n"(desc_high(BGROUP))
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem].
template <int ACC>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a_tmem), "r"(b), "r"(idesc), "n"(ACC), "n"(desc_high(1024))
        : "memory");
}
// The warp's number as a value that is the same for the whole warp.
__device__ __forceinline__ int warp_id() { return __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two additions or multiply-adds by one instruction.
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 s, t;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\tadd.rn.f32x2 s, s, t;\n\tmov.b64 {%0, %1}, s;\n\t}" : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float factor, float term) {
    asm("{\n\t.reg .b64 s, f, t;\n\tmov.b64 s, {%2, %3};\n\tmov.b64 f, {%4, %4};\n\tmov.b64 t, {%5, %5};\n\tfma.rn.f32x2 s, s, f, t;\n\tmov.b64 {%0, %1}, s;\n\t}"
        : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(factor), "f"(term));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return BF ? pa::pack_bf2(a, b) : pa::pack_h2(a, b);
}
template <bool BF>
__device__ __forceinline__ uint16_t pack1(float a) {
    return (uint16_t)(pack2<BF>(a, 0.f) & 0xffffu);
}
template <bool BF>
__device__ __forceinline__ float unpack1(uint16_t b) {
    return BF ? __bfloat162float(__ushort_as_bfloat16(b)) : __half2float(__ushort_as_half(b));
}

// 16 lanes x 64 columns of a 64-row accumulator: a warp's 16 rows lie in the first 16 of its lanes.  Thread t gets, for every
// group i of eight columns, row t / 4: r[4 i], r[4 i + 1] and row t / 4 + 8: r[4 i + 2], r[4 i + 3], at columns 8 i + 2 (t % 4) and the next.
__device__ __forceinline__ void ld_16x256b_x8(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

}  // namespace latent
