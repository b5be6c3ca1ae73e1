// Tensor-core products, their TMEM and their descriptors (sm_100a).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace swb {

constexpr int kScaleBlock = 512;  // bytes: scales of 128 rows x 4 blocks of 32 values, as tcgen05.cp reads them

__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives on `bar` once every tcgen05 operation this thread issued so far is done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void scale_copy(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(uint32_t(accumulate)) : "memory");
}
__device__ __forceinline__ void mma_mxf8f6f4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                             bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(uint32_t(accumulate)) : "memory");
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate)) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptors: K-major rows of 128 swizzled bytes, groups of eight
// rows 1024 bytes apart; scale blocks: unswizzled 16-byte rows, groups of eight 128 apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
    return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(1) << 16) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}

// Instruction descriptors: K-major operands, fp32 sums, M x N. `id`: the byte of a scale word that
// the step takes (kind::mxf8f6f4: one block of 32 values), or the first of two (kind::mxf4).
__device__ __forceinline__ constexpr uint32_t mxf4_desc(int m, int n, int id) {  // e2m1 x e2m1, E8M0 scales
    return (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(m >> 7) << 27) |
           (uint32_t(id) << 4) | (uint32_t(id) << 29);
}
__device__ __forceinline__ constexpr uint32_t mxf8f6f4_desc(int m, int n, int id) {  // e2m1 x e4m3, E8M0 scales
    return (5u << 7) | (0u << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(m >> 7) << 27) |
           (uint32_t(id) << 4) | (uint32_t(id) << 29);
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t f16_desc(int m, int n) {
    constexpr uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (f << 7) | (f << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// One window of a row's scale bytes: bytes [b0, b0 + 16) of `blocks`, zero beyond.
__device__ __forceinline__ uint4 load_scales(const unsigned char* row, int b0, int blocks) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if ((blocks & 15) == 0 && (reinterpret_cast<uintptr_t>(row) & 15) == 0) {
        if (b0 < blocks) return __ldg(reinterpret_cast<const uint4*>(row + b0));
    } else if ((blocks & 3) == 0 && (reinterpret_cast<uintptr_t>(row) & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (b0 + 4 * i < blocks) w[i] = __ldg(reinterpret_cast<const uint32_t*>(row + b0) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (b0 + i < blocks) w[i >> 2] |= uint32_t(__ldg(row + b0 + i)) << (8 * (i & 3));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace swb
