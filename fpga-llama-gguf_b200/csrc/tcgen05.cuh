// Tensor memory and FP16 products on the fifth-generation tensor cores (tcgen05), as the prompt attention uses them.
// Waits for the products are mbarrier waits (pipeline.cuh) on a commit.
#pragma once
#include <cstdint>

#include "pipeline.cuh"

namespace b200q {

__device__ __forceinline__ void tm_alloc(uint32_t *dst, unsigned cols) {  // a whole warp; cols a power of two
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_free(uint32_t at, unsigned cols) {  // a whole warp
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory");
}
__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand without swizzle, core matrices of 8 x 16 bytes. K-major (the 16 bytes run along k): `lead` bytes
// between core matrices along k, `stride` bytes along rows. MN-major (the 16 bytes run along rows): `stride` along rows,
// `lead` along k.
__device__ __forceinline__ uint64_t tm_operand(uint32_t addr, unsigned lead, unsigned stride) {
    return uint64_t(addr >> 4 & 0x3FFFu) | uint64_t(lead >> 4) << 16 | uint64_t(stride >> 4) << 32 | uint64_t(1) << 46;
}
// kind::f16, FP16 operands, FP32 sums: M 128, N n; the B operand MN-major or K-major
__device__ __forceinline__ constexpr uint32_t tm_f16(unsigned n, bool b_mn) {
    return 1u << 4 | uint32_t(b_mn) << 16 | (n >> 3) << 17 | (128u >> 4) << 24;
}
// d (tensor memory, 128 lanes) = or += a b^T for 16 of k
__device__ __forceinline__ void tm_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
                 "l"(b), "r"(kind), "r"(uint32_t(add))
                 : "memory");
}
// the same with a in tensor memory (lane: row, a column: two of k)
__device__ __forceinline__ void tm_mma_t(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a),
                 "l"(b), "r"(kind), "r"(uint32_t(add))
                 : "memory");
}
// one arrival on the mbarrier when every product this thread issued before is done
__device__ __forceinline__ void tm_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// N consecutive columns of the warp's 32 lanes (the loads wait for themselves)
__device__ __forceinline__ void tm_load16(uint32_t at, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tm_load32(uint32_t at, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tm_store16(uint32_t at, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
        "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tm_store8(uint32_t at, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

}  // namespace b200q
