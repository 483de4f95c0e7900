// mbarriers, tcgen05 and TMEM: the PTX that the tiled and the clustered kernels share.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace gsb {

constexpr unsigned kWaitLimit = 1u << 22; // polls of about a microsecond at most

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(unsigned long long *b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void mbar_expect(unsigned long long *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(unsigned long long *b, uint32_t phase) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done)
                 : "r"(smem_u32(b)), "r"(phase), "r"(1000u)
                 : "memory");
    return done != 0;
}
// False when the wait ran out, here or in another role of the block.
__device__ __forceinline__ bool mbar_wait(unsigned long long *b, uint32_t phase, volatile int *abort) {
    for (unsigned i = 0; i < kWaitLimit; ++i) {
        if (mbar_try(b, phase)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    return false;
}

// Products are issued by a whole warp under the predicate `leader`, true in one lane: the
// descriptors are then computed in uniform registers, where the instruction wants them. Issued from a
// branch of one thread, each took 85 cycles, more than most products last.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0); }
__device__ __forceinline__ uint32_t elect_leader() {
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
    return e;
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t leader) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned long long *bar, uint32_t leader) {
    asm volatile("{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
                 " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar)), "r"(leader)
                 : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, float v[32]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
                 "tcgen05.wait::ld.sync.aligned;" // in one statement: nothing that uses v comes between
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void tmem_load16(uint32_t addr, float v[16]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}

// Shared-memory descriptor of a 128-byte-swizzled fp16 operand. Depth-major (K-major):
// rows of 128 bytes, groups of 8 rows 1024 bytes apart (chunk unused). The other way
// (N-major): 64 columns x 8 depths a 1024-byte group, the next 64 columns `chunk` bytes on.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool k_major, uint32_t chunk) {
    const uint64_t lbo = k_major ? 1 : chunk / 16, sbo = 1024 / 16;
    return (uint64_t)((addr & 0x3ffff) >> 4) | lbo << 16 | sbo << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: fp16 x fp16 -> fp32, 128 rows x n, Q N-major or not.
__device__ __forceinline__ uint32_t mma_desc(int n, bool q_k_major) {
    return 1u << 4 | (q_k_major ? 0u : 1u << 16) | (uint32_t)(n / 8) << 17 | (uint32_t)(128 / 16) << 24;
}

} // namespace gsb
