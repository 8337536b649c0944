// Copies by the copy engine into shared memory, counted by barriers whose waits end, for the operators on learned and compressed rows.
#pragma once
#include "common.cuh"

namespace legion {

__device__ __forceinline__ uint32_t shared_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void init_barrier(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Both addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Waits until the barrier's phase of that parity is over: at most `tries` times kTryUs microseconds (once, where tries is 0), then false.
constexpr int kTryUs = 20;
__device__ __forceinline__ bool wait_barrier(uint32_t bar, uint32_t parity, uint32_t tries)
{
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, %3;\n"
        "TRY:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n @p bra DONE;\n sub.u32 n, n, 1;\n setp.gt.s32 q, n, 0;\n @q bra TRY;\n"
        "DONE:\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(tries) : "memory");
    return ok != 0;
}

// What a launch asks for once per device and kernel: more than 48 KB of shared memory.
inline int allow_smem(const void *kernel, int bytes, bool *done)
{
    int dev = 0;
    LG_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !done[dev]) {
        LG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) done[dev] = true;
    }
    return LEGION_OK;
}

// Tries of a wait inside a launch made now (legion_operator_wait_limit): two seconds' worth, unless the caller has set another limit.
uint32_t operator_wait_tries();

// Kernels of two files raise errors, each in a word of its own file's (legion_operator_error reads both).
cudaError_t norm_error_word(void **word);

}  // namespace legion
