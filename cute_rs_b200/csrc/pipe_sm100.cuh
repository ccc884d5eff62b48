// What the tcgen05 kernels of this library share: descriptors, bounded waits,
// the driver's tensor-map encoder.  Internal.
#pragma once

#include <cuda.h>

#include <mutex>

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace cb {
namespace {

constexpr uint64_t WAIT_LIMIT_NS = 4ull * 1000 * 1000 * 1000;

// Report codes written to the status word.
enum : uint32_t {
    WHERE_PRODUCER = 1,
    WHERE_MMA_FULL = 2,
    WHERE_MMA_TMEM = 3,
    WHERE_EPILOGUE = 4,
    WHERE_DRAIN = 5,
    WHERE_PUSHER = 6,
    WHERE_SIGNAL = 7  // cute_b200_wait_signal: the counter did not reach the expected value in time
};

// Instruction descriptor of tcgen05.mma.kind::f16: f32 accumulator (bit 4), A and B format (0 = f16,
// 1 = bf16) at bits 7 and 10, both operands K-major (bits 15, 16 clear), N >> 3 at bit 17, M >> 4 at
// bit 24, M counting the rows of the whole CTA group.
__host__ __device__ constexpr uint32_t make_idesc(bool bf16, int umma_m, int bn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | (uint32_t(bn >> 3) << 17) |
           (uint32_t(umma_m >> 4) << 24);
}

// Shared-memory matrix descriptor of a K-major tile stored as 128-byte rows
// with the 128B swizzle (what TMA writes with CU_TENSOR_MAP_SWIZZLE_128B):
// start address >> 4, leading byte offset 1 (unused by swizzled K-major),
// stride byte offset 1024 (eight rows), descriptor version 1, layout 2.
__host__ __device__ __forceinline__ constexpr uint64_t sw128_desc(uint32_t saddr) {
    return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

__device__ __noinline__ void report_timeout(uint32_t *status, uint32_t where, uint32_t detail, uint32_t parity) {
    if (atomicCAS(status, 0u, where) == 0u) {
        status[1] = detail;
        status[2] = blockIdx.x;
        status[3] = parity;
        __threadfence();
    }
}

// Wait for phase `parity` of `bar`.  false = gave up (limit or CTA abort).
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag,
                                         uint32_t *status, uint32_t where, uint32_t detail,
                                         uint64_t limit_ns = WAIT_LIMIT_NS) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = ptx::globaltimer_ns();
    uint32_t spins = 0;
    for (;;) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        if ((++spins & 255u) == 0u) {
            if (*abort_flag) return false;
            if (ptx::globaltimer_ns() - t0 > limit_ns) {
                *abort_flag = 1u;
                report_timeout(status, where, detail, parity);
                return false;
            }
        }
    }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cute_b200_status encode_fn(EncodeTiledFn *out) {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    static cudaError_t err = cudaSuccess;
    std::call_once(once, [] {
        void *sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        err = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &sym, 12000, cudaEnableDefault, &q);
        if (err == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = reinterpret_cast<EncodeTiledFn>(sym);
    });
    if (!fn) return fail(CUTE_B200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    *out = fn;
    return CUTE_B200_OK;
}

}  // namespace
}  // namespace cb
