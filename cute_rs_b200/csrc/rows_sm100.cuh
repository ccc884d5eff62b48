// Shared by the products whose weights are chosen row by row: 16-bit
// conversions, tensor maps of row-major 16-bit matrices, small device helpers.
// Internal.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pipe_sm100.cuh"

namespace cb {
namespace {

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t v) {
    if constexpr (BF16) return __uint_as_float(uint32_t(v) << 16);
    else return __half2float(__ushort_as_half(v));
}
template <bool BF16>
__device__ __forceinline__ uint16_t from_f32(float v) {
    if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
    else return __half_as_ushort(__float2half_rn(v));
}
// The two values of a 32-bit word, the lower address first.
template <bool BF16>
__device__ __forceinline__ float2 pair_f32(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ uint32_t pack_16(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}

// The sum of four floats at the same place of the shared memory of a cluster's `kc` <= 8 CTAs, in ascending order; the loads
// are all on their way before the first is used.
__device__ __forceinline__ float4 cluster_sum(uint32_t at, int kc) {
    if (kc == 1) return ptx::ld_shared_cluster_v4(at);
    float4 part[8];
#pragma unroll
    for (int c = 0; c < 8; c++)
        if (c < kc) part[c] = ptx::ld_shared_cluster_v4(ptx::mapa(at, uint32_t(c)));
    float4 v = part[0];
#pragma unroll
    for (int c = 1; c < 8; c++)
        if (c < kc) v.x += part[c].x, v.y += part[c].y, v.z += part[c].z, v.w += part[c].w;
    return v;
}

// The final sums of a cluster: out(i, sum of the CTAs' floats at at(i)) for items i of 0 .. items - 1, shared by the cluster's
// threads.  TURN items per turn: their loads are on their way together (a turn takes some 0.8 us with any number of them).
template <int TURN, typename At, typename Out>
__device__ __forceinline__ void cluster_sums(int items, int rank, int kc, int threads, At at, Out out) {
    const int stride = kc * threads;
    for (int first = rank * threads; first < items; first += TURN * stride) {  // the same for the whole CTA
        const int i0 = first + int(threadIdx.x);
        float4 v[TURN];
#pragma unroll
        for (int u = 0; u < TURN; u++)
            if (first + u * stride < items) v[u] = cluster_sum(at(min(i0 + u * stride, items - 1)), kc);
#pragma unroll
        for (int u = 0; u < TURN; u++)
            if (i0 + u * stride < items) out(i0 + u * stride, v[u]);
    }
}

// i / n by a product, for i * n < 2^20.
struct Divider {
    uint32_t factor;
    __device__ __forceinline__ explicit Divider(int n) : factor((1u << 20) / uint32_t(n) + 1u) {}
    __device__ __forceinline__ int operator()(int i) const { return int((uint32_t(i) * factor) >> 20); }
};

// Tensor map of a row-major 16-bit matrix of `rows` x `cols`, `pitch` elements between rows, in boxes of 64 columns
// (one 128-byte swizzled row) by box_rows; what lies outside reads as zero.  Encoded anew for every call: it takes
// a fraction of a microsecond on the host, and nothing is kept by an operand's address.
inline cute_b200_status rows_tensor_map(CUtensorMap *tm, uint64_t base, bool bf16, uint64_t rows, uint64_t cols, uint64_t pitch, int box_rows) {
    EncodeTiledFn encode;
    CB_TRY(encode_fn(&encode));
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {pitch * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(box_rows)};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult r = encode(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                              reinterpret_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(CUTE_B200_ERR_CUDA, "cuTensorMapEncodeTiled failed: CUresult %d (rows %llu, columns %llu, box %d)", int(r),
                    (unsigned long long)rows, (unsigned long long)cols, box_rows);
    return CUTE_B200_OK;
}

// The same of `count` matrices one behind the other: a box lies within one of them, what lies outside reads as zero.
inline cute_b200_status stack_tensor_map(CUtensorMap *tm, uint64_t base, bool bf16, uint64_t count, uint64_t rows, uint64_t cols, int box_rows) {
    EncodeTiledFn encode;
    CB_TRY(encode_fn(&encode));
    const cuuint64_t dims[3] = {cols, rows, count};
    const cuuint64_t strides[2] = {cols * 2, rows * cols * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(box_rows), 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult r = encode(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                              reinterpret_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(CUTE_B200_ERR_CUDA, "cuTensorMapEncodeTiled failed: CUresult %d (%llu matrices of %llu x %llu, box %d)", int(r),
                    (unsigned long long)count, (unsigned long long)rows, (unsigned long long)cols, box_rows);
    return CUTE_B200_OK;
}

// Shared-memory matrix descriptor of an MN-major tile in 128-byte rows with the 128B swizzle: 64 values of M or N per
// row, the rows are k.  Leading byte offset: from 64 values to the next 64, one box of `box_bytes`; stride byte offset:
// from eight k to the next eight.  16 k further: MN_K_STEP in the address field.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr, uint32_t box_bytes) {
    return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(box_bytes >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}
constexpr uint32_t MN_K_STEP = (16 * 128) >> 4;
constexpr uint32_t IDESC_A_MN = 1u << 15, IDESC_B_MN = 1u << 16;  // instruction descriptor: that operand is MN-major

// Launch as a programmatic dependent of the kernel before it in the stream, in clusters of `cluster` CTAs.
template <typename... P, typename... A>
cute_b200_status launch_dependent(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream,
                                  const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[3];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[2].id = cudaLaunchAttributeClusterSchedulingPolicyPreference;
    attr[2].val.clusterSchedulingPolicyPreference = cudaClusterSchedulingPolicySpread;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 3 : 1;
    CB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    count_launch();
    return CUTE_B200_OK;
}

// How many clusters of `size` CTAs of a kernel the current device can hold at once.
template <typename... P>
cute_b200_status max_clusters(void (*kernel)(P...), int threads, size_t smem, int size, int *out) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(size));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CB_CUDA(cudaOccupancyMaxActiveClusters(out, kernel, &cfg));
    return CUTE_B200_OK;
}

// k blocks per ring stage of a product that streams `bn` rows of a weight past `rows` rows: 10 to 40 KB of the weight (more or
// less with another `wide`, the rows that make a stage alone), but at least four stages in a ring of `ring` bytes.
inline int stream_blocks(int bn, int rows, uint32_t ring, int wide = 160) {
    int blocks = bn >= wide ? 1 : (2 * bn >= wide ? 2 : 4);
    while (blocks > 1 && ring / (uint32_t(blocks * (rows + bn)) * 128u) < 4) blocks /= 2;
    return blocks;
}

// How a product that streams an (n, k) weight past a few rows is cut: bn rows of the weight per tile, a cluster of kc CTAs per tile.  The launch is one wave
// where it can be; the cut with the least time for the slowest CTA wins.  A CTA streams at most what an even share of
// HBM gives it, and no faster than its MMAs are issued (per k block four of 65 clocks or bn / 2 each, and some 80 of loop).
// `more`: rows of another matrix that every tile streams beside its own.
inline void stream_cut(int n, int k_blocks, const int (&max_clusters)[4], int *bn, int *kc, int more = 0) {
    double best = 1e300;
    for (int c = 0; c < 4; c++) {
        const int parts = 1 << c, ctas_at_once = max_clusters[c] * parts;
        if (parts > k_blocks || max_clusters[c] < 1) continue;
        for (int b = 16; b + more <= 256; b += 16) {
            const int64_t ctas = int64_t((n + b - 1) / b) * parts;
            const int64_t waves = (ctas + ctas_at_once - 1) / ctas_at_once;
            const double share = 6.5e12 / double(ctas < ctas_at_once ? ctas : ctas_at_once);
            const double rate = share < 7.0e10 ? share : 7.0e10;
            const int cols = b + more;
            const double load = cols * 128.0 / rate, math = (4.0 * (cols / 2 > 65 ? cols / 2 : 65) + 80.0) / 1.8e9;
            const double t = double(waves) * (((k_blocks + parts - 1) / parts) * (load > math ? load : math) + 2.0e-6) + (parts > 1 ? 1.0e-6 : 0.0);
            if (t < best * 0.999) best = t, *bn = b, *kc = parts;
        }
    }
}

}  // namespace
}  // namespace cb
