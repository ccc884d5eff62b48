// Shared by the translation units of lora_tn and its gradients.  Internal.
#pragma once

#include "rows_sm100.cuh"

namespace cb {

struct LoraParams {
    const uint16_t *x, *w, *a, *b;
    const int32_t *ids;
    const float *scale;
    void *y;
    uint16_t *t;    // (m, t_planes() rp): the inner products, see store_t
    uint32_t *plan; // which adapters each tile of rows names (tiled kernels)
    int m, n, k, rank, rp, adapters, c_dtype;
    int64_t ldx, ldy;
    // The backward product: `a` is (adapters, k, rank) and `b` (adapters, rank, n), the forward's matrices as they lie, read
    // as MN-major operands; and the kernel before T's is one that T's need not wait for (the row lists).
    bool low_mn;
};

// The tiled forward product (any m; cut 0..3 names a tile, a negative one chooses) and the bytes of its plan.
cute_b200_status lora_tiled(const LoraParams &p, bool bf16, int cut, int debug, const DeviceState &dev, cudaStream_t stream);
uint64_t lora_plan_bytes(int m, int adapters);
cute_b200_status lora_tiled_init(DeviceState &dev);

// The adapters' gradients: [0] dA from X and U, [1] dB from dY and T.  `first` (adapters + 1) and `list` (m) are the row lists.
struct LoraGrads {
    float *out[2];
    const uint16_t *wide[2], *low[2];
    int64_t pitch[2];
    int cols[2], m, rank, rp, adapters;
    const int32_t *first, *list;
};
cute_b200_status lora_row_lists(const int32_t *ids, int m, int adapters, int32_t *first, int32_t *list, cudaStream_t stream);
cute_b200_status lora_grads(const LoraGrads &g, bool bf16, int debug, const DeviceState &dev, cudaStream_t stream);
cute_b200_status lora_grad_init();

namespace {

__device__ __forceinline__ void store_c(void *c, int dtype, size_t i, float v) {
    if (dtype == CUTE_B200_F32) static_cast<float *>(c)[i] = v;
    else if (dtype == CUTE_B200_BF16) static_cast<__nv_bfloat16 *>(c)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(c)[i] = __float2half_rn(v);
}

// Width of the rank in T: 16, 32, 64 or 128.
__host__ __device__ constexpr int padded_rank(int rank) { return rank <= 16 ? 16 : (rank <= 32 ? 32 : (rank <= 64 ? 64 : 128)); }

// How T is stored: per row `t_planes` planes of rp numbers.  A value v is split into its rounding and a remainder, v = hi + lo.
//   bf16  hi, lo:           16 bits of v at any magnitude.
//   f16   lo, hi, lo 2^11:  the remainder of a value below 1/4 falls below f16's smallest step, so hi + lo is off by up to
//         2^-25 whatever v is.  Towards Y, whose accumulator takes hi and lo as they are, that is f16's own resolution.  A gradient
//         has no such floor: its kernel sums the scaled remainders in columns of their own and scales them back in f32, which
//         keeps 22 bits down to 2^-14 and is off by 2^-36 below.  (2^12 would overflow for values above 2^15.)
// Y reads planes 0 and 1, or hi alone; the gradients two planes from hi on.
__host__ __device__ constexpr int t_planes(bool bf16) { return bf16 ? 2 : 3; }
__host__ __device__ constexpr int t_hi(int rp, bool bf16) { return bf16 ? 0 : rp; }
constexpr float LOW_SCALE = 2048.0f;
template <bool BF16>
__device__ __forceinline__ void store_t(uint16_t *t, int rp, float v) {
    const uint16_t hi = from_f32<BF16>(v);
    const float lo = v - to_f32<BF16>(hi);
    t[t_hi(rp, BF16)] = hi;
    t[BF16 ? rp : 0] = from_f32<BF16>(lo);
    if constexpr (!BF16) t[2 * rp] = from_f32<BF16>(lo * LOW_SCALE);
}
// Four of them, 8-byte aligned.  Returns hi + lo.
__device__ __forceinline__ float4 store_t4(uint16_t *t, int rp, const float4 &v, bool bf16, bool store = true) {
    const uint32_t h0 = pack_16(v.x, v.y, bf16), h1 = pack_16(v.z, v.w, bf16);
    const float2 f0 = bf16 ? pair_f32<true>(h0) : pair_f32<false>(h0), f1 = bf16 ? pair_f32<true>(h1) : pair_f32<false>(h1);
    const float4 lo = make_float4(v.x - f0.x, v.y - f0.y, v.z - f1.x, v.w - f1.y);
    const uint32_t l0 = pack_16(lo.x, lo.y, bf16), l1 = pack_16(lo.z, lo.w, bf16);
    if (store) {
        *reinterpret_cast<uint2 *>(t + t_hi(rp, bf16)) = make_uint2(h0, h1);
        *reinterpret_cast<uint2 *>(t + (bf16 ? rp : 0)) = make_uint2(l0, l1);
        if (!bf16)
            *reinterpret_cast<uint2 *>(t + 2 * rp) = make_uint2(pack_16(lo.x * LOW_SCALE, lo.y * LOW_SCALE, bf16), pack_16(lo.z * LOW_SCALE, lo.w * LOW_SCALE, bf16));
    }
    const float2 g0 = bf16 ? pair_f32<true>(l0) : pair_f32<false>(l0), g1 = bf16 ? pair_f32<true>(l1) : pair_f32<false>(l1);
    return make_float4(f0.x + g0.x, f0.y + g0.y, f1.x + g1.x, f1.y + g1.y);
}

// First occurrences of ids by a hash table in shared memory.
template <int ROWS>
struct IdTable {
    static constexpr int SIZE = 2 * ROWS;  // 256, 512 or 1024: at most half full, so a probe ends
    static_assert(ROWS == 128 || ROWS == 256 || ROWS == 512, "the hash keeps log2(SIZE) bits");
    int32_t key[SIZE], first[SIZE], entry[SIZE], before[4];
};

// The distinct ids of ROWS rows (128, 256 or 512; negative = none) in the order of their first row, by 128 threads that all
// call this: thread t holds rows t, t + 128, ..  emit(e, id) receives the list; mine[i] becomes the place in it of row
// t + 128 i (-1 = none).  Returns the length.  The order does not depend on timing: `first` is a minimum over rows.
template <int ROWS, typename Emit>
__device__ __forceinline__ int distinct_ids(const int32_t (&id)[ROWS / 128], IdTable<ROWS> &h, int t, int32_t (&mine)[ROWS / 128], Emit emit) {
    constexpr int N = ROWS / 128;
    const int lane = t & 31, w = t >> 5;
    for (int i = t; i < h.SIZE; i += 128) h.key[i] = -1, h.first[i] = 0x7fffffff;
    ptx::named_barrier(1, 128);
    uint32_t slot[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        slot[i] = (uint32_t(id[i]) * 2654435761u) >> (ROWS == 128 ? 24 : (ROWS == 256 ? 23 : 22));  // SIZE slots
        if (id[i] >= 0) {
            for (;;) {
                const int old = atomicCAS(&h.key[slot[i]], -1, id[i]);
                if (old == -1 || old == id[i]) break;
                slot[i] = (slot[i] + 1u) & uint32_t(h.SIZE - 1);
            }
            atomicMin(&h.first[slot[i]], t + 128 * i);
        }
    }
    ptx::named_barrier(1, 128);
    int total = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const bool first = id[i] >= 0 && h.first[slot[i]] == t + 128 * i;
        __syncwarp();
        const uint32_t firsts = __ballot_sync(0xffffffffu, first);
        if (lane == 0) h.before[w] = __popc(firsts);
        ptx::named_barrier(1, 128);
        int at = total + __popc(firsts & ((1u << lane) - 1u));
        for (int j = 0; j < 4; j++) {
            if (j < w) at += h.before[j];
            total += h.before[j];
        }
        if (first) {
            h.entry[slot[i]] = at;
            emit(at, id[i]);
        }
        ptx::named_barrier(1, 128);
    }
#pragma unroll
    for (int i = 0; i < N; i++) mine[i] = id[i] >= 0 ? h.entry[slot[i]] : -1;
    return total;
}

// An adapter's part of the product runs over columns of T in blocks of 64: block q pairs columns t_col.. of T with columns
// b_col.. of B; `steps` MMAs of 16, whose step of B is s & b_mask.  An f32 result takes both numbers of a value of T, the
// rounded one and the remainder (with rp <= 32 they lie in one block and B's columns serve both).  A 16-bit result takes
// the rounded one alone: its own rounding is as coarse, and the tensor core's share of an adapter halves.
struct ExtBlock {
    int t_col, b_col, steps, b_mask;
};
__host__ __device__ __forceinline__ bool whole_t(int c_dtype) { return c_dtype == CUTE_B200_F32; }
__host__ __device__ __forceinline__ int ext_blocks(int rp, bool whole) { return rp <= 32 ? 1 : (whole ? rp / 32 : rp / 64); }
__device__ __forceinline__ ExtBlock ext_block(int q, int rp, int rank, bool whole, bool bf16) {
    const int first = whole ? 0 : t_hi(rp, bf16);
    if (rp <= 32) return {first, 0, whole ? rp / 8 : rp / 16, rp / 16 - 1};
    const int half = whole ? q >> 1 : q, left = (rank - 64 * half + 15) / 16;  // at least 1: rank > rp / 2
    return {first + (whole ? (q & 1) * rp : 0) + 64 * half, 64 * half, left < 4 ? left : 4, 3};
}

}  // namespace
}  // namespace cb
