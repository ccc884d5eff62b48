// A projection shared by all rows with a low-rank adapter chosen row by row:
//     y[i] = W x[i] + scale[a] * B[a] (A[a] x[i]),   a = ids[i]
// and its gradients.  The inner product T[i] = scale[a] * A[a] x[i] (`rank`
// values per row) goes to the workspace as two 16-bit numbers per value, their
// sum: the second product can then run on 16-bit operands and still carry 16
// (bf16) or 22 (f16) bits of T.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx_sm100.cuh"

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
__device__ __forceinline__ void store_c(void *c, int dtype, size_t i, float v) {
    if (dtype == CUTE_B200_F32) static_cast<float *>(c)[i] = v;
    else if (dtype == CUTE_B200_BF16) static_cast<__nv_bfloat16 *>(c)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(c)[i] = __float2half_rn(v);
}

// Width of the rank in T: 16, 32, 64 or 128.
__host__ __device__ constexpr int padded_rank(int rank) { return rank <= 16 ? 16 : (rank <= 32 ? 32 : (rank <= 64 ? 64 : 128)); }

struct LoraParams {
    const uint16_t *x, *w, *a, *b;
    const int32_t *ids;
    const float *scale;
    void *y;
    uint16_t *t;
    int m, n, k, rank, rp, adapters, c_dtype;
    int64_t ldx, ldy;
};

template <bool BF16>
__global__ void shrink_simple(const LoraParams p) {
    const int row = blockIdx.x, lane = threadIdx.x & 31;
    const int id = p.ids[row];
    const bool has = id >= 0 && id < p.adapters;
    for (int j = threadIdx.x >> 5; j < p.rp; j += blockDim.x >> 5) {
        float acc = 0.0f;
        if (has && j < p.rank) {
            const uint16_t *a = p.a + (int64_t(id) * p.rank + j) * p.k;
            for (int l = lane; l < p.k; l += 32) acc = fmaf(to_f32<BF16>(a[l]), to_f32<BF16>(p.x[row * p.ldx + l]), acc);
            for (int s = 16; s > 0; s >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, s);
            acc *= p.scale[id];
        }
        if (lane == 0) {
            const uint16_t hi = from_f32<BF16>(acc);
            const float rest = acc - to_f32<BF16>(hi);
            p.t[int64_t(row) * 2 * p.rp + j] = hi;
            p.t[int64_t(row) * 2 * p.rp + p.rp + j] = from_f32<BF16>(rest);
        }
    }
}

template <bool BF16>
__global__ void product_simple(const LoraParams p) {
    __shared__ float xs[16][17], ws[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t row = int64_t(blockIdx.y) * 16 + ty;
    const int64_t col = int64_t(blockIdx.x) * 16 + tx, wrow = int64_t(blockIdx.x) * 16 + ty;
    float acc = 0.0f;
    for (int l = 0; l < p.k; l += 16) {
        xs[ty][tx] = row < p.m && l + tx < p.k ? to_f32<BF16>(p.x[row * p.ldx + l + tx]) : 0.0f;
        ws[ty][tx] = wrow < p.n && l + tx < p.k ? to_f32<BF16>(p.w[wrow * p.k + l + tx]) : 0.0f;
        __syncthreads();
        for (int i = 0; i < 16; i++) acc = fmaf(xs[ty][i], ws[tx][i], acc);
        __syncthreads();
    }
    if (row >= p.m || col >= p.n) return;
    const int id = p.ids[row];
    if (id >= 0 && id < p.adapters)
        for (int j = 0; j < p.rank; j++) {
            const float t = to_f32<BF16>(p.t[row * 2 * p.rp + j]) + to_f32<BF16>(p.t[row * 2 * p.rp + p.rp + j]);
            acc = fmaf(t, to_f32<BF16>(p.b[(int64_t(id) * p.n + col) * p.rank + j]), acc);
        }
    store_c(p.y, p.c_dtype, row * p.ldy + col, acc);
}

// (rows, cols) -> (cols, rows) of each of `count` 16-bit matrices.
__global__ void transpose_simple(const uint16_t *in, uint16_t *out, int rows, int cols) {
    const int64_t base = int64_t(blockIdx.y) * rows * cols;
    const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= int64_t(rows) * cols) return;
    out[base + (i % cols) * rows + i / cols] = in[base + i];
}

// out[a][j * sj + c * sc] = sum over rows i with ids[i] == a of (hi + lo of t[i][j]) * v[i][c]
template <bool BF16>
__global__ void grad_simple(const uint16_t *t, const uint16_t *v, int64_t ldv, const int32_t *ids, float *out, int m, int cols, int rank,
                            int rp, int64_t sj, int64_t sc) {
    const int a = blockIdx.z, j = blockIdx.y;
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= cols) return;
    float acc = 0.0f;
    for (int64_t i = 0; i < m; i++)
        if (ids[i] == a)
            acc = fmaf(to_f32<BF16>(t[i * 2 * rp + j]) + to_f32<BF16>(t[i * 2 * rp + rp + j]), to_f32<BF16>(v[i * ldv + c]), acc);
    out[int64_t(a) * rank * cols + j * sj + c * sc] = acc;
}

constexpr uint64_t kAlign = 256;
uint64_t round_up(uint64_t v) { return (v + kAlign - 1) / kAlign * kAlign; }
uint64_t t_bytes(const cute_b200_lora_desc &d) { return round_up(uint64_t(d.m) * padded_rank(d.rank) * 4); }

cute_b200_status check_desc(const cute_b200_lora_desc &d, const char *who) {
    if (d.m < 0 || d.n < 1 || d.k < 8)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: invalid size %dx%dx%d", who, d.m, d.n, d.k);
    if (d.k % 8) return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: k must be a multiple of 8, got %d", who, d.k);
    if (d.rank < 8 || d.rank > 128 || d.rank % 8)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: rank must be a multiple of 8 in 8..128, got %d", who, d.rank);
    if (d.adapters < 1) return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: at least one adapter is needed, got %d", who, d.adapters);
    const int64_t widest = d.n > d.k ? (d.n > d.rank ? d.n : d.rank) : (d.k > d.rank ? d.k : d.rank);
    if (d.adapters * widest > 0x7fffffffll)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: %d adapters of %lld rows are more than 2^31 rows", who, d.adapters,
                    (long long)widest);
    if (d.ab_dtype != CUTE_B200_F16 && d.ab_dtype != CUTE_B200_BF16)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s takes f16 or bf16 operands, not dtype %d", who, d.ab_dtype);
    if (d.c_dtype != CUTE_B200_F32 && d.c_dtype != CUTE_B200_F16 && d.c_dtype != CUTE_B200_BF16)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s writes f32, f16 or bf16, not dtype %d", who, d.c_dtype);
    if (d.ldx != 0 && (d.ldx < d.k || d.ldx % 8))
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: ldx must be 0 or a multiple of 8 of at least k = %d, got %d", who, d.k, d.ldx);
    if (d.ldy != 0 && d.ldy < d.n)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: ldy must be 0 or at least n = %d, got %d", who, d.n, d.ldy);
    if (d.tuning[0] < 0 || d.tuning[0] > 2 || (d.tuning[0] == 1 && d.m > 128))
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: tuning[0] must be 0, 1 (with m <= 128) or 2, got %d", who, d.tuning[0]);
    return CUTE_B200_OK;
}

cute_b200_status check_ptr(const char *who, const char *name, uint64_t p, uint64_t align, bool need) {
    if (!p && need) return fail(CUTE_B200_ERR_NULL_POINTER, "%s: %s is null", who, name);
    if (p % align) return fail(CUTE_B200_ERR_MISALIGNED, "%s: %s must be %llu-byte aligned", who, name, (unsigned long long)align);
    return CUTE_B200_OK;
}

uint64_t elem_bytes(int dtype) { return dtype == CUTE_B200_F32 ? 4 : 2; }

template <bool BF16>
cute_b200_status forward(const LoraParams &p, cudaStream_t stream) {
    if (p.m == 0) return CUTE_B200_OK;
    shrink_simple<BF16><<<p.m, 128, 0, stream>>>(p);
    CB_CUDA(cudaGetLastError());
    product_simple<BF16><<<dim3(unsigned((p.n + 15) / 16), unsigned((p.m + 15) / 16)), 256, 0, stream>>>(p);
    CB_CUDA(cudaGetLastError());
    count_launch(2);
    return CUTE_B200_OK;
}

}  // namespace

cute_b200_status lora_workspace(const cute_b200_lora_desc &d, uint64_t *forward, uint64_t *backward) {
    CB_TRY(check_desc(d, "lora_workspace"));
    *forward = t_bytes(d) + kAlign;
    *backward = t_bytes(d) + round_up(uint64_t(d.adapters) * d.rank * d.k * 2) + round_up(uint64_t(d.adapters) * d.rank * d.n * 2) + kAlign;
    return CUTE_B200_OK;
}

// ptr: X, W, A, B, ids, scale, Y, workspace
cute_b200_status lora_tn_check(const cute_b200_lora_desc &d, const uint64_t ptr[8]) {
    const char *who = "lora_tn";
    CB_TRY(check_desc(d, who));
    const bool rows = d.m > 0;
    CB_TRY(check_ptr(who, "X", ptr[0], 16, rows));
    CB_TRY(check_ptr(who, "W", ptr[1], 16, rows));
    CB_TRY(check_ptr(who, "A", ptr[2], 16, rows));
    CB_TRY(check_ptr(who, "B", ptr[3], 16, rows));
    CB_TRY(check_ptr(who, "ids", ptr[4], 4, rows));
    CB_TRY(check_ptr(who, "scale", ptr[5], 4, rows));
    CB_TRY(check_ptr(who, "Y", ptr[6], elem_bytes(d.c_dtype), rows));
    CB_TRY(check_ptr(who, "the workspace", ptr[7], kAlign, rows));
    return CUTE_B200_OK;
}

cute_b200_status lora_tn(const cute_b200_lora_desc &d, const uint64_t ptr[8], cudaStream_t stream, const DeviceState &) {
    LoraParams p = {};
    p.x = reinterpret_cast<const uint16_t *>(ptr[0]);
    p.w = reinterpret_cast<const uint16_t *>(ptr[1]);
    p.a = reinterpret_cast<const uint16_t *>(ptr[2]);
    p.b = reinterpret_cast<const uint16_t *>(ptr[3]);
    p.ids = reinterpret_cast<const int32_t *>(ptr[4]);
    p.scale = reinterpret_cast<const float *>(ptr[5]);
    p.y = reinterpret_cast<void *>(ptr[6]);
    p.t = reinterpret_cast<uint16_t *>(ptr[7]);
    p.m = d.m, p.n = d.n, p.k = d.k, p.rank = d.rank, p.rp = padded_rank(d.rank), p.adapters = d.adapters, p.c_dtype = d.c_dtype;
    p.ldx = d.ldx ? d.ldx : d.k;
    p.ldy = d.ldy ? d.ldy : d.n;
    return d.ab_dtype == CUTE_B200_BF16 ? forward<true>(p, stream) : forward<false>(p, stream);
}

// ptr: X, W transposed, A, B, ids, scale, dY, forward workspace, dX, dA, dB, workspace
cute_b200_status lora_tn_backward_check(const cute_b200_lora_desc &d, const uint64_t ptr[12]) {
    const char *who = "lora_tn_backward";
    CB_TRY(check_desc(d, who));
    if (d.n % 8) return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: n must be a multiple of 8, got %d", who, d.n);
    if (d.ldy % 8) return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: ldy must be a multiple of 8, got %d", who, d.ldy);
    const bool rows = d.m > 0, dx = ptr[8] != 0, dw = ptr[9] != 0 || ptr[10] != 0;
    CB_TRY(check_ptr(who, "X", ptr[0], 16, rows && dw));
    CB_TRY(check_ptr(who, "W transposed", ptr[1], 16, rows && dx));
    CB_TRY(check_ptr(who, "A", ptr[2], 16, rows));
    CB_TRY(check_ptr(who, "B", ptr[3], 16, rows));
    CB_TRY(check_ptr(who, "ids", ptr[4], 4, rows));
    CB_TRY(check_ptr(who, "scale", ptr[5], 4, rows));
    CB_TRY(check_ptr(who, "dY", ptr[6], 16, rows));
    CB_TRY(check_ptr(who, "the forward workspace", ptr[7], kAlign, rows && dw));
    CB_TRY(check_ptr(who, "dX", ptr[8], elem_bytes(d.c_dtype), false));
    CB_TRY(check_ptr(who, "dA", ptr[9], 4, dw));
    CB_TRY(check_ptr(who, "dB", ptr[10], 4, dw));
    CB_TRY(check_ptr(who, "the workspace", ptr[11], kAlign, rows));
    return CUTE_B200_OK;
}

cute_b200_status lora_tn_backward(const cute_b200_lora_desc &d, const uint64_t ptr[12], cudaStream_t stream, const DeviceState &) {
    const int64_t ldx = d.ldx ? d.ldx : d.k, ldy = d.ldy ? d.ldy : d.n;
    const bool bf16 = d.ab_dtype == CUTE_B200_BF16;
    float *da = reinterpret_cast<float *>(ptr[9]), *db = reinterpret_cast<float *>(ptr[10]);
    if (d.m == 0) {
        if (da) CB_CUDA(cudaMemsetAsync(da, 0, size_t(d.adapters) * d.rank * d.k * 4, stream));
        if (db) CB_CUDA(cudaMemsetAsync(db, 0, size_t(d.adapters) * d.rank * d.n * 4, stream));
        return CUTE_B200_OK;
    }
    uint16_t *u = reinterpret_cast<uint16_t *>(ptr[11]);
    uint16_t *at = reinterpret_cast<uint16_t *>(ptr[11] + t_bytes(d));
    uint16_t *bt = reinterpret_cast<uint16_t *>(ptr[11] + t_bytes(d) + round_up(uint64_t(d.adapters) * d.rank * d.k * 2));
    transpose_simple<<<dim3(unsigned((int64_t(d.rank) * d.k + 255) / 256), unsigned(d.adapters)), 256, 0, stream>>>(
        reinterpret_cast<const uint16_t *>(ptr[2]), at, d.rank, d.k);
    transpose_simple<<<dim3(unsigned((int64_t(d.rank) * d.n + 255) / 256), unsigned(d.adapters)), 256, 0, stream>>>(
        reinterpret_cast<const uint16_t *>(ptr[3]), bt, d.n, d.rank);
    CB_CUDA(cudaGetLastError());
    count_launch(2);
    LoraParams p = {};
    p.x = reinterpret_cast<const uint16_t *>(ptr[6]);
    p.w = reinterpret_cast<const uint16_t *>(ptr[1]);
    p.a = bt;
    p.b = at;
    p.ids = reinterpret_cast<const int32_t *>(ptr[4]);
    p.scale = reinterpret_cast<const float *>(ptr[5]);
    p.y = reinterpret_cast<void *>(ptr[8]);
    p.t = u;
    p.m = d.m, p.n = d.k, p.k = d.n, p.rank = d.rank, p.rp = padded_rank(d.rank), p.adapters = d.adapters, p.c_dtype = d.c_dtype;
    p.ldx = ldy;
    p.ldy = ldx;
    if (p.y) {
        CB_TRY(bf16 ? forward<true>(p, stream) : forward<false>(p, stream));
    } else {
        if (bf16) shrink_simple<true><<<p.m, 128, 0, stream>>>(p);
        else shrink_simple<false><<<p.m, 128, 0, stream>>>(p);
        CB_CUDA(cudaGetLastError());
        count_launch();
    }
    if (da) {
        const uint16_t *x = reinterpret_cast<const uint16_t *>(ptr[0]), *dy = p.x, *t = reinterpret_cast<const uint16_t *>(ptr[7]);
        const dim3 ga(unsigned((d.k + 127) / 128), unsigned(d.rank), unsigned(d.adapters));
        const dim3 gb(unsigned((d.n + 127) / 128), unsigned(d.rank), unsigned(d.adapters));
        if (bf16) {
            grad_simple<true><<<ga, 128, 0, stream>>>(u, x, ldx, p.ids, da, d.m, d.k, d.rank, p.rp, d.k, 1);
            grad_simple<true><<<gb, 128, 0, stream>>>(t, dy, ldy, p.ids, db, d.m, d.n, d.rank, p.rp, 1, d.rank);
        } else {
            grad_simple<false><<<ga, 128, 0, stream>>>(u, x, ldx, p.ids, da, d.m, d.k, d.rank, p.rp, d.k, 1);
            grad_simple<false><<<gb, 128, 0, stream>>>(t, dy, ldy, p.ids, db, d.m, d.n, d.rank, p.rp, 1, d.rank);
        }
        CB_CUDA(cudaGetLastError());
        count_launch(2);
    }
    return CUTE_B200_OK;
}

cute_b200_status lora_init(const DeviceState &) { return CUTE_B200_OK; }

}  // namespace cb
