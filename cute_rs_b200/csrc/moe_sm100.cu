// A mixture-of-experts layer for a few tokens: router, softmax, top-k, gated
// experts, weighted sum.
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
__device__ __forceinline__ float warp_sum(float v) {
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}

struct MoeParams {
    const uint16_t *x, *r, *g, *u, *dn;
    uint16_t *y;
    float *logits;   // (tokens, experts)
    int32_t *ids;    // (tokens, top)
    float *weights;  // (tokens, top)
    uint16_t *h;     // (tokens, top, f)
    int tokens, experts, top, d, f, renorm;
};

template <bool BF16>
__global__ void logits_simple(const MoeParams p) {
    const int e = blockIdx.x, t = blockIdx.y, lane = threadIdx.x;
    float acc = 0.0f;
    for (int l = lane; l < p.d; l += 32) acc = fmaf(to_f32<BF16>(p.x[int64_t(t) * p.d + l]), to_f32<BF16>(p.r[int64_t(e) * p.d + l]), acc);
    acc = warp_sum(acc);
    if (lane == 0) p.logits[t * p.experts + e] = acc;
}

// One warp per token.
__global__ void top_simple(const MoeParams p) {
    const int t = blockIdx.x, lane = threadIdx.x;
    float v[16];
    float best = -INFINITY;
    for (int j = 0; j < 16; j++) {
        const int e = j * 32 + lane;
        v[j] = e < p.experts ? p.logits[t * p.experts + e] : 0.0f;
        if (e < p.experts) best = fmaxf(best, v[j]);
    }
    for (int s = 16; s > 0; s >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, s));
    float total = 0.0f;
    for (int j = 0; j < 16; j++)
        if (j * 32 + lane < p.experts) total += expf(v[j] - best);
    total = warp_sum(total);
    uint32_t open = 0;
    for (int j = 0; j < 16; j++) open |= (j * 32 + lane < p.experts ? 1u : 0u) << j;
    float chosen_sum = 0.0f;
    for (int i = 0; i < p.top; i++) {
        float key = 0.0f;
        int at = 0x7fffffff;
        for (int j = 0; j < 16; j++)
            if ((open >> j) & 1u) {
                const float c = v[j] == v[j] ? v[j] : -INFINITY;
                if (at == 0x7fffffff || c > key) key = c, at = j * 32 + lane;
            }
        for (int s = 16; s > 0; s >>= 1) {
            const float k2 = __shfl_xor_sync(0xffffffffu, key, s);
            const int a2 = __shfl_xor_sync(0xffffffffu, at, s);
            if (a2 != 0x7fffffff && (at == 0x7fffffff || k2 > key || (k2 == key && a2 < at))) key = k2, at = a2;
        }
        if ((at & 31) == lane) open &= ~(1u << (at >> 5));
        const float w = expf(key - best) / total;
        chosen_sum += w;
        if (lane == 0) p.ids[t * p.top + i] = at, p.weights[t * p.top + i] = w;
    }
    __syncwarp();
    if (p.renorm && lane < p.top) p.weights[t * p.top + lane] /= chosen_sum;
}

template <bool BF16>
__global__ void up_simple(const MoeParams p) {
    const int slot = blockIdx.y, t = slot / p.top, lane = threadIdx.x & 31;
    const int j = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (j >= p.f) return;
    const int64_t row = (int64_t(p.ids[slot]) * p.f + j) * p.d;
    float g = 0.0f, u = 0.0f;
    for (int l = lane; l < p.d; l += 32) {
        const float x = to_f32<BF16>(p.x[int64_t(t) * p.d + l]);
        g = fmaf(to_f32<BF16>(p.g[row + l]), x, g);
        u = fmaf(to_f32<BF16>(p.u[row + l]), x, u);
    }
    g = warp_sum(g), u = warp_sum(u);
    if (lane == 0) p.h[int64_t(slot) * p.f + j] = from_f32<BF16>(p.weights[slot] * (g / (1.0f + expf(-g))) * u);
}

template <bool BF16>
__global__ void down_simple(const MoeParams p) {
    const int t = blockIdx.y, lane = threadIdx.x & 31;
    const int j = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (j >= p.d) return;
    float acc = 0.0f;
    for (int s = t * p.top; s < (t + 1) * p.top; s++) {
        const int64_t row = (int64_t(p.ids[s]) * p.d + j) * p.f;
        for (int l = lane; l < p.f; l += 32) acc = fmaf(to_f32<BF16>(p.dn[row + l]), to_f32<BF16>(p.h[int64_t(s) * p.f + l]), acc);
    }
    acc = warp_sum(acc);
    if (lane == 0) p.y[int64_t(t) * p.d + j] = from_f32<BF16>(acc);
}

constexpr uint64_t kAlign = 256;
uint64_t round_up(uint64_t v) { return (v + kAlign - 1) / kAlign * kAlign; }

cute_b200_status check_desc(const cute_b200_moe_desc &d, const char *who) {
    if (d.tokens < 0 || d.tokens > 64)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s takes 0 to 64 tokens, got %d", who, d.tokens);
    if (d.experts < 1 || d.experts > 512)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s takes 1 to 512 experts, got %d", who, d.experts);
    if (d.top < 1 || d.top > 16 || d.top > d.experts)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: top must be 1 to 16 and at most the %d experts, got %d", who, d.experts, d.top);
    if (d.d < 8 || d.f < 8 || d.d % 8 || d.f % 8)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: d and f must be positive multiples of 8, got %d and %d", who, d.d, d.f);
    if (int64_t(d.experts) * (d.d > d.f ? d.d : d.f) > 0x7fffffffll)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: %d experts of %d rows are more than 2^31 rows", who, d.experts,
                    d.d > d.f ? d.d : d.f);
    if (d.dtype != CUTE_B200_F16 && d.dtype != CUTE_B200_BF16)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s takes f16 or bf16, not dtype %d", who, d.dtype);
    return CUTE_B200_OK;
}

struct Layout {
    uint64_t logits, ids, weights, h, total;
};
Layout layout(const cute_b200_moe_desc &d) {
    Layout l;
    l.logits = 0;
    l.ids = l.logits + round_up(uint64_t(d.tokens) * d.experts * 4);
    l.weights = l.ids + round_up(uint64_t(d.tokens) * d.top * 4);
    l.h = l.weights + round_up(uint64_t(d.tokens) * d.top * 4);
    l.total = l.h + round_up(uint64_t(d.tokens) * d.top * d.f * 2) + kAlign;
    return l;
}

template <bool BF16>
cute_b200_status run(const MoeParams &p, cudaStream_t stream) {
    logits_simple<BF16><<<dim3(unsigned(p.experts), unsigned(p.tokens)), 32, 0, stream>>>(p);
    top_simple<<<p.tokens, 32, 0, stream>>>(p);
    up_simple<BF16><<<dim3(unsigned((p.f + 7) / 8), unsigned(p.tokens * p.top)), 256, 0, stream>>>(p);
    down_simple<BF16><<<dim3(unsigned((p.d + 7) / 8), unsigned(p.tokens)), 256, 0, stream>>>(p);
    CB_CUDA(cudaGetLastError());
    count_launch(4);
    return CUTE_B200_OK;
}

}  // namespace

cute_b200_status moe_workspace(const cute_b200_moe_desc &d, uint64_t *bytes) {
    CB_TRY(check_desc(d, "moe_workspace"));
    *bytes = layout(d).total;
    return CUTE_B200_OK;
}

// ptr: X, router, gate, up, down, Y, workspace
cute_b200_status moe_tn_check(const cute_b200_moe_desc &d, const uint64_t ptr[7]) {
    static const char *names[7] = {"X", "the router", "the gate weights", "the up weights", "the down weights", "Y", "the workspace"};
    CB_TRY(check_desc(d, "moe_tn"));
    for (int i = 0; i < 7; i++) {
        const uint64_t align = i == 6 ? kAlign : 16;
        if (!ptr[i] && d.tokens > 0) return fail(CUTE_B200_ERR_NULL_POINTER, "moe_tn: %s is null", names[i]);
        if (ptr[i] % align)
            return fail(CUTE_B200_ERR_MISALIGNED, "moe_tn: %s must be %llu-byte aligned", names[i], (unsigned long long)align);
    }
    return CUTE_B200_OK;
}

cute_b200_status moe_tn(const cute_b200_moe_desc &d, const uint64_t ptr[7], cudaStream_t stream, const DeviceState &) {
    if (d.tokens == 0) return CUTE_B200_OK;
    const Layout l = layout(d);
    MoeParams p = {};
    p.x = reinterpret_cast<const uint16_t *>(ptr[0]);
    p.r = reinterpret_cast<const uint16_t *>(ptr[1]);
    p.g = reinterpret_cast<const uint16_t *>(ptr[2]);
    p.u = reinterpret_cast<const uint16_t *>(ptr[3]);
    p.dn = reinterpret_cast<const uint16_t *>(ptr[4]);
    p.y = reinterpret_cast<uint16_t *>(ptr[5]);
    p.logits = reinterpret_cast<float *>(ptr[6] + l.logits);
    p.ids = reinterpret_cast<int32_t *>(ptr[6] + l.ids);
    p.weights = reinterpret_cast<float *>(ptr[6] + l.weights);
    p.h = reinterpret_cast<uint16_t *>(ptr[6] + l.h);
    p.tokens = d.tokens, p.experts = d.experts, p.top = d.top, p.d = d.d, p.f = d.f, p.renorm = d.renormalise;
    return d.dtype == CUTE_B200_BF16 ? run<true>(p, stream) : run<false>(p, stream);
}

cute_b200_status moe_init(const DeviceState &) { return CUTE_B200_OK; }

}  // namespace cb
