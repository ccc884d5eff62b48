// A mixture-of-experts layer for a few tokens, in three kernels:
//   router   logits, softmax, top-k: a cluster of eight CTAs for four tokens;
//   up       the gate and up weights of the experts that anybody chose stream past all the tokens, each byte once;
//   down     the down weights likewise, summed over the experts in the accumulator.
// Bound by HBM: 6 d f bytes per chosen expert.  The tokens (at most 64 of the M = 128 rows of an MMA) are the lanes of
// the accumulators, the weights' rows its columns, so that nothing is gathered or sorted: an expert's product is
// computed for all tokens - the tensor core has time to spare, an MMA of N columns costs the same for 1 and for 128 rows -
// and used, or added, only in the lanes of the tokens that chose it.
#include "rows_sm100.cuh"

namespace cb {
namespace {

constexpr int MAX_TOKENS = 64, MAX_TOP = 16, MAX_EXPERTS = 512;

struct MoeParams {
    const uint16_t *x, *r;
    uint16_t *y, *h;  // h: (chosen experts in ascending order, token_rows, f)
    int32_t *ids;     // (tokens, top)
    float *weights;   // (tokens, top)
    int tokens, token_rows, experts, top, d, f, renorm;
    int kc, bn, stages, kps;
    uint32_t stage_bytes, tmem_cols;
    bool bf16;
    uint32_t *status;
    int debug;
};

// ---- router -----------------------------------------------------------------
// 128 warps share the experts' rows of four tokens; with fewer experts each row is cut into `parts` ranges of d.  The
// sums go to the CTA that owns the token (the cluster's CTAs 0-3), which adds the parts in order and chooses.  Bound by
// latency: what it reads is asked into L2 while the kernel before still runs (which is safe whatever that kernel
// writes), the loads of two steps are on their way at once, a round of the choice is two warp-wide reductions.
constexpr int ROUTER_THREADS = 512, ROUTER_CLUSTER = 8, ROUTER_TOKENS = 4;

template <bool BF16>
__global__ void __launch_bounds__(ROUTER_THREADS) moe_router_kernel(const MoeParams p) {
    __shared__ float part[MAX_EXPERTS];
    {
        const int64_t cta = ptx::cluster_ctarank(), t0 = int64_t(blockIdx.x) / ROUTER_CLUSTER * ROUTER_TOKENS;
        const int64_t r_bytes = int64_t(p.experts) * p.d * 2, x_bytes = int64_t(min(ROUTER_TOKENS, p.tokens - int(t0))) * p.d * 2;
        const char *r = reinterpret_cast<const char *>(p.r), *x = reinterpret_cast<const char *>(p.x + t0 * p.d);
        for (int64_t i = (cta * ROUTER_THREADS + threadIdx.x) * 128; i < r_bytes; i += ROUTER_CLUSTER * ROUTER_THREADS * 128) ptx::prefetch_l2(r + i);
        for (int64_t i = int64_t(threadIdx.x) * 128; i < x_bytes; i += ROUTER_THREADS * 128) ptx::prefetch_l2(x + i);
    }
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = int(ptx::cluster_ctarank()), t0 = int(blockIdx.x) / ROUTER_CLUSTER * ROUTER_TOKENS;
    const int warps = ROUTER_CLUSTER * ROUTER_THREADS / 32, count = min(ROUTER_TOKENS, p.tokens - t0);
    int parts = 1;
    while (parts * 2 * p.experts <= warps && parts * 2 <= 16) parts *= 2;  // experts * parts <= MAX_EXPERTS
    const int vecs = p.d / 8;
    ptx::cluster_arrive();
    ptx::cluster_wait();  // every CTA of the cluster runs: its shared memory may be written
    for (int item = rank * (ROUTER_THREADS / 32) + warp; item < p.experts * parts; item += warps) {
        const int e = item / parts, q = item - e * parts;
        const uint16_t *r = p.r + int64_t(e) * p.d, *x = p.x + int64_t(t0) * p.d;
        float acc[ROUTER_TOKENS] = {};
        const int end = int(int64_t(vecs) * (q + 1) / parts);
#pragma unroll 2
        for (int c = int(int64_t(vecs) * q / parts) + lane; c < end; c += 32) {
            const uint4 rv = *reinterpret_cast<const uint4 *>(r + 8 * c);
            const uint32_t rw[4] = {rv.x, rv.y, rv.z, rv.w};
            uint4 xv[ROUTER_TOKENS];  // a token past the last is the first once more: no branch between the loads
#pragma unroll
            for (int t = 0; t < ROUTER_TOKENS; t++) xv[t] = *reinterpret_cast<const uint4 *>(x + (t < count ? int64_t(t) * p.d : 0) + 8 * c);
#pragma unroll
            for (int t = 0; t < ROUTER_TOKENS; t++) {
                const uint32_t xw[4] = {xv[t].x, xv[t].y, xv[t].z, xv[t].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 a = pair_f32<BF16>(rw[i]), b = pair_f32<BF16>(xw[i]);
                    acc[t] = fmaf(a.y, b.y, fmaf(a.x, b.x, acc[t]));
                }
            }
        }
#pragma unroll
        for (int t = 0; t < ROUTER_TOKENS; t++) {
            const float sum = warp_sum(acc[t]);
            if (lane == 0 && t < count) ptx::st_shared_cluster(ptx::mapa(ptx::smem_u32(&part[item]), uint32_t(t)), sum);
        }
    }
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (rank >= count || warp != 0) return;  // nothing reads another CTA's shared memory from here on
    // One warp chooses for the token: lane l holds experts l, l + 32, ..
    const int t = t0 + rank;
    const int per_lane = (p.experts + 31) / 32;
    float v[MAX_EXPERTS / 32];
    float best = -INFINITY;
#pragma unroll
    for (int j = 0; j < MAX_EXPERTS / 32; j++) {
        if (j >= per_lane) break;
        const int e = j * 32 + lane;
        v[j] = -INFINITY;
        if (e < p.experts) {
            float sum = part[e * parts];
            for (int q = 1; q < parts; q++) sum += part[e * parts + q];
            v[j] = sum;
            best = fmaxf(best, sum);
        }
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, s));
    float total = 0.0f;
    uint32_t open = 0;
#pragma unroll
    for (int j = 0; j < MAX_EXPERTS / 32; j++) {
        if (j >= per_lane) break;
        if (j * 32 + lane < p.experts) {
            total += expf(v[j] - best);
            open |= 1u << j;
        }
    }
    total = warp_sum(total);
    // A logit as an unsigned number of the same order (-0 as +0); a NaN counts as the smallest, its weight is a NaN.
    auto order = [](float f) -> uint32_t {
        if (!(f == f)) return 0u;
        const uint32_t u = __float_as_uint(f + 0.0f);
        return (u >> 31) ? ~u : u | 0x80000000u;
    };
    float my_logit = 0.0f;
    int my_id = 0;
    for (int i = 0; i < p.top; i++) {
        // The largest open logit, the lowest index among equals.  The lane's own first.
        uint32_t key = 0u;
        int at = 0x7fffffff;
        float logit = 0.0f;
#pragma unroll
        for (int j = 0; j < MAX_EXPERTS / 32; j++) {
            if (j >= per_lane) break;
            if ((open >> j) & 1u) {
                const uint32_t k = order(v[j]);
                if (at == 0x7fffffff || k > key) key = k, at = j * 32 + lane, logit = v[j];
            }
        }
        const uint32_t best_key = __reduce_max_sync(0xffffffffu, key);
        const int winner = int(__reduce_min_sync(0xffffffffu, key == best_key ? uint32_t(at) : 0x7fffffffu));
        const float w = __shfl_sync(0xffffffffu, logit, winner & 31);
        if ((winner & 31) == lane) open &= ~(1u << (winner >> 5));
        if (lane == i) my_logit = w, my_id = winner;
    }
    const float w = lane < p.top ? expf(my_logit - best) / total : 0.0f, chosen_sum = warp_sum(w);
    if (lane < p.top) {
        p.ids[t * p.top + lane] = my_id;
        p.weights[t * p.top + lane] = p.renorm ? w / chosen_sum : w;
    }
}

// ---- which experts are chosen, and by whom ----------------------------------------
struct MoeHead {
    uint64_t full[16], empty[16], tfull[2], tempty[2], plan, done, drain;
    uint32_t tmem, abort, stop;
    int32_t active, before[4];
    int32_t expert[MAX_EXPERTS];                     // the chosen experts, ascending
    unsigned long long who[MAX_EXPERTS];             // by expert: which tokens chose it
    int32_t ids[MAX_TOKENS * MAX_TOP];
    float weights[MAX_TOKENS * MAX_TOP];
    int32_t row[MAX_TOKENS];  // of the chunk at hand: the tokens that chose its expert
    float row_weight[MAX_TOKENS];
};
constexpr uint32_t MOE_HEAD = 16 * 1024;
static_assert(sizeof(MoeHead) <= MOE_HEAD, "head");

// By 128 threads (t = 0..127).  The router's output is read from L2: the down kernel reads it ahead of its griddepcontrol.wait.
__device__ __forceinline__ void find_active(MoeHead &h, const MoeParams &p, int t) {
    const int lane = t & 31, w = t >> 5;
    for (int e = t; e < MAX_EXPERTS; e += 128) h.who[e] = 0ull;
    for (int i = t; i < p.tokens * p.top; i += 128) h.ids[i] = __ldcg(p.ids + i), h.weights[i] = __ldcg(p.weights + i);
    ptx::named_barrier(1, 128);
    for (int i = t; i < p.tokens * p.top; i += 128) atomicOr(&h.who[h.ids[i]], 1ull << (i / p.top));
    ptx::named_barrier(1, 128);
    int mine = 0;
    for (int j = 0; j < 4; j++) mine += h.who[4 * t + j] != 0ull;
    int upto = mine;
    for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, s);
        if (lane >= s) upto += o;
    }
    if (lane == 31) h.before[w] = upto;
    ptx::named_barrier(1, 128);
    int at = upto - mine, total = 0;
    for (int i = 0; i < 4; i++) {
        if (i < w) at += h.before[i];
        total += h.before[i];
    }
    for (int j = 0; j < 4; j++)
        if (h.who[4 * t + j] != 0ull) h.expert[at++] = 4 * t + j;
    if (t == 0) h.active = total;
    ptx::named_barrier(1, 128);
}

constexpr int MOE_THREADS = 192, MOE_MAX_STAGES = 16;
constexpr uint32_t MOE_SMEM = 216 * 1024;  // leaves room for the next kernels' first CTAs, the router's among them

// ---- up ---------------------------------------------------------------------------
// The rows of the chosen experts' gate and up weights, eight of each to a group, are dealt out evenly over the CTAs;
// a CTA takes its range in chunks of up to sixteen groups of one expert.  A chunk's MMA has N = 16 columns per group:
// first the chunk's gate rows, then its up rows.
//   warp 0  TMA: per stage one, two or four k blocks of X and of the weights, 8 g rows of each matrix as boxes of 64, 32,
//           16 and 8 rows, a lane per box (boxes of 8 rows alone would cap the stream at 4 TB/s, those of 16 at 6.5: measured).
//   warp 1  MMA, two accumulators in turn.
//   warps 2-5  epilogue: silu, product, routing weight, rounding.  Only the tokens that chose the expert count, one lane
//           of 64 for a single token, so 32 pairs of columns at a time go through shared memory, where all 128 threads
//           share them (a thread per token took 1.2 us per group: 15 us after the last weight, 8 of 4096 x 14336).
constexpr int UP_GROUPS = 16, UP_PAIRS = 32;
constexpr uint32_t UP_PITCH = (2 * UP_PAIRS + 4) * 4;  // a token's pairs of one step: gate, up
struct UpMaps {
    CUtensorMap gate[4], up[4];  // boxes of 64, 32, 16 and 8 rows
};
// k blocks per stage: what a stage of 2 token_rows + 256 rows holds.
__device__ __forceinline__ int up_blocks(int groups, int token_rows) {
    return groups > 8 ? 1 : (groups <= 4 && 4 * (token_rows + 16 * groups) <= 2 * token_rows + 256 ? 4 : 2);
}

__host__ __device__ __forceinline__ uint32_t up_step_bytes(int token_rows) { return (uint32_t(token_rows) * UP_PITCH + 1023u) & ~1023u; }

// Calls f(expert's place in the list, first group, groups) for every chunk of this CTA; f returns false to stop.
template <typename F>
__device__ __forceinline__ void up_chunks(const MoeHead &h, const MoeParams &p, F f) {
    const int per = p.f / 8;
    const int64_t all = int64_t(h.active) * per;
    int64_t g = all * blockIdx.x / gridDim.x;
    const int64_t end = all * (blockIdx.x + 1) / gridDim.x;
    while (g < end) {
        const int a = int(g / per), g0 = int(g - int64_t(a) * per);
        const int piece = int(min(end - g, int64_t(per - g0))), chunks = (piece + UP_GROUPS - 1) / UP_GROUPS;
        for (int c = 0; c < chunks; c++) {
            const int lo = piece * c / chunks, hi = piece * (c + 1) / chunks;
            if (!f(a, g0 + lo, hi - lo)) return;
        }
        g += piece;
    }
}

__global__ void __launch_bounds__(MOE_THREADS, 1)
    moe_up_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ UpMaps maps, const MoeParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    MoeHead &h = *reinterpret_cast<MoeHead *>(smem_raw + (base - raw));
    // The head, the epilogue's step, the ring.
    const uint32_t pairs = base + MOE_HEAD, ring = pairs + up_step_bytes(p.token_rows), x_bytes = uint32_t(p.token_rows) * 128u;
    auto bar = [&](uint64_t &b) { return ptx::smem_u32(&b); };
    volatile uint32_t *abort_flag = &h.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k_blocks = (p.d + 63) / 64;
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            ptx::mbar_init(bar(h.full[s]), 1);
            ptx::mbar_init(bar(h.empty[s]), 1);
        }
        for (int b = 0; b < 2; b++) {
            ptx::mbar_init(bar(h.tfull[b]), 1);
            ptx::mbar_init(bar(h.tempty[b]), 4);
        }
        ptx::mbar_init(bar(h.plan), 1);
        ptx::mbar_init(bar(h.drain), 1);
        h.abort = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<1>(ptx::smem_u32(&h.tmem), 512);
        ptx::tmem_relinquish<1>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&h.tmem);
    ptx::griddep_wait();
    if (threadIdx.x == 0) ptx::griddep_launch_dependents();

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 0, filled = 0, filled_parity = 0;
        bool ok = !(p.debug & 4) && wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_PRODUCER, 100u, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (ok)
            up_chunks(h, p, [&](int a, int g0, int groups) {
                const int kps = up_blocks(groups, p.token_rows), w_bytes = groups * 2048;
                // Lanes issue the boxes of a stage's k blocks, per matrix two of 64 rows, then 32, 16, 8 (up to four groups: from
                // 32 on), and, from lane 28 or 30 on, the blocks of X.
                const int boxes = kps == 4 ? 3 : 5, weights = kps == 4 ? 24 : 20;
                const bool x_lane = lane >= 32 - (kps == 4 ? 4 : 2);
                const int kk = x_lane ? lane - (32 - (kps == 4 ? 4 : 2)) : lane / (2 * boxes), up = lane / boxes % 2, box = lane % boxes + 5 - boxes;
                const int size = box < 2 ? 64 : 128 >> box;
                const int off = box < 2 ? 64 * box : (8 * groups) & ~(2 * size - 1);  // the larger boxes lie before it
                const bool mine = lane < weights && (box < 2 ? groups >= 8 * (box + 1) : (8 * groups & size) != 0);
                const CUtensorMap *map = (up ? maps.up : maps.gate) + (box < 2 ? 0 : box - 1);
                const uint32_t to = uint32_t(kps) * x_bytes + uint32_t(kk * w_bytes + up * groups * 1024 + off * 128);
                const int row = h.expert[a] * p.f + 8 * g0 + off;
                for (int kb = 0; kb < k_blocks; kb += kps) {
                    const int nk = min(kps, k_blocks - kb);
                    ok = wait_bar(bar(h.empty[s]), ph ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(s), limit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return false;
                    const uint32_t dst = ring + uint32_t(s) * p.stage_bytes, full = bar(h.full[s]);
                    if (lane == 0) ptx::mbar_arrive_expect_tx(full, uint32_t(nk) * (x_bytes + uint32_t(w_bytes)));
                    __syncwarp();
                    if (mine && kk < nk) ptx::tma_load_2d(dst + to, map, full, (kb + kk) * 64, row);
                    if (x_lane && kk < nk) ptx::tma_load_2d(dst + uint32_t(kk) * x_bytes, &tmX, full, (kb + kk) * 64, 0);
                    __syncwarp();
                    filled |= 1u << s, filled_parity = (filled_parity & ~(1u << s)) | (ph << s);
                    if (++s == p.stages) s = 0, ph ^= 1u;
                }
                return true;
            });
        if (!ok && lane == 0) {  // giving up: let the copies in flight land (bounded)
            const uint64_t t0 = ptx::globaltimer_ns();
            for (int i = 0; i < p.stages; i++)
                while ((filled >> i & 1u) && !ptx::mbar_try_wait(bar(h.full[i]), (filled_parity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp runs the loop and one thread issues: see lora_few_kernel.
        const bool leader = ptx::elect_one();
        int s = 0, it = 0;
        uint32_t ph = 0;
        bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_MMA_TMEM, 100u, limit)), issued = false;
        if (ok)
            up_chunks(h, p, [&](int, int, int groups) {
                const int buf = it & 1, kps = up_blocks(groups, p.token_rows);
                const uint32_t idesc = make_idesc(p.bf16, 128, 16 * groups), d = tmem + uint32_t(buf) * 256u;
                ok = __all_sync(0xffffffffu, wait_bar(bar(h.tempty[buf]), (uint32_t(it >> 1) & 1u) ^ 1u, abort_flag, p.status, WHERE_MMA_TMEM, uint32_t(buf), limit));
                if (!ok) return false;
                ptx::tc_fence_after();
                for (int kb = 0; kb < k_blocks; kb += kps) {
                    ok = __all_sync(0xffffffffu, wait_bar(bar(h.full[s]), ph, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(s), limit));
                    if (!ok) return false;
                    ptx::tc_fence_after();
                    const uint32_t src = ring + uint32_t(s) * p.stage_bytes;
                    const int nk = min(kps, k_blocks - kb);
                    for (int kk = 0; kk < nk; kk++) {
                        const uint64_t a = sw128_desc(src + uint32_t(kk) * x_bytes), b = sw128_desc(src + uint32_t(kps) * x_bytes + uint32_t(kk * groups) * 2048u);
                        const uint32_t more = kb > 0 || kk > 0 ? 1u : 0u;
                        if (leader) {
#pragma unroll
                            for (int j = 0; j < 4; j++) ptx::umma_f16<1>(d, a + 2u * j, b + 2u * j, idesc, j > 0 ? 1u : more);
                        }
                        __syncwarp();
                    }
                    issued = true;
                    if (leader) ptx::umma_commit<1>(bar(h.empty[s]));
                    __syncwarp();
                    if (++s == p.stages) s = 0, ph ^= 1u;
                }
                if (leader) ptx::umma_commit<1>(bar(h.tfull[buf]));
                __syncwarp();
                it++;
                return true;
            });
        if (!ok && issued && leader) {
            ptx::umma_commit<1>(bar(h.drain));
            const uint64_t t0 = ptx::globaltimer_ns();
            while (!ptx::mbar_try_wait(bar(h.drain), 0u))
                if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else {
        find_active(h, p, threadIdx.x - 64);
        if (threadIdx.x == 64) ptx::mbar_arrive(bar(h.plan));
        const int q = warp & 3, token = 32 * q + lane;
        int it = 0;
        up_chunks(h, p, [&](int a, int g0, int groups) {
            const int buf = it & 1;
            wait_bar(bar(h.tfull[buf]), uint32_t(it >> 1) & 1u, abort_flag, p.status, WHERE_EPILOGUE, uint32_t(buf), limit);
            // The four warps go on or stop together: the barriers below count all of them.
            ptx::named_barrier(1, 128);
            if (threadIdx.x == 64) h.stop = *abort_flag;
            ptx::named_barrier(1, 128);
            if (h.stop) return false;
            ptx::tc_fence_after();
            // The tokens that chose the expert, in order, and their weights.
            const int e = h.expert[a];
            const unsigned long long who = h.who[e];
            const int count = __popcll(who), thread = threadIdx.x - 64;
            const bool mine = q < 2 && ((who >> (token & 63)) & 1ull);
            const int place = __popcll(who & ((1ull << (token & 63)) - 1ull));
            if (mine) {
                h.row[place] = token;
                for (int i = 0; i < p.top; i++)
                    if (h.ids[token * p.top + i] == e) h.row_weight[place] = h.weights[token * p.top + i];
            }
            const int columns = 8 * groups;
            for (int c0 = 0; c0 < columns; c0 += UP_PAIRS) {
                const int pairs_here = min(UP_PAIRS, columns - c0);
                if (q < 2 && uint32_t(who >> (32 * q)) != 0u) {
                    uint32_t vg[32], vu[32];
                    const uint32_t at = tmem + (uint32_t(32 * q) << 16) + uint32_t(256 * buf + c0);
                    ptx::tmem_ld_32x32(at, vg);
                    ptx::tmem_ld_32x32(at + uint32_t(columns), vu);
                    ptx::tmem_ld_wait_all();
                    ptx::pin(vg);
                    ptx::pin(vu);
                    if (mine) {
                        const uint32_t dst = pairs + uint32_t(place) * UP_PITCH;
#pragma unroll
                        for (int g = 0; g < 8; g++) {
                            ptx::st_shared_v4(dst + 16u * g, vg[4 * g], vg[4 * g + 1], vg[4 * g + 2], vg[4 * g + 3]);
                            ptx::st_shared_v4(dst + 128u + 16u * g, vu[4 * g], vu[4 * g + 1], vu[4 * g + 2], vu[4 * g + 3]);
                        }
                    }
                }
                ptx::named_barrier(1, 128);
                // Two columns of one token per thread and turn.
                for (int i = thread; i < count * (UP_PAIRS / 2); i += 128) {
                    const int r = i / (UP_PAIRS / 2), c = i % (UP_PAIRS / 2) * 2;
                    if (c >= pairs_here) continue;
                    const float *v = reinterpret_cast<const float *>(smem_raw + (pairs - raw) + uint32_t(r) * UP_PITCH) + c;
                    const float weight = h.row_weight[r];
                    float o[2];
#pragma unroll
                    for (int j = 0; j < 2; j++) o[j] = weight * (v[j] / (1.0f + expf(-v[j]))) * v[UP_PAIRS + j];
                    // Rounded once, to the operands' type: the last product runs on 16-bit tensor-core operands.
                    uint16_t *out = p.h + (int64_t(a) * p.token_rows + h.row[r]) * p.f + 8 * g0 + c0 + c;
                    *reinterpret_cast<uint32_t *>(out) = pack_16(o[0], o[1], p.bf16);
                }
                ptx::named_barrier(1, 128);
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(h.tempty[buf]));
            it++;
            return true;
        });
        __syncwarp();
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, 512);
}

// ---- down -------------------------------------------------------------------------
// A tile of bn columns of Y; the k of its product runs over all the chosen experts, f each, shared by a cluster of kc
// CTAs.  An expert's MMAs are masked to the lanes of the tokens that chose it, so the accumulator, which starts
// from zeros, is the sum over the experts.  The weights do not depend on the kernel before (which has waited for the
// router): the first ring-full is loaded before griddepcontrol.wait, the h it is multiplied by after.
__global__ void __launch_bounds__(MOE_THREADS, 1)
    moe_down_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmD, const MoeParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    MoeHead &h = *reinterpret_cast<MoeHead *>(smem_raw + (base - raw));
    const uint32_t ring = base + MOE_HEAD, h_bytes = uint32_t(p.token_rows) * 128u;
    auto bar = [&](uint64_t &b) { return ptx::smem_u32(&b); };
    volatile uint32_t *abort_flag = &h.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, f_blocks = (p.f + 63) / 64;
    const uint32_t rank = p.kc > 1 ? ptx::cluster_ctarank() : 0u;
    const int n0 = int(blockIdx.x) / p.kc * p.bn;
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            ptx::mbar_init(bar(h.full[s]), 1);
            ptx::mbar_init(bar(h.empty[s]), 1);
        }
        ptx::mbar_init(bar(h.plan), 1);
        ptx::mbar_init(bar(h.done), 1);
        ptx::mbar_init(bar(h.drain), 1);
        h.abort = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<1>(ptx::smem_u32(&h.tmem), p.tmem_cols);
        ptx::tmem_relinquish<1>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&h.tmem);
    if (threadIdx.x == 0) ptx::griddep_launch_dependents();

    const uint32_t w_bytes = uint32_t(p.bn) * 128u, w0 = uint32_t(p.kps) * h_bytes;
    if (warp == 0) {
        if (lane == 0) {
            ptx::prefetch_tensormap(&tmH);
            ptx::prefetch_tensormap(&tmD);
        }
        bool ok = !(p.debug & 4) && wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_PRODUCER, 100u, limit);
        ok = __all_sync(0xffffffffu, ok);
        uint32_t filled = 0, filled_parity = 0;
        if (ok) {
            const int64_t all = int64_t(h.active) * f_blocks;
            const int i0 = int(all * rank / p.kc), i1 = int(all * (rank + 1) / p.kc);
            const int ahead = min((i1 - i0 + p.kps - 1) / p.kps, p.stages);  // stages filled at once
            const int kk = lane & 7;                                         // lanes 0-7 issue weights, lanes 8-15 rows of h
            // Lane kk follows block i0 + kk, i0 + kps + kk, ..: expert a, block kb of its f.
            struct At {
                int a, kb;
            };
            auto start = [&] { return At{(i0 + kk) / f_blocks, (i0 + kk) % f_blocks}; };
            auto step = [&](At &at) {
                at.kb += p.kps;
                while (at.kb >= f_blocks) at.kb -= f_blocks, at.a++;
            };
            At w = start(), r = start();
            auto weights = [&](int i, int s) {
                const int nk = min(p.kps, i1 - i);
                if (lane == 0) ptx::mbar_arrive_expect_tx(bar(h.full[s]), uint32_t(nk) * (h_bytes + w_bytes));
                __syncwarp();
                if (kk < nk && lane < 8)
                    ptx::tma_load_2d(ring + uint32_t(s) * p.stage_bytes + w0 + uint32_t(kk) * w_bytes, &tmD, bar(h.full[s]), w.kb * 64, h.expert[w.a] * p.d + n0);
                step(w);
            };
            auto rows = [&](int i, int s) {
                const int nk = min(p.kps, i1 - i);
                if (kk < nk && lane >= 8 && lane < 16)
                    ptx::tma_load_2d(ring + uint32_t(s) * p.stage_bytes + uint32_t(kk) * h_bytes, &tmH, bar(h.full[s]), r.kb * 64, r.a * p.token_rows);
                step(r);
                __syncwarp();
            };
            for (int i = 0; i < ahead; i++) weights(i0 + i * p.kps, i);
            ptx::griddep_wait();
            for (int i = 0; i < ahead; i++) rows(i0 + i * p.kps, i);
            filled = (1u << ahead) - 1u;
            int s = ahead == p.stages ? 0 : ahead;
            uint32_t ph = ahead == p.stages ? 1u : 0u;
            for (int i = i0 + ahead * p.kps; i < i1; i += p.kps) {
                ok = __all_sync(0xffffffffu, wait_bar(bar(h.empty[s]), ph ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(s), limit));
                if (!ok) break;
                weights(i, s);
                rows(i, s);
                filled_parity = (filled_parity & ~(1u << s)) | (ph << s);
                if (++s == p.stages) s = 0, ph ^= 1u;
            }
        } else {
            ptx::griddep_wait();
        }
        if (!ok && lane == 0) {
            const uint64_t t0 = ptx::globaltimer_ns();
            for (int i = 0; i < p.stages; i++)
                while ((filled >> i & 1u) && !ptx::mbar_try_wait(bar(h.full[i]), (filled_parity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp runs the loop and one thread issues: see lora_few_kernel.
        const bool leader = ptx::elect_one();
        bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_MMA_TMEM, 100u, limit)), issued = false;
        ptx::tc_fence_after();  // the zeros in the accumulator
        const int64_t all = ok ? int64_t(h.active) * f_blocks : 0;
        const int i0 = int(all * rank / p.kc), i1 = int(all * (rank + 1) / p.kc);
        const uint32_t idesc = make_idesc(p.bf16, 128, p.bn);
        int s = 0, kk = 0, a_at = i0 / f_blocks, left = f_blocks - i0 % f_blocks;  // blocks left of this expert
        uint32_t ph = 0, src = 0;
        for (int i = i0; i < i1 && ok; a_at++, left = f_blocks) {
            const unsigned long long who = h.who[h.expert[a_at]];
            const uint32_t off0 = __shfl_sync(0xffffffffu, ~uint32_t(who), 0), off1 = __shfl_sync(0xffffffffu, ~uint32_t(who >> 32), 0);
            for (const int end = min(i1, i + left); i < end; i++) {
                if (kk == 0) {
                    ok = __all_sync(0xffffffffu, wait_bar(bar(h.full[s]), ph, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(s), limit));
                    if (!ok) break;
                    ptx::tc_fence_after();
                    src = ring + uint32_t(s) * p.stage_bytes;
                }
                const uint64_t a = sw128_desc(src + uint32_t(kk) * h_bytes), b = sw128_desc(src + w0 + uint32_t(kk) * w_bytes);
                if (leader) {
#pragma unroll
                    for (int j = 0; j < 4; j++) ptx::umma_f16_lanes(tmem, a + 2u * j, b + 2u * j, idesc, 1u, off0, off1, 0xffffffffu, 0xffffffffu);
                }
                __syncwarp();
                issued = true;
                if (++kk == p.kps || i + 1 == i1) {
                    if (leader) ptx::umma_commit<1>(bar(h.empty[s]));
                    __syncwarp();
                    kk = 0;
                    if (++s == p.stages) s = 0, ph ^= 1u;
                }
            }
        }
        if (leader) {
            if (ok) {
                ptx::umma_commit<1>(bar(h.done));
            } else if (issued) {
                ptx::umma_commit<1>(bar(h.drain));
                const uint64_t t0 = ptx::globaltimer_ns();
                while (!ptx::mbar_try_wait(bar(h.drain), 0u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            }
        }
        __syncwarp();
    } else {
        const int q = warp & 3;
        const uint32_t lanes = tmem + (uint32_t(32 * q) << 16);
        if (q < 2) {
            for (int c = 0; c < p.bn; c += 32) ptx::tmem_zero_32x32(lanes + uint32_t(c));
            ptx::tc_fence_before();
        }
        find_active(h, p, threadIdx.x - 64);  // ends with a barrier of these warps: the zeros are in place
        if (threadIdx.x == 64) ptx::mbar_arrive(bar(h.plan));
        const bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.done), 0, abort_flag, p.status, WHERE_EPILOGUE, 0u, limit));
        const uint32_t pitch = uint32_t(p.bn + 4) * 4u;
        if (ok && 32 * q < p.tokens) {
            ptx::tc_fence_after();
            ptx::fence_proxy_async_shared();
            for (int c = 0; c < p.bn; c += 32) {
                uint32_t v[32];
                ptx::tmem_ld_32x32(lanes + uint32_t(c), v);
                ptx::tmem_ld_wait(v);
                if (32 * q + lane < p.tokens) {
                    const uint32_t dst = ring + uint32_t(32 * q + lane) * pitch + uint32_t(c) * 4u;
#pragma unroll
                    for (int g = 0; g < 8; g++)
                        if (c + 4 * g < p.bn) ptx::st_shared_v4(dst + 16u * g, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
                }
            }
        }
        ptx::griddep_wait();  // Y is written below: nothing of an earlier kernel may still read it
        __syncwarp();
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (p.kc > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (!*abort_flag) {
        const int quads = p.bn / 4, items = p.tokens * quads;
        const uint32_t pitch = uint32_t(p.bn + 4) * 4u;
        for (int i = int(rank) * MOE_THREADS + int(threadIdx.x); i < items; i += p.kc * MOE_THREADS) {
            const int row = i / quads, col = (i - row * quads) * 4;
            const uint32_t at = ring + uint32_t(row) * pitch + uint32_t(col) * 4u;
            const float4 v = cluster_sum(at, p.kc);
            if (n0 + col < p.d)  // d is a multiple of 8: four columns are in or out together
                *reinterpret_cast<uint2 *>(p.y + int64_t(row) * p.d + n0 + col) = make_uint2(pack_16(v.x, v.y, p.bf16), pack_16(v.z, v.w, p.bf16));
        }
    }
    __syncthreads();
    if (p.kc > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, p.tmem_cols);
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

int token_rows(const cute_b200_moe_desc &d) { return (d.tokens + 7) / 8 * 8; }
int most_active(const cute_b200_moe_desc &d) { return d.experts < d.tokens * d.top ? d.experts : d.tokens * d.top; }

struct Layout {
    uint64_t ids, weights, h, total;
};
Layout layout(const cute_b200_moe_desc &d) {
    Layout l;
    l.ids = 0;
    l.weights = l.ids + round_up(uint64_t(d.tokens) * d.top * 4);
    l.h = l.weights + round_up(uint64_t(d.tokens) * d.top * 4);
    l.total = l.h + round_up(uint64_t(most_active(d)) * token_rows(d) * d.f * 2) + kAlign;
    return l;
}

// Stages of `bytes` behind the head; an MMA reads 128 rows of 128 bytes from up to `last` bytes behind a stage's start.
int ring_stages(uint32_t bytes, uint32_t last, uint32_t before = 0) {
    const uint32_t ring = MOE_SMEM - MOE_HEAD - 1024 - before, reach = last + 16384, over = bytes < reach ? reach - bytes : 0;
    const int stages = int((ring - over) / bytes);
    return stages < MOE_MAX_STAGES ? stages : MOE_MAX_STAGES;
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

cute_b200_status moe_tn(const cute_b200_moe_desc &d, const uint64_t ptr[7], cudaStream_t stream, const DeviceState &dev) {
    if (d.tokens == 0) return CUTE_B200_OK;
    const Layout l = layout(d);
    MoeParams p = {};
    p.x = reinterpret_cast<const uint16_t *>(ptr[0]);
    p.r = reinterpret_cast<const uint16_t *>(ptr[1]);
    p.y = reinterpret_cast<uint16_t *>(ptr[5]);
    p.ids = reinterpret_cast<int32_t *>(ptr[6] + l.ids);
    p.weights = reinterpret_cast<float *>(ptr[6] + l.weights);
    p.h = reinterpret_cast<uint16_t *>(ptr[6] + l.h);
    p.tokens = d.tokens, p.token_rows = token_rows(d), p.experts = d.experts, p.top = d.top, p.d = d.d, p.f = d.f, p.renorm = d.renormalise;
    p.bf16 = d.dtype == CUTE_B200_BF16;
    p.status = dev.status_word;
    p.debug = d.tuning[1];

    const dim3 groups(unsigned((d.tokens + ROUTER_TOKENS - 1) / ROUTER_TOKENS * ROUTER_CLUSTER));
    CB_TRY(launch_dependent(p.bf16 ? moe_router_kernel<true> : moe_router_kernel<false>, groups, ROUTER_THREADS, 0, ROUTER_CLUSTER, stream, p));

    CUtensorMap tmX, tmH, tmD;
    UpMaps maps;
    CB_TRY(rows_tensor_map(&tmX, ptr[0], p.bf16, d.tokens, d.d, d.d, p.token_rows));
    for (int i = 0; i < 4; i++) {
        CB_TRY(rows_tensor_map(&maps.gate[i], ptr[2], p.bf16, uint64_t(d.experts) * d.f, d.d, d.d, 64 >> i));
        CB_TRY(rows_tensor_map(&maps.up[i], ptr[3], p.bf16, uint64_t(d.experts) * d.f, d.d, d.d, 64 >> i));
    }
    p.stage_bytes = uint32_t(2 * p.token_rows + 16 * UP_GROUPS) * 128u;
    p.stages = ring_stages(p.stage_bytes, 0, up_step_bytes(p.token_rows));
    CB_TRY(launch_dependent(moe_up_kernel, dim3(unsigned(dev.sm_count)), MOE_THREADS, MOE_SMEM, 1, stream, tmX, maps, p));

    p.bn = 16, p.kc = 1;
    const int f_blocks = (d.f + 63) / 64, expected = most_active(d);
    int fits[4];
    for (int c = 0; c < 4; c++) fits[c] = (1 << c) <= f_blocks ? dev.down_clusters[c] : 0;  // every CTA has a block of one expert at least
    stream_cut(d.d, f_blocks * expected, fits, &p.bn, &p.kc);
    p.kps = stream_blocks(p.bn, p.token_rows, MOE_SMEM - MOE_HEAD - 1024);
    p.stage_bytes = uint32_t(p.kps * (p.token_rows + p.bn)) * 128u;
    p.stages = ring_stages(p.stage_bytes, uint32_t((p.kps - 1) * p.token_rows) * 128u);
    p.tmem_cols = p.bn <= 32 ? 32 : (p.bn <= 64 ? 64 : (p.bn <= 128 ? 128 : 256));
    CB_TRY(rows_tensor_map(&tmH, ptr[6] + l.h, p.bf16, uint64_t(expected) * p.token_rows, d.f, d.f, p.token_rows));
    CB_TRY(rows_tensor_map(&tmD, ptr[4], p.bf16, uint64_t(d.experts) * d.d, d.f, d.f, p.bn));
    return launch_dependent(moe_down_kernel, dim3(unsigned((d.d + p.bn - 1) / p.bn * p.kc)), MOE_THREADS, MOE_SMEM, p.kc, stream, tmH, tmD, p);
}

cute_b200_status moe_init(DeviceState &dev) {
    CB_CUDA(cudaFuncSetAttribute(moe_up_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOE_SMEM));
    CB_CUDA(cudaFuncSetAttribute(moe_down_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOE_SMEM));
    for (int c = 0; c < 4; c++) CB_TRY(max_clusters(moe_down_kernel, MOE_THREADS, MOE_SMEM, 1 << c, &dev.down_clusters[c]));
    return CUTE_B200_OK;
}

}  // namespace cb
