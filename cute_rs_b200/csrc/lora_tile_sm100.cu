// lora_tn for more rows than one accumulator holds: the inner products T by a
// tensor-core kernel of its own, then a persistent tiled GEMM whose k loop runs
// on, behind the last block of W, over the adapters that the tile's rows name.
#include "lora_sm100.cuh"

namespace cb {
namespace {

constexpr int BM = 128, BK = 64;

// The plan: for every tile of P rows (P = the rows of the GEMM's tile) the adapters its rows name, in the order of
// their first row, each with P / 32 words whose bit is set for a row of another adapter.  Words per tile: a header of
// four (count first), then per entry four (id first) and the masks; at most min(P, adapters) entries.
__host__ __device__ constexpr uint64_t plan_stride(int P, int adapters) {
    return 4 + uint64_t(P < adapters ? P : adapters) * uint64_t(4 + P / 32);
}

// ---- T --------------------------------------------------------------------------
// T[i] = scale * A[ids[i]] x_i for 128 rows per CTA, the k range of a tile shared by
// a cluster.  M = the rows, N = the padded rank: every adapter's MMAs are masked to
// the lanes of its rows, so one accumulator serves all of them.  Bound by reading X
// (and, where nearly every row has an adapter of its own, A).
//   warp 0  TMA: per k block a (128 x 64) block of X into one ring, then for every
//           adapter of the tile a (rp x 64) block of A into another.
//   warp 1  MMA.   warps 2-5  plan (own rows for the masks; the cluster's first CTA also
//           the plan of the GEMM's tile that starts at its rows), then the sum over the
//           cluster, scale, split into two 16-bit numbers.
constexpr int SHRINK_THREADS = 192, X_STAGES = 7, A_STAGES = 16;
constexpr uint32_t X_BYTES = BM * BK * 2, A_RING = 64 * 1024, SHRINK_HEAD = 8192;
constexpr uint32_t SHRINK_SMEM = 1024 + SHRINK_HEAD + X_STAGES * X_BYTES + A_RING;

struct ShrinkParams {
    const int32_t *ids;
    const float *scale;
    uint16_t *t;
    uint32_t *plan;
    int m, rank, rp, adapters, k_blocks, kc, plan_rows, a_stages;
    uint32_t idesc, tmem_cols;
    uint32_t *status;
    int debug;
};

struct ShrinkHead {
    uint64_t xfull[X_STAGES], xempty[X_STAGES], afull[A_STAGES], aempty[A_STAGES], plan, done, drain;
    uint32_t tmem, abort;
    int32_t entries, entry_id[BM], before[4];
    uint32_t off[BM][4];
    int32_t id[BM], wide[512];  // this CTA's rows; the rows of the GEMM's tile
};
static_assert(sizeof(ShrinkHead) <= SHRINK_HEAD, "head");

// Which of `rows` (a multiple of 128, at most 512) ids are the first of their kind, and the list of those, by 128 threads:
// thread `t` holds rows t, t + 128, ..  `id` is in shared memory, negative = none.  `emit(e, id)` receives the list,
// the count is returned to every thread.
template <typename Emit>
__device__ __forceinline__ int distinct_ids(const int32_t *id, int rows, int t, int32_t (&before)[4], Emit emit) {
    const int lane = t & 31, w = t >> 5;
    int total = 0;
    for (int r0 = 0; r0 < rows; r0 += 128) {
        const int r = r0 + t, mine = id[r];
        bool first = mine >= 0 && (r == 0 || id[r - 1] != mine);
        if (first)
            for (int i = 0; i + 1 < r; i++)
                if (id[i] == mine) {
                    first = false;
                    break;
                }
        __syncwarp();
        const uint32_t firsts = __ballot_sync(0xffffffffu, first);
        if (lane == 0) before[w] = __popc(firsts);
        ptx::named_barrier(1, 128);
        int at = total + __popc(firsts & ((1u << lane) - 1u));
        for (int i = 0; i < 4; i++) {
            if (i < w) at += before[i];
            total += before[i];
        }
        if (first) emit(at, mine);
        ptx::named_barrier(1, 128);
    }
    return total;
}

template <bool BF16>
__global__ void __launch_bounds__(SHRINK_THREADS, 1)
    shrink_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, const ShrinkParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    ShrinkHead &h = *reinterpret_cast<ShrinkHead *>(smem_raw + (base - raw));
    const uint32_t xring = base + SHRINK_HEAD, aring = xring + X_STAGES * X_BYTES, a_bytes = uint32_t(p.rp) * 128u;
    auto bar = [&](uint64_t &b) { return ptx::smem_u32(&b); };
    volatile uint32_t *abort_flag = &h.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = p.kc > 1 ? ptx::cluster_ctarank() : 0u;
    const int tile = int(blockIdx.x) / p.kc, row0 = tile * BM;
    const int kb0 = int(int64_t(p.k_blocks) * rank / p.kc), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / p.kc);
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < X_STAGES; s++) {
            ptx::mbar_init(bar(h.xfull[s]), 1);
            ptx::mbar_init(bar(h.xempty[s]), 1);
        }
        for (int s = 0; s < A_STAGES; s++) {
            ptx::mbar_init(bar(h.afull[s]), 1);
            ptx::mbar_init(bar(h.aempty[s]), 1);
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
    ptx::griddep_wait();
    if (threadIdx.x == 0) ptx::griddep_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            ptx::prefetch_tensormap(&tmX);
            ptx::prefetch_tensormap(&tmA);
            bool ok = !(p.debug & 4) && wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_PRODUCER, 100u, limit);
            const int entries = ok ? h.entries : 0;
            int sx = 0, sa = 0;
            uint32_t px = 0, pa = 0, xfilled = 0, xparity = 0, afilled = 0, aparity = 0;
            for (int kb = kb0; kb < kb1 && ok && entries > 0; kb++) {
                if (!(ok = wait_bar(bar(h.xempty[sx]), px ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(sx), limit))) break;
                ptx::mbar_arrive_expect_tx(bar(h.xfull[sx]), X_BYTES);
                ptx::tma_load_2d(xring + uint32_t(sx) * X_BYTES, &tmX, bar(h.xfull[sx]), kb * BK, row0);
                xfilled |= 1u << sx, xparity = (xparity & ~(1u << sx)) | (px << sx);
                if (++sx == X_STAGES) sx = 0, px ^= 1u;
                for (int e = 0; e < entries; e++) {
                    if (!(ok = wait_bar(bar(h.aempty[sa]), pa ^ 1u, abort_flag, p.status, WHERE_PRODUCER, 32u + uint32_t(sa), limit))) break;
                    ptx::mbar_arrive_expect_tx(bar(h.afull[sa]), a_bytes);
                    ptx::tma_load_2d(aring + uint32_t(sa) * a_bytes, &tmA, bar(h.afull[sa]), kb * BK, h.entry_id[e] * p.rank);
                    afilled |= 1u << sa, aparity = (aparity & ~(1u << sa)) | (pa << sa);
                    if (++sa == p.a_stages) sa = 0, pa ^= 1u;
                }
            }
            if (!ok) {  // giving up: let the copies in flight land (bounded)
                const uint64_t t0 = ptx::globaltimer_ns();
                for (int i = 0; i < X_STAGES; i++)
                    while ((xfilled >> i & 1u) && !ptx::mbar_try_wait(bar(h.xfull[i]), (xparity >> i) & 1u))
                        if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
                for (int i = 0; i < A_STAGES; i++)
                    while ((afilled >> i & 1u) && !ptx::mbar_try_wait(bar(h.afull[i]), (aparity >> i) & 1u))
                        if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_MMA_TMEM, 100u, limit), issued = false;
            const int entries = ok ? h.entries : 0;
            int sx = 0, sa = 0;
            uint32_t px = 0, pa = 0;
            for (int kb = kb0; kb < kb1 && ok && entries > 0; kb++) {
                if (!(ok = wait_bar(bar(h.xfull[sx]), px, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(sx), limit))) break;
                const uint64_t a = sw128_desc(xring + uint32_t(sx) * X_BYTES);
                for (int e = 0; e < entries; e++) {
                    if (!(ok = wait_bar(bar(h.afull[sa]), pa, abort_flag, p.status, WHERE_MMA_FULL, 32u + uint32_t(sa), limit))) break;
                    ptx::tc_fence_after();
                    const uint64_t b = sw128_desc(aring + uint32_t(sa) * a_bytes);
                    const uint32_t o0 = h.off[e][0], o1 = h.off[e][1], o2 = h.off[e][2], o3 = h.off[e][3];
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        ptx::umma_f16_lanes(tmem, a + 2u * j, b + 2u * j, p.idesc, (kb > kb0 || j > 0) ? 1u : 0u, o0, o1, o2, o3);
                    issued = true;
                    ptx::umma_commit<1>(bar(h.aempty[sa]));
                    if (++sa == p.a_stages) sa = 0, pa ^= 1u;
                }
                if (!ok) break;
                ptx::umma_commit<1>(bar(h.xempty[sx]));
                if (++sx == X_STAGES) sx = 0, px ^= 1u;
            }
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
        const int t = threadIdx.x - 64, w = t >> 5;
        auto read_id = [&](int row) {
            const int id = row < p.m ? p.ids[row] : -1;
            return id < 0 || id >= p.adapters ? -1 : id;
        };
        h.id[t] = read_id(row0 + t);
        ptx::named_barrier(1, 128);
        const int total = distinct_ids(h.id, 128, t, h.before, [&](int e, int id) { h.entry_id[e] = id; });
        if (t == 0) h.entries = total;
        for (int e = 0; e < total; e++) {
            const uint32_t mine = __ballot_sync(0xffffffffu, h.id[t] == h.entry_id[e]);
            if (lane == 0) h.off[e][w] = ~mine;
        }
        ptx::named_barrier(1, 128);
        if (t == 0) ptx::mbar_arrive(bar(h.plan));
        // The GEMM's plan, by the first CTA of the cluster at the tile's first 128 rows.
        if (rank == 0 && row0 % p.plan_rows == 0) {
            const int P = p.plan_rows, words = P / 32;
            uint32_t *plan = p.plan + uint64_t(row0 / P) * plan_stride(P, p.adapters);
            for (int i = t; i < P; i += 128) h.wide[i] = read_id(row0 + i);
            ptx::named_barrier(1, 128);
            const int count = distinct_ids(h.wide, P, t, h.before, [&](int e, int id) { plan[4 + e * (4 + words)] = uint32_t(id); });
            if (t == 0) plan[0] = uint32_t(count);
            __threadfence_block();
            ptx::named_barrier(1, 128);  // the ids above are read below by the other threads
            for (int e = 0; e < count; e++) {
                uint32_t *entry = plan + 4 + e * (4 + words);
                const int id = int(*reinterpret_cast<volatile uint32_t *>(entry));
                for (int r0 = 0; r0 < P; r0 += 128) {
                    const uint32_t mine = __ballot_sync(0xffffffffu, h.wide[r0 + t] == id);
                    if (lane == 0) entry[4 + r0 / 32 + w] = ~mine;
                }
            }
        }
        // Partial sums to shared memory: the rings are idle.
        const bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.done), 0, abort_flag, p.status, WHERE_EPILOGUE, 0u, limit));
        const int q = warp & 3;
        const uint32_t pitch = uint32_t(p.rp + 4) * 4u;
        if (ok) {
            ptx::tc_fence_after();
            ptx::fence_proxy_async_shared();
            for (int c = 0; c < p.rp; c += 32) {
                uint32_t v[32];
                ptx::tmem_ld_32x32(tmem + (uint32_t(32 * q) << 16) + uint32_t(c), v);
                ptx::tmem_ld_wait(v);
                const uint32_t dst = xring + uint32_t(32 * q + lane) * pitch + uint32_t(c) * 4u;
#pragma unroll
                for (int g = 0; g < 8; g++)
                    if (c + 4 * g < p.rp) ptx::st_shared_v4(dst + 16u * g, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            }
        }
        __syncwarp();
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (p.kc > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (!*abort_flag) {
        const int quads = p.rp / 4;
        const uint32_t pitch = uint32_t(p.rp + 4) * 4u;
        for (int i = int(rank) * SHRINK_THREADS + int(threadIdx.x); i < BM * quads; i += p.kc * SHRINK_THREADS) {
            const int row = i / quads, col = (i - row * quads) * 4;
            if (row0 + row >= p.m) break;
            const int id = h.id[row];
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (id >= 0 && col < p.rank) {  // lanes of rows without an adapter hold nothing; past the rank lie the next adapter's sums
                const uint32_t at = xring + uint32_t(row) * pitch + uint32_t(col) * 4u;
                v = cluster_sum(at, p.kc);
                const float s = p.scale[id];
                v.x *= s, v.y *= s, v.z *= s, v.w *= s;
            }
            const uint32_t h0 = pack_16(v.x, v.y, BF16), h1 = pack_16(v.z, v.w, BF16);
            const float2 f0 = pair_f32<BF16>(h0), f1 = pair_f32<BF16>(h1);
            uint16_t *t = p.t + int64_t(row0 + row) * 2 * p.rp + col;
            *reinterpret_cast<uint2 *>(t) = make_uint2(h0, h1);
            *reinterpret_cast<uint2 *>(t + p.rp) = make_uint2(pack_16(v.x - f0.x, v.y - f0.y, BF16), pack_16(v.z - f1.x, v.w - f1.y, BF16));
        }
    }
    __syncthreads();
    if (p.kc > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, p.tmem_cols);
}

// ---- Y --------------------------------------------------------------------------
// The structure of the library's GEMM: persistent CTAs or CTA pairs, a TMA warp, an MMA warp, eight epilogue warps, a
// ring of 192 KiB.  G: CTAs per MMA; BN: columns per tile; MH: 128-row accumulators per CTA.  Behind a tile's k blocks
// of W come, for every adapter its rows name, the blocks of T (in place of X) and of B[a] (in place of W), their MMAs
// masked to the lanes of the adapter's rows.  One adapter of rank 64 costs 2 blocks beside the 64 of k = 4096.
constexpr uint32_t RING_BYTES = 192 * 1024;
constexpr int TILE_THREADS = 64 + 256;

template <int G, int BN, int MH>
struct Tile {
    static constexpr int CTA_ROWS = BM * MH, ROWS = CTA_ROWS * G, B_ROWS = BN / G;
    static constexpr uint32_t A_BYTES = CTA_ROWS * BK * 2, B_BYTES = B_ROWS * BK * 2, KB_BYTES = A_BYTES + B_BYTES;
    static constexpr int KPS = MH == 1 && BN == 128 ? 2 : 1;  // k blocks per stage: a 128 x 128 tile is short on math per block
    static constexpr uint32_t STAGE_BYTES = KPS * KB_BYTES;
    static constexpr int STAGES = int(RING_BYTES / STAGE_BYTES);
    static constexpr int ACC_COLS = MH * BN, ACC_BUFS = 2 * ACC_COLS <= 512 ? 2 : 1;
    static constexpr uint32_t TMEM_COLS = ACC_COLS * ACC_BUFS;
    static constexpr uint32_t SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 512;
    static constexpr uint32_t EXPECT = G * KB_BYTES;
    static constexpr int CH = BN / 64;  // 32-column chunks of an accumulator per epilogue warp
    static_assert(STAGES >= 3 && TMEM_COLS <= 512 && SMEM_BYTES <= 227 * 1024 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "tile");
};

struct TileParams {
    const uint32_t *plan;
    void *y;
    int64_t ldy;
    int m, n, rank, rp, adapters, c_dtype, vec;
    int k_blocks, m_tiles, n_tiles, group_m;
    uint32_t idesc;
    uint32_t *status;
    int debug;
};

struct TileAt {
    int tm, tn;
};
// `group_m` row tiles are walked before the column advances, so that the CTAs running at one time share panels in L2.
__device__ __forceinline__ TileAt tile_at(int t, const TileParams &p) {
    const int size = p.group_m * p.n_tiles, g = t / size, first = g * p.group_m, gm = min(p.group_m, p.m_tiles - first), r = t - g * size;
    return {first + r % gm, r / gm};
}

__device__ __forceinline__ void store_32(const TileParams &p, int row, int col, const uint32_t (&v)[32]) {
    if (row >= p.m || col >= p.n) return;
    const int64_t at = int64_t(row) * p.ldy + col;
    if (p.vec && col + 32 <= p.n) {
        if (p.c_dtype == CUTE_B200_F32) {
            float *c = static_cast<float *>(p.y) + at;
            if (p.vec == 2) {
#pragma unroll
                for (int g = 0; g < 4; g++)
                    ptx::st_global_v8(c + 8 * g, v[8 * g], v[8 * g + 1], v[8 * g + 2], v[8 * g + 3], v[8 * g + 4], v[8 * g + 5], v[8 * g + 6], v[8 * g + 7]);
            } else {
#pragma unroll
                for (int g = 0; g < 8; g++) *reinterpret_cast<uint4 *>(c + 4 * g) = make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            }
        } else {
            const bool bf16 = p.c_dtype == CUTE_B200_BF16;
            uint16_t *c = static_cast<uint16_t *>(p.y) + at;
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; j++) w[j] = pack_16(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]), bf16);
            if (p.vec == 2) {
                ptx::st_global_v8(c, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
                ptx::st_global_v8(c + 16, w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15]);
            } else {
#pragma unroll
                for (int g = 0; g < 4; g++) *reinterpret_cast<uint4 *>(c + 8 * g) = make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (col + j < p.n) store_c(p.y, p.c_dtype, size_t(at + j), __uint_as_float(v[j]));
    }
}

template <int G, int BN, int MH>
__global__ void __launch_bounds__(TILE_THREADS, 1)
    lora_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmT,
                     const __grid_constant__ CUtensorMap tmB, const TileParams p) {
    using C = Tile<G, BN, MH>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), ring = (raw + 1023u) & ~1023u, bars = ring + C::STAGES * C::STAGE_BYTES;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
    auto tfull_bar = [&](int b) { return bars + 8u * (2 * C::STAGES + b); };
    auto tempty_bar = [&](int b, int h) { return bars + 8u * (2 * C::STAGES + 2 + 2 * b + h); };
    const uint32_t drain_bar = bars + 8u * (2 * C::STAGES + 6);
    uint8_t *tail = smem_raw + (bars - raw) + 8u * (2 * C::STAGES + 7);
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(tail);
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(tail + 4);
    static_assert(8 * (2 * C::STAGES + 7) + 8 <= 512, "barriers");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = G == 1 ? 0u : ptx::cluster_ctarank();
    const int first = int(blockIdx.x) / G, step = int(gridDim.x) / G, tiles = p.m_tiles * p.n_tiles;
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;
    const uint64_t stride = plan_stride(C::ROWS, p.adapters);
    constexpr int ENTRY = 4 + C::ROWS / 32;
    const int q_blocks = ext_blocks(p.rp);

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; b++) {
            ptx::mbar_init(tfull_bar(b), 1);
            for (int h = 0; h < 2; h++) ptx::mbar_init(tempty_bar(b, h), 8 * G);
        }
        ptx::mbar_init(drain_bar, 1);
        *abort_flag = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<G>(ptx::smem_u32(const_cast<uint32_t *>(tmem_slot)), C::TMEM_COLS);
        ptx::tmem_relinquish<G>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (G == 2) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (threadIdx.x == 0) ptx::griddep_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            ptx::prefetch_tensormap(&tmX);
            ptx::prefetch_tensormap(&tmW);
            ptx::prefetch_tensormap(&tmT);
            ptx::prefetch_tensormap(&tmB);
            int s = 0;
            uint32_t ph = 0, filled = 0, filled_parity = 0;
            bool ok = !(p.debug & 4), waited = false;
            // One stage of `nk` k blocks from column ax of `rows` and bx of `weights`.
            auto load = [&](int nk, const CUtensorMap *rows, int ax, int ay, const CUtensorMap *weights, int bx, int by) {
                if (!wait_bar(empty_bar(s), ph ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(s), limit)) return false;
                const uint32_t dst = ring + uint32_t(s) * C::STAGE_BYTES;
                if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(s), uint32_t(nk) * C::EXPECT);
                const uint32_t bar = G == 1 ? full_bar(s) : ptx::mapa(full_bar(s), 0);
#pragma unroll
                for (int kk = 0; kk < C::KPS; kk++)
                    if (kk < nk) {
                        if constexpr (G == 1) {
                            ptx::tma_load_2d(dst + kk * C::KB_BYTES, rows, bar, ax + kk * BK, ay);
                            ptx::tma_load_2d(dst + kk * C::KB_BYTES + C::A_BYTES, weights, bar, bx + kk * BK, by);
                        } else {
                            ptx::tma_load_2d_pair(dst + kk * C::KB_BYTES, rows, bar, ax + kk * BK, ay);
                            ptx::tma_load_2d_pair(dst + kk * C::KB_BYTES + C::A_BYTES, weights, bar, bx + kk * BK, by);
                        }
                    }
                filled |= 1u << s, filled_parity = (filled_parity & ~(1u << s)) | (ph << s);
                if (++s == C::STAGES) s = 0, ph ^= 1u;
                return true;
            };
            for (int t = first; t < tiles && ok; t += step) {
                const TileAt at = tile_at(t, p);
                const int row = at.tm * C::ROWS + int(rank) * C::CTA_ROWS, col = at.tn * BN + int(rank) * C::B_ROWS;
                for (int kb = 0; kb < p.k_blocks && ok; kb += C::KPS)
                    ok = load(min(C::KPS, p.k_blocks - kb), &tmX, kb * BK, row, &tmW, kb * BK, col);
                if (!ok) break;
                if (!waited) ptx::griddep_wait(), waited = true;  // T and the plan; X and W are older than their kernel
                const uint32_t *plan = p.plan + uint64_t(at.tm) * stride;
                const int entries = int(plan[0]);
                for (int e = 0; e < entries && ok; e++) {
                    const int id = int(plan[4 + e * ENTRY]);
                    for (int q = 0; q < q_blocks && ok; q++) {
                        const ExtBlock b = ext_block(q, p.rp, p.rank);
                        ok = load(1, &tmT, b.t_col, row, &tmB, b.b_col, id * p.n + col);
                    }
                }
            }
            if (!ok && rank == 0) {  // giving up: let the copies in flight land (bounded)
                const uint64_t t0 = ptx::globaltimer_ns();
                for (int i = 0; i < C::STAGES; i++)
                    while ((filled >> i & 1u) && !ptx::mbar_try_wait(full_bar(i), (filled_parity >> i) & 1u))
                        if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            }
            if (!waited) ptx::griddep_wait();
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int s = 0, it = 0;
            uint32_t ph = 0;
            bool ok = true, issued = false, waited = false;
            auto ready = [&] {
                if (!wait_bar(full_bar(s), ph, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(s), limit)) return false;
                ptx::tc_fence_after();
                return true;
            };
            auto free_stage = [&] {
                issued = true;
                ptx::umma_commit<G>(empty_bar(s));
                if constexpr (G == 2) ptx::umma_commit<G>(ptx::mapa(empty_bar(s), 1));
                if (++s == C::STAGES) s = 0, ph ^= 1u;
            };
            for (int t = first; t < tiles && ok; t += step, it++) {
                const TileAt at = tile_at(t, p);
                const int buf = it % C::ACC_BUFS;
                const uint32_t aph = uint32_t(it / C::ACC_BUFS) & 1u, d = tmem + uint32_t(buf * C::ACC_COLS);
                for (int k0 = 0; k0 < p.k_blocks; k0 += C::KPS) {
                    if (!(ok = ready())) break;
                    const uint32_t stage = ring + uint32_t(s) * C::STAGE_BYTES;
#pragma unroll
                    for (int kk = 0; kk < C::KPS; kk++) {
                        if (k0 + kk >= p.k_blocks) break;
                        const bool fresh = k0 == 0 && kk == 0;
                        const uint32_t src = stage + kk * C::KB_BYTES;
                        const uint64_t b = sw128_desc(src + C::A_BYTES);
#pragma unroll
                        for (int h = 0; h < MH; h++) {
                            if (fresh) {  // the epilogue must have drained this half of the buffer
                                if (!(ok = wait_bar(tempty_bar(buf, h), aph ^ 1u, abort_flag, p.status, WHERE_MMA_TMEM, uint32_t(buf * 2 + h), limit))) break;
                                ptx::tc_fence_after();
                            }
                            const uint64_t a = sw128_desc(src + uint32_t(h) * (BM * BK * 2));
#pragma unroll
                            for (int j = 0; j < 4; j++) ptx::umma_f16<G>(d + uint32_t(h * BN), a + 2u * j, b + 2u * j, p.idesc, (!fresh || j > 0) ? 1u : 0u);
                            issued = true;
                        }
                        if (!ok) break;
                    }
                    if (!ok) break;
                    free_stage();
                }
                if (!ok) break;
                if (!waited) ptx::griddep_wait(), waited = true;
                const uint32_t *plan = p.plan + uint64_t(at.tm) * stride;
                const int entries = int(plan[0]);
                for (int e = 0; e < entries && ok; e++) {
                    uint32_t off[C::ROWS / 32];
#pragma unroll
                    for (int i = 0; i < C::ROWS / 32; i += 4) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(plan + 4 + e * ENTRY + 4 + i);
                        off[i] = v.x, off[i + 1] = v.y, off[i + 2] = v.z, off[i + 3] = v.w;
                    }
                    for (int q = 0; q < q_blocks; q++) {
                        const ExtBlock x = ext_block(q, p.rp, p.rank);
                        if (!(ok = ready())) break;
                        const uint32_t src = ring + uint32_t(s) * C::STAGE_BYTES;
                        const uint64_t b = sw128_desc(src + C::A_BYTES);
#pragma unroll
                        for (int h = 0; h < MH; h++) {
                            const uint64_t a = sw128_desc(src + uint32_t(h) * (BM * BK * 2));
                            uint32_t m[4 * G];
#pragma unroll
                            for (int i = 0; i < 4 * G; i++) m[i] = off[(i / 4) * (C::CTA_ROWS / 32) + 4 * h + i % 4];
                            uint32_t all = 0xffffffffu;
#pragma unroll
                            for (int i = 0; i < 4 * G; i++) all &= m[i];
                            if (all == 0xffffffffu) continue;  // no row of these accumulators
                            for (int j = 0; j < x.steps; j++) {
                                if constexpr (G == 1)
                                    ptx::umma_f16_lanes(d + uint32_t(h * BN), a + 2u * j, b + 2u * (j & x.b_mask), p.idesc, 1u, m[0], m[1], m[2], m[3]);
                                else
                                    ptx::umma_f16_lanes_pair(d + uint32_t(h * BN), a + 2u * j, b + 2u * (j & x.b_mask), p.idesc, 1u, m);
                            }
                        }
                        free_stage();
                    }
                }
                if (!ok) break;
                ptx::umma_commit<G>(tfull_bar(buf));
                if constexpr (G == 2) ptx::umma_commit<G>(ptx::mapa(tfull_bar(buf), 1));
            }
            if (!ok && issued) {
                ptx::umma_commit<G>(drain_bar);
                const uint64_t t0 = ptx::globaltimer_ns();
                while (!ptx::mbar_try_wait(drain_bar, 0u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            }
        }
        __syncwarp();
    } else {
        const uint32_t q = uint32_t(warp) & 3u;
        const int e = (warp - 2) >> 2;  // of two groups of four warps, each takes every other 32-column chunk
        int it = 0;
        for (int t = first; t < tiles; t += step, it++) {
            const TileAt at = tile_at(t, p);
            const int buf = it % C::ACC_BUFS;
            const bool ok = wait_bar(tfull_bar(buf), uint32_t(it / C::ACC_BUFS) & 1u, abort_flag, p.status, WHERE_EPILOGUE, uint32_t(buf), limit);
            if (!__all_sync(0xffffffffu, ok)) break;
            ptx::tc_fence_after();
            const int row0 = at.tm * C::ROWS + int(rank) * C::CTA_ROWS + int(q) * 32 + lane;
            const uint32_t taddr = tmem + ((q * 32u) << 16) + uint32_t(buf * C::ACC_COLS);
#pragma unroll 1
            for (int h = 0; h < MH; h++) {
                // All of this warp's part of a half is read out and the half handed back before anything is converted
                // or stored: the next tile's first MMA may be waiting for it.
                uint32_t v[C::CH][32];
#pragma unroll
                for (int c = 0; c < C::CH; c++) ptx::tmem_ld_32x32(taddr + uint32_t(h * BN + (2 * c + e) * 32), v[c]);
                ptx::tmem_ld_wait_all();
#pragma unroll
                for (int c = 0; c < C::CH; c++) ptx::pin(v[c]);
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (G == 1) ptx::mbar_arrive(tempty_bar(buf, h));
                    else ptx::mbar_arrive_cluster(ptx::mapa(tempty_bar(buf, h), 0));
                }
#pragma unroll
                for (int c = 0; c < C::CH; c++) store_32(p, row0 + h * BM, at.tn * BN + (2 * c + e) * 32, v[c]);
            }
        }
        __syncwarp();
    }

    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (G == 2) {  // the peer may still arrive on our barriers or read our shared memory
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) ptx::tmem_dealloc<G>(tmem, C::TMEM_COLS);
}

// ---- host -------------------------------------------------------------------------
int g_shrink_clusters[64][4];  // clusters of 1, 2, 4, 8 CTAs of the T kernel that fit each device at once

template <bool BF16>
cute_b200_status shrink(const LoraParams &p, int plan_rows, int debug, const DeviceState &dev, cudaStream_t stream) {
    ShrinkParams s = {};
    s.ids = p.ids, s.scale = p.scale, s.t = p.t, s.plan = p.plan;
    s.m = p.m, s.rank = p.rank, s.rp = p.rp, s.adapters = p.adapters;
    s.k_blocks = (p.k + BK - 1) / BK;
    s.plan_rows = plan_rows;
    s.a_stages = int(A_RING / (uint32_t(p.rp) * 128u));
    if (s.a_stages > A_STAGES) s.a_stages = A_STAGES;
    s.idesc = make_idesc(BF16, 128, p.rp);
    s.tmem_cols = p.rp <= 32 ? 32 : uint32_t(p.rp);
    s.status = dev.status_word;
    s.debug = debug;
    const int tiles = (p.m + BM - 1) / BM;
    // k is cut while that puts more CTAs to work and leaves each at least four blocks.
    int device = 0;
    CB_CUDA(cudaGetDevice(&device));
    s.kc = 1;
    for (int c = 1; c < 4; c++)
        if (tiles <= g_shrink_clusters[device][c] && s.k_blocks >= (4 << c)) s.kc = 1 << c;
    CUtensorMap tmX, tmA;
    CB_TRY(rows_tensor_map(&tmX, reinterpret_cast<uint64_t>(p.x), BF16, p.m, p.k, p.ldx, BM));
    CB_TRY(rows_tensor_map(&tmA, reinterpret_cast<uint64_t>(p.a), BF16, uint64_t(p.adapters) * p.rank, p.k, p.k, p.rp));
    return launch_dependent(shrink_tile_kernel<BF16>, dim3(unsigned(tiles * s.kc)), SHRINK_THREADS, SHRINK_SMEM, s.kc, stream, tmX, tmA, s);
}

template <int G, int BN, int MH>
cute_b200_status launch_tile(const LoraParams &p, bool bf16, int debug, const DeviceState &dev, cudaStream_t stream) {
    using C = Tile<G, BN, MH>;
    TileParams t = {};
    t.plan = p.plan, t.y = p.y, t.ldy = p.ldy;
    t.m = p.m, t.n = p.n, t.rank = p.rank, t.rp = p.rp, t.adapters = p.adapters, t.c_dtype = p.c_dtype;
    const uint64_t esize = p.c_dtype == CUTE_B200_F32 ? 4 : 2, y = reinterpret_cast<uint64_t>(p.y);
    t.vec = y % 32 == 0 && uint64_t(p.ldy) * esize % 32 == 0 ? 2 : (y % 16 == 0 && uint64_t(p.ldy) * esize % 16 == 0 ? 1 : 0);
    t.k_blocks = (p.k + BK - 1) / BK;
    t.m_tiles = (p.m + C::ROWS - 1) / C::ROWS;
    t.n_tiles = (p.n + BN - 1) / BN;
    const int64_t tiles = int64_t(t.m_tiles) * t.n_tiles;
    if (tiles > 0x7fffffff) return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "lora_tn: %d x %d is more than 2^31 tiles", p.m, p.n);
    int clusters = dev.sm_count / G;
    if (tiles < clusters) clusters = int(tiles);
    int gm = 1;
    while (gm * gm * 2 <= clusters) gm *= 2;
    t.group_m = gm < t.m_tiles ? gm : t.m_tiles;
    t.idesc = make_idesc(bf16, 128 * G, BN);
    t.status = dev.status_word;
    t.debug = debug;
    CUtensorMap tmX, tmW, tmT, tmB;
    CB_TRY(rows_tensor_map(&tmX, reinterpret_cast<uint64_t>(p.x), bf16, p.m, p.k, p.ldx, C::CTA_ROWS));
    CB_TRY(rows_tensor_map(&tmW, reinterpret_cast<uint64_t>(p.w), bf16, p.n, p.k, p.k, C::B_ROWS));
    CB_TRY(rows_tensor_map(&tmT, reinterpret_cast<uint64_t>(p.t), bf16, p.m, 2 * p.rp, 2 * p.rp, C::CTA_ROWS));
    CB_TRY(rows_tensor_map(&tmB, reinterpret_cast<uint64_t>(p.b), bf16, uint64_t(p.adapters) * p.n, p.rank, p.rank, C::B_ROWS));
    return launch_dependent(lora_tile_kernel<G, BN, MH>, dim3(unsigned(clusters * G)), TILE_THREADS, C::SMEM_BYTES, G, stream, tmX, tmW, tmT, tmB, t);
}

// Rows of the GEMM's tile, and its columns: whole waves of tiles, each its MMA time at the rate this tiling was measured at
// beside the 512 x 256 pair tile (1.0) plus the time to fill the ring and drain the accumulator.
struct Cut {
    int rows, cols;
    double rate;
};
constexpr Cut CUTS[3] = {{512, 256, 1.0}, {128, 256, 0.86}, {128, 128, 0.7}};
int choose_cut(int m, int n, int k, int sm_count) {
    int best = 0;
    double best_t = 1e300;
    for (int i = 0; i < 3; i++) {
        const int pair = CUTS[i].rows == 512 ? 2 : 1;
        const int64_t tiles = int64_t((m + CUTS[i].rows - 1) / CUTS[i].rows) * ((n + CUTS[i].cols - 1) / CUTS[i].cols);
        const int64_t at_once = sm_count / pair, waves = (tiles + at_once - 1) / at_once;
        const double unit = 2.0 * CUTS[i].rows * CUTS[i].cols * k / (pair * 1.0e13 * CUTS[i].rate);
        const double t = double(waves) * (unit + 2.5e-6) + (pair == 2 ? 2.0e-6 : 0.0);
        if (t < best_t) best_t = t, best = i;
    }
    return best;
}

}  // namespace

uint64_t lora_plan_bytes(int m, int adapters) {
    uint64_t most = 0;
    for (int rows : {128, 512}) {
        const uint64_t b = uint64_t((int64_t(m) + rows - 1) / rows) * plan_stride(rows, adapters) * 4;
        if (b > most) most = b;
    }
    return most;
}

cute_b200_status lora_tiled(const LoraParams &p, bool bf16, int cut, int debug, const DeviceState &dev, cudaStream_t stream) {
    if (cut < 0) cut = choose_cut(p.m, p.n, p.k, dev.sm_count);
    CB_TRY(bf16 ? shrink<true>(p, CUTS[cut].rows, debug, dev, stream) : shrink<false>(p, CUTS[cut].rows, debug, dev, stream));
    if (!p.y) return CUTE_B200_OK;
    if (cut == 0) return launch_tile<2, 256, 2>(p, bf16, debug, dev, stream);
    if (cut == 1) return launch_tile<1, 256, 1>(p, bf16, debug, dev, stream);
    return launch_tile<1, 128, 1>(p, bf16, debug, dev, stream);
}

cute_b200_status lora_tiled_init() {
    int device = 0;
    CB_CUDA(cudaGetDevice(&device));
    CB_CUDA(cudaFuncSetAttribute(shrink_tile_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SHRINK_SMEM));
    CB_CUDA(cudaFuncSetAttribute(shrink_tile_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SHRINK_SMEM));
    CB_CUDA(cudaFuncSetAttribute(lora_tile_kernel<2, 256, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<2, 256, 2>::SMEM_BYTES));
    CB_CUDA(cudaFuncSetAttribute(lora_tile_kernel<1, 256, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<1, 256, 1>::SMEM_BYTES));
    CB_CUDA(cudaFuncSetAttribute(lora_tile_kernel<1, 128, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<1, 128, 1>::SMEM_BYTES));
    for (int c = 0; c < 4; c++)
        CB_TRY(max_clusters(shrink_tile_kernel<true>, SHRINK_THREADS, SHRINK_SMEM, 1 << c, &g_shrink_clusters[device][c]));
    return CUTE_B200_OK;
}

}  // namespace cb
