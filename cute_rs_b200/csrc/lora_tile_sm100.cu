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
// a cluster.  M = the rows, N = the padded ranks of several adapters side by side (an
// MMA of N = 128 takes the 65 clocks that one of N = 16 takes); each row reads its own
// adapter's columns of the accumulator.  Entry e of the tile's adapters has the columns
// of slot e % slots; where there are more entries than slots, the MMAs of entries g slots
// to (g + 1) slots - 1 are masked to the lanes of those entries' rows.  Bound by reading X
// (and, where nearly every row has an adapter of its own, A).
//   warp 0  TMA: two (128 x 64) blocks of X per stage of one ring, then the blocks of A
//           of the tile's adapters for them through another, a lane each (with one block
//           per stage the issuing warp was the bound: 0.3 us a stage).  Both rings are three
//           or four stages deep, as the rank allows: the shorter one is what keeps X coming.
//   warp 1  MMA.   warps 2-5  the adapters the rows name (and, by the cluster's first CTA,
//           the plan of the GEMM's tile that starts at its rows), then the sum over the
//           cluster, scale, split into 16-bit numbers.
// On the way back A is B[a] as it lies, (n, rank): rank is the fast index, so it is an MN-major operand.
// A CTA's k range goes to 1, 2 or 4 accumulators in turn, added in f32 at the end: the tensor core cuts its sums off instead
// of rounding them, an error of the same sign that grows with the products added into one accumulator (256 MMAs of 16: 5e-6
// of the sum, measured), and T enters f32 gradients.
constexpr int SHRINK_THREADS = 192, MAX_X_STAGES = 4, MAX_A_STAGES = 4, X_BLOCKS = 2;
constexpr uint32_t X_BYTES = BM * BK * 2, SHRINK_HEAD = 20 * 1024, SHRINK_RINGS = 192 * 1024;
constexpr int T_PARTS = 4, T_COLS = 512;  // at most; TMEM columns of all accumulators
constexpr uint32_t SHRINK_SMEM = 1024 + SHRINK_HEAD + SHRINK_RINGS;

struct ShrinkParams {
    const int32_t *ids;
    const float *scale;
    uint16_t *t;
    uint32_t *plan;
    int m, rank, rp, adapters, k_blocks, kc;
    int boxes;       // of A per adapter and k block
    uint32_t box_bytes, a_bytes;  // a_bytes: of a stage of A
    int x_stages, a_stages;
    uint32_t idesc;  // without N
    int parts, slot_shift, slot_cols;  // slot_cols: of an entry; an accumulator has slot_cols << slot_shift columns
    bool bf16, mn, early;
    uint32_t *status;
    int debug;
};

template <int P>
struct ShrinkHead {
    uint64_t xfull[MAX_X_STAGES], xempty[MAX_X_STAGES], afull[MAX_A_STAGES], aempty[MAX_A_STAGES], plan, done, drain;
    uint32_t tmem, abort;
    int32_t entries, entry_id[BM], id[BM], entry[BM];  // entry: of a row, -1 = none
    float scale[BM];
    uint32_t off[BM][4];  // by group of slots: lanes of other rows
    IdTable<128> rows;  // of this CTA's rows
    IdTable<P> tile;    // of the GEMM's tile
};

template <int P>
__global__ void __launch_bounds__(SHRINK_THREADS, 1)
    shrink_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, const ShrinkParams p) {
    static_assert(sizeof(ShrinkHead<P>) <= SHRINK_HEAD, "head");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    ShrinkHead<P> &h = *reinterpret_cast<ShrinkHead<P> *>(smem_raw + (base - raw));
    const uint32_t xring = base + SHRINK_HEAD, aring = xring + uint32_t(p.x_stages * X_BLOCKS) * X_BYTES;
    auto bar = [&](uint64_t &b) { return ptx::smem_u32(&b); };
    volatile uint32_t *abort_flag = &h.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = p.kc > 1 ? ptx::cluster_ctarank() : 0u;
    const int row0 = int(blockIdx.x) / p.kc * BM;
    const int kb0 = int(int64_t(p.k_blocks) * rank / p.kc), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / p.kc);
    const uint32_t entry_bytes = uint32_t(p.boxes) * p.box_bytes;
    const int group = min(int(p.a_bytes / entry_bytes), 32 / p.boxes);  // (k block, adapter) pairs per stage of A: 2 to 16
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.x_stages; s++) {
            ptx::mbar_init(bar(h.xfull[s]), 1);
            ptx::mbar_init(bar(h.xempty[s]), 1);
        }
        for (int s = 0; s < p.a_stages; s++) {
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
        ptx::tmem_alloc<1>(ptx::smem_u32(&h.tmem), T_COLS);
        ptx::tmem_relinquish<1>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&h.tmem);
    // early: nothing here depends on the kernel before, which has waited for all before it; it is waited for at the end.
    if (!p.early) ptx::griddep_wait();
    if (threadIdx.x == 0) ptx::griddep_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            ptx::prefetch_tensormap(&tmX);
            ptx::prefetch_tensormap(&tmA);
        }
        bool ok = !(p.debug & 4);
        ok = __all_sync(0xffffffffu, ok && wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_PRODUCER, 100u, limit));
        const int entries = ok ? h.entries : 0, my_item = lane / p.boxes, my_box = lane % p.boxes;
        int sx = 0, sa = 0;
        uint32_t px = 0, pa = 0, xfilled = 0, xparity = 0, afilled = 0, aparity = 0;
        for (int kb = kb0; kb < kb1 && ok && entries > 0; kb += X_BLOCKS) {
            const int nk = min(X_BLOCKS, kb1 - kb), items = nk * entries;
            ok = __all_sync(0xffffffffu, wait_bar(bar(h.xempty[sx]), px ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(sx), limit));
            if (!ok) break;
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar(h.xfull[sx]), uint32_t(nk) * X_BYTES);
            __syncwarp();
            if (lane < nk) ptx::tma_load_2d(xring + uint32_t(sx * X_BLOCKS + lane) * X_BYTES, &tmX, bar(h.xfull[sx]), (kb + lane) * BK, row0);
            __syncwarp();
            xfilled |= 1u << sx, xparity = (xparity & ~(1u << sx)) | (px << sx);
            if (++sx == p.x_stages) sx = 0, px ^= 1u;
            for (int i0 = 0; i0 < items; i0 += group) {
                ok = __all_sync(0xffffffffu, wait_bar(bar(h.aempty[sa]), pa ^ 1u, abort_flag, p.status, WHERE_PRODUCER, 32u + uint32_t(sa), limit));
                if (!ok) break;
                const int count = min(group, items - i0);
                if (lane == 0) ptx::mbar_arrive_expect_tx(bar(h.afull[sa]), uint32_t(count) * entry_bytes);
                __syncwarp();
                if (my_item < count) {
                    const int second = i0 + my_item >= entries ? 1 : 0, id = h.entry_id[i0 + my_item - second * entries];
                    const uint32_t dst = aring + uint32_t(sa) * p.a_bytes + uint32_t(lane) * p.box_bytes;
                    if (p.mn) ptx::tma_load_3d(dst, &tmA, bar(h.afull[sa]), 64 * my_box, (kb + second) * BK, id);
                    else ptx::tma_load_2d(dst, &tmA, bar(h.afull[sa]), (kb + second) * BK, id * p.rank);
                }
                __syncwarp();
                afilled |= 1u << sa, aparity = (aparity & ~(1u << sa)) | (pa << sa);
                if (++sa == p.a_stages) sa = 0, pa ^= 1u;
            }
        }
        if (!ok && lane == 0) {  // giving up: let the copies in flight land (bounded)
            const uint64_t t0 = ptx::globaltimer_ns();
            for (int i = 0; i < p.x_stages; i++)
                while ((xfilled >> i & 1u) && !ptx::mbar_try_wait(bar(h.xfull[i]), (xparity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            for (int i = 0; i < p.a_stages; i++)
                while ((afilled >> i & 1u) && !ptx::mbar_try_wait(bar(h.afull[i]), (aparity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp runs the loop and one thread issues: see lora_few_kernel.
        const bool leader = ptx::elect_one();
        bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_MMA_TMEM, 100u, limit)), issued = false;
        const int entries = ok ? h.entries : 0;
        // The blocks at which the second to fourth accumulator begin.
        static_assert(T_PARTS == 4, "three beginnings");
        const int blocks = kb1 - kb0, never = 0x7fffffff;
        const int begin1 = p.parts > 1 ? (blocks + p.parts - 1) / p.parts : never, begin2 = p.parts > 2 ? (blocks + 1) / 2 : never,
                  begin3 = p.parts > 2 ? (3 * blocks + 3) / 4 : never;
        const int slots = 1 << p.slot_shift;
        const uint32_t part_cols = uint32_t(p.slot_cols) << p.slot_shift;
        int sx = 0, sa = 0;
        uint32_t px = 0, pa = 0;
        for (int kb = kb0; kb < kb1 && ok && entries > 0; kb += X_BLOCKS) {
            const int items = min(X_BLOCKS, kb1 - kb) * entries;
            ok = __all_sync(0xffffffffu, wait_bar(bar(h.xfull[sx]), px, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(sx), limit));
            if (!ok) break;
            for (int i0 = 0; i0 < items; i0 += group) {
                ok = __all_sync(0xffffffffu, wait_bar(bar(h.afull[sa]), pa, abort_flag, p.status, WHERE_MMA_FULL, 32u + uint32_t(sa), limit));
                if (!ok) break;
                ptx::tc_fence_after();
                const int count = min(group, items - i0);
                for (int i = 0; i < count;) {
                    // As many adapters as lie side by side: in this stage, of one k block and one group of slots.
                    const int second = i0 + i >= entries ? 1 : 0, e = i0 + i - second * entries, slot = e & (slots - 1);
                    const int run = min(min(count - i, entries - e), slots - slot), at = kb + second - kb0;
                    const uint32_t src = aring + uint32_t(sa) * p.a_bytes + uint32_t(i) * entry_bytes;
                    const uint64_t a = sw128_desc(xring + uint32_t(sx * X_BLOCKS + second) * X_BYTES);
                    const uint64_t b = p.mn ? mn_desc(src, p.box_bytes) : sw128_desc(src);
                    const uint32_t k_step = p.mn ? MN_K_STEP : 2u, idesc = p.idesc | uint32_t(run * p.slot_cols / 8) << 17;
                    const uint32_t d = tmem + (uint32_t(at >= begin1) + uint32_t(at >= begin2) + uint32_t(at >= begin3)) * part_cols + uint32_t(slot * p.slot_cols);
                    const uint32_t more = at != 0 && at != begin1 && at != begin2 && at != begin3 ? 1u : 0u;
                    const uint32_t *off = h.off[e >> p.slot_shift];
                    const uint32_t o0 = off[0], o1 = off[1], o2 = off[2], o3 = off[3];
                    if (leader) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            ptx::umma_f16_lanes(d, a + 2u * j, b + k_step * j, idesc, j > 0 ? 1u : more, o0, o1, o2, o3);
                    }
                    __syncwarp();
                    i += run;
                }
                issued = true;
                if (leader) ptx::umma_commit<1>(bar(h.aempty[sa]));
                __syncwarp();
                if (++sa == p.a_stages) sa = 0, pa ^= 1u;
            }
            if (!ok) break;
            if (leader) ptx::umma_commit<1>(bar(h.xempty[sx]));
            __syncwarp();
            if (++sx == p.x_stages) sx = 0, px ^= 1u;
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
        const int t = threadIdx.x - 64;
        auto read_id = [&](int row) {
            const int id = row < p.m ? __ldcg(p.ids + row) : -1;
            return id < 0 || id >= p.adapters ? -1 : id;
        };
        {
            const int32_t ids[1] = {read_id(row0 + t)};
            int32_t mine[1];
            h.id[t] = ids[0];
            h.scale[t] = ids[0] >= 0 ? __ldcg(p.scale + ids[0]) : 0.0f;
            for (int i = t; i < BM * 4; i += 128) h.off[i / 4][i % 4] = 0xffffffffu;
            const int total = distinct_ids<128>(ids, h.rows, t, mine, [&](int e, int id) { h.entry_id[e] = id; });
            h.entry[t] = mine[0];
            if (mine[0] >= 0) atomicAnd(&h.off[mine[0] >> p.slot_shift][t / 32], ~(1u << (t % 32)));
            if (t == 0) h.entries = total;
            ptx::named_barrier(1, 128);
            if (t == 0) ptx::mbar_arrive(bar(h.plan));
        }
        if (rank == 0 && row0 % P == 0 && p.plan) {
            constexpr int WORDS = P / 32, ENTRY = 4 + WORDS;
            uint32_t *plan = p.plan + uint64_t(row0 / P) * plan_stride(P, p.adapters);
            int32_t ids[P / 128], mine[P / 128];
#pragma unroll
            for (int i = 0; i < P / 128; i++) ids[i] = read_id(row0 + t + 128 * i);
            const int count = distinct_ids<P>(ids, h.tile, t, mine, [&](int e, int id) { plan[4 + e * ENTRY] = uint32_t(id); });
            if (t == 0) plan[0] = uint32_t(count);
            for (int i = t; i < count * WORDS; i += 128) plan[4 + i / WORDS * ENTRY + 4 + i % WORDS] = 0xffffffffu;
            __threadfence();  // the words above are in place before another thread clears bits of them
            ptx::named_barrier(1, 128);
#pragma unroll
            for (int i = 0; i < P / 128; i++)
                if (mine[i] >= 0) atomicAnd(plan + 4 + mine[i] * ENTRY + 4 + (t + 128 * i) / 32, ~(1u << (t % 32)));
        }
        // Partial sums to shared memory: the rings are idle.
        const bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.done), 0, abort_flag, p.status, WHERE_EPILOGUE, 0u, limit));
        const int q = warp & 3;
        const uint32_t pitch = uint32_t(p.rp + 4) * 4u;
        if (ok) {
            ptx::tc_fence_after();
            ptx::fence_proxy_async_shared();
            // The slots that this warp's rows read, in pieces of 16 columns of one accumulator, eight of them on their way at
            // a time (one slot after another: 0.3 us each).
            const int entry = h.entry[32 * q + lane], own = entry >= 0 ? entry & ((1 << p.slot_shift) - 1) : -1;
            const uint32_t part_cols = uint32_t(p.slot_cols) << p.slot_shift, from = tmem + (uint32_t(32 * q) << 16);
            const uint32_t dst = xring + uint32_t(32 * q + lane) * pitch;
            uint32_t left = __reduce_or_sync(0xffffffffu, own >= 0 ? 1u << own : 0u);
            int slot = __ffs(int(left)) - 1, c = 0;
            while (slot >= 0) {
                uint32_t v[8][16];
                int slot_of[8], c_of[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    slot_of[i] = slot, c_of[i] = c;
                    if (slot < 0) continue;
                    ptx::tmem_ld_32x16(from + uint32_t(i & (p.parts - 1)) * part_cols + uint32_t(slot * p.slot_cols + c), v[i]);
                    if (((i + 1) & (p.parts - 1)) == 0 && (c += 16) == p.rp) {
                        c = 0;
                        left &= left - 1u;
                        slot = __ffs(int(left)) - 1;
                    }
                }
                ptx::tmem_ld_wait_all();
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (slot_of[i] >= 0) ptx::pin16(v[i]);
                auto add = [&](uint32_t (&to)[16], const uint32_t (&w)[16]) {
#pragma unroll
                    for (int k = 0; k < 16; k++) to[k] = __float_as_uint(__uint_as_float(to[k]) + __uint_as_float(w[k]));
                };
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    if (slot_of[i] < 0) continue;
                    if (p.parts == 2) {
                        add(v[i], v[i + 1]);
                        if (slot_of[i + 2] >= 0) add(v[i + 2], v[i + 3]);
                    } else if (p.parts == 4) {
                        add(v[i], v[i + 1]);
                        add(v[i], v[i + 2]);
                        add(v[i], v[i + 3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if ((i & (p.parts - 1)) == 0 && slot_of[i] >= 0 && slot_of[i] == own) {
#pragma unroll
                        for (int g = 0; g < 4; g++) ptx::st_shared_v4(dst + uint32_t(c_of[i]) * 4u + 16u * g, v[i][4 * g], v[i][4 * g + 1], v[i][4 * g + 2], v[i][4 * g + 3]);
                    }
                __syncwarp();
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
        const int shift = __ffs(quads) - 1;  // a power of two, as rp is
        cluster_sums<2>(
            min(BM, p.m - row0) * quads, int(rank), p.kc, SHRINK_THREADS,
            [&](int i) { return xring + uint32_t(i >> shift) * pitch + uint32_t(i & (quads - 1)) * 16u; },
            [&](int i, const float4 &v) {
                const int row = i >> shift, col = (i & (quads - 1)) * 4;
                // Rows without an adapter have nothing there, and past the rank may lie another adapter's sums.
                const float s = h.scale[row];
                const bool has = h.id[row] >= 0 && col < p.rank;
                const float4 w = has ? make_float4(v.x * s, v.y * s, v.z * s, v.w * s) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                store_t4(p.t + int64_t(row0 + row) * t_planes(p.bf16) * p.rp + col, p.rp, w, p.bf16);
            });
    }
    if (p.early) ptx::griddep_wait();
    __syncthreads();
    if (p.kc > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, T_COLS);
}

// ---- Y --------------------------------------------------------------------------
// The structure of the library's GEMM: persistent CTAs or CTA pairs, a TMA warp, an MMA warp, eight epilogue warps, a
// ring of 192 KiB.  G: CTAs per MMA; BN: columns per tile; MH: 128-row accumulators per CTA.  Behind a tile's k blocks
// of W come, for every adapter its rows name, the blocks of T (in place of X) and of B[a] (in place of W), their MMAs
// masked to the lanes of the adapter's rows.  One adapter of rank 64 costs 1 block (2 for
// an f32 result) beside the 64 of k = 4096.  A block of T serves all adapters of the tile: it
// keeps its stage until the last of them, and their blocks of B fill the rest of that stage and
// the others, as many as fit into each (a stage costs its issuing warps 0.3 us).
// On the way back B is A[a] as it lies, (rank, k): an MN-major operand, in boxes of 64 columns by up to 64 ranks.
// An f32 result of a long k is summed in `parts` accumulators (see T_PARTS), one set instead of two.
constexpr uint32_t RING_BYTES = 192 * 1024;
constexpr int TILE_THREADS = 64 + 256, TURN_PITCH = 33;  // words per row of a warp's piece of Y in shared memory, see store_32

template <int G, int BN, int MH>
struct Tile {
    static constexpr int CTA_ROWS = BM * MH, ROWS = CTA_ROWS * G, B_ROWS = BN / G;
    static constexpr uint32_t A_BYTES = CTA_ROWS * BK * 2, B_BYTES = B_ROWS * BK * 2, KB_BYTES = A_BYTES + B_BYTES;
    static constexpr int KPS = MH == 1 && BN == 128 ? 2 : 1;  // k blocks per stage: a 128 x 128 tile is short on math per block
    static constexpr uint32_t STAGE_BYTES = KPS * KB_BYTES;
    static constexpr int STAGES = int(RING_BYTES / STAGE_BYTES);
    static constexpr int ACC_COLS = MH * BN, ACC_BUFS = 2 * ACC_COLS <= 512 ? 2 : 1;
    static constexpr uint32_t TMEM_COLS = MH == 1 ? 512 : ACC_COLS * ACC_BUFS;
    static constexpr uint32_t SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 512 + 8 * 32 * TURN_PITCH * 4;
    static constexpr int CH = BN / 64;  // 32-column chunks of an accumulator per epilogue warp
    // Blocks of B in a stage that holds one or two blocks of T, and in one without.  Two of them, the values' two numbers,
    // where they fit: they are multiplied by the same block of B.
    static constexpr bool PAIRS = 2 * A_BYTES <= STAGE_BYTES;
    static constexpr int FIRST = int((STAGE_BYTES - A_BYTES) / B_BYTES), FIRST_PAIR = PAIRS ? int((STAGE_BYTES - 2 * A_BYTES) / B_BYTES) : 0;
    static constexpr int REST = int(STAGE_BYTES / B_BYTES);
    static constexpr int WORDS = ROWS / 32, BATCH = 32 / WORDS;  // mask words of an entry; entries whose words a warp reads at once
    static_assert(STAGES >= 3 && TMEM_COLS <= 512 && SMEM_BYTES <= 227 * 1024 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "tile");
};

struct TileParams {
    const uint32_t *plan;
    void *y;
    int64_t ldy;
    int m, n, rank, rp, adapters, c_dtype, vec;
    int k_blocks, m_tiles, n_tiles, group_m, parts;
    uint32_t idesc, low_idesc, low_box;  // low_box: bytes of an MN-major box of B, 0 = B is K-major
    bool bf16;
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

// A warp's 32 x 32 piece of Y from row row0 and column col on, a row per lane.  Lanes that hold whole aligned vectors store
// them as they are; others turn the piece through shared memory, so that a row is stored by neighbouring lanes (from a row
// per lane, stores of 4 bytes took 10 us of 777 x 2050 values in f32: each touches 32 sectors).
__device__ __forceinline__ void store_32(const TileParams &p, int row0, int col, const uint32_t (&v)[32], float *turn) {
    if (col >= p.n || row0 >= p.m) return;
    const int lane = int(threadIdx.x) & 31;
    if (p.vec && col + 32 <= p.n) {
        if (row0 + lane >= p.m) return;
        const int64_t at = int64_t(row0 + lane) * p.ldy + col;
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
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 32; j++) turn[lane * TURN_PITCH + j] = __uint_as_float(v[j]);
        __syncwarp();
        const int rows = min(32, p.m - row0);
        if (col + lane < p.n)
#pragma unroll 8
            for (int r = 0; r < rows; r++) store_c(p.y, p.c_dtype, size_t(int64_t(row0 + r) * p.ldy + col + lane), turn[r * TURN_PITCH + lane]);
        __syncwarp();
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
    const int bufs = p.parts > 1 ? 1 : C::ACC_BUFS;
    const bool whole = whole_t(p.c_dtype);
    const int t_blocks = C::PAIRS && whole && p.rp > 32 ? 2 : 1, q_blocks = ext_blocks(p.rp, whole);  // t_blocks: of T taken together
    const int first_blocks = t_blocks == 2 ? C::FIRST_PAIR : C::FIRST;

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
        }
        int s = 0, held = -1;  // held: the stage that keeps a block of T, passed over until its adapters are done
        uint32_t phases = 0, filled = 0, filled_parity = 0;  // phases: bit s = the parity of stage s's next use
        bool ok = !(p.debug & 4), waited = false;
        // Waits for the next stage and announces `bytes` per CTA.
        auto next = [&](uint32_t bytes) {
            if (s == held) s = s + 1 == C::STAGES ? 0 : s + 1;
            ok = __all_sync(0xffffffffu, wait_bar(empty_bar(s), ~(phases >> s) & 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(s), limit));
            if (ok && lane == 0 && rank == 0) ptx::mbar_arrive_expect_tx(full_bar(s), uint32_t(G) * bytes);
            __syncwarp();
            return ok;
        };
        auto issued = [&] {
            __syncwarp();
            filled |= 1u << s, filled_parity = (filled_parity & ~(1u << s)) | (phases & 1u << s);
            phases ^= 1u << s;
            if (++s == C::STAGES) s = 0;
        };
        auto load = [&](uint32_t dst, const CUtensorMap *map, int x, int y) {
            if constexpr (G == 1) ptx::tma_load_2d(dst, map, full_bar(s), x, y);
            else ptx::tma_load_2d_pair(dst, map, ptx::mapa(full_bar(s), 0), x, y);
        };
        const uint32_t low_bytes = p.low_box ? uint32_t(C::B_ROWS / 64) * p.low_box : C::B_BYTES;
        for (int t = first; t < tiles && ok; t += step) {
            const TileAt at = tile_at(t, p);
            const int row = at.tm * C::ROWS + int(rank) * C::CTA_ROWS, col = at.tn * BN + int(rank) * C::B_ROWS;
            const int kk = lane >> 1;  // lane 2 kk issues k block kk of X, lane 2 kk + 1 that of W
            const uint32_t *plan = p.plan + uint64_t(at.tm) * stride;
            // Lane l holds the id of entry l, 32 of them at a time, on their way while the tile's blocks of W are issued.
            int entries = 0, ids = 0;
            auto read_ids = [&](int e0) { ids = e0 + lane < entries ? int(plan[4 + (e0 + lane) * ENTRY]) : 0; };
            auto read_plan = [&] {
                entries = int(plan[0]);
                read_ids(0);
            };
            if (waited) read_plan();
            for (int kb = 0; kb < p.k_blocks && ok; kb += C::KPS) {
                const int nk = min(C::KPS, p.k_blocks - kb);
                if (!next(uint32_t(nk) * C::KB_BYTES)) break;
                const uint32_t dst = ring + uint32_t(s) * C::STAGE_BYTES + uint32_t(kk) * C::KB_BYTES;
                if (kk < nk) load(dst + (lane & 1 ? C::A_BYTES : 0u), lane & 1 ? &tmW : &tmX, (kb + kk) * BK, lane & 1 ? col : row);
                issued();
            }
            if (!ok) break;
            if (!waited) {
                ptx::griddep_wait();  // T and the plan; X and W are older than their kernel
                waited = true;
                read_plan();
            }
            const int boxes = p.low_box ? C::B_ROWS / 64 : 1;  // of B per adapter
            for (int q = 0; q < q_blocks && entries > 0 && ok; q += t_blocks) {
                const ExtBlock b = ext_block(q, p.rp, p.rank, whole, p.bf16);
                if (q > 0 && entries > 32) read_ids(0);
                bool head = true;  // this stage begins with T
                for (int e = 0; e < entries && ok; head = false) {
                    if (e > 0 && e % 32 == 0) read_ids(e);
                    // Entries of one stage, all of one reading of the ids.
                    const int count = min(min(head ? first_blocks : C::REST, entries - e), 32 - e % 32);
                    const int item = head ? lane - t_blocks : lane, mine = item / boxes, box = item % boxes;  // the first lanes issue T
                    const int id = __shfl_sync(0xffffffffu, ids, (e + mine) & 31);
                    const uint32_t t_bytes = head ? uint32_t(t_blocks) * C::A_BYTES : 0u;
                    if (!next(t_bytes + uint32_t(count) * low_bytes)) break;
                    const uint32_t dst = ring + uint32_t(s) * C::STAGE_BYTES, low = dst + t_bytes + uint32_t(mine) * C::B_BYTES;
                    if (head && lane < t_blocks) load(dst + uint32_t(lane) * C::A_BYTES, &tmT, b.t_col + lane * p.rp, row);
                    if (item >= 0 && mine < count) {
                        if (p.low_box == 0) {
                            load(low, &tmB, b.b_col, id * p.n + col);
                        } else {
                            const uint32_t to = low + uint32_t(box) * p.low_box;
                            if constexpr (G == 1) ptx::tma_load_3d(to, &tmB, full_bar(s), col + 64 * box, b.b_col, id);
                            else ptx::tma_load_3d_pair(to, &tmB, ptx::mapa(full_bar(s), 0), col + 64 * box, b.b_col, id);
                        }
                    }
                    if (head) held = s;
                    issued();
                    e += count;
                }
                held = -1;
            }
        }
        if (!ok && rank == 0 && lane == 0) {  // giving up: let the copies in flight land (bounded)
            const uint64_t t0 = ptx::globaltimer_ns();
            for (int i = 0; i < C::STAGES; i++)
                while ((filled >> i & 1u) && !ptx::mbar_try_wait(full_bar(i), (filled_parity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        if (!waited) ptx::griddep_wait();
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            // The whole warp runs the loop and one thread issues: see lora_few_kernel.
            const bool leader = ptx::elect_one();
            int s = 0, it = 0, held = -1;
            uint32_t phases = 0;
            bool ok = true, issued = false, waited = false;
            auto ready = [&] {
                if (s == held) s = s + 1 == C::STAGES ? 0 : s + 1;
                ok = __all_sync(0xffffffffu, wait_bar(full_bar(s), phases >> s & 1u, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(s), limit));
                ptx::tc_fence_after();
                return ok;
            };
            auto release = [&](int stage) {
                if (leader) {
                    ptx::umma_commit<G>(empty_bar(stage));
                    if constexpr (G == 2) ptx::umma_commit<G>(ptx::mapa(empty_bar(stage), 1));
                }
                __syncwarp();
            };
            auto advance = [&] {
                issued = true;
                phases ^= 1u << s;
                if (++s == C::STAGES) s = 0;
            };
            for (int t = first; t < tiles && ok; t += step, it++) {
                const TileAt at = tile_at(t, p);
                const int buf = it % bufs;
                const uint32_t aph = uint32_t(it / bufs) & 1u, d0 = tmem + uint32_t(buf * C::ACC_COLS);
                uint32_t d = d0;
                int part = 0, part_end = (p.k_blocks + p.parts - 1) / p.parts;  // the k block the next accumulator begins at
                const uint32_t *plan = p.plan + uint64_t(at.tm) * stride;
                // Lane l holds word l % WORDS of the masks of entry l / WORDS of a batch, read one batch ahead.
                int entries = 0;
                uint32_t ahead = 0;
                auto read_off = [&](int e0) {
                    const int e = e0 + lane / C::WORDS;
                    ahead = e < entries ? plan[4 + e * ENTRY + 4 + lane % C::WORDS] : 0u;
                };
                auto read_plan = [&] {
                    entries = int(plan[0]);
                    read_off(0);
                };
                if (waited) read_plan();
                for (int k0 = 0; k0 < p.k_blocks; k0 += C::KPS) {
                    if (!ready()) break;
                    const uint32_t stage = ring + uint32_t(s) * C::STAGE_BYTES;
#pragma unroll
                    for (int kk = 0; kk < C::KPS; kk++) {
                        if (k0 + kk >= p.k_blocks) break;
                        bool fresh = k0 == 0 && kk == 0;
                        if (k0 + kk == part_end && part + 1 < p.parts) {
                            part++;
                            part_end = (p.k_blocks * (part + 1) + p.parts - 1) / p.parts;
                            d = d0 + uint32_t(part * C::ACC_COLS);
                            fresh = true;
                        }
                        const uint32_t src = stage + kk * C::KB_BYTES;
                        const uint64_t b = sw128_desc(src + C::A_BYTES);
#pragma unroll
                        for (int h = 0; h < MH; h++) {
                            if (fresh && part == 0) {  // the epilogue must have drained this half of the buffer
                                ok = __all_sync(0xffffffffu, wait_bar(tempty_bar(buf, h), aph ^ 1u, abort_flag, p.status, WHERE_MMA_TMEM, uint32_t(buf * 2 + h), limit));
                                if (!ok) break;
                                ptx::tc_fence_after();
                            }
                            const uint64_t a = sw128_desc(src + uint32_t(h) * (BM * BK * 2));
                            if (leader) {
#pragma unroll
                                for (int j = 0; j < 4; j++) ptx::umma_f16<G>(d + uint32_t(h * BN), a + 2u * j, b + 2u * j, p.idesc, (!fresh || j > 0) ? 1u : 0u);
                            }
                            __syncwarp();
                            issued = true;
                        }
                        if (!ok) break;
                    }
                    if (!ok) break;
                    release(s);
                    advance();
                }
                if (!ok) break;
                if (!waited) {
                    ptx::griddep_wait();
                    waited = true;
                    read_plan();
                }
                const uint32_t k_step = p.low_box ? MN_K_STEP : 2u;
                for (int q = 0; q < q_blocks && entries > 0 && ok; q += t_blocks) {
                    const ExtBlock x = ext_block(q, p.rp, p.rank, whole, p.bf16);
                    uint32_t words = 0, t_block = 0, b_block = 0;
                    uint32_t step[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) step[j] = k_step * uint32_t(j & x.b_mask);
                    int first_stage = 0, left = 0;  // left: entries of this stage still to come
                    bool head = false;              // this stage holds T
                    if (q > 0 && entries > C::BATCH) read_off(0);
                    for (int e = 0; e < entries; e++) {
                        if (e % C::BATCH == 0) {
                            words = ahead;
                            if (entries > C::BATCH) read_off(e + C::BATCH);
                        }
                        if (e == 0) {
                            if (!ready()) break;
                            first_stage = s, t_block = ring + uint32_t(s) * C::STAGE_BYTES, b_block = t_block + uint32_t(t_blocks) * C::A_BYTES;
                            left = min(min(first_blocks, entries), 32);
                            head = true;
                            if (left == 0) {
                                held = s, head = false;
                                advance();
                            }
                        }
                        if (left == 0) {
                            if (!ready()) break;
                            left = min(min(C::REST, entries - e), 32 - e % 32);
                            b_block = ring + uint32_t(s) * C::STAGE_BYTES;
                        }
                        const uint64_t b = p.low_box ? mn_desc(b_block, p.low_box) : sw128_desc(b_block);
#pragma unroll
                        for (int h = 0; h < MH; h++) {
                            const uint64_t a = sw128_desc(t_block + uint32_t(h) * (BM * BK * 2));
                            uint32_t m[4 * G], all = 0xffffffffu;
#pragma unroll
                            for (int i = 0; i < 4 * G; i++) {
                                m[i] = __shfl_sync(0xffffffffu, words, e % C::BATCH * C::WORDS + (i / 4) * (C::CTA_ROWS / 32) + 4 * h + i % 4);
                                all &= m[i];
                            }
                            if (leader && all != 0xffffffffu) {  // else no row of these accumulators
                                auto multiply = [&](uint64_t from) {
#pragma unroll
                                    for (int j = 0; j < 4; j++) {
                                        if (j >= x.steps) continue;
                                        const uint64_t bj = b + uint64_t(step[j]);
                                        if constexpr (G == 1) ptx::umma_f16_lanes(d0 + uint32_t(h * BN), from + 2u * j, bj, p.low_idesc, 1u, m[0], m[1], m[2], m[3]);
                                        else ptx::umma_f16_lanes_pair(d0 + uint32_t(h * BN), from + 2u * j, bj, p.low_idesc, 1u, m);
                                    }
                                };
                                multiply(a);
                                if (t_blocks == 2) multiply(a + (C::A_BYTES >> 4));
                            }
                            __syncwarp();
                        }
                        b_block += C::B_BYTES;
                        if (--left == 0) {  // T's stage is kept until the last entry
                            if (head) held = s, head = false;
                            else release(s);
                            advance();
                        }
                    }
                    if (!ok) break;
                    release(first_stage);
                    held = -1;
                }
                if (!ok) break;
                if (leader) {
                    ptx::umma_commit<G>(tfull_bar(buf));
                    if constexpr (G == 2) ptx::umma_commit<G>(ptx::mapa(tfull_bar(buf), 1));
                }
                __syncwarp();
            }
            if (!ok && issued && leader) {
                ptx::umma_commit<G>(drain_bar);
                const uint64_t t0 = ptx::globaltimer_ns();
                while (!ptx::mbar_try_wait(drain_bar, 0u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            }
        }
        __syncwarp();
    } else {
        const uint32_t q = uint32_t(warp) & 3u;
        float *turn = reinterpret_cast<float *>(smem_raw + (bars - raw) + 512) + (warp - 2) * 32 * TURN_PITCH;
        const int e = (warp - 2) >> 2;  // of two groups of four warps, each takes every other 32-column chunk
        int it = 0;
        for (int t = first; t < tiles; t += step, it++) {
            const TileAt at = tile_at(t, p);
            const int buf = it % bufs;
            const bool ok = wait_bar(tfull_bar(buf), uint32_t(it / bufs) & 1u, abort_flag, p.status, WHERE_EPILOGUE, uint32_t(buf), limit);
            if (!__all_sync(0xffffffffu, ok)) break;
            ptx::tc_fence_after();
            const int row0 = at.tm * C::ROWS + int(rank) * C::CTA_ROWS + int(q) * 32;
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
                if constexpr (MH == 1)
                    for (int i = 1; i < p.parts; i++) {
#pragma unroll
                        for (int c = 0; c < C::CH; c++) {
                            uint32_t o[32];
                            ptx::tmem_ld_32x32(taddr + uint32_t(i * C::ACC_COLS + (2 * c + e) * 32), o);
                            ptx::tmem_ld_wait(o);
#pragma unroll
                            for (int j = 0; j < 32; j++) v[c][j] = __float_as_uint(__uint_as_float(v[c][j]) + __uint_as_float(o[j]));
                        }
                    }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (G == 1) ptx::mbar_arrive(tempty_bar(buf, h));
                    else ptx::mbar_arrive_cluster(ptx::mapa(tempty_bar(buf, h), 0));
                }
#pragma unroll
                for (int c = 0; c < C::CH; c++) store_32(p, row0 + h * BM, at.tn * BN + (2 * c + e) * 32, v[c], turn);
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
template <int P>
cute_b200_status shrink(const LoraParams &p, int product_ctas, bool bf16, int debug, const DeviceState &dev, cudaStream_t stream) {
    ShrinkParams s = {};
    s.ids = p.ids, s.scale = p.scale, s.t = p.t, s.plan = p.y ? p.plan : nullptr;
    s.m = p.m, s.rank = p.rank, s.rp = p.rp, s.adapters = p.adapters;
    s.k_blocks = (p.k + BK - 1) / BK;
    s.mn = s.early = p.low_mn;
    s.boxes = p.low_mn ? (p.rp + 63) / 64 : 1;
    s.box_bytes = p.low_mn ? BK * 128 : uint32_t(p.rp) * 128u;
    // A stage of A holds the blocks of two k blocks of one adapter, or 16 KB of them.
    s.a_bytes = 2 * uint32_t(s.boxes) * s.box_bytes;
    if (s.a_bytes < 16 * 1024) s.a_bytes = 16 * 1024;
    s.x_stages = s.a_bytes > 16 * 1024 ? 3 : 4;
    s.a_stages = int((SHRINK_RINGS - uint32_t(s.x_stages * X_BLOCKS) * X_BYTES) / s.a_bytes);
    if (s.a_stages > MAX_A_STAGES) s.a_stages = MAX_A_STAGES;
    s.bf16 = bf16;
    s.idesc = make_idesc(bf16, 128, 0) | (p.low_mn ? IDESC_B_MN : 0u);
    s.status = dev.status_word;
    s.debug = debug;
    const int tiles = (p.m + BM - 1) / BM;
    // k is cut while that puts more CTAs to work and leaves each at least two blocks.
    s.kc = 1;
    for (int c = 1; c < 4; c++)
        if (tiles <= dev.shrink_clusters[c] && s.k_blocks >= (2 << c)) s.kc = 1 << c;
    // Where the product's CTAs (an SM each, like these) leave SMs free, T's kernel keeps to those, so that the product's k loop
    // over W runs beside it; unless that takes longer than both one after the other, at 0.25 us per k block of the product
    // and, per k block of T, 0.2 us and 0.25 per 128 rows of A.
    const int free = dev.sm_count - product_ctas, entries = p.adapters < BM ? p.adapters : BM;
    if (p.y && free >= tiles && tiles * s.kc > free) {
        int kc = s.kc;
        while (tiles * kc > free) kc /= 2;
        const double block = 0.2 + 0.25 * entries * p.rp / 128.0;
        if (block * s.k_blocks / kc <= block * s.k_blocks / s.kc + 0.25 * s.k_blocks) s.kc = kc;
    }
    // At most 8 k blocks (32 MMAs of 16) per accumulator where one or two are enough: fewer of them have more slots.
    const int blocks = (s.k_blocks + s.kc - 1) / s.kc;
    s.parts = blocks <= 8 ? 1 : (blocks <= 16 ? 2 : T_PARTS);
    s.slot_cols = p.low_mn ? 64 * s.boxes : p.rp;
    while ((s.slot_cols << (s.slot_shift + 1)) * s.parts <= T_COLS) s.slot_shift++;
    CUtensorMap tmX, tmA;
    CB_TRY(rows_tensor_map(&tmX, reinterpret_cast<uint64_t>(p.x), bf16, p.m, p.k, p.ldx, BM));
    if (p.low_mn) CB_TRY(stack_tensor_map(&tmA, reinterpret_cast<uint64_t>(p.a), bf16, p.adapters, p.k, p.rank, BK));
    else CB_TRY(rows_tensor_map(&tmA, reinterpret_cast<uint64_t>(p.a), bf16, uint64_t(p.adapters) * p.rank, p.k, p.k, p.rp));
    return launch_dependent(shrink_tile_kernel<P>, dim3(unsigned(tiles * s.kc)), SHRINK_THREADS, SHRINK_SMEM, s.kc, stream, tmX, tmA, s);
}

// Accumulators an f32 result of this k asks for: 4096 of k in one cost 5e-6 of the sum.
int result_parts(int k, int c_dtype) { return c_dtype != CUTE_B200_F32 || k <= 4096 ? 1 : (k <= 8192 ? 2 : 4); }

template <int G, int BN, int MH>
cute_b200_status launch_tile(const LoraParams &p, bool bf16, int debug, const DeviceState &dev, cudaStream_t stream) {
    using C = Tile<G, BN, MH>;
    TileParams t = {};
    t.plan = p.plan, t.y = p.y, t.ldy = p.ldy;
    t.m = p.m, t.n = p.n, t.rank = p.rank, t.rp = p.rp, t.adapters = p.adapters, t.c_dtype = p.c_dtype;
    const uint64_t esize = p.c_dtype == CUTE_B200_F32 ? 4 : 2, y = reinterpret_cast<uint64_t>(p.y);
    t.vec = y % 32 == 0 && uint64_t(p.ldy) * esize % 32 == 0 ? 2 : (y % 16 == 0 && uint64_t(p.ldy) * esize % 16 == 0 ? 1 : 0);
    t.k_blocks = (p.k + BK - 1) / BK;
    t.parts = result_parts(p.k, p.c_dtype);
    if (t.parts > 512 / C::ACC_COLS) t.parts = 512 / C::ACC_COLS;
    t.m_tiles = (p.m + C::ROWS - 1) / C::ROWS;
    t.n_tiles = (p.n + BN - 1) / BN;
    const int64_t tiles = int64_t(t.m_tiles) * t.n_tiles;
    if (tiles > (1 << 30)) return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "lora_tn: %d x %d is more than 2^30 tiles", p.m, p.n);
    int clusters = dev.sm_count / G;
    if (tiles < clusters) clusters = int(tiles);
    // With a tile per CTA there is no second buffer to keep free: an f32 result takes all accumulators (777 x 2050, k = 1032:
    // relative error 4e-7 in 27.6 us, 1.3e-6 in 27.1 from one).
    if (p.c_dtype == CUTE_B200_F32 && tiles <= dev.sm_count / G && MH == 1)
        while (t.parts * 2 * C::ACC_COLS <= 512 && t.parts * 2 <= t.k_blocks) t.parts *= 2;
    int gm = 1;
    while (gm * gm * 2 <= clusters) gm *= 2;
    t.group_m = gm < t.m_tiles ? gm : t.m_tiles;
    t.idesc = make_idesc(bf16, 128 * G, BN);
    const int low_rows = p.rp < 64 ? p.rp : 64;  // ranks per box of an MN-major B
    t.low_idesc = t.idesc | (p.low_mn ? IDESC_B_MN : 0u);
    t.low_box = p.low_mn ? uint32_t(low_rows) * 128u : 0u;
    t.bf16 = bf16;
    t.status = dev.status_word;
    t.debug = debug;
    CUtensorMap tmX, tmW, tmT, tmB;
    CB_TRY(rows_tensor_map(&tmX, reinterpret_cast<uint64_t>(p.x), bf16, p.m, p.k, p.ldx, C::CTA_ROWS));
    CB_TRY(rows_tensor_map(&tmW, reinterpret_cast<uint64_t>(p.w), bf16, p.n, p.k, p.k, C::B_ROWS));
    CB_TRY(rows_tensor_map(&tmT, reinterpret_cast<uint64_t>(p.t), bf16, p.m, t_planes(bf16) * p.rp, t_planes(bf16) * p.rp, C::CTA_ROWS));
    if (p.low_mn) CB_TRY(stack_tensor_map(&tmB, reinterpret_cast<uint64_t>(p.b), bf16, p.adapters, p.rank, p.n, low_rows));
    else CB_TRY(rows_tensor_map(&tmB, reinterpret_cast<uint64_t>(p.b), bf16, uint64_t(p.adapters) * p.n, p.rank, p.rank, C::B_ROWS));
    return launch_dependent(lora_tile_kernel<G, BN, MH>, dim3(unsigned(clusters * G)), TILE_THREADS, C::SMEM_BYTES, G, stream, tmX, tmW, tmT, tmB, t);
}

// Rows of the GEMM's tile, and its columns: whole waves of tiles, each its MMA time at the rate this tiling was measured at
// beside the 512 x 256 pair tile (1.0) plus the time to fill the ring and drain the accumulator.
struct Cut {
    int rows, cols;
    double rate;
};
constexpr int NUM_CUTS = 4;
constexpr Cut CUTS[NUM_CUTS] = {{512, 256, 1.0}, {256, 256, 0.92}, {128, 256, 0.86}, {128, 128, 0.7}};
int choose_cut(int m, int n, int k, int c_dtype, int sm_count) {
    int best = 0;
    double best_t = 1e300;
    for (int i = 0; i < NUM_CUTS; i++) {
        if (result_parts(k, c_dtype) * CUTS[i].cols * (CUTS[i].rows == 512 ? 2 : 1) > 512) continue;
        const int pair = CUTS[i].rows >= 256 ? 2 : 1;
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
    for (int rows : {128, 256, 512}) {
        const uint64_t b = uint64_t((int64_t(m) + rows - 1) / rows) * plan_stride(rows, adapters) * 4;
        if (b > most) most = b;
    }
    return most;
}

cute_b200_status lora_tiled(const LoraParams &p, bool bf16, int cut, int debug, const DeviceState &dev, cudaStream_t stream) {
    if (cut < 0) cut = choose_cut(p.m, p.n, p.k, p.c_dtype, dev.sm_count);
    const int64_t tiles = int64_t((p.m + CUTS[cut].rows - 1) / CUTS[cut].rows) * ((p.n + CUTS[cut].cols - 1) / CUTS[cut].cols);
    const int pair = CUTS[cut].rows >= 256 ? 2 : 1, ctas = tiles * pair < dev.sm_count ? int(tiles) * pair : dev.sm_count;
    if (CUTS[cut].rows == 512) CB_TRY(shrink<512>(p, ctas, bf16, debug, dev, stream));
    else if (CUTS[cut].rows == 256) CB_TRY(shrink<256>(p, ctas, bf16, debug, dev, stream));
    else CB_TRY(shrink<128>(p, ctas, bf16, debug, dev, stream));
    if (!p.y) return CUTE_B200_OK;
    if (cut == 0) return launch_tile<2, 256, 2>(p, bf16, debug, dev, stream);
    if (cut == 1) return launch_tile<2, 256, 1>(p, bf16, debug, dev, stream);
    if (cut == 2) return launch_tile<1, 256, 1>(p, bf16, debug, dev, stream);
    return launch_tile<1, 128, 1>(p, bf16, debug, dev, stream);
}

cute_b200_status lora_tiled_init(DeviceState &dev) {
    CB_CUDA(cudaFuncSetAttribute(shrink_tile_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, SHRINK_SMEM));
    CB_CUDA(cudaFuncSetAttribute(shrink_tile_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, SHRINK_SMEM));
    CB_CUDA(cudaFuncSetAttribute(shrink_tile_kernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize, SHRINK_SMEM));
    CB_CUDA(cudaFuncSetAttribute(lora_tile_kernel<2, 256, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<2, 256, 2>::SMEM_BYTES));
    CB_CUDA(cudaFuncSetAttribute(lora_tile_kernel<2, 256, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<2, 256, 1>::SMEM_BYTES));
    CB_CUDA(cudaFuncSetAttribute(lora_tile_kernel<1, 256, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<1, 256, 1>::SMEM_BYTES));
    CB_CUDA(cudaFuncSetAttribute(lora_tile_kernel<1, 128, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<1, 128, 1>::SMEM_BYTES));
    for (int c = 0; c < 4; c++)
        CB_TRY(max_clusters(shrink_tile_kernel<128>, SHRINK_THREADS, SHRINK_SMEM, 1 << c, &dev.shrink_clusters[c]));
    return CUTE_B200_OK;
}

}  // namespace cb
