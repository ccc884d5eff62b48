// A projection shared by all rows with a low-rank adapter chosen row by row:
//     y[i] = W x[i] + scale[a] * B[a] (A[a] x[i]),   a = ids[i]
// and its gradients.  The inner product T[i] = scale[a] * A[a] x[i] (`rank`
// values per row) goes to the workspace as 16-bit numbers whose sum is the
// value (store_t): the second product can then run on 16-bit operands and still
// carry 16 (bf16) or 22 (f16, but no finer than 2^-25) bits of T.
#include "lora_sm100.cuh"

namespace cb {
namespace {

// ---- few rows (m <= 128) ------------------------------------------------------
// T: a CTA takes J of an adapter's `rank` rows and up to four rows of X that name it; its 256 threads walk k in 16-byte pieces.
// Of the rows that share an adapter every fourth brings its CTA to work, on itself and the next three; the others return.
// Both operands come from L2 but for the first time (100 rows of 4 adapters, rank 128, k = 8192: 90 MB; a CTA per row and
// four ranks read 256 MB).  It is over before the weights have streamed past (below).
constexpr int FEW_ROWS = 128, SHRINK_THREADS = 256, SHRINK_ROWS = 4;

template <bool BF16, int J>
__global__ void __launch_bounds__(SHRINK_THREADS) shrink_rows_kernel(const LoraParams p) {
    __shared__ float part[SHRINK_THREADS / 32][SHRINK_ROWS * J];
    __shared__ int rows[SHRINK_ROWS], counts[4], before;
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int j0 = blockIdx.y * J, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int id = p.ids[blockIdx.x];
    if (id < 0 || id >= p.adapters) return;
    // Place of every row among those that share this adapter; `first` is this CTA's.
    const bool same = tid < p.m && p.ids[tid] == id;
    const uint32_t votes = __ballot_sync(0xffffffffu, same);
    if (warp < 4 && lane == 0) counts[warp] = __popc(votes);
    if (tid < SHRINK_ROWS) rows[tid] = blockIdx.x;  // a batch of fewer rows takes this one once more
    __syncthreads();
    int at = __popc(votes & ((1u << lane) - 1u)), count = 0;
    for (int i = 0; i < 4; i++) {
        if (i < warp) at += counts[i];
        count += counts[i];
    }
    if (tid == int(blockIdx.x)) before = at;
    __syncthreads();
    const int first = before;
    if (first % SHRINK_ROWS) return;
    if (same && at >= first && at < first + SHRINK_ROWS) rows[at - first] = tid;
    __syncthreads();
    const bool live = j0 < p.rank;  // else the padding of the rank: zeros
    const float scale = p.scale[id];
    const uint16_t *a = p.a + (int64_t(id) * p.rank + j0) * p.k;
    const int vecs = live ? p.k / 8 : 0, batch = min(SHRINK_ROWS, count - first);
    const uint16_t *x[SHRINK_ROWS];
#pragma unroll
    for (int r = 0; r < SHRINK_ROWS; r++) x[r] = p.x + rows[r] * p.ldx;
    float acc[SHRINK_ROWS][J] = {};
#pragma unroll 1
    for (int c = tid; c < vecs; c += SHRINK_THREADS) {
        uint4 av[J], xv[SHRINK_ROWS];
#pragma unroll
        for (int j = 0; j < J; j++) av[j] = __ldg(reinterpret_cast<const uint4 *>(a + int64_t(j) * p.k + 8 * c));
#pragma unroll
        for (int r = 0; r < SHRINK_ROWS; r++) xv[r] = *reinterpret_cast<const uint4 *>(x[r] + 8 * c);  // no branch between the loads
#pragma unroll
        for (int r = 0; r < SHRINK_ROWS; r++) {
            if (r > 0 && batch == 1) break;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 xf = pair_f32<BF16>(i == 0 ? xv[r].x : (i == 1 ? xv[r].y : (i == 2 ? xv[r].z : xv[r].w)));
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const float2 af = pair_f32<BF16>(i == 0 ? av[j].x : (i == 1 ? av[j].y : (i == 2 ? av[j].z : av[j].w)));
                    acc[r][j] = fmaf(af.y, xf.y, fmaf(af.x, xf.x, acc[r][j]));
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < SHRINK_ROWS; r++) {
        if (r > 0 && batch == 1) break;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const float sum = warp_sum(acc[r][j]);
            if (lane == 0) part[warp][r * J + j] = sum;
        }
    }
    __syncthreads();
    if (tid < batch * J) {
        float sum = 0.0f;
        for (int w = 0; w < SHRINK_THREADS / 32; w++) sum += part[w][tid];
        sum = live ? sum * scale : 0.0f;
        store_t<BF16>(p.t + int64_t(rows[tid / J]) * t_planes(BF16) * p.rp + j0 + tid % J, p.rp, sum);
    }
}

// Y: the weight streams past the rows.  The (up to 128) rows of X are the M = 128
// lanes of one accumulator, `bn` rows of W its columns; a cluster of `kc` CTAs
// shares a tile's k blocks and, after them, the adapters its rows name, and adds
// its partial sums through shared memory.  Bound by HBM: every byte of W is
// read once, the ring keeps ~190 KB of it in flight per SM.
//   warp 0  TMA: per stage `kps` k blocks, each (xr x 64) of X and (bn x 64) of W;
//           then T, once, and per adapter blocks of B[a].  A stage costs the
//           issuing warp about 0.3 us whatever it holds (measured: 32 x 64 blocks, one per
//           stage, stream at 1.9 TB/s, four per stage at 4.4 when lanes issue side by side),
//           so a stage is made to hold 10 to 40 KB of W (stream_blocks) and every block is another lane's.
//   warp 1  MMA: M 128, N bn.  The MMA always reads 128 rows of X; those past
//           the loaded xr rows are whatever lies behind them in shared memory (in
//           bounds, see forward_few), and end up in lanes that nothing reads.  An
//           adapter's product is masked to the lanes of the rows that name it,
//           so that nothing of it reaches another row.
//   warps 2-5  which adapters the rows name, while the weights stream; then
//           the accumulator's rows to shared memory, the sum over the cluster
//           and the stores.
// W and X do not depend on the kernel that computes T, which has waited for all
// before it: they are loaded before griddepcontrol.wait, T and the ids after.
constexpr int FEW_THREADS = 192, FEW_MAX_STAGES = 16;
constexpr uint32_t FEW_HEAD = 8192;  // barriers, masks and ids, ahead of the ring

struct FewParams {
    const int32_t *ids;
    void *y;
    int64_t ldy;
    int m, n, rank, rp, adapters, c_dtype, vec;
    int k_blocks, bn, kc, xr, stages, kps, b_blocks, parts;  // parts: accumulators the k range goes to in turn
    uint32_t stage_bytes, x_bytes, w_bytes, low_bytes, idesc, tmem_cols;
    const uint16_t *t, *b;
    bool bf16;
    uint32_t *status;
    int debug;
};

struct FewHead {
    uint64_t full[FEW_MAX_STAGES], empty[FEW_MAX_STAGES], low, plan, done, drain;
    uint32_t tmem, abort;
    int32_t entries, entry_id[FEW_ROWS];
    uint32_t off[FEW_ROWS][4];  // lanes of entry e that keep their sums: bit set = not a row of this adapter
    int32_t id[FEW_ROWS];
    IdTable<FEW_ROWS> table;
};
static_assert(sizeof(FewHead) <= FEW_HEAD, "head");

// Where the adapters' products are taken.  On the tensor core, through the ring, in blocks of 64 columns of B[a]
// (b_blocks > 0); or, b_blocks == 0, as dot products by the epilogue's 128 threads, idle while W streams, a thread per column
// of Y, into `low` in f32, which the final sum adds.  The second way serves ranks up to 32, whose rows of B[a] are 16 to
// 64 bytes: TMA fetches those no faster than full rows of 128 (0.5 us for a box of 128 rows, measured; 48 rows with an
// adapter each, rank 16, n = 8192: 35 us by the tensor core).  Its results must leave the ring most of shared memory.
constexpr uint32_t FEW_DOTS = 40 * 1024;
// Blocks of B that this CTA of the cluster takes: every kc-th adapter.
__device__ __forceinline__ int low_blocks(int entries, int rank, int kc, int b_blocks) {
    return b_blocks > 0 && entries > rank ? (entries - rank + kc - 1) / kc * b_blocks : 0;
}

// The adapters' part of columns n0.. of Y for rows rank, rank + kc, .. (row r of `t` and `out` is row rank + r kc of Y), by
// 128 threads; id[row] < 0 = no adapter.  V: 16-byte pieces of a row of B; R: rows of a batch, whose B is fetched at once.
// Of ranks up to 16 two batches are on their way (one row at a time took 0.7 us each, the latency of its loads; a batch at a
// time, behind W's stream, 2.5), the first two while T is still being computed: 48 rows of 64 adapters, 8192 x 4096, rank 16:
// 21.2 us, 22.1 a batch at a time; of higher ranks their traffic holds T up (16 rows, rank 32, 11008 x 4096: 25.4 us, 22.7 a batch at
// a time).
template <bool BF16, int V, int R, int AHEAD>
__device__ __forceinline__ void few_dots(const FewParams &p, const int32_t *id, float *t, float *out, int rank, int n0, int thread) {
    const int rows = (p.m - rank + p.kc - 1) / p.kc, cols = min(p.bn, p.n - n0), groups = (rows + R - 1) / R, batches = groups * ((cols + 127) / 128);
    uint4 b[AHEAD][R][V];
    auto load = [&](int q, uint4 (&to)[R][V]) {
        const int pass = q / groups, r0 = (q - pass * groups) * R, c = 128 * pass + thread;
        if (c >= cols) return;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int a = r0 + r < rows ? id[rank + (r0 + r) * p.kc] : -1;
            const uint4 *src = reinterpret_cast<const uint4 *>(p.b + (int64_t(a) * p.n + n0 + c) * p.rank);
#pragma unroll
            for (int v = 0; v < V; v++) to[r][v] = a >= 0 ? __ldg(src + v) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    auto multiply = [&](int q, const uint4 (&from)[R][V]) {
        const int pass = q / groups, r0 = (q - pass * groups) * R, c = 128 * pass + thread;
        if (c >= cols) return;
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (r0 + r >= rows) break;
            const float *tv = t + (r0 + r) * p.rp;  // zeros where the row has no adapter
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < V; v++) {
                const uint32_t w[4] = {from[r][v].x, from[r][v].y, from[r][v].z, from[r][v].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = pair_f32<BF16>(w[i]);
                    sum = fmaf(f.y, tv[8 * v + 2 * i + 1], fmaf(f.x, tv[8 * v + 2 * i], sum));
                }
            }
            out[(r0 + r) * p.bn + c] = sum;
        }
    };
    if (AHEAD == 2 && batches > 0) load(0, b[0]);
    if (AHEAD == 2 && batches > 1) load(1, b[1]);
    ptx::griddep_wait();
    for (int i = thread; i < rows * p.rp; i += 128) {
        const int r = i / p.rp, j = i - r * p.rp;
        const uint16_t *src = p.t + int64_t(rank + r * p.kc) * t_planes(BF16) * p.rp + j;
        t[i] = id[rank + r * p.kc] >= 0 ? to_f32<BF16>(src[0]) + to_f32<BF16>(src[p.rp]) : 0.0f;
    }
    ptx::named_barrier(1, 128);
    for (int q = 0; q < batches; q += AHEAD) {
        if constexpr (AHEAD == 1) load(q, b[0]);
        multiply(q, b[0]);
        if constexpr (AHEAD == 2) {
            if (q + 2 < batches) load(q + 2, b[0]);
            if (q + 1 < batches) multiply(q + 1, b[1]);
            if (q + 3 < batches) load(q + 3, b[1]);
        }
    }
}

template <bool BF16>
__device__ __forceinline__ void few_dots(const FewParams &p, const int32_t *id, float *t, float *out, int rank, int n0, int thread) {
    if (p.rank == 8) few_dots<BF16, 1, 8, 2>(p, id, t, out, rank, n0, thread);
    else if (p.rank == 16) few_dots<BF16, 2, 8, 2>(p, id, t, out, rank, n0, thread);
    else if (p.rank == 24) few_dots<BF16, 3, 4, 1>(p, id, t, out, rank, n0, thread);
    else few_dots<BF16, 4, 4, 1>(p, id, t, out, rank, n0, thread);
}

// 168 registers at most (what two CTAs per SM would allow; shared memory holds one), so that a CTA fits beside one of T's kernel.
__global__ void __launch_bounds__(FEW_THREADS, 2)
    lora_few_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmT,
                    const __grid_constant__ CUtensorMap tmB, const FewParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    FewHead &h = *reinterpret_cast<FewHead *>(smem_raw + (base - raw));
    const bool whole = whole_t(p.c_dtype);
    const int b_blocks = p.b_blocks, t_blocks = ext_blocks(p.rp, whole);
    // T's blocks for the tensor core, or T and the dot products, then the ring.
    const uint32_t low = base + FEW_HEAD, ring = low + p.low_bytes;
    auto bar = [&](uint64_t &b) { return ptx::smem_u32(&b); };
    volatile uint32_t *abort_flag = &h.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = p.kc > 1 ? ptx::cluster_ctarank() : 0u;
    const int n0 = int(blockIdx.x) / p.kc * p.bn;
    const int kb0 = int(int64_t(p.k_blocks) * rank / p.kc), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / p.kc);
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            ptx::mbar_init(bar(h.full[s]), 1);
            ptx::mbar_init(bar(h.empty[s]), 1);
        }
        ptx::mbar_init(bar(h.low), 1);
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

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 0, filled = 0, filled_parity = 0;
        bool ok = !(p.debug & 4);
        // Waits for the next stage and announces `bytes`: its address, 0 when giving up.
        auto next = [&](uint32_t bytes) -> uint32_t {
            ok = __all_sync(0xffffffffu, wait_bar(bar(h.empty[s]), ph ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(s), limit));
            if (!ok) return 0u;
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar(h.full[s]), bytes);
            __syncwarp();
            return ring + uint32_t(s) * p.stage_bytes;
        };
        auto issued = [&] {
            __syncwarp();
            filled |= 1u << s;
            filled_parity = (filled_parity & ~(1u << s)) | (ph << s);
            if (++s == p.stages) s = 0, ph ^= 1u;
        };
        if (lane == 0) {
            ptx::prefetch_tensormap(&tmX);
            ptx::prefetch_tensormap(&tmW);
            if (b_blocks > 0) {
                ptx::prefetch_tensormap(&tmT);
                ptx::prefetch_tensormap(&tmB);
            }
        }
        const uint32_t w0 = uint32_t(p.kps) * p.x_bytes;
        const int kk = lane & 7;  // lanes 0-7 issue blocks of W, lanes 8-15 of X
        for (int kb = kb0; kb < kb1 && ok; kb += p.kps) {
            const int nk = min(p.kps, kb1 - kb);
            const uint32_t dst = next(uint32_t(nk) * (p.x_bytes + p.w_bytes));
            if (!ok) break;
            if (kk < nk && lane < 8) ptx::tma_load_2d(dst + w0 + uint32_t(kk) * p.w_bytes, &tmW, bar(h.full[s]), (kb + kk) * 64, n0);
            if (kk < nk && lane >= 8 && lane < 16) ptx::tma_load_2d(dst + uint32_t(kk) * p.x_bytes, &tmX, bar(h.full[s]), (kb + kk) * 64, 0);
            issued();
        }
        ptx::griddep_wait();
        ok = __all_sync(0xffffffffu, ok && wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_PRODUCER, 100u, limit));
        const int mine = ok ? low_blocks(h.entries, int(rank), p.kc, b_blocks) : 0;
        const bool has_low = mine > 0;
        if (has_low) {
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar(h.low), uint32_t(t_blocks) * p.x_bytes);
            __syncwarp();
            if (lane < t_blocks) ptx::tma_load_2d(low + uint32_t(lane) * p.x_bytes, &tmT, bar(h.low), ext_block(lane, p.rp, p.rank, whole, p.bf16).t_col, 0);
        }
        for (int i = 0; i < mine && ok; i += p.kps) {
            const int nk = min(p.kps, mine - i);
            const uint32_t dst = next(uint32_t(nk) * p.w_bytes);
            if (!ok) break;
            if (lane < nk) {
                const int e = int(rank) + (i + lane) / b_blocks * p.kc, q = (i + lane) % b_blocks;
                ptx::tma_load_2d(dst + w0 + uint32_t(lane) * p.w_bytes, &tmB, bar(h.full[s]), 64 * q, h.entry_id[e] * p.n + n0);
            }
            issued();
        }
        if (!ok && lane == 0) {  // giving up: let the copies in flight land (bounded) before the shared memory is handed back
            const uint64_t t0 = ptx::globaltimer_ns();
            for (int i = 0; i < p.stages; i++)
                while ((filled >> i & 1u) && !ptx::mbar_try_wait(bar(h.full[i]), (filled_parity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            while (has_low && !ptx::mbar_try_wait(bar(h.low), 0u))
                if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp runs the loop and one thread issues: the descriptors are then the same in every lane for the
        // compiler too, and an MMA of N <= 128 goes out every 65 clocks (from a loop of one lane: 115 and more, measured).
        const bool leader = ptx::elect_one();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true, issued = false;
        const uint32_t w0 = uint32_t(p.kps) * p.x_bytes;
        auto ready = [&] {
            ok = __all_sync(0xffffffffu, wait_bar(bar(h.full[s]), ph, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(s), limit));
            ptx::tc_fence_after();
            return ok;
        };
        auto free_stage = [&] {
            issued = true;
            if (leader) ptx::umma_commit<1>(bar(h.empty[s]));
            __syncwarp();
            if (++s == p.stages) s = 0, ph ^= 1u;
        };
        const int part_cols = (p.bn + 31) / 32 * 32;
        int part = 0, part_end = kb0 + (kb1 - kb0 + p.parts - 1) / p.parts;  // the k block the next accumulator begins at
        for (int kb = kb0; kb < kb1; kb += p.kps) {
            if (!ready()) break;
            const uint32_t src = ring + uint32_t(s) * p.stage_bytes;
            const int nk = min(p.kps, kb1 - kb);
            for (int kk = 0; kk < nk; kk++) {
                const uint64_t a = sw128_desc(src + uint32_t(kk) * p.x_bytes), b = sw128_desc(src + w0 + uint32_t(kk) * p.w_bytes);
                const bool next_part = kb + kk == part_end && part + 1 < p.parts;
                if (next_part) part++, part_end = kb0 + ((kb1 - kb0) * (part + 1) + p.parts - 1) / p.parts;
                const uint32_t more = (kb > kb0 || kk > 0) && !next_part ? 1u : 0u, d = tmem + uint32_t(part * part_cols);
                if (leader) {
#pragma unroll
                    for (int j = 0; j < 4; j++) ptx::umma_f16<1>(d, a + 2u * j, b + 2u * j, p.idesc, j > 0 ? 1u : more);
                }
                __syncwarp();
            }
            free_stage();
        }
        if (ok) ok = __all_sync(0xffffffffu, wait_bar(bar(h.plan), 0, abort_flag, p.status, WHERE_MMA_TMEM, 100u, limit));
        const int mine = ok ? low_blocks(h.entries, int(rank), p.kc, b_blocks) : 0;
        if (mine > 0) ok = __all_sync(0xffffffffu, wait_bar(bar(h.low), 0, abort_flag, p.status, WHERE_MMA_FULL, 101u, limit));
        for (int i = 0; i < mine && ok; i += p.kps) {
            if (!ready()) break;
            const uint32_t src = ring + uint32_t(s) * p.stage_bytes;
            const int nk = min(p.kps, mine - i);
            for (int kk = 0; kk < nk; kk++) {
                const int e = int(rank) + (i + kk) / b_blocks * p.kc, q = (i + kk) % b_blocks;
                const uint32_t o0 = h.off[e][0], o1 = h.off[e][1], o2 = h.off[e][2], o3 = h.off[e][3];
                const uint64_t b = sw128_desc(src + w0 + uint32_t(kk) * p.w_bytes);
                // The blocks of T that go with this block of B.
                const int parts = t_blocks / b_blocks;
                for (int part = 0; part < parts; part++) {
                    const ExtBlock x = ext_block(parts * q + part, p.rp, p.rank, whole, p.bf16);
                    const uint64_t a = sw128_desc(low + uint32_t(parts * q + part) * p.x_bytes);
                    if (leader)
                        for (int j = 0; j < x.steps; j++) ptx::umma_f16_lanes(tmem, a + 2u * j, b + 2u * (j & x.b_mask), p.idesc, 1u, o0, o1, o2, o3);
                    __syncwarp();
                }
            }
            free_stage();
        }
        if (leader) {
            if (ok) {
                ptx::umma_commit<1>(bar(h.done));
            } else if (issued) {  // giving up: wait (bounded) until the tensor core is done with shared memory and TMEM
                ptx::umma_commit<1>(bar(h.drain));
                const uint64_t t0 = ptx::globaltimer_ns();
                while (!ptx::mbar_try_wait(bar(h.drain), 0u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
            }
        }
        __syncwarp();
    } else {
        // The adapters the rows name, in the order of their first row.  The ids, like W, are older than the kernel that
        // computes T.
        const int row = threadIdx.x - 64;
        int id = row < p.m ? p.ids[row] : -1;
        if (id < 0 || id >= p.adapters) id = -1;
        h.id[row] = id;
        if (b_blocks > 0) {
            for (int i = row; i < FEW_ROWS * 4; i += 128) h.off[i / 4][i % 4] = 0xffffffffu;
            const int32_t ids[1] = {id};
            int32_t mine[1];
            const int total = distinct_ids<FEW_ROWS>(ids, h.table, row, mine, [&](int e, int which) { h.entry_id[e] = which; });
            if (mine[0] >= 0) atomicAnd(&h.off[mine[0]][row / 32], ~(1u << (row % 32)));
            if (row == 0) h.entries = total;
        }
        ptx::named_barrier(1, 128);
        if (row == 0) ptx::mbar_arrive(bar(h.plan));
        if (b_blocks == 0) {
            float *t = reinterpret_cast<float *>(smem_raw + (low - raw)), *dots = t + (p.m + p.kc - 1) / p.kc * p.rp;
            if (p.bf16) few_dots<true>(p, h.id, t, dots, int(rank), n0, row);
            else few_dots<false>(p, h.id, t, dots, int(rank), n0, row);
        } else {
            ptx::griddep_wait();
        }

        // The accumulator's rows to shared memory (the ring is idle: every load has been consumed).
        const bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.done), 0, abort_flag, p.status, WHERE_EPILOGUE, 0u, limit));
        const int q = warp & 3;  // the TMEM lanes this warp may read: rows 32 q ..
        const uint32_t pitch = uint32_t(p.bn + 4) * 4u;
        if (ok && 32 * q < p.m) {
            ptx::tc_fence_after();
            ptx::fence_proxy_async_shared();
            for (int c = 0; c < p.bn; c += 32) {
                uint32_t v[32];
                const uint32_t from = tmem + (uint32_t(32 * q) << 16) + uint32_t(c);
                ptx::tmem_ld_32x32(from, v);
                ptx::tmem_ld_wait(v);
                for (int i = 1; i < p.parts; i++) {
                    uint32_t o[32];
                    ptx::tmem_ld_32x32(from + uint32_t(i * ((p.bn + 31) / 32 * 32)), o);
                    ptx::tmem_ld_wait(o);
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(o[j]));
                }
                if (32 * q + lane < p.m) {
                    const uint32_t dst = ring + uint32_t(32 * q + lane) * pitch + uint32_t(c) * 4u;
#pragma unroll
                    for (int g = 0; g < 8; g++)
                        if (c + 4 * g < p.bn) ptx::st_shared_v4(dst + 16u * g, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
                }
            }
        }
        __syncwarp();
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (p.kc > 1) {  // every CTA of the cluster has its partial sums in shared memory (or has given up)
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (!*abort_flag) {
        const int quads = p.bn / 4, items = p.m * quads;
        const uint32_t pitch = uint32_t(p.bn + 4) * 4u;
        const Divider by_quads(quads);
        constexpr int TURN = 4;
        const int shift = __ffs(p.kc) - 1, stride = p.kc * FEW_THREADS;
        const uint32_t dots = low + uint32_t(((p.m + p.kc - 1) >> shift) * p.rp) * 4u;
        for (int first = int(rank) * FEW_THREADS; first < items; first += TURN * stride) {  // as in cluster_sums
            const int i0 = first + int(threadIdx.x);
            float4 v[TURN], dot[TURN];
#pragma unroll
            for (int u = 0; u < TURN; u++) {
                if (first + u * stride >= items) continue;
                const int i = min(i0 + u * stride, items - 1), row = by_quads(i), col = (i - row * quads) * 4;
                v[u] = cluster_sum(ring + uint32_t(row) * pitch + uint32_t(col) * 4u, p.kc);
                if (b_blocks == 0) {  // the dot products of this row were taken by CTA row % kc
                    const uint32_t from = dots + uint32_t((row >> shift) * p.bn + col) * 4u;
                    dot[u] = ptx::ld_shared_cluster_v4(p.kc > 1 ? ptx::mapa(from, uint32_t(row & (p.kc - 1))) : from);
                }
            }
#pragma unroll
            for (int u = 0; u < TURN; u++) {
                const int i = i0 + u * stride, row = by_quads(i), col = (i - row * quads) * 4;
                if (i >= items) break;
                if (b_blocks == 0) v[u].x += dot[u].x, v[u].y += dot[u].y, v[u].z += dot[u].z, v[u].w += dot[u].w;
                const int64_t gcol = n0 + col, out = int64_t(row) * p.ldy + gcol;
                if (p.vec && gcol + 4 <= p.n) {
                    if (p.c_dtype == CUTE_B200_F32) *reinterpret_cast<float4 *>(static_cast<float *>(p.y) + out) = v[u];
                    else {
                        const bool bf16 = p.c_dtype == CUTE_B200_BF16;
                        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.y) + out) =
                            make_uint2(pack_16(v[u].x, v[u].y, bf16), pack_16(v[u].z, v[u].w, bf16));
                    }
                } else {
                    const float f[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
                    for (int j = 0; j < 4; j++)
                        if (gcol + j < p.n) store_c(p.y, p.c_dtype, size_t(out + j), f[j]);
                }
            }
        }
    }
    __syncthreads();
    if (p.kc > 1) {  // until every CTA has read its peers' shared memory
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, p.tmem_cols);
}

// Less than all of it: the CTAs of the kernel that computes T (1.2 KB each) have to fit beside, or W would not stream until
// they are gone.
constexpr uint32_t FEW_SMEM = 216 * 1024;

// ---- one row of a rank up to 16 ---------------------------------------------------
// T and Y by one kernel: the 16 rows of the row's A lie behind the tile's rows of W as further columns of the same MMA, so T
// comes out of the stream that Y comes out of (every cluster computes it anew; A comes from L2 but for the first time), and
// the adapter's part is dot products with rows of B fetched meanwhile, by the first CTA of a cluster.  A second kernel's launch
// falls away, 2 us on the host; on the device 4096 x 4096 takes 11.3 us (11.6 by two kernels), 32000 x 2048 24.6 (26.4), 1024 x 1024
// 6.1 (6.7), 512 x 8192 8.6 (8.4).  With more rows or ranks the stream of A costs what the launch saves (64 columns of A: 13.9
// and 11.8).  Bound by latency, then HBM.
//   warp 0  TMA: W, X and, once the id is there, A.   warp 1  MMA, M 128, N = bn + 16.
//   warps 2-5  the slice of B to shared memory; then the accumulators' row.  All: T, the sums over the cluster, Y.
// T is rounded to the sum of two 16-bit numbers, as everywhere.
constexpr int ONE_RANK = 16;
constexpr uint32_t ONE_HEAD = 2048;

struct OneParams {
    const int32_t *ids;
    const float *scale;
    const uint16_t *b;
    uint16_t *t;
    void *y;
    int n, rank, adapters, c_dtype, vec;
    int k_blocks, bn, kc, cols, stages, kps, parts;  // cols: bn + ONE_RANK
    uint32_t stage_bytes, w_bytes, b_bytes, idesc, tmem_cols;
    bool bf16;
    uint32_t *status;
    int debug;
};
constexpr uint32_t ONE_X_BYTES = 8 * 128;

struct OneHead {
    uint64_t full[FEW_MAX_STAGES], empty[FEW_MAX_STAGES], done, drain;
    uint32_t tmem, abort;
    int32_t id;  // -1 = none
    float scale, t[ONE_RANK];
};
static_assert(sizeof(OneHead) <= ONE_HEAD, "head");

__global__ void __launch_bounds__(FEW_THREADS, 1)
    lora_one_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                    const OneParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    OneHead &h = *reinterpret_cast<OneHead *>(smem_raw + (base - raw));
    const uint32_t slice = base + ONE_HEAD, ring = slice + p.b_bytes;
    auto bar = [&](uint64_t &b) { return ptx::smem_u32(&b); };
    volatile uint32_t *abort_flag = &h.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = p.kc > 1 ? ptx::cluster_ctarank() : 0u;
    const int n0 = int(blockIdx.x) / p.kc * p.bn;
    const int kb0 = int(int64_t(p.k_blocks) * rank / p.kc), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / p.kc);
    const int part_cols = (p.cols + 31) / 32 * 32;
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; s++) {
            ptx::mbar_init(bar(h.full[s]), 1);
            ptx::mbar_init(bar(h.empty[s]), 1);
        }
        ptx::mbar_init(bar(h.done), 1);
        ptx::mbar_init(bar(h.drain), 1);
        h.abort = 0u;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmX);
        ptx::prefetch_tensormap(&tmW);
        ptx::prefetch_tensormap(&tmA);
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

    const uint32_t w0 = uint32_t(p.kps) * ONE_X_BYTES;
    if (warp == 0) {
        // Lanes 0-3 issue blocks of W, 8-11 of X, 16-19 of A (some adapter's, where the row has none: nothing reads those
        // columns).  One instruction for all of them: a step costs 0.3 us per instruction.
        const bool w_lane = lane < 8, a_lane = lane >= 16;
        const int kk = lane & 7;
        const bool mine = kk < p.kps && lane < 24;
        const CUtensorMap *map = a_lane ? &tmA : (w_lane ? &tmW : &tmX);
        const uint32_t to = ring + (a_lane || w_lane ? w0 + uint32_t(kk) * p.w_bytes + (a_lane ? uint32_t(p.bn) * 128u : 0u) : uint32_t(kk) * ONE_X_BYTES);
        const int id = a_lane ? __ldcg(p.ids) : 0;
        int y = w_lane ? n0 : 0;
        bool ok = !(p.debug & 4);
        int s = 0;
        uint32_t ph = 0, filled = 0, filled_parity = 0;
        const int steps = (kb1 - kb0 + p.kps - 1) / p.kps, early = min(2, steps);  // early: steps issued before the id is there
        auto issue = [&](int i, int stage, bool go) {
            const int kb = kb0 + i * p.kps + kk;
            if (go && mine && kb < kb1) ptx::tma_load_2d(to + uint32_t(stage) * p.stage_bytes, map, bar(h.full[stage]), kb * 64, y);
            __syncwarp();
        };
        for (int i = 0; i < steps && ok; i++) {
            if (i >= p.stages) ok = __all_sync(0xffffffffu, wait_bar(bar(h.empty[s]), ph ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(s), limit));
            if (!ok) break;
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar(h.full[s]), uint32_t(min(p.kps, kb1 - kb0 - i * p.kps)) * (ONE_X_BYTES + p.w_bytes));
            __syncwarp();
            issue(i, s, i >= early || !a_lane);
            filled |= 1u << s, filled_parity = (filled_parity & ~(1u << s)) | (ph << s);
            if (++s == p.stages) s = 0, ph ^= 1u;
            if (i + 1 == early) {  // stages 0 and 1
                if (a_lane) y = id >= 0 && id < p.adapters ? id * p.rank : 0;
                for (int e = 0; e < early; e++) issue(e, e, a_lane);
            }
        }
        if (!ok && lane == 0) {  // giving up: let the copies in flight land (bounded)
            const uint64_t t0 = ptx::globaltimer_ns();
            for (int i = 0; i < p.stages; i++)
                while ((filled >> i & 1u) && !ptx::mbar_try_wait(bar(h.full[i]), (filled_parity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        const bool leader = ptx::elect_one();  // see lora_few_kernel
        int s = 0, part = 0, part_end = kb0 + (kb1 - kb0 + p.parts - 1) / p.parts;
        uint32_t ph = 0;
        bool ok = true, issued = false;
        for (int kb = kb0; kb < kb1; kb += p.kps) {
            ok = __all_sync(0xffffffffu, wait_bar(bar(h.full[s]), ph, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(s), limit));
            if (!ok) break;
            ptx::tc_fence_after();
            const uint32_t src = ring + uint32_t(s) * p.stage_bytes;
            const int nk = min(p.kps, kb1 - kb);
            for (int kk = 0; kk < nk; kk++) {
                const uint64_t a = sw128_desc(src + uint32_t(kk) * ONE_X_BYTES), b = sw128_desc(src + w0 + uint32_t(kk) * p.w_bytes);
                const bool next_part = kb + kk == part_end && part + 1 < p.parts;
                if (next_part) part++, part_end = kb0 + ((kb1 - kb0) * (part + 1) + p.parts - 1) / p.parts;
                const uint32_t more = (kb > kb0 || kk > 0) && !next_part ? 1u : 0u, d = tmem + uint32_t(part * part_cols);
                if (leader) {
#pragma unroll
                    for (int j = 0; j < 4; j++) ptx::umma_f16<1>(d, a + 2u * j, b + 2u * j, p.idesc, j > 0 ? 1u : more);
                }
                __syncwarp();
            }
            issued = true;
            if (leader) ptx::umma_commit<1>(bar(h.empty[s]));
            __syncwarp();
            if (++s == p.stages) s = 0, ph ^= 1u;
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
        const int t = threadIdx.x - 64, named = __ldcg(p.ids), id = named >= 0 && named < p.adapters ? named : -1;
        if (t == 0) h.id = id, h.scale = id >= 0 ? __ldcg(p.scale + id) : 0.0f;
        if (id >= 0 && rank == 0) {  // the tile's rows of B lie one after another; the first CTA of a cluster multiplies them
            const int pieces = min(p.bn, p.n - n0) * p.rank / 8;
            const uint4 *src = reinterpret_cast<const uint4 *>(p.b + (int64_t(id) * p.n + n0) * p.rank);
#pragma unroll 4
            for (int i = t; i < pieces; i += 128) {
                const uint4 v = __ldg(src + i);
                ptx::st_shared_v4(slice + uint32_t(i) * 16u, v.x, v.y, v.z, v.w);
            }
        }
        const bool ok = __all_sync(0xffffffffu, wait_bar(bar(h.done), 0, abort_flag, p.status, WHERE_EPILOGUE, 0u, limit));
        if (ok && (warp & 3) == 0) {  // the warp that may read row 0
            ptx::tc_fence_after();
            ptx::fence_proxy_async_shared();
            for (int c = 0; c < p.cols; c += 16) {
                uint32_t v[4][16];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (i < p.parts) ptx::tmem_ld_32x16(tmem + uint32_t(i * part_cols + c), v[i]);
                ptx::tmem_ld_wait_all();
                ptx::pin16(v[0]);
#pragma unroll
                for (int i = 1; i < 4; i++) {
                    if (i >= p.parts) continue;
                    ptx::pin16(v[i]);
#pragma unroll
                    for (int j = 0; j < 16; j++) v[0][j] = __float_as_uint(__uint_as_float(v[0][j]) + __uint_as_float(v[i][j]));
                }
                if (lane == 0) {
#pragma unroll
                    for (int g = 0; g < 4; g++) ptx::st_shared_v4(ring + uint32_t(c) * 4u + 16u * g, v[0][4 * g], v[0][4 * g + 1], v[0][4 * g + 2], v[0][4 * g + 3]);
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
    const bool good = !*abort_flag;
    if (good && rank == 0 && threadIdx.x < ONE_RANK / 4) {  // T; the first cluster stores it
        const int j = 4 * int(threadIdx.x);
        const float4 v = cluster_sum(ring + uint32_t(p.bn + j) * 4u, p.kc);
        const float s = h.scale;
        const bool has = h.id >= 0 && j < p.rank;  // past the rank may lie another adapter's sums
        const float4 w = has ? make_float4(v.x * s, v.y * s, v.z * s, v.w * s) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float4 t = store_t4(p.t + j, ONE_RANK, w, p.bf16, blockIdx.x == 0);
        h.t[j] = t.x, h.t[j + 1] = t.y, h.t[j + 2] = t.z, h.t[j + 3] = t.w;
    }
    __syncthreads();
    const int i = int(threadIdx.x);  // four columns; bn / 4 is less than the CTA's threads
    if (good && rank == 0 && i < p.bn / 4) {
        const float4 v = cluster_sum(ring + uint32_t(i) * 16u, p.kc);
        float f[4] = {v.x, v.y, v.z, v.w};
        const int gcol = n0 + 4 * i;
        if (h.id >= 0) {
            const uint4 *b = reinterpret_cast<const uint4 *>(smem_raw + (slice - raw)) + 4 * i * p.rank / 8;
#pragma unroll 1
            for (int c = 0; c < 4; c++) {
                float dot = 0.0f;
                for (int j = 0; j < p.rank; j += 8) {
                    const uint4 q = b[(c * p.rank + j) / 8];
                    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 x = p.bf16 ? pair_f32<true>(w[e]) : pair_f32<false>(w[e]);
                        dot = fmaf(x.y, h.t[j + 2 * e + 1], fmaf(x.x, h.t[j + 2 * e], dot));
                    }
                }
                f[c] += dot;
            }
        }
        if (p.vec && gcol + 4 <= p.n) {
            if (p.c_dtype == CUTE_B200_F32) *reinterpret_cast<float4 *>(static_cast<float *>(p.y) + gcol) = make_float4(f[0], f[1], f[2], f[3]);
            else {
                const bool bf16 = p.c_dtype == CUTE_B200_BF16;
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.y) + gcol) = make_uint2(pack_16(f[0], f[1], bf16), pack_16(f[2], f[3], bf16));
            }
        } else {
            for (int c = 0; c < 4; c++)
                if (gcol + c < p.n) store_c(p.y, p.c_dtype, size_t(gcol + c), f[c]);
        }
    }
    __syncthreads();
    if (p.kc > 1) {  // until every CTA has read its peers' shared memory
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, p.tmem_cols);
}

cute_b200_status forward_one(const LoraParams &p, bool bf16, const DeviceState &dev, int debug, cudaStream_t stream) {
    OneParams f = {};
    f.ids = p.ids, f.scale = p.scale, f.b = p.b, f.t = p.t, f.y = p.y;
    f.n = p.n, f.rank = p.rank, f.adapters = p.adapters, f.c_dtype = p.c_dtype;
    f.vec = reinterpret_cast<uint64_t>(p.y) % (p.c_dtype == CUTE_B200_F32 ? 16 : 8) == 0;
    f.k_blocks = (p.k + 63) / 64;
    f.bn = 16, f.kc = 1;
    stream_cut(p.n, f.k_blocks, dev.few_clusters, &f.bn, &f.kc, ONE_RANK);
    f.cols = f.bn + ONE_RANK;
    f.w_bytes = uint32_t(f.cols) * 128u;
    f.b_bytes = (uint32_t(f.bn * p.rank) * 2u + 1023u) / 1024u * 1024u;
    // The head, B, the ring, and behind the last stage as much as an MMA reads past its rows of X.
    const uint32_t ring = FEW_SMEM - ONE_HEAD - 1024 - f.b_bytes;
    f.kps = stream_blocks(f.cols, 8, ring, 320);
    f.stage_bytes = uint32_t(f.kps) * (ONE_X_BYTES + f.w_bytes);
    const uint32_t reach = uint32_t(f.kps - 1) * ONE_X_BYTES + 16384, over = f.stage_bytes < reach ? reach - f.stage_bytes : 0;
    f.stages = int((ring - over) / f.stage_bytes);
    if (f.stages > FEW_MAX_STAGES) f.stages = FEW_MAX_STAGES;
    f.idesc = make_idesc(bf16, 128, f.cols);
    f.parts = f.cols <= 128 ? 4 : 2;  // accumulators added in f32: see T_PARTS of the tiled kernels
    while (f.parts > f.k_blocks / f.kc && f.parts > 1) f.parts /= 2;
    for (f.tmem_cols = 32; f.tmem_cols < uint32_t(f.parts * ((f.cols + 31) / 32 * 32)); f.tmem_cols *= 2) {}
    f.bf16 = bf16;
    f.status = dev.status_word;
    f.debug = debug;
    CUtensorMap tmX, tmW, tmA;
    CB_TRY(rows_tensor_map(&tmX, reinterpret_cast<uint64_t>(p.x), bf16, p.m, p.k, p.ldx, 8));
    CB_TRY(rows_tensor_map(&tmW, reinterpret_cast<uint64_t>(p.w), bf16, p.n, p.k, p.k, f.bn));
    CB_TRY(rows_tensor_map(&tmA, reinterpret_cast<uint64_t>(p.a), bf16, uint64_t(p.adapters) * p.rank, p.k, p.k, ONE_RANK));
    const unsigned grid = unsigned((p.n + f.bn - 1) / f.bn) * unsigned(f.kc);
    return launch_dependent(lora_one_kernel, dim3(grid), FEW_THREADS, FEW_SMEM, f.kc, stream, tmX, tmW, tmA, f);
}

// How the few-row kernels would run a problem, and in what time.  The terms are fitted to measurements of both ways (graphs of
// 60 calls, us, few / tiled; rows with one of a adapters each):
//   n 4096 k 4096 rank 16 a 64: 8 rows 12 / 22, 64 rows 17 / 39, 128 rows 22 / 49
//   n 8192 k 4096 rank 16 a 4: 8 rows 17 / 33, 32 rows 19 / 22, 64 rows 23 / 23, 128 rows 26 / 23
//   n 16384 k 2048 rank 32 a 8: 8 rows 17 / 25, 32 rows 20 / 19, 128 rows 28 / 19
//   n 1000 k 8192 rank 128 a 4: 8 rows 15 / 33, 128 rows 30 / 35
// The tiled kernels read every adapter's weights tile by tile and do not cut k; the few-row kernels pay for every row: its
// part of X per k block, its dot products (or its adapter's masked product), its place in the final sum.
struct FewPlan {
    int bn = 16, kc = 1;
    bool dots = false;  // the adapters' part as dot products
    double time = 0.0;
};
FewPlan few_plan(const LoraParams &p, const DeviceState &dev) {
    FewPlan f;
    const int k_blocks = (p.k + 63) / 64, entries = p.adapters < p.m ? p.adapters : p.m;
    stream_cut(p.n, k_blocks, dev.few_clusters, &f.bn, &f.kc);
    const int own = (p.m + f.kc - 1) / f.kc, at_once = p.rank <= 16 ? 8 : 4;
    const double dots = (own + at_once - 1) / at_once * ((f.bn + 127) / 128) * 0.8e-6;
    const double masked = (entries + f.kc - 1) / f.kc * (p.rp <= 64 ? 1 : 2) * 0.5e-6;
    f.dots = p.rp <= 32 && uint64_t(own) * uint64_t(p.rp + f.bn) * 4 <= FEW_DOTS && dots <= masked;
    const double stream = double(p.n) * p.k * 2 / 6.0e12 + double(k_blocks) / f.kc * p.m * 128 / 9.0e10;
    const double low = 2.5e-6 + double(p.m) / SHRINK_ROWS * p.rp / (p.rank >= 64 ? 8 : 4) / (2.0 * dev.sm_count) * (p.k / 2048.0 * 1.0e-6 + 1.5e-6);
    f.time = 5.5e-6 + (stream > low ? stream : low) + (f.dots ? dots : masked) + double(p.m) * f.bn / (4.0 * f.kc * 2 * FEW_THREADS) * 0.6e-6;
    return f;
}
double tiled_time(const LoraParams &p, const DeviceState &dev) {
    const int k_blocks = (p.k + 63) / 64, entries = p.adapters < p.m ? p.adapters : p.m;
    const double waves = double(((p.n + 127) / 128 + dev.sm_count - 1) / dev.sm_count), weight = double(p.n) * p.k * 2 / 5.5e12;
    const double product = waves * k_blocks * 0.19e-6;
    return 8.0e-6 + (weight > product ? weight : product) + entries * (0.05e-6 * p.k / 1024 * p.rp / 16 + 0.3e-6 * ext_blocks(p.rp, whole_t(p.c_dtype)));
}

template <bool BF16>
cute_b200_status forward_few(const LoraParams &p, const FewPlan &plan, const DeviceState &dev, int debug, cudaStream_t stream) {
    if (p.rank >= 64) CB_TRY(launch_dependent(shrink_rows_kernel<BF16, 8>, dim3(unsigned(p.m), unsigned(p.rp / 8)), SHRINK_THREADS, 0, 1, stream, p));
    else CB_TRY(launch_dependent(shrink_rows_kernel<BF16, 4>, dim3(unsigned(p.m), unsigned(p.rp / 4)), SHRINK_THREADS, 0, 1, stream, p));
    FewParams f = {};
    f.ids = p.ids, f.y = p.y, f.ldy = p.ldy;
    f.m = p.m, f.n = p.n, f.rank = p.rank, f.rp = p.rp, f.adapters = p.adapters, f.c_dtype = p.c_dtype;
    const uint64_t esize = p.c_dtype == CUTE_B200_F32 ? 4 : 2;
    f.vec = reinterpret_cast<uint64_t>(p.y) % (4 * esize) == 0 && p.ldy % 4 == 0;
    f.k_blocks = (p.k + 63) / 64;
    f.bn = plan.bn, f.kc = plan.kc;
    f.xr = (p.m + 7) / 8 * 8;
    f.x_bytes = uint32_t(f.xr) * 128u;
    f.w_bytes = uint32_t(f.bn) * 128u;
    // The head, T, the ring, and behind the last stage as much as an MMA reads past its rows of X.
    const uint64_t dots = uint64_t((p.m + f.kc - 1) / f.kc) * uint64_t(p.rp + f.bn) * 4;
    f.b_blocks = plan.dots ? 0 : (p.rp <= 64 ? 1 : 2);
    f.low_bytes = f.b_blocks == 0 ? uint32_t((dots + 1023) / 1024 * 1024) : uint32_t(ext_blocks(p.rp, whole_t(p.c_dtype))) * f.x_bytes;
    f.t = p.t, f.b = p.b, f.bf16 = BF16;
    const uint32_t ring = FEW_SMEM - FEW_HEAD - 1024 - f.low_bytes;
    f.kps = stream_blocks(f.bn, f.xr, ring);
    f.stage_bytes = uint32_t(f.kps) * (f.x_bytes + f.w_bytes);
    const uint32_t reach = uint32_t(f.kps - 1) * f.x_bytes + 16384, over = f.stage_bytes < reach ? reach - f.stage_bytes : 0;
    f.stages = int((ring - over) / f.stage_bytes);
    if (f.stages > FEW_MAX_STAGES) f.stages = FEW_MAX_STAGES;
    f.idesc = make_idesc(BF16, 128, f.bn);
    // An f32 result: two or four accumulators, added in f32 (the tensor core's own sums are cut off, not rounded).
    f.parts = p.c_dtype != CUTE_B200_F32 ? 1 : (f.bn <= 128 ? 4 : 2);
    while (f.parts > f.k_blocks / f.kc && f.parts > 1) f.parts /= 2;  // every one of them is written
    for (f.tmem_cols = 32; f.tmem_cols < uint32_t(f.parts * ((f.bn + 31) / 32 * 32)); f.tmem_cols *= 2) {}
    f.status = dev.status_word;
    f.debug = debug;
    CUtensorMap tmX, tmW, tmT = {}, tmB = {};
    CB_TRY(rows_tensor_map(&tmX, reinterpret_cast<uint64_t>(p.x), BF16, p.m, p.k, p.ldx, f.xr));
    CB_TRY(rows_tensor_map(&tmW, reinterpret_cast<uint64_t>(p.w), BF16, p.n, p.k, p.k, f.bn));
    if (f.b_blocks > 0) {
        CB_TRY(rows_tensor_map(&tmT, reinterpret_cast<uint64_t>(p.t), BF16, p.m, t_planes(BF16) * p.rp, t_planes(BF16) * p.rp, f.xr));
        CB_TRY(rows_tensor_map(&tmB, reinterpret_cast<uint64_t>(p.b), BF16, uint64_t(p.adapters) * p.n, p.rank, p.rank, f.bn));
    }
    const unsigned grid = unsigned((p.n + f.bn - 1) / f.bn) * unsigned(f.kc);
    return launch_dependent(lora_few_kernel, dim3(grid), FEW_THREADS, FEW_SMEM, f.kc, stream, tmX, tmW, tmT, tmB, f);
}

constexpr uint64_t kAlign = 256;
uint64_t round_up(uint64_t v) { return (v + kAlign - 1) / kAlign * kAlign; }
uint64_t t_bytes(const cute_b200_lora_desc &d) { return round_up(uint64_t(d.m) * padded_rank(d.rank) * 2 * t_planes(d.ab_dtype == CUTE_B200_BF16)); }

uint64_t plan_bytes(const cute_b200_lora_desc &d) { return round_up(lora_plan_bytes(d.m, d.adapters)) + kAlign; }

// The backward call's workspace: U and the plan of its product, the row lists.
struct BackLayout {
    uint64_t first, list, total;
};
BackLayout back_layout(const cute_b200_lora_desc &d) {
    BackLayout l;
    l.first = t_bytes(d) + plan_bytes(d);
    l.list = l.first + round_up((uint64_t(d.adapters) + 1) * 4);
    l.total = l.list + round_up(uint64_t(d.m) * 4) + kAlign;
    return l;
}

cute_b200_status check_desc(const cute_b200_lora_desc &d, const char *who) {
    if (d.m < 0 || d.n < 1 || d.k < 8)
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: invalid size %dx%dx%d", who, d.m, d.n, d.k);
    if (d.m > (1 << 30) || d.n > (1 << 30) || d.k > (1 << 30))
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: m, n and k may be at most 2^30, got %dx%dx%d", who, d.m, d.n, d.k);
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
    if (d.tuning[0] < 0 || d.tuning[0] > 6 || (d.tuning[0] == 1 && d.m > 128))
        return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "%s: tuning[0] must be 0, 1 (with m <= 128) or 2 to 6, got %d", who, d.tuning[0]);
    return CUTE_B200_OK;
}

cute_b200_status check_ptr(const char *who, const char *name, uint64_t p, uint64_t align, bool need) {
    if (!p && need) return fail(CUTE_B200_ERR_NULL_POINTER, "%s: %s is null", who, name);
    if (p % align) return fail(CUTE_B200_ERR_MISALIGNED, "%s: %s must be %llu-byte aligned", who, name, (unsigned long long)align);
    return CUTE_B200_OK;
}

uint64_t elem_bytes(int dtype) { return dtype == CUTE_B200_F32 ? 4 : 2; }

cute_b200_status forward(const LoraParams &p, bool bf16, const int32_t (&tuning)[2], const DeviceState &dev, cudaStream_t stream) {
    if (p.m == 0) return CUTE_B200_OK;
    if (tuning[0] == 1 || (tuning[0] == 0 && p.m <= FEW_ROWS)) {
        if (p.m == 1 && p.rp == ONE_RANK) return forward_one(p, bf16, dev, tuning[1], stream);
        const FewPlan plan = few_plan(p, dev);
        if (tuning[0] == 1 || plan.time <= tiled_time(p, dev))
            return bf16 ? forward_few<true>(p, plan, dev, tuning[1], stream) : forward_few<false>(p, plan, dev, tuning[1], stream);
    }
    return lora_tiled(p, bf16, tuning[0] - 3, tuning[1], dev, stream);
}

}  // namespace

cute_b200_status lora_workspace(const cute_b200_lora_desc &d, uint64_t *forward, uint64_t *backward) {
    CB_TRY(check_desc(d, "lora_workspace"));
    *forward = t_bytes(d) + plan_bytes(d);
    *backward = back_layout(d).total;
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

cute_b200_status lora_tn(const cute_b200_lora_desc &d, const uint64_t ptr[8], cudaStream_t stream, const DeviceState &dev) {
    LoraParams p = {};
    p.x = reinterpret_cast<const uint16_t *>(ptr[0]);
    p.w = reinterpret_cast<const uint16_t *>(ptr[1]);
    p.a = reinterpret_cast<const uint16_t *>(ptr[2]);
    p.b = reinterpret_cast<const uint16_t *>(ptr[3]);
    p.ids = reinterpret_cast<const int32_t *>(ptr[4]);
    p.scale = reinterpret_cast<const float *>(ptr[5]);
    p.y = reinterpret_cast<void *>(ptr[6]);
    p.t = reinterpret_cast<uint16_t *>(ptr[7]);
    p.plan = reinterpret_cast<uint32_t *>(ptr[7] + t_bytes(d));
    p.m = d.m, p.n = d.n, p.k = d.k, p.rank = d.rank, p.rp = padded_rank(d.rank), p.adapters = d.adapters, p.c_dtype = d.c_dtype;
    p.ldx = d.ldx ? d.ldx : d.k;
    p.ldy = d.ldy ? d.ldy : d.n;
    return forward(p, d.ab_dtype == CUTE_B200_BF16, d.tuning, dev, stream);
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

cute_b200_status lora_tn_backward(const cute_b200_lora_desc &d, const uint64_t ptr[12], cudaStream_t stream, const DeviceState &dev) {
    const int64_t ldx = d.ldx ? d.ldx : d.k, ldy = d.ldy ? d.ldy : d.n;
    const bool bf16 = d.ab_dtype == CUTE_B200_BF16;
    float *da = reinterpret_cast<float *>(ptr[9]), *db = reinterpret_cast<float *>(ptr[10]);
    if (d.m == 0) {
        if (da) CB_CUDA(cudaMemsetAsync(da, 0, size_t(d.adapters) * d.rank * d.k * 4, stream));
        if (db) CB_CUDA(cudaMemsetAsync(db, 0, size_t(d.adapters) * d.rank * d.n * 4, stream));
        return CUTE_B200_OK;
    }
    uint16_t *u = reinterpret_cast<uint16_t *>(ptr[11]);
    const BackLayout l = back_layout(d);
    int32_t *first = reinterpret_cast<int32_t *>(ptr[11] + l.first), *list = reinterpret_cast<int32_t *>(ptr[11] + l.list);
    CB_TRY(lora_row_lists(reinterpret_cast<const int32_t *>(ptr[4]), d.m, d.adapters, first, list, stream));
    LoraParams p = {};
    p.x = reinterpret_cast<const uint16_t *>(ptr[6]);
    p.w = reinterpret_cast<const uint16_t *>(ptr[1]);
    p.a = reinterpret_cast<const uint16_t *>(ptr[3]);
    p.b = reinterpret_cast<const uint16_t *>(ptr[2]);
    p.low_mn = true;
    p.ids = reinterpret_cast<const int32_t *>(ptr[4]);
    p.scale = reinterpret_cast<const float *>(ptr[5]);
    p.y = reinterpret_cast<void *>(ptr[8]);
    p.t = u;
    p.plan = reinterpret_cast<uint32_t *>(ptr[11] + t_bytes(d));
    p.m = d.m, p.n = d.k, p.k = d.n, p.rank = d.rank, p.rp = padded_rank(d.rank), p.adapters = d.adapters, p.c_dtype = d.c_dtype;
    p.ldx = ldy;
    p.ldy = ldx;
    CB_TRY(lora_tiled(p, bf16, d.tuning[0] - 3, d.tuning[1], dev, stream));
    if (da) {
        LoraGrads g = {};
        g.out[0] = da, g.out[1] = db;
        g.wide[0] = reinterpret_cast<const uint16_t *>(ptr[0]), g.wide[1] = p.x;
        g.low[0] = u, g.low[1] = reinterpret_cast<const uint16_t *>(ptr[7]);
        g.pitch[0] = ldx, g.pitch[1] = ldy;
        g.cols[0] = d.k, g.cols[1] = d.n;
        g.m = d.m, g.rank = d.rank, g.rp = p.rp, g.adapters = d.adapters;
        g.first = first, g.list = list;
        CB_TRY(lora_grads(g, bf16, d.tuning[1], dev, stream));
    }
    return CUTE_B200_OK;
}

cute_b200_status lora_init(DeviceState &dev) {
    CB_CUDA(cudaFuncSetAttribute(lora_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM));
    CB_CUDA(cudaFuncSetAttribute(lora_one_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM));
    for (int c = 0; c < 4; c++) CB_TRY(max_clusters(lora_few_kernel, FEW_THREADS, FEW_SMEM, 1 << c, &dev.few_clusters[c]));
    CB_TRY(lora_tiled_init(dev));
    CB_TRY(lora_grad_init());
    return CUTE_B200_OK;
}

}  // namespace cb
