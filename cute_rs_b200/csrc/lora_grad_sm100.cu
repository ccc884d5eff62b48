// Gradients of the adapters:
//     dA[a] = sum over rows i of adapter a of U[i] x[i]^T        (rank, k)
//     dB[a] = sum over rows i of adapter a of dY[i] T[i]^T       (n, rank)
// Both are products over the rows of one adapter of a wide matrix V (X or dY)
// with a narrow one L (U or T, each value the sum of two 16-bit numbers, of
// which f16's second is scaled, see store_t).
//
// A row list per adapter comes first (rows in ascending order).  Then one CTA
// takes 128 columns of V for one adapter: M = the columns, N = the 2 rp columns
// of L, the rows are the k of the MMA, so both operands lie in shared memory
// with k slow ("MN-major").  64 rows make a block: a plain TMA box where the
// list's next 64 rows follow one another, else gathered four rows at a time;
// rows past the end of the list read as zero in both operands, so nothing of
// another adapter's row, not even a NaN, takes part.  A cluster shares the rows
// of a tile and adds its partial sums in order: the result does not depend on
// timing.  Bound by reading X and dY once.
//
// The tensor core cuts its f32 sums off instead of rounding them, an error of
// one sign that grows with the MMAs added into one accumulator.  An accumulator
// therefore takes a few blocks only; the epilogue warps then add it to sums in
// their registers while the next one is filled.  The error then does not grow
// with the rows: sums of one sign over 16 k to 256 k rows are off by 1.1e-6 up to
// rank 32 and 2.2e-6 above (8 and 16 blocks; all blocks of a CTA in one
// accumulator: 5e-6 to 1.7e-4), at the same speed (65,536 rows, rank 128, 1024 +
// 1024 columns, with the products: 505 us, was 505; half the blocks: 508).
#include "lora_sm100.cuh"

namespace cb {
namespace {

constexpr int LIST_THREADS = 1024;

// list[first[a] .. first[a + 1]) = the rows that name adapter a.  A CTA per adapter counts the rows of lower adapters (its
// place in the list) and its own, then writes its own: no CTA waits for another.
__global__ void __launch_bounds__(LIST_THREADS) row_list_kernel(const int32_t *ids, int m, int adapters, int32_t *first, int32_t *list) {
    __shared__ int lower_sum[LIST_THREADS / 32], own_sum[LIST_THREADS / 32];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int a = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lower = 0, own = 0;
    for (int i = threadIdx.x; i < m; i += LIST_THREADS) {
        const int id = ids[i];
        lower += id >= 0 && id < a;
        own += id == a;
    }
    lower = __reduce_add_sync(0xffffffffu, lower);
    own = __reduce_add_sync(0xffffffffu, own);
    if (lane == 0) lower_sum[warp] = lower, own_sum[warp] = own;
    __syncthreads();
    int begin = 0, count = 0;
    for (int w = 0; w < LIST_THREADS / 32; w++) begin += lower_sum[w], count += own_sum[w];
    if (threadIdx.x == 0) {
        first[a] = begin;
        if (a == adapters - 1) first[adapters] = begin + count;
    }
    __syncthreads();
    int at = begin;
    for (int i0 = 0; i0 < m && at < begin + count; i0 += LIST_THREADS) {
        const int i = i0 + int(threadIdx.x);
        const bool mine = i < m && ids[i] == a;
        const uint32_t votes = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) own_sum[warp] = __popc(votes);
        __syncthreads();
        int before = __popc(votes & ((1u << lane) - 1u)), total = 0;
        for (int w = 0; w < LIST_THREADS / 32; w++) {
            if (w < warp) before += own_sum[w];
            total += own_sum[w];
        }
        if (mine) list[at + before] = i;
        at += total;
        __syncthreads();
    }
}

constexpr int GRAD_M = 128, GRAD_ROWS = 64, GRAD_STAGES = 4, GRAD_BUFS = 4;
constexpr uint32_t GRAD_BOX = GRAD_ROWS * 128, GRAD_HEAD = 1024;

// How a tile is cut by rank.  What bounds the kernel beside HBM is the way from L2 to the SMs (some 100 GB/s each): per 64
// rows a tile fetches 8 KB per 64 columns of V and 8 KB per 64 columns of L, so a high rank takes two accumulators of 128
// columns of V (rank 128, 8192 rows, 8192 + 2048 columns: 491 MB with one, 335 MB with two), and the SM to itself.
__host__ __device__ constexpr int grad_halves(int rp) { return rp >= 64 ? 2 : 1; }
__host__ __device__ constexpr int grad_threads(int rp) { return 64 + 128 * grad_halves(rp); }  // an epilogue thread's sums: rp of them, of one column
// Two CTAs share an SM up to rank 64 and have 256 columns of TMEM each: four accumulators of up to 64, or one of 256; above, one
// of 512.  Where there is one, the MMAs wait while it is read: it takes more blocks.
__host__ __device__ constexpr int grad_bufs(int rp) { return rp <= 32 ? GRAD_BUFS : 1; }
__host__ __device__ constexpr int grad_depth(int rp) { return rp <= 32 ? 8 : 16; }
__host__ __device__ constexpr int grad_low_boxes(int rp) { return (2 * rp + 63) / 64; }
constexpr uint32_t grad_ring(int rp) { return (rp == 128 ? 192u : 96u) * 1024; }
constexpr uint32_t grad_smem(int rp) { return 1024 + GRAD_HEAD + grad_ring(rp); }

struct GradMaps {
    CUtensorMap wide[2], wide_rows[2], low[2], low_rows[2];  // [0] for dA: X and U, [1] for dB: dY and T; boxes of 64 rows, and of one
};

struct GradParams {
    float *out[2];
    const int32_t *first, *list;
    int cols[2], tiles[2], m, rank, kc, stages, vec;
    uint32_t stage_bytes, idesc;
    int low_col;      // of L: where the two planes begin
    float low_scale;  // of the second plane's sums
    uint32_t *status;
    int debug;
};

struct GradHead {
    uint64_t full[GRAD_STAGES], empty[GRAD_STAGES], tfull[GRAD_BUFS], tempty[GRAD_BUFS], drain;
    uint32_t tmem, abort;
};

template <int RP>
__global__ void __launch_bounds__(grad_threads(RP), RP == 128 ? 1 : 2) lora_grad_kernel(const __grid_constant__ GradMaps maps, const GradParams p) {
    constexpr int HALVES = grad_halves(RP), THREADS = grad_threads(RP), BUFS = grad_bufs(RP), DEPTH = grad_depth(RP);
    constexpr uint32_t ACC_COLS = 2 * RP * HALVES, TMEM_COLS = BUFS * ACC_COLS;
    static_assert(TMEM_COLS >= 32 && TMEM_COLS <= (RP == 128 ? 512 : 256) && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "TMEM");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    GradHead &h = *reinterpret_cast<GradHead *>(smem_raw + (base - raw));
    const uint32_t ring = base + GRAD_HEAD;
    auto bar = [&](uint64_t &b) { return ptx::smem_u32(&b); };
    volatile uint32_t *abort_flag = &h.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = p.kc > 1 ? ptx::cluster_ctarank() : 0u;
    const int unit = int(blockIdx.x) / p.kc, per = p.tiles[0] + p.tiles[1], a = unit / per;
    int tile = unit - a * per;
    const int job = tile >= p.tiles[0] ? 1 : 0;
    if (job) tile -= p.tiles[0];
    const int c0 = tile * GRAD_M * HALVES, wide_boxes = 2 * HALVES, low_boxes = grad_low_boxes(RP);
    const uint64_t limit = (p.debug & 8) ? 20ull * 1000 * 1000 : WAIT_LIMIT_NS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < GRAD_STAGES; s++) {
            ptx::mbar_init(bar(h.full[s]), 1);
            ptx::mbar_init(bar(h.empty[s]), 1);
        }
        for (int b = 0; b < BUFS; b++) {
            ptx::mbar_init(bar(h.tfull[b]), 1);
            ptx::mbar_init(bar(h.tempty[b]), 4 * HALVES);
        }
        ptx::mbar_init(bar(h.drain), 1);
        h.abort = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<1>(ptx::smem_u32(&h.tmem), TMEM_COLS);
        ptx::tmem_relinquish<1>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&h.tmem);
    ptx::griddep_wait();
    if (threadIdx.x == 0) ptx::griddep_launch_dependents();
    const int begin = p.first[a], count = p.first[a + 1] - begin, blocks = (count + GRAD_ROWS - 1) / GRAD_ROWS;
    const int b0 = int(int64_t(blocks) * rank / p.kc), b1 = int(int64_t(blocks) * (rank + 1) / p.kc);

    if (warp == 0) {
        if (lane == 0) {
            ptx::prefetch_tensormap(&maps.wide[job]);
            ptx::prefetch_tensormap(&maps.low[job]);
        }
        int s = 0;
        uint32_t ph = 0, filled = 0, filled_parity = 0;
        bool ok = !(p.debug & 4);
        const uint32_t bytes = uint32_t(wide_boxes + low_boxes) * GRAD_BOX;
        // Lanes 0-15 hold four rows of a block each, read one block ahead; past the end of the list a row that no matrix has.
        int next[4];
        auto read_rows = [&](int b) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = b * GRAD_ROWS + 4 * (lane & 15) + i;
                next[i] = b < b1 && at < count ? p.list[begin + at] : p.m;
            }
        };
        read_rows(b0);
        for (int b = b0; b < b1 && ok; b++) {
            int row[4];
#pragma unroll
            for (int i = 0; i < 4; i++) row[i] = next[i];
            read_rows(b + 1);
            const int first_row = __shfl_sync(0xffffffffu, row[0], 0), last_row = __shfl_sync(0xffffffffu, row[3], 15);
            const bool run = last_row < p.m && last_row - first_row == GRAD_ROWS - 1;
            ok = wait_bar(bar(h.empty[s]), ph ^ 1u, abort_flag, p.status, WHERE_PRODUCER, uint32_t(s), limit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint32_t dst = ring + uint32_t(s) * p.stage_bytes, full = bar(h.full[s]);
            if (lane == 0) ptx::mbar_arrive_expect_tx(full, bytes);
            __syncwarp();
            if (run) {  // a lane per box
                if (lane < wide_boxes) ptx::tma_load_2d(dst + lane * GRAD_BOX, &maps.wide[job], full, c0 + 64 * lane, first_row);
                else if (lane < wide_boxes + low_boxes) ptx::tma_load_2d(dst + lane * GRAD_BOX, &maps.low[job], full, p.low_col + 64 * (lane - wide_boxes), first_row);
            } else if (lane < 16) {
                for (int x = 0; x < wide_boxes; x++)
                    ptx::tma_gather4(dst + x * GRAD_BOX + 512u * lane, &maps.wide_rows[job], full, c0 + 64 * x, row[0], row[1], row[2], row[3]);
                for (int x = 0; x < low_boxes; x++)
                    ptx::tma_gather4(dst + (wide_boxes + x) * GRAD_BOX + 512u * lane, &maps.low_rows[job], full, p.low_col + 64 * x, row[0], row[1], row[2], row[3]);
            }
            __syncwarp();
            filled |= 1u << s, filled_parity = (filled_parity & ~(1u << s)) | (ph << s);
            if (++s == p.stages) s = 0, ph ^= 1u;
        }
        if (!ok && lane == 0) {  // giving up: let the copies in flight land (bounded)
            const uint64_t t0 = ptx::globaltimer_ns();
            for (int i = 0; i < GRAD_STAGES; i++)
                while ((filled >> i & 1u) && !ptx::mbar_try_wait(bar(h.full[i]), (filled_parity >> i) & 1u))
                    if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        // The whole warp runs the loop and one thread issues: see lora_few_kernel.
        const bool leader = ptx::elect_one();
        int s = 0;
        uint32_t ph = 0;
        bool ok = true, issued = false;
        for (int b = b0; b < b1; b++) {
            const int at = (b - b0) % DEPTH, turn = (b - b0) / DEPTH, buf = turn % BUFS;
            if (at == 0) {  // the epilogue must have read this accumulator
                ok = __all_sync(0xffffffffu, wait_bar(bar(h.tempty[buf]), (uint32_t(turn / BUFS) & 1u) ^ 1u, abort_flag, p.status, WHERE_MMA_TMEM, uint32_t(buf), limit));
                if (!ok) break;
            }
            ok = __all_sync(0xffffffffu, wait_bar(bar(h.full[s]), ph, abort_flag, p.status, WHERE_MMA_FULL, uint32_t(s), limit));
            if (!ok) break;
            ptx::tc_fence_after();
            const uint32_t src = ring + uint32_t(s) * p.stage_bytes;
            const uint64_t low = mn_desc(src + uint32_t(wide_boxes) * GRAD_BOX, GRAD_BOX);
            const uint32_t more = at > 0 ? 1u : 0u, d = tmem + uint32_t(buf) * ACC_COLS;
            if (leader) {
#pragma unroll
                for (int x = 0; x < HALVES; x++) {
                    const uint64_t wide = mn_desc(src + uint32_t(2 * x) * GRAD_BOX, GRAD_BOX);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        ptx::umma_f16<1>(d + uint32_t(2 * x * RP), wide + MN_K_STEP * j, low + MN_K_STEP * j, p.idesc, j > 0 ? 1u : more);
                }
                ptx::umma_commit<1>(bar(h.empty[s]));
                if (at == DEPTH - 1 || b + 1 == b1) ptx::umma_commit<1>(bar(h.tfull[buf]));
            }
            __syncwarp();
            issued = true;
            if (++s == p.stages) s = 0, ph ^= 1u;
        }
        if (leader && !ok && issued) {
            ptx::umma_commit<1>(bar(h.drain));
            const uint64_t t0 = ptx::globaltimer_ns();
            while (!ptx::mbar_try_wait(bar(h.drain), 0u))
                if (ptx::globaltimer_ns() - t0 > WAIT_LIMIT_NS / 4) break;
        }
        __syncwarp();
    } else {
        // A thread holds the sums of one column of V: row 32 q + lane of accumulator half x.
        const int q = warp & 3, x = HALVES == 1 ? 0 : (warp - 2) >> 2;
        float sum[RP] = {};
        bool ok = true;
        for (int b = b0, turn = 0; b < b1; b += DEPTH, turn++) {
            const int buf = turn % BUFS;
            ok = __all_sync(0xffffffffu, wait_bar(bar(h.tfull[buf]), uint32_t(turn / BUFS) & 1u, abort_flag, p.status, WHERE_EPILOGUE, uint32_t(buf), limit));
            if (!ok) break;
            ptx::tc_fence_after();
            // Columns j and RP + j belong to the two numbers of value j: their sum is the gradient's part.
            const uint32_t from = tmem + (uint32_t(32 * q) << 16) + uint32_t(buf) * ACC_COLS + uint32_t(2 * x * RP);
#pragma unroll
            for (int c = 0; c < RP; c += 16) {
                uint32_t hi[16], lo[16];
                ptx::tmem_ld_32x16(from + uint32_t(c), hi);
                ptx::tmem_ld_32x16(from + uint32_t(RP + c), lo);
                ptx::tmem_ld_wait_all();
                ptx::pin16(hi);
                ptx::pin16(lo);
#pragma unroll
                for (int j = 0; j < 16; j++) sum[c + j] += fmaf(__uint_as_float(lo[j]), p.low_scale, __uint_as_float(hi[j]));
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(h.tempty[buf]));
        }
        if (ok) {  // the ring is idle: every block has been multiplied
            ptx::fence_proxy_async_shared();
            const uint32_t dst = ring + uint32_t(GRAD_M * x + 32 * q + lane) * uint32_t(RP + 4) * 4u;
#pragma unroll
            for (int c = 0; c < RP; c += 4)
                ptx::st_shared_v4(dst + uint32_t(c) * 4u, __float_as_uint(sum[c]), __float_as_uint(sum[c + 1]), __float_as_uint(sum[c + 2]), __float_as_uint(sum[c + 3]));
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
        const uint32_t pitch = uint32_t(RP + 4) * 4u;
        // Four ranks of one column of V per step.  Neighbouring threads write neighbouring addresses: of dA the columns, of dB
        // the ranks, 16 bytes at once.
        const int cols = p.cols[job], columns = GRAD_M * HALVES, wide = min(columns, cols - c0), quads = p.rank / 4, items = columns * quads;
        float *out = p.out[job] + int64_t(a) * p.rank * cols;
        const Divider by_quads(quads);
        const int shift = __ffs(columns) - 1;  // a power of two
        auto column = [&](int i) { return job ? by_quads(i) : i & (columns - 1); };
        auto first_rank = [&](int i) { return 4 * (job ? i - by_quads(i) * quads : i >> shift); };
        cluster_sums<2>(
            items, int(rank), p.kc, THREADS, [&](int i) { return ring + uint32_t(column(i)) * pitch + uint32_t(first_rank(i)) * 4u; },
            [&](int i, const float4 &v) {
                const int c = column(i), j = first_rank(i);
                if (c >= wide) return;
                if (job) {
                    float *to = out + int64_t(c0 + c) * p.rank + j;
                    if (p.vec) *reinterpret_cast<float4 *>(to) = v;
                    else to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
                } else {
                    float *to = out + int64_t(j) * cols + c0 + c;
                    to[0] = v.x, to[cols] = v.y, to[2 * int64_t(cols)] = v.z, to[3 * int64_t(cols)] = v.w;
                }
            });
    }
    __syncthreads();
    if (p.kc > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, TMEM_COLS);
}

}  // namespace

cute_b200_status lora_row_lists(const int32_t *ids, int m, int adapters, int32_t *first, int32_t *list, cudaStream_t stream) {
    return launch_dependent(row_list_kernel, dim3(unsigned(adapters)), LIST_THREADS, 0, 1, stream, ids, m, adapters, first, list);
}

cute_b200_status lora_grads(const LoraGrads &g, bool bf16, int debug, const DeviceState &dev, cudaStream_t stream) {
    GradParams p = {};
    GradMaps maps;
    const int low_cols = t_planes(bf16) * g.rp;
    for (int i = 0; i < 2; i++) {
        p.out[i] = g.out[i];
        p.cols[i] = g.cols[i];
        p.tiles[i] = (g.cols[i] + GRAD_M * grad_halves(g.rp) - 1) / (GRAD_M * grad_halves(g.rp));
        const uint64_t wide = reinterpret_cast<uint64_t>(g.wide[i]), low = reinterpret_cast<uint64_t>(g.low[i]);
        CB_TRY(rows_tensor_map(&maps.wide[i], wide, bf16, g.m, g.cols[i], g.pitch[i], GRAD_ROWS));
        CB_TRY(rows_tensor_map(&maps.wide_rows[i], wide, bf16, g.m, g.cols[i], g.pitch[i], 1));
        CB_TRY(rows_tensor_map(&maps.low[i], low, bf16, g.m, low_cols, low_cols, GRAD_ROWS));
        CB_TRY(rows_tensor_map(&maps.low_rows[i], low, bf16, g.m, low_cols, low_cols, 1));
    }
    p.first = g.first, p.list = g.list;
    p.vec = reinterpret_cast<uint64_t>(g.out[1]) % 16 == 0;
    p.m = g.m, p.rank = g.rank;
    p.stage_bytes = uint32_t(2 * grad_halves(g.rp) + grad_low_boxes(g.rp)) * GRAD_BOX;
    p.stages = int(grad_ring(g.rp) / p.stage_bytes);
    if (p.stages > GRAD_STAGES) p.stages = GRAD_STAGES;
    p.idesc = make_idesc(bf16, GRAD_M, 2 * g.rp) | IDESC_A_MN | IDESC_B_MN;
    p.low_col = t_hi(g.rp, bf16);
    p.low_scale = bf16 ? 1.0f : 1.0f / LOW_SCALE;
    p.status = dev.status_word;
    p.debug = debug;
    // The rows of a tile are shared by a cluster of kc CTAs: the least time for whole waves of CTAs, each the blocks of an
    // adapter of average size and some twelve blocks' time to start, add up and store.
    const int64_t units = int64_t(p.tiles[0] + p.tiles[1]) * g.adapters, slots = int64_t(dev.sm_count) * (g.rp == 128 ? 1 : 2);
    const int blocks = int((int64_t(g.m) + int64_t(GRAD_ROWS) * g.adapters - 1) / (int64_t(GRAD_ROWS) * g.adapters));
    p.kc = 1;
    double best = 1e300;
    for (int kc = 1; kc <= 8 && kc <= blocks; kc++) {
        const double waves = double((units * kc + slots - 1) / slots), t = waves * ((blocks + kc - 1) / kc + 12.0);
        if (t < best) best = t, p.kc = kc;
    }
    if (units * p.kc > 0x7fffffff) return fail(CUTE_B200_ERR_INVALID_ARGUMENT, "lora_tn_backward: the adapters are too large");
    auto launch = [&](auto kernel) { return launch_dependent(kernel, dim3(unsigned(units * p.kc)), grad_threads(g.rp), grad_smem(g.rp), p.kc, stream, maps, p); };
    if (g.rp == 16) return launch(lora_grad_kernel<16>);
    if (g.rp == 32) return launch(lora_grad_kernel<32>);
    if (g.rp == 64) return launch(lora_grad_kernel<64>);
    return launch(lora_grad_kernel<128>);
}

cute_b200_status lora_grad_init() {
    CB_CUDA(cudaFuncSetAttribute(lora_grad_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, grad_smem(16)));
    CB_CUDA(cudaFuncSetAttribute(lora_grad_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, grad_smem(32)));
    CB_CUDA(cudaFuncSetAttribute(lora_grad_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, grad_smem(64)));
    CB_CUDA(cudaFuncSetAttribute(lora_grad_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, grad_smem(128)));
    return CUTE_B200_OK;
}

}  // namespace cb
