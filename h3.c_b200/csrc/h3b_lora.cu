/* Low-rank adapters of many requests beside a shared projection:
 *   out[r] = bf16( x[r].W^T + bias + scale[a] (x[r].down[a]^T).up[a]^T ),  a = row_adapter[r].
 *
 * On the tensor cores a call is two launches. h3b_lora_down_tc finds the adapters that occur in every tile of rows
 * (its entries, h3b_lora.cuh) and computes their low-rank rows t; the projection then takes t and up as
 * further K blocks of the tile's accumulation, so the adapters cost no pass over the output and there is
 * one rounding. The projection is launched as a programmatic dependent: it streams its own K blocks while
 * the first kernel finishes and waits for t only behind them. Many rows: the 128- and 256-row tiles of
 * h3b_gemm.cu. Few rows: h3b_lora_rows, which streams the weight through the M side of the instruction.
 *
 * Kernels that take any shape and alignment (one F32 fmaf chain per sum): h3b_lora_down_simt computes
 * the low-rank row t[r] = scale[a] x[r].down[a]^T once, h3b_lora_simt the projection with t[r].up[a]^T
 * added to every output before its one rounding (18 TFLOP/s: 6,400 rows, 5,376 -> 21,504, rank 64 83.8 ms; on the
 * tensor cores 1.13, of which the bare projection is 0.95).
 */
#include "h3b_common.cuh"
#include "h3b_lora.cuh"
#include "h3b_sm100.cuh"

#include <cstdlib>

namespace {

/* round to nearest even; NaN stays NaN (h3b_narrow's integer formula turns some into zeros) */
__device__ __forceinline__ uint16_t to_bf16(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }

/* One warp per (row, rank index): t[row][j] = scale[a] * x[row] . down[a][j], F32; 0 without an adapter. */
__global__ void __launch_bounds__(256)
h3b_lora_down_simt(const uint16_t *x, const uint16_t *down, const float *scale, const uint32_t *row_adapter,
                   float *t, uint32_t rows, uint32_t k, uint32_t adapters, uint32_t rank) {
    const size_t unit = (size_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (unit >= size_t(rows) * rank) return;
    const uint32_t lane = threadIdx.x & 31, row = uint32_t(unit / rank), j = uint32_t(unit % rank);
    const uint32_t a = row_adapter ? row_adapter[row] : 0;
    float sum = 0.0f;
    if (a < adapters) {
        const uint16_t *xr = x + size_t(row) * k, *d = down + (size_t(a) * rank + j) * k;
        for (uint32_t i = lane; i < k; i += 32) sum = fmaf(h3b_widen(xr[i]), h3b_widen(d[i]), sum);
        sum = h3b_warp_sum(sum) * (scale ? scale[a] : 1.0f);
    }
    if (lane == 0) t[unit] = sum;
}

/* 64 x 64 tile, 16 x 16 threads, 4 x 4 outputs per thread: the projection, then the row's own adapter. */
__global__ void __launch_bounds__(256)
h3b_lora_simt(const uint16_t *x, const uint16_t *w, const uint16_t *bias, const uint16_t *up, const float *t,
              const uint32_t *row_adapter, uint16_t *out, uint32_t rows, uint32_t k, uint32_t n,
              uint32_t adapters, uint32_t rank) {
    __shared__ float xs[16][65];
    __shared__ float ws[16][65];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const uint32_t columns = uint32_t((uint64_t(n) + 63) / 64), row0 = blockIdx.x / columns * 64, col0 = blockIdx.x % columns * 64;
    float acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t col = col0 + tx + 16 * j;
        const float start = bias && col < n ? h3b_widen(bias[col]) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i][j] = start;
    }
    for (uint32_t k0 = 0; k0 < k; k0 += 16) {
        for (int e = threadIdx.x; e < 64 * 16; e += 256) {
            const int r = e >> 4, kk = e & 15;
            const uint32_t gr = row0 + r, gc = col0 + r, gk = k0 + kk;
            xs[kk][r] = gr < rows && gk < k ? h3b_widen(x[size_t(gr) * k + gk]) : 0.0f;
            ws[kk][r] = gc < n && gk < k ? h3b_widen(w[size_t(gc) * k + gk]) : 0.0f;
        }
        __syncthreads();
        const uint32_t limit = min(16u, k - k0);
        for (uint32_t kk = 0; kk < limit; kk++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = fmaf(xs[kk][ty + 16 * i], ws[kk][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t row = row0 + ty + 16 * i;
        if (row >= rows) continue;
        const uint32_t a = row_adapter ? row_adapter[row] : 0;
        const float *tr = t + size_t(row) * rank;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t col = col0 + tx + 16 * j;
            if (col >= n) continue;
            float v = acc[i][j];
            if (a < adapters) {
                const uint16_t *u = up + (size_t(a) * n + col) * rank;
                for (uint32_t q = 0; q < rank; q++) v = fmaf(tr[q], h3b_widen(u[q]), v);
            }
            out[size_t(row) * n + col] = to_bf16(v);
        }
    }
}

/* ------------------------------------------------------------- tensor cores */

constexpr int LR_M = 128;                    /* rows of an instruction: x rows (down) or weight rows (projection) */
constexpr int LR_K = 64;                     /* one 128-byte swizzle line */
constexpr int LR_A_BYTES = LR_M * LR_K * 2;
constexpr int LR_THREADS = 192;              /* TMA, MMA, 4 epilogue warps */
static_assert(LR_THREADS == int(H3B_LORA_THREADS), "the repair of adapter tiles is written for it");
constexpr uint32_t LR_SPLIT = 8;             /* CTAs of a cluster, at most */
constexpr int LR_STAGES = 8;                 /* barriers laid out; a launch uses `stages` of them */
constexpr int LR_BAR_BYTES = 256;
constexpr uint32_t kMaxRank = 256, kMaxAdapters = 1024;

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

struct RingArgs {
    int *status;
    long long wait_cycles;
    uint32_t stages, stage_bytes, tmem_columns;
};

/* barriers, the pipeline's shared memory and the accumulator of a CTA of the two kernels below */
struct Ring {
    uint32_t stage0, full, empty, done, info, holder;
    volatile int *stop;
};
/* addresses, and (thread 0) the barriers: `arrivals` per full barrier */
__device__ __forceinline__ Ring ring_begin(const RingArgs &args, uint8_t *raw, int *stop_flag, uint32_t arrivals) {
    Ring r;
    r.stage0 = (smem_u32(raw) + 1023u) & ~1023u;
    r.full = r.stage0 + args.stages * args.stage_bytes;
    r.empty = r.full + 8 * LR_STAGES;
    r.done = r.empty + 8 * LR_STAGES;
    r.info = r.done + 8;
    r.holder = r.info + 8;
    r.stop = stop_flag;
    if (threadIdx.x == 0) {
        *stop_flag = 0;
        for (uint32_t i = 0; i < args.stages; i++) {
            mbar_init(r.full + 8 * i, arrivals);
            mbar_init(r.empty + 8 * i, 1);
        }
        mbar_init(r.done, 1);
        mbar_init(r.info, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x >> 5 == 1) tmem_alloc(r.holder, args.tmem_columns);
    return r;
}
/* behind the block barrier that follows ring_begin: the accumulator's address */
__device__ __forceinline__ uint32_t ring_tmem(const Ring &r) {
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(r.holder));
    return tmem;
}
/* Behind the last use of the accumulator: tensor memory goes back. After a wait that ran out: the status, and time for
 * copies and products that may be in flight to land first. */
__device__ __forceinline__ void ring_close(const RingArgs &args, const Ring &r, uint32_t tmem) {
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*r.stop) {
        if (threadIdx.x == 0) atomicMax(args.status, int(H3B_STATUS_GEMM_TIMEOUT));
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
        __syncthreads();
    }
    if (threadIdx.x >> 5 == 1) {
        tc_fence_after();
        tmem_free(tmem, args.tmem_columns);
    }
    __syncwarp();
}

/* The entries of a tile: the adapters that occur among its rows, ascending. Every CTA finds them for itself. */
struct Entries {
    uint32_t present[kMaxAdapters / 32], before[kMaxAdapters / 32];
    uint16_t adapter[256];          /* of an entry */
    uint32_t without;
};
constexpr uint32_t kNone = 0xffffffffu;
__device__ __forceinline__ uint32_t adapter_of(const h3b_lora_task &task, uint32_t row) {
    const uint32_t a = row >= task.rows ? kNone : task.row_adapter ? task.row_adapter[row] : 0;
    return a < task.adapters ? a : kNone;
}
/* A thread's rows of the tile, threadIdx.x and the one blockDim.x on: with 192 threads or more two loads cover any
 * tile. Asked for first of all and used behind the set-up: one after the other, the row's adapter, the tile's
 * second rows and the scale cost three memory latencies (3.5 us of a kernel of 13 us). */
struct TileRows {
    uint32_t a[2], rows;        /* rows: how many of the two exist */
};
__device__ __forceinline__ TileRows load_rows(const h3b_lora_task &task, uint32_t tile) {
    TileRows r = {{kNone, kNone}, 0};
#pragma unroll
    for (uint32_t i = 0; i < 2; i++) {
        const uint32_t at = threadIdx.x + i * blockDim.x;
        if (at < task.tile_rows && tile * task.tile_rows + at < task.rows) {
            r.a[i] = adapter_of(task, tile * task.tile_rows + at);
            r.rows = i + 1;
        }
    }
    return r;
}
/* all threads; returns the number of entries */
__device__ __forceinline__ uint32_t find_entries(Entries &s, const TileRows &rows) {
    const uint32_t lane = threadIdx.x & 31;
    if (threadIdx.x < kMaxAdapters / 32) s.present[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.without = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2; i++) {
        if (i >= rows.rows) break;
        if (rows.a[i] != kNone) atomicOr(&s.present[rows.a[i] >> 5], 1u << (rows.a[i] & 31));
        else s.without = 1;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        uint32_t mine = s.present[lane], sum = __popc(mine);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= uint32_t(o)) sum += v;
        }
        uint32_t at = sum - __popc(mine);
        s.before[lane] = at;
        for (; mine; mine &= mine - 1) s.adapter[at++] = uint16_t(lane * 32 + __ffs(mine) - 1);
    }
    __syncthreads();
    return s.before[31] + __popc(s.present[31]);
}
__device__ __forceinline__ uint32_t entry_of(const Entries &s, uint32_t a) {
    return a == kNone ? kNone : s.before[a >> 5] + __popc(s.present[a >> 5] & ((1u << (a & 31)) - 1));
}
__device__ __forceinline__ void publish_entries(const Entries &s, const h3b_lora_task &task, uint32_t tile, uint32_t count) {
    for (uint32_t e = threadIdx.x; e < count; e += blockDim.x) task.entries[size_t(tile) * task.max_entries + e] = s.adapter[e];
    if (threadIdx.x == 0) task.counts[tile] = count | (count > 1 || (count && s.without) ? H3B_LORA_MIXED : 0u);
}

/* t of one 128-row block for up to `group` entries of its tile: x block . [down of the entries]^T, K split over
 * the CTAs of a cluster, partial sums joined through distributed shared memory in rank order. Every row
 * then takes its own adapter's columns. Bound by reading x once (6,400 x 5,376: 69 MB, 10.5 us). The x
 * copies of the first stages go out before the entries are known. */
struct DownArgs {
    h3b_lora_task task;
    RingArgs ring;
    uint32_t k_blocks, rank16, group;        /* columns per entry (rank rounded up to 16); entries at a time */
};
__global__ void __launch_bounds__(LR_THREADS)
h3b_lora_down_tc(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_down,
                 const __grid_constant__ DownArgs args) {
    extern __shared__ uint8_t raw_smem[];
    __shared__ int stop_flag;
    __shared__ Entries found;
    __shared__ uint32_t own[LR_M];           /* entry of a row of the block */
    __shared__ float own_scale[LR_M];
    const h3b_lora_task &task = args.task;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = gridDim.x, part = blockIdx.x, row0 = blockIdx.y * LR_M, tile = row0 / task.tile_rows;
    const uint32_t kb0 = part * args.k_blocks / split, kb1 = (part + 1) * args.k_blocks / split;
    if (threadIdx.x == 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_down) : "memory");
    /* Tensor memory behind the wait for what is in front, and the launch behind let go behind that: nobody ever waits for
     * columns of a CTA that waits for it. */
    if (task.first) h3b_wait_for_launch();
    Ring ring = ring_begin(args.ring, raw_smem, &stop_flag, 2);
    if (warp == 1) h3b_let_next_launch();
    const TileRows rows = load_rows(task, tile);
    const uint32_t own_a = threadIdx.x < LR_M ? adapter_of(task, row0 + threadIdx.x) : kNone;
    const float own_s = own_a != kNone && task.scale ? task.scale[own_a] : 1.0f;
    const uint32_t early = blockIdx.z == 0 ? min(args.ring.stages, kb1 - kb0) : 0;
    if (threadIdx.x == 0)
        for (uint32_t i = 0; i < early; i++) {
            mbar_expect_tx(ring.full + 8 * i, LR_A_BYTES);
            tma_load_2d(ring.stage0 + i * args.ring.stage_bytes, &map_x, ring.full + 8 * i, int((kb0 + i) * LR_K), int(row0));
        }
    const uint32_t count = find_entries(found, rows);
    if (blockIdx.z == 0 && part == 0 && row0 == tile * task.tile_rows) publish_entries(found, task, tile, count);
    if (threadIdx.x < LR_M) own[threadIdx.x] = entry_of(found, own_a);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ring_tmem(ring);
    if (count == 0 && threadIdx.x == 0)
        /* nothing to compute; copies that went out have to land before the CTA leaves */
        for (uint32_t i = 0; i < early; i++) {
            mbar_arrive(ring.full + 8 * i);
            mbar_wait(ring.full + 8 * i, 0, ring.stop, args.ring.wait_cycles);
        }
    /* Groups of entries blockIdx.z, blockIdx.z + gridDim.z, ...: as many turns in every CTA of the cluster, whatever
     * any of them runs into. Stages and phases count on in the two roles that use them. */
    uint32_t stage = 0, phase = 0, turn = 0;
    for (uint32_t e0 = blockIdx.z * args.group; e0 < count; e0 += gridDim.z * args.group, turn++) {
        const uint32_t e1 = min(count, e0 + args.group), columns = (e1 - e0) * args.rank16;
        if (warp == 0) {
            if (lane == 0) {
                for (uint32_t kb = kb0; kb < kb1; kb++) {
                    const uint32_t bar = ring.full + 8 * stage, dst = ring.stage0 + stage * args.ring.stage_bytes;
                    if (turn || kb - kb0 >= early) {
                        if (!mbar_wait(ring.empty + 8 * stage, phase ^ 1, ring.stop, args.ring.wait_cycles)) break;
                        mbar_expect_tx(bar, LR_A_BYTES);
                        tma_load_2d(dst, &map_x, bar, int(kb * LR_K), int(row0));
                    }
                    mbar_expect_tx(bar, columns * LR_K * 2);
                    for (uint32_t e = e0; e < e1; e++)
                        tma_load_2d(dst + LR_A_BYTES + (e - e0) * args.rank16 * LR_K * 2, &map_down, bar, int(kb * LR_K),
                                    int(found.adapter[e] * task.rank));
                    if (++stage == args.ring.stages) { stage = 0; phase ^= 1; }
                }
            }
        } else if (warp == 1) {
            const uint32_t leader = lane == 0, idesc = instruction_desc(LR_M, int(columns));
            bool alive = true;
            for (uint32_t kb = kb0; kb < kb1; kb++) {
                alive = __all_sync(0xffffffffu, mbar_wait(ring.full + 8 * stage, phase, ring.stop, args.ring.wait_cycles));
                if (!alive) break;
                tc_fence_after();
                const uint32_t a_lo = desc_lo_kmajor(ring.stage0 + stage * args.ring.stage_bytes);
                const uint32_t b_lo = a_lo + (LR_A_BYTES >> 4);
                if (kb == kb0) umma_ss<false>(tmem, a_lo, b_lo, idesc, leader);
                else umma_ss<true>(tmem, a_lo, b_lo, idesc, leader);
#pragma unroll
                for (int k = 1; k < LR_K / 16; k++) umma_ss<true>(tmem, a_lo + 2 * k, b_lo + 2 * k, idesc, leader);
                umma_commit_if(ring.empty + 8 * stage, leader);
                if (++stage == args.ring.stages) { stage = 0; phase ^= 1; }
            }
            if (alive) umma_commit_if(ring.done, leader);
        } else {
            /* accumulator -> this CTA's shared memory, [row][columns] F32 with 16-byte pieces XOR-swizzled by row
             * (every copy and product of this CTA is complete, the stages are free) */
            const uint32_t quarter = warp & 3, row = quarter * 32 + lane;
            if (__all_sync(0xffffffffu, mbar_wait(ring.done, turn & 1u, ring.stop, args.ring.wait_cycles))) {
                tc_fence_after();
                for (uint32_t c = 0; c < columns; c += 16) {
                    uint32_t v[16];
                    asm volatile(
                        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                        : "r"(tmem + ((quarter * 32) << 16) + c) : "memory");
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) {
                        const uint32_t piece = (c / 4 + i) ^ (row & 3);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(ring.stage0 + (row * columns + piece * 4) * 4),
                                     "r"(v[4 * i]), "r"(v[4 * i + 1]), "r"(v[4 * i + 2]), "r"(v[4 * i + 3]) : "memory");
                    }
                }
                tc_fence_before();
            }
        }
        if (threadIdx.x < LR_M) own_scale[threadIdx.x] = own_s;
        __syncwarp();
        cluster_sync_all();
        if (!*ring.stop) {
            /* rows part, part + split, ...: the row's own columns of all CTAs, scaled and rounded; zeros for the
             * entries that are not its own */
            const uint32_t mine = (LR_M - part + split - 1) / split, pieces = task.rank8 / 4, log2 = 32 - __clz(pieces - 1);
            uint16_t *t_rows = task.t + (size_t(tile) * task.max_entries * task.tile_rows + row0 % task.tile_rows) * task.rank8;
            for (uint32_t i = threadIdx.x; i < mine << log2; i += LR_THREADS) {
                const uint32_t j = (i & ((1u << log2) - 1)) * 4, r = part + (i >> log2) * split;
                if (j >= task.rank8 || row0 + r >= task.rows) continue;
                const uint32_t e_own = own[r];
                uint2 value = make_uint2(0, 0);
                if (e_own - e0 < e1 - e0) {
                    const uint32_t c = (e_own - e0) * args.rank16 + j;
                    const uint32_t at = ring.stage0 + (r * columns + ((c / 4) ^ (r & 3)) * 4) * 4;
                    float4 x[LR_SPLIT], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (uint32_t p = 0; p < LR_SPLIT; p++)      /* all on the way before the first is used */
                        if (p < split)
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(x[p].x), "=f"(x[p].y), "=f"(x[p].z), "=f"(x[p].w) : "r"(cluster_map(at, p)) : "memory");
#pragma unroll
                    for (uint32_t p = 0; p < LR_SPLIT; p++)
                        if (p < split) { v.x += x[p].x; v.y += x[p].y; v.z += x[p].z; v.w += x[p].w; }
                    const float s = own_scale[r];
                    value = make_uint2(pack_bf16(j < task.rank ? v.x * s : 0.0f, j + 1 < task.rank ? v.y * s : 0.0f),
                                       pack_bf16(j + 2 < task.rank ? v.z * s : 0.0f, j + 3 < task.rank ? v.w * s : 0.0f));
                }
                for (uint32_t e = e0; e < e1; e++)
                    *reinterpret_cast<uint2 *>(t_rows + (size_t(e) * task.tile_rows + r) * task.rank8 + j) = e == e_own ? value : make_uint2(0, 0);
            }
        }
        /* nobody leaves, or loads over its shared memory, while that may be read */
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        cluster_sync_all();
        tc_fence_after();
    }
    ring_close(args.ring, ring, tmem);
    h3b_wait_for_launch();               /* the padded up rows, where a launch in front writes them: done before this one is */
}

/* t of a call of few rows (one tile): a CTA per row and pair of rank indices, four warps to each sum, so that the
 * kernel costs little more than one memory latency; the tensor-core form above takes 8 us for its set-up,
 * copies and cluster barriers whatever the size (one row, rank 16, k = 7,168). */
constexpr int LF_SUMS = 2, LF_WARPS = 4 * LF_SUMS;
__global__ void __launch_bounds__(32 * LF_WARPS)
h3b_lora_down_few(const __grid_constant__ h3b_lora_task task) {
    __shared__ Entries found;
    __shared__ float part[LF_WARPS];
    if (task.first) h3b_wait_for_launch();
    h3b_let_next_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t row = blockIdx.x, j = blockIdx.y * LF_SUMS + warp / 4, a = adapter_of(task, row);
    const TileRows rows = load_rows(task, 0);
    const float s = a != kNone && task.scale ? task.scale[a] : 1.0f;
    float sum = 0.0f;
    if (a != kNone && j < task.rank) {
        const uint4 *x = reinterpret_cast<const uint4 *>(task.x + size_t(row) * task.k);
        const uint4 *d = reinterpret_cast<const uint4 *>(task.down + (size_t(a) * task.rank + j) * task.k);
        float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (uint32_t i = (warp & 3) * 32 + lane; i < task.k / 8; i += 128) {
            const uint4 u = x[i], v = d[i];
            const uint32_t us[4] = {u.x, u.y, u.z, u.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int q = 0; q < 4; q++) sums[q] = fmaf(h3b_hi(us[q]), h3b_hi(vs[q]), fmaf(h3b_lo(us[q]), h3b_lo(vs[q]), sums[q]));
        }
        sum = h3b_warp_sum((sums[0] + sums[1]) + (sums[2] + sums[3]));
    }
    if (lane == 0) part[warp] = sum;
    const uint32_t count = find_entries(found, rows);          /* has block barriers */
    if (blockIdx.x == 0 && blockIdx.y == 0) publish_entries(found, task, 0, count);
    const uint32_t mine = entry_of(found, a);
    for (uint32_t i = threadIdx.x; i < count * LF_SUMS; i += 32 * LF_WARPS) {
        const uint32_t e = i / LF_SUMS, q = i % LF_SUMS, jj = blockIdx.y * LF_SUMS + q;
        const float v = ((part[4 * q] + part[4 * q + 1]) + (part[4 * q + 2] + part[4 * q + 3])) * s;
        task.t[(size_t(e) * task.tile_rows + row) * task.rank8 + jj] = e == mine && jj < task.rank ? to_bf16(v) : 0;
    }
    h3b_wait_for_launch();
}

/* The projection of few rows: D[weight row][x row] = W.x^T for 128 weight rows and the up to 128 rows of the call, the
 * weight streamed once through the M side of the instruction. K is split over the CTAs of a cluster so
 * that every SM pulls on the weight (42 weight tiles of n = 5,376 would leave 106 SMs idle); the entries'
 * blocks are dealt out over the CTAs of the cluster. Partial sums are joined through distributed shared memory in rank order.
 * Bound by the weight's bytes: one row, 7,168 -> 5,376, 77 MB in 16 us. */
struct RowsArgs {
    h3b_lora_task task;
    RingArgs ring;
    uint32_t k_blocks, blocks;               /* blocks: K blocks of an entry */
};
__global__ void __launch_bounds__(LR_THREADS)
h3b_lora_rows(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
              const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_t,
              const __grid_constant__ RowsArgs args) {
    extern __shared__ uint8_t raw_smem[];
    __shared__ int stop_flag;
    const h3b_lora_task &task = args.task;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = gridDim.x, part = blockIdx.x, w0 = blockIdx.y * LR_M;
    const uint32_t kb0 = part * args.k_blocks / split, kb1 = (part + 1) * args.k_blocks / split;
    const uint32_t b_bytes = task.tile_rows * LR_K * 2;
    Ring ring = ring_begin(args.ring, raw_smem, &stop_flag, 1);
    __shared__ uint32_t entries, rows_differ;
    __shared__ uint16_t adapter[LR_M];
    /* the join's threads (the epilogue's warps) have two weight rows of every second of their CTA's x rows */
    const uint32_t col = w0 + 2 * (threadIdx.x & 63);
    uint32_t bias = 0;
    if (warp >= 2 && task.bias && col < task.n) bias = *reinterpret_cast<const uint32_t *>(task.bias + col);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ring_tmem(ring);
    /* The entries' blocks are dealt out over the CTAs of the cluster, behind their own: entry e to part e % split.
     * Which they are is read by a warp that is idle meanwhile: count, adapter and copy in a row would cost the
     * end of the stream three latencies. */
    auto extra_blocks = [&] { return (entries + split - 1 - part) / split * args.blocks; };
    if (warp == 0) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            auto next_stage = [&]() -> uint32_t {
                alive = mbar_wait(ring.empty + 8 * stage, phase ^ 1, ring.stop, args.ring.wait_cycles);
                if (alive) mbar_expect_tx(ring.full + 8 * stage, LR_A_BYTES + b_bytes);
                return ring.stage0 + stage * args.ring.stage_bytes;
            };
            auto advance = [&] { if (++stage == args.ring.stages) { stage = 0; phase ^= 1; } };
            for (uint32_t kb = kb0; alive && kb < kb1; kb++) {
                const uint32_t dst = next_stage(), bar = ring.full + 8 * stage;
                if (!alive) break;
                tma_load_2d(dst, &map_w, bar, int(kb * LR_K), int(w0));
                tma_load_2d(dst + LR_A_BYTES, &map_x, bar, int(kb * LR_K), 0);
                advance();
            }
            alive = alive && mbar_wait(ring.info, 0, ring.stop, args.ring.wait_cycles);
            const uint32_t extra = alive ? extra_blocks() : 0;
            for (uint32_t i = 0; alive && i < extra; i++) {
                const uint32_t e = part + i / args.blocks * split, c = i % args.blocks * LR_K;
                const uint32_t dst = next_stage(), bar = ring.full + 8 * stage;
                if (!alive) break;
                tma_load_3d(dst, &map_up, bar, int(c), int(w0), int(adapter[e]));
                tma_load_2d(dst + LR_A_BYTES, &map_t, bar, int(c), int(e * task.tile_rows));
                advance();
            }
        }
    } else if (warp == 1) {
        const uint32_t leader = lane == 0, idesc = instruction_desc(LR_M, int(task.tile_rows));
        uint32_t stage = 0, phase = 0, blocks = kb1 - kb0;
        bool alive = true;
        for (uint32_t i = 0; alive && i <= blocks; i++) {
            if (i == kb1 - kb0) {      /* how many there are in all is known by now, or soon */
                alive = __all_sync(0xffffffffu, mbar_wait(ring.info, 0, ring.stop, args.ring.wait_cycles));
                if (alive) blocks += extra_blocks();
            }
            if (!alive || i == blocks) break;
            alive = __all_sync(0xffffffffu, mbar_wait(ring.full + 8 * stage, phase, ring.stop, args.ring.wait_cycles));
            if (!alive) break;
            tc_fence_after();
            const uint32_t a_lo = desc_lo_kmajor(ring.stage0 + stage * args.ring.stage_bytes);
            const uint32_t b_lo = a_lo + (LR_A_BYTES >> 4), c = i < kb1 - kb0 ? 0 : (i - (kb1 - kb0)) % args.blocks * LR_K;
            const uint32_t k16 = i < kb1 - kb0 ? LR_K / 16 : (min(task.rank - c, uint32_t(LR_K)) + 15) / 16;
            for (uint32_t k = 0; k < k16; k++) {
                if (i == 0 && k == 0) umma_ss<false>(tmem, a_lo, b_lo, idesc, leader);
                else umma_ss<true>(tmem, a_lo + 2 * k, b_lo + 2 * k, idesc, leader);
            }
            umma_commit_if(ring.empty + 8 * stage, leader);
            if (++stage == args.ring.stages) { stage = 0; phase ^= 1; }
        }
        if (alive) umma_commit_if(ring.done, leader);
    } else {
        if (warp == 2) {
            /* what the launch in front found */
            h3b_wait_for_launch();
            const uint32_t found = task.counts[0], count = found & ~H3B_LORA_MIXED;
            for (uint32_t e = lane; e < count; e += 32) adapter[e] = uint16_t(task.entries[e]);
            if (lane == 0) {
                entries = count;
                rows_differ = found & H3B_LORA_MIXED;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(ring.info);
        }
        /* accumulator -> shared memory [x row][128 weight rows] F32 */
        const uint32_t quarter = warp & 3;
        if (__all_sync(0xffffffffu, mbar_wait(ring.done, 0, ring.stop, args.ring.wait_cycles))) {
            tc_fence_after();
            for (uint32_t c = 0; c < task.rows; c += 16) {
                uint32_t v[16];
                asm volatile(
                    "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                    : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                      "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                    : "r"(tmem + ((quarter * 32) << 16) + c) : "memory");
                tmem_ld_wait();
#pragma unroll
                for (uint32_t i = 0; i < 16; i++)
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(ring.stage0 + ((c + i) * LR_M + quarter * 32 + lane) * 4), "r"(v[i]) : "memory");
            }
        }
    }
    ring_close(args.ring, ring, tmem);      /* tensor memory goes back while the cluster meets */
    cluster_sync_all();
    bool repair = false;
    if (!*ring.stop && warp >= 2) {
        /* rows part, part + split, ... */
        const bool mixed = rows_differ;
        if (col < task.n) {
            const float b0 = h3b_lo(bias), b1 = h3b_hi(bias);
            for (uint32_t r = part + split * ((threadIdx.x >> 6) - 1); r < task.rows; r += 2 * split) {
                const uint32_t at = ring.stage0 + (r * LR_M + 2 * (threadIdx.x & 63)) * 4;
                float v0 = 0.0f, v1 = 0.0f;
                float x0[LR_SPLIT], x1[LR_SPLIT];
#pragma unroll
                for (uint32_t p = 0; p < LR_SPLIT; p++)      /* all on the way before the first is used */
                    if (p < split)
                        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x0[p]), "=f"(x1[p]) : "r"(cluster_map(at, p)) : "memory");
#pragma unroll
                for (uint32_t p = 0; p < LR_SPLIT; p++)
                    if (p < split) { v0 += x0[p]; v1 += x1[p]; }
                v0 += b0;
                v1 += b1;
                repair |= mixed && (h3b_not_finite(v0) || h3b_not_finite(v1));
                *reinterpret_cast<uint32_t *>(task.out + size_t(r) * task.n + col) = pack_bf16(v0, v1);
            }
        }
    }
    __syncwarp();
    cluster_sync_all();      /* nobody leaves, or writes over its shared memory, while that may be read */
    if (__syncthreads_or(repair)) {
        h3b_wait_for_launch();
        h3b_lora_repair(task, reinterpret_cast<float *>(raw_smem + (ring.stage0 - smem_u32(raw_smem))), part, split,
                        (task.rows - part + split - 1) / split, w0, min(uint32_t(LR_M), task.n - w0));
    }
}

/* up with rows of rank8 elements, zeros behind the rank: TMA wants row strides of 16 bytes. 8 elements a thread. */
__global__ void __launch_bounds__(256)
h3b_lora_pad_up(const uint16_t *__restrict__ up, uint16_t *up8, size_t rows, uint32_t rank, uint32_t rank8) {
    h3b_wait_for_launch();
    h3b_let_next_launch();
    const uint32_t pieces = rank8 / 8;
    const size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= rows * pieces) return;
    const size_t row = i / pieces;
    const uint32_t j = uint32_t(i % pieces) * 8;
    uint16_t v[8];
#pragma unroll
    for (uint32_t q = 0; q < 8; q++) v[q] = j + q < rank ? up[row * rank + j + q] : 0;
    *reinterpret_cast<uint4 *>(up8 + i * 8) = make_uint4(v[0] | uint32_t(v[1]) << 16, v[2] | uint32_t(v[3]) << 16,
                                                         v[4] | uint32_t(v[5]) << 16, v[6] | uint32_t(v[7]) << 16);
}

/* row-major BF16 [rows][k], box of 64 columns x box_rows, 128-byte swizzle */
bool lora_map(CUtensorMap *map, const uint16_t *data, uint64_t rows, uint64_t k, uint32_t box_rows) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    cuuint64_t dims[2] = {k, rows};
    cuuint64_t strides[1] = {k * 2};
    cuuint32_t box[2] = {LR_K, box_rows};
    cuuint32_t elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t *>(data), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool lora_env(const char *name) {
    const char *v = getenv(name);
    return v && *v && strcmp(v, "0") != 0;
}

/* shared memory of a launch of the two kernels above: `stages` stages, at least what the joined accumulators
 * need, and the barriers */
size_t ring_smem(const RingArgs &ring) { return size_t(ring.stages) * ring.stage_bytes + 1024 + LR_BAR_BYTES; }

bool lora_configure(int device) {
    static std::mutex mutex;
    static bool done[64];
    std::lock_guard<std::mutex> guard(mutex);
    if (!done[device & 63]) {
        if (cudaFuncSetAttribute(h3b_lora_down_tc, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 << 10) != cudaSuccess ||
            cudaFuncSetAttribute(h3b_lora_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 << 10) != cudaSuccess ||
            /* two CTAs of 100 KB per SM */
            cudaFuncSetAttribute(h3b_lora_down_tc, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
            cudaFuncSetAttribute(h3b_lora_rows, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        done[device & 63] = true;
    }
    return true;
}

/* `dependent`: the launch may begin while the kernel in front of it runs, and waits for it inside */
template <class Kernel, class... Args>
void launch_cluster(h3_gpu *gpu, Kernel *kernel, dim3 grid, uint32_t threads, uint32_t cluster, size_t smem, bool dependent, const Args &...args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = gpu->stream;
    cudaLaunchAttribute attributes[2];
    int count = 0;
    if (cluster > 1) {
        attributes[count].id = cudaLaunchAttributeClusterDimension;
        attributes[count].val.clusterDim.x = cluster;
        attributes[count].val.clusterDim.y = 1;
        attributes[count].val.clusterDim.z = 1;
        count++;
    }
    if (dependent) {
        attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[count].val.programmaticStreamSerializationAllowed = 1;
        count++;
    }
    config.attrs = attributes;
    config.numAttrs = count;
    cudaLaunchKernelEx(&config, kernel, args...);      /* an error is reported by h3b_launched */
}

uint32_t tmem_columns_for(uint32_t columns) {
    uint32_t n = 32;
    while (n < columns) n *= 2;
    return n;
}

/* clusters of `split` CTAs that the device runs beside each other with one CTA per SM; asked once per size. (The
 * runtime answers for one CTA per SM for kernels that allocate tensor memory, whatever their shared memory;
 * two of 100 KB do run side by side, checked by their SM numbers and start times.) */
template <class Kernel>
uint64_t resident_clusters(int device, Kernel *kernel, uint32_t split, size_t smem) {
    static std::mutex mutex;
    static std::unordered_map<uint64_t, int> known;
    const uint64_t key = uint64_t(device) << 40 | uint64_t(smem) << 8 | split;
    std::lock_guard<std::mutex> guard(mutex);
    auto found = known.find(key);
    if (found != known.end()) return uint64_t(found->second);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(split, 1024);
    config.blockDim = dim3(LR_THREADS);
    config.dynamicSmemBytes = smem;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = split;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) {
        cudaGetLastError();
        clusters = 0;
    }
    return uint64_t(known[key] = clusters);
}

/* CTAs of a cluster that split K: the most with which all tiles run in one round (a GPC holds whole clusters
 * only, so clusters of 7 or 8 leave SMs empty), with at least 4 K blocks each. One row, 7,168 -> 5,376, two
 * CTAs per SM: 21.6 us in 3 parts, 18.5 in 4, 16.8 in 5, 15.9 in 6, 26.3 in 7 (a second round). */
template <class Kernel>
uint32_t split_for(h3_gpu *gpu, Kernel *kernel, size_t smem, uint32_t per_sm, uint64_t tiles, uint32_t k_blocks) {
    for (uint32_t split = LR_SPLIT; split > 1; split--)
        if (split * 4 <= k_blocks && tiles <= per_sm * resident_clusters(gpu->device, kernel, split, smem)) return split;
    return 1;
}

/* Rows [0, task.rows) on the tensor cores; scratch as laid out by the caller. The first launch of a call may begin while
 * the one in front of the call ends and waits inside; not while capturing, where the node in front is the
 * scratch's allocation. */
int lora_tensor_cores(h3_gpu *gpu, const h3b_lora_task &task, bool few, bool captured) {
    const bool dependent = !captured || !task.first;
    const uint32_t k_blocks = (task.k + LR_K - 1) / LR_K;
    const uint32_t row_blocks = (task.rows + LR_M - 1) / LR_M;
    CUtensorMap map_x, map_down;
    DownArgs down = {};
    down.task = task;
    down.k_blocks = k_blocks;
    down.rank16 = (task.rank + 15) & ~15u;
    /* 128 columns at a time, or one entry of a larger rank (64 columns: 1,003 rows of rank 12 69.2 us instead of 66,
     * 1,664 rows of rank 64 121.7 instead of 118.5: x is read again for every group) */
    down.group = (down.rank16 <= 128 ? 128 : 256) / down.rank16;
    if (down.group > task.max_entries) down.group = task.max_entries;
    const uint32_t groups = (task.max_entries + down.group - 1) / down.group, columns = down.group * down.rank16;
    down.ring.status = gpu->status_device;
    down.ring.wait_cycles = gpu->wait_cycles;
    down.ring.stage_bytes = LR_A_BYTES + columns * LR_K * 2;
    down.ring.tmem_columns = tmem_columns_for(columns);
    /* Two CTAs per SM where they would fill more than half of the SMs alone and the joined accumulators (128 x columns F32)
     * leave room for it, so that the projection can begin on the others (1,664 rows, 7,168 -> 5,376, rank 64, 104
     * CTAs: 122 us, one per SM 127); else deeper rings, since a CTA's stream is its bytes in flight over the memory's
     * latency (800 rows, 14,336 -> 5,376, rank 128, 56 CTAs: 138 us, two per SM 139.3). */
    const bool two = columns <= 128 && uint64_t(row_blocks) * 2 * LR_SPLIT > uint64_t(gpu->sm_count);
    const uint32_t want = two ? 106 << 10 : 200 << 10;
    down.ring.stages = want / down.ring.stage_bytes;
    if (down.ring.stages > uint32_t(LR_STAGES)) down.ring.stages = LR_STAGES;
    const uint32_t per_sm = two ? 2 : 1, down_split = split_for(gpu, h3b_lora_down_tc, ring_smem(down.ring), per_sm, row_blocks, k_blocks);
    /* Groups of entries run side by side while all run in one round, and in turn beyond that: most tiles hold few of
     * many adapters, and a CTA that finds nothing to do costs its set-up (6,400 rows, 5,376 -> 5,376, 4 of 256
     * adapters of rank 64 occur: 265 us in turn, 534 with every group side by side; 300 rows of 16 adapters of rank 64,
     * which fit: 48 side by side, 83 in turn) */
    const uint64_t room = per_sm * resident_clusters(gpu->device, h3b_lora_down_tc, down_split, ring_smem(down.ring)) / row_blocks;
    const uint32_t side = groups < room ? groups : room < 1 ? 1 : uint32_t(room);
    if (!lora_map(&map_x, task.x, task.rows, task.k, LR_M) ||
        !lora_map(&map_down, task.down, uint64_t(task.adapters) * task.rank, task.k, down.rank16))
        return h3b_fail(gpu, "linear_lora_bf16: cannot encode the tensor maps");
    /* By warps where that is the shorter way and there is no long weight stream to hide it behind (us, by warps / tensor
     * cores: 4 rows 1,024 -> 5,376 rank 16 8.6 / 11.7, 128 rows 15.1 / 17.5, rank 64 22.2 / 18.5; 2,048 -> 5,376 16
     * rows 12.0 / 13.3; 2,688 -> 10,752 16 rows 18.9 / 17.0; 5,376 -> 5,376 64 rows 21.8 / 19.5), and up to 8 CTAs (2
     * stored sums each) beside any weight: more of them take SMs that the streaming kernel's clusters wait for. 1 row of
     * rank 16 or 2 of rank 8, 8 CTAs: 5,376 -> 5,376 16.0 / 17.1, 7,168 -> 5,376 18.0 / 18.5, 14,336 -> 5,376 29.1 / 29.6,
     * 5,376 -> 21,504 42.6 / 43.0, 2,688 -> 96,768 84.9 / 85.3; 1 row of rank 32 or 4 of rank 4, 16 CTAs: 24.5 / 17.5,
     * 28.2 / 19.7, 46.1 / 29.5, 42.6 / 43.1, 84.8 / 85.4. */
    const uint64_t sums = uint64_t(task.rows) * task.rank;
    if (few && (uint64_t(task.rows) * task.rank8 <= 16 || (sums <= 2048 && uint64_t(task.n) * task.k <= 12000000)))
        launch_cluster(gpu, h3b_lora_down_few, dim3(task.rows, task.rank8 / LF_SUMS), 32 * LF_WARPS, 1, 0, dependent, task);
    else
        launch_cluster(gpu, h3b_lora_down_tc, dim3(down_split, row_blocks, side), LR_THREADS, down_split, ring_smem(down.ring), dependent,
                       map_x, map_down, down);
    if (cudaGetLastError() != cudaSuccess) return h3b_fail(gpu, "linear_lora_bf16: the low-rank rows cannot be launched");
    if (!few) {
        if (!h3b_gemm_lora(gpu, task, captured)) return h3b_fail(gpu, "linear_lora_bf16: cannot set up the tensor-core GEMM");
        return 1;
    }
    RowsArgs rows = {};
    rows.task = task;
    rows.k_blocks = k_blocks;
    rows.blocks = (task.rank + LR_K - 1) / LR_K;
    rows.ring.status = gpu->status_device;
    rows.ring.wait_cycles = gpu->wait_cycles;
    rows.ring.stage_bytes = LR_A_BYTES + task.tile_rows * LR_K * 2;
    rows.ring.tmem_columns = tmem_columns_for(task.tile_rows);
    rows.ring.stages = (106 << 10) / rows.ring.stage_bytes;
    if (rows.ring.stages > uint32_t(LR_STAGES)) rows.ring.stages = LR_STAGES;
    const uint32_t weight_tiles = (task.n + LR_M - 1) / LR_M;
    const uint32_t split = split_for(gpu, h3b_lora_rows, ring_smem(rows.ring), 2, weight_tiles, k_blocks);
    CUtensorMap map_w, map_rows, map_up, map_t;
    EncodeTiled encode = encode_tiled();
    cuuint64_t dims[3] = {task.rank8, task.n, task.adapters};
    cuuint64_t strides[2] = {cuuint64_t(task.rank8) * 2, cuuint64_t(task.n) * task.rank8 * 2};
    cuuint32_t box[3] = {LR_K, LR_M, 1};
    cuuint32_t elem[3] = {1, 1, 1};
    if (!lora_map(&map_w, task.w, task.n, task.k, LR_M) || !lora_map(&map_rows, task.x, task.rows, task.k, task.tile_rows) ||
        !lora_map(&map_t, task.t, uint64_t(task.max_entries) * task.tile_rows, task.rank8, task.tile_rows) ||
        encode(&map_up, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t *>(task.up8), dims, strides, box, elem,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return h3b_fail(gpu, "linear_lora_bf16: cannot encode the tensor maps");
    launch_cluster(gpu, h3b_lora_rows, dim3(split, weight_tiles), LR_THREADS, split, ring_smem(rows.ring), true, map_w, map_rows, map_up, map_t, rows);
    return 1;
}

}  // namespace

extern "C" int h3x_linear_lora_bf16(h3_gpu *gpu, h3_gpu_tensor *output, const h3_gpu_tensor *input,
                                    const h3_gpu_tensor *weight, const h3_gpu_tensor *bias,
                                    const h3_gpu_tensor *down, const h3_gpu_tensor *up,
                                    const h3_gpu_tensor *scale, const h3_gpu_tensor *row_adapter, uint32_t rows,
                                    uint32_t input_dim, uint32_t output_dim, uint32_t adapters, uint32_t rank) {
    if (!gpu) return 0;
    if (!adapters) return h3_gpu_linear_bf16(gpu, output, input, weight, bias, rows, input_dim, output_dim);
    if (adapters > kMaxAdapters || !rank || rank > kMaxRank)
        return h3b_fail(gpu, "adapters must be 0..%u and rank 1..%u", kMaxAdapters, kMaxRank);
    if (!h3b_need(gpu, input, H3_GPU_BF16, size_t(rows) * input_dim, "adapter projection input") ||
        !h3b_need(gpu, weight, H3_GPU_BF16, size_t(output_dim) * input_dim, "adapter projection weight") ||
        !h3b_need(gpu, output, H3_GPU_BF16, size_t(rows) * output_dim, "adapter projection output") ||
        (bias && !h3b_need(gpu, bias, H3_GPU_BF16, output_dim, "adapter projection bias")) ||
        !h3b_need(gpu, down, H3_GPU_BF16, size_t(adapters) * rank * input_dim, "adapter down") ||
        !h3b_need(gpu, up, H3_GPU_BF16, size_t(adapters) * output_dim * rank, "adapter up") ||
        (scale && !h3b_need(gpu, scale, H3_GPU_F32, adapters, "adapter scale")) ||
        (row_adapter && !h3b_need(gpu, row_adapter, H3_GPU_U32, rows, "row adapter")) || !h3b_need_command(gpu))
        return 0;
    for (const h3_gpu_tensor *t : {input, weight, bias, down, up, scale, row_adapter})
        if (t && h3b_overlap(output->data, size_t(rows) * output_dim * 2, t->data, t->bytes))
            return h3b_fail(gpu, "the adapter projection's output overlaps one of its inputs");
    const h3b_kind kind = rows >= 32 && input_dim >= 256 && output_dim >= 256 ? H3B_LINEAR : H3B_DIRECT;
    if (!rows || !output_dim) return h3b_launched(gpu, "linear_lora_bf16", kind);
    h3b_on_device device(gpu);
    const uint16_t *x = h3b_ptr<uint16_t>(input), *w = h3b_ptr<uint16_t>(weight);
    const uint16_t *b = bias ? h3b_ptr<uint16_t>(bias) : nullptr;
    const uint16_t *d = h3b_ptr<uint16_t>(down), *u = h3b_ptr<uint16_t>(up);
    const float *s = scale ? h3b_ptr<float>(scale) : nullptr;
    const uint32_t *map = row_adapter ? h3b_ptr<uint32_t>(row_adapter) : nullptr;
    uint16_t *y = h3b_ptr<uint16_t>(output);

    const bool aligned = h3b_aligned16(x) && h3b_aligned16(w) && (!b || h3b_aligned16(b)) && h3b_aligned16(d) && h3b_aligned16(u) && h3b_aligned16(y);
    if (aligned && input_dim && input_dim % 8 == 0 && output_dim % 8 == 0 && input_dim <= INT32_MAX && output_dim <= INT32_MAX && !lora_env("H3B_NO_TENSOR_CORES") &&
        double(rows) * output_dim * input_dim >= 32.0 * 256 * 256) {      /* tiny problems are latency bound either way */
        if (!lora_configure(gpu->device)) return h3b_fail(gpu, "cannot reserve shared memory for the adapter kernels");
        h3b_lora_task task = {};
        task.x = x; task.w = w; task.bias = b; task.down = d; task.up = task.up8 = u;
        task.scale = s;
        task.row_adapter = map;
        task.out = y;
        task.rows = rows; task.k = input_dim; task.n = output_dim; task.adapters = adapters; task.rank = rank;
        task.rank8 = (rank + 7) & ~7u;
        /* The weight-streaming kernel takes calls of one row tile: up to 16 rows of any width, and more while the GEMM's tiles
         * would leave two thirds of the SMs idle (us, streaming / GEMM, 5,376 and 2,688 inputs: 1 row -> 21,504 43.8 / 59.6,
         * 25.6 / 34.1; 16 rows -> 28,672 53.5 / 53.7, 31.4 / 36.9, -> 96,768 164 / 164, 91 / 111; 100 rows -> 5,376 22 / 39
         * (5,376), -> 10,752 30.5 / 41.2, 21.2 / 25.5, -> 16,384 41.2 / 43.2, 27.3 / 26.0, -> 21,504 58.7 / 47.6, 37.8 / 29.3) */
        const uint64_t gemm_tiles = (uint64_t(output_dim) + 255) / 256;
        const bool few = (rows <= 16 && gemm_tiles < 32768) || (rows <= uint32_t(LR_M) && 3 * gemm_tiles <= uint64_t(gpu->sm_count));
        const uint32_t tile_rows = few ? (rows + 15) & ~15u : h3b_gemm_lora_tile_rows(gpu, rows, output_dim);
        task.tile_rows = tile_rows;
        task.max_entries = adapters < tile_rows ? adapters : tile_rows;
        auto rounded = [](size_t bytes) { return (bytes + 255) & ~size_t(255); };
        /* room for every adapter in every tile; so many rows at a time that it stays within a gigabyte */
        const size_t tile_bytes = size_t(task.max_entries) * tile_rows * task.rank8 * 2;
        size_t chunk_tiles = (size_t(1) << 30) / tile_bytes;
        if (chunk_tiles > 32767) chunk_tiles = 32767;          /* two 128-row blocks each, counted in a grid's y */
        const size_t all_tiles = (size_t(rows) + tile_rows - 1) / tile_rows;
        if (chunk_tiles > all_tiles) chunk_tiles = all_tiles;
        const size_t t_bytes = rounded(chunk_tiles * tile_bytes);
        const size_t up_bytes = task.rank8 == rank ? 0 : rounded(size_t(adapters) * output_dim * task.rank8 * 2);
        const size_t count_bytes = rounded(chunk_tiles * 4), entry_bytes = rounded(chunk_tiles * task.max_entries * 4);
        h3b_scratch scratch(gpu, t_bytes + up_bytes + count_bytes + entry_bytes);
        if (!scratch.data) return h3b_fail(gpu, "linear_lora_bf16: cannot allocate the low-rank rows");
        uint8_t *at = static_cast<uint8_t *>(scratch.data);
        task.t = reinterpret_cast<uint16_t *>(at);
        task.counts = reinterpret_cast<uint32_t *>(at + t_bytes + up_bytes);
        task.entries = reinterpret_cast<uint32_t *>(at + t_bytes + up_bytes + count_bytes);
        if (up_bytes) {
            uint16_t *up8 = reinterpret_cast<uint16_t *>(at + t_bytes);
            const size_t up_rows = size_t(adapters) * output_dim;
            launch_cluster(gpu, h3b_lora_pad_up, dim3(unsigned((up_rows * (task.rank8 / 8) + 255) / 256)), 256, 1, 0, !scratch.captured, u, up8,
                           up_rows, rank, task.rank8);
            task.up8 = up8;
        }
        for (size_t tile = 0; tile < all_tiles; tile += chunk_tiles) {
            const size_t row0 = tile * tile_rows;
            h3b_lora_task part = task;
            part.rows = uint32_t(rows - row0 < chunk_tiles * tile_rows ? rows - row0 : chunk_tiles * tile_rows);
            part.x = x + row0 * input_dim;
            part.out = y + row0 * output_dim;
            part.row_adapter = map ? map + row0 : nullptr;
            part.first = !up_bytes || tile;
            if (!lora_tensor_cores(gpu, part, few, scratch.captured)) return 0;
        }
        return h3b_launched(gpu, "linear_lora_bf16", kind);
    }
    /* so many rows at a time that their low-rank rows stay within 256 MB and grids within their limits */
    const size_t most = (size_t(1) << 26) / rank, chunk = rows < most ? rows : most;
    h3b_scratch scratch(gpu, chunk * rank * sizeof(float));
    if (!scratch.data) return h3b_fail(gpu, "linear_lora_bf16: cannot allocate the low-rank rows");
    float *t = static_cast<float *>(scratch.data);
    for (size_t row0 = 0; row0 < rows; row0 += chunk) {
        const uint32_t part = uint32_t(rows - row0 < chunk ? rows - row0 : chunk);
        const uint32_t *part_map = map ? map + row0 : nullptr;
        h3b_lora_down_simt<<<unsigned((size_t(part) * rank + 7) / 8), 256, 0, gpu->stream>>>(x + row0 * input_dim, d, s, part_map, t, part,
                                                                                            input_dim, adapters, rank);
        const size_t tiles = size_t((part + 63) / 64) * ((size_t(output_dim) + 63) / 64);
        h3b_lora_simt<<<unsigned(tiles), 256, 0, gpu->stream>>>(x + row0 * input_dim, w, b, u, t, part_map, y + row0 * output_dim, part,
                                                                input_dim, output_dim, adapters, rank);
    }
    return h3b_launched(gpu, "linear_lora_bf16", kind);
}
