/* What the kernels of the adapter projection share (h3b_lora.cu, the adapter epilogue of h3b_gemm.cu).
 *
 * The rows of a call are cut into tiles of tile_rows. A tile's entries are the adapters that occur in it,
 * ascending; entry e has a block of tile_rows low-rank rows t (BF16, rank8 = rank rounded up to 8 columns,
 * zeros behind rank): scale[a] x.down[a]^T where the row's adapter is the entry's, zeros elsewhere. Then
 *   out tile = x.W^T + sum_e t_e . up[a_e]^T
 * is one accumulation on the tensor cores: the entries are more K blocks behind the projection's own.
 *
 * t is F32 until it is scaled and then rounded to BF16 once, since both operands of an instruction have one type
 * and up is BF16: 2^-8 of |t| . |up| at most, of a term that is small beside x.W^T. A second block of what the
 * rounding left would take that to 2^-16 for twice the entries' K blocks; the result's own rounding is 2^-8 of all of it. */
#pragma once

#include "h3b_common.cuh"

#include <cuda_bf16.h>

struct h3b_lora_task {
    const uint16_t *x, *w, *bias, *down, *up;
    const uint16_t *up8;            /* up with rows of rank8 elements (up itself where rank is a multiple of 8) */
    const float *scale;
    const uint32_t *row_adapter;
    uint16_t *out;
    uint32_t rows, k, n, adapters, rank, rank8;
    uint32_t tile_rows, max_entries;
    uint32_t first;                 /* the low-rank rows are the call's first launch: it waits for what is in front of the call */
    uint32_t *counts;               /* [tile]: entries, bit 31: rows of the tile differ in their adapter */
    uint32_t *entries;              /* [tile][max_entries]: adapter of the entry */
    uint16_t *t;                    /* [tile][max_entries][tile_rows][rank8] */
};
constexpr uint32_t H3B_LORA_MIXED = 0x80000000u;

/* The projection with adapter epilogue on 128- or 256-row tiles (h3b_gemm.cu); its launch may begin before
 * the kernel in front of it on the stream has ended and waits inside for it. */
uint32_t h3b_gemm_lora_tile_rows(h3_gpu *gpu, uint32_t rows, uint32_t n);
int h3b_gemm_lora(h3_gpu *gpu, const h3b_lora_task &task, bool captured);

#ifdef __CUDACC__
/* In a tile whose rows differ in their adapter, a row meets the other adapters' up rows times zeros. Where
 * those are not finite the accumulator is NaN although the row's own result may be finite. Such a tile is stored as it
 * comes, and behind its last tile, where no wait of the kernel runs any more, the CTA that stored it computes what is
 * not finite in it again, from each row's own adapter alone: F32 chains over k and then the rank, 64 x 64 outputs at a
 * time, 8 x 4 of them a thread, both operands through shared memory (one element at a time, inside the epilogue,
 * 400 rows 7,168 -> 768 of three adapters, one of infinities, took 139 ms and held up the accumulators' waits). */
constexpr uint32_t H3B_LORA_THREADS = 192, H3B_LORA_REPAIR_K = 32, H3B_LORA_REPAIR_PITCH = 68;
/* Rows row0, row0 + stride, ... (`count` of them) of output columns col0 .. col0 + columns - 1, by all threads of the CTA;
 * smem: 2 * 32 * 68 floats, 16-byte aligned. */
static __device__ __noinline__ void h3b_lora_repair(const h3b_lora_task &task, float *smem, uint32_t row0, uint32_t stride,
                                                    uint32_t count, uint32_t col0, uint32_t columns) {
    constexpr uint32_t SIDE = 64, K = H3B_LORA_REPAIR_K, PITCH = H3B_LORA_REPAIR_PITCH, PIECES = 2 * SIDE * K / 8;
    constexpr uint32_t LOADS = (PIECES + H3B_LORA_THREADS - 1) / H3B_LORA_THREADS;
    const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;      /* ty 8 and up: loads only */
    for (uint32_t r0 = 0; r0 < count; r0 += SIDE)
        for (uint32_t c0 = 0; c0 < columns; c0 += SIDE) {
            const uint32_t col = col0 + c0 + 4 * tx;
            uint32_t bad = 0;                                         /* bit 4 i + j: row i, column j of the thread's */
            if (ty < 8 && c0 + 4 * tx < columns)
                for (uint32_t i = 0; i < 8 && r0 + 8 * ty + i < count; i++) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(task.out + size_t(row0 + (r0 + 8 * ty + i) * stride) * task.n + col);
                    const uint32_t words[2] = {v.x, v.y};
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) bad |= uint32_t((words[j / 2] >> (16 * (j & 1)) & 0x7f80u) == 0x7f80u) << (4 * i + j);
                }
            if (!__syncthreads_or(bad != 0)) continue;
            float acc[8][4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const float start = task.bias && c0 + 4 * tx < columns ? h3b_widen(task.bias[col + j]) : 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) acc[i][j] = start;
            }
            /* 8 values of k at a time (k is a multiple of 8): piece p is of x (p < 256) or w, row p & 63 */
            uint4 next[LOADS];
            auto load = [&](uint32_t k0) {
#pragma unroll
                for (uint32_t l = 0; l < LOADS; l++) {
                    const uint32_t p = threadIdx.x + l * H3B_LORA_THREADS, r = p & (SIDE - 1), k = k0 + 8 * (p / SIDE & 3);
                    next[l] = make_uint4(0, 0, 0, 0);
                    if (p >= PIECES || k >= task.k) continue;
                    if (p < PIECES / 2) {
                        if (r0 + r < count) next[l] = *reinterpret_cast<const uint4 *>(task.x + size_t(row0 + (r0 + r) * stride) * task.k + k);
                    } else if (c0 + r < columns) {
                        next[l] = *reinterpret_cast<const uint4 *>(task.w + size_t(col0 + c0 + r) * task.k + k);
                    }
                }
            };
            load(0);
            for (uint32_t k0 = 0; k0 < task.k; k0 += K) {
#pragma unroll
                for (uint32_t l = 0; l < LOADS; l++) {
                    const uint32_t p = threadIdx.x + l * H3B_LORA_THREADS;
                    if (p >= PIECES) break;
                    float *at = smem + (p < PIECES / 2 ? 0 : K * PITCH) + 8 * (p / SIDE & 3) * PITCH + (p & (SIDE - 1));
                    const uint32_t words[4] = {next[l].x, next[l].y, next[l].z, next[l].w};
#pragma unroll
                    for (uint32_t q = 0; q < 4; q++) {
                        at[2 * q * PITCH] = h3b_lo(words[q]);
                        at[(2 * q + 1) * PITCH] = h3b_hi(words[q]);
                    }
                }
                __syncthreads();
                if (k0 + K < task.k) load(k0 + K);
                if (ty < 8) {
#pragma unroll 4
                    for (uint32_t k = 0; k < K; k++) {
                        const float4 a0 = *reinterpret_cast<const float4 *>(smem + k * PITCH + 8 * ty);
                        const float4 a1 = *reinterpret_cast<const float4 *>(smem + k * PITCH + 8 * ty + 4);
                        const float4 b = *reinterpret_cast<const float4 *>(smem + (K + k) * PITCH + 4 * tx);
                        const float as[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w}, bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                        for (uint32_t i = 0; i < 8; i++)
#pragma unroll
                            for (uint32_t j = 0; j < 4; j++) acc[i][j] = fmaf(as[i], bs[j], acc[i][j]);
                    }
                }
                __syncthreads();
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                if (!(bad >> (4 * i) & 15u)) continue;
                const uint32_t row = row0 + (r0 + 8 * ty + i) * stride, tile = row / task.tile_rows;
                const uint32_t a = task.row_adapter ? task.row_adapter[row] : 0;
                const uint32_t entries = a < task.adapters ? task.counts[tile] & ~H3B_LORA_MIXED : 0;
                for (uint32_t e = 0; e < entries; e++) {
                    if (task.entries[size_t(tile) * task.max_entries + e] != a) continue;
                    const uint16_t *t = task.t + ((size_t(tile) * task.max_entries + e) * task.tile_rows + row % task.tile_rows) * task.rank8;
                    const uint16_t *u = task.up + (size_t(a) * task.n + col) * task.rank;
                    for (uint32_t q = 0; q < task.rank; q++)
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) acc[i][j] = fmaf(h3b_widen(t[q]), h3b_widen(u[size_t(j) * task.rank + q]), acc[i][j]);
                    break;
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; j++)
                    if (bad >> (4 * i + j) & 1u) task.out[size_t(row) * task.n + col + j] = __bfloat16_as_ushort(__float2bfloat16_rn(acc[i][j]));
            }
        }
}
__device__ __forceinline__ bool h3b_not_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }

/* The launch in front of this one on the stream has ended and its writes are visible (programmatic
 * dependent launch); returns at once in a launch without that attribute. */
__device__ __forceinline__ void h3b_wait_for_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void h3b_let_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif
