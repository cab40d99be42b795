/* What the kernels of the adapter projection share (h3b_lora.cu, the adapter epilogue of h3b_gemm.cu).
 *
 * The rows of a call are cut into tiles of tile_rows. A tile's entries are the adapters that occur in it,
 * ascending; entry e has a block of tile_rows low-rank rows t (BF16, rank8 = rank rounded up to 8 columns,
 * zeros behind rank): scale[a] x.down[a]^T where the row's adapter is the entry's, zeros elsewhere. Then
 *   out tile = x.W^T + sum_e t_e . up[a_e]^T
 * is one accumulation on the tensor cores: the entries are more K blocks behind the projection's own. */
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
 * those are not finite the accumulator is NaN although the row's own result may be finite: such an element
 * is computed again on its own, in F32, from its row's adapter alone. */
static __device__ __noinline__ float h3b_lora_element(const h3b_lora_task &task, uint32_t row, uint32_t col) {
    float v = task.bias ? h3b_widen(task.bias[col]) : 0.0f;
    const uint16_t *x = task.x + size_t(row) * task.k, *w = task.w + size_t(col) * task.k;
    for (uint32_t i = 0; i < task.k; i++) v = fmaf(h3b_widen(x[i]), h3b_widen(w[i]), v);
    const uint32_t a = task.row_adapter ? task.row_adapter[row] : 0, tile = row / task.tile_rows;
    const uint32_t count = a < task.adapters ? task.counts[tile] & ~H3B_LORA_MIXED : 0;
    for (uint32_t e = 0; e < count; e++)
        if (task.entries[size_t(tile) * task.max_entries + e] == a) {
            const uint16_t *t = task.t + ((size_t(tile) * task.max_entries + e) * task.tile_rows + row % task.tile_rows) * task.rank8;
            const uint16_t *u = task.up + (size_t(a) * task.n + col) * task.rank;
            for (uint32_t j = 0; j < task.rank; j++) v = fmaf(h3b_widen(t[j]), h3b_widen(u[j]), v);
        }
    return v;
}
__device__ __forceinline__ bool h3b_not_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }

/* The launch in front of this one on the stream has ended and its writes are visible (programmatic
 * dependent launch); returns at once in a launch without that attribute. */
__device__ __forceinline__ void h3b_wait_for_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void h3b_let_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif
