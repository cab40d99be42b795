/* Low-rank adapters of many requests beside a shared projection:
 *   out[r] = bf16( x[r].W^T + bias + scale[a] (x[r].down[a]^T).up[a]^T ),  a = row_adapter[r].
 *
 * Kernels that take any shape and alignment (one F32 fmaf chain per sum): h3b_lora_down_simt computes
 * the low-rank row t[r] = scale[a] x[r].down[a]^T once, h3b_lora_simt the projection with t[r].up[a]^T
 * added to every output before its one rounding.
 */
#include "h3b_common.cuh"

#include <cuda_bf16.h>

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
    const uint32_t row0 = blockIdx.y * 64, col0 = blockIdx.x * 64;
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

constexpr uint32_t kMaxRank = 256, kMaxAdapters = 1024;

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

    h3b_scratch scratch(gpu, size_t(rows) * rank * sizeof(float));
    if (!scratch.data) return h3b_fail(gpu, "linear_lora_bf16: cannot allocate the low-rank rows");
    float *t = static_cast<float *>(scratch.data);
    const size_t warps = size_t(rows) * rank;
    h3b_lora_down_simt<<<unsigned((warps + 7) / 8), 256, 0, gpu->stream>>>(x, d, s, map, t, rows, input_dim, adapters, rank);
    h3b_lora_simt<<<dim3((output_dim + 63) / 64, (rows + 63) / 64), 256, 0, gpu->stream>>>(
        x, w, b, u, t, map, y, rows, input_dim, output_dim, adapters, rank);
    return h3b_launched(gpu, "linear_lora_bf16", kind);
}
