/* Cross attention: query rows of several requests to an encoder's states of other lengths.
 *
 * h3b_cross_simt takes any head size, alignment and scale: one CTA per (query row, head) walks the keys
 * of the row's segment with the online softmax recurrence in F32.
 */
#include "h3b_common.cuh"

#include <cuda_bf16.h>

#include <cmath>

namespace {

/* round to nearest even; NaN stays NaN (h3b_narrow's integer formula turns some into zeros) */
__device__ __forceinline__ uint16_t to_bf16(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }

/* Rows of one segment after clipping to the tensors */
struct Segment {
    uint32_t q0, queries, k0, keys;
};

__device__ __forceinline__ Segment load_segment(const uint32_t *segments, uint32_t index, uint32_t query_rows,
                                                uint32_t key_rows) {
    if (!segments) return {0u, query_rows, 0u, key_rows};
    const uint4 raw = make_uint4(__ldg(segments + 4 * index), __ldg(segments + 4 * index + 1),
                                 __ldg(segments + 4 * index + 2), __ldg(segments + 4 * index + 3));
    Segment s;
    s.q0 = min(raw.x, query_rows);
    s.queries = min(raw.y, query_rows - s.q0);
    s.k0 = min(raw.z, key_rows);
    s.keys = min(raw.w, key_rows - s.k0);
    return s;
}

constexpr int kSimtThreads = 128;
constexpr int kSimtMaxDimsPerThread = 4;   /* head_dim <= 512 */

__global__ void __launch_bounds__(kSimtThreads)
h3b_cross_simt(const uint16_t *q, const uint16_t *k, const uint16_t *v, uint16_t *out, const uint32_t *segments,
               uint32_t segment_count, uint32_t query_rows, uint32_t key_rows, uint32_t heads, uint32_t kv_heads,
               uint32_t hd, float scale) {
    extern __shared__ float cross_smem[];
    float *qs = cross_smem;             /* hd           */
    float *ps = cross_smem + hd;        /* kSimtThreads */
    __shared__ float red[kSimtThreads / 32];
    const uint32_t row = blockIdx.x, head = blockIdx.y, kv_head = head / (heads / kv_heads);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Segment s = {0, 0, 0, 0};
    uint32_t at = 0;
    for (; at < segment_count; at++) {
        s = load_segment(segments, at, query_rows, key_rows);
        if (row - s.q0 < s.queries) break;
    }
    if (at == segment_count) return;                /* a row of no segment */
    const uint16_t *qp = q + (size_t(row) * heads + head) * hd;
    for (uint32_t d = tid; d < hd; d += kSimtThreads) qs[d] = h3b_widen(qp[d]);
    __syncthreads();
    float m = -INFINITY, l = 0.0f;
    float acc[kSimtMaxDimsPerThread] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t j0 = 0; j0 < s.keys; j0 += kSimtThreads) {
        const uint32_t j = j0 + tid;
        float score = -INFINITY;
        if (j < s.keys) {
            const uint16_t *kp = k + (size_t(s.k0 + j) * kv_heads + kv_head) * hd;
            float dot = 0.0f;
            for (uint32_t d = 0; d < hd; d++) dot = fmaf(qs[d], h3b_widen(kp[d]), dot);
            score = dot * scale;
        }
        float most = score;
#pragma unroll
        for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (lane == 0) red[warp] = most;
        __syncthreads();
        most = m;
        for (int w = 0; w < kSimtThreads / 32; w++) most = fmaxf(most, red[w]);
        const float base = most == -INFINITY ? 0.0f : most;     /* all scores -inf so far */
        const float alpha = expf(m - base);
        const float p = j < s.keys ? expf(score - base) : 0.0f;
        ps[tid] = p;
        const float part = h3b_warp_sum(p);
        __syncthreads();
        if (lane == 0) red[warp] = part;
        __syncthreads();
        float total = 0.0f;
        for (int w = 0; w < kSimtThreads / 32; w++) total += red[w];
        l = l * alpha + total;
        m = most;
        const uint32_t live = min(uint32_t(kSimtThreads), s.keys - j0);
#pragma unroll
        for (int i = 0; i < kSimtMaxDimsPerThread; i++) {
            const uint32_t d = tid + i * kSimtThreads;
            if (d >= hd) break;
            float a = acc[i] * alpha;
            for (uint32_t t = 0; t < live; t++)
                a = fmaf(ps[t], h3b_widen(v[(size_t(s.k0 + j0 + t) * kv_heads + kv_head) * hd + d]), a);
            acc[i] = a;
        }
        __syncthreads();
    }
    /* no keys, or no key with a score above -inf: zeros. A sum that is NaN stays NaN. */
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < kSimtMaxDimsPerThread; i++) {
        const uint32_t d = tid + i * kSimtThreads;
        if (d >= hd) break;
        out[(size_t(row) * heads + head) * hd + d] = to_bf16(acc[i] * inv);
    }
}

}  // namespace

extern "C" int h3x_cross_sdpa_bf16(h3_gpu *gpu, h3_gpu_tensor *output, const h3_gpu_tensor *query,
                                   const h3_gpu_tensor *key, const h3_gpu_tensor *value,
                                   const h3_gpu_tensor *segments, uint32_t segment_count, uint32_t query_rows,
                                   uint32_t key_rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                   float scale) {
    if (!gpu) return 0;
    if (!heads || !kv_heads || !head_dim) return h3b_fail(gpu, "cross attention shape is empty");
    if (heads % kv_heads) return h3b_fail(gpu, "cross attention heads must divide by the key heads");
    if (head_dim > uint32_t(kSimtThreads * kSimtMaxDimsPerThread))
        return h3b_fail(gpu, "cross attention head dimension is too large");
    if (heads > 65535) return h3b_fail(gpu, "cross attention has too many heads");
    if (!segments && segment_count) return h3b_fail(gpu, "cross attention segments tensor has the wrong dtype");
    const size_t q_count = size_t(query_rows) * heads * head_dim, k_count = size_t(key_rows) * kv_heads * head_dim;
    if (!h3b_need(gpu, query, H3_GPU_BF16, q_count, "cross attention query") ||
        !h3b_need(gpu, key, H3_GPU_BF16, k_count, "cross attention key") ||
        !h3b_need(gpu, value, H3_GPU_BF16, k_count, "cross attention value") ||
        !h3b_need(gpu, output, H3_GPU_BF16, q_count, "cross attention output") ||
        (segments && !h3b_need(gpu, segments, H3_GPU_U32, size_t(segment_count) * 4, "cross attention segments")) ||
        !h3b_need_command(gpu))
        return 0;
    for (const h3_gpu_tensor *t : {key, value, segments})
        if (t && h3b_overlap(output->data, q_count * 2, t->data, t->bytes))
            return h3b_fail(gpu, "the cross attention's output overlaps its keys, values or segments");
    if (output->data != query->data && h3b_overlap(output->data, q_count * 2, query->data, q_count * 2))
        return h3b_fail(gpu, "the cross attention's output overlaps part of its query");
    const uint32_t *table = segments ? h3b_ptr<uint32_t>(segments) : nullptr;
    if (!segments) segment_count = 1;
    if (!query_rows || !segment_count) return h3b_launched(gpu, "cross_sdpa_bf16", H3B_SDPA);
    h3b_on_device device(gpu);
    const uint16_t *q = h3b_ptr<uint16_t>(query), *k = h3b_ptr<uint16_t>(key), *v = h3b_ptr<uint16_t>(value);
    uint16_t *out = h3b_ptr<uint16_t>(output);

    const size_t smem = (size_t(head_dim) + kSimtThreads) * sizeof(float);
    h3b_cross_simt<<<dim3(query_rows, heads), kSimtThreads, smem, gpu->stream>>>(
        q, k, v, out, table, segment_count, query_rows, key_rows, heads, kv_heads, head_dim, scale);
    return h3b_launched(gpu, "cross_sdpa_bf16", H3B_SDPA);
}
