/* Cross attention: query rows of several requests to an encoder's states of other lengths.
 *
 * h3b_cross_tc (head_dim 64 and 128) runs on the tensor cores, described at its definition;
 * h3b_cross_merge joins its partial results where the keys of a segment are cut into pieces. h3b_cross_simt takes
 * any head size, alignment and scale: one CTA per (query row, head) walks the keys of the row's segment
 * with the online softmax recurrence in F32 (1.0 TFLOP/s, bound by its loads and shuffles: 50,476 rows x
 * 512 keys x 56 heads 698 ms).
 */
#include "h3b_common.cuh"
#include "h3b_sm100.cuh"

#include <cuda_bf16.h>

#include <cmath>
#include <cstdlib>
#include <type_traits>

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
    /* Read-only loads (plain ones cost single rows 0.5 us of 25): behind griddepcontrol.wait what is in front of the call
     * has ended, and nothing of this launch has touched the table before. */
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


/* ------------------------------------------------------------- tensor cores
 * A query tile is 128 rows of tensor memory: 128 / pack query rows of `pack` neighbouring heads that
 * share a key head (pack = the largest power of two in heads / kv_heads), so that shared key heads are
 * read once per tile. A work unit is GROUPS neighbouring tiles of one segment and head set over a range of
 * 128-key tiles ("steps"); persistent CTAs walk units w, w + grid, ... The steps of all units of a CTA
 * count on in t: t names buffers and barrier phases, and step t + 1 may be the next unit's first.
 *
 *   warp 0   TMA. Stage t % STAGES holds what the tensor core reads after the softmax of step t: V(t) and
 *            K(t + 1). With a unit's last step come the next unit's queries (one buffer per group: the
 *            scores of the last step have been computed by then).
 *   warp 1   tcgen05.mma, per step and group: O += P(t).V(t), then the group's scores Q.K(t + 1)^T, at a unit's
 *            end those of the next unit once its queries are there (the groups write their outputs meanwhile). The
 *            tensor pipe does not drain between units: states are short (one to four steps), and a CTA per
 *            tile would spend half of its time filling and draining. All the group waits for collects on
 *            two barriers: go[group][t % 2], the softmax warps' arrivals for the first half of P(t) and, for
 *            the first group, the bytes of V(t) and K(t + 1); go2, the second half, whose exponentials are
 *            computed while the first half is multiplied (1,664 rows x 257 keys x 24 heads 21.7 us, all of P
 *            at once 22.0). The issuing warp is one instruction stream of 4 to 5 cycles an
 *            instruction: with a barrier each for P, K, V and Q it needed 3,270 cycles per step of two
 *            groups without a single MMA. P (BF16) overwrites the scores it came from and is the A
 *            operand of P.V; the in-order pipe keeps the next scores behind it. BF16 since V is (one type for
 *            both operands): the results are off by about 0.0023 of themselves, by 0.0017 with F32 probabilities;
 *            the row's sum adds the unrounded ones.
 *   warps 2+ softmax, 8 warps per group: two threads own a row, each 64 of a step's 128 keys and half of
 *            the output; they exchange their maxima through shared memory and a named barrier of their
 *            two warps, which also carries the vote to go on. Scores of a step complete imply that
 *            the group's P.V before them is complete (issued earlier on one pipe), so a raise of the
 *            reference maximum may rescale O at once. While one group computes exponentials, the
 *            tensor pipe works for the other.
 * Keys past the segment get -inf scores by selection; value rows past it that belong to somebody else
 * are cleared in shared memory before P.V reads them (0 * NaN is NaN).
 * Tensor memory: S of group g at 128 g, O behind the scores. All waits are bounded.
 *
 * 6,400 rows x 512 keys x 56 heads: 98 us at 1.8 GHz, 116 in long runs (the power cap's 1.5 GHz), of 57 for the
 * products at the GEMM peak; 50,476 rows 844 of 449. Bound by a group's chain per step, softmax 1,820 cycles and
 * P.V and the next scores 1,620 (of two groups the products are 2,048 cycles, the exponentials 2,048), and 1,900
 * cycles of output per unit beyond a step's. */
constexpr int CT = 128;                              /* rows of a query tile, keys of a key tile */
constexpr int CT_BOX = CT * 64 * 2;                  /* a TMA box: 128 rows x 64 dims            */
constexpr float CT_RAISE = 8.0f;                     /* raise the reference by more than 2^8 only */

template <int D> constexpr int ct_tile() { return CT * D * 2; }
template <int GROUPS> constexpr int ct_stages() { return GROUPS; }
template <int GROUPS> constexpr int ct_threads() { return 64 + 256 * GROUPS; }
constexpr int CT_BARS = 256;
constexpr int CT_OUT = 32 * 64;                      /* output staging of a warp: 32 rows x 32 dims */
template <int GROUPS> constexpr int ct_out() { return GROUPS == 2 ? GROUPS * 8 * CT_OUT : 0; }
template <int GROUPS> constexpr int ct_xchg() { return GROUPS * 2 * CT * 4; }    /* [group][half][row] */
template <int D, int GROUPS> constexpr size_t ct_smem() {
    return size_t(GROUPS + 2 * ct_stages<GROUPS>()) * ct_tile<D>() + ct_out<GROUPS>() + CT_BARS + ct_xchg<GROUPS>();
}
static_assert(ct_smem<128, 2>() <= 232448, "cross attention needs at most 227 KiB of shared memory");
static_assert(2 * (ct_smem<128, 1>() + 1024) <= 233472, "two one-group CTAs per SM");

struct CrossArgs {
    uint16_t *out;
    const uint32_t *segments;
    float *partial_o, *partial_ml;       /* segments in several pieces: [piece][query row][head][D], [piece][query row][head][2] */
    int *status;
    long long wait_cycles;
    uint32_t segment_count, query_rows, key_rows, heads, kv_heads;
    uint32_t pack, pack_log2, head_units;    /* head_units = heads / pack */
    uint32_t units_per_kv;                   /* head units that share a key head */
    uint32_t per_piece;                      /* how the keys of a segment are cut: ct_pieces */
    uint32_t step_h, step_i;                 /* the grid as (head unit, item) digits */
    uint32_t block_stores;                   /* whole tiles leave through map_out */
    float scale_log2;
};

/* The keys of a segment go to this many units, of about the same number of key tiles: tiles / length, rounded up. As
 * the high half of a product with 2^31 / length, rounded down (2 tiles - 1 halves away from every multiple, so exact
 * while tiles * length < 2^30, else a piece fewer): every cursor asks for every segment, and with a division 64
 * segments of one row took 139 instead of 126 us. per_piece 0: one unit. */
__device__ __forceinline__ uint32_t ct_pieces(uint32_t keys, uint32_t per_piece) {
    return 1 + __umulhi(2 * ((max(keys, 1u) - 1) / CT) + 1, per_piece);
}

/* One work unit; every role walks the same units with a cursor of its own */
struct CrossUnit {
    uint32_t q_row, rows;        /* first query row, live query rows (of all groups) */
    uint32_t head0, kv_head;
    uint32_t k_row, keys;        /* first key row of the range; keys of the segment from there on */
    uint32_t steps, piece;
    bool cut;                    /* one of several pieces of the segment's keys */
    bool dirty;                  /* the last tile reaches rows that are not the segment's */
};

template <int GROUPS>
struct CrossCursor {
    uint32_t h, item;               /* the next unit: head unit (fastest), item (a piece of a pair of tiles) */
    uint32_t index, before, items;  /* the segment that item is looked for in, items in front of it, its items */
    uint32_t pieces;
    Segment segment;
    __device__ __forceinline__ void enter(const CrossArgs &a) {
        segment = load_segment(a.segments, index, a.query_rows, a.key_rows);
        const uint32_t per_item = GROUPS * CT >> a.pack_log2;
        pieces = ct_pieces(segment.keys, a.per_piece);
        items = ((segment.queries + per_item - 1) >> ((GROUPS == 2 ? 8 : 7) - a.pack_log2)) * pieces;
    }
    __device__ __forceinline__ explicit CrossCursor(const CrossArgs &a) : index(0), before(0) {
        h = blockIdx.x % a.head_units;
        item = blockIdx.x / a.head_units;
        enter(a);
    }
    __device__ __forceinline__ bool next(const CrossArgs &a, CrossUnit &u) {
        while (item - before >= items) {
            before += items;
            if (++index >= a.segment_count) return false;
            enter(a);
        }
        const uint32_t tiles = (segment.keys + CT - 1) / CT;
        uint32_t at = item - before, t0 = 0, t1 = tiles;
        u.cut = pieces > 1;
        if (u.cut) {
            u.piece = at % pieces;
            at /= pieces;
            t0 = uint32_t(uint64_t(u.piece) * tiles / pieces);
            t1 = uint32_t(uint64_t(u.piece + 1) * tiles / pieces);
        }
        const uint32_t tile_rows = CT >> a.pack_log2, first = at * GROUPS * tile_rows, left = segment.queries - first;
        u.q_row = segment.q0 + first;
        u.rows = min(GROUPS * tile_rows, left);
        u.head0 = h << a.pack_log2;
        u.kv_head = a.units_per_kv == 1 ? h : h / a.units_per_kv;
        u.k_row = segment.k0 + t0 * CT;
        u.keys = segment.keys - t0 * CT;
        u.steps = t1 - t0;
        u.dirty = t1 == tiles && (segment.keys & (CT - 1)) && segment.k0 + segment.keys < a.key_rows;
        h += a.step_h;
        item += a.step_i;
        if (h >= a.head_units) { h -= a.head_units; item++; }
        return true;
    }
};

__device__ __forceinline__ void ct_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void ct_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void ct_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
/* good to 2^-22, far below the BF16 rounding of the probability */
__device__ __forceinline__ float ct_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

/* 32 scores -> 32 probabilities (16 packed columns), their sum added in two packed accumulators */
__device__ __forceinline__ void ct_exponentials(const uint32_t *s, uint64_t scale2, uint64_t neg_m2, uint32_t (&packed)[16],
                                                uint64_t &sum_a, uint64_t &sum_b) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint64_t xa = fma_f32x2(pack_f32x2(__uint_as_float(s[4 * i]), __uint_as_float(s[4 * i + 1])), scale2, neg_m2);
        const uint64_t xb = fma_f32x2(pack_f32x2(__uint_as_float(s[4 * i + 2]), __uint_as_float(s[4 * i + 3])), scale2, neg_m2);
        float x0, x1, x2, x3;
        unpack_f32x2(xa, x0, x1);
        unpack_f32x2(xb, x2, x3);
        const float p0 = ct_exp2(x0), p1 = ct_exp2(x1), p2 = ct_exp2(x2), p3 = ct_exp2(x3);
        sum_a = add_f32x2(sum_a, pack_f32x2(p0, p1));
        sum_b = add_f32x2(sum_b, pack_f32x2(p2, p3));
        packed[2 * i] = pack_bf16(p0, p1);
        packed[2 * i + 1] = pack_bf16(p2, p3);
    }
}

template <int D, int GROUPS>
__global__ void __launch_bounds__(ct_threads<GROUPS>(), GROUPS == 2 ? 1 : 2)
h3b_cross_tc(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
             const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
             const __grid_constant__ CrossArgs args) {
    constexpr int TILE = ct_tile<D>(), STAGES = ct_stages<GROUPS>();
    constexpr uint32_t COL_O = GROUPS * CT, TMEM_COLS = GROUPS * 256;
    extern __shared__ __align__(1024) uint8_t ct_smem_raw[];
    const uint32_t base = smem_u32(ct_smem_raw);
    const uint32_t q_smem = base;                                   /* [group]               */
    const uint32_t k_smem = q_smem + GROUPS * TILE;                 /* [stage]               */
    const uint32_t v_smem = k_smem + STAGES * TILE;                 /* [stage]               */
    const uint32_t out_smem = v_smem + STAGES * TILE;               /* [softmax warp]        */
    const uint32_t bars = out_smem + ct_out<GROUPS>();
    const uint32_t first = bars;                                    /* K(0)                  */
    const uint32_t queries = first + 8;                             /* a unit's query tiles  */
    const uint32_t go = queries + 8;                                /* [group][step % 2] = 4 */
    const uint32_t go2 = go + 32;                                   /* [group][step % 2]: P complete */
    const uint32_t s_full = go2 + 32;                               /* [group] = 2: scores   */
    const uint32_t o_done = s_full + 16;                            /* [group] = 2           */
    const uint32_t seen = o_done + 16;                              /* [step % 2]: scores of all groups seen complete */
    const uint32_t tail = seen + 16;                                /* [step % 2]: V tile that has to be cleared in part */
    const uint32_t holder = tail + 16;
    volatile int *stop = reinterpret_cast<volatile int *>(ct_smem_raw + (holder + 8 - base));
    volatile float *xchg = reinterpret_cast<volatile float *>(ct_smem_raw + (bars - base) + CT_BARS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long budget = args.wait_cycles;
    if ((base & 1023u) != 0) {       /* swizzled tiles need 1024-byte alignment */
        if (threadIdx.x == 0) atomicMax(args.status, int(H3B_STATUS_ATTN_TIMEOUT));
        return;
    }
    if (threadIdx.x == 0) {
        *stop = 0;
        mbar_init(first, 1);
        mbar_init(queries, 1);
        for (int i = 0; i < 2 * GROUPS; i++) {
            mbar_init(go + 8 * i, i < 2 ? 9 : 8);      /* 8 softmax warps, the producer */
            mbar_init(go2 + 8 * i, 8);
        }
        for (int i = 0; i < 2; i++) { mbar_init(seen + 8 * i, 1); mbar_init(tail + 8 * i, 1); }
        for (int g = 0; g < GROUPS; g++) {
            mbar_init(s_full + 8 * g, 1);
            mbar_init(o_done + 8 * g, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_out) : "memory");
    }
    /* The launch in front of this one has ended. Tensor memory is taken behind that, so that nothing in front can wait for
     * it; the merge, which waits for this one's end, may begin. */
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 1) tmem_alloc(holder, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(holder));

    CrossCursor<GROUPS> cursor(args);
    CrossUnit u;
    if (warp == 0) {
        /* ---------------------------------------------------------------- TMA producer */
        if (lane == 0) {
            auto load = [&](const CUtensorMap *map, uint32_t bar, uint32_t dst, uint32_t head, uint32_t row) {
                ct_load(dst, map, bar, 0, int(head), int(row));
                if (D == 128) ct_load(dst + CT_BOX, map, bar, 64, int(head), int(row));
            };
            auto ahead = [&](const CUtensorMap *map, uint32_t head, uint32_t row) {
                for (int box = 0; box < D / 64; box++)
                    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];"
                                 ::"l"(map), "r"(box * 64), "r"(int(head)), "r"(int(row)) : "memory");
            };
            auto next_unit = [&](CrossUnit &n) {
                while (cursor.next(args, n))
                    if (n.steps) return true;
                return false;
            };
            CrossUnit n = {};
            uint32_t t = 0;
            bool have = next_unit(u), alive = true;
            if (have) {
                mbar_expect_tx(queries, GROUPS * TILE);
                for (int g = 0; g < GROUPS; g++)
                    load(&map_q, queries, q_smem + g * TILE, u.head0, u.q_row + g * (CT >> args.pack_log2));
                mbar_expect_tx(first, TILE);
                load(&map_k, first, k_smem + (STAGES - 1) * TILE, u.kv_head, u.k_row);
            }
            /* has step `e`'s "all scores seen" been waited for? (every one is, in order) */
            uint32_t events = 0;
            auto scores_seen = [&](uint32_t e) {
                while (alive && events <= e) {
                    alive = mbar_wait(seen + 8 * (events & 1u), (events >> 1) & 1u, stop, budget);
                    events++;
                }
                return alive;
            };
            while (have && alive) {
                const bool more = next_unit(n);
                /* into L2 by the time the single query buffers are free: from memory the load would take longer
                 * than the last softmax hides (2,800 cycles measured, against 1,000) */
                for (int g = 0; more && g < GROUPS; g++) ahead(&map_q, n.head0, n.q_row + g * (CT >> args.pack_log2));
                for (uint32_t j = 0; j < u.steps; j++, t++) {
                    const bool last = j + 1 == u.steps, dirty = last && u.dirty;
                    /* V(t), K(t + 1) into their stage: V(t - STAGES) and K(t + 1 - STAGES) are dead when the scores
                     * of step t + 1 - STAGES are complete */
                    if (t + 1 >= uint32_t(STAGES) && !scores_seen(t + 1 - STAGES)) break;
                    const uint32_t stage = t % STAGES, bar = go + 8 * (t & 1u);
                    const bool next_k = !last || more;
                    mbar_expect_tx(bar, (dirty ? 0 : TILE) + (next_k ? TILE : 0));
                    if (dirty) mbar_expect_tx(tail + 8 * (t & 1u), TILE);
                    if (next_k)
                        load(&map_k, bar, k_smem + stage * TILE, last ? n.kv_head : u.kv_head, last ? n.k_row : u.k_row + (j + 1) * CT);
                    load(&map_v, dirty ? tail + 8 * (t & 1u) : bar, v_smem + stage * TILE, u.kv_head, u.k_row + j * CT);
                    if (GROUPS == 1) {
                        /* One stage: what the next step loads is on its way into L2 by then (skewed batch of single rows
                         * 48.8 us, without 52.7; one row over 8,192 keys 19.9, 19.2) */
                        if (j + 1 < u.steps) ahead(&map_v, u.kv_head, u.k_row + (j + 1) * CT);
                        if (j + 2 < u.steps) ahead(&map_k, u.kv_head, u.k_row + (j + 2) * CT);
                    }
                    if (last && more) {
                        /* the next queries: their buffers are free when the last scores are complete */
                        if (!scores_seen(t)) break;
                        mbar_expect_tx(queries, GROUPS * TILE);
                        for (int g = 0; g < GROUPS; g++)
                            load(&map_q, queries, q_smem + g * TILE, n.head0, n.q_row + g * (CT >> args.pack_log2));
                    }
                }
                u = n;
                have = more;
            }
        }
    } else if (warp == 1) {
        /* ------------------------------------------------------------------ MMA issuer */
        const uint32_t leader = lane == 0;
        constexpr uint32_t idesc_qk = instruction_desc(CT, CT);
        constexpr uint32_t idesc_pv = instruction_desc(CT, D) | (1u << 16);     /* V is N-major */
        constexpr uint32_t HALF = CT_BOX >> 4, STAGE = TILE >> 4;
        const uint32_t q_lo0 = desc_lo_kmajor(q_smem), k_lo0 = desc_lo_kmajor(k_smem);
        const uint32_t v_lo0 = desc_lo_nmajor(v_smem, CT_BOX);
        auto wait = [&](uint32_t bar, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop, budget));
        };
        using std::integral_constant;
        /* instructions FROM .. TO - 1 of the D / 16 of a group's scores against the K tile of a stage */
        auto issue_qk = [&](auto g_const, auto stage_const, auto from_const, auto to_const) {
            constexpr int g = decltype(g_const)::value, from = decltype(from_const)::value, to = decltype(to_const)::value;
            const uint32_t d = tmem_base + g * CT, q_lo = q_lo0 + g * STAGE, k_lo = k_lo0 + decltype(stage_const)::value * STAGE;
#pragma unroll
            for (int kk = from; kk < to; kk++) {
                if (kk == 0) umma_ss<false>(d, q_lo, k_lo, idesc_qk, leader);
                else umma_ss<true>(d, q_lo + (kk >> 2) * HALF + 2 * (kk & 3), k_lo + (kk >> 2) * HALF + 2 * (kk & 3), idesc_qk, leader);
            }
            if (to == D / 16) umma_commit_if(s_full + 8 * g, leader);
        };
        auto next_unit = [&] {
            uint32_t steps = 0;
            while (!steps && cursor.next(args, u)) steps = u.steps;
            return steps;
        };
        constexpr integral_constant<int, 0> zero{};
        constexpr integral_constant<int, D / 16 - 2> most{};
        constexpr integral_constant<int, D / 16> all{};
        /* steps left of this unit (this one included) and steps of the next */
        uint32_t left = next_unit(), n_steps = 0;
        uint32_t q_phase = 0;
        bool going = left && wait(first, 0) && wait(queries, 0);
        if (going) {
            tc_fence_after();
            issue_qk(zero, integral_constant<int, STAGES - 1>{}, zero, all);
            if constexpr (GROUPS == 2) issue_qk(integral_constant<int, 1>{}, integral_constant<int, STAGES - 1>{}, zero, all);
            q_phase = 1;
            n_steps = next_unit();
        }
        /* Unrolled by the step's parity, so that descriptors and barrier addresses are constants; the
         * barrier that comes next is tested between two MMAs, where that hides behind the pipe. */
        uint32_t phase = 0, ready = 0, start = 1;      /* start: the unit's first step, which overwrites O */
        auto step = [&](auto parity_const) {
            constexpr int PARITY = decltype(parity_const)::value;
            constexpr integral_constant<int, PARITY % STAGES> stage{};
            const bool last = left == 1, more = !last || n_steps;
            auto group = [&](auto g_const) {
                constexpr int g = decltype(g_const)::value;
                if (!__all_sync(0xffffffffu, ready != 0u) && !wait(go + 16 * g + 8 * PARITY, phase)) return false;
                tc_fence_after();
                const uint32_t d = tmem_base + COL_O + g * D, a = tmem_base + g * CT, v_lo = v_lo0 + stage.value * STAGE;
                if (start) umma_ts<false>(d, a, v_lo, idesc_pv, leader);
                else umma_ts<true>(d, a, v_lo, idesc_pv, leader);
                /* P of keys 64.. lies on the columns of their scores; first the halves' first 32 keys */
                auto pv = [&](uint32_t kk) { umma_ts<true>(d, a + (kk >> 2) * 64 + (kk & 3) * 8, v_lo + kk * (2048 >> 4), idesc_pv, leader); };
                pv(1);
                pv(4);
                const uint32_t complete = mbar_test(go2 + 16 * g + 8 * PARITY, phase);
                pv(5);
                if (!__all_sync(0xffffffffu, complete != 0u) && !wait(go2 + 16 * g + 8 * PARITY, phase)) return false;
                tc_fence_after();
                pv(2);
                pv(3);
                pv(6);
                pv(7);
                if (last) {
                    umma_commit_if(o_done + 8 * g, leader);
                    if (g == 0 && more) {                 /* the next unit's queries */
                        if (!wait(queries, q_phase)) return false;
                        q_phase ^= 1;
                        tc_fence_after();
                    }
                }
                if (more) issue_qk(g_const, stage, zero, most);
                if (g + 1 < GROUPS) ready = mbar_test(go + 16 + 8 * PARITY, phase);
                else ready = mbar_test(go + 8 * (PARITY ^ 1), phase ^ PARITY);
                if (more) issue_qk(g_const, stage, most, all);
                return true;
            };
            if (!group(integral_constant<int, 0>{})) return false;
            if constexpr (GROUPS == 2)
                if (!group(integral_constant<int, 1>{})) return false;
            start = last;
            left--;
            if (last) {
                left = n_steps;
                if (left) n_steps = next_unit();
            }
            return left != 0;
        };
        while (going) {
            going = step(zero);
            if (going) going = step(integral_constant<int, 1>{});
            phase ^= 1;
        }
    } else {
        /* --------------------------------------------------------------------- softmax */
        const int g = (warp - 2) >> 3;
        const uint32_t half = ((warp - 2) >> 2) & 1, quarter = warp & 3, local_row = quarter * 32 + lane;
        const uint32_t lane_base = (quarter * 32) << 16;
        const uint32_t tmem_s = tmem_base + g * CT + half * 64 + lane_base;
        const uint32_t tmem_o = tmem_base + COL_O + g * D + half * (D / 2) + lane_base;      /* this thread's half of O */
        const uint32_t pair = 1 + g * 4 + quarter;                                          /* named barrier of a row's two warps */
        volatile float *my_x = xchg + (g * 2 + half) * CT + local_row, *their_x = xchg + (g * 2 + (half ^ 1)) * CT + local_row;
        const float scale_log2 = args.scale_log2;
        const uint64_t scale2 = pack_f32x2(scale_log2, scale_log2);
        /* the two warps of a row meet; both carry on or neither does */
        auto meet = [&](bool ok) {
            uint32_t both;
            asm volatile("{\n\t.reg .pred pin, pout;\n\tsetp.ne.u32 pin, %2, 0;\n\t"
                         "bar.red.and.pred pout, %1, 64, pin;\n\tselp.u32 %0, 1, 0, pout;\n\t}"
                         : "=r"(both) : "r"(pair), "r"(uint32_t(ok)) : "memory");
            return both != 0;
        };
        uint32_t t = 0, o_phase = 0, tail_phase = 0;
        bool alive = true;
        bool have = cursor.next(args, u);
        while (have) {
            const uint32_t tile_rows = CT >> args.pack_log2, row_in_tile = local_row >> args.pack_log2;
            const uint32_t q_row = u.q_row + g * tile_rows;                       /* of the tile */
            const bool live = g * tile_rows + row_in_tile < u.rows, whole = (g + 1) * tile_rows <= u.rows;
            /* (row, head) this thread's accumulators belong to */
            auto unit_of_row = [&] { return size_t(q_row + row_in_tile) * args.heads + u.head0 + (local_row & (args.pack - 1)); };
            const uint32_t steps = u.steps;
            if (!steps) {
                if (live) {            /* no keys: zeros */
                    uint4 *dst = reinterpret_cast<uint4 *>(args.out + unit_of_row() * D + half * (D / 2));
#pragma unroll
                    for (int i = 0; i < D / 16; i++) dst[i] = make_uint4(0, 0, 0, 0);
                }
                have = cursor.next(args, u);
                continue;
            }
            auto clear_tail = [&](uint32_t j) {
                if (!u.dirty || j + 1 != steps || g != 0) return;
                /* value rows that are not the segment's: cleared before anybody's P.V, which is issued
                 * behind this group's arrival */
                const bool ok = __all_sync(0xffffffffu, mbar_wait(tail + 8 * (t & 1u), tail_phase >> (t & 1u) & 1u, stop, budget));
                if (ok && local_row >= u.keys - j * CT) {
                    const uint32_t at = v_smem + (t % STAGES) * TILE + local_row * 128 + (D == 128 ? half * CT_BOX : half * 64);
#pragma unroll
                    for (int i = 0; i < D / 16; i++)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + i * 16), "r"(0) : "memory");
                }
                fence_async_smem();
                tail_phase ^= 1u << (t & 1u);
            };
            /* None of the warp's rows is the segment's: whatever its scores make of its rows of O is stored by nobody, and the
             * others have the exponentials to themselves (64 rows of 300 keys each x 56 heads 121.5 us, 129.4 with
             * the dead rows; 8 x 1,000 keys, dim 64 20.9, 22.6; a ragged batch 76.3, 78.0). */
            const bool idle = g * tile_rows + ((quarter * 32) >> args.pack_log2) >= u.rows;
            float reference = -INFINITY, sum = 0.0f;
            for (uint32_t j = 0; j < steps; j++, t++) {
                const bool ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * g, t & 1u, stop, budget));
                tc_fence_after();
                /* the last group's scores are the last to be complete: the stage before is free */
                if (g == GROUPS - 1 && half == 0 && quarter == 0 && lane == 0) mbar_arrive(seen + 8 * (t & 1u));
                if (idle) {
                    alive = meet(ok);
                    if (!alive) break;
                    clear_tail(j);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(go + 16 * g + 8 * (t & 1u));
                        mbar_arrive(go2 + 16 * g + 8 * (t & 1u));
                    }
                    continue;
                }
                const int valid = int(min(u.keys - j * CT, uint32_t(CT))) - int(half * 64);
                /* 32 scores at a time, read from tensor memory twice (for the maximum, for the exponentials):
                 * holding all 64 spills at the 96 registers there are for 18 warps */
                uint32_t s[32];
                auto scores = [&](int c) {
                    tmem_ld32(tmem_s + 32 * c, s);
                    tmem_ld_wait();
                    if (valid < 32 * c + 32) {
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (32 * c + i >= valid) s[i] = 0xff800000u;      /* -inf */
                    }
                };
                float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
                for (int c = 1; c >= 0; c--) {       /* the first 32 stay in registers */
                    scores(c);
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        m0 = max3_f32(m0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                        m1 = max3_f32(m1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
                        m2 = max3_f32(m2, __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
                        m3 = max3_f32(m3, __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
                    }
                }
                float m_step = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
                /* The row's other half. A slot is read before it is written again: these scores imply P.V of the
                 * step before, which implies that both halves had read theirs. */
                *my_x = m_step;
                alive = meet(ok);
                if (!alive) break;
                m_step = fmaxf(m_step, *their_x) * scale_log2;
                const bool raise = m_step - reference > CT_RAISE;      /* true at the first finite score */
                if (j > 0 && __any_sync(0xffffffffu, raise)) {
                    const float alpha = raise ? ct_exp2(reference - m_step) : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < D / 2; c += 16) {
                        uint32_t o[16];
                        ct_ld16(tmem_o + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        ct_st16(tmem_o + c, o);
                    }
                }
                if (raise) {
                    sum *= ct_exp2(reference - m_step);      /* 0 from -inf */
                    reference = m_step;
                }
                /* a row whose scores are all -inf so far: probabilities 0, not exp2(-inf + inf) */
                const float neg_m = reference == -INFINITY ? 0.0f : -reference;
                const uint64_t neg_m2 = pack_f32x2(neg_m, neg_m);
                uint64_t sum_a = 0, sum_b = 0;
                clear_tail(j);
                /* P of 32 keys lands on columns in front of the scores that are still to be read */
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t packed[16];
                    if (c) scores(c);
                    ct_exponentials(s, scale2, neg_m2, packed, sum_a, sum_b);
                    ct_st16(tmem_s + c * 16, packed);
                    if (c == 0) {
                        tmem_st_wait_all();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(go + 16 * g + 8 * (t & 1u));
                    }
                }
                tmem_st_wait_all();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(go2 + 16 * g + 8 * (t & 1u));
                float s0, s1, s2, s3;
                unpack_f32x2(sum_a, s0, s1);
                unpack_f32x2(sum_b, s2, s3);
                sum += (s0 + s1) + (s2 + s3);
            }
            if (!alive) break;
            /* While P.V runs: the row's sum, through the slots the other way round (each thread writes the one
             * it has read and reads the one it wrote, so nobody's pending read is overwritten) */
            *their_x = sum;
            alive = meet(true);
            if (!alive) break;
            sum += *my_x;
            const size_t unit = unit_of_row();
            const uint32_t head0 = u.head0, piece = u.piece;
            const bool cut = u.cut;
            have = cursor.next(args, u);
            alive = meet(__all_sync(0xffffffffu, mbar_wait(o_done + 8 * g, o_phase, stop, budget)));
            if (!alive) break;
            o_phase ^= 1;
            tc_fence_after();
            if (cut) {
                const size_t at = size_t(piece) * args.query_rows * args.heads + unit;
                if (live && !half) *reinterpret_cast<float2 *>(args.partial_ml + at * 2) = make_float2(reference, sum);
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem_o + c, o);
                    tmem_ld_wait();
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            reinterpret_cast<uint4 *>(args.partial_o + at * D + half * (D / 2) + c)[i] =
                                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            } else {
                /* All scores -inf: zeros; a NaN sum stays NaN. Rows of a whole tile leave through the warp's
                 * staging area and the copy engine, 32 rows x 32 dims at a time: stored row by row they cost
                 * the shared-memory path a cycle per 16 or 32 bytes, and the tensor core reads its operands
                 * through the same path. */
                const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
                const bool block = GROUPS == 2 && whole && args.block_stores;
                const uint32_t area = out_smem + (warp - 2) * CT_OUT, line = area + lane * 64, turn = (lane >> 1) & 3;
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 32) {
                    uint32_t o[32], packed[16];
                    tmem_ld32(tmem_o + c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        packed[i] = pack_bf16(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                    if (block) {
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      /* the area's last block */
                        __syncwarp();
#pragma unroll
                        for (uint32_t i = 0; i < 4; i++)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(line + ((i ^ turn) << 4)),
                                         "r"(packed[4 * i]), "r"(packed[4 * i + 1]), "r"(packed[4 * i + 2]), "r"(packed[4 * i + 3]) : "memory");
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                                         ::"l"(&map_out), "r"(area), "r"(int(half * (D / 2) + c)), "r"(int(head0)),
                                           "r"(int(q_row + (quarter * 32 >> args.pack_log2))) : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    } else if (live) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            reinterpret_cast<uint4 *>(args.out + unit * D + half * (D / 2) + c)[i] =
                                make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
                    }
                }
            }
            /* O has been read: the next unit's P.V waits for this group's next P */
            tc_fence_before();
        }
        if (GROUPS == 2 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*stop) {
        if (threadIdx.x == 0) atomicMax(args.status, int(H3B_STATUS_ATTN_TIMEOUT));
        /* give copies that may still be in flight time to land before the CTA retires */
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem_base, TMEM_COLS);
    }
}

/* out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over a segment's pieces s in order, one warp per (row, head);
 * rows of no segment, and of segments in one piece, are left alone. 32 pieces at a time: their statistics one per lane, their rows loaded
 * eight ahead (one after the other they cost a memory latency each: 20 us for 32). */
template <int D>
__global__ void __launch_bounds__(256)
h3b_cross_merge(const CrossArgs args) {
    using Vector = std::conditional_t<D == 128, float4, float2>;
    constexpr int PER = D / 32;
    const size_t unit = (size_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5, all = size_t(args.query_rows) * args.heads;
    const uint32_t lane = threadIdx.x & 31, row = uint32_t(unit / args.heads);
    /* the segment table is the caller's: no launch of this call writes it */
    uint32_t pieces = 0;
    if (!args.segments) pieces = unit < all ? ct_pieces(args.key_rows, args.per_piece) : 0;
    for (uint32_t i = lane; args.segments && unit < all && i < args.segment_count; i += 32) {
        const Segment s = load_segment(args.segments, i, args.query_rows, args.key_rows);
        if (row - s.q0 < s.queries) pieces = ct_pieces(s.keys, args.per_piece);
    }
    pieces = __reduce_max_sync(0xffffffffu, pieces);
    asm volatile("griddepcontrol.wait;" ::: "memory");      /* every warp: this launch does not end before the one in front */
    if (pieces < 2) return;
    float most = -INFINITY;
    bool nan = false;
    for (uint32_t s = lane; s < pieces; s += 32) {
        const float m = args.partial_ml[(s * all + unit) * 2];
        most = fmaxf(most, m);
        nan = nan || m != m;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (__any_sync(0xffffffffu, nan)) most = NAN;
    float sum = 0.0f, o[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) o[i] = 0.0f;
    for (uint32_t s0 = 0; s0 < pieces; s0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (s0 + lane < pieces) ml = *reinterpret_cast<const float2 *>(args.partial_ml + ((s0 + lane) * all + unit) * 2);
        /* A piece without a score above -inf: weight 0, not 2^(-inf + inf). Its rows take part all the same: they are
         * zeros, and NaN where a value is not finite, as 0 times it is in a segment in one piece. */
        const float weight = ml.x == -INFINITY ? 0.0f : ct_exp2(ml.x - most);
        float part = ml.y * weight;
#pragma unroll
        for (int q = 16; q; q >>= 1) part += __shfl_xor_sync(0xffffffffu, part, q);
        sum += part;
        const uint32_t count = min(32u, pieces - s0);
#pragma unroll 8
        for (uint32_t s = 0; s < count; s++) {
            const Vector v = reinterpret_cast<const Vector *>(args.partial_o + ((s0 + s) * all + unit) * D)[lane];
            const float w = __shfl_sync(0xffffffffu, weight, s);
#pragma unroll
            for (int i = 0; i < PER; i++) o[i] = fmaf(reinterpret_cast<const float *>(&v)[i], w, o[i]);
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint32_t packed[PER / 2];
#pragma unroll
    for (int i = 0; i < PER / 2; i++) packed[i] = pack_bf16(o[2 * i] * inv, o[2 * i + 1] * inv);
#pragma unroll
    for (int i = 0; i < PER / 2; i++) reinterpret_cast<uint32_t *>(args.out + unit * D)[lane * (PER / 2) + i] = packed[i];
}

/* [rows][heads][D] BF16 as a 3-D tensor (dim, head, row); box = box_dims (64 or 32, one swizzled line) x
 * box_heads x box_rows */
bool ct_map(CUtensorMap *map, const uint16_t *data, uint32_t rows, uint32_t heads, uint32_t dim, uint32_t box_dims,
            uint32_t box_heads, uint32_t box_rows) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    cuuint64_t dims[3] = {dim, heads, rows};
    cuuint64_t strides[2] = {cuuint64_t(dim) * 2, cuuint64_t(heads) * dim * 2};
    cuuint32_t box[3] = {box_dims, box_heads, box_rows};
    cuuint32_t elem[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t *>(data), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, box_dims == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

/* cudaFuncSetAttribute belongs to a device; one answer per device and kernel */
template <int D, int GROUPS>
bool ct_configure(int device) {
    static std::mutex mutex;
    static bool done[64];
    std::lock_guard<std::mutex> guard(mutex);
    if (!done[device & 63]) {
        if (cudaFuncSetAttribute(h3b_cross_tc<D, GROUPS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(ct_smem<D, GROUPS>())) != cudaSuccess ||
            cudaFuncSetAttribute(h3b_cross_tc<D, GROUPS>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        done[device & 63] = true;
    }
    return true;
}

template <int D, int GROUPS>
int ct_launch(h3_gpu *gpu, CrossArgs &args, const uint16_t *q, const uint16_t *k, const uint16_t *v) {
    if (!ct_configure<D, GROUPS>(gpu->device)) return h3b_fail(gpu, "cannot reserve shared memory for the cross attention kernel");
    CUtensorMap map_q, map_k, map_v, map_out;
    /* a warp's block of the output is 32 tile rows */
    args.block_stores = args.pack <= 32;
    if (!ct_map(&map_out, args.out, args.query_rows, args.heads, D, 32, args.block_stores ? args.pack : 1,
                args.block_stores ? 32 >> args.pack_log2 : 32) ||
        !ct_map(&map_q, q, args.query_rows, args.heads, D, 64, args.pack, CT >> args.pack_log2) ||
        !ct_map(&map_k, k, args.key_rows, args.kv_heads, D, 64, 1, CT) ||
        !ct_map(&map_v, v, args.key_rows, args.kv_heads, D, 64, 1, CT))
        return h3b_fail(gpu, "cannot encode the cross attention tensor maps");
    const uint64_t per_item = uint64_t(GROUPS) * CT >> args.pack_log2, tiles = (uint64_t(args.key_rows) + CT - 1) / CT;
    const uint64_t resident = uint64_t(gpu->sm_count) * (GROUPS == 2 ? 1 : 2);
    /* The keys of a segment are cut into pieces of about so many key tiles. If rows and keys are spread evenly over the
     * segments: the length with which the rounds of units take least, a unit costing its tiles and two more. One
     * row, 32,768 keys, 8 heads: 37 us with a round's worth of pieces, 58 with three rounds', 460 uncut; 16 rows x
     * 2,048 keys x 32 heads on 8: 34 in two pieces, 41 in three (two rounds). A longer segment than the others is cut
     * to the same pieces (single rows over 512, 77, 2,048 and 1 keys x 56 heads: 25 us, uncut 37), but where CTAs
     * have many units anyway not finer than a CTA's share. Every piece writes its rows in F32 and they are read
     * again: no more of that than there is to read of keys and values (1,000 rows, 16 heads on 2, 700 keys: 26 us in
     * two parts, 19 in one). Two groups: two key tiles or more each. */
    const uint64_t worth = uint64_t(args.key_rows) * args.kv_heads / (uint64_t(args.query_rows) * args.heads * 2);
    const uint64_t spread = (args.query_rows + per_item - 1) / per_item;
    const uint64_t even_units = (spread > args.segment_count ? spread : args.segment_count) * args.head_units;
    const uint64_t even_tiles = (tiles + args.segment_count - 1) / args.segment_count;
    uint64_t piece = even_tiles, least = ~0ull;
    for (uint64_t cuts = 1; cuts * GROUPS <= even_tiles; cuts++) {
        const uint64_t rounds = (even_units * cuts + resident - 1) / resident, length = (even_tiles + cuts - 1) / cuts;
        if (rounds * (GROUPS + 2) >= least) break;           /* no finer cut is faster */
        if (rounds * (length + 2) < least) {
            least = rounds * (length + 2);
            piece = length;
        }
    }
    const uint64_t share = even_units * even_tiles / resident;
    if (piece < share) piece = share;
    if (!worth || piece > tiles) piece = tiles;
    if (worth && piece * worth < tiles) piece = (tiles + worth - 1) / worth;
    const uint64_t pieces = (tiles + piece - 1) / piece;
    args.per_piece = pieces > 1 ? uint32_t((1ull << 31) / piece) : 0;
    /* most units there can be: every segment may end in a part of a tile, and have all key rows */
    const uint64_t units = (args.query_rows / per_item + args.segment_count) * pieces * args.head_units;
    if (units > 0xffffffffull - 2 * resident) return h3b_fail(gpu, "cross attention has too many tiles");
    const unsigned grid = unsigned(units < resident ? units : resident);
    args.step_h = grid % args.head_units;
    args.step_i = grid / args.head_units;
    h3b_scratch scratch(gpu, pieces > 1 ? size_t(pieces) * args.query_rows * args.heads * (D + 2) * sizeof(float) : 0);
    if (pieces > 1) {
        if (!scratch.data) return h3b_fail(gpu, "cross_sdpa_bf16: cannot allocate the partial results");
        args.partial_o = static_cast<float *>(scratch.data);
        args.partial_ml = args.partial_o + size_t(pieces) * args.query_rows * args.heads * D;
    }
    /* Both launches may begin while what is in front of them ends, and wait inside: their set-up comes out of
     * its time. Not the first one while capturing, where an allocation is in front of it. */
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(ct_threads<GROUPS>());
    config.dynamicSmemBytes = ct_smem<D, GROUPS>();
    config.stream = gpu->stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = scratch.captured ? 0 : 1;
    cudaLaunchKernelEx(&config, h3b_cross_tc<D, GROUPS>, map_q, map_k, map_v, map_out, args);      /* an error is reported by h3b_launched */
    if (pieces > 1) {
        const size_t warps = size_t(args.query_rows) * args.heads;
        config.gridDim = dim3(unsigned((warps + 7) / 8));
        config.blockDim = dim3(256);
        config.dynamicSmemBytes = 0;
        config.numAttrs = 1;
        cudaLaunchKernelEx(&config, h3b_cross_merge<D>, args);
    }
    /* the form of the call is part of its name in the op profile */
    const char *name = GROUPS == 2 ? (pieces > 1 ? "cross_sdpa_bf16, two tiles, cut" : "cross_sdpa_bf16, two tiles")
                                   : (pieces > 1 ? "cross_sdpa_bf16, one tile, cut" : "cross_sdpa_bf16, one tile");
    return h3b_launched(gpu, name, H3B_SDPA);
}

bool cross_env_on(const char *name) {
    const char *v = getenv(name);
    return v && *v && strcmp(v, "0") != 0;
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
    if (query_rows > 0x7ffffe00u || key_rows > 0x7ffffe00u) return h3b_fail(gpu, "cross attention has too many rows");
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

    const bool aligned = h3b_aligned16(q) && h3b_aligned16(k) && h3b_aligned16(v) && h3b_aligned16(out);
    if ((head_dim == 64 || head_dim == 128) && aligned && key_rows && scale > 0.0f && !cross_env_on("H3B_SDPA_SIMT")) {
        CrossArgs args = {};
        args.out = out;
        args.segments = table;
        args.status = gpu->status_device;
        args.wait_cycles = gpu->wait_cycles;
        args.segment_count = segment_count;
        args.query_rows = query_rows;
        args.key_rows = key_rows;
        args.heads = heads;
        args.kv_heads = kv_heads;
        const uint32_t group = heads / kv_heads;
        while (args.pack_log2 < 7 && group % (2u << args.pack_log2) == 0) args.pack_log2++;
        args.pack = 1u << args.pack_log2;
        args.head_units = heads / args.pack;
        args.units_per_kv = group / args.pack;
        args.scale_log2 = scale * 1.4426950408889634f;
        /* One group per CTA, two CTAs per SM: where segments hold a tile of rows or less on average, and where units of two
         * tiles would leave more than half of the SMs idle (900 rows x 24 heads x 300 keys, 96 such units: two
         * groups 13.9 us, one 16.0); with head_dim 64, where loads and products are half as long, up to two rounds of
         * them (1,797 rows x 32 heads on 8 x 77 keys, 232 units: 12.0, one group 11.0; 6,400 rows x 56 heads x 77
         * keys, 1,456 units: 33.4, 41.2). */
        const uint64_t tile_rows = CT >> args.pack_log2, pairs = (query_rows / (2 * tile_rows) + segment_count) * args.head_units;
        const uint64_t sms = uint64_t(gpu->sm_count);
        const bool few = query_rows <= segment_count * tile_rows || (head_dim == 64 ? pairs <= 2 * sms : 2 * pairs <= sms);
        if (few) return head_dim == 128 ? ct_launch<128, 1>(gpu, args, q, k, v) : ct_launch<64, 1>(gpu, args, q, k, v);
        return head_dim == 128 ? ct_launch<128, 2>(gpu, args, q, k, v) : ct_launch<64, 2>(gpu, args, q, k, v);
    }
    const size_t smem = (size_t(head_dim) + kSimtThreads) * sizeof(float);
    h3b_cross_simt<<<dim3(query_rows, heads), kSimtThreads, smem, gpu->stream>>>(
        q, k, v, out, table, segment_count, query_rows, key_rows, heads, kv_heads, head_dim, scale);
    return h3b_launched(gpu, "cross_sdpa_bf16, any shape", H3B_SDPA);
}
