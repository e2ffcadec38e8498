// Joining the parts that several blocks left of the same query rows (cache_attn.cu, cache_attn_tc5.cu).
#pragma once

#include <algorithm>

#include "cache_attn.cuh"

namespace prism {

// A part of `rows` query rows: [HD / 4][rows][4] sums of weight times value, then the rows' maxima (in powers of two), then their sums of
// weights, all on those maxima.
__host__ __device__ constexpr size_t cache_part_floats(uint32_t rows, uint32_t hd) { return (size_t)rows * (hd + 2); }

struct CacheJoinDev {
    CacheAttnDev a;
    uint32_t splits, tiles, rows;  // parts of a row tile, row tiles of an entry and head, rows of a tile
    const float *part;             // [item][split]
};

constexpr uint32_t CJ_THREADS = 256, CJ_ROWS = 8, CJ_MAX_SPLIT = 256;

// A block takes 8 rows: weights of their parts, then every thread its groups of four columns over all parts in order.  A row
// whose result is not finite is taken again by itself.  Bound: L2, the parts are read where they were just written.
template <int KIND, int HD>
__global__ void __launch_bounds__(CJ_THREADS) cache_join_kernel(const __grid_constant__ CacheJoinDev d) {
    __shared__ float wgt[CJ_MAX_SPLIT][CJ_ROWS];
    __shared__ float sums[CJ_ROWS];
    __shared__ uint32_t again;
    const CacheAttnDev &a = d.a;
    constexpr uint32_t R = CJ_ROWS;
    const uint32_t tid = threadIdx.x, item = blockIdx.y, r0 = blockIdx.x * R;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tile = item % d.tiles, kh = item / d.tiles % a.c.kv_heads, e = item / d.tiles / a.c.kv_heads;
    CacheEntry x;
    if (!cache_entry(a, e, x)) return;
    const uint32_t n_rows = x.n * a.group, first = tile * d.rows + r0;
    if (first >= n_rows) return;
    const uint32_t here = min(R, n_rows - first);
    const size_t size = cache_part_floats(d.rows, HD);
    const float *all = d.part + (size_t)item * d.splits * size;
    {
        const uint32_t r = tid >> 5, k = tid & 31;                     // a warp a row
        const float *ml = all + (size_t)d.rows * HD + r0 + r;
        float top = -INFINITY, sum = 0.0f;
        for (uint32_t s = k; s < d.splits; s += 32) top = fmaxf(top, __ldcg(ml + s * size));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const float sub = top == -INFINITY ? 0.0f : top;
        for (uint32_t s = k; s < d.splits; s += 32) {
            const float f = exp2f(__ldcg(ml + s * size) - sub);
            wgt[s][r] = f;
            sum += __ldcg(ml + s * size + d.rows) * f;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (k == 0) sums[r] = sum;
        if (tid == 0) again = 0;
    }
    __syncthreads();
    for (uint32_t u = tid; u < R * (HD / 4); u += CJ_THREADS) {
        const uint32_t r = u % R, c = u / R;
        const float4 *p = reinterpret_cast<const float4 *>(all) + (size_t)c * d.rows + r0 + r;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (uint32_t s = 0; s < d.splits; s++) {
            const float4 w = __ldcg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + s * size));
            const float f = wgt[s][r];
            v.x = fmaf(w.x, f, v.x);
            v.y = fmaf(w.y, f, v.y);
            v.z = fmaf(w.z, f, v.z);
            v.w = fmaf(w.w, f, v.w);
        }
        if (r >= here) continue;
        const float inv = 1.0f / sums[r];
        v.x *= inv;
        v.y *= inv;
        v.z *= inv;
        v.w *= inv;
        if (!(sums[r] > 0.0f) || !isfinite(v.x) || !isfinite(v.y) || !isfinite(v.z) || !isfinite(v.w)) {
            atomicOr(&again, 1u << r);
            continue;
        }
        const uint32_t rr = first + r;
        uint16_t *dst = a.out + (size_t)(x.row0 + rr / a.group) * a.out_stride + (size_t)(kh * a.group + rr % a.group) * HD + c * 4;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(kv_round2(v.x, v.y, a.c.rows_bf16), kv_round2(v.z, v.w, a.c.rows_bf16));
    }
    __syncthreads();
    for (uint32_t r = tid >> 5; r < here; r += CJ_THREADS / 32)
        if (again >> r & 1) cache_plain_row<KIND, HD>(a, x, (first + r) / a.group, kh * a.group + (first + r) % a.group, tid & 31);
}

template <int KIND, int HD>
inline int launch_cache_join(prism_cuda_ctx *ctx, const CacheJoinDev &d) {
    const uint32_t items = d.a.n_entries * d.a.c.kv_heads * d.tiles;  // fewer than the GPU has room for: at most 65535
    launch_pdl(ctx, "cache_join_kernel", cache_join_kernel<KIND, HD>, dim3((d.rows + CJ_ROWS - 1) / CJ_ROWS, items), dim3(CJ_THREADS), 0, d);
    return after_launch(ctx, "cache_join_kernel");
}

}  // namespace prism
