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

constexpr uint32_t CJ_THREADS = 256, CJ_MAX_SPLIT = 256, CJ_FEW = 8;
template <int HD, bool MANY>
constexpr uint32_t CJ_ROWS = MANY ? 2 : CJ_THREADS * 4 / HD;

// A block takes some rows: weights of their parts, then every thread four columns over its group's share of the parts, in order.  A row
// whose result is not finite is taken again by itself.  Bound: L2, the parts are read where they were just written, and its latency.
// MANY: two rows, whose parts several groups of threads share (64 rows of 128 in 55 parts: 8 rows a block 10 us, two 5 us; 14 rows of 64
// in 222 parts: 17 and 3 us).  To CJ_FEW parts: a group that fills the block (16384 rows of 128 in two parts: two rows a block 24 us, eight 8 us).
template <int KIND, int HD, bool MANY>
__global__ void __launch_bounds__(CJ_THREADS) cache_join_kernel(const __grid_constant__ CacheJoinDev d) {
    constexpr uint32_t R = CJ_ROWS<HD, MANY>, GROUPS = CJ_THREADS / (R * HD / 4);
    __shared__ float wgt[MANY ? CJ_MAX_SPLIT : CJ_FEW][R];
    __shared__ float sums[R];
    __shared__ float4 group_sum[GROUPS > 1 ? CJ_THREADS : 1];
    __shared__ uint32_t again;
    const CacheAttnDev &a = d.a;
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
    if (tid == 0) again = 0;
    for (uint32_t r = tid >> 5; r < R; r += CJ_THREADS / 32) {         // a warp a row
        const uint32_t k = tid & 31;
        const float *ml = all + (size_t)d.rows * HD + r0 + r;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll 4
        for (uint32_t s = k; s < d.splits; s += 32) top = fmaxf(top, __ldcg(ml + s * size));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const float sub = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
        for (uint32_t s = k; s < d.splits; s += 32) {
            const float f = exp2f(__ldcg(ml + s * size) - sub);
            wgt[s][r] = f;
            sum += __ldcg(ml + s * size + d.rows) * f;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (k == 0) sums[r] = sum;
    }
    const uint32_t r = tid % R, c = tid / R % (HD / 4), group = tid / (R * HD / 4);
    const float *p = all + ((size_t)c * d.rows + r0 + r) * 4;
    const uint32_t s_lo = d.splits * group / GROUPS, s_hi = d.splits * (group + 1) / GROUPS;
    __syncthreads();
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (uint32_t s = s_lo; s < s_hi; s++) {
        const float4 w = __ldcg(reinterpret_cast<const float4 *>(p + s * size));
        const float f = wgt[s][r];
        v.x = fmaf(w.x, f, v.x);
        v.y = fmaf(w.y, f, v.y);
        v.z = fmaf(w.z, f, v.z);
        v.w = fmaf(w.w, f, v.w);
    }
    if constexpr (GROUPS > 1) {
        group_sum[tid] = v;
        __syncthreads();
    }
    if (group == 0 && r < here) {
#pragma unroll
        for (uint32_t i = 1; i < GROUPS; i++) {
            const float4 w = group_sum[i * (R * HD / 4) + tid];
            v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
        }
        const float inv = 1.0f / sums[r];
        v.x *= inv;
        v.y *= inv;
        v.z *= inv;
        v.w *= inv;
        if (!(sums[r] > 0.0f) || !isfinite(v.x) || !isfinite(v.y) || !isfinite(v.z) || !isfinite(v.w)) {
            atomicOr(&again, 1u << r);
        } else {
            const uint32_t rr = first + r;
            uint16_t *dst = a.out + (size_t)(x.row0 + rr / a.group) * a.out_stride + (size_t)(kh * a.group + rr % a.group) * HD + c * 4;
            *reinterpret_cast<uint2 *>(dst) = make_uint2(kv_round2(v.x, v.y, a.c.rows_bf16), kv_round2(v.z, v.w, a.c.rows_bf16));
        }
    }
    __syncthreads();
    for (uint32_t r = tid >> 5; r < here; r += CJ_THREADS / 32)
        if (again >> r & 1) cache_plain_row<KIND, HD>(a, x, (first + r) / a.group, kh * a.group + (first + r) % a.group, tid & 31);
}

template <int KIND, int HD>
inline int launch_cache_join(prism_cuda_ctx *ctx, const CacheJoinDev &d) {
    const uint32_t items = d.a.n_entries * d.a.c.kv_heads * d.tiles;  // fewer than the GPU has room for: at most 65535
    auto go = [&](auto kernel, uint32_t rows) {
        launch_pdl(ctx, "cache_join_kernel", kernel, dim3((d.rows + rows - 1) / rows, items), dim3(CJ_THREADS), 0, d);
    };
    if (d.splits > CJ_FEW) go(cache_join_kernel<KIND, HD, true>, (uint32_t)CJ_ROWS<HD, true>);
    else go(cache_join_kernel<KIND, HD, false>, (uint32_t)CJ_ROWS<HD, false>);
    return after_launch(ctx, "cache_join_kernel");
}

}  // namespace prism
