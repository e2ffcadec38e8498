// What the kernels of attention over a caller-owned cache share: the call, the entries, which positions a row sees, and a row taken
// position by position.
#pragma once

#include "kv_cache.cuh"

namespace prism {

struct CacheAttnDev {
    KvDev c;
    const uint16_t *q;
    uint16_t *out;
    uint64_t q_stride, out_stride;
    uint32_t n_rows, n_entries;
    const int32_t *seq, *q_start, *length;
    uint32_t max_tokens;
    uint32_t heads, group;   // query heads, and how many share a cached one
    uint32_t window, sinks;
    float scale;
    const uint64_t *tree;
    uint32_t tree_words;
    const int32_t *q_pos;
};

#ifdef __CUDACC__
// An entry after its checks: rows row0 .. row0 + n - 1, positions 0 .. len - 1, the first `first` of them committed.
struct CacheEntry {
    uint32_t seq, row0, n;
    int32_t len, first;
};
__device__ __forceinline__ bool cache_entry(const CacheAttnDev &a, uint32_t e, CacheEntry &x) {
    const int32_t s = __ldg(a.seq + e), r0 = __ldg(a.q_start + e), r1 = __ldg(a.q_start + e + 1), len = __ldg(a.length + e);
    if (s < 0 || r1 == r0) return false;
    if ((uint32_t)s >= a.c.n_seqs || r0 < 0 || r1 < r0 || (uint32_t)r1 > a.n_rows || (uint32_t)(r1 - r0) > a.max_tokens || len < 0 ||
        (uint32_t)len > (a.c.stride << a.c.shift)) {
        kv_flag(a.c);
        return false;
    }
    x.seq = (uint32_t)s;
    x.row0 = (uint32_t)r0;
    x.n = (uint32_t)(r1 - r0);
    x.len = len;
    x.first = len - (int32_t)x.n;
    return true;
}

// Where a row stands: a position c is visible if c <= last and (c > low or c < sinks), c < len throughout; of a tree's drafted
// positions (c >= first) the row's mask says it.
struct CacheRow {
    int32_t last, low;
    const uint64_t *mask;
};
__device__ __forceinline__ CacheRow cache_row(const CacheAttnDev &a, const CacheEntry &x, uint32_t token) {
    CacheRow r;
    const uint32_t row = x.row0 + token;
    r.mask = a.tree ? a.tree + (size_t)row * a.tree_words : nullptr;
    const int32_t at = x.first + (int32_t)token;
    r.last = a.tree ? x.first - 1 : at;
    // in 64 bits: a window may be larger than any position
    r.low = a.window ? (int32_t)max((int64_t)(a.tree ? __ldg(a.q_pos + row) : at) - (int64_t)a.window, (int64_t)-1) : -1;
    return r;
}
__device__ __forceinline__ bool cache_sees(const CacheAttnDev &a, const CacheEntry &x, const CacheRow &r, int32_t c) {
    if (c < 0 || c >= x.len) return false;
    if (r.mask && c >= x.first) {
        const uint32_t j = (uint32_t)(c - x.first);  // below n, and so below 64 * tree_words
        return __ldg(r.mask + (j >> 6)) >> (j & 63) & 1;
    }
    return c <= r.last && (c > r.low || (uint32_t)c < a.sinks);
}

// One token's output for one head by one warp in 32 bits, position by position, in three passes: the largest score, the sum of the weights, the
// values over that sum, which is no larger than the largest of them (values near bf16's largest overflow the sums of the other kernels).  What the formula gives for infinities and NaN is what this gives; positions that the row does not see take no part.
template <int KIND, int HD>
__device__ __noinline__ void cache_plain_row(const CacheAttnDev &a, const CacheEntry &x, uint32_t token, uint32_t head, uint32_t lane) {
    constexpr int VEC = HD / 32;
    constexpr uint32_t ROWB = HD * kv_bits<KIND>() / 8;
    const uint32_t kh = head / a.group, col = lane * VEC;
    const CacheRow r = cache_row(a, x, token);
    float q[VEC], acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        q[i] = kv_row_value(a.q[(size_t)(x.row0 + token) * a.q_stride + (size_t)head * HD + col + i], a.c.rows_bf16);
        acc[i] = 0.0f;
    }
    float top = -INFINITY, sum = 0.0f;
    bool any = false;
    for (int pass = 0; pass < 3; pass++) {
        // positions that no row under this window sees are stepped over
        const int32_t gap_lo = (int32_t)min(a.sinks, 0x7FFFFFFFu), gap_hi = min(r.low, x.first - 1);
        for (int32_t p = 0; p < x.len; p++) {
            if (p >= gap_lo && p <= gap_hi) {
                p = gap_hi;
                continue;
            }
            uint32_t page;
            if (!cache_sees(a, x, r, p) || !kv_page(a.c, x.seq, (uint32_t)p, page)) continue;
            const size_t at = kv_row(a.c, page, kh, (uint32_t)p);
            float k[VEC], v[VEC], d = 0.0f;
            kv_values<KIND, VEC>(a.c.k + at * ROWB, a.c.ks + at * kv_scales<KIND>(), col, k);
#pragma unroll
            for (int i = 0; i < VEC; i++) d = fmaf(q[i], k[i], d);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
            d *= a.scale;
            any = true;
            if (pass == 0) {
                top = fmaxf(top, d);
            } else if (pass == 1) {
                sum += expf(d - top);
            } else {
                const float w = expf(d - top) / sum;
                kv_values<KIND, VEC>(a.c.v + at * ROWB, a.c.vs + at * kv_scales<KIND>(), col, v);
#pragma unroll
                for (int i = 0; i < VEC; i++) acc[i] = fmaf(w, v[i], acc[i]);
            }
        }
    }
    uint16_t *dst = a.out + (size_t)(x.row0 + token) * a.out_stride + (size_t)head * HD + col;
#pragma unroll
    for (int i = 0; i < VEC; i++) dst[i] = kv_round(any ? acc[i] : 0.0f, a.c.rows_bf16);
}
#endif

// Scratch of a call (cache_attn.cu): `part_bytes` and `counts` counters that are zero.
int cache_scratch(prism_cuda_ctx *ctx, size_t part_bytes, size_t counts, float **part, unsigned int **count);
// cache_attn_tc5.cu: many rows per cached head; cache_tiles_fit: head size and pool are for it
bool cache_tiles_fit(const CacheAttnDev &a, uint32_t hd);
int launch_cache_tiles(prism_cuda_ctx *ctx, int kind, uint32_t hd, const CacheAttnDev &a, uint32_t max_length);

}  // namespace prism
