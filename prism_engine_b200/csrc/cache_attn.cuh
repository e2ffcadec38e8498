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

// One token's output for one head by one warp in 32 bits, in three passes: the largest score, the sum of the weights, the values over that
// sum, which is no larger than the largest of them (values near bf16's largest overflow the sums of the other kernels).  What the formula
// gives for infinities and NaN is what this gives; positions that the row does not see take no part.  Scores are a position a lane, the
// values' sums HD / 32 columns a lane: bound by the latency of the loads, once for 32 positions (60000 positions of a 64-wide head, 256 rows
// by the 20 warps of a block: 342 ms; a position at a time by the whole warp 1610 ms).
template <int KIND, int HD>
__device__ __noinline__ void cache_plain_row(const CacheAttnDev &a, const CacheEntry &x, uint32_t token, uint32_t head, uint32_t lane) {
    constexpr int VEC = HD / 32, PIECE = 128 / (int)kv_bits<KIND>();  // columns of a lane; values of 16 bytes
    constexpr uint32_t ROWB = HD * kv_bits<KIND>() / 8, ALL = 0xFFFFFFFFu;
    const uint32_t kh = head / a.group, col = lane * VEC;
    const CacheRow r = cache_row(a, x, token);
    const uint16_t *q = a.q + (size_t)(x.row0 + token) * a.q_stride + (size_t)head * HD;
    float acc[VEC], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; i++) acc[i] = 0.0f;
    bool any = false;
    const int32_t gap_lo = (int32_t)min(a.sinks, 0x7FFFFFFFu), gap_hi = min(r.low, x.first - 1);  // what the window leaves out
    for (int pass = 0; pass < 3; pass++) {
        for (int32_t p0 = 0; p0 < x.len; p0 += 32) {
            if (p0 >= gap_lo && p0 + 31 <= gap_hi) {       // none of these 32: on to those that gap_hi + 1 is one of
                p0 = (gap_hi + 1) / 32 * 32 - 32;
                continue;
            }
            const int32_t p = p0 + (int32_t)lane;
            uint32_t page = 0;
            const bool see = cache_sees(a, x, r, p) && kv_page(a.c, x.seq, (uint32_t)p, page);
            unsigned long long at = 0;
            float d = 0.0f;
            if (see) {
                at = kv_row(a.c, page, kh, (uint32_t)p);
                const uint4 *row = reinterpret_cast<const uint4 *>(a.c.k + at * ROWB);
#pragma unroll 2
                for (int c = 0; c < HD / PIECE; c++) {
                    const uint4 w = __ldg(row + c);
                    float k[PIECE];
                    kv_values<KIND, PIECE>(reinterpret_cast<const uint8_t *>(&w), a.c.ks + at * kv_scales<KIND>(), 0, k);
#pragma unroll
                    for (int i = 0; i < PIECE; i++) d = fmaf(kv_row_value(__ldg(q + c * PIECE + i), a.c.rows_bf16), k[i], d);
                }
                d *= a.scale;
                any = true;
            }
            if (pass == 0) {
                if (see) top = fmaxf(top, d);
            } else if (pass == 1) {
                if (see) sum += expf(d - top);
            } else {
                const float w = see ? expf(d - top) / sum : 0.0f;
                const uint32_t seen = __ballot_sync(ALL, see);
#pragma unroll 8
                for (int u = 0; u < 32; u++) {
                    const float f = __shfl_sync(ALL, w, u);
                    const unsigned long long from = __shfl_sync(ALL, at, u);
                    if (seen >> u & 1) {
                        float v[VEC];
                        kv_values<KIND, VEC>(a.c.v + from * ROWB, a.c.vs + from * kv_scales<KIND>(), col, v);
#pragma unroll
                        for (int i = 0; i < VEC; i++) acc[i] = fmaf(f, v[i], acc[i]);
                    }
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            if (pass == 0) top = fmaxf(top, __shfl_xor_sync(ALL, top, o));
            if (pass == 1) sum += __shfl_xor_sync(ALL, sum, o);
        }
    }
    any = __any_sync(ALL, any);
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
