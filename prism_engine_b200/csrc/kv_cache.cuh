// A caller-owned key/value cache of several sequences (prism_cache, include/prism_cuda.h) as the kernels see it: a pool of pages
// [page][kv head][position in page][head], 16-bit values or 8- / 4-bit codes, and beside codes 32-bit scales
// [page][kv head][position in page].
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace prism {

// What a cached value is held in: the two 16-bit kinds of row, then the codes.
enum KvKind { KV_F16 = 0, KV_BF16 = 1, KV_INT8 = 2, KV_E4M3 = 3, KV_INT4 = 4 };

template <int KIND>
__host__ __device__ constexpr uint32_t kv_bits() { return KIND <= KV_BF16 ? 16 : KIND == KV_INT4 ? 4 : 8; }
// 32-bit numbers of a head of one position: a scale, or a scale and a zero
template <int KIND>
__host__ __device__ constexpr uint32_t kv_scales() { return KIND <= KV_BF16 ? 0 : KIND == KV_INT4 ? 2 : 1; }

struct KvDev {
    uint8_t *k, *v;
    float *ks, *vs;
    const int32_t *table;    // [n_seqs][stride] page numbers, or nullptr: sequence s owns pages s * stride ..
    uint32_t shift, stride, n_pages, n_seqs, kv_heads;
    uint32_t rows_bf16;      // rows (q, k, v, outputs) are bf16, not fp16
    unsigned int *err;       // the context's error word: code 8, a place outside the cache was skipped
};

#ifdef __CUDACC__
__device__ __forceinline__ void kv_flag(const KvDev &c) { atomicExch(c.err, 8u); }

// Page of position p of sequence s, both inside the cache's bounds, as the table has it; whether it is one (if not, the error word is set).
__device__ __forceinline__ uint32_t kv_page_number(const KvDev &c, uint32_t s, uint32_t p) {
    const uint32_t at = p >> c.shift;
    return c.table ? (uint32_t)__ldg(c.table + (size_t)s * c.stride + at) : s * c.stride + at;
}
__device__ __forceinline__ bool kv_page_ok(const KvDev &c, uint32_t page) {
    if (page < c.n_pages) return true;
    kv_flag(c);
    return false;
}
__device__ __forceinline__ bool kv_page(const KvDev &c, uint32_t s, uint32_t p, uint32_t &page) {
    page = kv_page_number(c, s, p);
    return kv_page_ok(c, page);
}
// Row of a head of a page's position: rows are what codes and scales are counted in.
__device__ __forceinline__ size_t kv_row(const KvDev &c, uint32_t page, uint32_t head, uint32_t p) {
    return (((size_t)page * c.kv_heads + head) << c.shift) + (p & ((1u << c.shift) - 1u));
}
// The row of (sequence, position) for a list of places: 1 = there, 0 = none (a negative number: padding; outside the cache: also flagged).
__device__ __forceinline__ bool kv_place(const KvDev &c, int32_t s, int32_t p, uint32_t &page) {
    if (s < 0 || p < 0) return false;
    if ((uint32_t)s >= c.n_seqs || ((uint32_t)p >> c.shift) >= c.stride) {
        kv_flag(c);
        return false;
    }
    return kv_page(c, (uint32_t)s, (uint32_t)p, page);
}

__device__ __forceinline__ float kv_f16(uint16_t v) { return __half2float(__ushort_as_half(v)); }
__device__ __forceinline__ float kv_row_value(uint16_t v, bool bf16) { return bf16 ? __uint_as_float((uint32_t)v << 16) : kv_f16(v); }
__device__ __forceinline__ uint16_t kv_round(float v, bool bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ uint32_t kv_round2(float a, float b, bool bf16) {  // a in the low half
    return (uint32_t)kv_round(a, bf16) | (uint32_t)kv_round(b, bf16) << 16;
}

// N values from column `at` of a cached row (codes at `row`, its scales at `sc`); N even for 4-bit codes.
template <int KIND, int N>
__device__ __forceinline__ void kv_values(const uint8_t *row, const float *sc, uint32_t at, float (&out)[N]) {
    if constexpr (KIND <= KV_BF16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(row) + at;
#pragma unroll
        for (int i = 0; i < N; i++) out[i] = kv_row_value(p[i], KIND == KV_BF16);
    } else if constexpr (KIND == KV_INT4) {
        const float s = sc[0], z = sc[1];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t b = row[(at + i) >> 1], c = (at + i) & 1 ? b >> 4 : b & 15;
            out[i] = __fadd_rn(__fmul_rn((float)((int)c - 8), s), z);
        }
    } else {
        const float s = sc[0];
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (KIND == KV_INT8) out[i] = __fmul_rn((float)(int8_t)row[at + i], s);
            else out[i] = __fmul_rn(__half2float(__half(__nv_cvt_fp8_to_halfraw(row[at + i], __NV_E4M3))), s);
        }
    }
}
#endif

// Whether arrays of 32-bit numbers lie on 4-byte boundaries; others would fault the kernels that read them.
template <typename... P>
inline bool kv_words(const P *...p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & 3) == 0; }

// The library's own record of a prism_cache, after its checks.
int kv_check(prism_cuda_ctx *ctx, const prism_cache *c, KvDev *out, int *kind);

// The context's device for the length of a call; the caller's afterwards.
struct DeviceGuard {
    int before = -1;
    cudaError_t err;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) (void)cudaSetDevice(before);
    }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;
};

}  // namespace prism
