// Writing rows of keys and values into a caller-owned cache (prism_cache), quantised to 8 or 4 bits as they are written, reading
// them back, and moving accepted drafted tokens up behind the committed ones.
//
//   int8   scale = amax / 127, code = rint(x * (127 / amax))             amax, lo, hi: over one head of one position
//   e4m3   scale = amax / 448, code = e4m3(x * (448 / amax))
//   int4   scale = (hi - lo) / 15, zero = lo + 8 scale, code = rint((x - lo) * (15 / (hi - lo))), value = (code - 8) scale + zero
//
// Every step is one rounded 32-bit operation, so codes and scales are the same numbers wherever they are computed.  A span below
// 2^-100 (its reciprocal would overflow) is written with scale 0; a head with a value that is not finite gets the scale NaN.
//
// A head of one position is a unit of hd / 8 lanes with 16 bytes of the row each: its extremes take log2(hd / 8) shuffles, and
// loads and stores of neighbouring heads are whole lines.  Bound: HBM for long lists, launch latency for a decode step's rows; a
// thread has KV_UNITS units in flight.
#include <stdexcept>

#include "kv_cache.cuh"

namespace prism {

constexpr uint32_t KV_THREADS = 256, KV_UNITS = 4;

struct KvRowsDev {
    KvDev c;
    uint16_t *k, *v;             // rows, k_stride / v_stride values apart
    uint64_t k_stride, v_stride;
    const int32_t *seq, *pos;    // place of every row
    uint32_t units;              // n_rows * 2 * kv_heads
};

namespace {

template <int LANES>
__device__ __forceinline__ float kv_max_of(float v) {
#pragma unroll
    for (int x = LANES / 2; x > 0; x >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, x));
    return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t kv_umax_of(uint32_t v) {
#pragma unroll
    for (int x = LANES / 2; x > 0; x >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, x));
    return v;
}

// Unit u of a list: its row, which of k and v, and its head.
__device__ __forceinline__ void kv_unit(uint32_t u, uint32_t heads, uint32_t &row, uint32_t &which, uint32_t &head) {
    const uint32_t t = u / heads;
    head = u - t * heads;
    which = t & 1;
    row = t >> 1;
}

// Codes of 8 values of a head that LANES lanes share, and the head's scales (the same in all its lanes).
template <int KIND, int LANES>
__device__ __forceinline__ uint2 kv_encode(const float (&x)[8], float &scale, float &zero) {
    constexpr float TOP = KIND == KV_INT8 ? 127.0f : KIND == KV_E4M3 ? 448.0f : 15.0f;
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) big = max(big, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    big = kv_umax_of<LANES>(big);            // as integers: NaN above infinity above every number
    float lo = 0.0f, span = __uint_as_float(big);
    if (KIND == KV_INT4) {
        float hi = x[0];
        lo = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
        }
        lo = -kv_max_of<LANES>(-lo);
        hi = kv_max_of<LANES>(hi);
        span = __fsub_rn(hi, lo);
    }
    const bool real = span >= 0x1p-100f, odd = big >= 0x7F800000u || __float_as_uint(span) >= 0x7F800000u;
    scale = real ? __fdiv_rn(span, TOP) : 0.0f;
    const float inv = real && !odd ? __fdiv_rn(TOP, span) : 0.0f;
    if (KIND == KV_INT4) zero = __fadd_rn(lo, __fmul_rn(8.0f, scale));
    if (odd) scale = zero = __uint_as_float(0x7FC00000u);
    uint32_t w[2] = {0, 0};
    if (KIND == KV_INT4) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = real && !odd ? __float2int_rn(__fmul_rn(__fsub_rn(x[i], lo), inv)) : 8;
            w[0] |= (uint32_t)c << (4 * i);
        }
    } else if (odd) {
        // codes 0
    } else if (KIND == KV_INT8) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i >> 2] |= (uint32_t)(__float2int_rn(__fmul_rn(x[i], inv)) & 0xFF) << (8 * (i & 3));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[2 * i], inv), __fmul_rn(x[2 * i + 1], inv)), __NV_SATFINITE, __NV_E4M3)
                         << (16 * (i & 1));
    }
    return make_uint2(w[0], w[1]);
}

}  // namespace

template <int KIND, int HD>
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const KvRowsDev a) {
    constexpr uint32_t LANES = HD / 8, PER = KV_THREADS / LANES, ROWB = HD * kv_bits<KIND>() / 8;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x % LANES, first = blockIdx.x * PER * KV_UNITS + threadIdx.x / LANES;
    uint4 data[KV_UNITS];
    size_t to[KV_UNITS];
    bool there[KV_UNITS];
    uint32_t which[KV_UNITS];
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        const uint32_t u = first + j * PER;
        uint32_t row, head, page = 0;
        kv_unit(min(u, a.units - 1), a.c.kv_heads, row, which[j], head);
        const int32_t s = __ldg(a.seq + row), p = __ldg(a.pos + row);
        data[j] = __ldg(reinterpret_cast<const uint4 *>((which[j] ? a.v + row * a.v_stride : a.k + row * a.k_stride) + head * HD) + lane);
        there[j] = u < a.units && kv_place(a.c, s, p, page);
        to[j] = there[j] ? kv_row(a.c, page, head, (uint32_t)p) : 0;
    }
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        uint8_t *dst = (which[j] ? a.c.v : a.c.k) + to[j] * ROWB;
        if constexpr (KIND <= KV_BF16) {
            if (there[j]) reinterpret_cast<uint4 *>(dst)[lane] = data[j];
        } else {
            float x[8], scale, zero = 0.0f;
            const uint32_t w[4] = {data[j].x, data[j].y, data[j].z, data[j].w};
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = kv_row_value((uint16_t)(w[i >> 1] >> (16 * (i & 1))), a.c.rows_bf16);
            const uint2 codes = kv_encode<KIND, LANES>(x, scale, zero);  // every lane of the warp takes part
            if (!there[j]) continue;
            float *sc = (which[j] ? a.c.vs : a.c.ks) + to[j] * kv_scales<KIND>();
            if constexpr (KIND == KV_INT4) {
                reinterpret_cast<uint32_t *>(dst)[lane] = codes.x;
                if (lane == 0) *reinterpret_cast<float2 *>(sc) = make_float2(scale, zero);
            } else {
                reinterpret_cast<uint2 *>(dst)[lane] = codes;
                if (lane == 0) *sc = scale;
            }
        }
    }
}

template <int KIND, int HD>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const KvRowsDev a) {
    constexpr uint32_t LANES = HD / 8, PER = KV_THREADS / LANES, ROWB = HD * kv_bits<KIND>() / 8;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x % LANES, first = blockIdx.x * PER * KV_UNITS + threadIdx.x / LANES;
    uint4 data[KV_UNITS];
    float2 sc[KV_UNITS];
    bool there[KV_UNITS];
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        const uint32_t u = first + j * PER;
        uint32_t row, which, head, page = 0;
        kv_unit(min(u, a.units - 1), a.c.kv_heads, row, which, head);
        const int32_t s = __ldg(a.seq + row), p = __ldg(a.pos + row);
        there[j] = u < a.units && kv_place(a.c, s, p, page);
        data[j] = make_uint4(0, 0, 0, 0);
        sc[j] = make_float2(0.0f, 0.0f);
        if (!there[j]) continue;
        const size_t from = kv_row(a.c, page, head, (uint32_t)p);
        const uint8_t *src = (which ? a.c.v : a.c.k) + from * ROWB;
        const float *scp = (which ? a.c.vs : a.c.ks) + from * kv_scales<KIND>();
        if constexpr (KIND <= KV_BF16) data[j] = reinterpret_cast<const uint4 *>(src)[lane];
        else if constexpr (KIND == KV_INT4) {
            data[j].x = reinterpret_cast<const uint32_t *>(src)[lane];
            sc[j] = *reinterpret_cast<const float2 *>(scp);
        } else {
            const uint2 w = reinterpret_cast<const uint2 *>(src)[lane];
            data[j].x = w.x;
            data[j].y = w.y;
            sc[j].x = *scp;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        if (!there[j]) continue;
        uint32_t row, which, head;
        kv_unit(first + j * PER, a.c.kv_heads, row, which, head);
        uint4 *dst = reinterpret_cast<uint4 *>((which ? a.v + row * a.v_stride : a.k + row * a.k_stride) + head * HD) + lane;
        if constexpr (KIND <= KV_BF16) {
            *dst = data[j];
        } else {
            float x[8];
            const float both[2] = {sc[j].x, sc[j].y};
            const uint32_t w[2] = {data[j].x, data[j].y};
            kv_values<KIND, 8>(reinterpret_cast<const uint8_t *>(w), both, 0, x);
            *dst = make_uint4(kv_round2(x[0], x[1], a.c.rows_bf16), kv_round2(x[2], x[3], a.c.rows_bf16), kv_round2(x[4], x[5], a.c.rows_bf16),
                              kv_round2(x[6], x[7], a.c.rows_bf16));
        }
    }
}

// Accepted tokens: row base + path[j] goes to base + j, j ascending.  A thread owns 16 bytes of one head's rows (or its scales) and
// reads KV_KEEP of them before it writes them; as path[j] >= j rises, what it reads later has not been written by then.
constexpr uint32_t KV_KEEP = 8;
struct KvKeepDev {
    KvDev c;
    const int32_t *seq, *base, *path, *kept;
    uint32_t path_stride, n_entries, pieces, scale_pieces, rowb;  // 16-byte pieces of a row, 4- or 8-byte ones of its scales (0 or 1)
};
__global__ void __launch_bounds__(KV_THREADS) kv_keep_kernel(const KvKeepDev a) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t e = blockIdx.y, per = a.pieces + a.scale_pieces, i = blockIdx.x * KV_THREADS + threadIdx.x;
    if (i >= per * a.c.kv_heads * 2) return;
    const uint32_t piece = i % per, head = i / per % a.c.kv_heads, which = i / per / a.c.kv_heads;
    const int32_t s = __ldg(a.seq + e), base = __ldg(a.base + e), n = min(__ldg(a.kept + e), (int32_t)a.path_stride);
    if (s < 0 || base < 0) return;
    for (int32_t j0 = 0; j0 < n; j0 += KV_KEEP) {
        uint4 data[KV_KEEP];
        size_t to[KV_KEEP];
        bool moves[KV_KEEP];
#pragma unroll
        for (uint32_t j = 0; j < KV_KEEP; j++) {
            moves[j] = false;
            const int32_t at = j0 + (int32_t)j;
            if (at >= n) continue;
            const int32_t d = __ldg(a.path + (size_t)e * a.path_stride + at);
            uint32_t from_page, to_page;
            if (d < at || d > 0x7FFFFFFF - base) {  // not a later token of this sequence
                kv_flag(a.c);
                continue;
            }
            if (d == at || !kv_place(a.c, s, base + d, from_page) || !kv_place(a.c, s, base + at, to_page)) continue;
            const size_t from = kv_row(a.c, from_page, head, (uint32_t)(base + d));
            to[j] = kv_row(a.c, to_page, head, (uint32_t)(base + at));
            moves[j] = true;
            if (piece < a.pieces) {
                data[j] = *(reinterpret_cast<const uint4 *>((which ? a.c.v : a.c.k) + from * a.rowb) + piece);
            } else {
                const uint32_t *sc = reinterpret_cast<const uint32_t *>(which ? a.c.vs : a.c.ks);
                data[j].x = sc[from * a.scale_pieces];
                if (a.scale_pieces == 2) data[j].x = sc[from * 2 + (piece - a.pieces)];
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < KV_KEEP; j++) {
            if (!moves[j]) continue;
            if (piece < a.pieces) {
                *(reinterpret_cast<uint4 *>((which ? a.c.v : a.c.k) + to[j] * a.rowb) + piece) = data[j];
            } else {
                uint32_t *sc = reinterpret_cast<uint32_t *>(which ? a.c.vs : a.c.ks);
                sc[to[j] * a.scale_pieces + (a.scale_pieces == 2 ? piece - a.pieces : 0)] = data[j].x;
            }
        }
    }
}

// ---- host side -----------------------------------------------------------------------------------
int kv_check(prism_cuda_ctx *ctx, const prism_cache *c, KvDev *out, int *kind) {
    if (c->rows != PRISM_CACHE_ROWS_F16 && c->rows != PRISM_CACHE_ROWS_BF16) return fail(ctx, PRISM_E_ARG, "cache: rows must be fp16 or bf16");
    if (c->format > PRISM_CACHE_INT4) return fail(ctx, PRISM_E_ARG, "cache: unknown format");
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(ctx, PRISM_E_ARG, "cache: head_dim must be 32, 64, 128 or 256");
    if (!c->kv_heads || c->kv_heads > 4096 || !c->n_pages || !c->n_seqs || !c->table_stride) return fail(ctx, PRISM_E_ARG, "cache: zero dimension, or over 4096 kv heads");
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1))) return fail(ctx, PRISM_E_ARG, "cache: page_size must be a power of two of at least 16");
    if ((uint64_t)c->table_stride * c->page_size > (1ull << 30)) return fail(ctx, PRISM_E_ARG, "cache: a sequence may hold at most 2^30 positions");
    if (c->n_seqs > 0x7FFFFFFFu || c->n_pages > 0x7FFFFFFFu) return fail(ctx, PRISM_E_ARG, "cache: sequences and pages are counted in 31 bits");
    if (!c->page_table && (uint64_t)c->n_seqs * c->table_stride > c->n_pages)
        return fail(ctx, PRISM_E_ARG, "cache: without a page table n_seqs * table_stride pages are needed");
    if (!c->k || !c->v || (c->format != PRISM_CACHE_16BIT && (!c->k_scale || !c->v_scale))) return fail(ctx, PRISM_E_NULL, "cache: null buffer");
    const void *all[4] = {c->k, c->v, c->format == PRISM_CACHE_16BIT ? nullptr : c->k_scale, c->format == PRISM_CACHE_16BIT ? nullptr : c->v_scale};
    for (const void *p : all)
        if (reinterpret_cast<uintptr_t>(p) & 15) return fail(ctx, PRISM_E_ARG, "cache: buffers must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(c->page_table) & 3) return fail(ctx, PRISM_E_ARG, "cache: the page table must be 4-byte aligned");
    uint32_t shift = 4;
    while ((1u << shift) < c->page_size) shift++;
    *out = KvDev{static_cast<uint8_t *>(c->k), static_cast<uint8_t *>(c->v), c->k_scale, c->v_scale, c->page_table, shift, c->table_stride, c->n_pages,
                 c->n_seqs, c->kv_heads, c->rows == PRISM_CACHE_ROWS_BF16, ctx->dev_err};
    *kind = c->format == PRISM_CACHE_16BIT ? (c->rows == PRISM_CACHE_ROWS_BF16 ? KV_BF16 : KV_F16) : c->format == PRISM_CACHE_INT8 ? KV_INT8
          : c->format == PRISM_CACHE_E4M3 ? KV_E4M3 : KV_INT4;
    return PRISM_OK;
}

template <int KIND>
static void launch_rows(prism_cuda_ctx *ctx, bool write, uint32_t hd, const KvRowsDev &a) {
    const uint32_t per = KV_THREADS / (hd / 8) * KV_UNITS;
    const dim3 grid((a.units + per - 1) / per), block(KV_THREADS);
    auto go = [&](void (*w)(KvRowsDev), void (*r)(KvRowsDev)) {
        if (write) launch_pdl(ctx, "kv_write_kernel", w, grid, block, 0, a);
        else launch_pdl(ctx, "kv_read_kernel", r, grid, block, 0, a);
    };
    switch (hd) {
    case 32: return go(kv_write_kernel<KIND, 32>, kv_read_kernel<KIND, 32>);
    case 64: return go(kv_write_kernel<KIND, 64>, kv_read_kernel<KIND, 64>);
    case 128: return go(kv_write_kernel<KIND, 128>, kv_read_kernel<KIND, 128>);
    default: return go(kv_write_kernel<KIND, 256>, kv_read_kernel<KIND, 256>);
    }
}

static int cache_rows(prism_cuda_ctx *ctx, const prism_cache *c, bool write, const void *k, const void *v, uint64_t k_stride, uint64_t v_stride, uint32_t n_rows,
                      const int32_t *seq, const int32_t *pos) {
    const char *name = write ? "cache_write" : "cache_read";
    if (!ctx || !c) return fail(ctx, PRISM_E_NULL, std::string(name) + ": null argument");
    KvRowsDev a{};
    int kind;
    PRISM_TRY(kv_check(ctx, c, &a.c, &kind));
    if (n_rows == 0) return PRISM_OK;
    if (!k || !v || !seq || !pos) return fail(ctx, PRISM_E_NULL, std::string(name) + ": null argument");
    const uint64_t width = (uint64_t)c->kv_heads * c->head_dim;
    if (k_stride < width || v_stride < width || k_stride % 8 || v_stride % 8 || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15))
        return fail(ctx, PRISM_E_ARG, std::string(name) + ": rows must be 16-byte aligned and at least kv_heads * head_dim values apart");
    if ((uint64_t)n_rows * 2 * c->kv_heads > 0x7FFFFFFFull) return fail(ctx, PRISM_E_ARG, std::string(name) + ": too many rows in one call");
    DeviceGuard on(ctx->device);
    if (on.err != cudaSuccess) return cuda_fail(ctx, on.err, "cudaSetDevice");
    a.k = static_cast<uint16_t *>(const_cast<void *>(k));
    a.v = static_cast<uint16_t *>(const_cast<void *>(v));
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.seq = seq;
    a.pos = pos;
    a.units = n_rows * 2 * c->kv_heads;
    switch (kind) {
    case KV_F16:
    case KV_BF16: launch_rows<KV_F16>(ctx, write, c->head_dim, a); break;  // 16-bit rows are copied as they are
    case KV_INT8: launch_rows<KV_INT8>(ctx, write, c->head_dim, a); break;
    case KV_E4M3: launch_rows<KV_E4M3>(ctx, write, c->head_dim, a); break;
    default: launch_rows<KV_INT4>(ctx, write, c->head_dim, a); break;
    }
    return after_launch(ctx, write ? "kv_write_kernel" : "kv_read_kernel");
}

static int cache_keep(prism_cuda_ctx *ctx, const prism_cache *c, uint32_t n_entries, const int32_t *seq, const int32_t *base, const int32_t *path,
                      uint32_t path_stride, const int32_t *kept) {
    if (!ctx || !c) return fail(ctx, PRISM_E_NULL, "cache_keep: null argument");
    KvKeepDev a{};
    int kind;
    PRISM_TRY(kv_check(ctx, c, &a.c, &kind));
    if (n_entries == 0 || path_stride == 0) return PRISM_OK;
    if (!seq || !base || !path || !kept) return fail(ctx, PRISM_E_NULL, "cache_keep: null argument");
    if (n_entries > 65535) return fail(ctx, PRISM_E_ARG, "cache_keep: at most 65535 entries a call");
    if (path_stride > 0x7FFFFFFFu) return fail(ctx, PRISM_E_ARG, "cache_keep: path_stride is counted in 31 bits");
    DeviceGuard on(ctx->device);
    if (on.err != cudaSuccess) return cuda_fail(ctx, on.err, "cudaSetDevice");
    a.seq = seq;
    a.base = base;
    a.path = path;
    a.kept = kept;
    a.path_stride = path_stride;
    a.n_entries = n_entries;
    a.rowb = c->head_dim * (kind <= KV_BF16 ? 16 : kind == KV_INT4 ? 4 : 8) / 8;
    a.pieces = a.rowb / 16;
    a.scale_pieces = kind <= KV_BF16 ? 0 : kind == KV_INT4 ? 2 : 1;
    const uint32_t threads = (a.pieces + a.scale_pieces) * c->kv_heads * 2;
    launch_pdl(ctx, "kv_keep_kernel", kv_keep_kernel, dim3((threads + KV_THREADS - 1) / KV_THREADS, n_entries), dim3(KV_THREADS), 0, a);
    return after_launch(ctx, "kv_keep_kernel");
}

}  // namespace prism

using namespace prism;

extern "C" {

int prism_cuda_cache_write_dev(prism_cuda_ctx *ctx, const prism_cache *cache, const void *k, const void *v, uint64_t k_stride, uint64_t v_stride,
                               uint32_t n_rows, const int32_t *seq, const int32_t *pos) {
    try {
        return cache_rows(ctx, cache, true, k, v, k_stride, v_stride, n_rows, seq, pos);
    } catch (const std::exception &) {
        return PRISM_E_STATE;  // no memory for a message
    }
}

int prism_cuda_cache_read_dev(prism_cuda_ctx *ctx, const prism_cache *cache, void *k, void *v, uint64_t k_stride, uint64_t v_stride, uint32_t n_rows,
                              const int32_t *seq, const int32_t *pos) {
    try {
        return cache_rows(ctx, cache, false, k, v, k_stride, v_stride, n_rows, seq, pos);
    } catch (const std::exception &) {
        return PRISM_E_STATE;
    }
}

int prism_cuda_cache_keep_dev(prism_cuda_ctx *ctx, const prism_cache *cache, uint32_t n_entries, const int32_t *seq, const int32_t *base,
                              const int32_t *path, uint32_t path_stride, const int32_t *kept) {
    try {
        return cache_keep(ctx, cache, n_entries, seq, base, path, path_stride, kept);
    } catch (const std::exception &) {
        return PRISM_E_STATE;
    }
}

}  // extern "C"
