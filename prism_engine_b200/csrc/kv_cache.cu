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
// hd / 16 lanes share a head of a position (a unit), 8 values from each half of it a lane, so loads and stores are whole lines and the extremes take
// log2(hd / 16) shuffles; a task is two units of one row.  Codes are rounded by adding 1.5 * 2^23, whose last bits they then are, and gathered by
// byte permutes.  Bound: HBM for long lists of 16-bit rows; for codes the time goes by tasks, not by bytes (a thread group does one, with its place,
// page and data in turn, and ends); launch latency for a decode step's rows.
// Reading up to 6 x 8000 rows of 8 heads of 128: from 16 bits 38.7 us (6.3 TB/s), e4m3 37.5 (4.9 TB/s), int4 36.6; four units a task 43.5 from e4m3
// and 41.3 from 16 bits, one 38.1 and 42.0.  Up to 4 x 2048 such rows, which L2 holds: written in 16 bits 5.4 us, int8 7.4, e4m3 7.1, int4 9.0 (3.4 TB/s),
// written in int4 and read back 15.7; four units 16.8, one 16.5.
#include <stdexcept>

#include "kv_cache.cuh"

namespace prism {

constexpr uint32_t KV_THREADS = 256, KV_UNITS = 2;

struct KvRowsDev {
    KvDev c;
    uint16_t *k, *v;             // rows, k_stride / v_stride values apart
    uint64_t k_stride, v_stride;
    const int32_t *seq, *pos;    // place of every row
    uint32_t tasks, per_row;     // of all rows, of one: KV_UNITS of its 2 * kv_heads units each
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
template <bool BF16>
__device__ __forceinline__ void kv_unpack(const uint4 &w, float *x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BF16) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
template <bool BF16>
__device__ __forceinline__ uint4 kv_pack(const float *x) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
// A rounded number of at most 22 bits (ties to even) in the last bits.
__device__ __forceinline__ uint32_t kv_rint(float x) { return __float_as_uint(__fadd_rn(x, 12582912.0f)); }
__device__ __forceinline__ uint32_t kv_four(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // their low bytes
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Codes of 2 * 8 values of a head that LANES lanes share (w[0], w[1]: the first eight, w[2], w[3]: the others; 4-bit codes: w[0] and w[2]),
// and the head's scales (the same in all its lanes).
template <int KIND, int LANES>
__device__ __forceinline__ void kv_encode(const float (&x)[16], uint32_t (&w)[4], float &scale, float &zero) {
    constexpr float TOP = KIND == KV_INT8 ? 127.0f : KIND == KV_E4M3 ? 448.0f : 15.0f;
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) big = max(big, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    big = kv_umax_of<LANES>(big);            // as integers: NaN above infinity above every number
    float lo = 0.0f, span = __uint_as_float(big);
    if (KIND == KV_INT4) {
        float hi = x[0];
        lo = x[0];
#pragma unroll
        for (int i = 1; i < 16; i++) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
        }
        lo = -kv_max_of<LANES>(-lo);
        hi = kv_max_of<LANES>(hi);
        span = __fsub_rn(hi, lo);
    }
    const bool odd = big >= 0x7F800000u || __float_as_uint(span) >= 0x7F800000u, real = span >= 0x1p-100f && !odd;
    scale = real ? __fdiv_rn(span, TOP) : 0.0f;
    const float inv = real ? __fdiv_rn(TOP, span) : 0.0f;
    if (KIND == KV_INT4) zero = __fadd_rn(lo, __fmul_rn(8.0f, scale));
    if (odd) scale = zero = __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const float *y = x + 8 * h;
        w[2 * h] = w[2 * h + 1] = KIND == KV_INT4 ? 0x88888888u : 0;
        if (KIND == KV_E4M3 ? odd : !real) continue;  // e4m3 keeps the signs of zeros
        uint32_t c[8];
        if constexpr (KIND == KV_INT4) {
#pragma unroll
            for (int i = 0; i < 8; i++) c[i] = kv_rint(__fmul_rn(__fsub_rn(y[i], lo), inv));
            uint32_t a = kv_four(c[0], c[1], c[2], c[3]), b = kv_four(c[4], c[5], c[6], c[7]);
            a |= a >> 4;                     // two codes in bytes 0 and 2
            b |= b >> 4;
            w[2 * h] = __byte_perm(a, b, 0x6420);
        } else if constexpr (KIND == KV_INT8) {
#pragma unroll
            for (int i = 0; i < 8; i++) c[i] = kv_rint(__fmul_rn(y[i], inv));
            w[2 * h] = kv_four(c[0], c[1], c[2], c[3]);
            w[2 * h + 1] = kv_four(c[4], c[5], c[6], c[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(y[2 * i], inv), __fmul_rn(y[2 * i + 1], inv)), __NV_SATFINITE, __NV_E4M3);
            w[2 * h] = c[0] | c[1] << 16;
            w[2 * h + 1] = c[2] | c[3] << 16;
        }
    }
}
// Eight values of codes: a product in 32 bits, and a sum where there is a zero.
template <int KIND>
__device__ __forceinline__ void kv_decode(uint32_t w0, uint32_t w1, float scale, float zero, float *x) {
    if constexpr (KIND == KV_INT4) {
#pragma unroll
        for (int i = 0; i < 8; i++)          // 2^23 + code
            x[i] = __fadd_rn(__fmul_rn(__uint_as_float((w0 >> (4 * i) & 15u) | 0x4B000000u) - 8388616.0f, scale), zero);
    } else if constexpr (KIND == KV_INT8) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t u = (i < 4 ? w0 : w1) ^ 0x80808080u;
            x[i] = __fmul_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + (i & 3))) - 8388736.0f, scale);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t h;
            asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}\n" : "=r"(h) : "r"((i < 2 ? w0 : w1) >> (16 * (i & 1))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            x[2 * i] = __fmul_rn(f.x, scale);
            x[2 * i + 1] = __fmul_rn(f.y, scale);
        }
    }
}

// A task's row, its place, and its first unit (of 2 * kv_heads: k's heads, then v's).
struct KvTask {
    uint32_t row, page, unit;
    int32_t pos;
    bool there;
};
__device__ __forceinline__ KvTask kv_task(const KvRowsDev &a, uint32_t i) {
    KvTask t;
    const uint32_t at = min(i, a.tasks - 1);
    t.row = at / a.per_row;
    t.unit = (at - t.row * a.per_row) * KV_UNITS;
    t.pos = __ldg(a.pos + t.row);
    t.page = 0;
    t.there = kv_place(a.c, __ldg(a.seq + t.row), t.pos, t.page) && i < a.tasks;
    return t;
}

}  // namespace

template <int KIND, int HD, bool BF16>
__global__ void __launch_bounds__(KV_THREADS, 3) kv_write_kernel(const KvRowsDev a) {
    constexpr uint32_t LANES = HD / 16, PER = KV_THREADS / LANES, ROWB = HD * kv_bits<KIND>() / 8;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x % LANES, units = 2 * a.c.kv_heads, index = blockIdx.x * PER + threadIdx.x / LANES;
    const uint32_t row = min(index, a.tasks - 1) / a.per_row, first = (min(index, a.tasks - 1) - row * a.per_row) * KV_UNITS;
    uint4 data[KV_UNITS][2];                 // asked for before the place is looked up
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        const uint32_t u = min(first + j, units - 1), which = u >= a.c.kv_heads, head = u - (which ? a.c.kv_heads : 0);
        const uint4 *src = reinterpret_cast<const uint4 *>((which ? a.v + row * a.v_stride : a.k + row * a.k_stride) + head * HD);
        data[j][0] = __ldg(src + lane);
        data[j][1] = __ldg(src + lane + LANES);
    }
    const KvTask t = kv_task(a, index);
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        const uint32_t u = t.unit + j, which = u >= a.c.kv_heads, head = u - (which ? a.c.kv_heads : 0);
        const bool there = t.there && u < units;
        const size_t to = there ? kv_row(a.c, t.page, head, (uint32_t)t.pos) : 0;
        uint8_t *dst = (which ? a.c.v : a.c.k) + to * ROWB;
        if constexpr (KIND <= KV_BF16) {
            if (there) {
                reinterpret_cast<uint4 *>(dst)[lane] = data[j][0];
                reinterpret_cast<uint4 *>(dst)[lane + LANES] = data[j][1];
            }
        } else {
            float x[16], scale, zero = 0.0f;
            uint32_t w[4];
            kv_unpack<BF16>(data[j][0], x);
            kv_unpack<BF16>(data[j][1], x + 8);
            kv_encode<KIND, LANES>(x, w, scale, zero);  // every lane of the warp takes part
            if (there) {
                float *sc = (which ? a.c.vs : a.c.ks) + to * kv_scales<KIND>();
                if constexpr (KIND == KV_INT4) {
                    reinterpret_cast<uint32_t *>(dst)[lane] = w[0];
                    reinterpret_cast<uint32_t *>(dst)[lane + LANES] = w[2];
                    if (lane == 0) *reinterpret_cast<float2 *>(sc) = make_float2(scale, zero);
                } else {
                    reinterpret_cast<uint2 *>(dst)[lane] = make_uint2(w[0], w[1]);
                    reinterpret_cast<uint2 *>(dst)[lane + LANES] = make_uint2(w[2], w[3]);
                    if (lane == 0) *sc = scale;
                }
            }
        }
    }
}

template <int KIND, int HD, bool BF16>
__global__ void __launch_bounds__(KV_THREADS, 3) kv_read_kernel(const KvRowsDev a) {
    constexpr uint32_t LANES = HD / 16, PER = KV_THREADS / LANES, ROWB = HD * kv_bits<KIND>() / 8;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x % LANES, units = 2 * a.c.kv_heads;
    const KvTask t = kv_task(a, blockIdx.x * PER + threadIdx.x / LANES);
    if (!t.there) return;
    uint4 data[KV_UNITS][2];
    float2 sc[KV_UNITS];
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        const uint32_t u = min(t.unit + j, units - 1), which = u >= a.c.kv_heads, head = u - (which ? a.c.kv_heads : 0);
        const size_t from = kv_row(a.c, t.page, head, (uint32_t)t.pos);
        const uint8_t *src = (which ? a.c.v : a.c.k) + from * ROWB;
        const float *scp = (which ? a.c.vs : a.c.ks) + from * kv_scales<KIND>();
        if constexpr (KIND <= KV_BF16) {
            data[j][0] = __ldg(reinterpret_cast<const uint4 *>(src) + lane);
            data[j][1] = __ldg(reinterpret_cast<const uint4 *>(src) + lane + LANES);
        } else if constexpr (KIND == KV_INT4) {
            data[j][0].x = __ldg(reinterpret_cast<const uint32_t *>(src) + lane);
            data[j][1].x = __ldg(reinterpret_cast<const uint32_t *>(src) + lane + LANES);
            sc[j] = __ldg(reinterpret_cast<const float2 *>(scp));
        } else {
            const uint2 p = __ldg(reinterpret_cast<const uint2 *>(src) + lane), q = __ldg(reinterpret_cast<const uint2 *>(src) + lane + LANES);
            data[j][0] = make_uint4(p.x, p.y, 0, 0);
            data[j][1] = make_uint4(q.x, q.y, 0, 0);
            sc[j] = make_float2(__ldg(scp), 0.0f);
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < KV_UNITS; j++) {
        const uint32_t u = t.unit + j, which = u >= a.c.kv_heads, head = u - (which ? a.c.kv_heads : 0);
        if (u >= units) break;
        uint4 *dst = reinterpret_cast<uint4 *>((which ? a.v + t.row * a.v_stride : a.k + t.row * a.k_stride) + head * HD) + lane;
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) {
            if constexpr (KIND <= KV_BF16) {
                dst[h * LANES] = data[j][h];
            } else {
                float x[8];
                kv_decode<KIND>(data[j][h].x, data[j][h].y, sc[j].x, sc[j].y, x);
                dst[h * LANES] = kv_pack<BF16>(x);
            }
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

template <int KIND, bool BF16>
static void launch_rows(prism_cuda_ctx *ctx, bool write, uint32_t hd, const KvRowsDev &a) {
    const uint32_t per = KV_THREADS / (hd / 16);
    const dim3 grid((a.tasks + per - 1) / per), block(KV_THREADS);
    auto go = [&](void (*w)(KvRowsDev), void (*r)(KvRowsDev)) {
        if (write) launch_pdl(ctx, "kv_write_kernel", w, grid, block, 0, a);
        else launch_pdl(ctx, "kv_read_kernel", r, grid, block, 0, a);
    };
    switch (hd) {
    case 32: return go(kv_write_kernel<KIND, 32, BF16>, kv_read_kernel<KIND, 32, BF16>);
    case 64: return go(kv_write_kernel<KIND, 64, BF16>, kv_read_kernel<KIND, 64, BF16>);
    case 128: return go(kv_write_kernel<KIND, 128, BF16>, kv_read_kernel<KIND, 128, BF16>);
    default: return go(kv_write_kernel<KIND, 256, BF16>, kv_read_kernel<KIND, 256, BF16>);
    }
}
template <int KIND>
static void launch_kind_rows(prism_cuda_ctx *ctx, bool write, uint32_t hd, const KvRowsDev &a) {
    if (a.c.rows_bf16) launch_rows<KIND, true>(ctx, write, hd, a);
    else launch_rows<KIND, false>(ctx, write, hd, a);
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
    if (!kv_words(seq, pos)) return fail(ctx, PRISM_E_ARG, std::string(name) + ": places must be 4-byte aligned");
    if ((uint64_t)n_rows * 2 * c->kv_heads > 0x7FFFFFFFull) return fail(ctx, PRISM_E_ARG, std::string(name) + ": too many rows in one call");
    DeviceGuard on(ctx->device);
    if (on.err != cudaSuccess) return cuda_fail(ctx, on.err, "cudaSetDevice");
    a.k = static_cast<uint16_t *>(const_cast<void *>(k));
    a.v = static_cast<uint16_t *>(const_cast<void *>(v));
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.seq = seq;
    a.pos = pos;
    a.per_row = (2 * c->kv_heads + KV_UNITS - 1) / KV_UNITS;
    a.tasks = n_rows * a.per_row;
    switch (kind) {
    case KV_F16:
    case KV_BF16: launch_rows<KV_F16, false>(ctx, write, c->head_dim, a); break;  // 16-bit rows are copied as they are
    case KV_INT8: launch_kind_rows<KV_INT8>(ctx, write, c->head_dim, a); break;
    case KV_E4M3: launch_kind_rows<KV_E4M3>(ctx, write, c->head_dim, a); break;
    default: launch_kind_rows<KV_INT4>(ctx, write, c->head_dim, a); break;
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
    if (!kv_words(seq, base, path, kept)) return fail(ctx, PRISM_E_ARG, "cache_keep: seq, base, path and kept must be 4-byte aligned");
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
