// Attention of the newest tokens of some sequences over a caller-owned cache on tcgen05 / TMEM: many query rows per cached head
// (portions of prompts, drafted trees), heads of 64 and 128.
//
// The rows that share a cached head -- the heads of its group, token after token -- are taken 256 at a time, two tiles of 128: while the
// softmax warps of one work, the tensor core has the other's products, and every key and value of the group is fetched once.  128
// positions a stage; S = Q K^T goes to TMEM, a thread owns one row, weights go back to TMEM over the scores they came from (16 bits, 2^12-fold
// in fp16) and meet V, read across its rows.  The running maximum moves only when it grows by more than 2^3.
//
//   16-bit rows   keys and values by TMA, page by page, straight from the pool
//   codes         three warps load them to registers a tile ahead and store them as fp16 in the swizzle the products read.  Keys stay
//                 exact codes, their scales multiply the scores; q enters as fp16 over a power of two.  Values are code * scale (+ zero) over
//                 a power of two of their tile, rounded once: code * (high part) + code * (low part) of the scale in fp16 pairs; a weight is shifted
//                 by the exponent in which its tile lies below the largest so far.  A value 2^27 below the largest of its tile loses bits.
//
// Positions past the end are zero.  A position that a row does not see meets weight 0, which an infinity there turns into NaN: a row whose
// result is not finite is taken again by itself (cache_plain_row).
// Fewer row tiles than SMs: the positions are cut into parts whose fp32 sums cache_join_kernel joins in order.
// Bound: the tensor core and the instructions about the scores together: 2 048 cycles of products for 256 rows and 128 positions of a 128-wide head,
// as many for their exponentials, and some 5 instructions a score (codes: 6 to 7) on four schedulers.
#include <algorithm>

#include "cache_join.cuh"
#include "tc5_ptx.cuh"
#include "tensor_map.cuh"

namespace prism {

constexpr int CT_ROWS = 256, CT_POS = 128, CT_ST = 2, CT_SC = 4;  // slots of scales
constexpr int CT_SOFT = 16;                                     // softmax warps: two threads a row, half of the positions each
constexpr float CT_GROW = 3.0f, CT_UP = 12.0f;  // powers of two: what a score may lie above the maximum in use; of the weights in fp16
template <int KIND, int HD>
struct CtCfg {
    static constexpr int PANELS = HD / 64, PANEL = 128 * 128, TILE = PANELS * PANEL;  // 128 rows of 64 values, in the 128-byte swizzle
    static constexpr int NSC = (int)kv_scales<KIND>(), ROWB = HD * (int)kv_bits<KIND>() / 8;
    static constexpr int SLOT = NSC ? 2 * CT_POS * NSC * 4 + 16 : 0;                   // key scales, value scales, each converting warp's largest of the latter
    static constexpr int K_OFF = 2 * TILE, V_OFF = K_OFF + CT_ST * TILE, SC_OFF = V_OFF + CT_ST * TILE, BAR_OFF = SC_OFF + CT_SC * SLOT;
    // barriers: kfull, kempty, vfull, vempty [2 each], sfull, pfull, ofull [2 each], qfull, scales [4]
    static constexpr int STATE_OFF = BAR_OFF + 8 * (4 * CT_ST + 7 + CT_SC);
    static constexpr int X_OFF = STATE_OFF + 16;                                       // what the two threads of a row tell each other
    static constexpr int R_OFF = X_OFF + 2 * 2 * CT_ROWS * 4;                          // CacheRow of each row
    static constexpr size_t SMEM = R_OFF + CT_ROWS * sizeof(CacheRow) + 1024;
    // behind the softmax warps three that convert (one of them copies, with 16-bit rows) and one of products: five warps a scheduler, 96 registers
    static constexpr int CONV = 96, ISSUER = CT_SOFT + 3, THREADS = (ISSUER + 1) * 32;
    static constexpr int RP = ROWB / 16, STEP = CONV / RP;                             // 16-byte pieces of a row; rows between a thread's pieces
    static constexpr int MINE = (CT_POS + STEP - 1) / STEP;                            // a thread's pieces of a tile
};

struct CtDev {
    CacheAttnDev a;
    uint32_t splits, tiles, box;  // parts of the positions, row tiles of an entry and head, positions of a copy
    uint32_t pool_rows;           // rows of the pool: one past the last
    float *part;                  // of the blocks, where there are several of a row tile (CacheJoinDev)
};

namespace {

__device__ __forceinline__ float ct_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t ct_below(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }
__device__ __forceinline__ float ct_pow2(int32_t e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// Exponent of the largest of four numbers, each not negative.
__device__ __forceinline__ int32_t ct_exponent(const float *top) {
    const float4 a = *reinterpret_cast<const float4 *>(top);
    return max((int32_t)(__float_as_uint(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w))) >> 23) - 127, -100);
}
// Which of 32 positions from c0 on a row sees: the last it sees of the committed, the window's end, the mask.
__device__ __forceinline__ uint32_t ct_seen(const CacheAttnDev &a, const CacheEntry &x, const CacheRow &r, int32_t c0) {
    uint32_t see = ct_below(r.last + 1 - c0) & (~ct_below(r.low + 1 - c0) | ct_below((int32_t)min(a.sinks, 0x7FFFFFFFu) - c0));
    if (r.mask && c0 + 32 > x.first && c0 < x.len) {
        const int32_t from = c0 - x.first;  // the bit of position c0
        uint32_t bits;
        if (from < 0) {
            bits = (uint32_t)(__ldg(r.mask) << -from);
        } else {
            uint64_t w = __ldg(r.mask + (from >> 6)) >> (from & 63);
            if ((from & 63) > 32 && (from >> 6) + 1 < (int32_t)a.tree_words) w |= __ldg(r.mask + (from >> 6) + 1) << (64 - (from & 63));
            bits = (uint32_t)w;
        }
        see |= bits & ct_below(x.len - c0) & ~ct_below(x.first - c0);
    }
    return see;
}

__device__ __forceinline__ uint32_t ct_u(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ __half2 ct_h(uint32_t u) { return *reinterpret_cast<const __half2 *>(&u); }

// A scale as it is kept for the values of a position: 8-bit codes, a high and a low fp16 part in one word; 4-bit codes, scale and zero.
template <int KIND>
__device__ __forceinline__ float2 ct_scale(float2 sc, float unit) {
    if constexpr (KIND == KV_INT4) return make_float2(sc.x * unit, sc.y * unit);
    const float v = sc.x * unit;
    const __half hi = __float2half_rn(v);
    return make_float2(__uint_as_float(ct_u(__halves2half2(hi, __float2half_rn(v - __half2float(hi))))), 0.0f);
}
// Two words of 8-bit codes, or one of 4-bit codes, as eight fp16: the codes (VALUES: code * scale, + zero, rounded once).  4-bit codes come
// in the order 0 4 1 5 2 6 3 7, which q's fragments and the columns of O follow (ct_order, ct_col).
template <int KIND, bool VALUES>
__device__ __forceinline__ uint4 ct_eight(uint32_t w0, uint32_t w1, float2 sc) {
    uint32_t h[4];
    if constexpr (KIND == KV_INT4) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t x = w0 >> (8 * i);
            h[2 * i] = ct_u(__hsub2(ct_h((x & 0x000F000Fu) | 0x64006400u), ct_h(0x64086408u)));
            h[2 * i + 1] = ct_u(__hfma2(ct_h((x & 0x00F000F0u) | 0x64006400u), ct_h(0x2C002C00u), ct_h(0xD480D480u)));  // (1024 + 16 c) / 16 - 72
        }
        if constexpr (VALUES) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = __half22float2(ct_h(h[i]));
                h[i] = ct_u(__floats2half2_rn(fmaf(f.x, sc.x, sc.y), fmaf(f.y, sc.x, sc.y)));
            }
        }
    } else {
        const uint32_t w[2] = {w0, w1};
#pragma unroll
        for (int q = 0; q < 2; q++) {
            if constexpr (KIND == KV_INT8) {
                const uint32_t x = w[q] ^ 0x80808080u;  // code + 128 in the low bits of 1024
                h[2 * q] = ct_u(__hsub2(ct_h(__byte_perm(x, 0x64646464u, 0x4140)), ct_h(0x64806480u)));
                h[2 * q + 1] = ct_u(__hsub2(ct_h(__byte_perm(x, 0x64646464u, 0x4342)), ct_h(0x64806480u)));
            } else {
                asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n" : "=r"(h[2 * q]), "=r"(h[2 * q + 1]) : "r"(w[q]));
            }
        }
        if constexpr (VALUES) {
            const uint32_t both = __float_as_uint(sc.x);
            const __half2 hi = ct_h(__byte_perm(both, 0, 0x1010)), lo = ct_h(__byte_perm(both, 0, 0x3232));
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = ct_u(__hfma2(ct_h(h[i]), hi, __hmul2(ct_h(h[i]), lo)));
        }
    }
    return make_uint4(h[0], h[1], h[2], h[3]);
}
// Eight 16-bit values in that order.
template <int KIND>
__device__ __forceinline__ uint4 ct_order(uint4 w) {
    if (KIND != KV_INT4) return w;
    return make_uint4(__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632), __byte_perm(w.y, w.w, 0x5410), __byte_perm(w.y, w.w, 0x7632));
}
// The register that holds column i of 32.
template <int KIND>
__device__ __forceinline__ constexpr int ct_col(int i) {
    return KIND != KV_INT4 ? i : (i & ~7) | (i & 3) << 1 | (i >> 2 & 1);
}

// In the order of the program: what a thread holds at once stays within its registers.
__device__ __forceinline__ void ct_sts(uint32_t at, const uint4 &v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float2 ct_lds2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float ct_lds(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// A 16-byte piece of codes into a tile: eight values a store.  `at`: where the pieces of fp16 go in the thread's first row, `flip`: what differs in
// this one; `swap`: the second half
// of the piece first, so that the stores of neighbouring lanes lie in different banks.
template <int KIND, bool VALUES>
__device__ __forceinline__ void ct_convert(uint32_t tile, uint32_t flip, const uint32_t (&at)[4], bool swap, const uint4 &codes, float2 sc) {
    const uint32_t w0 = swap ? codes.z : codes.x, w1 = swap ? codes.w : codes.y, w2 = swap ? codes.x : codes.z, w3 = swap ? codes.y : codes.w;
    if constexpr (KIND == KV_INT4) {
        ct_sts(tile + (at[0] ^ flip), ct_eight<KIND, VALUES>(w0, 0, sc));
        ct_sts(tile + (at[1] ^ flip), ct_eight<KIND, VALUES>(w1, 0, sc));
        ct_sts(tile + (at[2] ^ flip), ct_eight<KIND, VALUES>(w2, 0, sc));
        ct_sts(tile + (at[3] ^ flip), ct_eight<KIND, VALUES>(w3, 0, sc));
    } else {
        ct_sts(tile + (at[0] ^ flip), ct_eight<KIND, VALUES>(w0, w1, sc));
        ct_sts(tile + (at[1] ^ flip), ct_eight<KIND, VALUES>(w2, w3, sc));
    }
}

}  // namespace

template <int KIND, int HD>
__global__ void __launch_bounds__(CtCfg<KIND, HD>::THREADS, 1) cache_tiles_kernel(const __grid_constant__ CtDev d, const __grid_constant__ CUtensorMap kmap,
                                                                    const __grid_constant__ CUtensorMap vmap) {
    using C = CtCfg<KIND, HD>;
    constexpr bool CODES = KIND >= KV_INT8, BF16 = KIND == KV_BF16;
    constexpr int ST = CT_ST, NSC = C::NSC;
    const CacheAttnDev &a = d.a;
    extern __shared__ uint8_t ct_raw[];
    uint8_t *smem = ct_raw + (1024 - ((uint32_t)__cvta_generic_to_shared(ct_raw) & 1023u)) % 1024;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
    pdl_launch_dependents();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t b_kfull = base + C::BAR_OFF, b_kempty = b_kfull + 8 * ST, b_vfull = b_kempty + 8 * ST, b_vempty = b_vfull + 8 * ST,
                   b_sfull = b_vempty + 8 * ST, b_pfull = b_sfull + 16, b_ofull = b_pfull + 16, b_qfull = b_ofull + 16, b_sc = b_qfull + 8;
    volatile uint32_t *err_flag = reinterpret_cast<volatile uint32_t *>(smem + C::STATE_OFF);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::STATE_OFF + 8);
    if (tid == 0) {
        for (int s = 0; s < ST; s++) {
            t5::mbar_init(b_kfull + 8 * s, CODES ? C::CONV : 1); t5::mbar_init(b_kempty + 8 * s, 1);
            t5::mbar_init(b_vfull + 8 * s, CODES ? C::CONV : 1); t5::mbar_init(b_vempty + 8 * s, 1);
        }
        for (int q = 0; q < 2; q++) { t5::mbar_init(b_sfull + 8 * q, 1); t5::mbar_init(b_pfull + 8 * q, CT_SOFT / 2); t5::mbar_init(b_ofull + 8 * q, 1); }
        t5::mbar_init(b_qfull, CT_SOFT);
        for (int s = 0; s < CT_SC; s++) t5::mbar_init(b_sc + 8 * s, C::CONV);
        *err_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == C::ISSUER) t5::tmem_alloc(base + C::STATE_OFF + 8, 512);
    t5::fence_before();
    __syncthreads();
    t5::fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);  // S of tile q at column 128 q, O at 256 + HD q
    pdl_wait();                                                    // before any bounded wait: the kernel before this one may still be at work

    const uint32_t item = blockIdx.x / d.splits, split = blockIdx.x - item * d.splits;
    const uint32_t tile = item % d.tiles, kh = item / d.tiles % a.c.kv_heads, e = item / d.tiles / a.c.kv_heads;
    CacheEntry x;
    const bool is = cache_entry(a, e, x);                          // the same in all blocks of an item
    const uint32_t n_rows = is ? x.n * a.group : 0, r0 = tile * CT_ROWS;
    const uint32_t here = r0 < n_rows ? min((uint32_t)CT_ROWS, n_rows - r0) : 0, n_q = (here + 127) / 128;
    // ---- the positions that some row sees: the first tiles (a.sinks), then main_lo .. --------------------------------------
    int32_t i_lo = 0, i_hi = 0, first_tiles = 0, main_lo = 0;
    if (here) {
        const uint32_t tok_lo = r0 / a.group, tok_hi = (r0 + here - 1) / a.group;
        int32_t low = -1;
        if (a.window && !a.tree) low = cache_row(a, x, tok_lo).low;
        else if (a.window) {
            low = x.len;
            for (uint32_t i = tok_lo + lane; i <= tok_hi; i += 32) low = min(low, cache_row(a, x, i).low);
            low = __reduce_min_sync(0xFFFFFFFFu, low);
        }
        const int32_t end = a.tree ? x.len : min(x.len, x.first + (int32_t)tok_hi + 1), start = a.tree ? min(low + 1, max(x.first, 0)) : low + 1;
        const int32_t main_hi = end > 0 ? (end + CT_POS - 1) / CT_POS : 0;
        first_tiles = end > 0 ? (int32_t)(min((uint32_t)end, a.sinks) + CT_POS - 1) / CT_POS : 0;
        main_lo = max(start / CT_POS, first_tiles);
        const int32_t n_tiles = first_tiles + max(main_hi - main_lo, 0);
        i_lo = (int32_t)((int64_t)n_tiles * split / d.splits);
        i_hi = (int32_t)((int64_t)n_tiles * (split + 1) / d.splits);
    }
    const uint32_t n = (uint32_t)(i_hi - i_lo);
    auto pos_of = [&](uint32_t j) {
        const int32_t i = i_lo + (int32_t)j;
        return (i < first_tiles ? i : main_lo + (i - first_tiles)) * CT_POS;
    };

    if (here == 0) {
        // nothing of this entry
    } else if (warp < CT_SOFT) {
        // ================= softmax: two threads a query row, positions 0..63 and 64..127 of a tile =================
        const uint32_t q = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane, lanes = ((warp & 3) * 32) << 16, rr = r0 + q * 128 + row;
        const uint32_t s_col = tmem + lanes + q * 128, o_col = tmem + lanes + 256 + q * HD + half * (HD / 2);
        const bool there = q * 128 + row < here;
        float *xch = reinterpret_cast<float *>(smem + C::X_OFF) + q * 128 + row;  // [turn][half][256 rows]
        // The value of the row's other thread.  Turns alternate: both have read one turn's before either writes it again.
        auto other = [&](float v, uint32_t turn) {
            xch[(turn * 2 + half) * CT_ROWS] = v;
            asm volatile("bar.sync %0, 64;\n" ::"r"(1 + q * 4 + (warp & 3)) : "memory");
            return xch[(turn * 2 + (half ^ 1)) * CT_ROWS];
        };
        CacheRow *row_at = reinterpret_cast<CacheRow *>(smem + C::R_OFF) + q * 128 + row;  // the same in both threads
        int32_t all_to, all_low;
        {
            CacheRow r{0x7FFFFFF0, -1, nullptr};                   // a row that is not there: sees everything, is not stored
            if (there) r = cache_row(a, x, rr / a.group);
            all_to = __reduce_min_sync(0xFFFFFFFFu, r.last);
            all_low = __reduce_max_sync(0xFFFFFFFFu, r.low);
            *row_at = r;
        }
        float mul = fabsf(a.scale) * 1.4426950408889634f, qsum = 0.0f;
        {   // half of the row of q into its tile, its sign that of the scale
            constexpr int W = HD / 16;
            const uint32_t token = there ? rr / a.group : 0, head = kh * a.group + (there ? rr % a.group : 0);
            const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
            const uint4 *src = reinterpret_cast<const uint4 *>(a.q + (size_t)(x.row0 + token) * a.q_stride + (size_t)head * HD) + half * W;
            uint4 w[W];
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < W; i++) {
                w[i] = there ? src[i] : make_uint4(0, 0, 0, 0);
                uint32_t *u = reinterpret_cast<uint32_t *>(&w[i]);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    u[k] ^= flip;
                    if constexpr (CODES)
                        big = fmaxf(big, fmaxf(fabsf(kv_row_value((uint16_t)u[k], a.c.rows_bf16)), fabsf(kv_row_value((uint16_t)(u[k] >> 16), a.c.rows_bf16))));
                }
            }
            if constexpr (CODES) {                                 // over the power of two below the largest
                big = fmaxf(big, other(big, 0));
                const uint32_t ex = min(__float_as_uint(big) & 0x7F800000u, 253u << 23);
                const float inv = ex ? __uint_as_float((254u << 23) - ex) : 1.0f;
                if (ex) mul *= __uint_as_float(ex);
#pragma unroll
                for (int i = 0; i < W; i++) {
                    uint32_t *u = reinterpret_cast<uint32_t *>(&w[i]);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const __half2 h = __floats2half2_rn(kv_row_value((uint16_t)u[k], a.c.rows_bf16) * inv, kv_row_value((uint16_t)(u[k] >> 16), a.c.rows_bf16) * inv);
                        const float2 f = __half22float2(h);
                        qsum += f.x + f.y;
                        u[k] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                }
                if constexpr (NSC == 2) qsum += other(qsum, 1);
            }
#pragma unroll
            for (int i = 0; i < W; i++) {
                const uint32_t c = half * W + i;
                *reinterpret_cast<uint4 *>(smem + q * C::TILE + (c >> 3) * C::PANEL + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = ct_order<KIND>(w[i]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            asm volatile("bar.sync %0, 64;\n" ::"r"(1 + q * 4 + (warp & 3)) : "memory");  // the exchanged values have been read
            if (lane == 0) t5::mbar_arrive(b_qfull);
        }
        float m = -INFINITY, l = 0.0f;
        int32_t ref = 0;                                           // exponent that O is over
        const uint32_t mine = q < n_q ? n : 0;
        for (uint32_t j = 0; j < mine; j++) {
            int32_t ex = 0;
            const float *ksc = nullptr;
            if constexpr (CODES) {
                t5::mbar_wait_warp(b_sc + 8 * (j % CT_SC), (j / CT_SC) & 1, err_flag);
                ksc = reinterpret_cast<const float *>(smem + C::SC_OFF + (j % CT_SC) * C::SLOT);
                ex = ct_exponent(ksc + 2 * CT_POS * NSC);
                ksc += half * 64 * NSC;
            }
            t5::mbar_wait_warp(b_sfull + 8 * q, j & 1, err_flag);
            t5::fence_after();
            uint32_t s[2][32];
#pragma unroll
            for (int c = 0; c < 2; c++) t5::ld32(s_col + half * 64 + c * 32, s[c]);
            t5::wait_ld();
            const int32_t p0 = pos_of(j) + (int32_t)half * 64;
            if constexpr (NSC == 1) {
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(ksc + c * 32 + i);
                        s[c][i] = __float_as_uint(__uint_as_float(s[c][i]) * f.x);
                        s[c][i + 1] = __float_as_uint(__uint_as_float(s[c][i + 1]) * f.y);
                        s[c][i + 2] = __float_as_uint(__uint_as_float(s[c][i + 2]) * f.z);
                        s[c][i + 3] = __float_as_uint(__uint_as_float(s[c][i + 3]) * f.w);
                    }
            } else if constexpr (NSC == 2) {
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float4 f = *reinterpret_cast<const float4 *>(ksc + (c * 32 + i) * 2);
                        s[c][i] = __float_as_uint(fmaf(__uint_as_float(s[c][i]), f.x, qsum * f.y));
                        s[c][i + 1] = __float_as_uint(fmaf(__uint_as_float(s[c][i + 1]), f.z, qsum * f.w));
                    }
            }
            if (p0 + 63 > all_to || !(p0 > all_low || (uint32_t)(p0 + 64) <= a.sinks)) {  // some row of the warp does not see all 64
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const uint32_t see = there ? ct_seen(a, x, *row_at, p0 + c * 32) : 0xFFFFFFFFu;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (!(see & (1u << i))) s[c][i] = 0xFF800000u;
                }
            }
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; c++) mx[c] = __uint_as_float(s[c >> 1][(c & 1) * 16]);
#pragma unroll
            for (int i = 1; i < 16; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) mx[c] = fmaxf(mx[c], __uint_as_float(s[c >> 1][(c & 1) * 16 + i]));
            float best = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            best = fmaxf(best, other(best, j & 1));
            const float top = best == -INFINITY ? best : best * mul;  // mul may be 0
            const bool grow = top > m + CT_GROW;
            if (j == 0) {
                m = top;
                ref = ex;
            } else if (__any_sync(0xFFFFFFFFu, grow) || ex > ref) {
                // the products of the tile before are complete: the scores that were just waited for follow them
                float f = grow ? ct_ex2(m - top) : 1.0f;
                if (grow) m = top;
                l *= f;
                if (ex > ref) {
                    f *= ct_pow2(max(ref - ex, -126));
                    ref = ex;
                }
#pragma unroll 1
                for (int c = 0; c < HD / 32; c++) {
                    uint32_t o[16];
                    t5::ld16(o_col + c * 16, o);
                    t5::wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    t5::st16(o_col + c * 16, o);
                }
            }
            const float less = (m == -INFINITY ? 0.0f : m) - (BF16 ? 0.0f : CT_UP) - (CODES ? (float)max(ex - ref, -90) : 0.0f);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float e0 = ct_ex2(fmaf(__uint_as_float(s[c][2 * i]), mul, -less)), e1 = ct_ex2(fmaf(__uint_as_float(s[c][2 * i + 1]), mul, -less));
                    sum[(2 * i) & 3] += e0;
                    sum[(2 * i + 1) & 3] += e1;
                    if constexpr (BF16) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(e0, e1);
                        p[i] = *reinterpret_cast<const uint32_t *>(&h);
                    } else {
                        const __half2 h = __floats2half2_rn(e0, e1);
                        p[i] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                }
                t5::st16(s_col + half * 32 + c * 16, p);
            }
            float more = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if constexpr (CODES)
                if (ex != ref) more *= ct_pow2(min(ref - ex, 90));
            l += more;
            t5::wait_st();
            t5::fence_before();
            __syncwarp();
            if (lane == 0) t5::mbar_arrive(b_pfull + 8 * q);
        }
        l += other(l, mine & 1);
        if (mine) {
            t5::mbar_wait_warp(b_ofull + 8 * q, 0, err_flag);
            t5::fence_after();
        }
        // ---- results, half of the columns a thread: O times 2^(ref - 13) where V was over a power of two, as the weights' sum is 2^12-fold ----
        const float unit = CODES ? ct_pow2(ref - 13) : 1.0f;
        float inv = 1.0f / l, odd = l > 0.0f ? 0.0f : 1.0f;        // not 0 once an output was not finite
        uint16_t *dst = there ? a.out + (size_t)(x.row0 + rr / a.group) * a.out_stride + (size_t)(kh * a.group + rr % a.group) * HD + half * (HD / 2) : nullptr;
        auto store = [&](int c, const float (&o)[32]) {            // 32 columns
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float u = o[ct_col<KIND>(2 * i)] * inv, v = o[ct_col<KIND>(2 * i + 1)] * inv;
                odd = fmaf(u, 0.0f, fmaf(v, 0.0f, odd));
                w[i] = kv_round2(u, v, a.c.rows_bf16);
            }
            if (there)
#pragma unroll
                for (int i = 0; i < 4; i++) reinterpret_cast<uint4 *>(dst + c * 32)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        };
        if (d.splits == 1) {
#pragma unroll 1
            for (int c = 0; c < HD / 64; c++) {
                uint32_t o[32];
                float v[32];
                if (mine) {
                    t5::ld32(o_col + c * 32, o);
                    t5::wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = mine ? __uint_as_float(o[i]) * unit : 0.0f;
                store(c, v);
                __syncwarp();                                      // the next TMEM read takes the whole warp
            }
        } else {
            const size_t at = q * 128 + row, c_first = half * (HD / 8);  // groups of four columns
            float *to = d.part + (size_t)blockIdx.x * cache_part_floats(CT_ROWS, HD);
#pragma unroll 1
            for (int c = 0; c < HD / 64; c++) {
                uint32_t o[32];
                if (mine) {
                    t5::ld32(o_col + c * 32, o);
                    t5::wait_ld();
                }
                if (there) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const auto col = [&](int k) { return mine ? __uint_as_float(o[ct_col<KIND>(4 * i + k)]) * unit : 0.0f; };
                        const float4 v = make_float4(col(0), col(1), col(2), col(3));
                        __stcg(reinterpret_cast<float4 *>(to) + (c_first + c * 8 + i) * CT_ROWS + at, v);
                    }
                }
                __syncwarp();
            }
            if (half == 0) {
                __stcg(to + CT_ROWS * HD + at, m);
                __stcg(to + CT_ROWS * (HD + 1) + at, l);
            }
        }
        if (d.splits == 1) {
            const float theirs = other(odd, (mine & 1) ^ 1);       // every lane takes part; after what the other thread stored
            const bool again = there && (odd != 0.0f || theirs != 0.0f);
            if (half == 0)
                for (uint32_t rows = __ballot_sync(0xFFFFFFFFu, again); rows; rows &= rows - 1) {
                    const uint32_t i = rr - lane + (uint32_t)(__ffs(rows) - 1);
                    cache_plain_row<KIND, HD>(a, x, i / a.group, kh * a.group + i % a.group, lane);
                }
        }
        t5::fence_before();
    } else if (warp == C::ISSUER) {
        // ================= products: the whole warp walks the tiles (descriptors stay in uniform registers), an elected lane issues;
        // all lanes clear 16-bit value rows past the end =================
        const uint32_t types = BF16 ? 1u << 7 | 1u << 10 : 0u;
        const uint32_t id_s = t5::idesc_f16(128, CT_POS) | types, id_o = t5::idesc_f16(128, HD) | types | (1u << 16);  // V is read across its rows
        auto scores = [&](uint32_t q, uint32_t j) {
            const uint32_t qa = base + q * C::TILE, ka = base + C::K_OFF + (j % ST) * C::TILE;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                const uint32_t off = (k * 32 / 128) * C::PANEL + (k * 32) % 128;
                t5::mma_ss(tmem + q * 128, t5::desc_swizzled<128>(qa + off, 16), t5::desc_swizzled<128>(ka + off, 16), id_s, k != 0);
            }
            t5::commit(b_sfull + 8 * q);
        };
        if (n) {
            t5::mbar_wait_bounded(b_qfull, 0, err_flag);
            t5::mbar_wait_bounded(b_kfull, 0, err_flag);
            __syncwarp();
            t5::fence_after();
            if (t5::elect_one()) {
                for (uint32_t q = 0; q < n_q; q++) scores(q, 0);
                t5::commit(b_kempty);
            }
            __syncwarp();
        }
        for (uint32_t j = 0; j < n; j++) {
            const uint32_t st = j % ST, ph = (j / ST) & 1, va = base + C::V_OFF + st * C::TILE, jn = j + 1;
            t5::mbar_wait_bounded(b_vfull + 8 * st, ph, err_flag);
            __syncwarp();
            if constexpr (!CODES) {
                const int32_t left = x.len - pos_of(j);
                if (left < CT_POS) {
                    const uint32_t first = (uint32_t)left, cells = (CT_POS - first) * 8 * C::PANELS;
                    for (uint32_t i = lane; i < cells; i += 32) {
                        const uint32_t p = i / ((CT_POS - first) * 8), c = i % ((CT_POS - first) * 8);
                        *reinterpret_cast<uint4 *>(smem + C::V_OFF + st * C::TILE + p * C::PANEL + first * 128 + c * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                }
            }
            if (jn < n) t5::mbar_wait_bounded(b_kfull + 8 * (jn % ST), (jn / ST) & 1, err_flag);
#pragma unroll
            for (uint32_t q = 0; q < 2; q++) {
                if (q >= n_q) continue;
                t5::mbar_wait_bounded(b_pfull + 8 * q, j & 1, err_flag);
                __syncwarp();
                t5::fence_after();
                if (t5::elect_one()) {
#pragma unroll
                    for (int k = 0; k < CT_POS / 16; k++)
                        t5::mma_ts(tmem + 256 + q * HD, tmem + q * 128 + k * 8, t5::desc_swizzled<128>(va + k * 16 * 128, C::PANEL), id_o, k ? 1u : j);
                    if (jn < n) scores(q, jn);
                    else t5::commit(b_ofull + 8 * q);
                }
                __syncwarp();
            }
            if (t5::elect_one()) {
                t5::commit(b_vempty + 8 * st);
                if (jn < n) t5::commit(b_kempty + 8 * (jn % ST));
            }
            __syncwarp();
        }
        t5::fence_before();
    } else if constexpr (!CODES) {
        // ================= copies =================
        // A lane a box (of at most eight): its page is asked for a tile before it is needed.
        if (warp == CT_SOFT) {
            const uint32_t boxes = CT_POS / d.box, b = lane % boxes;
            auto look = [&](uint32_t j) {
                const int32_t p = j < n ? pos_of(j) + (int32_t)(b * d.box) : x.len;
                return p < x.len ? kv_page_number(a.c, x.seq, (uint32_t)p) : 0xFFFFFFFFu;
            };
            auto load = [&](const CUtensorMap *map, uint32_t dst, uint32_t at, uint32_t mbar) {
                if (lane == 0) t5::mbar_arrive_expect_tx(mbar, CT_POS * HD * 2);
                __syncwarp();
                if (lane < boxes)
                    for (uint32_t q = 0; q < (uint32_t)C::PANELS; q++)
                        t5::tma_2d(dst + q * C::PANEL + b * d.box * 128, map, (int32_t)(q * 64), (int32_t)at, mbar);
            };
            uint32_t page = look(0);
            for (uint32_t j = 0; j < n; j++) {
                const uint32_t st = j % ST, ph = (j / ST) & 1;
                const int32_t p = pos_of(j) + (int32_t)(b * d.box);
                // past the last row of the pool: zeros
                const uint32_t at = p < x.len && kv_page_ok(a.c, page) ? (uint32_t)kv_row(a.c, page, kh, (uint32_t)p) : d.pool_rows;
                page = look(j + 1);
                t5::mbar_wait_warp(b_kempty + 8 * st, ph ^ 1, err_flag);
                load(&kmap, base + C::K_OFF + st * C::TILE, at, b_kfull + 8 * st);
                t5::mbar_wait_warp(b_vempty + 8 * st, ph ^ 1, err_flag);
                load(&vmap, base + C::V_OFF + st * C::TILE, at, b_vfull + 8 * st);
            }
            // every copy in flight lands before the CTA leaves
            for (uint32_t j = n > (uint32_t)ST ? n - ST : 0; j < n; j++) {
                t5::mbar_wait_warp(b_kfull + 8 * (j % ST), (j / ST) & 1, err_flag);
                t5::mbar_wait_warp(b_vfull + 8 * (j % ST), (j / ST) & 1, err_flag);
            }
        }
        __syncwarp();
    } else {
        // ================= codes to fp16 =================
        // A thread has the same piece of every STEP-th row; its codes stay in registers: as soon as those of the keys are stored those of
        // the values are asked for, and so on.
        const uint32_t ct = tid - CT_SOFT * 32, cw = warp - CT_SOFT;
        constexpr int RP = C::RP, STEP = C::STEP, MINE = C::MINE, N = KIND == KV_INT4 ? 4 : 2;
        static_assert(STEP % 4 == 0, "neighbouring pieces of a thread lie alike in their swizzled rows, or four rows apart");
        const uint32_t row0 = ct / RP, piece = ct % RP;
        const bool swap = KIND == KV_INT4 ? piece & 2 : piece >> 2 & 1;
        uint32_t to[4];                                            // of its fp16 pieces in row0 of a tile
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t c = piece * N + ((i % N) ^ (swap ? N / 2 : 0));
            to[i] = (c >> 3) * C::PANEL + row0 * 128 + (((c & 7) ^ (row0 & 7)) << 4);
        }
        uint4 reg[MINE];
        float2 scr[2][2];                                          // keys', values' scales of positions ct and ct + 96
        uint32_t at_k = 0, at_v = 0;                               // lanes 0..7: the pool row of the tile's 16-position unit (0 where there is none)
        // Pages are asked for two tiles ahead, so that nothing waits for the table.
        auto look = [&](uint32_t j) {
            const int32_t p = j < n ? pos_of(j) + (int32_t)(lane & 7) * 16 : x.len;
            return p < x.len ? kv_page_number(a.c, x.seq, (uint32_t)p) : 0xFFFFFFFFu;
        };
        auto units = [&](uint32_t j, uint32_t page) {
            const int32_t p = j < n ? pos_of(j) + (int32_t)(lane & 7) * 16 : x.len;
            return p < x.len && kv_page_ok(a.c, page) ? (uint32_t)kv_row(a.c, page, kh, (uint32_t)p) : 0u;
        };
        uint32_t page = look(0);
        // Four pieces at a time, so that what they wait for overlaps.
        constexpr int G = 4;
        auto load = [&](const uint8_t *pool, int first, uint32_t of) {
            uint32_t at[G];
#pragma unroll
            for (int i = 0; i < G; i++) at[i] = __shfl_sync(0xFFFFFFFFu, of, ((row0 + (first + i) * STEP) >> 4) & 7);
#pragma unroll
            for (int i = 0; i < G; i++)
                if (first + i < MINE) reg[first + i] = t5::ldg128_nc(pool + (size_t)(at[i] + ((row0 + (first + i) * STEP) & 15)) * C::ROWB + piece * 16);
        };
        // Past the end some row of the pool is read; its scale is 0, but a code of e4m3 may be NaN.
        auto clear = [&](int32_t p0) {
            if (KIND == KV_E4M3 && p0 + CT_POS > x.len) {
#pragma unroll
                for (int i = 0; i < MINE; i++)
                    if (p0 + (int32_t)(row0 + i * STEP) >= x.len) reg[i] = make_uint4(0, 0, 0, 0);
            }
        };
        constexpr int FULL = CT_POS / STEP;                        // pieces that every thread has
        auto load_scales = [&](int32_t p0, uint32_t of) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t row = ct + h * 96, at = __shfl_sync(0xFFFFFFFFu, of, (row >> 4) & 7);
                scr[0][h] = scr[1][h] = make_float2(0.0f, 0.0f);
                if (row < CT_POS && p0 + (int32_t)row < x.len) {
                    const size_t from = ((size_t)at + (row & 15)) * NSC;
                    if constexpr (NSC == 2) {
                        scr[0][h] = __ldg(reinterpret_cast<const float2 *>(a.c.ks + from));
                        scr[1][h] = __ldg(reinterpret_cast<const float2 *>(a.c.vs + from));
                    } else {
                        scr[0][h].x = __ldg(a.c.ks + from);
                        scr[1][h].x = __ldg(a.c.vs + from);
                    }
                }
            }
        };
        if (n) {
            at_k = units(0, page);
            page = look(1);
#pragma unroll
            for (int i = 0; i < MINE; i += G) load(a.c.k, i, at_k);
            load_scales(pos_of(0), at_k);
        }
        for (uint32_t j = 0; j < n; j++) {
            const uint32_t st = j % ST, ph = (j / ST) & 1;
            const int32_t now = pos_of(j), next = j + 1 < n ? pos_of(j + 1) : x.len;  // nothing is loaded from the end on
            at_v = at_k;
            t5::mbar_wait_warp(b_kempty + 8 * st, ph ^ 1, err_flag);
            // the slot's last readers, the softmax of tile j - 4, came before the products that have just been waited for
            float *ksc = reinterpret_cast<float *>(smem + C::SC_OFF + (j % CT_SC) * C::SLOT), *vsc = ksc + CT_POS * NSC, *tops = vsc + CT_POS * NSC;
            float big = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t row = ct + h * 96;
                if (row < CT_POS) {
                    if constexpr (NSC == 2) reinterpret_cast<float2 *>(ksc)[row] = scr[0][h];
                    else ksc[row] = scr[0][h].x;
                }
                // no value is larger; scales that are not finite count for nothing, their values stay what they are
                const float most = KIND == KV_INT4 ? fmaf(8.0f, fabsf(scr[1][h].x), fabsf(scr[1][h].y)) : fabsf(scr[1][h].x) * (KIND == KV_INT8 ? 128.0f : 448.0f);
                if (most < INFINITY) big = fmaxf(big, most);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
            if (lane == 0) tops[cw] = big;
            if (ct == 0) tops[3] = 0.0f;                           // ct_exponent reads four
            t5::mbar_arrive(b_sc + 8 * (j % CT_SC));
            asm volatile("bar.sync 9, 96;\n" ::: "memory");        // the largest of all three warps
            const float unit = ct_pow2(13 - ct_exponent(tops));
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t row = ct + h * 96;
                const float2 sc = ct_scale<KIND>(scr[1][h], unit);
                if (row < CT_POS) {
                    if constexpr (NSC == 2) reinterpret_cast<float2 *>(vsc)[row] = sc;
                    else vsc[row] = sc.x;
                }
            }
            at_k = units(j + 1, page);
            page = look(j + 2);
            load_scales(next, at_k);
            const uint32_t kt = base + C::K_OFF + st * C::TILE, vt = base + C::V_OFF + st * C::TILE;
            clear(now);
#pragma unroll
            for (int g = 0; g < MINE; g += G) {
#pragma unroll
                for (int i = g; i < g + G && i < MINE; i++)
                    if (i < FULL || row0 + i * STEP < CT_POS) ct_convert<KIND, false>(kt + i * STEP * 128, STEP % 8 ? (i & 1) << 6 : 0, to, swap, reg[i], make_float2(1.0f, 0.0f));
                load(a.c.v, g, at_v);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            t5::mbar_arrive(b_kfull + 8 * st);
            asm volatile("bar.sync 9, 96;\n" ::: "memory");        // the scales of all three warps
            t5::mbar_wait_warp(b_vempty + 8 * st, ph ^ 1, err_flag);
            const uint32_t v_at = base + C::SC_OFF + (j % CT_SC) * C::SLOT + (CT_POS + row0) * NSC * 4;
            clear(now);
#pragma unroll
            for (int g = 0; g < MINE; g += G) {
                float2 sc[G];
#pragma unroll
                for (int i = 0; i < G; i++) {
                    sc[i] = make_float2(0.0f, 0.0f);
                    if (g + i < MINE && (g + i < FULL || row0 + (g + i) * STEP < CT_POS)) {
                        if constexpr (NSC == 2) sc[i] = ct_lds2(v_at + (g + i) * STEP * NSC * 4);
                        else sc[i].x = ct_lds(v_at + (g + i) * STEP * NSC * 4);
                    }
                }
#pragma unroll
                for (int i = g; i < g + G && i < MINE; i++)
                    if (i < FULL || row0 + i * STEP < CT_POS) ct_convert<KIND, true>(vt + i * STEP * 128, STEP % 8 ? (i & 1) << 6 : 0, to, swap, reg[i], sc[i - g]);
                load(a.c.k, g, at_k);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            t5::mbar_arrive(b_vfull + 8 * st);
        }
    }
    __syncthreads();
    t5::fence_after();
    if (warp == C::ISSUER) t5::tmem_dealloc(tmem, 512);
    if (tid == 0 && *err_flag) atomicExch(a.c.err, 5u);
}

// ---- host side -----------------------------------------------------------------------------------
template <int KIND, int HD>
static int launch_tiles(prism_cuda_ctx *ctx, const CacheAttnDev &a, uint32_t max_length) {
    using C = CtCfg<KIND, HD>;
    static bool configured[PRISM_MAX_DEVICES] = {false};
    if (!configured[ctx->device]) {
        PRISM_CUDA_TRY(ctx, cudaFuncSetAttribute(cache_tiles_kernel<KIND, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
        configured[ctx->device] = true;
    }
    CtDev d{};
    d.a = a;
    d.tiles = (uint32_t)(((uint64_t)a.max_tokens * a.group + CT_ROWS - 1) / CT_ROWS);
    const uint64_t items = (uint64_t)a.n_entries * a.c.kv_heads * d.tiles;
    uint64_t seen = max_length;
    if (a.window) seen = std::min<uint64_t>(seen, (uint64_t)a.window + a.sinks + 2 * CT_POS + CT_ROWS / a.group);
    const uint64_t most = std::max<uint64_t>(1, (seen + CT_POS - 1) / CT_POS);
    d.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, ctx->sm_count / items));
    if (items * d.splits > 0x7FFFFFFFull) return fail(ctx, PRISM_E_ARG, "cache_attention: too many rows");
    const uint64_t rows = ((uint64_t)a.c.n_pages * a.c.kv_heads) << a.c.shift;
    d.box = std::min<uint32_t>(CT_POS, 1u << a.c.shift);
    d.pool_rows = (uint32_t)rows;
    CUtensorMap k{}, v{};
    if constexpr (KIND <= KV_BF16) {
        PRISM_TRY(encode_tensor_map(ctx, &k, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.c.k, HD, rows, HD, 64, d.box, CU_TENSOR_MAP_SWIZZLE_128B));
        PRISM_TRY(encode_tensor_map(ctx, &v, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.c.v, HD, rows, HD, 64, d.box, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    if (d.splits > 1) PRISM_TRY(cache_scratch(ctx, (size_t)(items * d.splits) * cache_part_floats(CT_ROWS, HD) * 4, 0, &d.part, nullptr));
    launch_pdl(ctx, "cache_tiles_kernel", cache_tiles_kernel<KIND, HD>, dim3((uint32_t)(items * d.splits)), dim3(C::THREADS), C::SMEM, d, k, v);
    PRISM_TRY(after_launch(ctx, "cache_tiles_kernel"));
    return d.splits > 1 ? launch_cache_join<KIND, HD>(ctx, CacheJoinDev{a, d.splits, d.tiles, CT_ROWS, d.part}) : PRISM_OK;
}

bool cache_tiles_fit(const CacheAttnDev &a, uint32_t hd) {
    const uint64_t rows = ((uint64_t)a.c.n_pages * a.c.kv_heads) << a.c.shift;
    return (hd == 64 || hd == 128) && rows < 0x7FFFFFFFull;  // a copy's coordinate has 31 bits
}

int launch_cache_tiles(prism_cuda_ctx *ctx, int kind, uint32_t hd, const CacheAttnDev &a, uint32_t max_length) {
    auto go = [&](auto k) {
        constexpr int KIND = decltype(k)::value;
        return hd == 64 ? launch_tiles<KIND, 64>(ctx, a, max_length) : launch_tiles<KIND, 128>(ctx, a, max_length);
    };
    switch (kind) {
    case KV_F16: return go(std::integral_constant<int, KV_F16>());
    case KV_BF16: return go(std::integral_constant<int, KV_BF16>());
    case KV_INT8: return go(std::integral_constant<int, KV_INT8>());
    case KV_E4M3: return go(std::integral_constant<int, KV_E4M3>());
    default: return go(std::integral_constant<int, KV_INT4>());
    }
}

}  // namespace prism
