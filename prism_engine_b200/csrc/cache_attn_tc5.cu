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
//                 by the exponent in which its tile lies below the largest so far.  Where positions' values lie more than 2^16 apart, seen or
//                 not, the rows are taken by themselves.
//
// Why 16 bits where they are: the products take 16-bit operands at twice the rate of 32-bit ones, from tiles of half the size.  A weight is
// rounded once, to the rows' type or fp16 (2^-8 or 2^-11 of itself), as the result is; q over a power of two keeps its bits but for elements 2^-14 of
// its largest; a coded value is rounded once to fp16 (2^-11), where its scale kept apart would have to go into each row's weight.  The polynomial of a
// quarter of the 16-bit exponentials is off by 2.6e-6, far below the rounding of the weight that follows.  Scores, maxima, sums and O are 32 bits.
//
// Positions past the end are zero.  A position that a row does not see meets weight 0, which an infinity there turns into NaN: a row whose
// result is not finite is taken again by itself (cache_plain_row), after all parts of its block.
// Few row tiles: the positions are cut into parts whose fp32 sums cache_join_kernel joins in order.  More of them: the blocks, one an SM, share
// all tiles of positions evenly, whatever the lengths, and copies and conversions of a row tile begin under the results of the one before.
// Bound: the tensor core and the instructions about the scores together: 2 048 cycles of products for 256 rows and 128 positions of a 128-wide head,
// as many for their exponentials, and some 5 instructions a score (codes: 6 to 7) on four schedulers; a tile takes 4 300 cycles of 16-bit rows.
// Besides, 15 000 cycles a row tile: q, the first products, results.
// 28 heads of 128 over 4, 2 x 2048 tokens over 6001 positions, bf16: 316 us (0.92 PFLOP/s), under a window of 1024 129 us; int8 535 us, int4
// 570 us.  8 x 63 drafted tokens of 64 heads over 4100 positions: int8 99 us, 16 bits 76 us.
#include <algorithm>

#include "cache_join.cuh"
#include "tc5_ptx.cuh"
#include "tensor_map.cuh"

namespace prism {

constexpr int CT_ROWS = 256, CT_POS = 128, CT_ST = 2, CT_SC = 4;  // slots of scales
constexpr uint32_t CT_PAIRS = 1024;                            // row tiles of all entries that are dealt by their work
constexpr int CT_SOFT = 16;                                     // softmax warps: two threads a row, half of the positions each
// A row tile costs as many units as it has position tiles, but at least a CT_LEAST-th of the longest: with at most CT_ITEMS row tiles an SM a
// block has at most CT_ITEMS * CT_LEAST + 2 parts.
constexpr uint32_t CT_LEAST = 4, CT_ITEMS = 8, CT_SEGMENTS = CT_LEAST * CT_ITEMS + 2;
// Powers of two that the largest values of two positions of a part may lie apart, seen or not: their rows are taken by themselves else.  With values
// to 2^14 in fp16, the scale of one 2^16 below is held to 2^-15, and a weight of a tile that far below the others' to 2^-21 of its largest.
constexpr int CT_APART = 16;
constexpr float CT_GROW = 3.0f, CT_UP = 12.0f;  // powers of two: what a score may lie above the maximum in use; of the weights in fp16
// Part of a row tile that a block does.
struct CtSegment {
    CacheEntry x;
    uint32_t item, kh, r0, here, n_q, n;  // row tile of an entry and head, its head, first row, rows, tiles of 128 rows; position tiles of this part
    int32_t i_lo, first, main, start, end;  // the first of them; CtTiles
    uint32_t whole;                       // the whole row tile
    uint32_t units, from, take;           // of the row tile, of this part
    uint32_t b0, b1, slot, slot0;         // blocks that have parts of the item; places of this block's part and of b0's
    // barriers go on from part to part: position tiles before this one (T1: with a second tile of rows), parts with such tiles
    uint32_t T, T1, S0, S1;
    uint32_t again[CT_ROWS / 32];         // rows to be taken again by themselves: a bit each
    uint32_t wide;                        // values of its position tiles lie too far apart for fp16 (CT_APART)
};
template <int KIND, int HD>
struct CtCfg {
    static constexpr int PANELS = HD / 64, PANEL = 128 * 128, TILE = PANELS * PANEL;  // 128 rows of 64 values, in the 128-byte swizzle
    static constexpr int NSC = (int)kv_scales<KIND>(), ROWB = HD * (int)kv_bits<KIND>() / 8;
    static constexpr int SLOT = NSC ? 2 * CT_POS * NSC * 4 + 32 : 0;                   // key scales, value scales, each converting warp's largest value by the latter, its smallest but 0
    static constexpr int K_OFF = 2 * TILE, V_OFF = K_OFF + CT_ST * TILE, SC_OFF = V_OFF + CT_ST * TILE, BAR_OFF = SC_OFF + CT_SC * SLOT;
    // barriers: kfull, kempty, vfull, vempty [2 each], sfull, pfull, ofull, qfull [2 each], scales [4]
    static constexpr int STATE_OFF = BAR_OFF + 8 * (4 * CT_ST + 8 + CT_SC);
    static constexpr int X_OFF = STATE_OFF + 24;                                       // what the two threads of a row tell each other
    static constexpr int R_OFF = X_OFF + 2 * 2 * CT_ROWS * 4;                          // CacheRow of each row
    static constexpr int PRE_OFF = R_OFF + CT_ROWS * (int)sizeof(CacheRow);            // position tiles of the row tiles before each
    static constexpr int SEG_OFF = PRE_OFF + (CT_PAIRS + 4) * 4;                       // what the block does
    static constexpr size_t SMEM = SEG_OFF + CT_SEGMENTS * sizeof(CtSegment) + 1024;
    // behind the softmax warps three that convert (one of them copies, with 16-bit rows) and one of products: five warps a scheduler, 96 registers
    static constexpr int CONV = 96, ISSUER = CT_SOFT + 3, THREADS = (ISSUER + 1) * 32;
    static constexpr int RP = ROWB / 16, STEP = CONV / RP;                             // 16-byte pieces of a row; rows between a thread's pieces
    static constexpr int MINE = (CT_POS + STEP - 1) / STEP;                            // a thread's pieces of a tile
};

struct CtDev {
    CacheAttnDev a;
    uint32_t splits, tiles, box;  // parts of the positions (0: the blocks share the work, below), row tiles of an entry and head, positions of a copy
    uint32_t pool_rows;           // rows of the pool: one past the last
    float *part;                  // of the blocks, where there are several of a row tile (CacheJoinDev); shared work: two a block
    unsigned int *count;          // shared work: [row tile of an entry and head], zero between launches
};

namespace {

// The 128-position tiles that some row of a row tile sees: `first` of them from position 0 on (a.sinks), then those from `main` on.
struct CtTiles {
    uint32_t here;              // rows of the tile
    int32_t first, main, all;   // `all` of them
    int32_t start, end;         // seen by some row: positions below end that are not below start, and the first a.sinks
};
// WARP: called by whole warps, which share the rows of a tree.
template <bool WARP>
__device__ __forceinline__ CtTiles ct_tiles(const CacheAttnDev &a, const CacheEntry &x, uint32_t tile) {
    const uint32_t n_rows = x.n * a.group, r0 = tile * CT_ROWS;
    CtTiles t{r0 < n_rows ? min((uint32_t)CT_ROWS, n_rows - r0) : 0, 0, 0, 0, 0, 0};
    if (t.here == 0) return t;
    const uint32_t tok_lo = r0 / a.group, tok_hi = (r0 + t.here - 1) / a.group;
    int32_t low = -1;
    if (a.window && !a.tree) low = cache_row(a, x, tok_lo).low;
    else if (a.window) {
        low = x.len;
        for (uint32_t i = tok_lo + (WARP ? threadIdx.x & 31 : 0); i <= tok_hi; i += WARP ? 32 : 1) low = min(low, cache_row(a, x, i).low);
        if (WARP) low = __reduce_min_sync(0xFFFFFFFFu, low);
    }
    const int32_t end = a.tree ? x.len : min(x.len, x.first + (int32_t)tok_hi + 1), start = a.tree ? min(low + 1, max(x.first, 0)) : low + 1;
    const int32_t main_hi = end > 0 ? (end + CT_POS - 1) / CT_POS : 0;
    t.first = end > 0 ? (int32_t)(min((uint32_t)end, a.sinks) + CT_POS - 1) / CT_POS : 0;
    t.main = max(start / CT_POS, t.first);
    t.all = t.first + max(main_hi - t.main, 0);
    t.start = start;
    t.end = end;
    return t;
}

__device__ __forceinline__ float ct_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 numbers in neighbouring registers, and operations on both at once; the largest of three.
__device__ __forceinline__ uint64_t ct_two(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint64_t ct_two(float a, float b) { return ct_two(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ uint32_t ct_first(uint64_t v) { return (uint32_t)v; }
__device__ __forceinline__ uint32_t ct_second(uint64_t v) { return (uint32_t)(v >> 32); }
__device__ __forceinline__ uint64_t ct_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t ct_mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t ct_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// 2^x of two numbers on the multiply-add pipe, where the special function unit is the bound: x = n + f with n the nearest whole number (1.5 * 2^23
// added and taken off), 2^f by a polynomial of degree 4 fitted to the smallest relative error on [-1/2, 1/2] (2.6e-6), n added to the
// exponent.  LOW: numbers to 2^-126 give 0, as the unit gives (bf16 holds 2^-126, and a value may be 2^127): all results are less by what the
// polynomial makes of 2^-126.  Else they give 2^-126, of which fp16 keeps nothing.
template <bool LOW>
__device__ __forceinline__ uint64_t ct_exp2(uint64_t x) {
    float a, b;  // a NaN stays one, and ends as an infinite weight
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(a) : "f"(__uint_as_float(ct_first(x))), "f"(-126.0f));
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(b) : "f"(__uint_as_float(ct_second(x))), "f"(-126.0f));
    const uint64_t y = ct_two(a, b), t = ct_add2(y, ct_two(12582912.0f, 12582912.0f));
    const uint64_t f = ct_fma2(ct_add2(t, ct_two(-12582912.0f, -12582912.0f)), ct_two(-1.0f, -1.0f), y);
    uint64_t p = ct_fma2(ct_two(0.009570102207362652f, 0.009570102207362652f), f, ct_two(0.05591786280274391f, 0.05591786280274391f));
    p = ct_fma2(p, f, ct_two(0.240247443318367f, 0.240247443318367f));
    p = ct_fma2(p, f, ct_two(0.6931217908859253f, 0.6931217908859253f));
    p = ct_fma2(p, f, ct_two(0.9999992847442627f, 0.9999992847442627f));
    const uint64_t e = ct_two(ct_first(p) + (ct_first(t) << 23), ct_second(p) + (ct_second(t) << 23));
    return LOW ? ct_add2(e, ct_two(0x807FFFF4u, 0x807FFFF4u)) : e;
}
__device__ __forceinline__ float ct_max3(float a, uint32_t b, uint32_t c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return d;
}
__device__ __forceinline__ uint32_t ct_below(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }
__device__ __forceinline__ float ct_pow2(int32_t e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// Exponent of the largest of four numbers, each not negative; of the smallest.
__device__ __forceinline__ int32_t ct_exponent(const float *top) {
    const float4 a = *reinterpret_cast<const float4 *>(top);
    return max((int32_t)(__float_as_uint(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w))) >> 23) - 127, -100);
}
__device__ __forceinline__ int32_t ct_least_exponent(const float *low) {
    const float4 a = *reinterpret_cast<const float4 *>(low);
    return (int32_t)(__float_as_uint(fminf(fminf(a.x, a.y), fminf(a.z, a.w))) >> 23) - 127;
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

// Where 16-byte piece c of a row of q lies.
template <int HD>
__device__ __forceinline__ uint8_t *ct_q_piece(uint8_t *sm, uint32_t q, uint32_t row, uint32_t c) {
    return sm + q * CtCfg<KV_F16, HD>::TILE + (c >> 3) * CtCfg<KV_F16, HD>::PANEL + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

// The results of a row tile's part that this thread's row has, half of the columns: stored, or left as a part, which the last block to arrive joins.
// A function of its own: inlined into the loop over parts it took some 350 registers more than there are.
template <int KIND, int HD>
__device__ __noinline__ void ct_results(const CtDev &d, CtSegment &g, uint8_t *sm, uint32_t o_col, uint32_t warp, uint32_t lane, uint32_t mine, float m,
                                        float l, int32_t ref) {
    using C = CtCfg<KIND, HD>;
    constexpr bool CODES = KIND >= KV_INT8;
    const CacheAttnDev &a = d.a;
    const uint32_t q = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane, tid = warp * 32 + lane;
    const bool there = q * 128 + row < g.here;
    volatile uint32_t *last_flag = reinterpret_cast<volatile uint32_t *>(sm + C::STATE_OFF + 16);
    float *xch = reinterpret_cast<float *>(sm + C::X_OFF) + q * 128 + row;
    auto other = [&](float v, uint32_t turn) {
        xch[(turn * 2 + half) * CT_ROWS] = v;
        asm volatile("bar.sync %0, 64;\n" ::"r"(1 + q * 4 + (warp & 3)) : "memory");
        return xch[(turn * 2 + (half ^ 1)) * CT_ROWS];
    };
    // ---- results, half of the columns a thread: O times 2^(ref - 13) where V was over a power of two, as the weights' sum is 2^12-fold ----
    const float unit = CODES ? ct_pow2(ref - 13) : 1.0f;
    if (g.wide) l = __uint_as_float(0x7FC00000u);                  // and so is what this part is joined to
    float inv = 1.0f / l, odd = l > 0.0f && m > -INFINITY ? 0.0f : 1.0f;  // not 0 once an output was not finite; a row without a maximum saw nothing, or only -inf
    const uint32_t rr = g.r0 + q * 128 + row;
    // Half a row a thread, through where its half of q was: the products that read it are complete.
    constexpr int W = HD / 16, AT = 32 / W;                        // 16-byte pieces of half a row; rows that a warp stores at once
    uint16_t *dst = a.out + (size_t)(g.x.row0 + (there ? rr / a.group : 0)) * a.out_stride + (size_t)(g.kh * a.group + (there ? rr % a.group : 0)) * HD + half * (HD / 2);
    auto store = [&](int c, const float (&o)[32]) {            // 32 columns
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float u = o[ct_col<KIND>(2 * i)] * inv, v = o[ct_col<KIND>(2 * i + 1)] * inv;
            odd = fmaf(u, 0.0f, fmaf(v, 0.0f, odd));
            w[i] = kv_round2(u, v, a.c.rows_bf16);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(ct_q_piece<HD>(sm, q, row, half * W + c * 4 + i)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    };
    auto stored = [&]() {                                      // all columns
        __syncwarp();
#pragma unroll
        for (int i = 0; i < W; i++) {
            const uint32_t r = i * AT + lane / W, at = row - lane + r;
            const uint4 v = *reinterpret_cast<const uint4 *>(ct_q_piece<HD>(sm, q, at, half * W + lane % W));
            uint16_t *to = reinterpret_cast<uint16_t *>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(dst), r));
            if (q * 128 + at < g.here) reinterpret_cast<uint4 *>(to)[lane % W] = v;
        }
    };
    bool done = g.whole;
    if (g.whole) {
#pragma unroll 1
        for (int c = 0; c < HD / 64; c++) {
            uint32_t o[32];
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = 0;
            if (mine) {
                t5::ld32(o_col + c * 32, o);
                t5::wait_ld();
            }
#pragma unroll
            for (int i = 0; i < 32; i++) v[i] = __uint_as_float(o[i]) * unit;
            store(c, v);
            __syncwarp();                                      // the next TMEM read takes the whole warp
        }
        stored();
    } else {
        constexpr size_t PART = cache_part_floats(CT_ROWS, HD);
        const size_t at = q * 128 + row, c_first = half * (HD / 8);  // groups of four columns
        float *to = d.part + g.slot * PART;
#pragma unroll 1
        for (int c = 0; c < HD / 64; c++) {
            uint32_t o[32];
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = 0;
            if (mine) {
                t5::ld32(o_col + c * 32, o);
                t5::wait_ld();
            }
            if (there) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const auto col = [&](int k) { return __uint_as_float(o[ct_col<KIND>(4 * i + k)]) * unit; };
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
        if (d.splits == 0) {                                   // else cache_join_kernel follows
            __threadfence();
            asm volatile("bar.sync 10, 512;\n" ::: "memory");
            if (tid == 0) {
                const bool last = atomicAdd(d.count + g.item, 1u) == g.b1 - g.b0;
                if (last) d.count[g.item] = 0;                   // for the next launch
                *last_flag = last;
            }
            asm volatile("bar.sync 10, 512;\n" ::: "memory");
            done = *last_flag;
            if (done && q < g.n_q) {
                const uint32_t b0 = g.b0, b1 = g.b1;
                __threadfence();
                auto part = [&](uint32_t b) { return d.part + (b == b0 ? g.slot0 : 2 * b) * PART + at; };
                float best = -INFINITY;
                for (uint32_t b = b0; b <= b1; b++) best = fmaxf(best, __ldcg(part(b) + CT_ROWS * HD));
                const float sub = best == -INFINITY ? 0.0f : best;
                l = 0.0f;
                for (uint32_t b = b0; b <= b1; b++) l += __ldcg(part(b) + CT_ROWS * (HD + 1)) * ct_ex2(__ldcg(part(b) + CT_ROWS * HD) - sub);
                inv = 1.0f / l;
                odd = l > 0.0f ? 0.0f : 1.0f;
#pragma unroll 1
                for (int c = 0; c < HD / 64; c++) {
                    float v[32];                               // in the order that store() takes
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = 0.0f;
                    for (uint32_t b = b0; b <= b1 && there; b++) {
                        const float f = ct_ex2(__ldcg(part(b) + CT_ROWS * HD) - sub);
                        const float4 *p = reinterpret_cast<const float4 *>(part(b) - at) + (c_first + c * 8) * CT_ROWS + at;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float4 u = __ldcg(p + (size_t)i * CT_ROWS);
                            v[ct_col<KIND>(4 * i)] = fmaf(u.x, f, v[ct_col<KIND>(4 * i)]);
                            v[ct_col<KIND>(4 * i + 1)] = fmaf(u.y, f, v[ct_col<KIND>(4 * i + 1)]);
                            v[ct_col<KIND>(4 * i + 2)] = fmaf(u.z, f, v[ct_col<KIND>(4 * i + 2)]);
                            v[ct_col<KIND>(4 * i + 3)] = fmaf(u.w, f, v[ct_col<KIND>(4 * i + 3)]);
                        }
                    }
                    store(c, v);
                }
                stored();
            }
        }
    }
    const float theirs = other(odd, (mine & 1) ^ 1);           // every lane takes part; after what the other thread stored
    const uint32_t again = __ballot_sync(0xFFFFFFFFu, done && there && (odd != 0.0f || theirs != 0.0f));
    if (half == 0 && lane == 0) g.again[q * 4 + (warp & 3)] = again;
}

}  // namespace

template <int KIND, int HD>
__global__ void __launch_bounds__(CtCfg<KIND, HD>::THREADS, 1) cache_tiles_kernel(const __grid_constant__ CtDev d, const __grid_constant__ CUtensorMap kmap,
                                                                    const __grid_constant__ CUtensorMap vmap) {
    using C = CtCfg<KIND, HD>;
    constexpr bool CODES = KIND >= KV_INT8, BF16 = KIND == KV_BF16;
    // of 8 pairs of exponentials, those on the multiply-add pipe (ct_exp2): a group of 28 of 128-wide heads, 2048 tokens over 6144 positions, 16-bit
    // rows: none 344 us, 2 323 us, 4 356 us; int8, whose instructions are the bound already: none 513 us, 2 540 us
    constexpr int POLY = CODES ? 0 : 2;
    constexpr int ST = CT_ST, NSC = C::NSC;
    const CacheAttnDev &a = d.a;
    extern __shared__ uint8_t ct_raw[];
    uint8_t *smem = ct_raw + (1024 - ((uint32_t)__cvta_generic_to_shared(ct_raw) & 1023u)) % 1024;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
    pdl_launch_dependents();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t b_kfull = base + C::BAR_OFF, b_kempty = b_kfull + 8 * ST, b_vfull = b_kempty + 8 * ST, b_vempty = b_vfull + 8 * ST,
                   b_sfull = b_vempty + 8 * ST, b_pfull = b_sfull + 16, b_ofull = b_pfull + 16, b_qfull = b_ofull + 16, b_sc = b_qfull + 16;
    volatile uint32_t *err_flag = reinterpret_cast<volatile uint32_t *>(smem + C::STATE_OFF);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::STATE_OFF + 8);
    if (tid == 0) {
        for (int s = 0; s < ST; s++) {
            t5::mbar_init(b_kfull + 8 * s, CODES ? C::CONV : 1); t5::mbar_init(b_kempty + 8 * s, 1);
            t5::mbar_init(b_vfull + 8 * s, CODES ? C::CONV : 1); t5::mbar_init(b_vempty + 8 * s, 1);
        }
        for (int q = 0; q < 2; q++) { t5::mbar_init(b_sfull + 8 * q, 1); t5::mbar_init(b_pfull + 8 * q, CT_SOFT / 2); t5::mbar_init(b_ofull + 8 * q, 1); t5::mbar_init(b_qfull + 8 * q, CT_SOFT / 2); }
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

    // ---- what this block does ----------------------------------------------------------------------------------------------
    // d.splits > 0: one part of one row tile.  Else all blocks share the position tiles of all row tiles evenly, in order: a block has the rest of
    // a row tile, whole ones, the beginning of another.  Row tile i of entry e is pair e * d.tiles + i, an item is a pair and a head.
    uint32_t *pre = reinterpret_cast<uint32_t *>(smem + C::PRE_OFF);
    CtSegment *segs = reinterpret_cast<CtSegment *>(smem + C::SEG_OFF);
    {
        const uint32_t kvh = a.c.kv_heads, pairs = a.n_entries * d.tiles;
        if (d.splits == 0) {
            for (uint32_t i = tid; i < pairs; i += C::THREADS) {
                CacheEntry x;
                uint32_t c = 0;
                if (cache_entry(a, i / d.tiles, x)) {
                    const CtTiles t = ct_tiles<false>(a, x, i % d.tiles);
                    if (t.here) c = (uint32_t)max(t.all, 1);       // rows that see nothing are results, too
                }
                pre[i + 1] = c;
            }
            __syncthreads();
            if (warp == 0) {
                const uint32_t per = (pairs + 31) / 32, lo = min(lane * per, pairs), hi = min(lo + per, pairs);
                uint32_t longest = 0, sum = 0;
                for (uint32_t i = lo; i < hi; i++) longest = max(longest, pre[i + 1]);
                longest = __reduce_max_sync(0xFFFFFFFFu, longest);
                auto cost = [&](uint32_t c) { return c ? max(c, (longest + CT_LEAST - 1) / CT_LEAST) : 0; };
                for (uint32_t i = lo; i < hi; i++) sum += cost(pre[i + 1]);
                uint32_t all = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, all, o);
                    if (lane >= (uint32_t)o) all += v;
                }
                sum = all - sum;
                if (lane == 0) pre[0] = 0;
                for (uint32_t i = lo; i < hi; i++) pre[i + 1] = sum += cost(pre[i + 1]);
                __syncwarp();
                if (lane == 0) {
                    const uint64_t total = (uint64_t)pre[pairs] * kvh, G = min((uint64_t)gridDim.x, total);  // every block of G has a unit
                    const uint64_t end = blockIdx.x < G ? total * (blockIdx.x + 1) / G : 0;
                    uint64_t at = blockIdx.x < G ? total * blockIdx.x / G : 0;
                    uint32_t k = 0, p = 0, hi2 = pairs;
                    while (hi2 - p > 1) {                          // the last pair that begins at or before this unit
                        const uint32_t mid = (p + hi2) / 2;
                        if ((uint64_t)pre[mid] * kvh <= at) p = mid;
                        else hi2 = mid;
                    }
                    for (; at < end && k < CT_SEGMENTS; k++) {
                        while ((uint64_t)pre[p + 1] * kvh <= at) p++;
                        CtSegment &g = segs[k];
                        const uint32_t units = pre[p + 1] - pre[p], in = (uint32_t)(at - (uint64_t)pre[p] * kvh);
                        g.kh = in / units;
                        g.item = p * kvh + g.kh;
                        g.units = units;
                        g.from = in % units;
                        g.take = (uint32_t)min((uint64_t)(units - g.from), end - at);
                        g.whole = g.take == units;
                        const uint64_t item_unit = at - g.from;
                        g.b0 = (uint32_t)(((item_unit + 1) * G - 1) / total);
                        g.b1 = (uint32_t)(((item_unit + units) * G - 1) / total);
                        g.slot0 = 2 * g.b0 + (total * g.b0 / G < item_unit);  // a block's first part, or its last
                        g.slot = blockIdx.x == g.b0 ? g.slot0 : 2 * blockIdx.x;
                        at += g.take;
                    }
                    pre[CT_PAIRS + 1] = k;
                }
            }
        } else if (tid == 0) {
            CtSegment &g = segs[0];
            g.item = blockIdx.x / d.splits;
            g.kh = g.item / d.tiles % kvh;
            g.whole = d.splits == 1;
            g.slot = blockIdx.x;
            g.units = d.splits;
            g.from = blockIdx.x % d.splits;
            g.take = 1;
            pre[CT_PAIRS + 1] = 1;
        }
        __syncthreads();
        for (uint32_t k = warp; k < pre[CT_PAIRS + 1]; k += C::THREADS / 32) {
            CtSegment &g = segs[k];
            const uint32_t pair = d.splits ? g.item / d.tiles / kvh * d.tiles + g.item % d.tiles : g.item / kvh;
            CacheEntry x{};
            CtTiles t{};
            if (cache_entry(a, pair / d.tiles, x)) t = ct_tiles<true>(a, x, pair % d.tiles);  // the same in all blocks of an item
            if (lane < CT_ROWS / 32) g.again[lane] = 0;
            if (lane == 0) {
                g.wide = 0;
                g.x = x;
                g.r0 = pair % d.tiles * CT_ROWS;
                g.here = t.here;
                g.n_q = (t.here + 127) / 128;
                g.first = t.first;
                g.main = t.main;
                g.start = t.start;
                g.end = t.end;
                g.i_lo = (int32_t)((int64_t)t.all * g.from / g.units);
                g.n = (uint32_t)((int32_t)((int64_t)t.all * (g.from + g.take) / g.units) - g.i_lo);
            }
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t T = 0, T1 = 0, S0 = 0, S1 = 0;
            for (uint32_t k = 0; k < pre[CT_PAIRS + 1]; k++) {
                CtSegment &g = segs[k];
                g.T = T;
                g.T1 = T1;
                g.S0 = S0;
                g.S1 = S1;
                T += g.n;
                T1 += g.n_q == 2 ? g.n : 0;
                S0 += g.n > 0;
                S1 += g.n > 0 && g.n_q == 2;
            }
            pre[CT_PAIRS + 2] = T;
        }
        __syncthreads();
    }
    const uint32_t n_segs = pre[CT_PAIRS + 1];
    auto pos_of = [](const CtSegment &g, uint32_t j) {
        const int32_t i = g.i_lo + (int32_t)j;
        return (i < g.first ? i : g.main + (i - g.first)) * CT_POS;
    };

    // Whether some row of the part sees one of `span` positions from p on: pages of others are not asked for, they may be gone.
    auto wanted = [&](const CtSegment &g, int32_t p, int32_t span) { return p < g.end && (p + span > g.start || (uint32_t)p < a.sinks); };

    if (warp < CT_SOFT) {
        // ================= softmax: two threads a query row, positions 0..63 and 64..127 of a tile =================
        for (uint32_t k = 0; k < n_segs; k++) {
        // Taken anew for every part: kept over the loop, what follows from them would take more registers than there are.
        uint32_t w_now = warp, l_now = lane, t_now = tmem, s_now = 0;
        asm volatile("" : "+r"(w_now), "+r"(l_now), "+r"(t_now), "+r"(s_now));
        uint8_t *const sm = smem + s_now;
        const uint32_t q = w_now >> 3, half = w_now >> 2 & 1, row = (w_now & 3) * 32 + l_now, lanes = ((w_now & 3) * 32) << 16;
        const uint32_t s_col = t_now + lanes + q * 128, o_col = t_now + lanes + 256 + q * HD + half * (HD / 2);
        float *xch = reinterpret_cast<float *>(sm + C::X_OFF) + q * 128 + row;  // [turn][half][256 rows]
        // The value of the row's other thread.  Turns alternate: both have read one turn's before either writes it again.
        auto other = [&](float v, uint32_t turn) {
            xch[(turn * 2 + half) * CT_ROWS] = v;
            asm volatile("bar.sync %0, 64;\n" ::"r"(1 + q * 4 + (w_now & 3)) : "memory");
            return xch[(turn * 2 + (half ^ 1)) * CT_ROWS];
        };
        CacheRow *row_at = reinterpret_cast<CacheRow *>(sm + C::R_OFF) + q * 128 + row;  // the same in both threads
        CtSegment &g = *(reinterpret_cast<CtSegment *>(sm + C::SEG_OFF) + k);
        if (g.here == 0) continue;
        const bool there = q * 128 + row < g.here;
        const uint32_t mine = q < g.n_q ? g.n : 0, T = g.T, Tq = q ? g.T1 : T;
        int32_t all_to, all_low;
        {
            CacheRow r{0x7FFFFFF0, -1, nullptr};                   // a row that is not there: sees everything, is not stored
            if (there) r = cache_row(a, g.x, (g.r0 + q * 128 + row) / a.group);
            all_to = __reduce_min_sync(0xFFFFFFFFu, r.last);
            all_low = __reduce_max_sync(0xFFFFFFFFu, r.low);
            *row_at = r;
        }
        float mul = fabsf(a.scale) * 1.4426950408889634f, qsum = 0.0f;
        {   // half of the row of q into its tile, its sign that of the scale
            constexpr int W = HD / 16, AT = 32 / W;                // 16-byte pieces; rows that a warp fetches at once
            const uint32_t rr = g.r0 + q * 128 + row, token = there ? rr / a.group : 0, head = g.kh * a.group + (there ? rr % a.group : 0);
            const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
            const uint16_t *src = a.q + (size_t)(g.x.row0 + token) * a.q_stride + (size_t)head * HD + half * (HD / 2);
            uint4 w[W];
#pragma unroll
            for (int i = 0; i < W; i++) {
                const uint32_t r = i * AT + l_now / W;
                const uint16_t *from = reinterpret_cast<const uint16_t *>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(src), r));
                w[i] = q * 128 + row - l_now + r < g.here ? reinterpret_cast<const uint4 *>(from)[l_now % W] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < W; i++) {
                uint32_t *u = reinterpret_cast<uint32_t *>(&w[i]);
#pragma unroll
                for (int k = 0; k < 4; k++) u[k] ^= flip;
                *reinterpret_cast<uint4 *>(ct_q_piece<HD>(sm, q, row - l_now + i * AT + l_now / W, half * W + l_now % W)) = w[i];
            }
            if constexpr (CODES) {                                 // over the power of two below the largest
                __syncwarp();
                float big = 0.0f;
#pragma unroll
                for (int i = 0; i < W; i++) {
                    w[i] = *reinterpret_cast<const uint4 *>(ct_q_piece<HD>(sm, q, row, half * W + i));
                    uint32_t *u = reinterpret_cast<uint32_t *>(&w[i]);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        big = fmaxf(big, fmaxf(fabsf(kv_row_value((uint16_t)u[k], a.c.rows_bf16)), fabsf(kv_row_value((uint16_t)(u[k] >> 16), a.c.rows_bf16))));
                }
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
#pragma unroll
                for (int i = 0; i < W; i++) *reinterpret_cast<uint4 *>(ct_q_piece<HD>(sm, q, row, half * W + i)) = ct_order<KIND>(w[i]);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            asm volatile("bar.sync %0, 64;\n" ::"r"(1 + q * 4 + (w_now & 3)) : "memory");  // the exchanged values have been read
            // A phase only where the issuer waits for it: a wait tells a phase from the next by its parity alone, so no warp may be two ahead.
            if (l_now == 0 && mine) t5::mbar_arrive(b_qfull + 8 * q);
        }
        float m = -INFINITY, l = 0.0f;
        int32_t ref = 0;                                           // exponent that O is over
        // A warp that had no rows in the parts before may be phases ahead of the slots of scales, and parity would let it read an older tile's
        // exponent.  So it waits for the first scores, which follow their scales, and from then on is in step.  (Scores before scales in every
        // tile: 588 instead of 567 us for 28 heads of 128 over 4, 2 x 2048 tokens over 6001 positions, int4.)
        if (CODES && mine) t5::mbar_wait_warp(b_sfull + 8 * q, Tq & 1, err_flag);
        for (uint32_t j = 0; j < mine; j++) {
            int32_t ex = 0;
            const float *ksc = nullptr;
            if constexpr (CODES) {
                t5::mbar_wait_warp(b_sc + 8 * ((T + j) % CT_SC), ((T + j) / CT_SC) & 1, err_flag);
                ksc = reinterpret_cast<const float *>(sm + C::SC_OFF + ((T + j) % CT_SC) * C::SLOT);
                ex = ct_exponent(ksc + 2 * CT_POS * NSC);
                ksc += half * 64;                                  // scales of all positions, then zeros
            }
            t5::mbar_wait_warp(b_sfull + 8 * q, (Tq + j) & 1, err_flag);
            t5::fence_after();
            uint32_t s[2][32];
#pragma unroll
            for (int c = 0; c < 2; c++) t5::ld32(s_col + half * 64 + c * 32, s[c]);
            t5::wait_ld();
            const int32_t p0 = pos_of(g, j) + (int32_t)half * 64;
            if constexpr (NSC > 0) {
                const uint64_t qs = ct_two(qsum, qsum);
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(ksc + c * 32 + i);
                        uint64_t u = ct_two(s[c][i], s[c][i + 1]), v = ct_two(s[c][i + 2], s[c][i + 3]);
                        if constexpr (NSC == 2) {
                            const float4 z = *reinterpret_cast<const float4 *>(ksc + CT_POS + c * 32 + i);
                            u = ct_fma2(u, ct_two(f.x, f.y), ct_mul2(qs, ct_two(z.x, z.y)));
                            v = ct_fma2(v, ct_two(f.z, f.w), ct_mul2(qs, ct_two(z.z, z.w)));
                        } else {
                            u = ct_mul2(u, ct_two(f.x, f.y));
                            v = ct_mul2(v, ct_two(f.z, f.w));
                        }
                        s[c][i] = ct_first(u);
                        s[c][i + 1] = ct_second(u);
                        s[c][i + 2] = ct_first(v);
                        s[c][i + 3] = ct_second(v);
                    }
            }
            if (p0 + 63 > all_to || !(p0 > all_low || (uint32_t)(p0 + 64) <= a.sinks)) {  // some row of the warp does not see all 64
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const uint32_t see = there ? ct_seen(a, g.x, *row_at, p0 + c * 32) : 0xFFFFFFFFu;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (!(see & (1u << i))) s[c][i] = 0xFF800000u;
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 32; i += 4)
#pragma unroll
                for (int c = 0; c < 4; c++) mx[c] = ct_max3(mx[c], s[c >> 1][i + (c & 1) * 2], s[c >> 1][i + (c & 1) * 2 + 1]);
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
            const uint64_t mul2 = ct_two(mul, mul), less2 = ct_two(-less, -less);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const uint64_t x = ct_fma2(ct_two(s[c][2 * i], s[c][2 * i + 1]), mul2, less2);
                    uint64_t e;
                    if (i % 8 < POLY) e = ct_exp2<BF16>(x);
                    else e = ct_two(ct_ex2(__uint_as_float(ct_first(x))), ct_ex2(__uint_as_float(ct_second(x))));
                    const float e0 = __uint_as_float(ct_first(e)), e1 = __uint_as_float(ct_second(e));
                    sum[i & 1] = ct_add2(sum[i & 1], e);
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
            sum[0] = ct_add2(sum[0], sum[1]);
            float more = __uint_as_float(ct_first(sum[0])) + __uint_as_float(ct_second(sum[0]));
            if constexpr (CODES)
                if (ex != ref) more *= ct_pow2(min(ref - ex, 90));
            l += more;
            t5::wait_st();
            t5::fence_before();
            __syncwarp();
            if (l_now == 0) t5::mbar_arrive(b_pfull + 8 * q);
        }
        l += other(l, mine & 1);
        if (mine) {
            t5::mbar_wait_warp(b_ofull + 8 * q, (q ? g.S1 : g.S0) & 1, err_flag);
            t5::fence_after();
        }
        ct_results<KIND, HD>(d, g, sm, o_col, w_now, l_now, mine, m, l, ref);
        t5::fence_before();
        // the next segment's first exchange takes a turn whose last readers have been at this barrier
        asm volatile("bar.sync %0, 64;\n" ::"r"(1 + q * 4 + (w_now & 3)) : "memory");
        }
    } else if (warp == C::ISSUER) {
        // ================= products: the whole warp walks the tiles (descriptors stay in uniform registers), an elected lane issues;
        // all lanes clear 16-bit value rows past the end =================
        const uint32_t types = BF16 ? 1u << 7 | 1u << 10 : 0u;
        const uint32_t id_s = t5::idesc_f16(128, CT_POS) | types, id_o = t5::idesc_f16(128, HD) | types | (1u << 16);  // V is read across its rows
        auto scores = [&](uint32_t q, uint32_t J) {                // J: of all segments
            const uint32_t qa = base + q * C::TILE, ka = base + C::K_OFF + (J % ST) * C::TILE;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                const uint32_t off = (k * 32 / 128) * C::PANEL + (k * 32) % 128;
                t5::mma_ss(tmem + q * 128, t5::desc_swizzled<128>(qa + off, 16), t5::desc_swizzled<128>(ka + off, 16), id_s, k != 0);
            }
            t5::commit(b_sfull + 8 * q);
        };
        for (uint32_t i = 0; i < n_segs; i++) {
            const CtSegment &g = segs[i];
            const uint32_t n = g.n, n_q = g.n_q, T = g.T, T1 = g.T1;
            if (n) {
                t5::mbar_wait_bounded(b_kfull + 8 * (T % ST), (T / ST) & 1, err_flag);
                for (uint32_t q = 0; q < n_q; q++) {
                    t5::mbar_wait_bounded(b_qfull + 8 * q, (q ? g.S1 : g.S0) & 1, err_flag);
                    __syncwarp();
                    t5::fence_after();
                    if (t5::elect_one()) {
                        scores(q, T);
                        if (q + 1 == n_q) t5::commit(b_kempty + 8 * (T % ST));
                    }
                    __syncwarp();
                }
            }
            for (uint32_t j = 0; j < n; j++) {
                const uint32_t J = T + j, st = J % ST, ph = (J / ST) & 1, va = base + C::V_OFF + st * C::TILE;
                const bool more = j + 1 < n;
                t5::mbar_wait_bounded(b_vfull + 8 * st, ph, err_flag);
                __syncwarp();
                if constexpr (!CODES) {
                    const int32_t left = g.x.len - pos_of(g, j);
                    if (left < CT_POS) {
                        const uint32_t first = (uint32_t)left, cells = (CT_POS - first) * 8 * C::PANELS;
                        for (uint32_t u = lane; u < cells; u += 32) {
                            const uint32_t p = u / ((CT_POS - first) * 8), c = u % ((CT_POS - first) * 8);
                            *reinterpret_cast<uint4 *>(smem + C::V_OFF + st * C::TILE + p * C::PANEL + first * 128 + c * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                        __syncwarp();
                    }
                }
                if (more) t5::mbar_wait_bounded(b_kfull + 8 * ((J + 1) % ST), ((J + 1) / ST) & 1, err_flag);
#pragma unroll
                for (uint32_t q = 0; q < 2; q++) {
                    if (q >= n_q) continue;
                    t5::mbar_wait_bounded(b_pfull + 8 * q, ((q ? T1 : T) + j) & 1, err_flag);
                    __syncwarp();
                    t5::fence_after();
                    if (t5::elect_one()) {
#pragma unroll
                        for (int k = 0; k < CT_POS / 16; k++)
                            t5::mma_ts(tmem + 256 + q * HD, tmem + q * 128 + k * 8, t5::desc_swizzled<128>(va + k * 16 * 128, C::PANEL), id_o, k ? 1u : j);
                        if (more) scores(q, J + 1);
                        else t5::commit(b_ofull + 8 * q);
                    }
                    __syncwarp();
                }
                if (t5::elect_one()) {
                    t5::commit(b_vempty + 8 * st);
                    if (more) t5::commit(b_kempty + 8 * ((J + 1) % ST));
                }
                __syncwarp();
            }
        }
        t5::fence_before();
    } else if constexpr (!CODES) {
        // ================= copies =================
        // A lane a box (of at most eight): its page is asked for a tile before it is needed.
        if (warp == CT_SOFT) {
            const uint32_t boxes = CT_POS / d.box, b = lane % boxes;
            auto look = [&](const CtSegment &g, uint32_t j) {
                const int32_t p = j < g.n ? pos_of(g, j) + (int32_t)(b * d.box) : 0;
                return j < g.n && wanted(g, p, (int32_t)d.box) ? kv_page_number(a.c, g.x.seq, (uint32_t)p) : 0xFFFFFFFFu;
            };
            // `none`: boxes of a page that is none; keys there are NaN, so that the rows that look at them are taken again, which skips them
            auto load = [&](const CUtensorMap *map, uint32_t dst, uint32_t at, uint32_t mbar, uint32_t none) {
                for (uint32_t m = none; m; m &= m - 1)
                    for (uint32_t u = lane; u < d.box * 8 * C::PANELS; u += 32)
                        ct_sts(dst + u / (d.box * 8) * C::PANEL + (uint32_t)(__ffs(m) - 1) * d.box * 128 + u % (d.box * 8) * 16,
                               make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu));
                if (none) {
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                }
                if (lane == 0) t5::mbar_arrive_expect_tx(mbar, (boxes - __popc(none)) * d.box * HD * 2);
                __syncwarp();
                if (lane < boxes && !(none >> lane & 1))
                    for (uint32_t q = 0; q < (uint32_t)C::PANELS; q++)
                        t5::tma_2d(dst + q * C::PANEL + b * d.box * 128, map, (int32_t)(q * 64), (int32_t)at, mbar);
            };
            for (uint32_t k = 0; k < n_segs; k++) {
                const CtSegment &g = segs[k];
                uint32_t page = look(g, 0);
                for (uint32_t j = 0; j < g.n; j++) {
                    const uint32_t st = (g.T + j) % ST, ph = ((g.T + j) / ST) & 1;
                    const int32_t p = pos_of(g, j) + (int32_t)(b * d.box);
                    // past the last row of the pool: zeros
                    const bool some = wanted(g, p, (int32_t)d.box), there = some && kv_page_ok(a.c, page);
                    const uint32_t at = there ? (uint32_t)kv_row(a.c, page, g.kh, (uint32_t)p) : d.pool_rows, none = __ballot_sync(0xFFFFFFFFu, some && !there && lane < boxes);
                    page = look(g, j + 1);
                    t5::mbar_wait_warp(b_kempty + 8 * st, ph ^ 1, err_flag);
                    load(&kmap, base + C::K_OFF + st * C::TILE, at, b_kfull + 8 * st, none);
                    t5::mbar_wait_warp(b_vempty + 8 * st, ph ^ 1, err_flag);
                    load(&vmap, base + C::V_OFF + st * C::TILE, at, b_vfull + 8 * st, 0);
                }
            }
            // every copy in flight lands before the CTA leaves
            const uint32_t T = pre[CT_PAIRS + 2];
            for (uint32_t j = T > (uint32_t)ST ? T - ST : 0; j < T; j++) {
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
        // a bit for each unit of at_k: somebody looks at it, and it has a page or not (none: the scales of its keys are NaN, so that the rows that
        // look at it are taken again, which skips it)
        uint32_t some = 0, none = 0;
        // Pages are asked for two tiles ahead, so that nothing waits for the table.
        auto look = [&](const CtSegment &g, uint32_t j) {
            const int32_t p = j < g.n ? pos_of(g, j) + (int32_t)(lane & 7) * 16 : 0;
            return j < g.n && wanted(g, p, 16) ? kv_page_number(a.c, g.x.seq, (uint32_t)p) : 0xFFFFFFFFu;
        };
        auto units = [&](const CtSegment &g, uint32_t j, uint32_t page) {
            const int32_t p = j < g.n ? pos_of(g, j) + (int32_t)(lane & 7) * 16 : 0;
            const bool want = j < g.n && wanted(g, p, 16), ok = want && kv_page_ok(a.c, page);
            some = __ballot_sync(0xFFFFFFFFu, ok);
            none = __ballot_sync(0xFFFFFFFFu, want && !ok);
            return ok ? (uint32_t)kv_row(a.c, page, g.kh, (uint32_t)p) : 0u;
        };
        uint32_t page;
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
        // Where no row looks some row of the pool is read; its scale is 0, but a code of e4m3 may be NaN.
        auto clear = [&](const CtSegment &g, int32_t p0) {
            if (KIND == KV_E4M3 && (p0 + CT_POS > g.end || p0 < g.start)) {
#pragma unroll
                for (int i = 0; i < MINE; i++) {
                    const int32_t row = (int32_t)(row0 + i * STEP);
                    if (p0 + row >= g.x.len || !wanted(g, p0 + (row & ~15), 16)) reg[i] = make_uint4(0, 0, 0, 0);
                }
            }
        };
        constexpr int FULL = CT_POS / STEP;                        // pieces that every thread has
        auto load_scales = [&](int32_t p0, int32_t len, uint32_t of) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t row = ct + h * 96, at = __shfl_sync(0xFFFFFFFFu, of, (row >> 4) & 7);
                scr[0][h] = make_float2(none >> (row >> 4) & 1 ? __uint_as_float(0x7FC00000u) : 0.0f, 0.0f);
                scr[1][h] = make_float2(0.0f, 0.0f);
                if ((some >> (row >> 4) & 1) && row < CT_POS && p0 + (int32_t)row < len) {
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
        for (uint32_t k = 0; k < n_segs; k++) {
        CtSegment &g = segs[k];
        const uint32_t n = g.n, T = g.T;
        int32_t most_ex = -1000, least_ex = 1000;                  // of all tiles of the part so far
        if (n) {
            page = look(g, 0);
            at_k = units(g, 0, page);
            page = look(g, 1);
#pragma unroll
            for (int i = 0; i < MINE; i += G) load(a.c.k, i, at_k);
            load_scales(pos_of(g, 0), g.x.len, at_k);
        }
        for (uint32_t j = 0; j < n; j++) {
            const uint32_t st = (T + j) % ST, ph = ((T + j) / ST) & 1;
            const int32_t now = pos_of(g, j), next = j + 1 < n ? pos_of(g, j + 1) : g.x.len;  // nothing is loaded from the end on
            at_v = at_k;
            t5::mbar_wait_warp(b_kempty + 8 * st, ph ^ 1, err_flag);
            // the slot's last readers, the softmax of tile j - 4, came before the products that have just been waited for
            float *ksc = reinterpret_cast<float *>(smem + C::SC_OFF + ((T + j) % CT_SC) * C::SLOT), *vsc = ksc + CT_POS * NSC, *tops = vsc + CT_POS * NSC;
            float big = 0.0f, small = INFINITY;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t row = ct + h * 96;
                if (row < CT_POS) {
                    ksc[row] = scr[0][h].x;
                    if constexpr (NSC == 2) ksc[CT_POS + row] = scr[0][h].y;
                }
                // no value is larger; scales that are not finite count for nothing, their values stay what they are
                const float most = KIND == KV_INT4 ? fmaf(8.0f, fabsf(scr[1][h].x), fabsf(scr[1][h].y)) : fabsf(scr[1][h].x) * (KIND == KV_INT8 ? 128.0f : 448.0f);
                if (most < INFINITY) big = fmaxf(big, most);
                if (most > 0.0f) small = fminf(small, most);
            }
            // as whole numbers, which non-negative ones are ordered like
            big = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(big)));
            small = __uint_as_float(__reduce_min_sync(0xFFFFFFFFu, __float_as_uint(small)));
            if (lane == 0) {
                tops[cw] = big;
                tops[4 + cw] = small;
            }
            if (ct == 0) {                                         // four of each are read
                tops[3] = 0.0f;
                tops[7] = INFINITY;
            }
            asm volatile("bar.sync 9, 96;\n" ::: "memory");        // those of all three warps
            const float unit = ct_pow2(13 - ct_exponent(tops));
            most_ex = max(most_ex, ct_exponent(tops));
            least_ex = min(least_ex, ct_least_exponent(tops + 4));
            if (ct == 0 && most_ex - least_ex > CT_APART) g.wide = 1;
            t5::mbar_arrive(b_sc + 8 * ((T + j) % CT_SC));
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t row = ct + h * 96;
                const float2 sc = ct_scale<KIND>(scr[1][h], unit);
                if (row < CT_POS) {
                    if constexpr (NSC == 2) reinterpret_cast<float2 *>(vsc)[row] = sc;
                    else vsc[row] = sc.x;
                }
            }
            at_k = units(g, j + 1, page);
            page = look(g, j + 2);
            load_scales(next, g.x.len, at_k);
            const uint32_t kt = base + C::K_OFF + st * C::TILE, vt = base + C::V_OFF + st * C::TILE;
            clear(g, now);
#pragma unroll
            for (int f = 0; f < MINE; f += G) {
#pragma unroll
                for (int i = f; i < f + G && i < MINE; i++)
                    if (i < FULL || row0 + i * STEP < CT_POS) ct_convert<KIND, false>(kt + i * STEP * 128, STEP % 8 ? (i & 1) << 6 : 0, to, swap, reg[i], make_float2(1.0f, 0.0f));
                load(a.c.v, f, at_v);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            t5::mbar_arrive(b_kfull + 8 * st);
            asm volatile("bar.sync 9, 96;\n" ::: "memory");        // the scales of all three warps
            t5::mbar_wait_warp(b_vempty + 8 * st, ph ^ 1, err_flag);
            const uint32_t v_at = base + C::SC_OFF + ((T + j) % CT_SC) * C::SLOT + (CT_POS + row0) * NSC * 4;
            clear(g, now);
#pragma unroll
            for (int f = 0; f < MINE; f += G) {
                float2 sc[G];
#pragma unroll
                for (int i = 0; i < G; i++) {
                    sc[i] = make_float2(0.0f, 0.0f);
                    if (f + i < MINE && (f + i < FULL || row0 + (f + i) * STEP < CT_POS)) {
                        if constexpr (NSC == 2) sc[i] = ct_lds2(v_at + (f + i) * STEP * NSC * 4);
                        else sc[i].x = ct_lds(v_at + (f + i) * STEP * NSC * 4);
                    }
                }
#pragma unroll
                for (int i = f; i < f + G && i < MINE; i++)
                    if (i < FULL || row0 + i * STEP < CT_POS) ct_convert<KIND, true>(vt + i * STEP * 128, STEP % 8 ? (i & 1) << 6 : 0, to, swap, reg[i], sc[i - f]);
                load(a.c.k, f, at_k);
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            t5::mbar_arrive(b_vfull + 8 * st);
        }
        }
    }
    __syncthreads();
    t5::fence_after();
    if (warp == C::ISSUER) t5::tmem_dealloc(tmem, 512);
    if (tid == 0 && *err_flag) atomicExch(a.c.err, 5u);
    // Rows whose result is not finite, a warp each.  Not before: one may take as long as all else, and the waits above have a limit.
    for (uint32_t k = 0, turn = 0; k < pre[CT_PAIRS + 1]; k++) {
        const CtSegment &g = segs[k];
        for (uint32_t w = 0; w < CT_ROWS / 32; w++)
            for (uint32_t rows = g.again[w]; rows; rows &= rows - 1)
                if (turn++ % (C::THREADS / 32) == warp) {
                    const uint32_t i = g.r0 + w * 32 + (uint32_t)(__ffs(rows) - 1);
                    cache_plain_row<KIND, HD>(a, g.x, i / a.group, g.kh * a.group + i % a.group, lane);
                }
    }
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
    // Few row tiles: each cut into the same number of parts.  From half as many as SMs on: the blocks share the work, whatever the lengths
    // (a row tile has two or three parts then, and the last block joins them).  More than a block can list: a block a row tile.
    const uint64_t pairs = (uint64_t)a.n_entries * d.tiles, items = pairs * a.c.kv_heads;
    uint64_t seen = max_length;
    if (a.window) seen = std::min<uint64_t>(seen, (uint64_t)a.window + a.sinks + 2 * CT_POS + CT_ROWS / a.group);
    const uint64_t most = std::max<uint64_t>(1, (seen + CT_POS - 1) / CT_POS);
    const bool share = items * 2 > (uint64_t)ctx->sm_count && pairs <= CT_PAIRS && items <= (uint64_t)ctx->sm_count * CT_ITEMS;
    d.splits = share ? 0 : (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, ctx->sm_count / items));
    const uint64_t blocks = share ? (uint64_t)ctx->sm_count : items * d.splits;
    if (blocks > 0x7FFFFFFFull) return fail(ctx, PRISM_E_ARG, "cache_attention: too many rows");
    const uint64_t rows = ((uint64_t)a.c.n_pages * a.c.kv_heads) << a.c.shift;
    d.box = std::min<uint32_t>(CT_POS, 1u << a.c.shift);
    d.pool_rows = (uint32_t)rows;
    CUtensorMap k{}, v{};
    if constexpr (KIND <= KV_BF16) {
        PRISM_TRY(encode_tensor_map(ctx, &k, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.c.k, HD, rows, HD, 64, d.box, CU_TENSOR_MAP_SWIZZLE_128B));
        PRISM_TRY(encode_tensor_map(ctx, &v, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.c.v, HD, rows, HD, 64, d.box, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    if (d.splits != 1)
        PRISM_TRY(cache_scratch(ctx, (size_t)(share ? 2 * blocks : blocks) * cache_part_floats(CT_ROWS, HD) * 4, share ? (size_t)items : 0, &d.part, &d.count));
    launch_pdl(ctx, "cache_tiles_kernel", cache_tiles_kernel<KIND, HD>, dim3((uint32_t)blocks), dim3(C::THREADS), C::SMEM, d, k, v);
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
