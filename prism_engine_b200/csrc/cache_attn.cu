// Attention of the newest tokens of some sequences over a caller-owned cache (prism_cuda_cache_attention_dev): the kernel for few
// query rows per cached head.
//
// A block takes 8 or 16 query rows that share a cached head (the heads of its group, of one token or several) and a part of the
// positions that any of them sees; its four warps take tiles of 16 or 32 positions in turn, each with its own ring of stages
// (cp.async), running maximum and sums, so no warp waits for another before the end.  Products are mma.sync with positions, then columns,
// as M and eight query rows as N: S^T = K q^T, O^T += V^T P^T.  Codes go from shared memory to fragments in registers, with no
// 16-bit copy in between: a lane's fragments of K are consecutive codes of a row (the order of a contraction is free, so q's
// fragments follow it), those of V are the same columns of four rows, their bytes interleaved.  Codes are exact in fp16, so scales
// stay out of the products:
//   score = (q c) ks + (sum of q) kz,     o = sum of (w vs) c + sum of w vz.
// w vs enters the product as fp16 over the power of two below the row's largest so far, 2^14-fold, so no scale over- or underflows;
// with 16-bit rows w itself does (fp16: 2^13-fold, bf16: as it is), and the sum that divides is that of the rounded weights.  q of 8- and 4-bit caches enters
// as fp16 over a power of two.  Maxima, sums, O and everything that multiplies them are 32 bits.  The 16 bits are what the products
// take: a weight is rounded once (2^-8 of itself in bf16, 2^-11 in fp16), as the result is, and q over a power of two keeps its bits but for elements
// 2^-14 of its largest.
//
// Positions past the end are zero.  A position that some row of the block does not see meets weight 0, which an infinity there turns into
// NaN: a row whose result is not finite is taken again by itself (cache_plain_row).
//
// Where there are few row tiles the positions are cut into S parts.  Up to eight are the blocks of a cluster, each of which joins some rows out of
// the shared memory of all (through scratch and a counter: 14 heads of 64 over 711 positions 9.0 us, by clusters 5.5); more go through scratch to cache_join_kernel.
// Bound: HBM for long caches of 16-bit rows; the instructions about codes (some 850 a warp for 32 positions of a 128-wide head: places, copies, bytes to
// fragments, scales, softmax) at 8 and 4 bits; the latency of the chain (places, tiles, joining) for short ones.
// 64 heads of 128 over 8, a token of 32 sequences under a window of 4096: 16 bits 85 us (6.3 TB/s), int8 63 us (4.4 TB/s), int4 65 us; one sequence of 131071
// positions: 16 bits 91 us (5.9 TB/s), int4 56 us (2.7 TB/s); 14 heads of 64 over 2, 516 visible positions: 5.5 us.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <memory>
#include <stdexcept>
#include <vector>

#include "cache_join.cuh"

namespace prism {

constexpr int CR_W = 4, CR_THREADS = CR_W * 32;  // warps of a block
constexpr uint32_t CR_CLUSTER = 8;               // parts whose blocks are a cluster
constexpr uint32_t CR_NEAR = 512;                // positions of a part
// More than 32 rows of a cached head are for the tcgen05 kernel, whose blocks cost 6 us more to begin and to end, where 16-row tiles are more than
// two an SM or tiles times positions more than this.  8 cached heads of 128, 64 to 256 rows (int8): one sequence of 2000 positions 12 to 25 us here,
// 20 to 26 there; eight of 711 20 to 76 here, 27 to 35 there; eight of 8000 127 to 479 here, 134 to 151 there.  To 32 rows this one always:
// eight of 8000 positions, 32 rows: int8 71 us here, 128 there, 16 bits 68 and 75.
constexpr uint64_t CR_WORK = 200000;
constexpr float CR_UP = 16384.0f;                // weights of fp16 products of codes are 2^14-fold, and below 2; of fp16 rows 2^13-fold, and below 2^CR_GROW
constexpr float CR_GROW = 2.0f;                  // powers of two that a score may lie above the maximum in use
template <int KIND, int HD, int NQ>              // NQ: groups of eight query rows
struct CrCfg {
    static constexpr int ROWB = HD * (int)kv_bits<KIND>() / 8, R = 8 * NQ;
    static constexpr int TP = ROWB >= 256 ? 16 : 32, MT = TP / 16;   // positions of a tile
    static constexpr int NSC = (int)kv_scales<KIND>();
    static constexpr int TILE = TP * ROWB, SCB = TP * NSC * 4;       // bytes of a tile's keys (or values), of their scales
    static constexpr int STAGE = 2 * TILE + 2 * SCB;
    static constexpr int ST = ROWB >= 64 ? 2 : 3;
    static constexpr int KS = HD / 16, CPL = HD / 8, OT = HD / 16;   // contraction steps of a score; columns of a lane; tiles of O
    static constexpr bool Q_REGS = KS * NQ <= 16;
    static constexpr int PITCH = HD + 4;                             // floats of a row of the joined sums
    static constexpr int RING = CR_W * ST * STAGE, ACC_OFF = CR_W * R * HD * 4, PARTS = ACC_OFF + R * PITCH * 4;
    static constexpr int BODY = RING > PARTS ? RING : PARTS;         // also the warps' parts of O and their sum
    static constexpr int Q_OFF = BODY, FRAG_OFF = Q_OFF + R * HD * 2;  // q rows, then as fragments
    static constexpr int ROW_OFF = FRAG_OFF + R * HD * 2;            // CrRow of each row, then maxima and sums: the warps', the row's; flags
    static constexpr size_t SMEM = ROW_OFF + R * 32 + CR_W * R * 8 + R * 8 + 16;
    static constexpr int BLOCKS = HD <= 128 && NQ == 1 ? 3 : 2;      // of an SM, for the registers
};
struct CrRow {
    const uint64_t *mask;
    int32_t last, low;
    float mul, qsum;   // of the scores (in powers of two); the sum of q's fragments
    uint32_t there;
};
static_assert(sizeof(CrRow) == 32, "rows of 32 bytes");

struct CrDev {
    CacheAttnDev a;
    uint32_t splits, tiles;  // parts of the positions, row tiles of an entry and head
    float *part;             // of the blocks (CacheJoinDev)
};

namespace {

// Byte of a 16-byte piece c of tile row r: neighbouring rows' pieces are exchanged so that the lanes that read together (K: four
// neighbouring pieces of rows 2i and 2i + 1; V: the same columns of rows 0, 2, 4, 6 apart) lie in different banks.  Eight rows on it is
// 8 * ROWB bytes on, and piece c ^ k lies at the place of c with k << 4 exchanged.
template <int ROWB>
__host__ __device__ constexpr uint32_t cr_at(uint32_t r, uint32_t c) {
    if constexpr (ROWB == 512) return r * 512 + ((c ^ (((r >> 1) & 3) ^ ((r & 1) << 2))) << 4);
    else if constexpr (ROWB == 256) return r * 256 + ((c ^ ((((r >> 1) & 1) | ((r >> 2) & 1) << 2) ^ ((r & 1) << 2))) << 4);
    else if constexpr (ROWB == 128) return r * 128 + ((c ^ (((r >> 1) & 3) << 1 ^ ((r & 1) << 2))) << 4);
    else if constexpr (ROWB == 64) return (r >> 1) * 128 + ((r ^ (r >> 1)) & 1) * 64 + ((c ^ (((r >> 2) & 1) << 1)) << 4);
    else if constexpr (ROWB == 32) return ((r >> 3) * 2 + (r & 1)) * 128 + ((((r >> 1) & 3) ^ ((r & 1) << 1)) << 5) + (c << 4);
    else return r * 16;
}
// Place of slot j (of 4) of step ks in a head, for lane t of four: what the fragments of a row's codes hold.
template <int KIND, int HD>
__device__ __forceinline__ uint32_t cr_elem(uint32_t ks, uint32_t t, uint32_t j) {
    constexpr uint32_t LB = HD * kv_bits<KIND>() / 32;  // a lane's bytes of a row
    const uint32_t word = KIND <= KV_BF16 ? 2 * ks : KIND == KV_INT4 ? ks >> 1 : ks;
    const uint32_t byte = LB >= 16 ? (t + 4 * (word >> 2)) * 16 + (word & 3) * 4 : t * LB + word * 4;
    if (KIND <= KV_BF16) return byte / 2 + j;
    if (KIND == KV_INT4) return byte * 2 + ((ks & 1) << 1) + (j >> 1) + ((j & 1) << 2);
    return byte + j;
}

__device__ __forceinline__ float cr_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16>
__device__ __forceinline__ void cr_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Bytes copied, the rest of the 16 zero.
__device__ __forceinline__ void cr_cp16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// N words of shared memory (plain loads: the compiler takes them early).
template <int N>
__device__ __forceinline__ void cr_lds(uint32_t (&w)[N], const uint8_t *p) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x;
        w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}
__device__ __forceinline__ uint32_t cr_sub2(uint32_t h, uint32_t what) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&h), *reinterpret_cast<const __half2 *>(&what));
    return *reinterpret_cast<const uint32_t *>(&d);
}
// Four 8-bit codes as two fp16 pairs.
template <int KIND>
__device__ __forceinline__ void cr_bytes(uint32_t w, uint32_t &h0, uint32_t &h1) {
    if constexpr (KIND == KV_INT8) {
        const uint32_t x = w ^ 0x80808080u;  // code + 128 in the low bits of 1024
        h0 = cr_sub2(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u);
        h1 = cr_sub2(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n" : "=r"(h0), "=r"(h1) : "r"(w));
    }
}
// Codes 0..7 of a word as fp16 pairs (0, 4), (1, 5), (2, 6), (3, 7), less 8.
__device__ __forceinline__ void cr_nibbles(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t sixteenth = 0x2C002C00u, off = 0xD480D480u;  // 1 / 16, -(64 + 8)
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t x = w >> (8 * i);
        h[2 * i] = cr_sub2((x & 0x000F000Fu) | 0x64006400u, 0x64086408u);
        const uint32_t y = (x & 0x00F000F0u) | 0x64006400u;
        const __half2 d = __hfma2(*reinterpret_cast<const __half2 *>(&y), *reinterpret_cast<const __half2 *>(&sixteenth), *reinterpret_cast<const __half2 *>(&off));
        h[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&d);
    }
}
__device__ __forceinline__ float cr_pow2_below(float x) { return __uint_as_float(min(__float_as_uint(x) & 0x7F800000u, 253u << 23)); }
__device__ __forceinline__ float cr_inv_pow2(float p) { return p > 0.0f ? __uint_as_float((254u << 23) - __float_as_uint(p)) : 0.0f; }

}  // namespace

__device__ __forceinline__ void cr_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// From the same place of another block of the cluster.
__device__ __forceinline__ float cr_lds_of(uint32_t at, uint32_t block) {
    float v;
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %1, %2;\nld.shared::cluster.f32 %0, [r];\n}\n" : "=f"(v) : "r"(at), "r"(block) : "memory");
    return v;
}
__device__ __forceinline__ float4 cr_lds4_of(uint32_t at, uint32_t block) {
    float4 v;
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %4, %5;\nld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n}\n"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at), "r"(block)
                 : "memory");
    return v;
}

template <int KIND, int HD, int NQ>
__global__ void __launch_bounds__(CR_THREADS, CrCfg<KIND, HD, NQ>::BLOCKS) cache_rows_kernel(const __grid_constant__ CrDev d) {
    using C = CrCfg<KIND, HD, NQ>;
    constexpr int TP = C::TP, MT = C::MT, KS = C::KS, CPL = C::CPL, OT = C::OT, ROWB = C::ROWB, NSC = C::NSC, ST = C::ST, R = C::R, PITCH = C::PITCH;
    constexpr bool CODES = KIND >= KV_INT8, BF16 = KIND == KV_BF16;
    const CacheAttnDev &a = d.a;
    extern __shared__ __align__(128) uint8_t cr_smem[];
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t item = blockIdx.x / d.splits, split = blockIdx.x - item * d.splits;
    const uint32_t tile = item % d.tiles, kh = item / d.tiles % a.c.kv_heads, e = item / d.tiles / a.c.kv_heads;
    CacheEntry x;
    if (!cache_entry(a, e, x)) return;                     // the same in all blocks of an item
    const uint32_t n_rows = x.n * a.group, r0 = tile * R;
    if (r0 >= n_rows) return;
    const uint32_t here = min((uint32_t)R, n_rows - r0), tok_lo = r0 / a.group, tok_hi = (r0 + here - 1) / a.group;

    CrRow *rows = reinterpret_cast<CrRow *>(cr_smem + C::ROW_OFF);
    float *w_max = reinterpret_cast<float *>(cr_smem + C::ROW_OFF + R * 32), *w_sum = w_max + CR_W * R, *r_max = w_sum + CR_W * R, *r_sum = r_max + R;
    uint32_t *flags = reinterpret_cast<uint32_t *>(r_sum + R);  // rows to be taken again
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(cr_smem) + warp * ST * C::STAGE;

    // ---- the positions that some row sees: the first tiles (a.sinks), then main_lo .. ---------------------------------
    int32_t low = x.len, low_max = -1;
    if (!a.window) low = -1;
    else if (!a.tree) {
        low = cache_row(a, x, tok_lo).low;
        low_max = cache_row(a, x, tok_hi).low;
    } else {
        for (uint32_t i = tok_lo; i <= tok_hi; i++) {
            const int32_t l = cache_row(a, x, i).low;
            low = min(low, l);
            low_max = max(low_max, l);
        }
    }
    const int32_t end = a.tree ? x.len : min(x.len, x.first + (int32_t)tok_hi + 1);  // may be negative: nothing is seen
    const int32_t all_to = a.tree ? x.first - 1 : x.first + (int32_t)tok_lo;         // every row's last
    const int32_t start = a.tree ? min(low + 1, max(x.first, 0)) : low + 1;
    const uint32_t first_tiles = end > 0 ? (min((uint32_t)end, a.sinks) + TP - 1) / TP : 0;
    const uint32_t main_lo = max((uint32_t)start / TP, first_tiles), main_hi = end > 0 ? ((uint32_t)end + TP - 1) / TP : 0;
    const uint32_t n_tiles = first_tiles + (main_hi > main_lo ? main_hi - main_lo : 0);
    const uint32_t i_lo = (uint32_t)((uint64_t)n_tiles * split / d.splits), i_hi = (uint32_t)((uint64_t)n_tiles * (split + 1) / d.splits);
    auto pos_of = [&](uint32_t i) { return (int32_t)((i < first_tiles ? i : main_lo + (i - first_tiles)) * TP); };

    // Pages are asked for a tile before its rows, so that no warp waits for the table; pages[u] of 16 positions, the table's own number.  Only
    // where some row of the block sees one of them (bit u of `wanted`): others may be gone.
    uint32_t pages[TP / 16] = {}, wanted = 0;
    auto look = [&](uint32_t i) {
#pragma unroll
        for (int u = 0; u < TP / 16; u++) {
            const int32_t p = pos_of(i) + u * 16;
            const bool some = i < i_hi && p < end && (p + 15 >= start || (uint32_t)p < a.sinks);
            if (some) pages[u] = kv_page_number(a.c, x.seq, (uint32_t)p);
            wanted = (wanted & ~(1u << u)) | (uint32_t)some << u;
        }
    };
    const uint32_t f_at = cr_at<ROWB>(lane / (ROWB / 16), lane % (ROWB / 16));  // of the lane's first piece
    uint32_t skip = 0;                                     // two bits a stage: 16 positions whose page is none, nobody's from here on
    auto fetch = [&](uint32_t i, uint32_t st) {
        if (i < i_hi) {
            const uint32_t kt = ring + st * C::STAGE, vt = kt + C::TILE, ksc = vt + C::TILE, vsc = ksc + C::SCB;
            const int32_t p0 = pos_of(i);
#pragma unroll
            for (int u = 0; u < TP / 16; u++) {            // a page holds at least 16 positions
                const int32_t p = p0 + u * 16;
                int32_t left = wanted >> u & 1 ? x.len - p : 0;
                if (left && !kv_page_ok(a.c, pages[u])) {
                    left = 0;
                    skip |= 1u << (st * 2 + u);
                }
                const size_t row = left ? kv_row(a.c, pages[u], kh, (uint32_t)p) : 0;
                const uint8_t *ks = a.c.k + row * ROWB + lane * 16, *vs = a.c.v + row * ROWB + lane * 16;
                const bool all = left >= 16;
#pragma unroll
                for (int m = 0; m < (ROWB + 31) / 32; m++) {
                    constexpr uint32_t RP = ROWB / 16;
                    const uint32_t at = (f_at ^ (cr_at<ROWB>(m * 32 / RP, 0) - m * 512)) + u * 16 * ROWB + m * 512;
                    if (ROWB >= 32 || lane < (uint32_t)ROWB) {
                        const uint32_t bytes = all || (int32_t)((m * 32 + lane) / RP) < left ? 16 : 0;
                        cr_cp16(kt + at, ks + m * 512, bytes);
                        cr_cp16(vt + at, vs + m * 512, bytes);
                    }
                }
                if constexpr (NSC > 0) {
                    constexpr uint32_t PER = 4 * NSC;      // pieces of 16 positions' scales
                    if (lane < 2 * PER) {
                        const uint32_t which = lane / PER, piece = lane % PER, mine = piece * (4 / NSC);  // first position of the piece
                        const uint32_t bytes = (uint32_t)max(0, min(16, (left - (int32_t)mine) * 4 * NSC));
                        cr_cp16((which ? vsc : ksc) + u * 64 * NSC + piece * 16, (which ? a.c.vs : a.c.ks) + row * NSC + piece * 4, bytes);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    look(i_lo + warp);
#pragma unroll
    for (int s = 0; s < ST - 1; s++) {
        fetch(i_lo + warp + s * CR_W, s);
        look(i_lo + warp + (s + 1) * CR_W);
    }

    // ---- rows and q's fragments -----------------------------------------------------------------------------------------
    {
        constexpr int TR = CR_THREADS / R, PER = HD / TR;  // threads of a row, values of a thread
        const uint32_t r = tid / TR, part = tid % TR, token = (r0 + r) / a.group;
        const bool there = r < here;
        uint32_t w[PER / 2];
#pragma unroll
        for (int i = 0; i < PER / 2; i++) w[i] = 0;
        if (there) {
            const uint16_t *src = a.q + (size_t)(x.row0 + token) * a.q_stride + (size_t)(kh * a.group + (r0 + r) % a.group) * HD + part * PER;
            if constexpr (PER >= 8) {
#pragma unroll
                for (int i = 0; i < PER / 8; i++) reinterpret_cast<uint4 *>(w)[i] = reinterpret_cast<const uint4 *>(src)[i];
            } else if constexpr (PER == 4) {
                *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(src);
            } else {
                w[0] = *reinterpret_cast<const uint32_t *>(src);
            }
        }
        float mul = fabsf(a.scale) * 1.4426950408889634f, sum = 0.0f;
        if (a.scale < 0.0f) {                              // the sign of the scale is q's
#pragma unroll
            for (int i = 0; i < PER / 2; i++) w[i] ^= 0x80008000u;
        }
        if constexpr (CODES) {
            float v[PER], big = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                v[i] = kv_row_value((uint16_t)(w[i >> 1] >> (16 * (i & 1))), a.c.rows_bf16);
                big = fmaxf(big, fabsf(v[i]));
            }
#pragma unroll
            for (int o = TR / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
            const float unit = cr_pow2_below(big), inv = unit > 0.0f ? cr_inv_pow2(unit) : 1.0f;
            if (unit > 0.0f) mul *= unit;
#pragma unroll
            for (int i = 0; i < PER / 2; i++) {
                const __half2 h = __floats2half2_rn(v[2 * i] * inv, v[2 * i + 1] * inv);
                const float2 f = __half22float2(h);
                sum += f.x + f.y;
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
#pragma unroll
            for (int o = TR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        }
        uint32_t *dst = reinterpret_cast<uint32_t *>(cr_smem + C::Q_OFF) + (r * HD + part * PER) / 2;
#pragma unroll
        for (int i = 0; i < PER / 2; i++) dst[i] = w[i];
        if (part == 0) {
            CrRow y{nullptr, -1, -1, mul, sum, there};
            if (there) {
                const CacheRow c = cache_row(a, x, token);
                y.mask = c.mask;
                y.last = c.last;
                y.low = c.low;
            }
            rows[r] = y;
        }
        if (tid == 0) flags[0] = 0;
    }
    __syncthreads();
    {
        const uint16_t *q = reinterpret_cast<const uint16_t *>(cr_smem + C::Q_OFF);
        uint2 *frag = reinterpret_cast<uint2 *>(cr_smem + C::FRAG_OFF);
        for (uint32_t s = tid; s < NQ * KS * 32; s += CR_THREADS) {
            const uint32_t ks = (s >> 5) % KS, ln = s & 31, fr = (s >> 5) / KS * 8 + (ln >> 2), ft = ln & 3;
            auto pair = [&](int j) {
                return (uint32_t)q[fr * HD + cr_elem<KIND, HD>(ks, ft, j)] | (uint32_t)q[fr * HD + cr_elem<KIND, HD>(ks, ft, j + 1)] << 16;
            };
            frag[s] = make_uint2(pair(0), pair(2));
        }
    }
    __syncthreads();
    const uint8_t *frag_at = cr_smem + C::FRAG_OFF + lane * 8;
    uint32_t qf[C::Q_REGS ? NQ * KS : 1][2];
    if constexpr (C::Q_REGS) {
#pragma unroll
        for (int k = 0; k < NQ * KS; k++) cr_lds<2>(qf[k], frag_at + k * 256);
    }
    float mul[NQ][2], qsum[NQ][2];                         // of the lane's rows 2t and 2t + 1
#pragma unroll
    for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            mul[n][h] = rows[n * 8 + 2 * t + h].mul;
            qsum[n][h] = rows[n * 8 + 2 * t + h].qsum;
        }

    // ---- this warp's tiles ------------------------------------------------------------------------------------------------
    float o[NQ][OT][4], m[NQ][2], l[NQ][2], z[NQ][2], unit[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            m[n][h] = -INFINITY;
            l[n][h] = z[n][h] = 0.0f;
            unit[n][h] = 0x1p-100f;
        }
#pragma unroll
        for (int i = 0; i < OT; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[n][i][c] = 0.0f;
    }
    constexpr int LB = ROWB / 4, CB = ROWB / 8;            // a lane's bytes of a row of keys, of a row of values
    const uint32_t k_at = LB >= 16 ? cr_at<ROWB>(g, t) : LB == 8 ? cr_at<ROWB>(g, t >> 1) + (t & 1) * 8 : cr_at<ROWB>(g, 0) + t * 4;
    uint32_t v_at[2];                                      // of rows 2t and 2t + 1
#pragma unroll
    for (int h = 0; h < 2; h++)
        v_at[h] = C::TILE + (CB >= 16 ? cr_at<ROWB>(2 * t + h, g * (CB / 16)) : CB == 8 ? cr_at<ROWB>(2 * t + h, g >> 1) + (g & 1) * 8
                                        : CB == 4 ? cr_at<ROWB>(2 * t + h, g >> 2) + (g & 3) * 4 : cr_at<ROWB>(2 * t + h, 0) + g * 2);
    const uint32_t sc_at = 2 * C::TILE + g * 4 * NSC;
    uint32_t st = 0;
    for (uint32_t i = i_lo + warp; i < i_hi; i += CR_W) {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(ST - 2) : "memory");
        __syncwarp();                                      // and the whole warp is done with the tile before
        fetch(i + (ST - 1) * CR_W, st == 0 ? ST - 1 : st - 1);
        look(i + ST * CR_W);
        const uint8_t *stage = cr_smem + (warp * ST + st) * C::STAGE;
        const int32_t p0 = pos_of(i);
        // scores: rows g and g + 8 of 16 positions, query rows 2t and 2t + 1
        float s[MT][NQ][4];
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[j][n][c] = 0.0f;
        auto step = [&](int j, int k, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
            const uint32_t ka[4] = {a0, a1, a2, a3};
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                if constexpr (C::Q_REGS) {
                    cr_mma<BF16>(s[j][n], ka, qf[n * KS + k][0], qf[n * KS + k][1]);
                } else {
                    uint32_t q2[2];
                    cr_lds<2>(q2, frag_at + (n * KS + k) * 256);
                    cr_mma<BF16>(s[j][n], ka, q2[0], q2[1]);
                }
            }
        };
        constexpr int KW = LB >= 16 ? 4 : LB / 4;          // words of an access
#pragma unroll
        for (int pc = 0; pc < (LB + 15) / 16; pc++) {
            uint32_t w[MT][2][KW];                         // of rows g and g + 8 of each 16 positions
#pragma unroll
            for (int j = 0; j < MT; j++)
#pragma unroll
                for (int h = 0; h < 2; h++) cr_lds<KW>(w[j][h], stage + (k_at ^ (pc * 64)) + (j * 16 + 8 * h) * ROWB);
#pragma unroll
            for (int q = 0; q < KW; q++)
#pragma unroll
                for (int j = 0; j < MT; j++) {
                    if constexpr (KIND <= KV_BF16) {
                        if (q % 2 == 0) step(j, pc * 2 + q / 2, w[j][0][q], w[j][1][q], w[j][0][q + 1], w[j][1][q + 1]);
                    } else if constexpr (KIND == KV_INT4) {
                        uint32_t h0[4], h1[4];
                        cr_nibbles(w[j][0][q], h0);
                        cr_nibbles(w[j][1][q], h1);
                        step(j, (pc * 4 + q) * 2, h0[0], h1[0], h0[1], h1[1]);
                        step(j, (pc * 4 + q) * 2 + 1, h0[2], h1[2], h0[3], h1[3]);
                    } else {
                        uint32_t h0[2], h1[2];
                        cr_bytes<KIND>(w[j][0][q], h0[0], h0[1]);
                        cr_bytes<KIND>(w[j][1][q], h1[0], h1[1]);
                        step(j, pc * 4 + q, h0[0], h1[0], h0[1], h1[1]);
                    }
                }
        }
        float vs[MT][2], vz[MT][2];                        // of the lane's positions
#pragma unroll
        for (int j = 0; j < MT; j++) {
            float ks[2], kz[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t *at = stage + sc_at + (j * 16 + 8 * h) * 4 * NSC;
                if constexpr (NSC == 2) {
                    uint32_t w[2];
                    cr_lds<2>(w, at);
                    ks[h] = __uint_as_float(w[0]);
                    kz[h] = __uint_as_float(w[1]);
                    cr_lds<2>(w, at + C::SCB);
                    vs[j][h] = __uint_as_float(w[0]);
                    vz[j][h] = __uint_as_float(w[1]);
                } else if constexpr (NSC == 1) {
                    uint32_t w[1];
                    cr_lds<1>(w, at);
                    ks[h] = __uint_as_float(w[0]);
                    cr_lds<1>(w, at + C::SCB);
                    vs[j][h] = __uint_as_float(w[0]);
                }
            }
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    if constexpr (NSC == 2) s[j][n][c] = fmaf(s[j][n][c], ks[c >> 1], qsum[n][c & 1] * kz[c >> 1]);
                    else if constexpr (NSC == 1) s[j][n][c] *= ks[c >> 1];
                }
        }
        const bool whole = p0 + TP - 1 <= all_to && (p0 > low_max || (uint32_t)(p0 + TP) <= a.sinks);
        const uint32_t gone = skip >> (st * 2) & 3;
        if (!whole || gone) {
            skip &= ~(3u << (st * 2));
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const CrRow r = rows[n * 8 + 2 * t + h];
#pragma unroll
                    for (int j = 0; j < MT; j++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int32_t p = p0 + j * 16 + g + 8 * c;
                            bool see = p <= r.last && (p > r.low || (uint32_t)p < a.sinks);
                            if (a.tree && p >= x.first) {
                                see = r.mask && p < x.len;
                                if (see) see = __ldg(r.mask + ((uint32_t)(p - x.first) >> 6)) >> ((p - x.first) & 63) & 1;
                            }
                            if (!see || (gone >> j & 1)) s[j][n][2 * c + h] = -INFINITY;
                        }
                }
        }
        // weights
        uint32_t pf[MT][NQ][2];                            // P^T: positions 2t, 2t + 1 (and 8 on) of row g
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            // The maximum is moved only when some score of the tile lies above it by more than CR_GROW: else no lane asks the others.
            float top[2], alpha[2] = {1.0f, 1.0f};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                top[h] = fmaxf(s[0][n][h], s[0][n][2 + h]);
                if constexpr (MT == 2) top[h] = fmaxf(top[h], fmaxf(s[1][n][h], s[1][n][2 + h]));
                top[h] = top[h] == -INFINITY ? top[h] : top[h] * mul[n][h];  // mul may be 0
            }
            if (__any_sync(0xFFFFFFFFu, top[0] > m[n][0] + CR_GROW || top[1] > m[n][1] + CR_GROW)) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int q = 4; q < 32; q <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], q));
                    top[h] = fmaxf(top[h], m[n][h]);
                    alpha[h] = top[h] == -INFINITY ? 1.0f : cr_ex2(m[n][h] - top[h]);
                    m[n][h] = top[h];
                    l[n][h] *= alpha[h];
                    if constexpr (NSC == 2) z[n][h] *= alpha[h];
                }
            }
            float big[2] = {0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float sub = (m[n][h] == -INFINITY ? 0.0f : m[n][h]) - (KIND == KV_F16 ? 13.0f : 0.0f);  // nothing but -inf so far: weights 0
#pragma unroll
                for (int j = 0; j < MT; j++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float &w = s[j][n][2 * c + h];
                        w = cr_ex2(fmaf(w, mul[n][h], -sub));
                        if constexpr (CODES) {
                            l[n][h] += w;
                            if constexpr (NSC == 2) z[n][h] = fmaf(w, vz[j][c], z[n][h]);
                            w *= vs[j][c];
                            big[h] = fmaxf(big[h], fabsf(w));
                        }
                    }
            }
            if constexpr (CODES) {
                // What O is over: moved down with the weights so far, up when a product is twice as large.
                if (__any_sync(0xFFFFFFFFu, alpha[0] != 1.0f || alpha[1] != 1.0f || big[0] >= 2.0f * unit[n][0] || big[1] >= 2.0f * unit[n][1])) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
#pragma unroll
                        for (int q = 4; q < 32; q <<= 1) big[h] = fmaxf(big[h], __shfl_xor_sync(0xFFFFFFFFu, big[h], q));
                        float u = alpha[h] == 1.0f ? unit[n][h] : fmaxf(cr_pow2_below(unit[n][h] * alpha[h]), 0x1p-100f);
                        if (big[h] >= 2.0f * u) u = cr_pow2_below(big[h]);
                        alpha[h] = alpha[h] * unit[n][h] * cr_inv_pow2(u);
                        unit[n][h] = u;
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float inv = cr_inv_pow2(unit[n][h]) * CR_UP;
#pragma unroll
                    for (int j = 0; j < MT; j++) {
                        s[j][n][h] *= inv;
                        s[j][n][2 + h] *= inv;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < MT; j++)
#pragma unroll
                for (int h = 0; h < 2; h++) {              // positions g, g + 8
                    uint32_t p;
                    if constexpr (BF16) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(s[j][n][2 * h], s[j][n][2 * h + 1]);
                        p = *reinterpret_cast<const uint32_t *>(&b);
                        l[n][0] += __uint_as_float(p << 16);
                        l[n][1] += __uint_as_float(p & 0xFFFF0000u);
                    } else {
                        const __half2 b = __floats2half2_rn(s[j][n][2 * h], s[j][n][2 * h + 1]);
                        p = *reinterpret_cast<const uint32_t *>(&b);
                        if constexpr (!CODES) {
                            const float2 f = __half22float2(b);
                            l[n][0] += f.x;
                            l[n][1] += f.y;
                        }
                    }
                    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(pf[j][n][h]) : "r"(p));
                }
            if (__any_sync(0xFFFFFFFFu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int c = 0; c < OT; c++)
#pragma unroll
                    for (int q = 0; q < 4; q++) o[n][c][q] *= alpha[q & 1];
            }
        }
        // O^T += V^T P^T, 16 positions at a time: tile c of O is columns 2c and 2c + 1 of every lane's CPL
#pragma unroll
        for (int kk = 0; kk < MT; kk++) {
            constexpr int NW = CB >= 16 ? 4 : CB >= 4 ? CB / 4 : 1;  // words of an access
            auto step = [&](int c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                const uint32_t va[4] = {a0, a1, a2, a3};
#pragma unroll
                for (int n = 0; n < NQ; n++) cr_mma<BF16>(o[n][c], va, pf[kk][n][0], pf[kk][n][1]);
            };
#pragma unroll
            for (int pc = 0; pc < (CB + 15) / 16; pc++) {
                uint32_t w[4][NW];                         // of rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint8_t *at = stage + (v_at[q & 1] ^ (pc * 16)) + (kk * 16 + (q >> 1) * 8) * ROWB;
                    if constexpr (CB >= 4) cr_lds<NW>(w[q], at);
                    else w[q][0] = *reinterpret_cast<const uint16_t *>(at);
                }
#pragma unroll
                for (int v = 0; v < NW; v++) {
                    if constexpr (KIND <= KV_BF16) {
                        step(pc * 4 + v, __byte_perm(w[0][v], w[1][v], 0x5410), __byte_perm(w[0][v], w[1][v], 0x7632), __byte_perm(w[2][v], w[3][v], 0x5410),
                             __byte_perm(w[2][v], w[3][v], 0x7632));
                    } else if constexpr (KIND == KV_INT4) {
#pragma unroll
                        for (int half = 0; half < (CB == 2 ? 1 : 2); half++) {
                            const int c = (pc * 4 + v) * 4 + half * 2;
                            uint32_t b0[4], b1[4];
                            cr_nibbles(__byte_perm(w[0][v], w[1][v], half ? 0x7632 : 0x5410), b0);
                            cr_nibbles(__byte_perm(w[2][v], w[3][v], half ? 0x7632 : 0x5410), b1);
                            step(c, b0[0], b0[1], b1[0], b1[1]);
                            step(c + 1, b0[2], b0[3], b1[2], b1[3]);
                        }
                    } else {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            uint32_t b0[2], b1[2];
                            cr_bytes<KIND>(__byte_perm(w[0][v], w[1][v], half ? 0x7362 : 0x5140), b0[0], b0[1]);
                            cr_bytes<KIND>(__byte_perm(w[2][v], w[3][v], half ? 0x7362 : 0x5140), b1[0], b1[1]);
                            step((pc * 4 + v) * 2 + half, b0[0], b0[1], b1[0], b1[1]);
                        }
                    }
                }
            }
        }
        st = st + 1 == ST ? 0 : st + 1;
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");

    // ---- the warps' parts, in the order of fragments -------------------------------------------------------------------------
    __syncthreads();                                       // the rings are free
    float *parts = reinterpret_cast<float *>(cr_smem), *acc = reinterpret_cast<float *>(cr_smem + C::ACC_OFF);  // [warp][row group, tile][4][lane]; [R][PITCH]
    constexpr uint32_t VALUES = R * HD;
#pragma unroll
    for (int n = 0; n < NQ; n++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int q = 4; q < 32; q <<= 1) {
                l[n][h] += __shfl_xor_sync(0xFFFFFFFFu, l[n][h], q);
                if constexpr (NSC == 2) z[n][h] += __shfl_xor_sync(0xFFFFFFFFu, z[n][h], q);
            }
            if (g == 0) {
                w_max[warp * R + n * 8 + 2 * t + h] = m[n][h];
                w_sum[warp * R + n * 8 + 2 * t + h] = l[n][h];
            }
        }
#pragma unroll
        for (int c = 0; c < OT; c++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float v = o[n][c][q];
                if constexpr (CODES) v = v * (1.0f / CR_UP) * unit[n][q & 1];
                if constexpr (NSC == 2) v += z[n][q & 1];
                parts[warp * VALUES + ((n * OT + c) * 4 + q) * 32 + lane] = v;
            }
    }
    __syncthreads();
    if (tid < R) {
        float top = -INFINITY, sum = 0.0f;
        for (int w = 0; w < CR_W; w++) top = fmaxf(top, w_max[w * R + tid]);
        const float sub = top == -INFINITY ? 0.0f : top;
        for (int w = 0; w < CR_W; w++) {
            const float f = cr_ex2(w_max[w * R + tid] - sub);
            sum += w_sum[w * R + tid] * f;
            w_max[w * R + tid] = f;                        // from here on: the warp's weight
        }
        r_max[tid] = top;
        r_sum[tid] = sum;
    }
    __syncthreads();
    for (uint32_t b = warp; b < (uint32_t)NQ * OT * 4; b += CR_W) {
        const uint32_t q = b & 3, c = (b >> 2) % OT, row = (b >> 2) / OT * 8 + 2 * t + (q & 1);
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < CR_W; w++) v += parts[w * VALUES + b * 32 + lane] * w_max[w * R + row];
        acc[row * PITCH + g * CPL + 2 * c + (q >> 1)] = v;
    }
    __syncthreads();

    // ---- the blocks' parts: left to cache_join_kernel, or each block joins some rows out of the shared memory of all -----------------------------
    if (d.splits > CR_CLUSTER) {
        constexpr size_t PART = cache_part_floats(R, HD);
        float *mine = d.part + (size_t)blockIdx.x * PART;
        for (uint32_t i = tid; i < VALUES / 4; i += CR_THREADS)
            __stcg(reinterpret_cast<float4 *>(mine) + i, *reinterpret_cast<const float4 *>(acc + i % R * PITCH + i / R * 4));
        if (tid < R) {
            __stcg(mine + VALUES + tid, r_max[tid]);
            __stcg(mine + VALUES + R + tid, r_sum[tid]);
        }
        return;
    }
    const uint32_t lo = split * R / d.splits, hi = min((split + 1) * R / d.splits, here);  // rows of this block
    if (d.splits > 1) cr_cluster_sync();

    // ---- results: four columns of a row a thread ------------------------------------------------------------------------------
    for (uint32_t u = tid; u < (hi > lo ? hi - lo : 0) * (HD / 4); u += CR_THREADS) {
        const uint32_t r = lo + u / (HD / 4), c = u % (HD / 4) * 4;
        float sum = r_sum[r];
        float4 v = *reinterpret_cast<const float4 *>(acc + r * PITCH + c);
        if (d.splits > 1) {
            const uint32_t max_at = (uint32_t)__cvta_generic_to_shared(r_max + r), sum_at = (uint32_t)__cvta_generic_to_shared(r_sum + r),
                           acc_at = (uint32_t)__cvta_generic_to_shared(acc + r * PITCH + c);
            float f[CR_CLUSTER], part[CR_CLUSTER], top = -INFINITY;
            float4 w[CR_CLUSTER];
#pragma unroll
            for (uint32_t s = 0; s < CR_CLUSTER; s++) {
                const uint32_t from = s < d.splits ? s : 0;
                f[s] = cr_lds_of(max_at, from);
                part[s] = cr_lds_of(sum_at, from);
                w[s] = cr_lds4_of(acc_at, from);
                if (s < d.splits) top = fmaxf(top, f[s]);
            }
            const float sub = top == -INFINITY ? 0.0f : top;
            sum = 0.0f;
            v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t s = 0; s < CR_CLUSTER; s++)
                if (s < d.splits) {
                    const float k = cr_ex2(f[s] - sub);
                    sum = fmaf(part[s], k, sum);
                    v = make_float4(fmaf(w[s].x, k, v.x), fmaf(w[s].y, k, v.y), fmaf(w[s].z, k, v.z), fmaf(w[s].w, k, v.w));
                }
        }
        const float inv = 1.0f / sum;
        v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        if (!(sum > 0.0f) || !isfinite(v.x) || !isfinite(v.y) || !isfinite(v.z) || !isfinite(v.w)) {
            atomicOr(flags, 1u << r);
            continue;
        }
        const uint32_t rr = r0 + r;
        uint16_t *dst = a.out + (size_t)(x.row0 + rr / a.group) * a.out_stride + (size_t)(kh * a.group + rr % a.group) * HD + c;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(kv_round2(v.x, v.y, a.c.rows_bf16), kv_round2(v.z, v.w, a.c.rows_bf16));
    }
    __syncthreads();
    const uint32_t again = flags[0];
    for (uint32_t r = warp; r < here; r += CR_W)
        if (again >> r & 1) cache_plain_row<KIND, HD>(a, x, (r0 + r) / a.group, kh * a.group + (r0 + r) % a.group, lane);
    if (d.splits > 1) cr_cluster_sync();                   // nobody leaves before the others have read its part
}

// ---- scratch -----------------------------------------------------------------------------------------------------------------
// Parts and counters.  Eager calls of a context share a block, which grows when the stream is idle.  Calls that are being captured use
// a block of their capture: a replay finds it whatever ran in between, and no two captures share one.  The captured graph and what is
// instantiated from it hold a reference to the block; when the last of them is gone, and its launches with it, a later capture takes it.
struct CacheScratch {
    struct Block {
        unsigned long long capture;  // 0: eager
        uint8_t *mem;
        size_t part_bytes, counts;
        std::shared_ptr<std::atomic<bool>> left;  // of a capture: nothing refers to it any more
        bool fits(size_t bytes, size_t n) const { return part_bytes >= bytes && counts >= n; }
    };
    std::vector<Block> blocks;
};
void cache_scratch_free(CacheScratch *s) {
    if (!s) return;
    for (auto &b : s->blocks) cudaFree(b.mem);
    delete s;
}
static void CUDART_CB cache_block_left(void *p) {          // on a thread of the driver's: no CUDA calls
    auto *left = static_cast<std::shared_ptr<std::atomic<bool>> *>(p);
    (*left)->store(true);
    delete left;
}
// The block goes with this graph.
static int cache_block_of(prism_cuda_ctx *ctx, CacheScratch::Block &b, unsigned long long capture, cudaGraph_t graph) {
    auto flag = std::make_shared<std::atomic<bool>>(false);
    auto theirs = std::make_unique<std::shared_ptr<std::atomic<bool>>>(flag);
    cudaUserObject_t object;
    PRISM_CUDA_TRY(ctx, cudaUserObjectCreate(&object, theirs.get(), cache_block_left, 1, cudaUserObjectNoDestructorSync));
    theirs.release();
    b.capture = capture;
    b.left = std::move(flag);
    const cudaError_t e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) {
        (void)cudaUserObjectRelease(object, 1);
        return cuda_fail(ctx, e, "cudaGraphRetainUserObject");
    }
    return PRISM_OK;
}
int cache_scratch(prism_cuda_ctx *ctx, size_t part_bytes, size_t counts, float **part, unsigned int **count) {
    if (!ctx->cache_scratch) ctx->cache_scratch = new CacheScratch();
    auto &blocks = ctx->cache_scratch->blocks;
    cudaStreamCaptureStatus status;
    unsigned long long id = 0;
    cudaGraph_t graph = nullptr;
    PRISM_CUDA_TRY(ctx, cudaStreamGetCaptureInfo(ctx->stream, &status, &id, &graph));
    if (status == cudaStreamCaptureStatusNone) id = 0;
    auto use = [&](CacheScratch::Block &b) {
        *part = reinterpret_cast<float *>(b.mem);
        if (count) *count = reinterpret_cast<unsigned int *>(b.mem + b.part_bytes);
    };
    // kernels leave the counters at zero; in a capture this is a node before them
    auto clear = [&](CacheScratch::Block &b) -> int {
        if (b.counts) PRISM_CUDA_TRY(ctx, cudaMemsetAsync(b.mem + b.part_bytes, 0, b.counts * 4, ctx->stream));
        return PRISM_OK;
    };
    for (auto &b : blocks)
        if (b.capture == id && b.fits(part_bytes, counts)) {
            use(b);
            return PRISM_OK;
        }
    if (id == 0) {                                         // the block in use, and those that nothing refers to, make room for a larger one
        PRISM_CUDA_TRY(ctx, cudaStreamSynchronize(ctx->stream));
        for (size_t i = blocks.size(); i-- > 0;) {
            if (blocks[i].capture != 0 && !blocks[i].left->load()) continue;
            if (blocks[i].capture == 0) {
                part_bytes = std::max(part_bytes, blocks[i].part_bytes);
                counts = std::max(counts, blocks[i].counts);
            }
            cudaFree(blocks[i].mem);
            blocks.erase(blocks.begin() + i);
        }
    } else {
        CacheScratch::Block *best = nullptr;
        for (auto &b : blocks)
            if (b.capture != 0 && b.left->load() && b.fits(part_bytes, counts) && (!best || b.part_bytes < best->part_bytes)) best = &b;
        if (best) {
            PRISM_TRY(cache_block_of(ctx, *best, id, graph));
            PRISM_TRY(clear(*best));
            use(*best);
            return PRISM_OK;
        }
    }
    blocks.reserve(blocks.size() + 1);                     // nothing throws between the allocation and its place
    part_bytes = (part_bytes + 255) / 256 * 256;
    counts = (counts + 63) / 64 * 64;
    CacheScratch::Block b{id, nullptr, part_bytes, counts, nullptr};
    if (id == 0) {
        PRISM_CUDA_TRY(ctx, device_malloc(ctx, (void **)&b.mem, part_bytes + counts * 4));
    } else {
        b.left = std::make_shared<std::atomic<bool>>(true);  // until the graph has it
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // an allocation is no part of the capture
        PRISM_CUDA_TRY(ctx, cudaThreadExchangeStreamCaptureMode(&mode));
        const cudaError_t e = cudaMalloc((void **)&b.mem, part_bytes + counts * 4);
        (void)cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess) {
            (void)cudaGetLastError();
            return cuda_fail(ctx, e, "cudaMalloc(attention scratch of a capture)");
        }
    }
    blocks.push_back(std::move(b));
    if (id != 0) PRISM_TRY(cache_block_of(ctx, blocks.back(), id, graph));
    PRISM_TRY(clear(blocks.back()));
    use(blocks.back());
    return PRISM_OK;
}

template <int KIND, int HD, int NQ>
static int launch_rows_kernel(prism_cuda_ctx *ctx, const CacheAttnDev &a, uint32_t max_length) {
    using C = CrCfg<KIND, HD, NQ>;
    static int room[PRISM_MAX_DEVICES][CR_CLUSTER + 1] = {{0}};  // clusters of that many blocks that the device holds at once; [0]: asked already
    if (!room[ctx->device][0]) {
        PRISM_CUDA_TRY(ctx, cudaFuncSetAttribute(cache_rows_kernel<KIND, HD, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
        int n = 0;
        PRISM_CUDA_TRY(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, cache_rows_kernel<KIND, HD, NQ>, CR_THREADS, C::SMEM));
        if (n < 1) return fail(ctx, PRISM_E_CUDA, "cache_rows_kernel does not fit an SM");
        room[ctx->device][1] = n * ctx->sm_count;
        for (uint32_t size = 2; size <= CR_CLUSTER; size++) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(size);
            cfg.blockDim = dim3(CR_THREADS);
            cfg.dynamicSmemBytes = C::SMEM;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = size;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            PRISM_CUDA_TRY(ctx, cudaOccupancyMaxActiveClusters(&room[ctx->device][size], cache_rows_kernel<KIND, HD, NQ>, &cfg));
        }
        room[ctx->device][0] = 1;
    }
    CrDev d{};
    d.a = a;
    d.tiles = (uint32_t)(((uint64_t)a.max_tokens * a.group + C::R - 1) / C::R);
    const uint64_t items = (uint64_t)a.n_entries * a.c.kv_heads * d.tiles, slots = (uint64_t)room[ctx->device][1];
    uint64_t seen = max_length;
    if (a.window) seen = std::min<uint64_t>(seen, (uint64_t)a.window + a.sinks + 2 * C::TP);
    const uint64_t most = (seen + C::TP * CR_W - 1) / (C::TP * CR_W);  // parts in which every warp has a tile
    // Parts that fill the GPU once, where they are more than a cluster: a cluster joins in a microsecond, scratch and a second kernel in four, which
    // is worth it where a block of a cluster had more than CR_NEAR positions (8 heads of 128, 24 drafts of 8000 positions: 22 us by clusters, 18 by
    // parts; 6000 positions of one sequence: 13.1 and 12.6; 2000: 8.4 and 10.4).
    uint64_t parts = std::min<uint64_t>(std::min<uint64_t>(most, CJ_MAX_SPLIT), slots / items);
    if (parts <= CR_CLUSTER || seen <= CR_CLUSTER * CR_NEAR) {
        // Else the size of cluster with the smallest waves * (positions of a part + what a block costs besides, in positions).  A block costs 6 us:
        // 650 positions of 128 codes; 16-bit rows are bound by HBM from half of the blocks on, and lose more by a second wave.  256 row tiles of
        // 128-wide heads, one part and three: int8 over 8000 positions 113 and 76 us, over 2000 38 and 33; 16 bits 124 and 103, 38 and 37.
        constexpr uint64_t BESIDE = KIND >= KV_INT8 ? 650 : 2000;
        uint64_t least = UINT64_MAX;
        for (uint32_t size = 1; size <= CR_CLUSTER && size <= std::max<uint64_t>(most, 1); size++) {
            const uint64_t at_once = (uint64_t)std::max(room[ctx->device][size], 1);
            const uint64_t cost = (items + at_once - 1) / at_once * ((seen + size - 1) / size + BESIDE);
            if (cost < least) {
                least = cost;
                parts = size;
            }
        }
    }
    d.splits = (uint32_t)parts;
    if (items * parts > 0x7FFFFFFFull) return fail(ctx, PRISM_E_ARG, "cache_attention: too many rows");
    const bool join = parts > CR_CLUSTER;
    if (join) PRISM_TRY(cache_scratch(ctx, (size_t)(items * parts) * cache_part_floats(C::R, HD) * 4, 0, &d.part, nullptr));
    launch_cluster_pdl(ctx, cache_rows_kernel<KIND, HD, NQ>, dim3((uint32_t)(items * parts)), dim3(CR_THREADS), C::SMEM, join ? 1u : (unsigned)parts, d);
    PRISM_TRY(after_launch(ctx, "cache_rows_kernel"));
    return join ? launch_cache_join<KIND, HD>(ctx, CacheJoinDev{a, d.splits, d.tiles, (uint32_t)C::R, d.part}) : PRISM_OK;
}

template <int KIND>
static int launch_kind(prism_cuda_ctx *ctx, uint32_t hd, const CacheAttnDev &a, uint32_t max_length) {
    const bool one = (uint64_t)a.max_tokens * a.group <= 8;
    switch (hd) {
    case 32: return one ? launch_rows_kernel<KIND, 32, 1>(ctx, a, max_length) : launch_rows_kernel<KIND, 32, 2>(ctx, a, max_length);
    case 64: return one ? launch_rows_kernel<KIND, 64, 1>(ctx, a, max_length) : launch_rows_kernel<KIND, 64, 2>(ctx, a, max_length);
    case 128: return one ? launch_rows_kernel<KIND, 128, 1>(ctx, a, max_length) : launch_rows_kernel<KIND, 128, 2>(ctx, a, max_length);
    default: return one ? launch_rows_kernel<KIND, 256, 1>(ctx, a, max_length) : launch_rows_kernel<KIND, 256, 2>(ctx, a, max_length);
    }
}

static int cache_attention(prism_cuda_ctx *ctx, const prism_cache *c, const prism_cache_attention *p) {
    if (!ctx || !c || !p) return fail(ctx, PRISM_E_NULL, "cache_attention: null argument");
    CacheAttnDev a{};
    int kind;
    PRISM_TRY(kv_check(ctx, c, &a.c, &kind));
    if (p->num_heads == 0 || p->num_heads > 65536 || p->num_heads % c->kv_heads)
        return fail(ctx, PRISM_E_ARG, "cache_attention: num_heads must be a multiple of kv_heads, at most 65536");
    if (p->n_entries > 65535) return fail(ctx, PRISM_E_ARG, "cache_attention: at most 65535 entries a call");
    if (p->n_rows > 0x7FFFFFFFu || p->max_tokens > (1u << 24) || (uint64_t)p->max_tokens * p->num_heads > (1u << 30))
        return fail(ctx, PRISM_E_ARG, "cache_attention: too many rows");
    if (p->tree && (p->tree_words == 0 || (uint64_t)p->tree_words * 64 < p->max_tokens))
        return fail(ctx, PRISM_E_ARG, "cache_attention: a row's mask needs a bit for each of max_tokens tokens");
    if (p->tree && p->window && !p->q_pos) return fail(ctx, PRISM_E_NULL, "cache_attention: a tree under a window needs the rows' positions");
    if (!std::isfinite(p->scale)) return fail(ctx, PRISM_E_ARG, "cache_attention: the scale of the scores must be finite");
    if (p->n_entries == 0 || p->n_rows == 0 || p->max_tokens == 0) return PRISM_OK;
    if (!p->q || !p->out || !p->seq || !p->q_start || !p->length) return fail(ctx, PRISM_E_NULL, "cache_attention: null argument");
    const uint64_t width = (uint64_t)p->num_heads * c->head_dim;
    if (p->q_stride < width || p->out_stride < width || p->q_stride % 8 || p->out_stride % 8 ||
        ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out)) & 15))
        return fail(ctx, PRISM_E_ARG, "cache_attention: rows must be 16-byte aligned and at least num_heads * head_dim values apart");
    if (!kv_words(p->seq, p->q_start, p->length, p->q_pos))
        return fail(ctx, PRISM_E_ARG, "cache_attention: seq, q_start, length and q_pos must be 4-byte aligned");
    if (reinterpret_cast<uintptr_t>(p->tree) & 7) return fail(ctx, PRISM_E_ARG, "cache_attention: masks must be 8-byte aligned");
    if (p->q == p->out) return fail(ctx, PRISM_E_ARG, "cache_attention: results must not overlap the queries");  // a row may be taken again
    DeviceGuard on(ctx->device);
    if (on.err != cudaSuccess) return cuda_fail(ctx, on.err, "cudaSetDevice");
    a.q = static_cast<const uint16_t *>(p->q);
    a.out = static_cast<uint16_t *>(p->out);
    a.q_stride = p->q_stride;
    a.out_stride = p->out_stride;
    a.n_rows = p->n_rows;
    a.n_entries = p->n_entries;
    a.seq = p->seq;
    a.q_start = p->q_start;
    a.length = p->length;
    a.max_tokens = p->max_tokens;
    a.heads = p->num_heads;
    a.group = p->num_heads / c->kv_heads;
    a.window = p->window;
    a.sinks = p->window ? p->sinks : 0;
    a.scale = p->scale != 0.0f ? p->scale : 1.0f / sqrtf((float)c->head_dim);
    a.tree = p->tree;
    a.tree_words = p->tree_words;
    a.q_pos = p->q_pos;
    const uint64_t rows = (uint64_t)a.max_tokens * a.group, seen = a.window ? std::min<uint64_t>(p->max_length, (uint64_t)a.window + a.sinks) : p->max_length;
    const uint64_t items = (rows + 15) / 16 * a.n_entries * c->kv_heads;
    if (rows > 32 && (items > 2 * (uint64_t)ctx->sm_count || items * seen > CR_WORK) && cache_tiles_fit(a, c->head_dim))
        return launch_cache_tiles(ctx, kind, c->head_dim, a, p->max_length);
    switch (kind) {
    case KV_F16: return launch_kind<KV_F16>(ctx, c->head_dim, a, p->max_length);
    case KV_BF16: return launch_kind<KV_BF16>(ctx, c->head_dim, a, p->max_length);
    case KV_INT8: return launch_kind<KV_INT8>(ctx, c->head_dim, a, p->max_length);
    case KV_E4M3: return launch_kind<KV_E4M3>(ctx, c->head_dim, a, p->max_length);
    default: return launch_kind<KV_INT4>(ctx, c->head_dim, a, p->max_length);
    }
}

}  // namespace prism

using namespace prism;

extern "C" int prism_cuda_cache_attention_dev(prism_cuda_ctx *ctx, const prism_cache *cache, const prism_cache_attention *a) {
    try {
        return cache_attention(ctx, cache, a);
    } catch (const std::exception &) {
        return PRISM_E_STATE;  // no memory for a message
    }
}
