// Attention of single tokens (or a few drafted ones) over the 4-bit relay cache.
//
// Row (n, t, head): scores s_k = scale q.K_k over the keys of [shared prefix ; own sequence], the
// own keys of query t ending at lengths[n] - queries + t; m = max s, l = sum exp(s - m),
// o = sum exp(s - m) V / l, with the statistics [m, l] of the relay merge and its convention for a
// row without keys (o = 0, [0, 1]).
//
// The cache is read once and that bounds the work (1.25 D bytes a token and kv head), so the codes
// have to become operands of a matrix product at the rate at which they arrive.  With value =
// minimum + scale code for each group j of 32 channels,
//     s_k   = sum_j scale_kj (q_j . code_kj) + min_kj sum(q_j)
//     o_c   = sum_k (p_k scale_kj) code_kc + sum_k p_k min_kj
// and the products with the codes run on mma.sync m16n8k16 with f16 operands and f32 sums, tokens
// (K) or channels (V) in the 16 rows and up to 8 query rows in the 8 columns:
//   * a code needs no conversion: the 16-bit word with the code in four of its lowest 10 bits is an f16
//     subnormal, code * 2^-20 in bits 4 .. 7, so a shift and an AND make the operand register of two
//     keys' codes.  The powers of two go into q.  The products' sums drop what lies 24 bits below the
//     largest operand exponent, and a subnormal's counts as 2^-14, which leaves 18 to 22 bits (in the
//     lowest four bits it would be 14 to 18: an error of 1e-6 in the sums of small calls); for f32 rows the
//     codes go to the top of the mantissa (code * 2^-18, 20 to 24 bits).  The values' codes become normal
//     numbers around zero (code - 8), so that long sums neither drop bits nor cancel:
//     o = sum r (code - 8) + sum p (min + 8 scale), r the rounded p scale.  For f32 rows it is code - 7.5, the
//     codes' mean, for two shifts more: the sums truncate, and half a scale a token that grows in one of them
//     and is taken off in the other left an error of 2e-5 after 90000 tokens (now 1e-6).
//   * q is held in f16 relative to a power of two of its own row (bf16 q: exact down to 2^-31 of the row's
//     largest; f32 q: two f16 parts, 22 bits down to 2^-17 of it, then fewer), p scale in f16 relative to a power of two near the largest of its row and group of
//     channels (f32: again two parts), so that a group of small values is as exact as one of large ones.
//   * the minima are operands as they lie in memory: a token's (scale, minimum) words are the bf16
//     pairs of a row, met by zeros in the scales' places (keys), or read by a transposing ldmatrix
//     (values, which also gives the sums of p scale); sum(q) and p are given in bf16 parts.
//   * the scores arrive with tokens in rows and have to leave with tokens along the product's
//     inner dimension: movmatrix transposes the 8 x 8 blocks.
// The running maximum is only raised when a score passes it by 8 (in powers of two), so a step
// usually costs one vote instead of the shuffles of a maximum and the rescaling of the sums.  p is relative
// to that bound, not to the maximum, so it is never above 1 and the sums of large values stay in range.
//
// Work: an item is (sequence, kv head, up to 8 NR rows), or (kv head, up to 8 NR rows of all
// sequences) of a prefix that is worth a launch of its own, which is thus read once per head for 8 NR
// rows; other prefixes are read with every sequence's own tokens.  Items are cut into units of 128
// tokens, and the units of all items, one after another, are dealt to the CTAs that the GPU holds in
// equal runs, whatever the lengths are: a CTA finds its run in the lengths, so the host does not need
// them.  A CTA's four warps take turns at steps of 32 tokens, each with a ring of its own that bulk
// copies fill (tcgen05 needs 64 or 128 query rows to a tile, which only the rows of all sequences at a
// shared prefix make).  An item that one CTA holds whole is finished there; the others' sums go to the
// workspace, and the CTA that arrives last at an item joins them.  The prefix's launch comes before the
// sequences', which joins its sums to every item's and may start before it has ended: its CTAs come up
// as the prefix's leave (those of 16 rows hold an SM's registers two by two, so the two launches take
// 30 and 54 us alone and 85 together; what is saved is the gap between them).
//
// Bound: the codes' way from memory to operand.  131072 tokens of one sequence, 16 heads of 128 (336
// MB): 81.8 us = 4100 GB/s, 63% of the measured copy rate; 363 instructions a warp and tile of 16 tokens,
// issue slots 60% and ALU 54% busy (LOP3, shifts and byte permutes; a tile needs 64 + 32 + 8 of them).
// The slope is 78% of the copy rate (131072 to 262144 tokens); the rest is some 16 us of starts, joins
// and an uneven end.  CTAs of 2 and 8 warps instead of 4: 131072 tokens 91 and 79 us for 82, 64 sequences after
// a prefix 83.6 and 92 for 85.7, 48 ragged 47 and 48.6 for 43.2, six drafts 37.7 and 38.3 for 35; a rule by
// shape is not taken.  Tried in an earlier build and slower: 3 and 5 CTAs an SM, steps of 16 and 64 tokens,
// rings of 1, 3 and 4 stages, the next item's copies before this one's sums are joined (registers), shifts as
// high products.
#include <float.h>

#include <algorithm>

#include "relay_cache.cuh"
#include "tc_ptx.cuh"

namespace dbl {

namespace {

constexpr int W = 4;              // warps of a CTA
constexpr int TS = 2;             // tiles of a step
constexpr int STEP = TS * kCacheTile;
constexpr int NS = 2;             // stages of a warp's ring
constexpr int UNIT = W * STEP;    // tokens of a unit
constexpr int64_t kApart = 1 << 19;  // sequences x kv heads x tokens of a prefix with a launch of its own
constexpr int kStart = 3;         // units that the start and end of an item cost (about 6 us, a unit 2 us)
constexpr int kCounterBytes = DBL_RELAY_CACHE_COUNTER_BYTES;
// Units of a run.  16 f32 sequences of 131072 tokens whose values average out, 16 heads of 128, are off by 2.5e-5 of the
// result in runs of 443 units and by 7e-6 in runs of 148; 1048576 tokens, 16 heads, 700 us by one round and 708 by three.
constexpr int kRun = 128;
constexpr int WIN = 32 / TS;      // steps whose page numbers the lanes of a warp hold
constexpr int kCacheWaitFull = 40;  // wait-site code (dbl_device_error)
constexpr int kNoPage = -1, kPast = -2;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Tokens of a segment: tile * tiles_inv has its exact quotient below 2^32 / 256 tiles.
constexpr int64_t kMostTokens = (int64_t)1 << 27;
constexpr float kSlack = 8.f;     // how far a score may pass the running maximum (powers of two)
constexpr int kLift = 32;         // powers of two between the scores of queries from 2^120 on and their f
constexpr float kMostF16 = 60000.f;             // p scale mult stays below it
constexpr float kMostMult = 8.507059173e37f;    // 2^126
constexpr int kMostMultBits = 127 + 126;        // its exponent's bits

struct AttnParams {
    CacheView c;
    const void* q;
    int64_t qs[3];  // strides of sequence, query and head
    bool q_vec;     // 16-byte loads
    const int32_t *lengths, *prefix_pages;
    void* out;
    float *row_max, *row_sum;
    int N, Tq, H, group, prefix_len, prefix_width;
    float scale;
    uint32_t tiles_inv;  // ceil(2^32 / tiles of a page), 0 for 1: tile / tiles is the high word of a product
    bool pre;       // this launch: the prefix, or the sequences' own tokens (PRE on the device)
    int lead;       // tokens of the prefix's tiles where the sequences' launch reads them itself, 0 where not
    int tiles;      // row tiles: of a kv head over all sequences, or of a kv head and sequence
    int pre_tiles, pre_rows, pre_units, pre_run, pre_parts;  // the prefix: row tiles of a head, rows of a tile, units,
                                                             // units of a run, partials of a row at most
    unsigned* counter;     // [CTAs]: of the item that begins in a CTA's run and ends in another's
    float *part, *pre_part;  // rows of D sums, maximum, sum (D + 4 floats): [CTAs][2][R]; [heads, tiles, R][pre_parts]
    int* err;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero sums.
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Inner dimension 8.
__device__ __forceinline__ void mma_bf16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(b));
}
__device__ __forceinline__ void mma_bf16_k8_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(b), "f"(0.f));
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void bulk_load(void* sdst, const void* gsrc, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32addr(sdst)),
                 "l"(gsrc), "r"(bytes), "r"(smem_u32addr(bar))
                 : "memory");
}
// Waits for phase `parity` for at most kWaitLimitNs, whatever the block's error word says.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity))
        if (globaltimer_ns() - t0 > kWaitLimitNs) return;
}
__device__ __forceinline__ float f16x2_lo(uint32_t x) {
    float y;
    asm("{.reg .f16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, a;}" : "=f"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float f16x2_hi(uint32_t x) {
    float y;
    asm("{.reg .f16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, b;}" : "=f"(y) : "r"(x));
    return y;
}
// hi = (a, b) in f16, lo = what it leaves
__device__ __forceinline__ void split_f16x2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack_f16x2(a, b);
    lo = pack_f16x2(a - f16x2_lo(hi), b - f16x2_hi(hi));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float over_g_max(float x) {  // over the lanes of the same column pair
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float over_g_sum(float x) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// The power of two that takes w to 2^7 .. 2^8 (what is added later may be 2^8 times as large before it is lowered,
// and f16 holds what is 2^-22 of it to 11 bits), and the inverse of a power of two.
__device__ __forceinline__ float mult_for(float w) {
    const int e = min(max((int)(__float_as_uint(w) >> 23), 261 - kMostMultBits), 250);
    return __uint_as_float((uint32_t)(261 - e) << 23);
}
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }
__device__ __forceinline__ float pow2(int e) {  // 0 below 2^-126; e < 128
    return e < -126 ? 0.f : __uint_as_float((uint32_t)(127 + e) << 23);
}

// The operand registers of the 8 codes of w, codes (0, 4), (1, 5), (2, 6), (3, 7), and what they are
// multiplied by to be the codes (code_unit).
enum class Codes { kMid, kHigh, kCentred, kHalf };
// (x & mask) | bits in one instruction, which takes one constant: the other one stays in a register.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
    return r;
}
template <Codes C>
__device__ __forceinline__ void code_operands(uint32_t w, uint32_t (&r)[4]) {
    if constexpr (C == Codes::kHigh) {
        r[0] = (w << 6) & 0x03C003C0u, r[1] = (w << 2) & 0x03C003C0u;
        r[2] = (w >> 2) & 0x03C003C0u, r[3] = (w >> 6) & 0x03C003C0u;
    } else if constexpr (C == Codes::kMid) {
        r[0] = (w << 4) & 0x00F000F0u, r[1] = w & 0x00F000F0u;
        r[2] = (w >> 4) & 0x00F000F0u, r[3] = (w >> 8) & 0x00F000F0u;
    } else if constexpr (C == Codes::kHalf) {  // 1144 = 1024 + 16 * 7.5
        r[0] = and_or(w << 4, 0x00F000F0u, 0x64006400u), r[1] = and_or(w, 0x00F000F0u, 0x64006400u);
        r[2] = and_or(w >> 4, 0x00F000F0u, 0x64006400u), r[3] = and_or(w >> 8, 0x00F000F0u, 0x64006400u);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("add.rn.f16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(0xE478E478u));
    } else {  // 1024 + x is the f16 with mantissa x; 1032 = 1024 + 8, 1152 = 1024 + 16 * 8
        const uint32_t v = w >> 8;
        r[0] = and_or(w, 0x000F000Fu, 0x64006400u), r[1] = and_or(w, 0x00F000F0u, 0x64006400u);
        r[2] = and_or(v, 0x000F000Fu, 0x64006400u), r[3] = and_or(v, 0x00F000F0u, 0x64006400u);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            asm("add.rn.f16x2 %0, %0, %1;" : "+r"(r[i]) : "r"(i & 1 ? 0xE480E480u : 0xE408E408u));
    }
}
template <Codes C>
constexpr float code_unit(int i) {
    return C == Codes::kHigh ? 262144.f : C == Codes::kMid ? 1048576.f : C == Codes::kHalf || i & 1 ? 0.0625f : 1.f;
}

// The operand whose rows are the 2 G scales and minima of a tile's tokens (scale 0, minimum 0, scale 1,
// ...) and whose inner dimension are its 16 tokens (rows 8 .. 15 hold anything).
template <int G>
__device__ __forceinline__ void group_operands(const uint8_t* groups, int lane, uint32_t (&a)[4]) {
    if constexpr (G == 4) {  // a token's 8 numbers are a row of an 8 x 8 matrix
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                     : "r"(smem_u32addr(groups + (lane & 7) * 16 + (lane & 16) * 8)));
    } else {
        const int g = lane >> 2, t = lane & 3;
        const uint4 x = *reinterpret_cast<const uint4*>(groups + t * 16), y = *reinterpret_cast<const uint4*>(groups + 64 + t * 16);
        const uint32_t sel = g & 1 ? 0x7632u : 0x5410u;
        a[0] = a[1] = g & 2 ? __byte_perm(x.y, x.w, sel) : __byte_perm(x.x, x.z, sel);
        a[2] = a[3] = g & 2 ? __byte_perm(y.y, y.w, sel) : __byte_perm(y.x, y.z, sel);
    }
}

template <int G>
struct Words {  // the G words that a lane reads at once
    uint32_t w[G];
};
template <int G>
__device__ __forceinline__ Words<G> lds_words(const uint8_t* p) {
    Words<G> r;
    if constexpr (G == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        r.w[0] = x.x, r.w[1] = x.y, r.w[2] = x.z, r.w[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        r.w[0] = x.x, r.w[1] = x.y;
    }
    return r;
}

constexpr int kPartPad = 4;  // floats of a partial row after its D sums: maximum, sum, two unused

// Joins partial rows to the warp's own rows acc [rows][D] with (maximum, sum) ml [rows], in shared
// memory.  Lane r says where the partials of row r lie: the i-th of its `count` at from + off + i * stride,
// the first one `extra` further; the warp takes every W-th.
template <int D, int R>
__device__ __forceinline__ void fold_rows(float* acc, float2* ml, int rows, int warp, int lane, const float* from,
                                          int off, int stride, int extra, int count) {
    constexpr int V = D / 32;  // channels of a lane, neighbouring
    if (lane >= rows) count = 0;
    const int most = __reduce_max_sync(0xffffffffu, count);
    const float2 own = lane < rows ? ml[lane] : make_float2(-INFINITY, 0.f);
    float m = own.x;
#pragma unroll 8
    for (int i = warp; i < most; i += W)
        if (i < count) m = fmaxf(m, __ldcg(from + off + i * stride + (i ? 0 : extra) + D));
    const float c = own.x == -INFINITY ? 0.f : ex2(own.x - m);
    float l = own.y * c, o[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float cr = __shfl_sync(0xffffffffu, c, r);
#pragma unroll
        for (int v = 0; v < V; ++v) o[r][v] = r < rows ? acc[r * D + lane * V + v] * cr : 0.f;
    }
    constexpr int AT_ONCE = R == 1 ? 8 : R <= 4 ? 2 : 1;  // parts whose loads are on their way together
    for (int i0 = warp; i0 < most; i0 += W * AT_ONCE) {
        float w[AT_ONCE];
        float4 y[AT_ONCE][R];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int i = i0 + k * W, at = off + i * stride + (i ? 0 : extra);
            const float2 x = i < count ? __ldcg(reinterpret_cast<const float2*>(from + at + D)) : make_float2(-INFINITY, 0.f);
            w[k] = x.x == -INFINITY ? 0.f : ex2(x.x - m);
            l = fmaf(w[k], x.y, l);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float* a = from + __shfl_sync(0xffffffffu, at, r) + lane * V;
                const bool in = __shfl_sync(0xffffffffu, i < count, r);
                y[k][r] = make_float4(0.f, 0.f, 0.f, 0.f);
                if constexpr (V == 4) {
                    if (in) y[k][r] = __ldcg(reinterpret_cast<const float4*>(a));
                } else {
                    if (in) {
                        const float2 z = __ldcg(reinterpret_cast<const float2*>(a));
                        y[k][r].x = z.x, y[k][r].y = z.y;
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float wr = __shfl_sync(0xffffffffu, w[k], r);
                o[r][0] = fmaf(wr, y[k][r].x, o[r][0]), o[r][1] = fmaf(wr, y[k][r].y, o[r][1]);
                if constexpr (V == 4) o[r][2] = fmaf(wr, y[k][r].z, o[r][2]), o[r][3] = fmaf(wr, y[k][r].w, o[r][3]);
            }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r < rows)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[r * D + lane * V + v] = o[r][v];
    if (lane < rows) ml[lane] = make_float2(m, l);
}

template <int D, typename T, int R>
struct AttnLayout {
    static constexpr int TB = cache_tile_bytes(D), STAGE = TS * TB;
    static constexpr int RING = W * NS * STAGE;
    static constexpr int ACC = W * R * D * 4;  // the warps' sums, over the ring
    static constexpr int OFF_BAR = RING > ACC ? RING : ACC;
    static constexpr int OFF_ML = OFF_BAR + W * NS * 8;
    static constexpr int OFF_SCAN = OFF_ML + W * R * 8;  // error word, last-arrival flag, start of the run, warps' totals
    static constexpr int BYTES = OFF_SCAN + 32 + W * 4;
};

// NR groups of 8 columns; E = 2: a row in every column, E = 1 (up to 4 rows): in the even columns only,
// which saves the arithmetic of the others (a lane holds two neighbouring columns of every product).
// CTAs that an SM holds, by the registers that a tile's sums and operands take.  f32 rows, up to 4 of them, at 3 and 4
// CTAs: one sequence of 100000 tokens, 16 heads of 128, 84.5 and 99 us, 16 of 500 to 4000 tokens 49.5 and 56 us.
constexpr int held_at(int nr, int e, bool bf16) { return nr == 2 ? 2 : e == 2 || !bf16 ? 3 : 4; }
template <int NR, int E>
constexpr int rows_of_tile() { return NR * 4 * E; }

// PRE: the prefix's launch.  As a parameter of the launch it cost registers: 64 sequences after a prefix 88.0 us for 85.3.
template <int D, typename T, int NR, int E, bool PRE>
__global__ void __launch_bounds__(W * 32, held_at(NR, E, sizeof(T) == 2)) cache_attn_kernel(const AttnParams p) {
    constexpr int R = rows_of_tile<NR, E>();
    using L = AttnLayout<D, T, R>;
    using At = TileAt<D>;
    constexpr int G = D / 32;
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int NP = SPLIT ? 2 : 1;  // f16 parts of q and of p
    constexpr int PER = 16 / sizeof(T);
    constexpr Codes KX = SPLIT ? Codes::kHigh : Codes::kMid, VX = SPLIT ? Codes::kHalf : Codes::kCentred;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR) + warp * NS;
    float2* sml = reinterpret_cast<float2*>(smem + L::OFF_ML);      // [W][R]
    int* sint = reinterpret_cast<int*>(smem + L::OFF_SCAN);
    int* serr = sint;
    uint8_t* ring = smem + warp * NS * L::STAGE;
    const int TG = p.Tq * p.group, HT = p.c.heads * p.tiles;
    constexpr bool pre = PRE;
    if (lane == 0)
        for (int i = 0; i < NS; ++i) mbar_init(bar + i, 1);
    if (threadIdx.x == 0) *serr = 0;
    fence_mbar_init();

    if (pre) asm volatile("griddepcontrol.launch_dependents;");  // the sequences' launch may fill what this one leaves free

    // ---- the run: units [pos, end) of the items in the order (sequence, kv head, row tile); each item begins
    // with `start` units that stand for no tokens
    // An item's tokens: the prefix's where it has no launch of its own, to the end of their last tile, then
    // the sequence's.
    const int lead = p.lead, lead_end = lead ? p.prefix_len : 0;
    const int most = p.c.width * p.c.tiles * kCacheTile;  // own tokens that the table has entries for
    const int start = pre ? 0 : kStart;
    auto units_of = [&](int n) {
        const int len = pre ? p.prefix_len : lead + min(max(p.lengths[n], 0), most);
        return start + max(1, (len + UNIT - 1) / UNIT);
    };
    int run, pos, end, seq = 0, base = 0;  // base: units before sequence seq
    if (pre) {
        run = p.pre_run;
        pos = blockIdx.x * run;
        end = min(pos + run, HT * p.pre_units);
        __syncthreads();
    } else {
        const int each = (p.N + W * 32 - 1) / (W * 32), n0 = min(p.N, (int)threadIdx.x * each), n1 = min(p.N, n0 + each);
        int sum = 0;
        for (int n = n0; n < n1; ++n) sum += units_of(n);
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) sint[8 + warp] = upto;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) upto += sint[8 + w];
            total += sint[8 + w];
        }
        total *= HT;
        run = max((total + (int)gridDim.x - 1) / (int)gridDim.x, start + 1);
        pos = blockIdx.x * run;
        end = min(pos + run, total);
        upto *= HT;
        int before = upto - sum * HT;
        if (pos >= before && pos < upto) {  // one thread holds the sequence in which the run begins
            int n = n0;
            for (int u; pos >= before + (u = units_of(n) * HT); ++n) before += u;
            sint[2] = n;
            sint[3] = before;
        }
        __syncthreads();
        seq = sint[2];
        base = sint[3];
    }
    if (pos >= end) return;
    int slot = 0;  // of the warp's ring, and the parity of its phase
    uint32_t parity = 0;
    while (pos < end) {
    // ---- the item, and what the run holds of it
    int units = pre ? p.pre_units : units_of(seq);
    while (!pre && pos >= base + HT * units) base += HT * units, ++seq, units = units_of(seq);
    const int item = (pos - base) / units, item_pos = base + item * units;
    const int h = item / p.tiles, rt = item % p.tiles;
    pos = max(pos, item_pos + start);
    if (pos >= end) break;
    const int u0 = pos - item_pos - start, u1 = min(units - start, u0 + end - pos);
    const int cta_first = (item_pos + start) / run, cta_last = (item_pos + units - 1) / run;
    pos += u1 - u0;
    const int rows = min(R, (pre ? p.N * TG : TG) - rt * R);
    // row r of the tile: sequence, query, head; the number of keys it sees in this segment
    auto row_of = [&](int r, int& n, int& q, int& hq) {
        int x = rt * R + r;
        n = pre ? x / TG : seq;
        if (pre) x -= n * TG;
        q = x / p.group;
        hq = h * p.group + x % p.group;
    };
    const int len = pre ? p.prefix_len : max(p.lengths[seq], 0);
    auto row_at = [&](int nr, int e) { return E == 2 ? 8 * nr + 2 * t + e : 4 * nr + t; };  // of the lane's column e
    auto limit_of = [&](int r) {
        if (r >= rows) return 0;
        return pre ? len : lead + min(max(len - p.Tq + (rt * R + r) / p.group + 1, 0), most);
    };
    // Tokens that the table has no entries for are left out; the queries still count from the length.
    if (!pre && len > most && threadIdx.x == 0) atomicExch(p.err, kCacheErrorPage);
    const int c0 = u0 * UNIT, c1 = min(u1 * UNIT, limit_of(rows - 1));  // later rows see more
    const int steps = c1 > c0 ? (c1 - c0 + STEP - 1) / STEP : 0;
    const int mine = steps > warp ? (steps - warp + W - 1) / W : 0;
    const int tile_end = (c1 + kCacheTile - 1) / kCacheTile;

    // ---- q: column g of the products, channels 32 j + 8 t .. + 8 of each group j, as it lies in memory;
    // asked for before the copies, whose bytes would be ahead of it
    uint4 raw[NR][G][8 / PER];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        const int r = E == 2 ? 8 * nr + g : 4 * nr + g / 2;
        const bool live = r < rows && (E == 2 || g % 2 == 0);
        int n = 0, q = 0, hq = 0;
        if (live) row_of(r, n, q, hq);
        const T* src = static_cast<const T*>(p.q) + n * p.qs[0] + q * p.qs[1] + hq * p.qs[2] + 8 * t;
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 8 / PER; ++i) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (live && p.q_vec) {  // every row starts on 16 bytes
                    w = __ldg(reinterpret_cast<const uint4*>(src + 32 * j) + i);
                } else if (live) {
                    const T* e = src + 32 * j + PER * i;
                    if constexpr (SPLIT) {
                        w = make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]), __float_as_uint(e[3]));
                    } else {
                        const uint16_t* b = reinterpret_cast<const uint16_t*>(e);
                        w = make_uint4(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16, b[4] | (uint32_t)b[5] << 16,
                                       b[6] | (uint32_t)b[7] << 16);
                    }
                }
                raw[nr][j][i] = w;
            }
    }

    // ---- copies.  Lane l holds the place of tile l % TS of the warp's step (window) + l / TS in the
    // pool: kNoPage where the table has no page for it, kPast where the range has no such tile.
    auto place_of = [&](int step) -> int {
        const int tl = c0 / kCacheTile + ((step + lane / TS) * W + warp) * TS + lane % TS;
        if (tl >= tile_end) return kPast;
        const bool shared = pre || tl * kCacheTile < lead;
        const int at = shared ? tl : tl - lead / kCacheTile;
        const int slot = p.tiles_inv ? (int)__umulhi((uint32_t)at, p.tiles_inv) : at;
        int page = -1;
        if (slot < (shared ? p.prefix_width : p.c.width))
            page = shared ? p.prefix_pages[slot] : p.c.table[seq * p.c.table_stride + slot];
        return page >= 0 && page < p.c.pages ? (page * p.c.heads + h) * p.c.tiles + at - slot * p.c.tiles : kNoPage;
    };
    int win = place_of(0), win_next = kPast;
    uint32_t have_of = 0;  // TS bits for each slot: the tiles that its copy brings
    auto issue = [&](int step, int slot) {  // the warp's step'th
        if (step > 0 && step % WIN == 0) win = win_next;
        if (step % WIN == WIN / 2) win_next = place_of(step - step % WIN + WIN);
        int at[TS];
        uint32_t m = 0;
        bool row = true;  // the tiles are neighbours
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            at[i] = __shfl_sync(0xffffffffu, win, (step % WIN) * TS + i);
            m |= (uint32_t)(at[i] >= 0) << i;
            row = row && at[i] == at[0] + i;
        }
        have_of = (have_of & ~(((1u << TS) - 1) << (slot * TS))) | m << (slot * TS);
        if (lane == 0) {
            uint8_t* dst = ring + slot * L::STAGE;
            mbar_arrive_expect_tx(bar + slot, __popc(m) * L::TB);
            if (row && m == (1u << TS) - 1) {
                bulk_load(dst, p.c.pool + (int64_t)at[0] * L::TB, TS * L::TB, bar + slot);
            } else {
#pragma unroll
                for (int i = 0; i < TS; ++i) {
                    if (at[i] >= 0) bulk_load(dst + i * L::TB, p.c.pool + (int64_t)at[i] * L::TB, L::TB, bar + slot);
                    if (at[i] == kNoPage) atomicExch(p.err, kCacheErrorPage);
                }
            }
        }
        __syncwarp();
    };
    int issued = 0;
    for (; issued < min(NS, mine); ++issued) issue(issued, slot + issued < NS ? slot + issued : slot + issued - NS);

    // ---- q as operands
    uint32_t qf[NR][NP][G][4];
    // sums of q over the groups / f as three bf16 parts, in the odd places (the minima's) of the
    // operand for the (scale, minimum) words: group t
    uint32_t qm[NR][3];
    // the scale goes into f, which stays positive.  Where a row's f would leave f32, all rows of the tile take f 2^-kLift
    // and scores 2^kLift as large, by the path of masked steps.
    const float sign = p.scale > 0.f ? 1.f : p.scale < 0.f ? -1.f : 0.f;
    const float fscale = sign != 0.f ? fabsf(p.scale) * kLog2e : 1.f;
    float f[NR][E];  // of the columns 2 t, 2 t + 1: score = f * inner
    int fe[NR];      // of column g: f = fscale 2^fe
    bool lift = false;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        float x[G][8];
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 8 / PER; ++i) {
                const uint32_t u[4] = {raw[nr][j][i].x, raw[nr][j][i].y, raw[nr][j][i].z, raw[nr][j][i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (SPLIT) x[j][4 * i + k] = __uint_as_float(u[k]) * sign;
                    else x[j][2 * k] = bf16_lo(u[k]) * sign, x[j][2 * k + 1] = bf16_hi(u[k]) * sign;
                }
            }
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // top < 2^e; q 2^(14 - e) fits f16; score = f inner undoes it and the unit of the codes
        int e = (int)(__float_as_uint(top) >> 23) - 126;
        e = top == 0.f ? 0 : min(max(e, -112), 128);
        const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        constexpr int unit = KX == Codes::kHigh ? 18 : 20;  // log2 of code_unit<KX>(0)
        fe[nr] = unit - 14 + e;
        lift = lift || fe[nr] + (int)(__float_as_uint(fscale) >> 23) - 127 >= 126;
        float mine_sum = 0.f;
#pragma unroll
        for (int j = 0; j < G; ++j) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] *= up, sum += x[j][i];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (t == j) mine_sum = sum / code_unit<KX>(0);
            // the operands of the two products of a group, in the order of code_operands
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                static_assert(code_unit<KX>(0) == code_unit<KX>(1), "the keys' codes have one unit");
                if constexpr (SPLIT) split_f16x2(x[j][i], x[j][i + 4], qf[nr][0][j][i], qf[nr][NP - 1][j][i]);
                else qf[nr][0][j][i] = pack_f16x2(x[j][i], x[j][i + 4]);
            }
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            qm[nr][i] = pack_bf16x2(0.f, mine_sum);
            mine_sum -= bf16_hi(qm[nr][i]);
        }
    }
    lift = __any_sync(0xffffffffu, lift);
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        const float fr = ldexpf(fscale, fe[nr] - (lift ? kLift : 0));
#pragma unroll
        for (int e = 0; e < E; ++e) f[nr][e] = __shfl_sync(0xffffffffu, fr, (2 * t + e) * 4);
    }
    const int clear = lift ? -1 : min(limit_of(0), c1);  // steps that end here need no mask; -1: scores times 2^kLift

    float acc[NR][G][2][4];  // [group][channels 4 g + 0, 1 | 2, 3]: (ch 0, row 2t), (0, 2t+1), (1, 2t), (1, 2t+1)
    float omin[NR][E][G];    // f32: sum p (min + 7.5 scale) of this lane's tokens
    // bf16: sum p scale, sum p min: lanes g = 2 j, 2 j + 1 hold group j.  They grow with every token and are taken from
    // each other, so they are added up in f32 (a step's in the tensor cores, whose sums truncate).
    float pacc[NR][E];
    float l[NR][E], top[NR][E];      // sums; largest inner score of the lane
    // p = 2^(f (inner - ref) - kSlack) <= 1; the inner score at which ref is raised.  The difference comes first: it is
    // exact near ref, while f ref has a rounding of its own, of any size where the scores are large.
    float ref[NR][E], bar_[NR][E];
    float mult[NR][E][G];            // r = p scale mult, a power of two for each row and group
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[nr][j][i / 4][i % 4] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            l[nr][e] = ref[nr][e] = pacc[nr][e] = 0.f;
            top[nr][e] = bar_[nr][e] = -INFINITY;
#pragma unroll
            for (int j = 0; j < G; ++j) omin[nr][e][j] = 0.f, mult[nr][e][j] = kMostMult;
        }
    }

    // ---- the steps
    int done = 0;
    for (; done < mine; ++done) {
        if (!__all_sync(0xffffffffu, mbar_wait(bar + slot, parity, serr, kCacheWaitFull))) break;
        const uint8_t* st = ring + slot * L::STAGE;
        const uint32_t have = have_of >> (slot * TS) & ((1u << TS) - 1);
        const int tok0 = c0 + (done * W + warp) * STEP;
        const bool gap = tok0 < lead && tok0 + STEP > lead_end;  // holds the end of the prefix's last tile
        const bool masked = tok0 + STEP > clear || have != (1u << TS) - 1 || gap;
        if (masked) {  // what the groups of tokens that are not there hold is not a number that may be used
            // Drafted tokens that the tile's first rows do not see: a NaN group of their values would reach those rows as
            // 0 * NaN.  It is put into the sums of the rows that see the token instead.
            const int all_see = limit_of(0);
            if (tok0 + STEP > all_see && all_see < c1) {
                static_assert(STEP == 32, "a lane for each token of a step");
                const int at = tok0 + lane;
                const bool asked = at >= all_see && at < c1 && (have >> (lane / kCacheTile) & 1);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    uint32_t* word = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(st) + lane / kCacheTile * L::TB +
                                                                 At::value_group(lane % kCacheTile, j));
                    const float low = group_min(*word);
                    const bool nan = asked && low != low;
                    const unsigned who = __ballot_sync(0xffffffffu, nan);
                    if (who == 0) continue;
                    if (nan) *word = 0u;
                    const int first = tok0 + __ffs(who) - 1;
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (limit_of(row_at(nr, e)) > first)
#pragma unroll
                                for (int i = e; i < 8; i += 2) acc[nr][j][i / 4][i % 4] = NAN;
                }
            }
#pragma unroll
            for (int i = 0; i < TS; ++i)
                for (int w = lane; w < 2 * kCacheTile * G; w += 32) {
                    const int tok = w / G % kCacheTile;
                    const int at = tok0 + i * kCacheTile + tok;
                    if (!(have >> i & 1) || at >= c1 || (at >= lead_end && at < lead))
                        *reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(st) + i * L::TB +
                                                     (w < kCacheTile * G ? At::key_group(tok, w % G) : At::value_group(tok, w % G))) = 0u;
                }
            fence_proxy_async_smem();  // the slot's next copy comes after these writes
            __syncwarp();
        }

        float s[TS][NR][2 * E];  // token g: columns 2t (, 2t + 1), then token g + 8; inner scores, then p
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const uint8_t* tile = st + i * L::TB;
            const Words<G> ka = lds_words<G>(tile + At::key_word(g, t, 0)), kb = lds_words<G>(tile + At::key_word(g + 8, t, 0));
            const Words<G> pa = lds_words<G>(tile + At::key_group(g, 0)), pb = lds_words<G>(tile + At::key_group(g + 8, 0));
            // sum_j min_j sum(q_j): the (scale, minimum) words of group t as they are
            const uint32_t wa = *reinterpret_cast<const uint32_t*>(tile + At::key_group(g, t % G));
            const uint32_t wb = *reinterpret_cast<const uint32_t*>(tile + At::key_group(g + 8, t % G));
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float c[4];
                mma_bf16_k8_zero(c, wa, wb, qm[nr][0]);
                mma_bf16_k8(c, wa, wb, qm[nr][1]);
                mma_bf16_k8(c, wa, wb, qm[nr][2]);
#pragma unroll
                for (int e = 0; e < E; ++e) s[i][nr][e] = c[e], s[i][nr][E + e] = c[2 + e];
            }
#pragma unroll
            for (int j = 0; j < G; ++j) {
                uint32_t a[4], b[4];
                code_operands<KX>(ka.w[j], a);
                code_operands<KX>(kb.w[j], b);
                const float sa = group_scale(pa.w[j]), sb = group_scale(pb.w[j]);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float c[4];
                    const uint32_t* q = qf[nr][0][j];
                    mma_f16_zero(c, a[0], b[0], a[1], b[1], q[0], q[1]);
                    mma_f16(c, a[2], b[2], a[3], b[3], q[2], q[3]);
                    if constexpr (SPLIT) {
                        q = qf[nr][NP - 1][j];
                        mma_f16(c, a[0], b[0], a[1], b[1], q[0], q[1]);
                        mma_f16(c, a[2], b[2], a[3], b[3], q[2], q[3]);
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        s[i][nr][e] = fmaf(sa, c[e], s[i][nr][e]);
                        s[i][nr][E + e] = fmaf(sb, c[2 + e], s[i][nr][E + e]);
                    }
                }
            }
        }
        // tokens that a row does not see, or that are not there
        if (masked) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int lim = min(limit_of(row_at(nr, e)), c1);
#pragma unroll
                    for (int i = 0; i < TS; ++i)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int tok = tok0 + i * kCacheTile + g + 8 * b;
                            if (!(have >> i & 1) || tok >= lim || (tok >= lead_end && tok < lead)) s[i][nr][b * E + e] = -INFINITY;
                            if (clear < 0) s[i][nr][b * E + e] *= (float)(1ll << kLift);
                        }
                }
        }
        bool raise = false;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float m = top[nr][e];
#pragma unroll
                for (int i = 0; i < TS; ++i) m = fmaxf(m, fmaxf(s[i][nr][e], s[i][nr][E + e]));
                top[nr][e] = m;
                raise = raise || m > bar_[nr][e];
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float m = over_g_max(top[nr][e]);
                    const float to = m == -INFINITY ? 0.f : m;
                    // p, and with it what has been summed, shrinks by c; mult grows by the power of two in it
                    const float by = bar_[nr][e] == -INFINITY ? 0.f : fminf((to - ref[nr][e]) * f[nr][e], 400.f);
                    const float c = ex2(-by), rest = ex2(floorf(by) - by);
                    ref[nr][e] = to;
                    bar_[nr][e] = m + kSlack / f[nr][e];
                    l[nr][e] *= c;
                    pacc[nr][e] *= c;
#pragma unroll
                    for (int j = 0; j < G; ++j) {
                        if constexpr (SPLIT) omin[nr][e][j] *= c;
                        const int bits = (int)(__float_as_uint(mult[nr][e][j]) >> 23) + (int)by, past = max(bits - kMostMultBits, 0);
                        mult[nr][e][j] = __uint_as_float((uint32_t)(bits - past) << 23);
                        if (done == 0) continue;  // the sums are zero
#pragma unroll
                        for (int i = e; i < 8; i += 2) acc[nr][j][i / 4][i % 4] *= rest * pow2(-past);
                    }
                }
            }
        }
        // p, relative to ref
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < TS; ++i) {
                    s[i][nr][e] = ex2(fmaf(s[i][nr][e] - ref[nr][e], f[nr][e], -kSlack));
                    s[i][nr][E + e] = ex2(fmaf(s[i][nr][E + e] - ref[nr][e], f[nr][e], -kSlack));
                    l[nr][e] += s[i][nr][e] + s[i][nr][E + e];
                }
        // r = p scale mult of tile i as operands, and the largest of them
        uint32_t rw[NR][G][2][NP];  // tokens g and g + 8
        auto weigh = [&](int i) {
            const uint8_t* tile = st + i * L::TB;
            const Words<G> va = lds_words<G>(tile + At::value_group(g, 0)), vb = lds_words<G>(tile + At::value_group(g + 8, 0));
            float most = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const float sa = group_scale(va.w[j]), sb = group_scale(vb.w[j]);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float ra[2] = {0.f, 0.f}, rb[2] = {0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        ra[e] = s[i][nr][e] * sa * mult[nr][e][j];
                        rb[e] = s[i][nr][E + e] * sb * mult[nr][e][j];
                        most = max3(most, ra[e], rb[e]);
                    }
                    if constexpr (SPLIT) {
                        split_f16x2(ra[0], ra[1], rw[nr][j][0][0], rw[nr][j][0][NP - 1]);
                        split_f16x2(rb[0], rb[1], rw[nr][j][1][0], rw[nr][j][1][NP - 1]);
                    } else {
                        rw[nr][j][0][0] = pack_f16x2(ra[0], ra[1]);
                        rw[nr][j][1][0] = pack_f16x2(rb[0], rb[1]);
                    }
                }
            }
            return most;
        };
        auto lower = [&](int i) {  // mult of the rows and groups whose r left f16's range
            const uint8_t* tile = st + i * L::TB;
            const Words<G> va = lds_words<G>(tile + At::value_group(g, 0)), vb = lds_words<G>(tile + At::value_group(g + 8, 0));
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int j = 0; j < G; ++j) {
                        const float w = fmaxf(s[i][nr][e] * group_scale(va.w[j]), s[i][nr][E + e] * group_scale(vb.w[j]));
                        const float m = fminf(mult[nr][e][j], mult_for(over_g_max(w)));
                        const float c = pow2_inverse(mult[nr][e][j]) * m;
                        mult[nr][e][j] = m;
#pragma unroll
                        for (int x = e; x < 8; x += 2) acc[nr][j][x / 4][x % 4] *= c;
                    }
        };
        float pstep[NR][4];  // the step's part of pacc
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const uint8_t* tile = st + i * L::TB;
            if constexpr (!SPLIT) {  // p in two bf16 parts
                uint32_t w[4];
                group_operands<G>(tile + At::value_group(0, 0), lane, w);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float a0 = s[i][nr][0], a1 = E == 2 ? s[i][nr][E - 1] : 0.f, b0 = s[i][nr][E], b1 = E == 2 ? s[i][nr][2 * E - 1] : 0.f;
                    const uint32_t ha = pack_bf16x2(a0, a1), hb = pack_bf16x2(b0, b1);
                    if (i == 0) mma_bf16_zero(pstep[nr], w, transpose8x8(ha), transpose8x8(hb));
                    else mma_bf16(pstep[nr], w, transpose8x8(ha), transpose8x8(hb));
                    a0 -= bf16_lo(ha), b0 -= bf16_lo(hb);
                    if constexpr (E == 2) a1 -= bf16_hi(ha), b1 -= bf16_hi(hb);
                    mma_bf16(pstep[nr], w, transpose8x8(pack_bf16x2(a0, a1)), transpose8x8(pack_bf16x2(b0, b1)));
                    if (i == TS - 1)
#pragma unroll
                        for (int e = 0; e < E; ++e) pacc[nr][e] += pstep[nr][e];
                }
            }
            if (__any_sync(0xffffffffu, weigh(i) > kMostF16)) {
                lower(i);
                weigh(i);
            }
            // codes of channels 4 g .. + 3 of every group, of tokens 2 t, 2 t + 1 (+ 8): 16 bits each
            uint32_t x[2][G];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Words<G> w = lds_words<G>(tile + At::value_half(8 * u + 2 * t, g, 0));
#pragma unroll
                for (int j = 0; j < G; j += 2) {
                    x[u][j] = __byte_perm(w.w[j / 2], w.w[G / 2 + j / 2], 0x5410);
                    x[u][j + 1] = __byte_perm(w.w[j / 2], w.w[G / 2 + j / 2], 0x7632);
                }
            }
            const Words<G> va = lds_words<G>(tile + At::value_group(g, 0)), vb = lds_words<G>(tile + At::value_group(g + 8, 0));
#pragma unroll
            for (int j = 0; j < G; ++j) {
                uint32_t y[4], z[4];
                code_operands<VX>(x[0][j], y);
                code_operands<VX>(x[1][j], z);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    if constexpr (SPLIT) {
                        const float sa = group_scale(va.w[j]), sb = group_scale(vb.w[j]);
                        const float ma = fmaf(7.5f, sa, group_min(va.w[j])), mb = fmaf(7.5f, sb, group_min(vb.w[j]));
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            omin[nr][e][j] = fmaf(s[i][nr][e], ma, fmaf(s[i][nr][E + e], mb, omin[nr][e][j]));
                    }
#pragma unroll
                    for (int np = 0; np < NP; ++np) {
                        const uint32_t c0_ = transpose8x8(rw[nr][j][0][np]), c1_ = transpose8x8(rw[nr][j][1][np]);
                        mma_f16(acc[nr][j][0], y[0], y[1], z[0], z[1], c0_, c1_);
                        mma_f16(acc[nr][j][1], y[2], y[3], z[2], z[3], c0_, c1_);
                    }
                }
            }
        }
        __syncwarp();  // the slot has been read
        if (issued < mine) issue(issued, slot), ++issued;
        if (++slot == NS) slot = 0, parity ^= 1u;
    }
    // A warp that gave up at a wait still owns the copies it issued: let them land first.
    for (; done < issued; ++done) {
        mbar_drain(bar + slot, parity);
        if (++slot == NS) slot = 0, parity ^= 1u;
    }
    __syncthreads();

    // ---- the warps' sums, relative to the largest score of the warp, to shared memory
    float* sacc = reinterpret_cast<float*>(smem) + warp * R * D;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int r = row_at(nr, e);
            const float inner = over_g_max(top[nr][e]), m = inner * f[nr][e];  // -inf: nothing seen
            const float c = m == -INFINITY ? 0.f : ex2(fmaf(ref[nr][e] - inner, f[nr][e], kSlack));
            const float sum = over_g_sum(l[nr][e]) * c;
            float om[G];
#pragma unroll
            for (int j = 0; j < G; ++j) {
                if constexpr (SPLIT) om[j] = over_g_sum(omin[nr][e][j]);
                else om[j] = fmaf(8.f, __shfl_sync(0xffffffffu, pacc[nr][e], 8 * j + t),
                                  __shfl_sync(0xffffffffu, pacc[nr][e], 8 * j + 4 + t));
            }
            if (r < rows) {
                if (g == 0) sml[warp * R + r] = make_float2(m, sum);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    const float v = pow2_inverse(mult[nr][e][j]);
                    float4 o;
                    o.x = fmaf(acc[nr][j][0][e] * code_unit<VX>(0), v, om[j]) * c;
                    o.y = fmaf(acc[nr][j][0][e + 2] * code_unit<VX>(1), v, om[j]) * c;
                    o.z = fmaf(acc[nr][j][1][e] * code_unit<VX>(2), v, om[j]) * c;
                    o.w = fmaf(acc[nr][j][1][e + 2] * code_unit<VX>(3), v, om[j]) * c;
                    *reinterpret_cast<float4*>(sacc + r * D + 32 * j + 4 * g) = o;
                }
            }
        }
    __syncthreads();

    // ---- the CTA's sums
    const float* all = reinterpret_cast<const float*>(smem);
    auto joined = [&](int r, int d, float& m, float& sum) {  // of the warps, row r, channels d .. d + 3
        m = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, sml[w * R + r].x);
        sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 ml = sml[w * R + r];
            const float c = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
            const float4 a = *reinterpret_cast<const float4*>(all + (w * R + r) * D + d);
            sum = fmaf(c, ml.y, sum);
            o.x = fmaf(c, a.x, o.x), o.y = fmaf(c, a.y, o.y), o.z = fmaf(c, a.z, o.z), o.w = fmaf(c, a.w, o.w);
        }
        return o;
    };
    constexpr int PR = D + kPartPad;
    auto own_part = [&](int cta, int r) {  // an item begins as the last of a run and goes on as the first of others
        return p.part + ((int64_t)(cta * 2 + (cta == cta_first ? 1 : 0)) * R + r) * PR;
    };
    auto fold = [&](const float* from, int off, int stride, int extra, int count) {
        if (R <= 4 && rows == 1) fold_rows<D, 1>(sacc, sml + warp * R, 1, warp, lane, from, off, stride, extra, count);
        else fold_rows<D, R>(sacc, sml + warp * R, rows, warp, lane, from, off, stride, extra, count);
    };
    const bool whole = cta_first == cta_last;
    if (pre || !whole) {
        for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float m, sum;
            const float4 o = joined(r, d, m, sum);
            float* to = pre ? p.pre_part + ((int64_t)(item * R + r) * p.pre_parts + blockIdx.x - cta_first) * PR
                            : own_part(blockIdx.x, r);
            *reinterpret_cast<float4*>(to + d) = o;
            if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m, sum);
        }
    }
    bool finish = !pre && whole;
    if (!pre && !whole) {  // the CTA that arrives last at the item joins its parts, and leaves the counter at zero
        __syncthreads();
        if (threadIdx.x == 0) {  // the barriers make its fences the whole CTA's
            __threadfence();
            const bool last = atomicAdd(p.counter + cta_first, 1u) == (unsigned)(cta_last - cta_first);
            if (last) p.counter[cta_first] = 0;
            sint[1] = last;
            __threadfence();
        }
        __syncthreads();
        finish = sint[1];
        if (finish) {
            for (int i = lane; i < rows * D; i += 32) sacc[i] = 0.f;
            if (lane < rows) sml[warp * R + lane] = make_float2(-INFINITY, 0.f);
            __syncwarp();
            fold(p.part, (cta_first * 2 * R + lane) * PR, 2 * R * PR,
                            R * PR, cta_last - cta_first + 1);
            __syncthreads();
        }
    }
    if (finish) {
        if (p.pre_units) {
            asm volatile("griddepcontrol.wait;" ::: "memory");  // the prefix's launch has ended
            const int x = seq * TG + rt * R + min(lane, rows - 1), it = h * p.pre_tiles + x / p.pre_rows;
            const int first = it * p.pre_units / p.pre_run, last = ((it + 1) * p.pre_units - 1) / p.pre_run;
            __syncwarp();
            fold(p.pre_part,
                            (it * p.pre_rows + x % p.pre_rows) * p.pre_parts * PR, PR, 0, last - first + 1);
            __syncthreads();
        }
        for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float m, sum;
            const float4 o = joined(r, d, m, sum);
            int n, q, hq;
            row_of(r, n, q, hq);
            const int64_t row = ((int64_t)n * p.Tq + q) * p.H + hq;
            const bool empty = sum == 0.f;
            const float inv = empty ? 0.f : 1.f / sum;
            T* out = static_cast<T*>(p.out) + row * D + d;
            out[0] = from_f32<T>(o.x * inv), out[1] = from_f32<T>(o.y * inv);
            out[2] = from_f32<T>(o.z * inv), out[3] = from_f32<T>(o.w * inv);
            if (d == 0) {
                if (p.row_max) p.row_max[row] = empty ? 0.f : m * kLn2;
                if (p.row_sum) p.row_sum[row] = empty ? 1.f : sum;
            }
        }
    }
    fence_proxy_async_smem();  // the sums lie where the next item's copies go
    __syncthreads();
    }
    if (threadIdx.x == 0 && *serr != 0) atomicExch(p.err, *serr);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Segment {  // the prefix, or the sequences' own tokens
    int nr, e, rows, tiles;
    int64_t units, grid;  // of all items, at most
};

// `rows` rows share the tokens of an item.
Segment segment_of(int64_t rows, int64_t items, int64_t tokens, int start, bool bf16) {
    Segment s{};
    s.e = rows <= 4 ? 1 : 2;
    // two groups of columns share the codes' operands: 16 rows of 48 sequences 67 us, in two tiles of 8 73 us; 12 rows (six
    // drafts of two heads) 35 us both ways; the prefix of 64 sequences 85.7 and 83.9 us with what follows it (f32 rows
    // take the registers twice)
    s.nr = bf16 && rows > 8 ? 2 : 1;
    s.rows = 4 * s.e * s.nr;
    s.tiles = (int)ceil_div(rows, s.rows);
    s.units = items * s.tiles * (start + (tokens > UNIT ? ceil_div(tokens, UNIT) : 1));
    // As many CTAs as the GPU holds, in more rounds of them where a run would be longer than kRun units, as far as the
    // counters go: the tensor cores' sums truncate, and each is a run's.
    const int64_t held = 148 * held_at(s.nr, s.e, bf16), runs = ceil_div(s.units, start + 1);
    const int64_t rounds = std::min(ceil_div(s.units, held * kRun), (int64_t)kCounterBytes / 4 / held);
    s.grid = std::min(runs, held * rounds);
    return s;
}

struct Plan {
    Segment own, pre;
    int lead, pre_units, pre_run, pre_parts;
    size_t off_part, off_pre, bytes;
};

Plan plan_of(const dbl_relay_cache_attention_args* a) {
    Plan L{};
    const int64_t TG = a->queries * (a->heads / a->cache.kv_heads), H = a->cache.kv_heads, N = a->n_seq;
    const bool bf16 = a->dtype == DBL_BF16;
    const size_t row = (size_t)(a->cache.head_dim + kPartPad) * 4;
    // A prefix has a launch of its own where reading it with every sequence's own tokens costs more.  Measured at 16
    // heads of 128, 1024 own tokens, apart and with them: 64 sequences, prefix 512: 70 and 69 us, 1024: 71 and 85, 4096:
    // 85 and 183; 16 sequences, 512: 30 and 27, 1024: 31 and 31.6, 4096: 35 and 55; 4 sequences, 1024: 18 and 17, 4096:
    // 23.6 and 22.6.
    const bool apart = N >= 4 && N * H * a->prefix_len >= kApart;
    L.lead = a->prefix_len > 0 && !apart ? (int)(ceil_div(a->prefix_len, kCacheTile) * kCacheTile) : 0;
    L.own = segment_of(TG, N * H, L.lead + a->table_width * a->cache.page_size, kStart, bf16);
    L.off_part = kCounterBytes;
    L.off_pre = L.off_part + (size_t)(L.own.grid * 2 * L.own.rows) * row;
    L.bytes = L.off_pre;
    if (apart) {
        L.pre = segment_of(N * TG, H, a->prefix_len, 0, bf16);
        L.pre_units = (int)ceil_div(a->prefix_len, UNIT);
        L.pre_run = (int)ceil_div(L.pre.units, L.pre.grid);
        L.pre.grid = ceil_div(L.pre.units, L.pre_run);
        L.pre_parts = (L.pre_units + L.pre_run - 2) / L.pre_run + 1;
        L.bytes += (size_t)(H * L.pre.tiles * L.pre.rows * L.pre_parts) * row;
    }
    return L;
}

int attn_validate(const dbl_relay_cache_attention_args* a) {
    if (!a) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: null args");
    int rc = cache_validate(&a->cache, "relay cache attention");
    if (rc == DBL_OK)
        rc = cache_check_table(a->page_table, a->n_seq, a->table_width, a->table_stride, "relay cache attention");
    if (rc != DBL_OK) return rc;
    if (a->queries <= 0 || a->heads <= 0)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: queries and heads must be positive");
    if (a->heads % a->cache.kv_heads)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: heads must be a multiple of kv_heads");
    if (a->dtype != DBL_F32 && a->dtype != DBL_BF16)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: dtype must be f32 or bf16");
    if (a->prefix_len < 0 || a->prefix_len > kMostTokens || a->prefix_width < 0 || a->prefix_width > 0x7fffffff)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: prefix_len out of range");
    if (a->prefix_len > 0 && (!a->prefix_pages || a->prefix_width * a->cache.page_size < a->prefix_len))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: prefix_pages must hold prefix_len tokens");
    if (a->queries > 0x7fffffff || a->heads > 0x7fffffff || a->n_seq * a->queries > 0x7fffffff / a->heads ||
        a->table_width * a->cache.page_size > kMostTokens)
        return fail(DBL_ERR_UNSUPPORTED, "relay cache attention: sizes exceed 32-bit limits");
    return DBL_OK;
}

template <int D, typename T, int NR, int E, bool PRE>
int launch_with(const AttnParams& p, int64_t grid, cudaStream_t st) {
    constexpr int smem = AttnLayout<D, T, rows_of_tile<NR, E>()>::BYTES;
    static std::atomic<uint64_t> done{0};
    const int rc = once_per_device(done, [] {
        return cuda_status(
            cudaFuncSetAttribute(cache_attn_kernel<D, T, NR, E, PRE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
            "relay cache attention: cudaFuncSetAttribute");
    });
    if (rc != DBL_OK) return rc;
    // The sequences' launch after the prefix's starts without waiting for it, and waits where it joins its sums.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.pre_units && !p.pre ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, cache_attn_kernel<D, T, NR, E, PRE>, p), "cache_attn_kernel");
}

template <int D, typename T, int NR, int E>
int launch_attn(const AttnParams& p, int64_t grid, cudaStream_t st) {
    return p.pre ? launch_with<D, T, NR, E, true>(p, grid, st) : launch_with<D, T, NR, E, false>(p, grid, st);
}

template <int D>
int launch_segment(AttnParams p, const Segment& s, bool pre, bool bf16, cudaStream_t st) {
    p.pre = pre;
    p.tiles = s.tiles;
    if (!bf16) return s.e == 1 ? launch_attn<D, float, 1, 1>(p, s.grid, st) : launch_attn<D, float, 1, 2>(p, s.grid, st);
    if (s.nr == 2) return launch_attn<D, __nv_bfloat16, 2, 2>(p, s.grid, st);
    return s.e == 1 ? launch_attn<D, __nv_bfloat16, 1, 1>(p, s.grid, st)
                    : launch_attn<D, __nv_bfloat16, 1, 2>(p, s.grid, st);
}

}  // namespace
}  // namespace dbl

extern "C" size_t dbl_relay_cache_attention_workspace_bytes(const dbl_relay_cache_attention_args* a) {
    if (dbl::attn_validate(a) != DBL_OK) return 0;
    return dbl::plan_of(a).bytes;
}

extern "C" int dbl_relay_cache_attention(const dbl_relay_cache_attention_args* a, void* workspace,
                                         size_t workspace_bytes, dbl_stream_t stream) {
    using namespace dbl;
    int rc = attn_validate(a);
    if (rc != DBL_OK) return rc;
    if (!a->q || !a->out || !a->lengths)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: q, out and lengths are required");
    const int D = (int)a->cache.head_dim;
    const int64_t dims[4] = {a->n_seq, a->queries, a->heads, D};
    int64_t qs[4];
    resolve_strides(a->q_stride, dims, 4, qs);
    if (qs[3] != 1) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: the innermost stride of q must be 1");
    const Plan L = plan_of(a);
    if (L.own.units > 0x3fffffff || L.pre.units > 0x3fffffff || L.bytes > ((size_t)1 << 32))
        return fail(DBL_ERR_UNSUPPORTED, "relay cache attention: sizes exceed 32-bit limits");
    if (!workspace || workspace_bytes < L.bytes)
        return fail(DBL_ERR_WORKSPACE, "relay cache attention: workspace of %zu bytes required (got %zu)", L.bytes,
                    workspace_bytes);
    if (!aligned(workspace, 16))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: workspace must be 16-byte aligned");
    AttnParams p{};
    p.c = cache_view(&a->cache, a->page_table, a->table_width, a->table_stride);
    p.q = a->q;
    const int64_t per = 16 / (int64_t)dtype_size(a->dtype);
    p.q_vec = aligned(a->q, 16);
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = qs[i];
        p.q_vec = p.q_vec && qs[i] % per == 0;
    }
    p.lengths = a->lengths;
    p.prefix_pages = a->prefix_pages;
    p.out = a->out;
    p.row_max = a->row_max;
    p.row_sum = a->row_sum;
    p.N = (int)a->n_seq;
    p.Tq = (int)a->queries;
    p.H = (int)a->heads;
    p.group = (int)(a->heads / a->cache.kv_heads);
    p.tiles_inv = p.c.tiles == 1 ? 0u : (uint32_t)(((1ull << 32) + p.c.tiles - 1) / p.c.tiles);
    p.prefix_len = (int)a->prefix_len;
    p.prefix_width = (int)a->prefix_width;
    p.scale = a->scale;
    p.lead = L.lead;
    p.pre_tiles = L.pre.tiles;
    p.pre_rows = L.pre.rows;
    p.pre_units = L.pre_units;
    p.pre_run = L.pre_run;
    p.pre_parts = L.pre_parts;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.counter = reinterpret_cast<unsigned*>(ws);
    p.part = reinterpret_cast<float*>(ws + L.off_part);
    p.pre_part = reinterpret_cast<float*>(ws + L.off_pre);
    rc = device_error_record(&p.err);
    if (rc != DBL_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool bf16 = a->dtype == DBL_BF16;
    if (L.pre_units) {
        rc = D == 128 ? launch_segment<128>(p, L.pre, true, bf16, st) : launch_segment<64>(p, L.pre, true, bf16, st);
        if (rc != DBL_OK) return rc;
    }
    return D == 128 ? launch_segment<128>(p, L.own, false, bf16, st) : launch_segment<64>(p, L.own, false, bf16, st);
}
