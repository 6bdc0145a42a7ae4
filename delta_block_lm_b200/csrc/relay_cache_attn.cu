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
//   * a code needs no conversion: the 16-bit word with the code in its lowest 4 bits is the f16
//     subnormal code * 2^-24, with the code in the next 4 bits 16 times that, so one AND makes the
//     operand register of two codes.  The powers of two go into q (keys) or the output (values).
//     The products' sums drop what lies 24 bits below the largest operand exponent, and a
//     subnormal's counts as 2^-14: that leaves about 17 bits, ample beside p in f16.  For f32 rows
//     the keys' codes are shifted to the top of the mantissa (code * 2^-18, 22 bits) and the values'
//     become normal numbers around zero (code - 8), so that long sums neither drop bits nor cancel.
//   * q is held in f16 relative to a power of two of its own row (bf16 q: exact; f32 q: two f16
//     parts, 22 bits), p scale in f16 relative to a power of two near the row's largest (f32: again
//     two parts).  For bf16 the rounding of p scale, 2^-11, is kept off the values' mean: with r
//     the rounded p scale, o = sum r (code - 7.5) + sum p (min + 7.5 scale), where sum r is one
//     more product, with a row of ones (f32: sum r (code - 8) + sum p (min + 8 scale)).
//   * the scores arrive with tokens in rows and have to leave with tokens along the product's
//     inner dimension: movmatrix transposes the 8 x 8 blocks.
// The running maximum is only raised when a score passes it by 8 (in powers of two), so a step
// usually costs one vote instead of the shuffles of a maximum and the rescaling of the sums.
//
// Work: a CTA takes (kv head, up to 8 NR rows, a range of tokens) of the prefix -- rows of all
// sequences, so that it is read once per head for 8 NR sequences -- or of one sequence.  Its four
// warps take turns at steps of 32 tokens, each with a ring of its own that bulk copies fill.  The
// partial sums of the CTAs of a row go to the workspace, and the one that arrives last merges them.
#include <float.h>

#include "relay_cache.cuh"
#include "tc_ptx.cuh"

namespace dbl {

int cache_check_table(const int32_t* table, int64_t n_seq, int64_t width, int64_t stride, const char* what);

namespace {

constexpr int W = 4;              // warps of a CTA
constexpr int TS = 2;             // tiles of a step
constexpr int STEP = TS * kCacheTile;
constexpr int NS = 3;             // stages of a warp's ring
constexpr int WIN = 32 / TS;      // steps whose page numbers the lanes of a warp hold
constexpr int kCacheWaitFull = 40;  // wait-site code (dbl_device_error)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;     // how far a score may pass the running maximum (powers of two)
constexpr float kMostF16 = 60000.f;             // p scale mult stays below it
constexpr float kMostMult = 1.2676506e30f;      // 2^100
constexpr uint32_t kOnes = 0x3C003C00u;         // two f16 ones

struct AttnParams {
    CacheView c;
    const void* q;
    int64_t qs[3];  // strides of sequence, query and head
    const int32_t *lengths, *prefix_pages;
    void* out;
    float *row_max, *row_sum;
    int N, Tq, H, group, prefix_len, prefix_width;
    float scale;
    int tiles_pre, tiles_own;    // row tiles of a kv head over all sequences, of one sequence
    int splits_pre, splits_own;  // ranges of tokens
    int range_pre, range_own;    // tokens of a range
    float *part, *part_ml;       // [rows, splits, D], [rows, splits, 2]
    unsigned* counter;           // [rows]
    int* err;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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

// The power of two that takes w to 2^13 .. 2^14, and the inverse of a power of two.
__device__ __forceinline__ float mult_for(float w) {
    const int e = min(max((int)(__float_as_uint(w) >> 23), 40), 250);
    return __uint_as_float((uint32_t)(267 - e) << 23);
}
__device__ __forceinline__ float pow2_inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// The operand registers of the 8 codes of w, codes (0, 4), (1, 5), (2, 6), (3, 7), and what they are
// multiplied by to be the codes (kUnit of register i).
enum class Codes { kLow, kHigh, kCentred };
template <Codes C>
__device__ __forceinline__ void code_operands(uint32_t w, uint32_t (&r)[4]) {
    if constexpr (C == Codes::kHigh) {
        r[0] = (w << 6) & 0x03C003C0u, r[1] = (w << 2) & 0x03C003C0u;
        r[2] = (w >> 2) & 0x03C003C0u, r[3] = (w >> 6) & 0x03C003C0u;
    } else {
        r[0] = w & 0x000F000Fu, r[1] = w & 0x00F000F0u;
        r[2] = (w >> 8) & 0x000F000Fu, r[3] = (w >> 8) & 0x00F000F0u;
        if constexpr (C == Codes::kCentred) {  // 1024 + x is the f16 with mantissa x; 1032 = 1024 + 8, 1152 = 1024 + 16 * 8
#pragma unroll
            for (int i = 0; i < 4; ++i)
                asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(r[i] | 0x64006400u), "r"(i & 1 ? 0xE480E480u : 0xE408E408u));
        }
    }
}
template <Codes C>
constexpr float code_unit(int i) {
    return C == Codes::kHigh ? 262144.f : (i & 1 ? 0.0625f : 1.f) * (C == Codes::kLow ? 16777216.f : 1.f);
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

// Merges the S partials of output row `row`; one warp.
template <int D, typename T>
__device__ void merge_row(const AttnParams& p, int64_t row, int S) {
    constexpr int V = D / 32;  // channels of a lane, neighbouring
    const int lane = threadIdx.x & 31;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row * S;
    float m = -INFINITY;
    for (int i = lane; i < S; i += 32) m = fmaxf(m, __ldcg(ml + i).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f, acc[V] = {};
    for (int base = 0; base < S; base += 32) {
        float w = 0.f, li = 0.f;
        if (base + lane < S) {
            const float2 x = __ldcg(ml + base + lane);
            w = x.x == -INFINITY ? 0.f : ex2(x.x - m);
            li = x.y;
        }
        l += w * li;
        const int n = min(32, S - base);
        for (int i = 0; i < n; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            if (wi == 0.f) continue;
            const float* a = p.part + (row * S + base + i) * D + lane * V;
            if constexpr (V == 4) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(a));
                acc[0] = fmaf(wi, x.x, acc[0]), acc[1] = fmaf(wi, x.y, acc[1]);
                acc[2] = fmaf(wi, x.z, acc[2]), acc[3] = fmaf(wi, x.w, acc[3]);
            } else {
                const float2 x = __ldcg(reinterpret_cast<const float2*>(a));
                acc[0] = fmaf(wi, x.x, acc[0]), acc[1] = fmaf(wi, x.y, acc[1]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const bool empty = l == 0.f;
    const float inv = empty ? 0.f : 1.f / l;
    T* out = static_cast<T*>(p.out) + row * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = from_f32<T>(acc[i] * inv);
    if (lane == 0) {
        if (p.row_max) p.row_max[row] = empty ? 0.f : m * kLn2;
        if (p.row_sum) p.row_sum[row] = empty ? 1.f : l;
    }
}

template <int D, typename T, int NR>
struct AttnLayout {
    static constexpr int TB = cache_tile_bytes(D), STAGE = TS * TB;
    static constexpr int RING = W * NS * STAGE;
    static constexpr int ACC = W * 8 * NR * D * 4;  // the warps' sums, over the ring
    static constexpr int OFF_BAR = RING > ACC ? RING : ACC;
    static constexpr int OFF_MASK = OFF_BAR + W * NS * 8;
    static constexpr int OFF_ML = OFF_MASK + W * NS * 4;
    static constexpr int OFF_ROW = OFF_ML + W * 8 * NR * 8;
    static constexpr int OFF_ERR = OFF_ROW + 8 * NR * 8;
    static constexpr int BYTES = OFF_ERR + 16;
};

template <int D, typename T, int NR>
__global__ void __launch_bounds__(W * 32) cache_attn_kernel(const AttnParams p) {
    using L = AttnLayout<D, T, NR>;
    using At = TileAt<D>;
    constexpr int G = D / 32, R = 8 * NR;
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int NP = SPLIT ? 2 : 1;  // f16 parts of q and of p
    constexpr Codes KX = SPLIT ? Codes::kHigh : Codes::kLow, VX = SPLIT ? Codes::kCentred : Codes::kLow;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR) + warp * NS;
    uint32_t* smask = reinterpret_cast<uint32_t*>(smem + L::OFF_MASK) + warp * NS;
    float2* sml = reinterpret_cast<float2*>(smem + L::OFF_ML);      // [W][R]
    int64_t* srow = reinterpret_cast<int64_t*>(smem + L::OFF_ROW);  // output rows
    int* serr = reinterpret_cast<int*>(smem + L::OFF_ERR);
    uint8_t* ring = smem + warp * NS * L::STAGE;

    // ---- the item
    const int TG = p.Tq * p.group;
    int item = blockIdx.x;
    const int n_pre = p.splits_pre * p.tiles_pre * p.c.heads;
    const bool pre = item < n_pre;
    if (!pre) item -= n_pre;
    const int rt = item % (pre ? p.tiles_pre : p.tiles_own);
    item /= pre ? p.tiles_pre : p.tiles_own;
    const int h = item % p.c.heads;
    item /= p.c.heads;
    const int split = pre ? item : item % p.splits_own;
    const int seq = pre ? 0 : item / p.splits_own;
    const int rows = min(R, (pre ? p.N * TG : TG) - rt * R);
    // row r of the tile: sequence, query, head; the number of keys it sees in this segment
    auto row_of = [&](int r, int& n, int& q, int& hq) {
        int x = rt * R + r;
        n = pre ? x / TG : seq;
        if (pre) x -= n * TG;
        q = x / p.group;
        hq = h * p.group + x % p.group;
    };
    const int len = pre ? p.prefix_len : min(max(p.lengths[seq], 0), p.c.width * p.c.tiles * kCacheTile);
    auto limit_of = [&](int r) {
        if (r >= rows) return 0;
        return pre ? len : max(0, len - p.Tq + (rt * R + r) / p.group + 1);
    };
    const int range = pre ? p.range_pre : p.range_own;
    const int c0 = split * range, c1 = min(c0 + range, limit_of(rows - 1));  // later rows see more
    const int all_see = limit_of(0);                                         // tokens below it need no mask
    const int steps = c1 > c0 ? (c1 - c0 + STEP - 1) / STEP : 0;
    const int mine = steps > warp ? (steps - warp + W - 1) / W : 0;
    const int tile_end = (c1 + kCacheTile - 1) / kCacheTile;

    if (lane == 0)
        for (int i = 0; i < NS; ++i) mbar_init(bar + i, 1);
    if (threadIdx.x == 0) *serr = 0;
    fence_mbar_init();
    __syncthreads();

    // ---- copies.  Lane l holds the page of tile l % TS of the warp's step (window) + l / TS.
    auto page_of = [&](int step) -> int {  // of this lane's tile, for the window that begins at `step`
        const int tl = c0 / kCacheTile + ((step + lane / TS) * W + warp) * TS + lane % TS;
        if (tl >= tile_end) return -1;
        if (!pre) return cache_page(p.c, seq, tl);
        const int slot = tl / p.c.tiles;
        const int page = slot < p.prefix_width ? p.prefix_pages[slot] : -1;
        return page < p.c.pages ? page : -1;
    };
    int win = page_of(0), win_next = -1;
    auto issue = [&](int step) {  // the warp's step'th
        if (step > 0 && step % WIN == 0) win = win_next;
        if (step % WIN == WIN / 2) win_next = page_of(step - step % WIN + WIN);
        const int page = __shfl_sync(0xffffffffu, win, (step % WIN) * TS + lane % TS);
        const int tl = c0 / kCacheTile + (step * W + warp) * TS + lane;
        const bool want = lane < TS && tl < tile_end, have = want && page >= 0;
        if (want && !have) atomicExch(p.err, kCacheErrorPage);
        const uint32_t m = __ballot_sync(0xffffffffu, have);
        const int slot = step % NS;
        if (lane == 0) {
            smask[slot] = m;
            mbar_arrive_expect_tx(bar + slot, __popc(m) * L::TB);
        }
        __syncwarp();
        if (have)
            bulk_load(ring + slot * L::STAGE + lane * L::TB, cache_tile<D>(p.c, page, h, tl % p.c.tiles), L::TB,
                      bar + slot);
    };
    int issued = 0;
    for (; issued < min(NS, mine); ++issued) issue(issued);

    // ---- q: column g of the products, channels 32 j + 8 t .. + 8 of each group j
    uint32_t qf[NR][NP][G][4];
    // the scale goes into f, which stays positive
    const float sign = p.scale > 0.f ? 1.f : p.scale < 0.f ? -1.f : 0.f;
    const float fscale = sign != 0.f ? fabsf(p.scale) * kLog2e : 1.f;
    float qsum[NR][2][G], f[NR][2];  // of rows 2 t, 2 t + 1: sums of q over the groups / f; score = f * inner
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        const int r = 8 * nr + g;
        float x[G][8];
        float top = 0.f;
        if (r < rows) {
            int n, q, hq;
            row_of(r, n, q, hq);
            const T* src = static_cast<const T*>(p.q) + n * p.qs[0] + q * p.qs[1] + hq * p.qs[2] + 8 * t;
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = to_f32<T>(src[32 * j + i]) * sign;
        } else {
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // top < 2^e; q 2^(14 - e) fits f16; score = f inner undoes it and the unit of the codes
        int e = (int)(__float_as_uint(top) >> 23) - 126;
        e = top == 0.f ? 0 : min(max(e, -90), 110);
        const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        constexpr int unit = KX == Codes::kHigh ? 18 : 24;  // log2 of code_unit<KX>(0)
        const float fr = __uint_as_float((uint32_t)(127 - 14 + unit + e) << 23) * fscale;
        const float inv = __uint_as_float((uint32_t)(127 + 14 - unit - e) << 23);
        float sum[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += x[j][i];
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            sum[j] = s * inv;
            // the operands of the two products of a group, in the order of code_operands
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float by = up * (code_unit<KX>(i) / code_unit<KX>(0));
                if constexpr (SPLIT) split_f16x2(x[j][i] * by, x[j][i + 4] * by, qf[nr][0][j][i], qf[nr][NP - 1][j][i]);
                else qf[nr][0][j][i] = pack_f16x2(x[j][i] * by, x[j][i + 4] * by);
            }
        }
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) {
            const int from = (2 * t + e2) * 4;
            f[nr][e2] = __shfl_sync(0xffffffffu, fr, from);
#pragma unroll
            for (int j = 0; j < G; ++j) qsum[nr][e2][j] = __shfl_sync(0xffffffffu, sum[j], from);
        }
    }

    float acc[NR][G][2][4];  // [group][channels 4 g + 0, 1 | 2, 3]: (ch 0, row 2t), (0, 2t+1), (1, 2t), (1, 2t+1)
    float omin[NR][2][G];    // sum p min of this lane's tokens
    float racc[NR][4];       // sums of r: lanes g = j hold group j
    float l[NR][2], top[NR][2], ref[NR][2];  // sums; largest inner score of the lane; the reference of p
    float wtop[NR][2], mult[NR][2];          // largest p scale of the lane; r = p scale mult, a power of two
    int lim[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[nr][j][i / 4][i % 4] = 0.f;
        racc[nr][0] = racc[nr][1] = racc[nr][2] = racc[nr][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[nr][e] = wtop[nr][e] = 0.f;
            mult[nr][e] = kMostMult;
            top[nr][e] = ref[nr][e] = -INFINITY;
            lim[nr][e] = limit_of(8 * nr + 2 * t + e);
#pragma unroll
            for (int j = 0; j < G; ++j) omin[nr][e][j] = 0.f;
        }
    }

    // ---- the steps
    int done = 0;
    for (int it = 0; it < mine; ++it) {
        const int slot = it % NS;
        if (!__all_sync(0xffffffffu, mbar_wait(bar + slot, (uint32_t)(it / NS) & 1u, serr, kCacheWaitFull))) break;
        done = it + 1;
        const uint8_t* st = ring + slot * L::STAGE;
        const uint32_t have = smask[slot];
        const int tok0 = c0 + (it * W + warp) * STEP;
        const bool masked = tok0 + STEP > min(all_see, c1) || have != (1u << TS) - 1;

        float s[TS][NR][4];  // (token g, row 2t), (g, 2t+1), (g + 8, 2t), (g + 8, 2t+1); inner scores, then p
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const uint8_t* tile = st + i * L::TB;
            const Words<G> ka = lds_words<G>(tile + At::key_word(g, t, 0)), kb = lds_words<G>(tile + At::key_word(g + 8, t, 0));
            const Words<G> pa = lds_words<G>(tile + At::key_group(g, 0)), pb = lds_words<G>(tile + At::key_group(g + 8, 0));
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) s[i][nr][0] = s[i][nr][1] = s[i][nr][2] = s[i][nr][3] = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) {
                uint32_t a[4], b[4];
                code_operands<KX>(ka.w[j], a);
                code_operands<KX>(kb.w[j], b);
                const float sa = group_scale(pa.w[j]), sb = group_scale(pb.w[j]);
                const float ma = group_min(pa.w[j]), mb = group_min(pb.w[j]);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float c[4] = {};
#pragma unroll
                    for (int np = 0; np < NP; ++np) {
                        const uint32_t* q = qf[nr][np][j];
                        mma_f16(c, a[0], b[0], a[1], b[1], q[0], q[1]);
                        mma_f16(c, a[2], b[2], a[3], b[3], q[2], q[3]);
                    }
                    s[i][nr][0] = fmaf(sa, c[0], fmaf(ma, qsum[nr][0][j], s[i][nr][0]));
                    s[i][nr][1] = fmaf(sa, c[1], fmaf(ma, qsum[nr][1][j], s[i][nr][1]));
                    s[i][nr][2] = fmaf(sb, c[2], fmaf(mb, qsum[nr][0][j], s[i][nr][2]));
                    s[i][nr][3] = fmaf(sb, c[3], fmaf(mb, qsum[nr][1][j], s[i][nr][3]));
                }
            }
        }
        // tokens that a row does not see, or that are not there (their scores may be anything)
        if (masked) {
#pragma unroll
            for (int i = 0; i < TS; ++i)
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int tok = tok0 + i * kCacheTile + g + 8 * (e >> 1);
                        if (!(have >> i & 1) || tok >= min(lim[nr][e & 1], c1)) s[i][nr][e] = -INFINITY;
                    }
        }
        // values' groups, and each token's largest scale
        Words<G> va[TS], vb[TS];
        float sa_top[TS], sb_top[TS];
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const uint8_t* tile = st + i * L::TB;
            va[i] = lds_words<G>(tile + At::value_group(g, 0));
            vb[i] = lds_words<G>(tile + At::value_group(g + 8, 0));
            if (masked) {
                const int tok = tok0 + i * kCacheTile + g;
                const bool in = have >> i & 1;
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    if (!in || tok >= c1) va[i].w[j] = 0;
                    if (!in || tok + 8 >= c1) vb[i].w[j] = 0;
                }
            }
            sa_top[i] = sb_top[i] = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) {
                sa_top[i] = fmaxf(sa_top[i], group_scale(va[i].w[j]));
                sb_top[i] = fmaxf(sb_top[i], group_scale(vb[i].w[j]));
            }
        }
        bool raise = false;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float m = top[nr][e];
#pragma unroll
                for (int i = 0; i < TS; ++i) m = fmaxf(m, fmaxf(s[i][nr][e], s[i][nr][e + 2]));
                top[nr][e] = m;
                raise = raise || (m - ref[nr][e]) * f[nr][e] > kSlack || (ref[nr][e] == -INFINITY && m > -INFINITY);
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float c[2], back[2], forth[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float m = over_g_max(top[nr][e]);
                    c[e] = ref[nr][e] == -INFINITY ? 0.f : ex2((ref[nr][e] - m) * f[nr][e]);
                    ref[nr][e] = m;
                    l[nr][e] *= c[e];
                    wtop[nr][e] *= c[e];
                    back[e] = pow2_inverse(mult[nr][e]);
                    forth[e] = mult[nr][e] = mult_for(over_g_max(wtop[nr][e]));
#pragma unroll
                    for (int j = 0; j < G; ++j) omin[nr][e][j] *= c[e];
                }
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[nr][j][i / 4][i % 4] *= back[i & 1] * c[i & 1] * forth[i & 1];
#pragma unroll
                for (int i = 0; i < 2; ++i) racc[nr][i] *= back[i] * c[i] * forth[i];
            }
        }
        // p, relative to ref
        raise = false;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = ref[nr][e] == -INFINITY ? 0.f : -ref[nr][e] * f[nr][e];
                float w = 0.f;
#pragma unroll
                for (int i = 0; i < TS; ++i) {
                    s[i][nr][e] = ex2(fmaf(s[i][nr][e], f[nr][e], base));
                    s[i][nr][e + 2] = ex2(fmaf(s[i][nr][e + 2], f[nr][e], base));
                    l[nr][e] += s[i][nr][e] + s[i][nr][e + 2];
                    w = fmaxf(w, fmaxf(s[i][nr][e] * sa_top[i], s[i][nr][e + 2] * sb_top[i]));
                }
                wtop[nr][e] = fmaxf(wtop[nr][e], w);
                raise = raise || w * mult[nr][e] > kMostF16;
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float c[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float m = fminf(mult[nr][e], mult_for(over_g_max(wtop[nr][e])));
                    c[e] = pow2_inverse(mult[nr][e]) * m;
                    mult[nr][e] = m;
                }
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[nr][j][i / 4][i % 4] *= c[i & 1];
                racc[nr][0] *= c[0], racc[nr][1] *= c[1];
            }
        }
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const uint8_t* tile = st + i * L::TB;
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
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                const float p0 = s[i][nr][0] * mult[nr][0], p1 = s[i][nr][1] * mult[nr][1];
                const float p2 = s[i][nr][2] * mult[nr][0], p3 = s[i][nr][3] * mult[nr][1];
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    // a NaN group has a NaN minimum too; its scale must not meet the zeros of the row of ones
                    const float sa = fmaxf(group_scale(va[i].w[j]), 0.f), sb = fmaxf(group_scale(vb[i].w[j]), 0.f);
                    float ma = group_min(va[i].w[j]), mb = group_min(vb[i].w[j]);
                    constexpr float centre = SPLIT ? 8.f : 7.5f;
                    ma = fmaf(centre, sa, ma), mb = fmaf(centre, sb, mb);
                    omin[nr][0][j] = fmaf(s[i][nr][0], ma, fmaf(s[i][nr][2], mb, omin[nr][0][j]));
                    omin[nr][1][j] = fmaf(s[i][nr][1], ma, fmaf(s[i][nr][3], mb, omin[nr][1][j]));
                    uint32_t b0[NP], b1[NP];
                    if constexpr (SPLIT) {
                        split_f16x2(p0 * sa, p1 * sa, b0[0], b0[NP - 1]);
                        split_f16x2(p2 * sb, p3 * sb, b1[0], b1[NP - 1]);
                    } else {
                        b0[0] = pack_f16x2(p0 * sa, p1 * sa);
                        b1[0] = pack_f16x2(p2 * sb, p3 * sb);
                    }
                    uint32_t y[4], z[4];
                    code_operands<VX>(x[0][j], y);
                    code_operands<VX>(x[1][j], z);
#pragma unroll
                    for (int np = 0; np < NP; ++np) {
                        const uint32_t c0_ = transpose8x8(b0[np]), c1_ = transpose8x8(b1[np]);
                        mma_f16(acc[nr][j][0], y[0], y[1], z[0], z[1], c0_, c1_);
                        if constexpr (!SPLIT) mma_f16(racc[nr], g == j ? kOnes : 0u, 0u, g == j ? kOnes : 0u, 0u, c0_, c1_);
                        mma_f16(acc[nr][j][1], y[2], y[3], z[2], z[3], c0_, c1_);
                    }
                }
            }
        }
        __syncwarp();  // the slot has been read
        if (issued < mine) issue(issued), ++issued;
    }
    // A warp that gave up at a wait still owns the copies it issued: let them land first.
    for (int i = done; i < issued; ++i) mbar_drain(bar + i % NS, (uint32_t)(i / NS) & 1u);
    __syncthreads();
    if (threadIdx.x == 0 && *serr != 0) atomicExch(p.err, *serr);

    // ---- the warps' sums, relative to the largest score of the warp, to shared memory
    float* sacc = reinterpret_cast<float*>(smem) + warp * R * D;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * nr + 2 * t + e;
            const float m = over_g_max(top[nr][e]);
            const float c = ref[nr][e] == -INFINITY ? 0.f : ex2((ref[nr][e] - m) * f[nr][e]);
            const float sum = over_g_sum(l[nr][e]) * c;
            const float v = pow2_inverse(mult[nr][e]);
            float om[G], rs[G];
#pragma unroll
            for (int j = 0; j < G; ++j) {
                om[j] = over_g_sum(omin[nr][e][j]);
                rs[j] = SPLIT ? 0.f : -7.5f * __shfl_sync(0xffffffffu, racc[nr][e], j * 4 + t);
            }
            if (r < rows) {
                if (g == 0) sml[warp * R + r] = make_float2(m == -INFINITY ? m : m * f[nr][e], sum);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    float4 o;
                    o.x = fmaf(fmaf(acc[nr][j][0][e], code_unit<VX>(0), rs[j]), v, om[j]) * c;
                    o.y = fmaf(fmaf(acc[nr][j][0][e + 2], code_unit<VX>(1), rs[j]), v, om[j]) * c;
                    o.z = fmaf(fmaf(acc[nr][j][1][e], code_unit<VX>(2), rs[j]), v, om[j]) * c;
                    o.w = fmaf(fmaf(acc[nr][j][1][e + 2], code_unit<VX>(3), rs[j]), v, om[j]) * c;
                    *reinterpret_cast<float4*>(sacc + r * D + 32 * j + 4 * g) = o;
                }
            }
        }
    if (threadIdx.x < rows) {
        int n, q, hq;
        row_of(threadIdx.x, n, q, hq);
        srow[threadIdx.x] = ((int64_t)n * p.Tq + q) * p.H + hq;
    }
    __syncthreads();

    // ---- the CTA's sums: the output, or a partial
    const int S = p.splits_pre + p.splits_own, at = pre ? split : p.splits_pre + split;
    const float* all = reinterpret_cast<const float*>(smem);
    for (int i = threadIdx.x; i < rows * (D / 4); i += W * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, sml[w * R + r].x);
        float sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 ml = sml[w * R + r];
            const float c = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
            const float4 a = *reinterpret_cast<const float4*>(all + (w * R + r) * D + d);
            sum = fmaf(c, ml.y, sum);
            o.x = fmaf(c, a.x, o.x), o.y = fmaf(c, a.y, o.y), o.z = fmaf(c, a.z, o.z), o.w = fmaf(c, a.w, o.w);
        }
        const int64_t row = srow[r];
        if (S > 1) {
            *reinterpret_cast<float4*>(p.part + (row * S + at) * D + d) = o;
            if (d == 0) reinterpret_cast<float2*>(p.part_ml)[row * S + at] = make_float2(m, sum);
        } else {
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
    if (S == 1) return;
    // ---- the CTA that arrives last at a row merges it, and leaves its counter at zero
    __shared__ uint32_t s_last;
    if (threadIdx.x == 0) s_last = 0;
    __threadfence();
    __syncthreads();
    if (threadIdx.x < rows) {
        const unsigned before = atomicAdd(p.counter + srow[threadIdx.x], 1u);
        if (before == (unsigned)S - 1) {
            p.counter[srow[threadIdx.x]] = 0;
            atomicOr(&s_last, 1u << threadIdx.x);
        }
    }
    __syncthreads();
    const uint32_t last = s_last;
    if (last == 0) return;
    __threadfence();
    for (int r = warp; r < rows; r += W)
        if (last >> r & 1) merge_row<D, T>(p, srow[r], S);
}

struct Plan {
    int nr, tiles_pre, tiles_own, splits_pre, splits_own, range_pre, range_own;
    int64_t rows, grid;
    size_t off_ml, off_cnt, bytes;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Plan plan_of(const dbl_relay_cache_attention_args* a) {
    Plan L{};
    const int64_t G = a->heads / a->cache.kv_heads, TG = a->queries * G, H = a->cache.kv_heads, N = a->n_seq;
    const int64_t max_own = a->table_width * a->cache.page_size;
    L.nr = a->dtype == DBL_BF16 && (TG > 8 || (a->prefix_len > 0 && N * TG > 8)) ? 2 : 1;
    const int64_t R = 8 * L.nr;
    L.tiles_own = (int)ceil_div(TG, R);
    L.tiles_pre = a->prefix_len > 0 ? (int)ceil_div(N * TG, R) : 0;
    // CTAs enough for every SM to hold four, twice over; ranges of at least 256 tokens
    const int64_t want = 148 * 8;
    auto cut = [&](int64_t items, int64_t tokens, int& splits, int& range) {
        int64_t s = ceil_div(want, items);
        if (s > ceil_div(tokens, 256)) s = ceil_div(tokens, 256);
        if (s < 1) s = 1;
        int64_t r = ceil_div(ceil_div(tokens, s), W * STEP) * W * STEP;
        if (r < W * STEP) r = W * STEP;
        range = (int)r;
        splits = (int)ceil_div(tokens, r);
        if (splits < 1) splits = 1;
    };
    cut(N * H * L.tiles_own, max_own, L.splits_own, L.range_own);
    if (L.tiles_pre) cut(H * L.tiles_pre, a->prefix_len, L.splits_pre, L.range_pre);
    L.rows = N * a->queries * a->heads;
    L.grid = (int64_t)L.splits_pre * L.tiles_pre * H + (int64_t)L.splits_own * L.tiles_own * H * N;
    const int64_t S = L.splits_pre + L.splits_own;
    if (S > 1) {
        L.off_ml = (size_t)(L.rows * S * a->cache.head_dim) * 4;
        L.off_cnt = L.off_ml + (size_t)(L.rows * S) * 8;
        L.bytes = L.off_cnt + (size_t)L.rows * 4;
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
    if (a->prefix_len < 0 || a->prefix_len > 0x3fffffff || a->prefix_width < 0 || a->prefix_width > 0x7fffffff)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: prefix_len out of range");
    if (a->prefix_len > 0 && (!a->prefix_pages || a->prefix_width * a->cache.page_size < a->prefix_len))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: prefix_pages must hold prefix_len tokens");
    if (a->queries > 0x7fffffff || a->heads > 0x7fffffff || a->n_seq * a->queries > 0x7fffffff / a->heads ||
        a->table_width * a->cache.page_size > 0x3fffffff)
        return fail(DBL_ERR_UNSUPPORTED, "relay cache attention: sizes exceed 32-bit limits");
    return DBL_OK;
}

template <int D, typename T, int NR>
int launch_attn(const AttnParams& p, int64_t grid, cudaStream_t st) {
    constexpr int smem = AttnLayout<D, T, NR>::BYTES;
    static std::atomic<uint64_t> done{0};
    const int rc = once_per_device(done, [] {
        return cuda_status(cudaFuncSetAttribute(cache_attn_kernel<D, T, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                           "relay cache attention: cudaFuncSetAttribute");
    });
    if (rc != DBL_OK) return rc;
    cache_attn_kernel<D, T, NR><<<(unsigned)grid, W * 32, smem, st>>>(p);
    return launch_status("cache_attn_kernel");
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
    if (L.grid > 0x7fffffff) return fail(DBL_ERR_UNSUPPORTED, "relay cache attention: grid too large");
    if (L.bytes && (!workspace || workspace_bytes < L.bytes))
        return fail(DBL_ERR_WORKSPACE, "relay cache attention: workspace of %zu bytes required (got %zu)", L.bytes,
                    workspace_bytes);
    if (L.bytes && !aligned(workspace, 16))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: workspace must be 16-byte aligned");
    AttnParams p{};
    p.c = cache_view(&a->cache, a->page_table, a->table_width, a->table_stride);
    p.q = a->q;
    for (int i = 0; i < 3; ++i) p.qs[i] = qs[i];
    p.lengths = a->lengths;
    p.prefix_pages = a->prefix_pages;
    p.out = a->out;
    p.row_max = a->row_max;
    p.row_sum = a->row_sum;
    p.N = (int)a->n_seq;
    p.Tq = (int)a->queries;
    p.H = (int)a->heads;
    p.group = (int)(a->heads / a->cache.kv_heads);
    p.prefix_len = (int)a->prefix_len;
    p.prefix_width = (int)a->prefix_width;
    p.scale = a->scale;
    p.tiles_pre = L.tiles_pre;
    p.tiles_own = L.tiles_own;
    p.splits_pre = L.splits_pre;
    p.splits_own = L.splits_own;
    p.range_pre = L.range_pre;
    p.range_own = L.range_own;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.part = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + L.off_ml);
    p.counter = reinterpret_cast<unsigned*>(ws + L.off_cnt);
    rc = device_error_record(&p.err);
    if (rc != DBL_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == DBL_F32)
        return D == 128 ? launch_attn<128, float, 1>(p, L.grid, st) : launch_attn<64, float, 1>(p, L.grid, st);
    if (L.nr == 1)
        return D == 128 ? launch_attn<128, __nv_bfloat16, 1>(p, L.grid, st)
                        : launch_attn<64, __nv_bfloat16, 1>(p, L.grid, st);
    return D == 128 ? launch_attn<128, __nv_bfloat16, 2>(p, L.grid, st)
                    : launch_attn<64, __nv_bfloat16, 2>(p, L.grid, st);
}
