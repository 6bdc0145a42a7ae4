// Writing tokens into the 4-bit relay cache and reading them back.
//
// A group is 32 channels of one token's key or value at one head.  With x its values,
//   minimum = min(x) rounded down to bf16,      scale = (max(x) - minimum) / 15 rounded up to bf16,
//   code    = the smallest c of 0 .. 15 with x - minimum <= (c + 1/2) scale,
// so the values that the codes stand for reach from the minimum to at least max(x) whatever the two
// roundings did, and the error is at most scale / 2.  All of it is f32 arithmetic; (c + 1/2) scale
// has 13 significant bits and is exact.  A range below 2^-100 has scale 0 (1 / scale must be
// finite); a range that is not finite (an infinity or NaN among the values) makes the group NaN, so
// that it shows in what is computed from the token and from no other.
#include <type_traits>

#include "relay_cache.cuh"
#include "tc_ptx.cuh"

namespace dbl {
namespace {

struct AppendParams {
    CacheView c;
    const void *k, *v;
    int64_t ks[3], vs[3];  // strides of sequence, token and head
    const int32_t *lengths, *counts;
    int32_t* new_lengths;
    int T, tiles, blocks, per;  // tiles that T tokens can touch; blocks of a sequence; heads of a CTA
    bool vec;              // 16-byte loads
    int* err;
};

struct ReadParams {
    CacheView c;
    void *k, *v;
    const int32_t *lengths, *start;
    int T, tiles, blocks;
    int* err;
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Codes of NC channels of a group, of which 32 / NC neighbouring lanes hold NC each: 8 to a word, the
// first in the lowest four bits.  Returns the group's (scale, minimum) word.
//
// The code of d = x - minimum is the nearest integer to d / scale, ties down.  The guess, d times a
// reciprocal that is 2^-21 too small (rcp.approx is off by 2^-23 at most), rounded to an integer by adding
// 1.5 * 2^23, is the code or one less; d - guess * scale is exact (a multiple of d's last place, less than
// 2^24 of them) and says which.
template <int NC>
__device__ __forceinline__ uint32_t encode(const float (&x)[NC], uint32_t (&codes)[NC / 8]) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < NC; ++i) {
        lo = fminf(lo, x[i]);
        hi = max_nan(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 32 / NC; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    uint32_t lb = __float_as_uint(lo);
    lb = (lb & 0x80000000u) ? (lb + 0xFFFFu) & 0xFFFF0000u : lb & 0xFFFF0000u;
    const float base = __uint_as_float(lb);
    const float span = hi - base;
    uint32_t sb = (__float_as_uint(__fdiv_rn(span, 15.f)) + 0xFFFFu) & 0xFFFF0000u;
    if (span < 7.888609052e-31f) sb = 0;  // 2^-100
    const bool bad = !(span <= 3.402823466e38f);  // NaN too
    const float s = __uint_as_float(sb), half = 0.5f * s;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    inv *= 0.9999995232f;
    constexpr float kRound = 12582912.f;
#pragma unroll
    for (int w = 0; w < NC / 8; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            const float d = x[8 * w + i] - base, t = fmaf(d, inv, kRound);
            word = word * 16u + __float_as_uint(t);
            if (fmaf(kRound - t, s, d) > half) ++word;
        }
        codes[w] = bad || sb == 0 ? 0u : word - __float_as_uint(kRound) * 0x11111111u;  // kRound's bits of all eight
    }
    return bad ? 0x7FFF0000u /* scale 0, minimum NaN */ : (sb >> 16) | lb;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, bool vec, float (&x)[8]) {
    if (vec) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = bf16_lo(u[i]), x[2 * i + 1] = bf16_hi(u[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
    }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, bool vec, float (&x)[8]) {
    if (vec) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}

// Single tokens.  One thread: 8 channels of one (token, head), of the key and then of the value; four
// neighbouring lanes are a group.
template <int D, typename T>
__global__ void __launch_bounds__(256) cache_append_kernel(const AppendParams p) {
    using At = TileAt<D>;
    constexpr int LPT = D / 8;  // lanes of a token and head
    const int64_t n = blockIdx.x / p.blocks;
    const int i = blockIdx.x % p.blocks * 256 + threadIdx.x, row = i / LPT, part = i % LPT;  // row: (token, head)
    const int count = p.counts ? min(max(p.counts[n], 0), p.T) : p.T, len = p.lengths[n];
    if (p.new_lengths && i == 0) p.new_lengths[n] = len + count;
    // lanes past the end go along with the first row and write nothing: the shuffles need whole groups
    const bool inside = row < p.T * p.c.heads;
    const int t = inside ? row / p.c.heads : 0, h = inside ? row - t * p.c.heads : 0;
    float x[8], y[8];
    load8<T>(static_cast<const T*>(p.k) + n * p.ks[0] + t * p.ks[1] + h * p.ks[2] + part * 8, p.vec, x);
    load8<T>(static_cast<const T*>(p.v) + n * p.vs[0] + t * p.vs[1] + h * p.vs[2] + part * 8, p.vec, y);
    const bool live = inside && t < count;
    const int pos = len + t;
    const int page = live && pos >= 0 ? cache_page(p.c, n, pos / kCacheTile) : -1;
    if (live && page < 0) atomicExch(p.err, kCacheErrorPage);
    const int k = pos & (kCacheTile - 1);
    uint8_t* tile = cache_tile<D>(p.c, max(page, 0), h, max(pos, 0) / kCacheTile % p.c.tiles);
    const int j = part / 4, q = part % 4;  // group, quarter of the group
    uint32_t kc[1], vc[1];
    const uint32_t kw = encode<8>(x, kc), vw = encode<8>(y, vc);
    if (page < 0) return;
    *reinterpret_cast<uint32_t*>(tile + At::key_word(k, q, j)) = kc[0];
    *reinterpret_cast<uint16_t*>(tile + At::value_half(k, 2 * q, j)) = (uint16_t)vc[0];
    *reinterpret_cast<uint16_t*>(tile + At::value_half(k, 2 * q + 1, j)) = (uint16_t)(vc[0] >> 16);
    if (q == 0) {
        *reinterpret_cast<uint32_t*>(tile + At::key_group(k, j)) = kw;
        *reinterpret_cast<uint32_t*>(tile + At::value_group(k, j)) = vw;
    }
}

// Prompts.  A CTA writes one tile of positions for p.per heads, one after another: the tile is put together in shared
// memory and leaves in 16-byte words (in the pieces of single tokens where it is not written whole).  One
// thread: 16 channels of one token's key or value, two neighbouring lanes a group; its next head's
// values are on their way while it encodes.  8 x 4096 tokens, 16 heads of 128, bf16 (268 MB in, 84 MB out): 88 us
// = 4000 GB/s, 61% of the measured copy rate; bound by instructions (19 an element, issue slots 81% busy).  A
// correction on the FMA pipe alone (saturating products instead of compares) took the same time.
constexpr int kTileHeads = 4, kManyHeads = 16;
// Calls of at least so many tokens a sequence go by tiles.  256 sequences at all places in a tile, 16 heads of 128,
// by tiles and by single tokens: 8 tokens, append 26 and 12 us, read 13 and 10 us; 16 tokens 31 and 21, 16 and 17
// us; 64 tokens 66 and 78, 41 and 57 us.
constexpr int kTileTokens = 32;

template <int D, typename T>
__global__ void __launch_bounds__(256) cache_append_tiles_kernel(const AppendParams p) {
    using At = TileAt<D>;
    constexpr int TB = cache_tile_bytes(D), LPT = D / 16, HP = 128 / D;  // lanes of a token, heads of a pass
    constexpr int NW = 16 / (16 / (int)sizeof(T));                       // 16-byte words of 16 channels
    __shared__ __align__(16) uint8_t image[2][HP * TB];
    const unsigned hg = (p.c.heads + p.per - 1) / p.per;
    const unsigned b = blockIdx.x / hg, tn = b / p.tiles;
    const int h0 = (int)(blockIdx.x - b * hg) * p.per, h1 = min(h0 + p.per, p.c.heads), ti = (int)(b - tn * p.tiles);
    const int64_t n = tn;
    const int count = p.counts ? min(max(p.counts[n], 0), p.T) : p.T, len = p.lengths[n];
    if (p.new_lengths && ti == 0 && h0 == 0 && threadIdx.x == 0) p.new_lengths[n] = len + count;
    if (len < 0) {  // as single tokens: those at positions below zero are left out, and said to be
        if (count > 0 && threadIdx.x == 0) atomicExch(p.err, kCacheErrorPage);
        if (len <= -p.T) return;
    }
    const int tl = max(len, 0) / kCacheTile + ti, t0 = tl * kCacheTile - len;  // token of place 0
    if (t0 >= count) return;
    const int page = cache_page(p.c, n, tl);
    if (page < 0) {
        if (threadIdx.x == 0) atomicExch(p.err, kCacheErrorPage);
        return;
    }
    const int i = threadIdx.x, hp = i / (2 * D), which = i / D % 2, k = i / LPT % kCacheTile, part = i % LPT;
    const int t = t0 + k, j = part / 2, q = part % 2;
    const bool live = t >= 0 && t < count;
    const bool whole = t0 >= 0 && t0 + kCacheTile <= count;
    const T* src = static_cast<const T*>(which ? p.v : p.k) + n * (which ? p.vs[0] : p.ks[0]) +
                   (live ? t : 0) * (which ? p.vs[1] : p.ks[1]) + part * 16;
    const int64_t hs = which ? p.vs[2] : p.ks[2];
    uint4 raw[NW];
    auto load = [&](int h) {
        const T* at = src + min(h, h1 - 1) * hs;
        if (p.vec) {
#pragma unroll
            for (int w = 0; w < NW; ++w) raw[w] = __ldg(reinterpret_cast<const uint4*>(at) + w);
        } else {
            T v[16];
#pragma unroll
            for (int w = 0; w < 16; ++w) v[w] = at[w];
#pragma unroll
            for (int w = 0; w < NW; ++w) raw[w] = reinterpret_cast<const uint4*>(v)[w];
        }
    };
    load(h0 + hp);
    int buf = 0;
    for (int h = h0; h < h1; h += HP, buf ^= 1) {
        float x[16];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) x[4 * w + e] = __uint_as_float(u[e]);
                else x[8 * w + 2 * e] = bf16_lo(u[e]), x[8 * w + 2 * e + 1] = bf16_hi(u[e]);
            }
        }
        if (h + HP < h1) load(h + HP + hp);
        uint32_t codes[2];
        const uint32_t word = encode<16>(x, codes);
        uint8_t* img = image[buf] + hp * TB;
        if (which) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint16_t*>(img + At::value_half(k, 4 * q + e, j)) = (uint16_t)(codes[e / 2] >> (16 * (e % 2)));
            if (q == 0) *reinterpret_cast<uint32_t*>(img + At::value_group(k, j)) = word;
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) *reinterpret_cast<uint32_t*>(img + At::key_word(k, 2 * q + e, j)) = codes[e];
            if (q == 0) *reinterpret_cast<uint32_t*>(img + At::key_group(k, j)) = word;
        }
        __syncthreads();  // the image is complete; the other one has been written out (two images, one barrier each)
        const int heads = min(HP, h1 - h);
        uint8_t* to = cache_tile<D>(p.c, page, h, tl % p.c.tiles);
        const int64_t per = (int64_t)p.c.tiles * TB;  // from head to head
        if (whole) {
            for (int w = i; w < heads * (TB / 16); w += 256) {
                const int hh = w / (TB / 16), at = w % (TB / 16);
                reinterpret_cast<uint4*>(to + hh * per)[at] = reinterpret_cast<const uint4*>(image[buf] + hh * TB)[at];
            }
        } else {  // pieces of D / 16 bytes, each of one token
            using Piece = typename std::conditional<D == 128, uint2, uint32_t>::type;
            constexpr int NPC = TB / (int)sizeof(Piece), ROW = 8;
            for (int w = i; w < heads * NPC; w += 256) {
                const int hh = w / NPC, at = w % NPC, in = at % (NPC / 2);  // codes: 16 rows of 8 pieces, groups: 2 pieces
                int kk = in >= 16 * ROW ? (in - 16 * ROW) / 2 : at < NPC / 2 ? in / ROW : in / 64 * 8 + in % 8;
                const int tt = t0 + kk;
                if (tt >= 0 && tt < count)
                    reinterpret_cast<Piece*>(to + hh * per)[at] = reinterpret_cast<const Piece*>(image[buf] + hh * TB)[at];
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                              pack_bf16x2(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

__device__ __forceinline__ void decode8(uint32_t codes, uint32_t word, float (&x)[8]) {
    const float s = group_scale(word), m = group_min(word);
#pragma unroll
    for (int i = 0; i < 8; ++i)  // 2^23 + code as bits; the product is exact
        x[i] = fmaf(s, __uint_as_float((codes >> (4 * i) & 15u) | 0x4B000000u) - 8388608.f, m);
}

// Single tokens: as the append.
template <int D, typename T>
__global__ void __launch_bounds__(256) cache_read_kernel(const ReadParams p) {
    using At = TileAt<D>;
    constexpr int LPT = D / 8;
    const int64_t n = blockIdx.x / p.blocks;
    const int i = blockIdx.x % p.blocks * 256 + threadIdx.x, row = i / LPT, part = i % LPT;
    if (row >= p.T * p.c.heads) return;
    const int t = row / p.c.heads, h = row - t * p.c.heads;
    const int64_t pos = (p.start ? (int64_t)p.start[n] : 0) + t;
    const bool live = pos >= 0 && pos < p.lengths[n];
    const int page = live ? cache_page(p.c, n, (int)(pos / kCacheTile)) : -1;
    if (live && page < 0) atomicExch(p.err, kCacheErrorPage);
    float xk[8] = {}, xv[8] = {};
    if (page >= 0) {
        const int k = (int)(pos & (kCacheTile - 1));
        const uint8_t* tile = cache_tile<D>(p.c, page, h, (int)(pos / kCacheTile) % p.c.tiles);
        const int j = part / 4, q = part % 4;
        decode8(*reinterpret_cast<const uint32_t*>(tile + At::key_word(k, q, j)),
                *reinterpret_cast<const uint32_t*>(tile + At::key_group(k, j)), xk);
        const uint32_t lo = *reinterpret_cast<const uint16_t*>(tile + At::value_half(k, 2 * q, j));
        const uint32_t hi = *reinterpret_cast<const uint16_t*>(tile + At::value_half(k, 2 * q + 1, j));
        decode8(lo | hi << 16, *reinterpret_cast<const uint32_t*>(tile + At::value_group(k, j)), xv);
    }
    const int64_t at = ((n * p.T + t) * p.c.heads + h) * D + part * 8;
    store8<T>(static_cast<T*>(p.k) + at, xk);
    store8<T>(static_cast<T*>(p.v) + at, xv);
}

// Runs of tokens: a CTA reads one tile of positions for kTileHeads heads, all of them at once in 16-byte
// words to shared memory.  One thread: 16 channels of one token's key or value.  The prompts above (84 MB in,
// 268 MB out): 64.5 us = 5450 GB/s, 83% of the measured copy rate; one tile at a time took 79 us.
template <int D, typename T>
__global__ void __launch_bounds__(256) cache_read_tiles_kernel(const ReadParams p) {
    using At = TileAt<D>;
    constexpr int TB = cache_tile_bytes(D), LPT = D / 16, HP = 128 / D, WORDS = TB / 16;
    __shared__ __align__(16) uint8_t image[kTileHeads * TB];
    const unsigned hg = (p.c.heads + kTileHeads - 1) / kTileHeads;
    const unsigned b = blockIdx.x / hg, tn = b / p.tiles;
    const int h0 = (int)(blockIdx.x - b * hg) * kTileHeads, h1 = min(h0 + kTileHeads, p.c.heads), ti = (int)(b - tn * p.tiles);
    const int64_t n = tn;
    const int len = p.lengths[n];
    static_assert(kCacheTile == 16, "positions shift by 4");
    const int64_t first = p.start ? p.start[n] : 0;     // positions may pass 32 bits where the start is far out
    const int64_t tl = (first >> 4) + ti;               // rounded down
    const int t0 = (int)(tl * kCacheTile - first);      // token of place 0
    if (t0 >= p.T) return;
    const bool any = tl >= 0 && tl * kCacheTile < len;
    const int page = any ? cache_page(p.c, n, (int)tl) : -1;
    if (any && page < 0 && threadIdx.x == 0) atomicExch(p.err, kCacheErrorPage);
    const int i = threadIdx.x, hp = i / (2 * D), which = i / D % 2, k = i / LPT % kCacheTile, part = i % LPT;
    const int t = t0 + k, j = part / 2, q = part % 2;
    const bool wanted = t >= 0 && t < p.T, held = page >= 0 && first + t < len;
    const uint8_t* from = cache_tile<D>(p.c, max(page, 0), h0, any ? (int)tl % p.c.tiles : 0);
    const int64_t per = (int64_t)p.c.tiles * TB;  // from head to head
    if (page >= 0) {
        const int words = (h1 - h0) * WORDS;
        uint4 raw[(kTileHeads * WORDS + 255) / 256];
#pragma unroll
        for (int w = 0; w < (kTileHeads * WORDS + 255) / 256; ++w) {
            const int at = i + 256 * w, hh = at / WORDS;
            if (at < words) raw[w] = __ldg(reinterpret_cast<const uint4*>(from + hh * per) + (at - hh * WORDS));
        }
#pragma unroll
        for (int w = 0; w < (kTileHeads * WORDS + 255) / 256; ++w)
            if (i + 256 * w < words) reinterpret_cast<uint4*>(image)[i + 256 * w] = raw[w];
    }
    __syncthreads();
    if (!wanted) return;
    for (int h = h0 + hp; h < h1; h += HP) {
        const uint8_t* img = image + (h - h0) * TB;
        float x[2][8];
        uint32_t word, codes[2];
        if (which) {
            word = *reinterpret_cast<const uint32_t*>(img + At::value_group(k, j));
#pragma unroll
            for (int e = 0; e < 2; ++e)
                codes[e] = *reinterpret_cast<const uint16_t*>(img + At::value_half(k, 4 * q + 2 * e, j)) |
                           (uint32_t)*reinterpret_cast<const uint16_t*>(img + At::value_half(k, 4 * q + 2 * e + 1, j)) << 16;
        } else {
            word = *reinterpret_cast<const uint32_t*>(img + At::key_group(k, j));
#pragma unroll
            for (int e = 0; e < 2; ++e) codes[e] = *reinterpret_cast<const uint32_t*>(img + At::key_word(k, 2 * q + e, j));
        }
        if (!held) word = 0;  // zero, whatever the codes
        decode8(codes[0], word, x[0]);
        decode8(codes[1], word, x[1]);
        T* to = static_cast<T*>(which ? p.v : p.k) + ((n * p.T + t) * p.c.heads + h) * D + part * 16;
        store8<T>(to, x[0]);
        store8<T>(to + 8, x[1]);
    }
}

// Tiles or single tokens, and the grid; false where it is too large.
bool grid_for(int64_t n_seq, int64_t tokens, int64_t heads, int D, int per, int& tiles, int& blocks, bool& by_tiles,
              unsigned& grid) {
    if (tokens > 0x7ffffff0 || tokens * heads > 0x7fffffff / D) return false;
    tiles = (int)((tokens + 2 * kCacheTile - 2) / kCacheTile);
    blocks = (int)((tokens * heads * (D / 8) + 255) / 256);
    by_tiles = tokens >= kTileTokens;
    const int64_t ctas = n_seq * (by_tiles ? tiles * ((heads + per - 1) / per) : (int64_t)blocks);
    grid = (unsigned)ctas;
    return ctas <= 0x7fffffff;
}

}  // namespace

int cache_validate(const dbl_relay_cache* c, const char* what) {
    if (c->pages <= 0 || c->kv_heads <= 0)
        return fail(DBL_ERR_INVALID_ARGUMENT, "%s: pages and kv_heads must be positive", what);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(DBL_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128 (got %lld)", what, (long long)c->head_dim);
    if (c->page_size <= 0 || c->page_size % kCacheTile || c->page_size > 4096)
        return fail(DBL_ERR_UNSUPPORTED, "%s: page_size must be a multiple of 16 up to 4096 (got %lld)", what,
                    (long long)c->page_size);
    if (c->pages > 0x7fffffff || c->kv_heads > 65535 || c->pages * c->kv_heads > 0x7fffffff / (c->page_size / kCacheTile))
        return fail(DBL_ERR_UNSUPPORTED, "%s: sizes exceed 32-bit limits", what);
    if (!c->pool) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: pool is required", what);
    if (!aligned(c->pool, 16)) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: pool must be 16-byte aligned", what);
    return DBL_OK;
}

int cache_check_table(const int32_t* table, int64_t n_seq, int64_t width, int64_t stride, const char* what) {
    if (n_seq <= 0) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: n_seq must be positive", what);
    if (width <= 0 || stride < 0 || (stride && stride < width))
        return fail(DBL_ERR_INVALID_ARGUMENT, "%s: the page table needs a positive width and a row stride of at least it",
                    what);
    if (n_seq > 0x7fffffff || width > 0x7fffffff)
        return fail(DBL_ERR_UNSUPPORTED, "%s: sizes exceed 32-bit limits", what);
    if (!table) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: page_table is required", what);
    return DBL_OK;
}

}  // namespace dbl

extern "C" int dbl_relay_cache_append(const dbl_relay_cache_append_args* a, dbl_stream_t stream) {
    using namespace dbl;
    if (!a) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache append: null args");
    int rc = cache_validate(&a->cache, "relay cache append");
    if (rc == DBL_OK)
        rc = cache_check_table(a->page_table, a->n_seq, a->table_width, a->table_stride, "relay cache append");
    if (rc != DBL_OK) return rc;
    if (a->tokens <= 0) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache append: tokens must be positive");
    if (a->dtype != DBL_F32 && a->dtype != DBL_BF16)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache append: dtype must be f32 or bf16");
    if (!a->k || !a->v || !a->lengths)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache append: k, v and lengths are required");
    const int D = (int)a->cache.head_dim;
    const int64_t dims[4] = {a->n_seq, a->tokens, a->cache.kv_heads, D};
    int64_t ks[4], vs[4];
    resolve_strides(a->k_stride, dims, 4, ks);
    resolve_strides(a->v_stride, dims, 4, vs);
    if (ks[3] != 1 || vs[3] != 1)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache append: the innermost stride of k and v must be 1");
    AppendParams p{};
    p.c = cache_view(&a->cache, a->page_table, a->table_width, a->table_stride);
    p.k = a->k;
    p.v = a->v;
    for (int i = 0; i < 3; ++i) p.ks[i] = ks[i], p.vs[i] = vs[i];
    p.lengths = a->lengths;
    p.counts = a->counts;
    p.new_lengths = a->new_lengths;
    p.T = (int)a->tokens;
    // 16-byte loads where every row of k and v starts on 16 bytes
    const int64_t per = 16 / (int64_t)dtype_size(a->dtype);
    p.vec = aligned(a->k, 16) && aligned(a->v, 16);
    for (int i = 0; i < 3; ++i) p.vec = p.vec && ks[i] % per == 0 && vs[i] % per == 0;
    bool tiles;
    unsigned grid;
    // More heads a CTA spread its start over more work, where the GPU is full all the same: 8 x 4096 tokens of 16
    // heads take 98 us at 4 heads a CTA, 91 at 8, 88 at 16; one sequence of them (less than a round) 15 us at each.
    const int64_t full = a->n_seq * ((a->tokens + kCacheTile - 1) / kCacheTile) * a->cache.kv_heads / (148 * 4);
    p.per = full >= kManyHeads ? kManyHeads : kTileHeads;
    if (!grid_for(a->n_seq, a->tokens, a->cache.kv_heads, D, p.per, p.tiles, p.blocks, tiles, grid))
        return fail(DBL_ERR_UNSUPPORTED, "relay cache append: grid too large");
    rc = device_error_record(&p.err);
    if (rc != DBL_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(p); };
    if (a->dtype == DBL_BF16) {
        if (D == 128) launch(tiles ? cache_append_tiles_kernel<128, __nv_bfloat16> : cache_append_kernel<128, __nv_bfloat16>);
        else launch(tiles ? cache_append_tiles_kernel<64, __nv_bfloat16> : cache_append_kernel<64, __nv_bfloat16>);
    } else {
        if (D == 128) launch(tiles ? cache_append_tiles_kernel<128, float> : cache_append_kernel<128, float>);
        else launch(tiles ? cache_append_tiles_kernel<64, float> : cache_append_kernel<64, float>);
    }
    return launch_status("cache_append_kernel");
}

extern "C" int dbl_relay_cache_read(const dbl_relay_cache_read_args* a, dbl_stream_t stream) {
    using namespace dbl;
    if (!a) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: null args");
    int rc = cache_validate(&a->cache, "relay cache read");
    if (rc == DBL_OK) rc = cache_check_table(a->page_table, a->n_seq, a->table_width, a->table_stride, "relay cache read");
    if (rc != DBL_OK) return rc;
    if (a->tokens <= 0) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: tokens must be positive");
    if (a->dtype != DBL_F32 && a->dtype != DBL_BF16)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: dtype must be f32 or bf16");
    if (!a->k || !a->v || !a->lengths)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: k, v and lengths are required");
    if (!aligned(a->k, 16) || !aligned(a->v, 16))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: k and v must be 16-byte aligned");
    const int D = (int)a->cache.head_dim;
    ReadParams p{};
    p.c = cache_view(&a->cache, a->page_table, a->table_width, a->table_stride);
    p.k = a->k;
    p.v = a->v;
    p.lengths = a->lengths;
    p.start = a->start;
    p.T = (int)a->tokens;
    bool tiles;
    unsigned grid;
    if (!grid_for(a->n_seq, a->tokens, a->cache.kv_heads, D, kTileHeads, p.tiles, p.blocks, tiles, grid))
        return fail(DBL_ERR_UNSUPPORTED, "relay cache read: grid too large");
    rc = device_error_record(&p.err);
    if (rc != DBL_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const auto launch = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(p); };
    if (a->dtype == DBL_BF16) {
        if (D == 128) launch(tiles ? cache_read_tiles_kernel<128, __nv_bfloat16> : cache_read_kernel<128, __nv_bfloat16>);
        else launch(tiles ? cache_read_tiles_kernel<64, __nv_bfloat16> : cache_read_kernel<64, __nv_bfloat16>);
    } else {
        if (D == 128) launch(tiles ? cache_read_tiles_kernel<128, float> : cache_read_kernel<128, float>);
        else launch(tiles ? cache_read_tiles_kernel<64, float> : cache_read_kernel<64, float>);
    }
    return launch_status("cache_read_kernel");
}
