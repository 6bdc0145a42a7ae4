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
    int N, T;
    int* err;
};

struct ReadParams {
    CacheView c;
    void *k, *v;
    const int32_t *lengths, *start;
    int N, T;
    int* err;
};

// Codes of 8 channels of a group of which four neighbouring lanes hold 8 each.  Returns the eight
// codes (the first in the lowest four bits) and the group's (scale, minimum) word.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t& word) {
    // fminf and fmaxf pass over a NaN, the sum does not
    float lo = x[0], hi = x[0], sum = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        sum += x[i];
    }
    bool bad = sum != sum;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad = bad | (__shfl_xor_sync(0xffffffffu, (int)bad, o) != 0);
    }
    uint32_t lb = __float_as_uint(lo);
    lb = (lb & 0x80000000u) ? (lb + 0xFFFFu) & 0xFFFF0000u : lb & 0xFFFF0000u;
    const float base = __uint_as_float(lb);
    const float span = hi - base;
    bad = bad || !(span <= 3.402823466e38f);
    uint32_t sb = (__float_as_uint(__fdiv_rn(span, 15.f)) + 0xFFFFu) & 0xFFFF0000u;
    if (span < 7.888609052e-31f) sb = 0;  // 2^-100
    if (bad) {
        word = 0x7FFF0000u;  // scale 0, minimum NaN
        return 0;
    }
    word = (sb >> 16) | lb;
    if (sb == 0) return 0;
    const float s = __uint_as_float(sb), inv = __fdiv_rn(1.f, s);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float d = x[i] - base;
        // a first guess within one of the code, then the definition
        int c = __float2int_ru(fmaf(d, inv, -0.5f));
        c += d > ((float)c + 0.5f) * s ? 1 : 0;
        c -= d <= ((float)c - 0.5f) * s ? 1 : 0;
        codes |= (uint32_t)min(max(c, 0), 15) << (4 * i);
    }
    return codes;
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

// One thread: 8 channels of one (token, head), of the key and then of the value; four neighbouring
// lanes are a group.
template <int D, typename T>
__global__ void __launch_bounds__(256) cache_append_kernel(const AppendParams p, bool vec) {
    using At = TileAt<D>;
    constexpr int LPT = D / 8;  // lanes of a token and head
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t row = i / LPT;  // (sequence, token, head)
    const int part = (int)(i % LPT);
    const int64_t rows = (int64_t)p.N * p.T * p.c.heads;
    if (p.new_lengths && i < p.N) {
        const int cnt = p.counts ? min(max(p.counts[i], 0), p.T) : p.T;
        p.new_lengths[i] = p.lengths[i] + cnt;
    }
    // whole groups of lanes leave or stay, and the shuffles are among the four lanes of a group
    const bool inside = row < rows;
    const int h = inside ? (int)(row % p.c.heads) : 0;
    const int64_t nt = inside ? row / p.c.heads : 0;
    const int t = (int)(nt % p.T);
    const int64_t n = nt / p.T;
    const int count = p.counts ? min(max(p.counts[n], 0), p.T) : p.T;
    const bool live = inside && t < count;
    const int pos = p.lengths[n] + t;
    const int page = live && pos >= 0 ? cache_page(p.c, n, pos / kCacheTile) : -1;
    if (live && page < 0) atomicExch(p.err, kCacheErrorPage);
    const int k = pos & (kCacheTile - 1);
    uint8_t* tile = cache_tile<D>(p.c, max(page, 0), h, (pos / kCacheTile) % p.c.tiles);
    const int j = part / 4, q = part % 4;  // group, quarter of the group
    float x[8];
    uint32_t word;
    load8<T>(static_cast<const T*>(p.k) + n * p.ks[0] + t * p.ks[1] + h * p.ks[2] + part * 8, vec, x);
    uint32_t codes = encode8(x, word);
    if (page >= 0) {
        *reinterpret_cast<uint32_t*>(tile + At::key_word(k, q, j)) = codes;
        if (q == 0) *reinterpret_cast<uint32_t*>(tile + At::key_group(k, j)) = word;
    }
    load8<T>(static_cast<const T*>(p.v) + n * p.vs[0] + t * p.vs[1] + h * p.vs[2] + part * 8, vec, x);
    codes = encode8(x, word);
    if (page >= 0) {
        *reinterpret_cast<uint16_t*>(tile + At::value_half(k, 2 * q, j)) = (uint16_t)codes;
        *reinterpret_cast<uint16_t*>(tile + At::value_half(k, 2 * q + 1, j)) = (uint16_t)(codes >> 16);
        if (q == 0) *reinterpret_cast<uint32_t*>(tile + At::value_group(k, j)) = word;
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
    for (int i = 0; i < 8; ++i) x[i] = fmaf(s, (float)((codes >> (4 * i)) & 15u), m);  // the product is exact
}

template <int D, typename T>
__global__ void __launch_bounds__(256) cache_read_kernel(const ReadParams p) {
    using At = TileAt<D>;
    constexpr int LPT = D / 8;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t row = i / LPT;
    const int part = (int)(i % LPT);
    if (row >= (int64_t)p.N * p.T * p.c.heads) return;
    const int h = (int)(row % p.c.heads);
    const int64_t nt = row / p.c.heads;
    const int t = (int)(nt % p.T);
    const int64_t n = nt / p.T;
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
    store8<T>(static_cast<T*>(p.k) + row * D + part * 8, xk);
    store8<T>(static_cast<T*>(p.v) + row * D + part * 8, xv);
}

unsigned blocks_for(int64_t threads, int block) { return (unsigned)((threads + block - 1) / block); }

int check_table(const int32_t* table, int64_t n_seq, int64_t width, int64_t stride, const char* what) {
    if (n_seq <= 0) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: n_seq must be positive", what);
    if (width <= 0 || stride < 0 || (stride && stride < width))
        return fail(DBL_ERR_INVALID_ARGUMENT, "%s: the page table needs a positive width and a row stride of at least it",
                    what);
    if (n_seq > 0x7fffffff || width > 0x7fffffff)
        return fail(DBL_ERR_UNSUPPORTED, "%s: sizes exceed 32-bit limits", what);
    if (!table) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: page_table is required", what);
    return DBL_OK;
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
    return check_table(table, n_seq, width, stride, what);
}

}  // namespace dbl

extern "C" int dbl_relay_cache_append(const dbl_relay_cache_append_args* a, dbl_stream_t stream) {
    using namespace dbl;
    if (!a) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache append: null args");
    int rc = cache_validate(&a->cache, "relay cache append");
    if (rc == DBL_OK)
        rc = check_table(a->page_table, a->n_seq, a->table_width, a->table_stride, "relay cache append");
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
    const int64_t threads = a->n_seq * a->tokens * a->cache.kv_heads * (D / 8);
    if (a->tokens > 0x7fffffff || threads / 256 > 0x7ffffff0)
        return fail(DBL_ERR_UNSUPPORTED, "relay cache append: grid too large");
    AppendParams p{};
    p.c = cache_view(&a->cache, a->page_table, a->table_width, a->table_stride);
    p.k = a->k;
    p.v = a->v;
    for (int i = 0; i < 3; ++i) p.ks[i] = ks[i], p.vs[i] = vs[i];
    p.lengths = a->lengths;
    p.counts = a->counts;
    p.new_lengths = a->new_lengths;
    p.N = (int)a->n_seq;
    p.T = (int)a->tokens;
    rc = device_error_record(&p.err);
    if (rc != DBL_OK) return rc;
    // 16-byte loads where every row of k and v starts on 16 bytes
    const int64_t per = 16 / (int64_t)dtype_size(a->dtype);
    bool vec = aligned(a->k, 16) && aligned(a->v, 16);
    for (int i = 0; i < 3; ++i) vec = vec && ks[i] % per == 0 && vs[i] % per == 0;
    const unsigned grid = blocks_for(threads > p.N ? threads : p.N, 256);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == DBL_BF16) {
        if (D == 128) cache_append_kernel<128, __nv_bfloat16><<<grid, 256, 0, st>>>(p, vec);
        else cache_append_kernel<64, __nv_bfloat16><<<grid, 256, 0, st>>>(p, vec);
    } else {
        if (D == 128) cache_append_kernel<128, float><<<grid, 256, 0, st>>>(p, vec);
        else cache_append_kernel<64, float><<<grid, 256, 0, st>>>(p, vec);
    }
    return launch_status("cache_append_kernel");
}

extern "C" int dbl_relay_cache_read(const dbl_relay_cache_read_args* a, dbl_stream_t stream) {
    using namespace dbl;
    if (!a) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: null args");
    int rc = cache_validate(&a->cache, "relay cache read");
    if (rc == DBL_OK) rc = check_table(a->page_table, a->n_seq, a->table_width, a->table_stride, "relay cache read");
    if (rc != DBL_OK) return rc;
    if (a->tokens <= 0) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: tokens must be positive");
    if (a->dtype != DBL_F32 && a->dtype != DBL_BF16)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: dtype must be f32 or bf16");
    if (!a->k || !a->v || !a->lengths)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: k, v and lengths are required");
    if (!aligned(a->k, 16) || !aligned(a->v, 16))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache read: k and v must be 16-byte aligned");
    const int D = (int)a->cache.head_dim;
    const int64_t threads = a->n_seq * a->tokens * a->cache.kv_heads * (D / 8);
    if (a->tokens > 0x7fffffff || threads / 256 > 0x7ffffff0)
        return fail(DBL_ERR_UNSUPPORTED, "relay cache read: grid too large");
    ReadParams p{};
    p.c = cache_view(&a->cache, a->page_table, a->table_width, a->table_stride);
    p.k = a->k;
    p.v = a->v;
    p.lengths = a->lengths;
    p.start = a->start;
    p.N = (int)a->n_seq;
    p.T = (int)a->tokens;
    rc = device_error_record(&p.err);
    if (rc != DBL_OK) return rc;
    const unsigned grid = blocks_for(threads, 256);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == DBL_BF16) {
        if (D == 128) cache_read_kernel<128, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
        else cache_read_kernel<64, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    } else {
        if (D == 128) cache_read_kernel<128, float><<<grid, 256, 0, st>>>(p);
        else cache_read_kernel<64, float><<<grid, 256, 0, st>>>(p);
    }
    return launch_status("cache_read_kernel");
}
