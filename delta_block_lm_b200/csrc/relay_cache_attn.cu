// Attention of single tokens (or a few drafted ones) over the 4-bit relay cache.
//
// Row (n, t, head): scores s_k = scale q.K_k over the keys of [shared prefix ; own sequence], the
// own keys of query t ending at lengths[n] - queries + t; m = max s, l = sum exp(s - m),
// o = sum exp(s - m) V / l, with the statistics [m, l] of the relay merge and its convention for a
// row without keys (o = 0, [0, 1]).
#include <float.h>

#include "relay_cache.cuh"
#include "tc_ptx.cuh"

namespace dbl {

int cache_check_table(const int32_t* table, int64_t n_seq, int64_t width, int64_t stride, const char* what);

namespace {

struct AttnParams {
    CacheView c;
    const void* q;
    int64_t qs[3];  // strides of sequence, query and head
    const int32_t *lengths, *prefix_pages;
    void* out;
    float *row_max, *row_sum;
    int N, Tq, H, group, prefix_len, prefix_width;
    float scale;
    int* err;
};

__device__ __forceinline__ float wsum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// One CTA a row; a warp takes every fourth key, a lane D / 32 channels: lane l holds channels
// 32 j + l of every group j.
template <int D, typename T>
__global__ void __launch_bounds__(128) cache_attn_kernel(const AttnParams p) {
    using At = TileAt<D>;
    constexpr int G = D / 32, NW = 4;
    __shared__ float sm[NW], sl[NW], so[NW][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hq = blockIdx.x % p.H;
    const int t = (blockIdx.x / p.H) % p.Tq;
    const int64_t n = blockIdx.x / p.H / p.Tq;
    const int h = hq / p.group;
    float q[G], acc[G], m = -FLT_MAX, l = 0.f;
#pragma unroll
    for (int j = 0; j < G; ++j) {
        q[j] = to_f32<T>(static_cast<const T*>(p.q)[n * p.qs[0] + t * p.qs[1] + hq * p.qs[2] + 32 * j + lane]) * p.scale;
        acc[j] = 0.f;
    }
    const int own = max(0, p.lengths[n] - p.Tq + t + 1);
    for (int64_t i = warp; i < (int64_t)p.prefix_len + own; i += NW) {
        const bool pre = i < p.prefix_len;
        const int pos = (int)(pre ? i : i - p.prefix_len), tl = pos / kCacheTile;
        int page;
        if (pre) {
            page = tl / p.c.tiles < p.prefix_width ? p.prefix_pages[tl / p.c.tiles] : -1;
            if (page >= p.c.pages) page = -1;
        } else {
            page = cache_page(p.c, n, tl);
        }
        if (page < 0) {
            if (lane == 0) atomicExch(p.err, kCacheErrorPage);
            continue;
        }
        const uint8_t* tile = cache_tile<D>(p.c, page, h, tl % p.c.tiles);
        const int k = pos % kCacheTile;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + At::key_word(k, lane / 8, j));
            const uint32_t g = *reinterpret_cast<const uint32_t*>(tile + At::key_group(k, j));
            s = fmaf(q[j], fmaf(group_scale(g), (float)(w >> (4 * (lane % 8)) & 15u), group_min(g)), s);
        }
        s = wsum(s);
        const float mn = fmaxf(m, s), corr = expf(m - mn), e = expf(s - mn);
        m = mn;
        l = l * corr + e;
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const uint32_t w = *reinterpret_cast<const uint16_t*>(tile + At::value_half(k, lane / 4, j));
            const uint32_t g = *reinterpret_cast<const uint32_t*>(tile + At::value_group(k, j));
            acc[j] = acc[j] * corr + e * fmaf(group_scale(g), (float)(w >> (4 * (lane % 4)) & 15u), group_min(g));
        }
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int j = 0; j < G; ++j) so[warp][32 * j + lane] = acc[j];
    __syncthreads();
    float mx = -FLT_MAX;
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sm[w]);
    float sum = 0.f;
    for (int w = 0; w < NW; ++w) sum += sl[w] == 0.f ? 0.f : sl[w] * expf(sm[w] - mx);
    const bool empty = (int64_t)p.prefix_len + own == 0 || sum == 0.f;
    for (int d = threadIdx.x; d < D; d += 128) {
        float o = 0.f;
        for (int w = 0; w < NW; ++w) o += sl[w] == 0.f ? 0.f : so[w][d] * expf(sm[w] - mx);
        static_cast<T*>(p.out)[(int64_t)blockIdx.x * D + d] = from_f32<T>(empty ? 0.f : o / sum);
    }
    if (threadIdx.x == 0) {
        if (p.row_max) p.row_max[blockIdx.x] = empty ? 0.f : mx;
        if (p.row_sum) p.row_sum[blockIdx.x] = empty ? 1.f : sum;
    }
}

}  // namespace
}  // namespace dbl

extern "C" size_t dbl_relay_cache_attention_workspace_bytes(const dbl_relay_cache_attention_args* a) {
    (void)a;
    return 0;
}

extern "C" int dbl_relay_cache_attention(const dbl_relay_cache_attention_args* a, void* workspace,
                                         size_t workspace_bytes, dbl_stream_t stream) {
    using namespace dbl;
    (void)workspace;
    (void)workspace_bytes;
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
    if (!a->q || !a->out || !a->lengths)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: q, out and lengths are required");
    if (a->prefix_len < 0 || a->prefix_len > 0x7fffffff || a->prefix_width < 0 || a->prefix_width > 0x7fffffff)
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: prefix_len out of range");
    if (a->prefix_len > 0 && (!a->prefix_pages || a->prefix_width * a->cache.page_size < a->prefix_len))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: prefix_pages must hold prefix_len tokens");
    const int D = (int)a->cache.head_dim;
    const int64_t dims[4] = {a->n_seq, a->queries, a->heads, D};
    int64_t qs[4];
    resolve_strides(a->q_stride, dims, 4, qs);
    if (qs[3] != 1) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache attention: the innermost stride of q must be 1");
    if (a->queries > 0x7fffffff || a->heads > 0x7fffffff || a->n_seq * a->queries > 0x7fffffff / a->heads)
        return fail(DBL_ERR_UNSUPPORTED, "relay cache attention: sizes exceed 32-bit limits");
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
    rc = device_error_record(&p.err);
    if (rc != DBL_OK) return rc;
    const unsigned grid = (unsigned)(a->n_seq * a->queries * a->heads);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == DBL_BF16) {
        if (D == 128) cache_attn_kernel<128, __nv_bfloat16><<<grid, 128, 0, st>>>(p);
        else cache_attn_kernel<64, __nv_bfloat16><<<grid, 128, 0, st>>>(p);
    } else {
        if (D == 128) cache_attn_kernel<128, float><<<grid, 128, 0, st>>>(p);
        else cache_attn_kernel<64, float><<<grid, 128, 0, st>>>(p);
    }
    return launch_status("cache_attn_kernel");
}
