// Pages of the relay cache: releasing, forking, reserving (with copy on write), compacting, copying.
//
// The state is three int32 arrays on the device -- the page table [S, W] (-1: no page), lengths [S]
// and refs [P] (how many table entries hold a page) -- and every call works on the device alone, so
// that a serving loop neither waits for the host nor leaves a CUDA graph.  Where a call hands out
// pages it takes the free page with the lowest number first, in the order of sequences and slots,
// and integer atomics only count and take maxima, so the results do not depend on the order in which
// threads run.
//
// The integer work is one CTA of 1024 threads, or for large states a cluster of 8: its phases are
// separated by the barrier, which orders global memory among its threads, so each call is one launch
// (two with the copies of page data, which use the whole GPU).
#include "relay_cache.cuh"
#include "tc_ptx.cuh"

namespace dbl {

namespace {

constexpr int CT = 1024;             // threads of a CTA
constexpr int MOST_WARPS = 8 * CT / 32;
// Table entries and pages that one CTA deals with.  Measured, release + fork + reserve, by one CTA and by eight: 8
// sequences (74 entries and pages) and 32 (308) 18 and 25 us, 256 (14 K) 71 and 35 us.
constexpr int64_t kSmallState = 4096;

struct PageParams {
    const int32_t *table, *lengths, *refs;      // before
    int32_t *table_out, *lengths_out, *refs_out;  // after; may be the same arrays
    int64_t stride;                             // of table and table_out rows
    int S, W, P, page;
    const int32_t *a, *b;                       // the call's lists
    int n;                                      // their length
    int tokens;                                 // reserve: tokens of every sequence where b is null
    int32_t* result;                            // reserve: pages missing; compact: pages in use
    int32_t* scratch;
    int* err;
};

template <int CL>  // CTAs of the launch
__device__ __forceinline__ void sync_all() {
    if constexpr (CL == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ int gtid() { return blockIdx.x * CT + threadIdx.x; }
__device__ __forceinline__ int gwarp() { return gtid() >> 5; }
__device__ __forceinline__ int lane_id() { return threadIdx.x & 31; }
__device__ __forceinline__ int ld(const int32_t* p) { return __ldcg(p); }

__device__ __forceinline__ int wsum_i(int x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// Sum of v[0 .. count) by one warp.
__device__ __forceinline__ int warp_total(const int32_t* v, int count) {
    int s = 0;
    for (int i = lane_id(); i < count; i += 32) s += ld(v + i);
    return wsum_i(s);
}
__device__ __forceinline__ int64_t entry(const PageParams& p, int s, int w) { return (int64_t)s * p.stride + w; }

template <int CL>
__device__ void copy_state(const PageParams& p, bool lengths) {
    constexpr int NT = CL * CT;
    // in place there is nothing to copy
    if (p.table_out != p.table)
        for (int64_t i = gtid(); i < (int64_t)p.S * p.W; i += NT) {
            const int s = (int)(i / p.W), w = (int)(i % p.W);
            p.table_out[entry(p, s, w)] = p.table[entry(p, s, w)];
        }
    if (p.refs_out != p.refs)
        for (int i = gtid(); i < p.P; i += NT) p.refs_out[i] = p.refs[i];
    if (lengths && p.lengths_out != p.lengths)
        for (int i = gtid(); i < p.S; i += NT) p.lengths_out[i] = p.lengths[i];
}

// a = the sequences to release.  An entry that two list items name is released once.
template <int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(CT, 1) cache_release_kernel(const PageParams p) {
    constexpr int NT = CL * CT;
    copy_state<CL>(p, true);
    sync_all<CL>();
    for (int64_t i = gtid(); i < (int64_t)p.n * p.W; i += NT) {
        const int s = p.a[i / p.W];
        if (s < 0 || s >= p.S) {
            atomicExch(p.err, kCacheErrorPage);
            continue;
        }
        const int page = atomicExch(p.table_out + entry(p, s, (int)(i % p.W)), -1);
        if (page >= 0 && page < p.P) atomicSub(p.refs_out + page, 1);
        if (i % p.W == 0) p.lengths_out[s] = 0;
    }
}

// a = parents, b = children (each named once, none of them a parent), which give back the pages that they hold.
template <int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(CT, 1) cache_fork_kernel(const PageParams p) {
    constexpr int NT = CL * CT;
    copy_state<CL>(p, true);
    sync_all<CL>();
    for (int64_t i = gtid(); i < (int64_t)p.n * p.W; i += NT) {
        const int from = p.a[i / p.W], to = p.b[i / p.W], w = (int)(i % p.W);
        if (from < 0 || from >= p.S || to < 0 || to >= p.S || from == to) {
            atomicExch(p.err, kCacheErrorPage);
            continue;
        }
        const int len = ld(p.lengths_out + from);
        const int page = (int64_t)w * p.page < len ? ld(p.table_out + entry(p, from, w)) : -1;
        const int old = atomicExch(p.table_out + entry(p, to, w), page);  // reserve may have given it pages
        if (old >= 0 && old < p.P) atomicSub(p.refs_out + old, 1);
        if (page >= 0 && page < p.P) atomicAdd(p.refs_out + page, 1);
        if (w == 0) p.lengths_out[to] = len;
    }
}

// Gives every slot [first, end) of every sequence s to visit(s, w): a thread takes a sequence and its first slot; where
// there are more (prompts), its warp takes them together.  range(s, first, end) says which slots.
template <int CL, typename Range, typename Visit>
__device__ __forceinline__ void each_slot(int S, Range range, Visit visit) {
    for (int s0 = gwarp() * 32; s0 < S; s0 += CL * CT) {
        const int s = s0 + lane_id();
        int first = 0, end = 0;
        if (s < S) range(s, first, end);
        if (first < end) visit(s, first);
        for (unsigned more = __ballot_sync(0xffffffffu, end - first > 1); more; more &= more - 1) {
            const int l = __ffs(more) - 1, w1 = __shfl_sync(0xffffffffu, end, l);
            for (int w = __shfl_sync(0xffffffffu, first, l) + 1 + lane_id(); w < w1; w += 32) visit(s0 + l, w);
        }
    }
}

// b = tokens of each sequence, or null: p.tokens of each.
//   scratch: asked [P], last [P], list [P], src [S], dst [S], tiles [S], free [NWARP], want [NWARP]
template <int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(CT, 1) cache_reserve_kernel(const PageParams p) {
    constexpr int NT = CL * CT, NWARP = NT / 32;
    asm volatile("griddepcontrol.launch_dependents;");  // the copies' CTAs may come up meanwhile
    int32_t *asked = p.scratch, *last = asked + p.P, *list = last + p.P;
    int32_t *src = list + p.P, *dst = src + p.S, *tiles = dst + p.S, *nfree = tiles + p.S, *nwant = nfree + NWARP;
    const int warp = gwarp(), lane = lane_id();
    copy_state<CL>(p, false);
    // the slots that the next tokens of sequence s are written to: [len / page, end), cut to the table
    int len, add;
    auto range = [&](int s, int& first, int& end) -> bool {  // false: the table has no slots for some of the tokens
        len = max(p.lengths[s], 0);
        add = max(p.b ? p.b[s] : p.tokens, 0);
        first = len / p.page;
        const int64_t past = add ? ((int64_t)len + add + p.page - 1) / p.page : 0;
        end = (int)min(past, (int64_t)p.W);
        return past <= p.W;
    };
    auto held = [&](int s, int w) {  // the page that slot w holds, or -1
        const int page = ld(p.table + entry(p, s, w));
        return page >= 0 && page < p.P ? page : -1;
    };
    // Who is about to write to a page: how many, and the last of them.  Lengths are the caller's and may have been
    // lowered, so any page of a range may be one that others hold too, not only the one that the range begins in.
    each_slot<CL>(p.S, range, [&](int s, int w) {
        const int page = held(s, w);
        if (page >= 0) asked[page] = 0, last[page] = -1;
    });
    sync_all<CL>();
    each_slot<CL>(p.S, range, [&](int s, int w) {
        const int page = held(s, w);
        if (page >= 0) {
            atomicAdd(asked + page, 1);
            atomicMax(last + page, s);
        }
    });
    sync_all<CL>();
    // A holder replaces the page it is about to write where others hold it too; if all of its holders are about to
    // write, the last of them keeps it.  Only that last one asks for the page's references, which it alone changes below.
    auto replaces = [&](int s, int page) {
        if (ld(last + page) != s) return true;
        const int r = ld(p.refs + page);
        return r > 1 && ld(asked + page) < r;
    };
    // does slot w of sequence s need a page?
    auto wants = [&](int s, int w, int& page) {
        page = held(s, w);
        if (page >= 0) return replaces(s, page);
        return (int64_t)w * p.page >= len && ld(p.table + entry(p, s, w)) < 0;
    };
    const int rows = (p.S + NWARP - 1) / NWARP, s0 = min(p.S, warp * rows), s1 = min(p.S, s0 + rows);
    const int pages = (p.P + NWARP - 1) / NWARP, p0 = min(p.P, warp * pages), p1 = min(p.P, p0 + pages);
    int want = 0, first, end, page;
    bool beyond = false;
    for (int s = s0; s < s1; ++s) {
        if (!range(s, first, end)) beyond = true;
        if (lane == 0) src[s] = -1;
        for (int w = first; w < end; w += 32) {
            const bool need = w + lane < end && wants(s, w + lane, page);
            if (need && page >= 0 && lane == 0 && w == first && len % p.page) src[s] = page;  // it holds tokens: a copy
            want += __popc(__ballot_sync(0xffffffffu, need));
        }
    }
    int nf = 0;
    for (int i = p0 + lane; i < p1; i += 32) nf += p.refs[i] == 0;
    nf = wsum_i(nf);
    if (lane == 0) {
        nfree[warp] = nf;
        nwant[warp] = want;
        if (beyond) atomicExch(p.err, kCacheErrorPage);
    }
    sync_all<CL>();
    const int total_want = warp_total(nwant, NWARP), total_free = warp_total(nfree, NWARP);
    const bool ok = total_want <= total_free;
    if (gtid() == 0) p.result[0] = ok ? 0 : total_want - total_free;
    int at = warp_total(nfree, warp);
    for (int i = p0; i < p1 && at < total_want && ok; i += 32) {
        const bool f = i + lane < p1 && p.refs[i + lane] == 0;
        const unsigned m = __ballot_sync(0xffffffffu, f);
        const int r = at + __popc(m & ((1u << lane) - 1));
        if (f && r < total_want) list[r] = i + lane;
        at += __popc(m);
    }
    sync_all<CL>();
    at = warp_total(nwant, warp);
    for (int s = s0; s < s1; ++s) {
        range(s, first, end);
        if (lane == 0) {
            if (!ok) src[s] = -1;
            tiles[s] = (len % p.page + kCacheTile - 1) / kCacheTile;
        }
        if (!ok) continue;
        for (int w = first; w < end; w += 32) {
            const bool in = w + lane < end, need = in && wants(s, w + lane, page);
            const unsigned m = __ballot_sync(0xffffffffu, need);
            if (in && page >= 0 && ld(last + page) == s) {  // what the page's holders that are about to write leave
                const int r = ld(p.refs + page), a = ld(asked + page);
                if (r > 1) p.refs_out[page] = a < r ? r - a : 1;
            }
            if (need) {
                const int fresh = ld(list + at + __popc(m & ((1u << lane) - 1)));
                p.table_out[entry(p, s, w + lane)] = fresh;
                p.refs_out[fresh] = 1;
                if (w + lane == first) dst[s] = fresh;
            }
            at += __popc(m);
        }
    }
}

// Pages in use move to the front: the i-th page in use at or past `used` goes to the i-th free page
// below it.   scratch: count [2], src [P], dst [P], to [P], inuse [NWARP]
template <int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(CT, 1) cache_compact_kernel(const PageParams p) {
    constexpr int NT = CL * CT, NWARP = NT / 32;
    asm volatile("griddepcontrol.launch_dependents;");  // the copies' CTAs may come up meanwhile
    int32_t *count = p.scratch, *src = count + 2, *dst = src + p.P, *to = dst + p.P, *inuse = to + p.P;
    const int warp = gwarp(), lane = lane_id();
    const int pages = (p.P + NWARP - 1) / NWARP, p0 = min(p.P, warp * pages), p1 = min(p.P, p0 + pages);
    int nu = 0;
    for (int i = p0 + lane; i < p1; i += 32) nu += p.refs[i] > 0;
    nu = wsum_i(nu);
    if (lane == 0) inuse[warp] = nu;
    sync_all<CL>();
    const int used = warp_total(inuse, NWARP), before = warp_total(inuse, warp);
    if (gtid() == 0) p.result[0] = used;
    if (p0 <= used && used < p1) {  // pages in use below `used`
        int c = 0;
        for (int i = p0 + lane; i < used; i += 32) c += p.refs[i] > 0;
        c = wsum_i(c);
        if (lane == 0) count[1] = before + c;
    }
    if (used == p.P && gtid() == 0) count[1] = used;
    sync_all<CL>();
    const int below = ld(count + 1);
    if (gtid() == 0) count[0] = used - below;
    int at = before;
    for (int i = p0; i < p1; i += 32) {
        const bool in = i + lane < p1, u = in && p.refs[i + lane] > 0;
        const unsigned m = __ballot_sync(0xffffffffu, u);
        const int r = at + __popc(m & ((1u << lane) - 1)), page = i + lane;
        if (u && page >= used) src[r - below] = page;
        if (in && !u && page < used) dst[page - r] = page;
        if (in && !u && page >= used) to[page] = page;  // no entry names it
        at += __popc(m);
    }
    sync_all<CL>();
    for (int i = gtid(); i < used - below; i += NT) to[ld(src + i)] = ld(dst + i);
    if (p.refs_out != p.refs)
        for (int i = gtid(); i < p.P; i += NT) p.refs_out[i] = p.refs[i];
    sync_all<CL>();
    for (int i = gtid(); i < used - below; i += NT) {
        const int a = ld(src + i);
        p.refs_out[ld(dst + i)] = ld(p.refs + a);
        p.refs_out[a] = 0;
    }
    for (int64_t i = gtid(); i < (int64_t)p.S * p.W; i += NT) {
        const int64_t e = entry(p, (int)(i / p.W), (int)(i % p.W));
        const int page = p.table[e];
        p.table_out[e] = page >= used && page < p.P ? ld(to + page) : page;
    }
}

struct CopyParams {
    uint4* pool;
    const int32_t *src, *dst, *tiles;  // tiles: of each pair, or null: all
    const int32_t* count;              // on the device, or null
    int n, pages, heads, page_tiles, tile_words;
    int* err;
};

// Copies pages src[i] -> dst[i]; one CTA a (pair, head) at a time.  Bound by HBM: 1024 pages of 160 KB (335 MB
// read and written) take 57 of a compaction's 66 us (5900 GB/s, 90% of the measured copy rate).  Grids of 16, 64,
// 128 and 512 CTAs an SM: 70, 66, 66 and 87 us (a compaction's list is shorter than the host knows).
__global__ void __launch_bounds__(128) cache_copy_kernel(const CopyParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // after a plan: its lists are complete
    const int n = p.count ? min(*p.count, p.n) : p.n;
    const int64_t jobs = (int64_t)n * p.heads;
    for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const int i = (int)(job / p.heads), h = (int)(job % p.heads);
        const int a = p.src[i];
        if (a == -1 && p.tiles) continue;  // a pair that reserve left out
        const int b = p.dst[i];
        if (a < 0 || a >= p.pages || b < 0 || b >= p.pages) {
            if (threadIdx.x == 0) atomicExch(p.err, kCacheErrorPage);
            continue;
        }
        const int words = (p.tiles ? min(p.tiles[i], p.page_tiles) : p.page_tiles) * p.tile_words;
        const int64_t per = (int64_t)p.page_tiles * p.tile_words;
        const uint4* from = p.pool + ((int64_t)a * p.heads + h) * per;
        uint4* to = p.pool + ((int64_t)b * p.heads + h) * per;
        constexpr int U = 5;  // words of a thread on their way at once: 10 KB of a page of 64 tokens
        for (int w0 = threadIdx.x; w0 < words; w0 += 128 * U) {
            uint4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (w0 + 128 * u < words) x[u] = from[w0 + 128 * u];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (w0 + 128 * u < words) to[w0 + 128 * u] = x[u];
        }
    }
}

int launch_copy(const dbl_relay_cache& c, const int32_t* src, const int32_t* dst, const int32_t* tiles,
                const int32_t* count, int64_t n, int* err, bool after_plan, cudaStream_t st) {
    CopyParams q{};
    q.pool = static_cast<uint4*>(c.pool);
    q.src = src;
    q.dst = dst;
    q.tiles = tiles;
    q.count = count;
    q.n = (int)n;
    q.pages = (int)c.pages;
    q.heads = (int)c.kv_heads;
    q.page_tiles = (int)(c.page_size / kCacheTile);
    q.tile_words = cache_tile_bytes((int)c.head_dim) / 16;
    q.err = err;
    const int64_t jobs = n * c.kv_heads, most = 148 * 64;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(jobs < most ? jobs : most));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = after_plan ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, cache_copy_kernel, q), "cache_copy_kernel");
}

// Fills what every call has in common.
int page_params(const dbl_relay_cache_pages_args* a, PageParams& p, const char* what, bool lengths) {
    if (!a) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: null args", what);
    int rc = cache_validate(&a->cache, what);
    if (rc == DBL_OK) rc = cache_check_table(a->page_table, a->n_seq, a->table_width, a->table_stride, what);
    if (rc != DBL_OK) return rc;
    if (!a->refs || !a->page_table_out || !a->refs_out || (lengths && !a->lengths))
        return fail(DBL_ERR_INVALID_ARGUMENT, "%s: the page table, refs and lengths and their outputs are required", what);
    p.table = a->page_table;
    p.lengths = a->lengths;
    p.refs = a->refs;
    p.table_out = a->page_table_out;
    p.lengths_out = a->lengths_out;
    p.refs_out = a->refs_out;
    p.stride = a->table_stride ? a->table_stride : a->table_width;
    p.S = (int)a->n_seq;
    p.W = (int)a->table_width;
    p.P = (int)a->cache.pages;
    p.page = (int)a->cache.page_size;
    return DBL_OK;
}

// One CTA, or a cluster.
bool small_state(const PageParams& p) { return (int64_t)p.S * p.W + p.P <= kSmallState; }

size_t page_scratch(int64_t P, int64_t S) { return (size_t)(4 * P + 3 * S + 2 * MOST_WARPS + 16) * sizeof(int32_t); }

int check_scratch(const dbl_relay_cache_pages_args* a, PageParams& p, void* ws, size_t bytes, const char* what) {
    const size_t need = page_scratch(a->cache.pages, a->n_seq);
    if (!ws || bytes < need) return fail(DBL_ERR_WORKSPACE, "%s: workspace of %zu bytes required (got %zu)", what, need, bytes);
    if (!aligned(ws, 16)) return fail(DBL_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", what);
    p.scratch = static_cast<int32_t*>(ws);
    return DBL_OK;
}

}  // namespace
}  // namespace dbl

extern "C" size_t dbl_relay_cache_pages_workspace_bytes(int64_t pages, int64_t n_seq) {
    if (pages <= 0 || n_seq <= 0) return 0;
    return dbl::page_scratch(pages, n_seq);
}

extern "C" int dbl_relay_cache_release(const dbl_relay_cache_pages_args* a, const int32_t* sequences, int64_t count,
                                       dbl_stream_t stream) {
    using namespace dbl;
    PageParams p{};
    int rc = page_params(a, p, "relay cache release", true);
    if (rc != DBL_OK) return rc;
    if (!a->lengths_out) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache release: lengths_out is required");
    if (count < 0 || count > 0x7fffffff || (count > 0 && !sequences))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache release: bad list of sequences");
    p.a = sequences;
    p.n = (int)count;
    if ((rc = device_error_record(&p.err)) != DBL_OK) return rc;
    const auto st = reinterpret_cast<cudaStream_t>(stream);
    if (small_state(p)) cache_release_kernel<1><<<1, CT, 0, st>>>(p);
    else cache_release_kernel<8><<<8, CT, 0, st>>>(p);
    return launch_status("cache_release_kernel");
}

extern "C" int dbl_relay_cache_fork(const dbl_relay_cache_pages_args* a, const int32_t* parents, const int32_t* children,
                                    int64_t count, dbl_stream_t stream) {
    using namespace dbl;
    PageParams p{};
    int rc = page_params(a, p, "relay cache fork", true);
    if (rc != DBL_OK) return rc;
    if (!a->lengths_out) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache fork: lengths_out is required");
    if (count < 0 || count > 0x7fffffff || (count > 0 && (!parents || !children)))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache fork: bad lists of parents and children");
    p.a = parents;
    p.b = children;
    p.n = (int)count;
    if ((rc = device_error_record(&p.err)) != DBL_OK) return rc;
    const auto st = reinterpret_cast<cudaStream_t>(stream);
    if (small_state(p)) cache_fork_kernel<1><<<1, CT, 0, st>>>(p);
    else cache_fork_kernel<8><<<8, CT, 0, st>>>(p);
    return launch_status("cache_fork_kernel");
}

extern "C" int dbl_relay_cache_reserve(const dbl_relay_cache_pages_args* a, const int32_t* counts, int64_t tokens,
                                       int32_t* missing, void* workspace, size_t workspace_bytes, dbl_stream_t stream) {
    using namespace dbl;
    PageParams p{};
    int rc = page_params(a, p, "relay cache reserve", true);
    if (rc != DBL_OK) return rc;
    if (!missing) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache reserve: missing is required");
    if (!counts && (tokens < 0 || tokens > 0x3fffffff))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache reserve: tokens out of range");
    if ((rc = check_scratch(a, p, workspace, workspace_bytes, "relay cache reserve")) != DBL_OK) return rc;
    p.b = counts;
    p.tokens = (int)tokens;
    p.result = missing;
    if ((rc = device_error_record(&p.err)) != DBL_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (small_state(p)) cache_reserve_kernel<1><<<1, CT, 0, st>>>(p);
    else cache_reserve_kernel<8><<<8, CT, 0, st>>>(p);
    if ((rc = launch_status("cache_reserve_kernel")) != DBL_OK) return rc;
    const int32_t* src = p.scratch + 3 * (int64_t)p.P;
    return launch_copy(a->cache, src, src + p.S, src + 2 * (int64_t)p.S, nullptr, p.S, p.err, true, st);
}

extern "C" int dbl_relay_cache_compact(const dbl_relay_cache_pages_args* a, int32_t* used, void* workspace,
                                       size_t workspace_bytes, dbl_stream_t stream) {
    using namespace dbl;
    PageParams p{};
    int rc = page_params(a, p, "relay cache compact", false);
    if (rc != DBL_OK) return rc;
    if (!used) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache compact: used is required");
    if ((rc = check_scratch(a, p, workspace, workspace_bytes, "relay cache compact")) != DBL_OK) return rc;
    p.result = used;
    if ((rc = device_error_record(&p.err)) != DBL_OK) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (small_state(p)) cache_compact_kernel<1><<<1, CT, 0, st>>>(p);
    else cache_compact_kernel<8><<<8, CT, 0, st>>>(p);
    if ((rc = launch_status("cache_compact_kernel")) != DBL_OK) return rc;
    const int32_t* src = p.scratch + 2;
    return launch_copy(a->cache, src, src + p.P, nullptr, p.scratch, p.P, p.err, true, st);
}

extern "C" int dbl_relay_cache_copy_pages(const dbl_relay_cache* c, const int32_t* src, const int32_t* dst,
                                          int64_t count, dbl_stream_t stream) {
    using namespace dbl;
    if (!c) return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache copy: null cache");
    int rc = cache_validate(c, "relay cache copy");
    if (rc != DBL_OK) return rc;
    if (count < 0 || count > 0x7fffffff || (count > 0 && (!src || !dst)))
        return fail(DBL_ERR_INVALID_ARGUMENT, "relay cache copy: bad lists of pages");
    if (count == 0) return DBL_OK;
    int* err = nullptr;
    if ((rc = device_error_record(&err)) != DBL_OK) return rc;
    return launch_copy(*c, src, dst, nullptr, nullptr, count, err, false, reinterpret_cast<cudaStream_t>(stream));
}
