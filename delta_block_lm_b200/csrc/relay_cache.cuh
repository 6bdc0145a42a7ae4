// The 4-bit relay cache: where the bytes of a token lie, and the pool that a call names.
//
// A pool is [pages][kv_heads][page_size / 16] tiles; a tile holds 16 tokens of one head in 20 D
// bytes (G = D / 32 groups of 32 channels, two codes a byte, the lower code in the lower half):
//   0        key codes     [16 tokens][4 parts t][G groups j][8 codes i]           channel 32 j + 8 t + i
//   8 D      key groups    [16 tokens][G] (scale, minimum) in bf16
//   10 D     value codes   [2 halves u][8 parts g][8 tokens][G groups j][4 codes i]  channel 32 j + 4 g + i
//   18 D     value groups  [16 tokens][G] (scale, minimum) in bf16
// and a channel's value is minimum + scale * code.  The order of the codes is that of the operand
// registers of a 16 x 8 x 16 matrix product, so that a lane's codes of one token are one load: for
// keys a lane holds 8 channels of each group, for values 4.
#pragma once

#include "common.cuh"

namespace dbl {

constexpr int kCacheTile = 16;        // tokens of one tile
constexpr int kCacheErrorPage = 102;  // dbl_device_error: a token whose page is not in the pool

struct CacheView {
    uint8_t* pool;
    const int32_t* table;   // [sequences, table_stride]
    int64_t table_stride;
    int pages, heads, tiles;  // tiles: 16-token tiles of one page
    int width;                // entries of a table row
};

__host__ __device__ __forceinline__ constexpr int cache_tile_bytes(int D) { return 20 * D; }

// The tile of page `page`, head h, tile t of the page.
template <int D>
__device__ __forceinline__ uint8_t* cache_tile(const CacheView& c, int page, int h, int t) {
    return c.pool + (((int64_t)page * c.heads + h) * c.tiles + t) * cache_tile_bytes(D);
}
// The page that holds tile `tile` (counted from the start) of sequence n, or -1 where the table
// has no page of the pool for it.
__device__ __forceinline__ int cache_page(const CacheView& c, int64_t n, int tile) {
    const int slot = tile / c.tiles;
    if (slot >= c.width) return -1;
    const int page = c.table[n * c.table_stride + slot];
    return page >= 0 && page < c.pages ? page : -1;
}

// Offsets inside a tile, for token k (0 .. 15).
template <int D>
struct TileAt {
    static constexpr int G = D / 32;
    static __device__ __forceinline__ int key_word(int k, int t, int j) { return ((k * 4 + t) * G + j) * 4; }
    static __device__ __forceinline__ int key_group(int k, int j) { return 8 * D + (k * G + j) * 4; }
    static __device__ __forceinline__ int value_half(int k, int g, int j) {
        return 10 * D + ((((k >> 3) * 8 + g) * 8 + (k & 7)) * G + j) * 2;
    }
    static __device__ __forceinline__ int value_group(int k, int j) { return 18 * D + (k * G + j) * 4; }
};

// A group's (scale, minimum) word: scale in the lower half, minimum in the upper one.
__device__ __forceinline__ float group_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float group_min(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Check what a call says of its pool and of its page table; `what` names the call.
int cache_validate(const dbl_relay_cache* c, const char* what);
int cache_check_table(const int32_t* table, int64_t n_seq, int64_t width, int64_t stride, const char* what);

inline CacheView cache_view(const dbl_relay_cache* c, const int32_t* table, int64_t width, int64_t stride) {
    CacheView v;
    v.pool = static_cast<uint8_t*>(c->pool);
    v.table = table;
    v.table_stride = stride ? stride : width;
    v.pages = (int)c->pages;
    v.heads = (int)c->kv_heads;
    v.tiles = (int)(c->page_size / kCacheTile);
    v.width = (int)width;
    return v;
}

}  // namespace dbl
