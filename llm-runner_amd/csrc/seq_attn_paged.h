// seq_attn_paged.h - the matrix-core form of attention over a paged cache for requests of any
// number of new tokens (seq_attn.hip, mx4_attn.hip): where its tiles' keys come from, and how the
// tiles of all requests are shared out.
#pragma once

#include "seq_attn_few.h"
#include "seq_attn_tile.h"

namespace llmr {
namespace seqattn {
namespace {

constexpr uint32_t kBlockRows = 256;  // rows of a workgroup of paged_attn_tiles
constexpr uint32_t kPageCap = 4096;   // pages staged at a time: 1020 tiles of the smallest pages
constexpr uint32_t kStageTiles = 1020;

// Keys in the pages of a cache: fragment tiles of 64 keys from key0 on. The request's pages
// lie in LDS, kStageTiles tiles of them at a time, checked (~0: none).
template <uint32_t ROW>
struct PagedKeys {
    static constexpr bool kStages = true, kBlocks4 = false;
    const int32_t* table;  // the request's row of the table
    uint32_t* pages;       // LDS: [kPageCap], then a word: some page is none
    uint32_t key0, n_keys, kvh, n_kv_heads, n_pages, log2, wave;
    uint32_t end = 0, page0 = 0;  // tiles below `end` are staged; the table's column of pages[0]
    bool none = false;
    __device__ __forceinline__ uint32_t stage(uint32_t t, uint32_t n) {
        end = min(n, t + kStageTiles);
        page0 = (key0 + t * kKeys) >> log2;
        const uint32_t last = (key0 + min(n_keys, end * kKeys) - 1u) >> log2;
        for (uint32_t i = threadIdx.x; page0 + i <= last; i += blockDim.x) {
            const uint32_t p = (uint32_t)table[page0 + i];
            pages[i] = p < n_pages ? p : ~0u;
            if (p >= n_pages) pages[kPageCap] = 1u;
        }
        return end;
    }
    __device__ __forceinline__ void staged() { none = __builtin_amdgcn_readfirstlane(pages[kPageCap]) != 0; }
    __device__ __forceinline__ uint32_t page_of(uint32_t k) const {  // of the fragment's key k
        const uint32_t top = min(n_keys, end * kKeys);
        const uint32_t p = pages[((key0 + min(k, top - 1u)) >> log2) - page0];
        return k < top ? p : ~0u;
    }
    // the wave's keys of a tile: 8 wave .. + 7, on one page
    __device__ __forceinline__ uint32_t page(uint32_t t) const { return page_of(t * kKeys + 8u * wave); }
    __device__ __forceinline__ rsrc_t tile(const void* base, uint32_t t, uint32_t page) const {
        return rows_of<ROW>(base, t, page);
    }
    // those keys' rows of R bytes in pages at base
    template <uint32_t R>
    __device__ __forceinline__ rsrc_t rows_of(const void* base, uint32_t t, uint32_t page) const {
        const uint32_t k = t * kKeys + 8u * wave, in = (key0 + k) & ((1u << log2) - 1u);
        const uint32_t left = page == ~0u ? 0u : min(__builtin_elementwise_sub_sat(n_keys, k), 8u);
        const uint64_t off = ((((uint64_t)(page == ~0u ? 0u : page) * n_kv_heads + kvh) << log2) + in) * R;
        return __builtin_amdgcn_make_buffer_rsrc((uint8_t*)const_cast<void*>(base) + off, (short)0,
                                                 (int)__builtin_amdgcn_readfirstlane(left * R), 0x00020000);
    }
    __device__ __forceinline__ uint32_t voffset(uint32_t r, uint32_t chunk) const { return (r & 7u) * ROW + (chunk << 4); }
    __device__ __forceinline__ bool holes() const { return none; }
    __device__ __forceinline__ uint32_t groups(uint32_t t) const {
        uint32_t on = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++)
            on |= (uint32_t)__builtin_amdgcn_readfirstlane(page_of(t * kKeys + 16u * i)) != ~0u ? 1u << i : 0u;
        return on;
    }
    __device__ __forceinline__ const uint8_t* row(const void* base, uint32_t j) const {
        const uint32_t p = (uint32_t)table[(key0 + j) >> log2];
        if (p >= n_pages) return nullptr;
        return (const uint8_t*)base +
               ((((uint64_t)p * n_kv_heads + kvh) << log2) + ((key0 + j) & ((1u << log2) - 1u))) * ROW;
    }
};

// Row blocks of a request, and the keys and 64-key tiles of one (a tile at least: its rows are
// written).
__device__ __forceinline__ uint32_t blocks_of(const PagedRequest& rq, uint32_t G) {
    return (uint32_t)(((uint64_t)rq.rows * G + kBlockRows - 1u) / kBlockRows);
}
__device__ __forceinline__ uint32_t block_keys(const SeqAttnArgs& a, const PagedRequest& rq, uint32_t G, uint32_t b) {
    const uint32_t last = (uint32_t)(min((uint64_t)rq.rows * G, (uint64_t)(b + 1u) * kBlockRows) - 1u) / G;
    const int64_t cap = (int64_t)a.max_pages << a.page_log2;
    return (uint32_t)min(max((int64_t)rq.pos0 + last + 1, (int64_t)0), cap);
}
__device__ __forceinline__ uint32_t block_tiles(const SeqAttnArgs& a, const PagedRequest& rq, uint32_t G, uint32_t b) {
    return max((block_keys(a, rq, G, b) + kKeys - 1u) / kKeys, 1u);
}
// A block's units on the line: its tiles, the first of them kStart units more, for what
// beginning a block costs (pages staged, the first tiles waited for, the end written). Without
// it a workgroup that got ten blocks of one tile was the last by far: 24 requests of 1 to 511
// new tokens 72 us; with 2, 3, 4, 6, 8, 10, 14: 43.4, 41.6, 40.0, 37.3, 37.8, 38.5, 39.6.
constexpr uint32_t kStart = 6;
__device__ __forceinline__ uint64_t request_units(const SeqAttnArgs& a, const PagedRequest& rq, uint32_t G) {
    uint64_t n = 0;
    for (uint32_t b = 0; b < blocks_of(rq, G); b++) n += block_tiles(a, rq, G, b) + kStart;
    return n;
}
template <uint32_t D>
constexpr size_t tile_part_floats() { return kBlockRows * (D + 2u); }

// Attention over a paged cache for requests of any number of new tokens: the units of all
// (request, key/value head, block of 256 rows) make one line that the workgroups, one a CU,
// share evenly, as paged_attn_few's waves do; parts of a block that several workgroups take
// go to scratch, at most two a workgroup, and paged_attn_join joins them.
// keys(PagedKeys): the source of keys that reads what the pages hold.
template <uint32_t T, uint32_t D, typename Keys>
__device__ __forceinline__ void paged_tiles(const SeqAttnArgs& a, uint8_t* lds, JoinRecord* __restrict__ records,
                                            float* __restrict__ scratch, const Keys& keys_of) {
    constexpr uint32_t NW = 8, ROW = D * 2u;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t G = a.n_heads / a.n_kv_heads;
    uint32_t* const pages = (uint32_t*)(lds + lds_bytes<D>());

    const auto cost = [&](const PagedRequest& r) { return request_units(a, r, G); };
    RequestWindow win;
    const uint64_t w = batch_cost(a, win, lane, cost) * a.n_kv_heads;
    const uint32_t n = (uint32_t)min((uint64_t)gridDim.x, w);  // every workgroup has a unit
    JoinRecord rec{};
    if (blockIdx.x >= n) {
        if (tid == 0) records[blockIdx.x].last = 0;
        return;
    }
    uint64_t at = part_begin(blockIdx.x, w, n);
    const uint64_t end = part_begin(blockIdx.x + 1u, w, n);
    uint64_t base;  // units (all heads) before request s
    uint32_t s = find_request(a, win, lane, cost, a.n_kv_heads, at, base);

    while (at < end) {
        if (s - win.s0 >= 64u) win.load(a, s, lane);
        const PagedRequest rq = win.get(s);
        const uint64_t per_head = request_units(a, rq, G), all = per_head * a.n_kv_heads;
        if (all == 0 || at >= base + all) {
            base += all;
            s++;
            continue;
        }
        const uint32_t kvh = (uint32_t)((at - base) / per_head);
        uint64_t x = (at - base) % per_head;
        uint32_t b = 0, tiles;
        while (x >= (tiles = block_tiles(a, rq, G, b)) + kStart) {
            x -= tiles + kStart;
            b++;
        }
        const uint64_t y = min((uint64_t)tiles + kStart, x + (end - at));  // units [x, y) of the block
        const uint32_t t0 = x > kStart ? (uint32_t)x - kStart : 0u, t1 = y > kStart ? (uint32_t)y - kStart : 0u;
        at += y - x;
        if (t0 == t1) continue;  // (of the first tile's units none but the last carries it)
        const uint32_t keys = block_keys(a, rq, G, b), key0 = t0 * kKeys;
        const uint32_t n_keys = min(keys, t1 * kKeys) - min(keys, key0);

        const uint32_t rows = rq.rows * G, row0 = b * kBlockRows;
        const auto out_at = [&]() {
            const uint32_t r = min(row0 + 32u * wave + (lane & 31u), rows - 1u);
            return (uint64_t)(rq.first + r / G) * a.out_stride + (kvh * G + r % G) * D;
        };
        const uint32_t r = min(row0 + 32u * wave + (lane & 31u), rows - 1u), i = r / G;
        RowOfLane row;
        row.live = row0 + 32u * wave + (lane & 31u) < rows;
        const int64_t pos = (int64_t)rq.pos0 + i - key0;  // last key it sees, of this part
        row.lo = 0;
        // not past the part's keys: where a length passes the end of the table, which need not be
        // the end of a tile, what the last tile holds behind them is no key
        row.hi = row.live ? (int)min(max(pos, (int64_t)-1), (int64_t)n_keys - 1) : -1;
        row.q = (const uint8_t*)a.q + 2u * ((uint64_t)(rq.first + i) * a.q_stride + (uint64_t)(kvh * G + r % G) * a.q_head_stride);

        // (the workgroup's last part is done with LDS)
        __syncthreads();
        if (tid == 0) pages[kPageCap] = 0;
        __syncthreads();
        auto src = keys_of(PagedKeys<ROW>{a.table + (size_t)s * a.max_pages, pages, key0, n_keys, kvh, a.n_kv_heads, a.n_pages,
                           a.page_log2, wave});
        float* const part = t0 == 0 && t1 == tiles
                                ? nullptr
                                : scratch + (2u * blockIdx.x + (t0 == 0 ? 1u : 0u)) * tile_part_floats<D>();
        tile_rows<T, D, NW>(a, lds, src, n_keys, row, part, out_at);
        if (t0 == 0 && t1 != tiles)  // (the workgroup's last part: the record is its one)
            rec = JoinRecord{part_of(at + (tiles - t1) - 1u, w, n), rq.first, row0,
                                      min(rows - row0, kBlockRows), kvh, {}};
    }
    if (tid == 0) records[blockIdx.x] = rec;
}

// LDS of a workgroup: the tiles' rings, the staged pages and a flag.
template <uint32_t D>
constexpr uint32_t paged_lds_bytes() { return lds_bytes<D>() + 4u * (kPageCap + 4u); }

}  // namespace
}  // namespace seqattn
}  // namespace llmr
