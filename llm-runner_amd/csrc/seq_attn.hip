// seq_attn.hip - causal attention of a batch of requests (llmr_prompt_attention,
// llmr_paged_attention): grouped heads, packed rows, keys in the packed rows or in
// the pages of a cache.
//
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,  p_j = exp2(c (<q[t, h], k[j, h / G]> - m))
//
// c = scale * log2(e), m the largest of the row's products so far (subtracted before
// the scaling: a product of the type's lowest value times log2(e) is past f32).
#include "seq_attn_few.h"
#include "seq_attn_tile.h"

namespace llmr {
namespace {

// Keys in packed rows: a tile's descriptor starts at its first key and ends with the
// workgroup's last.
struct PackedKeys {
    static constexpr bool kStages = false;
    uint64_t first;    // element offset of key 0 of the key/value head
    uint32_t stride2;  // bytes between keys
    uint32_t n_keys;
    __device__ __forceinline__ uint32_t stage(uint32_t, uint32_t n) { return n; }
    __device__ __forceinline__ uint32_t page(uint32_t) const { return 0; }
    __device__ __forceinline__ rsrc_t tile(const void* base, uint32_t t, uint32_t) const {
        // a saturating subtraction, not a comparison and a difference: from the latter's
        // difference for K(t+4) hipcc took n_keys >= 64 (t+4) as given and left V(t+2) without
        // its end, which read past the rows
        const uint32_t k0 = t * seqattn::kKeys;
        const uint32_t left = min(__builtin_elementwise_sub_sat(n_keys, k0), seqattn::kKeys);
        // readfirstlane keeps the descriptor in scalar registers
        return __builtin_amdgcn_make_buffer_rsrc(
            (uint8_t*)const_cast<void*>(base) + 2u * first + (uint64_t)k0 * stride2, (short)0,
            (int)__builtin_amdgcn_readfirstlane(left * stride2), 0x00020000);
    }
    __device__ __forceinline__ uint32_t voffset(uint32_t r, uint32_t chunk) const { return r * stride2 + (chunk << 4); }
    __device__ __forceinline__ bool holes() const { return false; }
    __device__ __forceinline__ uint32_t groups(uint32_t) const { return 15u; }
    __device__ __forceinline__ const uint8_t* row(const void* base, uint32_t j) const {
        return (const uint8_t*)base + 2u * first + (uint64_t)j * stride2;
    }
};

// The request of row t: the first one that ends behind it (n_seqs: none).
__device__ __forceinline__ uint32_t request_of(const int32_t* offsets, uint32_t lo, uint32_t n_seqs, uint32_t t) {
    uint32_t hi = n_seqs;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (offsets[mid + 1u] > (int32_t)t) hi = mid;
        else lo = mid + 1u;
    }
    return lo;
}

// Workgroup L: key/value head L % n_kv_heads (heads side by side, so that with eight of
// them each has an XCD's L2 of its own), row blocks from the last one down (the longest
// of a prompt start first).
template <uint32_t T, uint32_t D, uint32_t NW>
__global__ void __launch_bounds__(64 * NW, 1) prompt_attn_tiles(SeqAttnArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[seqattn::lds_bytes<D>()];
    constexpr uint32_t ROWS = 32u * NW;
    const uint32_t kvh = blockIdx.x % a.n_kv_heads, G = a.n_heads / a.n_kv_heads;
    const uint32_t rows = a.n_tokens * G, blocks = (rows + ROWS - 1u) / ROWS;
    const uint32_t row0 = (blocks - 1u - blockIdx.x / a.n_kv_heads) * ROWS;
    const uint32_t t0 = row0 / G, t1 = min(row0 + ROWS - 1u, rows - 1u) / G;
    const uint32_t s0 = request_of(a.offsets, 0, a.n_seqs, t0);
    if (s0 == a.n_seqs) return;  // rows behind the last request
    const int32_t start0 = a.offsets[s0], end0 = a.offsets[s0 + 1u];
    // keys from the first request's first row (t0: no request has it) to the last row
    const uint32_t kv0 = start0 <= (int32_t)t0 ? (uint32_t)max(start0, 0) : t0;

    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t r = min(row0 + 32u * wave + (lane & 31u), rows - 1u);
    const uint32_t tok = r / G, head = kvh * G + r % G;
    seqattn::RowOfLane row;
    row.live = row0 + 32u * wave + (lane & 31u) < rows;
    int32_t start = start0;
    if ((int32_t)tok >= end0) {
        const uint32_t s = request_of(a.offsets, s0 + 1u, a.n_seqs, tok);
        start = s < a.n_seqs ? a.offsets[s] : 0x7fffffff;
    }
    row.live = row.live && start <= (int32_t)tok;
    const uint32_t lo = (uint32_t)max(start, 0);
    row.lo = lo > kv0 ? (int)(lo - kv0) : 0;
    row.hi = row.live ? (int)(tok - kv0) : -1;
    row.q = (const uint8_t*)a.q + 2u * ((uint64_t)tok * a.q_stride + (uint64_t)head * a.q_head_stride);
    PackedKeys src{(uint64_t)kv0 * a.kv_stride + (uint64_t)kvh * a.kv_head_stride, a.kv_stride * 2u, t1 + 1u - kv0};
    seqattn::tile_rows<T, D, NW>(a, lds, src, t1 + 1u - kv0, row, nullptr, [&]() {
        const uint32_t x = min(row0 + 32u * wave + (lane & 31u), rows - 1u);
        return (uint64_t)(x / G) * a.out_stride + (kvh * G + x % G) * D;
    });
}

template <uint32_t T, uint32_t D, uint32_t NW>
hipError_t launch_tiles(const SeqAttnArgs& a, hipStream_t st) {
    const uint32_t blocks = (a.n_tokens * (a.n_heads / a.n_kv_heads) + 32u * NW - 1u) / (32u * NW);
    hipLaunchKernelGGL((prompt_attn_tiles<T, D, NW>), dim3(blocks * a.n_kv_heads), dim3(64 * NW), 0, st, a);
    return hipGetLastError();
}

using seqattn::PagedRequest;
constexpr uint32_t kBlockRows = 256;  // rows of a workgroup of paged_attn_tiles
constexpr uint32_t kPageCap = 4096;   // pages staged at a time: 1020 tiles of the smallest pages
constexpr uint32_t kStageTiles = 1020;

// Keys in the pages of a cache: fragment tiles of 64 keys from key0 on. The request's pages
// lie in LDS, kStageTiles tiles of them at a time, checked (~0: none).
template <uint32_t ROW>
struct PagedKeys {
    static constexpr bool kStages = true;
    const int32_t* table;  // the request's row of the table
    uint32_t* pages;       // LDS: [kPageCap], then a word: some page is none
    uint32_t key0, n_keys, kvh, n_kv_heads, n_pages, log2, wave;
    uint32_t end = 0, page0 = 0;  // tiles below `end` are staged; the table's column of pages[0]
    bool none = false;
    __device__ __forceinline__ uint32_t stage(uint32_t t, uint32_t n) {
        end = min(n, t + kStageTiles);
        page0 = (key0 + t * seqattn::kKeys) >> log2;
        const uint32_t last = (key0 + min(n_keys, end * seqattn::kKeys) - 1u) >> log2;
        for (uint32_t i = threadIdx.x; page0 + i <= last; i += blockDim.x) {
            const uint32_t p = (uint32_t)table[page0 + i];
            pages[i] = p < n_pages ? p : ~0u;
            if (p >= n_pages) pages[kPageCap] = 1u;
        }
        return end;
    }
    __device__ __forceinline__ void staged() { none = __builtin_amdgcn_readfirstlane(pages[kPageCap]) != 0; }
    __device__ __forceinline__ uint32_t page_of(uint32_t k) const {  // of the fragment's key k
        const uint32_t top = min(n_keys, end * seqattn::kKeys);
        const uint32_t p = pages[((key0 + min(k, top - 1u)) >> log2) - page0];
        return k < top ? p : ~0u;
    }
    // the wave's keys of a tile: 8 wave .. + 7, on one page
    __device__ __forceinline__ uint32_t page(uint32_t t) const { return page_of(t * seqattn::kKeys + 8u * wave); }
    __device__ __forceinline__ rsrc_t tile(const void* base, uint32_t t, uint32_t page) const {
        const uint32_t k = t * seqattn::kKeys + 8u * wave, in = (key0 + k) & ((1u << log2) - 1u);
        const uint32_t left = page == ~0u ? 0u : min(__builtin_elementwise_sub_sat(n_keys, k), 8u);
        const uint64_t off = ((((uint64_t)(page == ~0u ? 0u : page) * n_kv_heads + kvh) << log2) + in) * ROW;
        return __builtin_amdgcn_make_buffer_rsrc((uint8_t*)const_cast<void*>(base) + off, (short)0,
                                                 (int)__builtin_amdgcn_readfirstlane(left * ROW), 0x00020000);
    }
    __device__ __forceinline__ uint32_t voffset(uint32_t r, uint32_t chunk) const { return (r & 7u) * ROW + (chunk << 4); }
    __device__ __forceinline__ bool holes() const { return none; }
    __device__ __forceinline__ uint32_t groups(uint32_t t) const {
        uint32_t on = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++)
            on |= (uint32_t)__builtin_amdgcn_readfirstlane(page_of(t * seqattn::kKeys + 16u * i)) != ~0u ? 1u << i : 0u;
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
    return max((block_keys(a, rq, G, b) + seqattn::kKeys - 1u) / seqattn::kKeys, 1u);
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
template <uint32_t T, uint32_t D>
__device__ __forceinline__ void paged_tiles(const SeqAttnArgs& a, uint8_t* lds, seqattn::JoinRecord* __restrict__ records,
                                            float* __restrict__ scratch) {
    constexpr uint32_t NW = 8, ROW = D * 2u;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t G = a.n_heads / a.n_kv_heads;
    uint32_t* const pages = (uint32_t*)(lds + seqattn::lds_bytes<D>());

    const auto cost = [&](const PagedRequest& r) { return request_units(a, r, G); };
    seqattn::RequestWindow win;
    const uint64_t w = seqattn::batch_cost(a, win, lane, cost) * a.n_kv_heads;
    const uint32_t n = (uint32_t)min((uint64_t)gridDim.x, w);  // every workgroup has a unit
    seqattn::JoinRecord rec{};
    if (blockIdx.x >= n) {
        if (tid == 0) records[blockIdx.x].last = 0;
        return;
    }
    uint64_t at = seqattn::part_begin(blockIdx.x, w, n);
    const uint64_t end = seqattn::part_begin(blockIdx.x + 1u, w, n);
    uint64_t base;  // units (all heads) before request s
    uint32_t s = seqattn::find_request(a, win, lane, cost, a.n_kv_heads, at, base);

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
        const uint32_t keys = block_keys(a, rq, G, b), key0 = t0 * seqattn::kKeys;
        const uint32_t n_keys = min(keys, t1 * seqattn::kKeys) - min(keys, key0);

        const uint32_t rows = rq.rows * G, row0 = b * kBlockRows;
        const auto out_at = [&]() {
            const uint32_t r = min(row0 + 32u * wave + (lane & 31u), rows - 1u);
            return (uint64_t)(rq.first + r / G) * a.out_stride + (kvh * G + r % G) * D;
        };
        const uint32_t r = min(row0 + 32u * wave + (lane & 31u), rows - 1u), i = r / G;
        seqattn::RowOfLane row;
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
        PagedKeys<ROW> src{a.table + (size_t)s * a.max_pages, pages, key0, n_keys, kvh, a.n_kv_heads, a.n_pages,
                           a.page_log2, wave};
        float* const part = t0 == 0 && t1 == tiles
                                ? nullptr
                                : scratch + (2u * blockIdx.x + (t0 == 0 ? 1u : 0u)) * tile_part_floats<D>();
        seqattn::tile_rows<T, D, NW>(a, lds, src, n_keys, row, part, out_at);
        if (t0 == 0 && t1 != tiles)  // (the workgroup's last part: the record is its one)
            rec = seqattn::JoinRecord{seqattn::part_of(at + (tiles - t1) - 1u, w, n), rq.first, row0,
                                      min(rows - row0, kBlockRows), kvh, {}};
    }
    if (tid == 0) records[blockIdx.x] = rec;
}

template <uint32_t T, uint32_t D>
__global__ void __launch_bounds__(512, 1)
paged_attn_tiles(SeqAttnArgs a, seqattn::JoinRecord* __restrict__ records, float* __restrict__ parts) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[seqattn::lds_bytes<D>() + 4u * (kPageCap + 4u)];
    paged_tiles<T, D>(a, lds, records, parts);
}

}  // namespace

hipError_t launch_prompt_attention(const SeqAttnArgs& a, uint32_t type, uint32_t dim, int num_cus, hipStream_t st) {
    auto go = [&](auto t, auto d) {
        constexpr uint32_t T = decltype(t)::value, D = decltype(d)::value;
        // 128 rows a workgroup where all of them are on the card at once (one a CU, two with
        // head_dim 64: their LDS): a tile takes a wave alone on its SIMD nearly as long as two, so
        // fewer rows on more CUs end earlier. With 256 and 128 rows, us: 512 tokens of 32/8 heads,
        // 128: 19.6, 16.9; 1000: 30.7, 27.1; 24/8 heads, 64, 1024: 23.3, 19.5; 2048: 41.9, 35.3.
        // Past that there is a second round: 10 x 200 tokens of 24/8 heads, 128: 17.7, 25.3; 4096
        // of 32/8: 139, 178.
        const uint64_t rows = (uint64_t)a.n_tokens * (a.n_heads / a.n_kv_heads);
        const bool fits = (rows + 127u) / 128u * a.n_kv_heads <= (uint64_t)num_cus * (D == 64u ? 2u : 1u);
        return fits ? launch_tiles<T, D, 4>(a, st) : launch_tiles<T, D, 8>(a, st);
    };
    using BF16 = std::integral_constant<uint32_t, kGgmlBF16>;
    using F16 = std::integral_constant<uint32_t, kGgmlF16>;
    using D64 = std::integral_constant<uint32_t, 64>;
    using D128 = std::integral_constant<uint32_t, 128>;
    if (type == kGgmlBF16) return dim == 128u ? go(BF16{}, D128{}) : go(BF16{}, D64{});
    return dim == 128u ? go(F16{}, D128{}) : go(F16{}, D64{});
}

// Row blocks of 16 of the kernel for few rows that holds max_new tokens of a group; 0: more rows.
// For the call's max_new, not a request's own new tokens. 64 ragged contexts, single tokens, 30/6
// heads: 116 us with few rows, 151 in 256-row blocks; four long contexts with 32 and 64 rows a
// head are faster in those (the figures beside paged_attn_few).
static uint32_t few_blocks(uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new) {
    const uint64_t rows = (uint64_t)max_new * (n_heads / n_kv_heads);
    return rows <= 16u ? 1u : rows <= 32u ? 2u : rows <= 64u ? 4u : 0u;
}
// Workers: waves a CU of paged_attn_few, as many as their LDS lets reside at head_dim 128 (at 64
// too, where it would let twice as many), or one workgroup a CU of paged_attn_tiles. Scratch: a
// record of each, then two parts of each.
static uint32_t paged_workers(uint32_t nr, int num_cus) {
    return (uint32_t)num_cus * (nr == 0u ? 1u : nr == 1u ? 4u : nr == 2u ? 3u : 2u);
}

size_t paged_attention_scratch_bytes(uint32_t dim, uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new, int num_cus) {
    const uint32_t nr = few_blocks(n_heads, n_kv_heads, max_new);
    const size_t part = (nr ? 16u * nr : kBlockRows) * (dim + 2u) * sizeof(float);
    return paged_workers(nr, num_cus) * (sizeof(seqattn::JoinRecord) + 2u * part);
}

template <uint32_t R>
using Rows = std::integral_constant<uint32_t, R>;

template <uint32_t T, uint32_t D>
static hipError_t launch_paged(const SeqAttnArgs& a, uint32_t nr, int num_cus, void* scratch, hipStream_t st) {
    using namespace seqattn;
    const uint32_t n = paged_workers(nr, num_cus);
    auto* const records = (seqattn::JoinRecord*)scratch;
    auto* const parts = (float*)(records + n);
    auto go = [&](auto work, uint32_t threads, auto join, auto part) {
        constexpr uint32_t PR = decltype(part)::value;
        hipLaunchKernelGGL(work, dim3(n), dim3(threads), 0, st, a, records, parts);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(join, dim3(PR / 16u, n), dim3(join_threads<D, PR>()), 0, st, a, records, parts);
        return hipGetLastError();
    };
    if (nr == 0u) return go(paged_attn_tiles<T, D>, 512, paged_attn_join<T, D, kBlockRows>, Rows<kBlockRows>{});
    if (nr == 1u) return go(paged_attn_few<T, D, 1>, 64, paged_attn_join<T, D, 16>, Rows<16>{});
    if (nr == 2u) return go(paged_attn_few<T, D, 2>, 64, paged_attn_join<T, D, 32>, Rows<32>{});
    return go(paged_attn_few<T, D, 4>, 64, paged_attn_join<T, D, 64>, Rows<64>{});
}

hipError_t launch_paged_attention(const SeqAttnArgs& a, uint32_t type, uint32_t dim, int num_cus, void* scratch,
                                  hipStream_t st) {
    const uint32_t nr = few_blocks(a.n_heads, a.n_kv_heads, a.max_new);
    if (type == kGgmlBF16)
        return dim == 128u ? launch_paged<kGgmlBF16, 128>(a, nr, num_cus, scratch, st)
                           : launch_paged<kGgmlBF16, 64>(a, nr, num_cus, scratch, st);
    return dim == 128u ? launch_paged<kGgmlF16, 128>(a, nr, num_cus, scratch, st)
                       : launch_paged<kGgmlF16, 64>(a, nr, num_cus, scratch, st);
}

}  // namespace llmr
