// seq_attn.hip - causal attention of a batch of requests (llmr_prompt_attention,
// llmr_paged_attention): grouped heads, packed rows, keys in the packed rows or in
// the pages of a cache.
//
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,  p_j = exp2(c (<q[t, h], k[j, h / G]> - m))
//
// c = scale * log2(e), m the largest of the row's products so far (subtracted before
// the scaling: a product of the type's lowest value times log2(e) is past f32).
#include "seq_attn_few.h"
#include "seq_attn_paged.h"
#include "seq_attn_tile.h"

namespace llmr {
namespace {

// Keys in packed rows: a tile's descriptor starts at its first key and ends with the
// workgroup's last.
struct PackedKeys {
    static constexpr bool kStages = false, kBlocks4 = false;
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

template <uint32_t T, uint32_t D>
__global__ void __launch_bounds__(512, 1)
paged_attn_tiles(SeqAttnArgs a, seqattn::JoinRecord* __restrict__ records, float* __restrict__ parts) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[seqattn::paged_lds_bytes<D>()];
    seqattn::paged_tiles<T, D>(a, lds, records, parts, [](const seqattn::PagedKeys<D * 2u>& keys) { return keys; });
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
    const size_t part = (nr ? 16u * nr : seqattn::kBlockRows) * (dim + 2u) * sizeof(float);
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
    if (nr == 0u) return go(paged_attn_tiles<T, D>, 512, paged_attn_join<T, D, seqattn::kBlockRows>, Rows<seqattn::kBlockRows>{});
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
