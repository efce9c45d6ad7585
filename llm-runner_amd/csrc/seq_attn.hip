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

template <uint32_t T>
__device__ __forceinline__ float widen(uint16_t x) {
    if constexpr (T == kGgmlBF16) return __uint_as_float((uint32_t)x << 16);
    else return (float)__builtin_bit_cast(_Float16, x);
}
template <uint32_t T>
__device__ __forceinline__ uint16_t narrow(float x) {
    if constexpr (T == kGgmlBF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
    else return __builtin_bit_cast(uint16_t, (_Float16)x);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// One wave per (row, query head): 64 keys a step, a lane one key's score, then
// D / 64 dims of the row.
template <uint32_t T, uint32_t D, bool PAGED>
__global__ void __launch_bounds__(256) seq_attn_rows(SeqAttnArgs a) {
    __shared__ float qs[4][D];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t t = blockIdx.x * 4u + wave, head = blockIdx.y;
    if (t >= a.n_tokens) return;
    uint32_t lo = 0, hi = a.n_seqs;  // the first request that ends behind row t
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (a.offsets[mid + 1u] > (int32_t)t) hi = mid;
        else lo = mid + 1u;
    }
    if (lo == a.n_seqs) return;
    const int32_t first = a.offsets[lo];
    if (first < 0 || first > (int32_t)t) return;
    const uint32_t i = t - (uint32_t)first;
    if (PAGED && i >= a.max_new) return;
    const uint32_t kvh = head / (a.n_heads / a.n_kv_heads);
    int64_t keys;  // seen by this row
    if constexpr (PAGED) {
        const int64_t n = min(a.offsets[lo + 1u], (int32_t)a.n_tokens) - first;
        keys = (int64_t)a.kv_len[lo] - n + i + 1;
        keys = min(keys, (int64_t)a.max_pages << a.page_log2);
    } else {
        keys = i + 1;
    }
    const uint16_t* qr = (const uint16_t*)a.q + (size_t)t * a.q_stride + (size_t)head * a.q_head_stride;
    for (uint32_t d = lane; d < D; d += 64u) qs[wave][d] = widen<T>(qr[d]);
    __builtin_amdgcn_wave_barrier();
    float m = -INFINITY, l = 0.0f, o[D / 64u] = {};
    bool sees = false;  // any key: a row that sees none is 0
    for (int64_t k0 = 0; k0 < keys; k0 += 64) {
        const int64_t j = k0 + lane;
        size_t row = 0;
        bool seen = j < keys;
        if (seen) {
            if constexpr (PAGED) {
                const int32_t page = a.table[(size_t)lo * a.max_pages + (uint32_t)(j >> a.page_log2)];
                seen = page >= 0 && (uint32_t)page < a.n_pages;
                row = ((((size_t)(uint32_t)page * a.n_kv_heads + kvh) << a.page_log2) +
                       ((uint32_t)j & ((1u << a.page_log2) - 1u))) * D;
            } else {
                row = (size_t)(first + (uint32_t)j) * a.kv_stride + (size_t)kvh * a.kv_head_stride;
            }
        }
        float s = -INFINITY;
        if (seen) {
            float acc = 0.0f;
            const uint16_t* kr = (const uint16_t*)a.k + row;
            for (uint32_t d = 0; d < D; d++) acc = fmaf(qs[wave][d], widen<T>(kr[d]), acc);
            s = acc;
        }
        const uint64_t any = __builtin_amdgcn_ballot_w64(seen);
        if (any == 0) continue;
        sees = true;
        // NaN scores go into the row by way of exp2
        const float mx = fmaxf(m, wave_max(s));
        const float mu = mx == -INFINITY ? 0.0f : mx;
        const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mu) * a.scale_log2);
        const float p = seen ? widen<T>(narrow<T>(__builtin_amdgcn_exp2f((s - mu) * a.scale_log2))) : 0.0f;
        m = mx;
        l = l * alpha + wave_add(p);
#pragma unroll
        for (uint32_t x = 0; x < D / 64u; x++) o[x] *= alpha;
        for (uint32_t b = 0; b < 64u; b++) {
            if (!((any >> b) & 1u)) continue;
            const float pb = __shfl(p, (int)b, 64);
            const size_t rb = ((size_t)__shfl((int)(row >> 32), (int)b, 64) << 32) |
                              (uint32_t)__shfl((int)(uint32_t)row, (int)b, 64);
            const uint16_t* vr = (const uint16_t*)a.v + rb;
#pragma unroll
            for (uint32_t x = 0; x < D / 64u; x++) o[x] = fmaf(pb, widen<T>(vr[lane + 64u * x]), o[x]);
        }
    }
    uint16_t* dst = (uint16_t*)a.out + (size_t)t * a.out_stride + (size_t)head * D;
#pragma unroll
    for (uint32_t x = 0; x < D / 64u; x++) dst[lane + 64u * x] = narrow<T>(sees ? o[x] / l : 0.0f);
}

// Keys in packed rows: a tile's descriptor starts at its first key and ends with the
// workgroup's last.
struct PackedKeys {
    uint64_t first;    // element offset of key 0 of the key/value head
    uint32_t stride2;  // bytes between keys
    uint32_t n_keys;
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
    seqattn::RowsOfLane row;
    row.live = row0 + 32u * wave + (lane & 31u) < rows;
    int32_t start = start0;
    if ((int32_t)tok >= end0) {
        const uint32_t s = request_of(a.offsets, s0 + 1u, a.n_seqs, tok);
        start = s < a.n_seqs ? a.offsets[s] : 0x7fffffff;
    }
    row.live = row.live && start <= (int32_t)tok;
    const uint32_t lo = (uint32_t)max(start, 0);
    row.jlo = row.live ? (lo > kv0 ? lo - kv0 : 0u) : 0x80000000u;
    row.span = row.live ? tok - kv0 - row.jlo : 0u;
    row.q = (const uint8_t*)a.q + 2u * ((uint64_t)tok * a.q_stride + (uint64_t)head * a.q_head_stride);
    row.out = (uint64_t)tok * a.out_stride + head * D;
    const uint32_t lo_max = (uint32_t)seqattn::wave_imax(row.live ? (int)row.jlo : 0);
    const uint32_t hi_min = (uint32_t)seqattn::wave_imin(row.live ? (int)(tok - kv0) : 0x7fffffff);
    const PackedKeys src{(uint64_t)kv0 * a.kv_stride + (uint64_t)kvh * a.kv_head_stride, a.kv_stride * 2u, t1 + 1u - kv0};
    seqattn::tile_rows<T, D, NW>(a, lds, src, t1 + 1u - kv0, row, lo_max, hi_min);
}

template <uint32_t T, uint32_t D, uint32_t NW>
hipError_t launch_tiles(const SeqAttnArgs& a, hipStream_t st) {
    const uint32_t blocks = (a.n_tokens * (a.n_heads / a.n_kv_heads) + 32u * NW - 1u) / (32u * NW);
    hipLaunchKernelGGL((prompt_attn_tiles<T, D, NW>), dim3(blocks * a.n_kv_heads), dim3(64 * NW), 0, st, a);
    return hipGetLastError();
}

template <bool PAGED>
hipError_t launch(const SeqAttnArgs& a, uint32_t type, uint32_t dim, hipStream_t st) {
    const dim3 grid((a.n_tokens + 3u) / 4u, a.n_heads), block(256);
    if (type == kGgmlBF16) {
        if (dim == 128u) hipLaunchKernelGGL((seq_attn_rows<kGgmlBF16, 128, PAGED>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((seq_attn_rows<kGgmlBF16, 64, PAGED>), grid, block, 0, st, a);
    } else {
        if (dim == 128u) hipLaunchKernelGGL((seq_attn_rows<kGgmlF16, 128, PAGED>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((seq_attn_rows<kGgmlF16, 64, PAGED>), grid, block, 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_prompt_attention(const SeqAttnArgs& a, uint32_t type, uint32_t dim, hipStream_t st) {
    if (type == kGgmlBF16)
        return dim == 128u ? launch_tiles<kGgmlBF16, 128, 8>(a, st) : launch_tiles<kGgmlBF16, 64, 8>(a, st);
    return dim == 128u ? launch_tiles<kGgmlF16, 128, 8>(a, st) : launch_tiles<kGgmlF16, 64, 8>(a, st);
}
// Row blocks of 16 of the kernel for few rows that holds max_new tokens of a group; 0: more rows.
static uint32_t few_blocks(uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new) {
    const uint64_t rows = (uint64_t)max_new * (n_heads / n_kv_heads);
    return rows <= 16u ? 1u : rows <= 32u ? 2u : rows <= 64u ? 4u : 0u;
}
constexpr uint32_t kFewPerCu = 4;  // waves a CU: their rings fill its LDS

size_t paged_attention_scratch_bytes(uint32_t dim, uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new, int num_cus) {
    const uint32_t nr = few_blocks(n_heads, n_kv_heads, max_new);
    return (size_t)2u * kFewPerCu * num_cus * 16u * nr * (dim + 2u) * sizeof(float);
}

template <uint32_t T, uint32_t D, uint32_t NR>
static hipError_t launch_few(const SeqAttnArgs& a, int num_cus, float* scratch, hipStream_t st) {
    const uint32_t n = kFewPerCu * (uint32_t)num_cus;
    hipLaunchKernelGGL((seqattn::paged_attn_few<T, D, NR>), dim3(n), dim3(64), 0, st, a, scratch);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((seqattn::paged_attn_join<T, D, NR>), dim3(a.n_seqs, a.n_kv_heads), dim3(256), 0, st, a, scratch, n);
    return hipGetLastError();
}

hipError_t launch_paged_attention(const SeqAttnArgs& a, uint32_t type, uint32_t dim, int num_cus, void* scratch,
                                  hipStream_t st) {
    const uint32_t nr = few_blocks(a.n_heads, a.n_kv_heads, a.max_new);
    if (nr == 0) return launch<true>(a, type, dim, st);
    float* const p = (float*)scratch;
    auto go = [&](auto t, auto d) {
        constexpr uint32_t T = decltype(t)::value, D = decltype(d)::value;
        return nr == 1u ? launch_few<T, D, 1>(a, num_cus, p, st)
                        : nr == 2u ? launch_few<T, D, 2>(a, num_cus, p, st) : launch_few<T, D, 4>(a, num_cus, p, st);
    };
    using BF16 = std::integral_constant<uint32_t, kGgmlBF16>;
    using F16 = std::integral_constant<uint32_t, kGgmlF16>;
    using D64 = std::integral_constant<uint32_t, 64>;
    using D128 = std::integral_constant<uint32_t, 128>;
    if (type == kGgmlBF16) return dim == 128u ? go(BF16{}, D128{}) : go(BF16{}, D64{});
    return dim == 128u ? go(F16{}, D128{}) : go(F16{}, D64{});
}

}  // namespace llmr
