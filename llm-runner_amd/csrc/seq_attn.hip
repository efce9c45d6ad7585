// seq_attn.hip - causal attention of a batch of requests (llmr_prompt_attention,
// llmr_paged_attention): grouped heads, packed rows, keys in the packed rows or in
// the pages of a cache.
//
//   out[t, h] = sum_j p_j v[j, h / G] / sum_j p_j,  p_j = exp2(c (<q[t, h], k[j, h / G]> - m))
//
// c = scale * log2(e), m the largest of the row's products so far (subtracted before
// the scaling: a product of the type's lowest value times log2(e) is past f32).
#include "llmr_device.h"
#include "llmr_internal.h"

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
    return launch<false>(a, type, dim, st);
}
size_t paged_attention_scratch_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, int) { return 0; }
hipError_t launch_paged_attention(const SeqAttnArgs& a, uint32_t type, uint32_t dim, int, void*, hipStream_t st) {
    return launch<true>(a, type, dim, st);
}

}  // namespace llmr
