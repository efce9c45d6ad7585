// mx4_attn.hip - attention of a batch of requests over a paged cache in 4 bits
// (llmr_paged_attention_mx4).
#include "mx4_attn_few.h"

namespace llmr {
namespace {

using seqattn::PagedRequest;

// Simplest form: a wave a row and head, a key at a time, lanes over the dims.
template <uint32_t T, uint32_t D>
__global__ void __launch_bounds__(64) mx4_attn_rows(SeqAttnArgs a, const uint8_t* k_scales, const uint8_t* v_scales) {
    constexpr uint32_t W = D / 2u;  // lanes with two dims each
    const uint32_t lane = threadIdx.x, l = lane < W ? lane : 0u;
    const uint32_t t = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, G = a.n_heads / a.n_kv_heads, kvh = h / G;
    for (uint32_t s = 0; s < a.n_seqs; s++) {
        const PagedRequest rq = seqattn::paged_request(a, s);
        if (t < rq.first || t - rq.first >= rq.rows) continue;
        const int32_t last = rq.pos0 + (int32_t)(t - rq.first);
        const uint32_t n = (uint32_t)min(max(last + 1, 0), (int32_t)rq.keys);
        const uint32_t qw = *(const uint32_t*)((const uint16_t*)a.q + (size_t)t * a.q_stride + (size_t)h * a.q_head_stride + 2u * l);
        const float q0 = lane < W ? seqattn::lo_f32<T>(qw) : 0.0f, q1 = lane < W ? seqattn::hi_f32<T>(qw) : 0.0f;
        float m = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
        bool seen = false;
        for (uint32_t j = 0; j < n; j++) {
            const int32_t p = a.table[(size_t)s * a.max_pages + (j >> a.page_log2)];
            if (p < 0 || (uint32_t)p >= a.n_pages) continue;
            const size_t row = (((size_t)(uint32_t)p * a.n_kv_heads + kvh) << a.page_log2) + (j & ((1u << a.page_log2) - 1u));
            const uint32_t kb = ((const uint8_t*)a.k)[row * W + l], vb = ((const uint8_t*)a.v)[row * W + l];
            const float ks = __uint_as_float((uint32_t)k_scales[row * (D / 32u) + l / 16u] << 23);
            const float vs = __uint_as_float((uint32_t)v_scales[row * (D / 32u) + l / 16u] << 23);
            const auto kf = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(kb, ks, 0), vf = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(vb, vs, 0);
            float d = q0 * kf[0] + q1 * kf[1];
            if (lane >= W) d = 0.0f;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o, 64);
            seen = true;
            const float mx = fmaxf(m, d);
            const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * a.scale_log2);
            const float e = __builtin_amdgcn_exp2f((d - mx) * a.scale_log2);
            sum = sum * al + e;
            o0 = o0 * al + e * vf[0];
            o1 = o1 * al + e * vf[1];
            m = mx;
        }
        if (lane < W)
            *(uint32_t*)((uint16_t*)a.out + (size_t)t * a.out_stride + (size_t)h * D + 2u * l) =
                seen ? seqattn::pack2<T>(o0 / sum, o1 / sum) : 0u;
        return;
    }
}

}  // namespace

// Row blocks of 16 of the kernel for few rows that holds max_new tokens of a group; 0: more rows.
static uint32_t mx4_blocks(uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new) {
    const uint64_t rows = (uint64_t)max_new * (n_heads / n_kv_heads);
    return rows <= 16u ? 1u : rows <= 32u ? 2u : rows <= 64u ? 4u : 0u;
}
static uint32_t mx4_workers(uint32_t nr, int num_cus) {
    return (uint32_t)num_cus * (nr == 1u ? mx4attn::few_waves<1>() : nr == 2u ? mx4attn::few_waves<2>() : mx4attn::few_waves<4>());
}

size_t paged_attention_mx4_scratch_bytes(uint32_t dim, uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new,
                                         int num_cus) {
    const uint32_t nr = mx4_blocks(n_heads, n_kv_heads, max_new);
    if (nr == 0) return 0;
    const size_t part = 16u * nr * (dim + 2u) * sizeof(float);
    return mx4_workers(nr, num_cus) * (sizeof(seqattn::JoinRecord) + 2u * part);
}

template <uint32_t R>
using Rows = std::integral_constant<uint32_t, R>;

template <uint32_t T, uint32_t D>
static hipError_t launch_mx4(const mx4attn::Mx4Args& m4, uint32_t nr, int num_cus, void* scratch, hipStream_t st) {
    using namespace mx4attn;
    const SeqAttnArgs& a = m4.a;
    if (nr == 0) {
        hipLaunchKernelGGL((mx4_attn_rows<T, D>), dim3(a.n_tokens * a.n_heads), dim3(64), 0, st, a, m4.k_scales, m4.v_scales);
        return hipGetLastError();
    }
    const uint32_t n = mx4_workers(nr, num_cus);
    auto* const records = (JoinRecord*)scratch;
    auto* const parts = (float*)(records + n);
    auto go = [&](auto work, uint32_t threads, auto join, auto part) {
        constexpr uint32_t PR = decltype(part)::value;
        hipLaunchKernelGGL(work, dim3(n), dim3(threads), 0, st, m4, records, parts);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(join, dim3(PR / 16u, n), dim3(join_threads<D, PR>()), 0, st, a, records, parts);
        return hipGetLastError();
    };
    if (nr == 1u) return go(mx4_attn_few<T, D, 1>, 64 * kWaves, paged_attn_join<T, D, 16>, Rows<16>{});
    if (nr == 2u) return go(mx4_attn_few<T, D, 2>, 64 * kWaves, paged_attn_join<T, D, 32>, Rows<32>{});
    return go(mx4_attn_few<T, D, 4>, 64 * kWaves, paged_attn_join<T, D, 64>, Rows<64>{});
}

hipError_t launch_paged_attention_mx4(const SeqAttnArgs& a, const uint8_t* k_scales, const uint8_t* v_scales,
                                      uint32_t type, uint32_t dim, int num_cus, void* scratch, hipStream_t st) {
    const uint32_t nr = mx4_blocks(a.n_heads, a.n_kv_heads, a.max_new);
    const mx4attn::Mx4Args m4{a, k_scales, v_scales};
    if (type == kGgmlBF16)
        return dim == 128u ? launch_mx4<kGgmlBF16, 128>(m4, nr, num_cus, scratch, st)
                           : launch_mx4<kGgmlBF16, 64>(m4, nr, num_cus, scratch, st);
    return dim == 128u ? launch_mx4<kGgmlF16, 128>(m4, nr, num_cus, scratch, st)
                       : launch_mx4<kGgmlF16, 64>(m4, nr, num_cus, scratch, st);
}

}  // namespace llmr
