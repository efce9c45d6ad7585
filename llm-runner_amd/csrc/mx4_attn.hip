// mx4_attn.hip - attention of a batch of requests over a paged cache in 4 bits
// (llmr_paged_attention_mx4). Few rows a head: mx4_attn_few.h. More: mx4_attn_tiles, the
// tiles of 16-bit caches (seq_attn_paged.h) with keys and values in blocks of 4 bits, which
// pass through registers, where they become 16-bit rows, on their way to LDS. Measured, us:
// 512 tokens behind 30001 keys of 32/8 heads of 128 255 to 261 in a graph with the join, as over a
// 16-bit cache (floor 203; in the tiles, 254 to 266 traced, 950 to 1000 TFLOP/s: matrix cores busy 45%
// of their cycles at 2.1 GHz, the vector ALU 50% beside them); 24 requests
// of 1 to 511 tokens at 16/4 heads of 64 39 to 41 (blocks of few rows one after another).
#include "mx4_attn_few.h"
#include "seq_attn_paged.h"

namespace llmr {
namespace {

// Keys in the pages of a cache of blocks: a lane fetches an eighth of a key's numbers and their power.
template <uint32_t D>
struct Mx4Keys : seqattn::PagedKeys<D / 2u> {
    static constexpr bool kBlocks4 = true;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
    __device__ __forceinline__ seqattn::Blocks4<D> fetch(const void* base, const uint8_t* scales, uint32_t t, uint32_t page,
                                                         uint32_t lane) const {
        const rsrc_t r = this->template rows_of<D / 2u>(base, t, page), sr = this->template rows_of<D / 32u>(scales, t, page);
        seqattn::Blocks4<D> x;
        if constexpr (D == 128u) {
            const u32x2 n = __builtin_amdgcn_raw_buffer_load_b64(r, 8u * lane, 0, 0);
            x.n[0] = n.x;
            x.n[1] = n.y;
            x.power = __builtin_amdgcn_raw_buffer_load_b8(sr, lane >> 1, 0, 0);
        } else {
            x.n[0] = __builtin_amdgcn_raw_buffer_load_b32(r, 4u * lane, 0, 0);
            x.power = __builtin_amdgcn_raw_buffer_load_b8(sr, lane >> 2, 0, 0);
        }
        return x;
    }
    // the cache's row of key j < n_keys (-1: on no page)
    __device__ __forceinline__ int64_t row_of(uint32_t j) const {
        const uint32_t at = this->key0 + j, p = (uint32_t)this->table[at >> this->log2];
        return p < this->n_pages ? (int64_t)((((uint64_t)p * this->n_kv_heads + this->kvh) << this->log2) +
                                             (at & ((1u << this->log2) - 1u)))
                                 : -1;
    }
    __device__ __forceinline__ bool far_value(uint32_t j) const {
        const int64_t row = row_of(j);
        bool far = false;
        if (row >= 0) {
#pragma unroll
            for (uint32_t i = 0; i < D / 32u; i++) far = far || v_scales[row * (D / 32u) + i] > mx4attn::kTopPower;
        }
        return far;
    }
    template <uint32_t T>
    __device__ __forceinline__ u32x2 value4(const void* v, uint32_t j, uint32_t dim) const {
        const int64_t row = row_of(j);
        const u32x4 w = values8<T>(*(const uint16_t*)((const uint8_t*)v + row * (D / 2u) + dim / 2u),
                                   power4(v_scales[row * (D / 32u) + dim / 32u]));
        return u32x2{w.x, w.y};
    }
};

template <uint32_t T, uint32_t D>
__global__ void __launch_bounds__(512, 1)
mx4_attn_tiles(mx4attn::Mx4Args m4, seqattn::JoinRecord* __restrict__ records, float* __restrict__ parts) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[seqattn::paged_lds_bytes<D>()];
    seqattn::paged_tiles<T, D>(m4.a, lds, records, parts, [&](const seqattn::PagedKeys<D * 2u>& k) {
        return Mx4Keys<D>{{k.table, k.pages, k.key0, k.n_keys, k.kvh, k.n_kv_heads, k.n_pages, k.log2, k.wave},
                          m4.k_scales, m4.v_scales};
    });
}

}  // namespace

// Row blocks of 16 of the kernel for few rows that holds max_new tokens of a group; 0: more rows, for
// which the tiles are faster at any length. In 32-row blocks and in tiles, us: four contexts of 40000 to
// 131000 keys of 32/8 heads of 128 with 8 new tokens (32 rows) 102, 212; 16 x 4 tokens at 28/4 heads of
// 64 (28 rows) 32, 48. With a kernel of 64 rows, and in tiles: the four contexts with 9 to 16 tokens 500,
// 215 (64: 154, 155), 32 contexts of 100 to 8000 keys 134 to 142, 85 to 91 (64: 52 to 58, 48), one of 500
// 24 to 29, 22 to 24 (64: 14.5 to 15.8, 13.9 to 15.0).
static uint32_t mx4_blocks(uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new) {
    const uint64_t rows = (uint64_t)max_new * (n_heads / n_kv_heads);
    return rows <= 16u ? 1u : rows <= 32u ? 2u : 0u;
}
// Workers: workgroups a CU, as many as the registers let reside, or one of mx4_attn_tiles.
static uint32_t mx4_workers(uint32_t nr, int num_cus) {
    return (uint32_t)num_cus * (nr == 0u ? 1u : nr == 1u ? mx4attn::few_waves<1>() : mx4attn::few_waves<2>());
}

size_t paged_attention_mx4_scratch_bytes(uint32_t dim, uint32_t n_heads, uint32_t n_kv_heads, uint32_t max_new,
                                         int num_cus) {
    const uint32_t nr = mx4_blocks(n_heads, n_kv_heads, max_new);
    const size_t part = (nr ? 16u * nr : seqattn::kBlockRows) * (dim + 2u) * sizeof(float);
    return mx4_workers(nr, num_cus) * (sizeof(seqattn::JoinRecord) + 2u * part);
}

template <uint32_t R>
using Rows = std::integral_constant<uint32_t, R>;

template <uint32_t T, uint32_t D>
static hipError_t launch_mx4(const mx4attn::Mx4Args& m4, uint32_t nr, int num_cus, void* scratch, hipStream_t st) {
    using namespace mx4attn;
    const SeqAttnArgs& a = m4.a;
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
    if (nr == 0u) return go(mx4_attn_tiles<T, D>, 512, paged_attn_join<T, D, kBlockRows>, Rows<kBlockRows>{});
    if (nr == 1u) return go(mx4_attn_few<T, D, 1>, 64 * kWaves, paged_attn_join<T, D, 16>, Rows<16>{});
    return go(mx4_attn_few<T, D, 2>, 64 * kWaves, paged_attn_join<T, D, 32>, Rows<32>{});
}

hipError_t launch_paged_attention_mx4(const SeqAttnArgs& a, const uint8_t* k_scales, const uint8_t* v_scales,
                                      uint32_t type, uint32_t dim, int num_cus, void* scratch, hipStream_t st) {
    const uint32_t nr = mx4_blocks(a.n_heads, a.n_kv_heads, a.max_new);
    mx4attn::Mx4Args m4{a, k_scales, v_scales};
    if (a.n_pages == 0) {  // mx4_attn_few reads a cache's first rows for a page that there is not, and drops them
        m4.a.k = m4.a.v = scratch;
        m4.k_scales = m4.v_scales = (const uint8_t*)scratch;
    }
    if (type == kGgmlBF16)
        return dim == 128u ? launch_mx4<kGgmlBF16, 128>(m4, nr, num_cus, scratch, st)
                           : launch_mx4<kGgmlBF16, 64>(m4, nr, num_cus, scratch, st);
    return dim == 128u ? launch_mx4<kGgmlF16, 128>(m4, nr, num_cus, scratch, st)
                       : launch_mx4<kGgmlF16, 64>(m4, nr, num_cus, scratch, st);
}

}  // namespace llmr
