// paged.hip - what fills the paged key/value cache of a batch of requests: the
// plan of a step's pages and slots (llmr_paged_plan) and the QKV projection's
// rows into query rows and cache slots (llmr_qkv_tokens).
#include "llmr_device.h"
#include "llmr_internal.h"

// products and sums round where the formulas write them, as in the other glue
#pragma clang fp contract(off)

namespace llmr {
namespace {

__device__ __forceinline__ uint32_t len_of(int32_t n) { return n > 0 ? (uint32_t)n : 0u; }

// Pages of n tokens, at most the table's columns.
__device__ __forceinline__ uint32_t pages_of(uint32_t n, uint32_t log2, uint32_t max_pages) {
    return min((uint32_t)(((uint64_t)n + (1u << log2) - 1u) >> log2), max_pages);
}

constexpr uint32_t kPlanThreads = 256;

// Every workgroup scans all the requests' lengths (the sums of new tokens and of
// pages to take before each request, into LDS), then writes its share of the
// requests' and tokens' entries: one launch, no workgroup waits for another.
// A token whose page is new takes it from the free list by the page's rank
// rather than from the table, which another workgroup writes.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedPlanArgs a) {
    extern __shared__ uint32_t lds[];
    uint32_t* const tok = lds;                  // [n_seqs + 1] new tokens before request s
    uint32_t* const pag = lds + a.n_seqs + 1u;  // [n_seqs + 1] pages taken before request s
    __shared__ uint32_t part[2][kPlanThreads / 64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    uint32_t tok0 = 0, pag0 = 0;
    for (uint32_t s0 = 0; s0 < a.n_seqs; s0 += kPlanThreads) {
        const uint32_t s = s0 + tid;
        uint32_t nt = 0, np = 0;
        if (s < a.n_seqs) {
            const uint32_t past = len_of(a.past_len[s]);
            nt = len_of(a.new_len[s]);
            np = pages_of(past + nt, a.page_log2, a.max_pages) - pages_of(past, a.page_log2, a.max_pages);
        }
        uint32_t it = nt, ip = np;
#pragma unroll
        for (uint32_t o = 1; o < 64u; o <<= 1) {
            const uint32_t t = __shfl_up(it, o, 64), p = __shfl_up(ip, o, 64);
            if (lane >= o) {
                it += t;
                ip += p;
            }
        }
        if (lane == 63u) {
            part[0][wave] = it;
            part[1][wave] = ip;
        }
        __syncthreads();
        uint32_t bt = tok0, bp = pag0;
#pragma unroll
        for (uint32_t w = 0; w < kPlanThreads / 64u; w++) {
            if (w < wave) {
                bt += part[0][w];
                bp += part[1][w];
            }
            tok0 += part[0][w];
            pag0 += part[1][w];
        }
        if (s < a.n_seqs) {
            tok[s] = bt + it - nt;
            pag[s] = bp + ip - np;
        }
        __syncthreads();
    }
    if (tid == 0) {
        tok[a.n_seqs] = tok0;
        pag[a.n_seqs] = pag0;
    }
    __syncthreads();
    const uint32_t n_free = min(len_of(*a.free_count), a.n_free);
    const uint32_t threads = gridDim.x * kPlanThreads, id = blockIdx.x * kPlanThreads + tid;

    // the last s with sum[s] <= x (sum[0] = 0; empty requests share a sum: the last one)
    auto find = [&](const uint32_t* sum, uint32_t x) {
        uint32_t lo = 0, hi = a.n_seqs;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2u;
            if (sum[mid + 1u] > x) hi = mid;
            else lo = mid + 1u;
        }
        return lo;
    };
    auto fresh = [&](uint32_t rank) { return rank < n_free ? a.free_pages[n_free - 1u - rank] : -1; };

    for (uint32_t s = id; s <= a.n_seqs; s += threads) {
        a.seq_offsets[s] = (int32_t)tok[s];
        if (s < a.n_seqs) a.kv_len[s] = (int32_t)(len_of(a.past_len[s]) + len_of(a.new_len[s]));
    }
    if (id < 2u) a.pages[id] = (int32_t)(id == 0 ? n_free - min(n_free, pag0) : pag0 - min(n_free, pag0));
    for (uint32_t r = id; r < pag0; r += threads) {
        const uint32_t s = find(pag, r);
        const uint32_t held = pages_of(len_of(a.past_len[s]), a.page_log2, a.max_pages);
        a.block_table[(size_t)s * a.max_pages + held + (r - pag[s])] = fresh(r);
    }
    for (uint32_t t = id; t < a.n_tokens; t += threads) {
        int32_t slot = -1;
        uint32_t pos = 0;
        if (t < tok0) {
            const uint32_t s = find(tok, t);
            const uint32_t past = len_of(a.past_len[s]);
            pos = past + (t - tok[s]);
            const uint32_t col = pos >> a.page_log2;
            if (col < a.max_pages) {
                const uint32_t held = pages_of(past, a.page_log2, a.max_pages);
                const int32_t page =
                    col < held ? a.block_table[(size_t)s * a.max_pages + col] : fresh(pag[s] + (col - held));
                const int64_t at = ((int64_t)page << a.page_log2) + (pos & ((1u << a.page_log2) - 1u));
                if (page >= 0 && at <= 0x7fffffff) slot = (int32_t)at;
            }
        }
        a.slots[t] = slot;
        a.positions[t] = (int32_t)pos;
    }
}

template <uint32_t OT>
__device__ __forceinline__ void put2(void* base, size_t idx, float x, float y) {
    *(uint32_t*)((uint16_t*)base + idx) = OT == kGgmlF16 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
}

// One wave per head of a row; lane l holds the pair the rotation takes together
// (D = 64: two heads a wave).
template <uint32_t OT, uint32_t D, bool HALVES>
__global__ void __launch_bounds__(256) qkv_tokens_kernel(QkvTokensArgs a) {
    constexpr uint32_t P = D / 2u;  // pairs, lanes of a head
    const uint32_t l = threadIdx.x % P, unit = threadIdx.x / P;
    const uint32_t r = blockIdx.x, heads = a.n_heads + 2u * a.n_kv_heads;
    const uint32_t pos = a.positions ? (uint32_t)min(max(a.positions[r], 0), (int32_t)(a.n_positions - 1u)) : r;
    const uint32_t e0 = HALVES ? l : 2u * l, e1 = HALVES ? l + P : 2u * l + 1u;
    float c = 1.0f, sn = 0.0f;
    if (a.rope_cos) {
        c = a.rope_cos[(size_t)pos * P + l];
        sn = a.rope_sin[(size_t)pos * P + l];
    }
    const int32_t slot = a.slots ? a.slots[r] : 0;
    for (uint32_t h = blockIdx.y * (256u / P) + unit; h < heads; h += gridDim.y * (256u / P)) {
        const float* src = a.qkv + (size_t)r * a.qkv_stride + (size_t)h * D;
        float x0 = src[e0], x1 = src[e1];
        const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv_heads;
        const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (w) {
            float ss = x0 * x0 + x1 * x1;
#pragma unroll
            for (uint32_t o = P / 2u; o > 0; o >>= 1) ss += __shfl_xor(ss, (int)o, 64);
            const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
            x0 = x0 * inv * w[e0];
            x1 = x1 * inv * w[e1];
        }
        if (a.rope_cos && !is_v) {
            const float y0 = x0 * c - x1 * sn, y1 = x0 * sn + x1 * c;
            x0 = y0;
            x1 = y1;
        }
        void* dst;
        size_t at;
        if (is_q) {
            dst = a.q;
            at = (size_t)r * a.q_stride + (size_t)h * D;
        } else {
            const uint32_t kh = h - a.n_heads - (is_v ? a.n_kv_heads : 0u);
            dst = is_v ? a.v : a.k;
            if (a.slots) {
                const uint32_t page = (uint32_t)slot >> a.page_log2;
                if (slot < 0 || page >= a.n_pages) continue;
                at = ((((size_t)page * a.n_kv_heads + kh) << a.page_log2) +
                      ((uint32_t)slot & ((1u << a.page_log2) - 1u))) * D;
            } else {
                at = (size_t)r * a.kv_stride + (size_t)kh * D;
            }
        }
        if constexpr (HALVES) {
            ((uint16_t*)dst)[at + e0] = (uint16_t)(OT == kGgmlF16 ? pack_f16x2(x0, 0.0f) : pack_bf16x2(x0, 0.0f));
            ((uint16_t*)dst)[at + e1] = (uint16_t)(OT == kGgmlF16 ? pack_f16x2(x1, 0.0f) : pack_bf16x2(x1, 0.0f));
        } else {
            put2<OT>(dst, at + e0, x0, x1);
        }
    }
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t st) {
    // tokens of a workgroup: 4 a thread; a small step is one workgroup
    const uint32_t items = a.n_tokens > a.n_seqs ? a.n_tokens : a.n_seqs;
    const uint32_t wgs = (items + 4u * kPlanThreads - 1u) / (4u * kPlanThreads);
    hipLaunchKernelGGL(paged_plan_kernel, dim3(wgs < 256u ? (wgs ? wgs : 1u) : 256u), dim3(kPlanThreads),
                       2u * (a.n_seqs + 1u) * 4u, st, a);
    return hipGetLastError();
}

hipError_t launch_qkv_tokens(const QkvTokensArgs& a, uint32_t dim, uint32_t otype, bool halves, hipStream_t st) {
    const dim3 grid(a.n_tokens, 1), block(256);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, a); };
    if (otype == kGgmlBF16) {
        if (dim == 128u) halves ? go(qkv_tokens_kernel<kGgmlBF16, 128, true>) : go(qkv_tokens_kernel<kGgmlBF16, 128, false>);
        else halves ? go(qkv_tokens_kernel<kGgmlBF16, 64, true>) : go(qkv_tokens_kernel<kGgmlBF16, 64, false>);
    } else {
        if (dim == 128u) halves ? go(qkv_tokens_kernel<kGgmlF16, 128, true>) : go(qkv_tokens_kernel<kGgmlF16, 128, false>);
        else halves ? go(qkv_tokens_kernel<kGgmlF16, 64, true>) : go(qkv_tokens_kernel<kGgmlF16, 64, false>);
    }
    return hipGetLastError();
}

}  // namespace llmr
