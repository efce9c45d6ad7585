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
constexpr uint32_t kMaxGridRows = 1u << 23;

template <uint32_t OT>
__device__ __forceinline__ uint32_t pack16(float x, float y) {
    return OT == kGgmlF16 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
}

// Every workgroup scans all the requests' lengths (the sums of new tokens and of
// pages to take before each request, into LDS), then writes its share of the
// requests' and tokens' entries: one launch, no workgroup waits for another.
// A token whose page is new takes it from the free list by the page's rank
// rather than from the table, which another workgroup writes. Bound by the launch and
// the scan: 32 requests of one token 4.2 us, 256 of 39000 tokens 4.7 (tokens in a loop
// over few workgroups: 7.4).
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

// D / 8 lanes a head, 8 elements a lane: four pairs of the rotation, as two vectors of four
// (pairs (j, j + D / 2): one from each half; pairs (2j, 2j + 1): one behind the other), so
// that every load is 16 bytes a lane and every store 8. A thread has one head of one row:
// nothing waits for anything but its own loads. HBM bound: 8192 rows of 32/8 heads (306 MB)
// 52 us, 5.9 TB/s; 64 rows 3.2 us, the launch (rows in a loop, 8-byte loads: 76 and 8.8).
template <uint32_t OT, uint32_t D, bool HALVES>
__global__ void __launch_bounds__(256) qkv_tokens_kernel(QkvTokensArgs a) {
    constexpr uint32_t L = D / 8u;  // lanes of a head
    const uint32_t l = threadIdx.x % L, h = blockIdx.y * (256u / L) + threadIdx.x / L;
    const uint32_t r = blockIdx.z * kMaxGridRows + blockIdx.x;
    if (r >= a.n_tokens || h >= a.n_heads + 2u * a.n_kv_heads) return;  // (whole heads: the reductions stay within one)
    const uint32_t e0 = HALVES ? 4u * l : 8u * l, e1 = HALVES ? e0 + D / 2u : e0 + 4u;
    const float* src = a.qkv + (size_t)r * a.qkv_stride + (size_t)h * D;
    f32x4 x0 = *(const f32x4*)(src + e0), x1 = *(const f32x4*)(src + e1);
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv_heads;
    const int32_t slot = a.slots && !is_q ? a.slots[r] : 0;
    const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    if (w) {
        const f32x4 w0 = *(const f32x4*)(w + e0), w1 = *(const f32x4*)(w + e1);
        const f32x4 q = x0 * x0 + x1 * x1;
        float ss = (q.x + q.y) + (q.z + q.w);
#pragma unroll
        for (uint32_t o = L / 2u; o > 0; o >>= 1) ss += __shfl_xor(ss, (int)o, 64);
        const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
        x0 = x0 * inv * w0;
        x1 = x1 * inv * w1;
    }
    if (a.rope_cos && !is_v) {
        const uint32_t pos = a.positions ? (uint32_t)min(max(a.positions[r], 0), (int32_t)(a.n_positions - 1u)) : r;
        const size_t at = (size_t)pos * (D / 2u) + 4u * l;
        const f32x4 c = *(const f32x4*)(a.rope_cos + at), sn = *(const f32x4*)(a.rope_sin + at);
        // the first and the second of each pair
        const f32x4 u = HALVES ? x0 : f32x4{x0.x, x0.z, x1.x, x1.z}, v = HALVES ? x1 : f32x4{x0.y, x0.w, x1.y, x1.w};
        const f32x4 y0 = u * c - v * sn, y1 = u * sn + v * c;
        x0 = HALVES ? y0 : f32x4{y0.x, y1.x, y0.y, y1.y};
        x1 = HALVES ? y1 : f32x4{y0.z, y1.z, y0.w, y1.w};
    }
    uint16_t* dst;
    if (is_q) {
        dst = (uint16_t*)a.q + (size_t)r * a.q_stride + (size_t)h * D;
    } else {
        const uint32_t kh = h - a.n_heads - (is_v ? a.n_kv_heads : 0u);
        dst = (uint16_t*)(is_v ? a.v : a.k);
        if (a.slots) {
            const uint32_t page = (uint32_t)slot >> a.page_log2;
            if (slot < 0 || page >= a.n_pages) return;
            dst += ((((size_t)page * a.n_kv_heads + kh) << a.page_log2) + ((uint32_t)slot & ((1u << a.page_log2) - 1u))) * D;
        } else {
            dst += (size_t)r * a.kv_stride + (size_t)kh * D;
        }
    }
    *(u32x2*)(dst + e0) = u32x2{pack16<OT>(x0.x, x0.y), pack16<OT>(x0.z, x0.w)};
    *(u32x2*)(dst + e1) = u32x2{pack16<OT>(x1.x, x1.y), pack16<OT>(x1.z, x1.w)};
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t st) {
    // a token a thread, up to two workgroups a CU; a small step is one workgroup
    const uint32_t items = a.n_tokens > a.n_seqs ? a.n_tokens : a.n_seqs;
    const uint32_t wgs = (items + kPlanThreads - 1u) / kPlanThreads;
    hipLaunchKernelGGL(paged_plan_kernel, dim3(wgs < 512u ? (wgs ? wgs : 1u) : 512u), dim3(kPlanThreads),
                       2u * (a.n_seqs + 1u) * 4u, st, a);
    return hipGetLastError();
}

hipError_t launch_qkv_tokens(const QkvTokensArgs& a, uint32_t dim, uint32_t otype, bool halves, hipStream_t st) {
    const uint32_t per = 256u / (dim / 8u);  // heads a workgroup
    // rows go on in z where there are more than x takes (its threads, 256 a row, stay under 2^32)
    const uint32_t x = a.n_tokens < kMaxGridRows ? a.n_tokens : kMaxGridRows;
    const dim3 grid(x, (a.n_heads + 2u * a.n_kv_heads + per - 1u) / per, (a.n_tokens + x - 1u) / x), block(256);
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
