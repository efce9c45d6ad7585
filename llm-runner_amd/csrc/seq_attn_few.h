// seq_attn_few.h - attention over a paged cache for requests of few new tokens
// (seq_attn.hip): at most 16 NR rows (new tokens x query heads of a group) a
// key/value head. Every key and value is read once for few products, so the
// kernel is a stream of the cache's pages; what it has to do is to keep enough
// of them in flight on every CU whatever the requests' lengths are.
//
// One wave a workgroup, four or so a CU, each with a ring of two tiles of 32 keys
// and values in its own LDS, filled by DMA; no wave waits for another. The keys
// of all (request, key/value head) pairs, cut into units of 32, make one line of
// W units; wave g of N <= W takes the units [g W / N, (g + 1) W / N) of it. A pair that one
// wave takes whole is written to `out` by it; the parts of the others go to
// `scratch` (f32 rows, their maximum and sum), at most two a wave (its first part,
// where the pair began before it, and its last), and a second launch joins them.
// So any mix of lengths fills the card to within one unit a wave, the scratch
// depends on no length, and the order of every sum is fixed.
//
// S^T = K Q^T by 16x16x32 MFMAs (16 keys x 16 rows), O^T += V^T P^T with P^T
// straight from the score registers: a lane's eight weights of a tile are the keys
// 4g .. 4g+3 and 16+4g .. of its row (g = lane / 16), and the transposing reads of V
// give the same keys.
#pragma once

#include "seq_attn_tile.h"

namespace llmr {
namespace seqattn {
namespace {

constexpr uint32_t kUnit = 32;  // keys of a unit

template <uint32_t T>
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (T == kGgmlBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// V: chunk c of key r at c ^ fswz(r): a transposing read's 16 keys x 2 chunks lie
// evenly over the 256 bytes the banks cover.
template <uint32_t D>
__device__ __forceinline__ uint32_t fswz(uint32_t r) {
    return D == 128u ? 2u * (r & 7u) : 2u * ((r >> 1) & 3u);
}

// One request of a paged call, from the device's lengths, in bounds whatever they hold.
struct PagedRequest {
    uint32_t first;  // its first row
    uint32_t rows;   // new tokens computed
    int32_t pos0;    // key that the first row sees last (negative: none)
    uint32_t keys;   // keys any row sees: 0 .. keys - 1
};
__device__ __forceinline__ PagedRequest paged_request(const SeqAttnArgs& a, uint32_t s) {
    const int64_t T = a.n_tokens, cap = (int64_t)a.max_pages << a.page_log2;
    const int64_t o0 = min(max((int64_t)a.offsets[s], (int64_t)0), T);
    const int64_t o1 = min(max((int64_t)a.offsets[s + 1u], (int64_t)0), T);
    const int64_t n = max(o1 - o0, (int64_t)0), rows = min(n, (int64_t)a.max_new);
    const int64_t pos0 = (int64_t)a.kv_len[s] - n;
    PagedRequest r;
    r.first = (uint32_t)o0;
    r.rows = (uint32_t)rows;
    r.pos0 = (int32_t)max(pos0, (int64_t)-0x7fffffff);  // (a row i < rows that sees no key stays so)
    r.keys = (uint32_t)min(max(pos0 + rows, (int64_t)0), cap);
    return r;
}
// Units of 32 keys of a request and head: one at least where it has rows (they are written).
__device__ __forceinline__ uint32_t units_of(const PagedRequest& r) {
    return r.rows ? max((r.keys + kUnit - 1u) / kUnit, 1u) : 0u;
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
    return ((uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)v, lane, 64);
}
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32) |
           (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
}
// Inclusive sum over the wave's lanes.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, uint32_t lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = shfl64(v, (int)lane - o);
        if (lane >= (uint32_t)o) v += x;
    }
    return v;
}

// Units before request `upto` (of one key/value head), by one wave.
__device__ __forceinline__ uint64_t units_before(const SeqAttnArgs& a, uint32_t upto, uint32_t lane) {
    uint64_t sum = 0;
    for (uint32_t s = lane; s < upto; s += 64u) sum += units_of(paged_request(a, s));
    return uniform64(shfl64(wave_scan(sum, lane), 63));
}

// Wave g of n takes the units [part_begin(g), part_begin(g + 1)) of w; the wave that has
// unit x. (w < 2^38 units x 1024 heads, n < 2^14.)
__device__ __forceinline__ uint64_t part_begin(uint64_t g, uint64_t w, uint32_t n) { return g * w / n; }
__device__ __forceinline__ uint32_t part_of(uint64_t x, uint64_t w, uint32_t n) {
    return (uint32_t)(((x + 1u) * n + w - 1u) / w - 1u);
}

// A part of a pair in scratch: O[16 NR][D], then m[16 NR], l[16 NR] (l = -1: the row
// sees no key of this part).
template <uint32_t D, uint32_t NR>
constexpr uint32_t part_floats() { return 16u * NR * (D + 2u); }

template <uint32_t T, uint32_t D, uint32_t NR>
__device__ __forceinline__ void few_rows(const SeqAttnArgs& a, uint8_t* lds, float* __restrict__ scratch) {
    constexpr uint32_t ROW = D * 2u, RPI = 1024u / ROW, CPR = ROW / 16u;
    constexpr uint32_t IPG = 16u / RPI;        // DMA instructions per 16 keys
    constexpr uint32_t TILE = kUnit * ROW;     // bytes of a K or V tile; lds: two of K, two of V
    constexpr int DMAS = 4 * (int)IPG;         // per unit: K and V, two groups of 16 keys each
    constexpr int CH = D / 32, DT = D / 16;
    constexpr float OFF = T == kGgmlF16 ? 7.0f : 0.0f;
    const uint32_t lane = threadIdx.x, n16 = lane & 15u, g = lane >> 4;
    const uint32_t G = a.n_heads / a.n_kv_heads;
    const float c = a.scale_log2, grow_by = 8.0f / c;

    // this wave's units
    const uint64_t w1 = units_before(a, a.n_seqs, lane), w = w1 * a.n_kv_heads;
    const uint32_t n = (uint32_t)min((uint64_t)gridDim.x, w);  // every wave has a unit
    if (blockIdx.x >= n) return;
    uint64_t at = part_begin(blockIdx.x, w, n);
    const uint64_t end = part_begin(blockIdx.x + 1u, w, n);
    // the request of unit `at`: the last one whose units begin at or before it
    uint32_t s = 0;
    uint64_t base = 0;  // units (all heads) before request s
    for (uint32_t s0 = 0; s0 < a.n_seqs; s0 += 64u) {
        const uint64_t u = s0 + lane < a.n_seqs ? (uint64_t)units_of(paged_request(a, s0 + lane)) * a.n_kv_heads : 0;
        const uint64_t inc = wave_scan(u, lane);
        const uint64_t here = __builtin_amdgcn_ballot_w64(base + inc > at);
        if (here != 0) {
            const int l = __builtin_ctzll(here);
            s = s0 + (uint32_t)l;
            base += uniform64(shfl64(inc - u, l));
            break;
        }
        base += uniform64(shfl64(inc, 63));
    }

    // DMA lane offsets within 16 keys; fragment addresses within a tile
    uint32_t kvo[IPG], vvo[IPG];
#pragma unroll
    for (uint32_t i = 0; i < IPG; i++) {
        const uint32_t r = RPI * i + lane / CPR, p = lane % CPR;
        kvo[i] = r * ROW + ((p ^ kswz<D>(r)) << 4);
        vvo[i] = r * ROW + ((p ^ fswz<D>(r)) << 4);
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds;
    uint32_t kfo[CH], vto[DT];
#pragma unroll
    for (int ch = 0; ch < CH; ch++) kfo[ch] = lds0 + n16 * ROW + (((4u * ch + g) ^ kswz<D>(n16)) << 4);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
        const uint32_t r = 4u * g + (n16 >> 2);
        vto[dt] = lds0 + 2u * TILE + r * ROW + (((2u * dt + ((n16 & 3u) >> 1)) ^ fswz<D>(r)) << 4) + 8u * (n16 & 1u);
    }

    while (at < end) {
        const PagedRequest rq = paged_request(a, s);
        const uint32_t units = units_of(rq);
        if (units == 0 || at >= base + (uint64_t)units * a.n_kv_heads) {  // (nothing new: no units)
            base += (uint64_t)units * a.n_kv_heads;
            s++;
            continue;
        }
        const uint32_t kvh = (uint32_t)((at - base) / units);
        const uint32_t u0 = (uint32_t)((at - base) % units);
        const uint32_t u1 = (uint32_t)min((uint64_t)units, u0 + (end - at));
        const int32_t* const table = a.table + (size_t)s * a.max_pages;

        // rows: 16 r + n16 = (token i, head of the group)
        const uint32_t rows = rq.rows * G;
        s16x8 qf[NR][CH];
        int32_t hi[NR];  // last key the row sees
        int32_t hi_min = 0x7fffffff;
#pragma unroll
        for (int r = 0; r < (int)NR; r++) {
            const uint32_t x = 16u * r + n16, xc = min(x, rows - 1u), i = xc / G;
            hi[r] = x < rows ? rq.pos0 + (int32_t)i : -1;
            if (x < rows) hi_min = min(hi_min, hi[r]);
            const uint16_t* q = (const uint16_t*)a.q + (size_t)(rq.first + i) * a.q_stride +
                                (size_t)(kvh * G + xc % G) * a.q_head_stride;
#pragma unroll
            for (int ch = 0; ch < CH; ch++) qf[r][ch] = *(const s16x8*)(q + 32 * ch + 8u * g);
        }
        hi_min = wave_imin(hi_min);

        f32x4 o[NR][DT];
        float m_ref[NR], l_i[NR];
        uint32_t fresh = (1u << NR) - 1u, sees = 0;  // per row block: no maximum yet; a key seen
        bool bad = false;                            // a masked tile's V has an infinity or NaN
#pragma unroll
        for (int r = 0; r < (int)NR; r++) {
            m_ref[r] = l_i[r] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[r][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // 16 keys from key k0 on: their page (negative: none)
        auto page_at = [&](uint32_t k0) -> int32_t {
            if (k0 >= rq.keys) return -1;
            const int32_t p = table[k0 >> a.page_log2];
            return p >= 0 && (uint32_t)p < a.n_pages ? p : -1;
        };
        auto dma = [&](uint32_t u, uint32_t slot) {
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                const uint32_t k0 = u * kUnit + 16u * h;
                const int32_t p = u < u1 ? page_at(k0) : -1;
                const uint64_t off = ((((uint64_t)(uint32_t)max(p, 0) * a.n_kv_heads + kvh) << a.page_log2) +
                                      (k0 & ((1u << a.page_log2) - 1u))) * ROW;
                const uint32_t left = p < 0 ? 0u : min(__builtin_elementwise_sub_sat(rq.keys, k0), 16u);
                const int bytes = (int)__builtin_amdgcn_readfirstlane(left * ROW);
                const rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)const_cast<void*>(a.k) + off, (short)0,
                                                                    bytes, 0x00020000);
                const rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)const_cast<void*>(a.v) + off, (short)0,
                                                                    bytes, 0x00020000);
                uint8_t* const kd = lds + slot * TILE + h * 16u * ROW;
#pragma unroll
                for (uint32_t i = 0; i < IPG; i++) {
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void*)(kd + 1024u * i), 16, kvo[i], 0, 0, 0);
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void*)(kd + 2u * TILE + 1024u * i), 16, vvo[i], 0,
                                                             0, 0);
                }
            }
        };
        // a row's weights of a tile are 0 where it does not see the key, and 0 times an
        // infinity or NaN is NaN: in masked tiles V's are set to 0, and the rows that do see
        // them, with a weight above 0, get them from memory after the last tile
        auto clean_v = [&](uint32_t u, uint32_t slot) {
#pragma unroll
            for (uint32_t i = 0; i < TILE / 1024u; i++) {
                u32x4* const p = (u32x4*)(lds + (2u + slot) * TILE + 1024u * i + 16u * lane);
                const u32x4 x = *p;
                const bool nf = nonfinite4<T>(x);
                if (__builtin_amdgcn_ballot_w64(nf) != 0) {
                    bad = true;
                    if (nf) *p = finite4<T>(x);
                }
            }
        };

        dma(u0, 0);
        dma(u0 + 1u, 1);
        for (uint32_t u = u0; u < u1; u++) {
            const uint32_t slot = (u - u0) & 1u;
            // keys past the last one, on no page, or unseen by a row: masked
            const bool v0 = page_at(u * kUnit) >= 0, v1 = page_at(u * kUnit + 16u) >= 0;
            const bool masked = !v0 || !v1 || (int32_t)(u * kUnit + kUnit - 1u) > hi_min;
            asm volatile("" ::: "memory");
            LLMR_WAIT_VMCNT(DMAS);  // this unit's K and V have landed
            asm volatile("" ::: "memory");
            if (masked) clean_v(u, slot);
            f32x4 sc[NR][2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int ch = 0; ch < CH; ch++) {
                    const s16x8 k = *(const lds_s16x8*)(uintptr_t)(kfo[ch] + slot * TILE + (uint32_t)kb * 16u * ROW);
#pragma unroll
                    for (int r = 0; r < (int)NR; r++)
                        sc[r][kb] = mfma16<T>(k, qf[r][ch], ch == 0 ? f32x4{} - m_ref[r] : sc[r][kb]);
                }
            s16x8 pf[NR];
#pragma unroll
            for (int r = 0; r < (int)NR; r++) {
                if (masked) {
                    const int32_t k0 = (int32_t)(u * kUnit + 4u * g);
                    bool any = false;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool a0 = v0 && k0 + i <= hi[r], a1 = v1 && k0 + 16 + i <= hi[r];
                        sc[r][0][i] = a0 ? sc[r][0][i] : -INFINITY;
                        sc[r][1][i] = a1 ? sc[r][1][i] : -INFINITY;
                        any = any || a0 || a1;
                    }
                    if (any) sees |= 1u << r;
                } else {
                    sees |= 1u << r;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; i++) mx = fmaxf(fmaxf(mx, sc[r][0][i]), sc[r][1][i]);
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const bool fr = (fresh >> r) & 1u;
                if (__builtin_amdgcn_ballot_w64(mx > grow_by || (fr && mx > -INFINITY)) != 0) {
                    const float d = fr ? (mx > -INFINITY ? mx : 0.0f) : fmaxf(mx, 0.0f);
                    const float alpha = fr ? 0.0f : __builtin_amdgcn_exp2f(-d * c);
                    m_ref[r] += d;
                    l_i[r] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[r][dt] *= alpha;
                    sc[r][0] -= d;
                    sc[r][1] -= d;
                    if (mx > -INFINITY) fresh &= ~(1u << r);
                }
                float p[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    p[i] = __builtin_amdgcn_exp2f(fmaf(sc[r][i >> 2][i & 3], c, OFF));
                    l_i[r] += p[i];
                }
                pf[r] = __builtin_bit_cast(s16x8, u32x4{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]), pack2<T>(p[4], p[5]),
                                                       pack2<T>(p[6], p[7])});
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(vto[dt] + slot * TILE));
                const s16x4 up =
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(vto[dt] + slot * TILE + 16u * ROW));
                const s16x8 v = s16x8{lo.x, lo.y, lo.z, lo.w, up.x, up.y, up.z, up.w};
#pragma unroll
                for (int r = 0; r < (int)NR; r++) o[r][dt] = mfma16<T>(v, pf[r], o[r][dt]);
            }
            // every read of this slot has arrived before its next tile is sent for
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
            asm volatile("" ::: "memory");
            dma(u + 2u, slot);
        }
        if (bad) {
            for (uint32_t u = u0; u < u1; u++) {
                const uint32_t j = u * kUnit + (lane & 31u);
                const int32_t p = j < rq.keys ? page_at(j & ~15u) : -1;
                if ((int32_t)(u * kUnit + kUnit - 1u) <= hi_min && __builtin_amdgcn_ballot_w64(p < 0) == 0) continue;
                const uint8_t* const vr =
                    (const uint8_t*)a.v + ((((uint64_t)(uint32_t)max(p, 0) * a.n_kv_heads + kvh) << a.page_log2) +
                                           (j & ((1u << a.page_log2) - 1u))) * ROW;
                bool nf = false;
                if (p >= 0)
                    for (uint32_t b = 0; b < CPR; b++) nf = nf || nonfinite4<T>(*(const u32x4*)(vr + 16u * b));
                for (uint64_t todo = __builtin_amdgcn_ballot_w64(nf) & 0xffffffffull; todo != 0; todo &= todo - 1u) {
                    const int l = __builtin_ctzll(todo);
                    const uint8_t* const row = (const uint8_t*)uniform64(shfl64((uint64_t)(uintptr_t)vr, l));
                    const int32_t key = (int32_t)(u * kUnit) + l;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        const u32x2 v = *(const u32x2*)(row + 32u * dt + 8u * g);
                        const float x[4] = {lo_f32<T>(v.x), hi_f32<T>(v.x), lo_f32<T>(v.y), hi_f32<T>(v.y)};
#pragma unroll
                        for (int r = 0; r < (int)NR; r++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                o[r][dt][e] += (int)(key <= hi[r]) & (int)!(fabsf(x[e]) < INFINITY) ? x[e] : 0.0f;
                    }
                }
            }
        }

        const bool whole = u0 == 0 && u1 == units;
        float* const part = scratch + (size_t)(2u * blockIdx.x + (u0 == 0 ? 1u : 0u)) * part_floats<D, NR>();
#pragma unroll
        for (int r = 0; r < (int)NR; r++) {
            float l = l_i[r];
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            // a row's four lanes have seen different keys of a masked tile
            uint32_t sn = (sees >> r) & 1u;
            sn |= (uint32_t)__shfl_xor((int)sn, 16, 64);
            sn |= (uint32_t)__shfl_xor((int)sn, 32, 64);
            const uint32_t x = 16u * r + n16;
            if (x >= rows) continue;
            if (whole) {
                const uint32_t i = x / G;
                uint16_t* const dst = (uint16_t*)a.out + (size_t)(rq.first + i) * a.out_stride + (kvh * G + x % G) * D + 4u * g;
                const float inv = 1.0f / l;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const f32x4 v = o[r][dt] * inv;
                    *(u32x2*)(dst + 16 * dt) = sn ? u32x2{pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)} : u32x2{0u, 0u};
                }
            } else {
#pragma unroll
                for (int dt = 0; dt < DT; dt++) *(f32x4*)(part + x * D + 16u * dt + 4u * g) = o[r][dt];
                if (g == 0) {
                    part[16u * NR * D + x] = (fresh >> r) & 1u ? -INFINITY : m_ref[r];
                    part[16u * NR * (D + 1u) + x] = sn ? l : -1.0f;
                }
            }
        }
        at += u1 - u0;
        asm volatile("" ::: "memory");
        LLMR_WAIT_VMCNT(0);  // the last tiles' DMAs (of no keys) are done with the ring
        asm volatile("" ::: "memory");
    }
}

template <uint32_t T, uint32_t D, uint32_t NR>
__global__ void __launch_bounds__(64, 1) paged_attn_few(SeqAttnArgs a, float* __restrict__ scratch) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[4u * kUnit * D * 2u];
    few_rows<T, D, NR>(a, lds, scratch);
}

// One row's dims d .. d + 3 of the parts g0 .. g1, in their order, divided by the sum; false:
// the row sees no key. part(g): O[rows][D], m[rows], l[rows] of part g.
template <typename Part>
__device__ __forceinline__ bool join_row(uint32_t g0, uint32_t g1, float c, const Part& part, uint32_t rows, uint32_t D,
                                         uint32_t x, uint32_t d, f32x4& out) {
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    bool sees = false;
    for (uint32_t g = g0; g <= g1; g++) {
        const float* const p = part(g);
        const float pm = p[rows * D + x], pl = p[rows * (D + 1u) + x];
        const f32x4 po = *(const f32x4*)(p + x * D + d);
        if (pl == -1.0f) continue;  // no key of this part is seen
        const float mx = fmaxf(m, pm);
        // (a part whose scores are all -inf has m = -inf and sums of 0 or NaN)
        const float fo = !sees || m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * c);
        const float fp = pm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((pm - mx) * c);
        o = o * fo + po * fp;
        l = l * fo + pl * fp;
        m = mx;
        sees = true;
    }
    out = o * (1.0f / l);
    return sees;
}

// Joins the parts of a (request, key/value head) pair that more than one wave took, in
// their order. waves: the grid of paged_attn_few.
template <uint32_t T, uint32_t D, uint32_t NR>
__global__ void __launch_bounds__(256) paged_attn_join(SeqAttnArgs a, const float* __restrict__ scratch, uint32_t waves) {
    const uint32_t s = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
    const uint32_t G = a.n_heads / a.n_kv_heads;
    const PagedRequest rq = paged_request(a, s);
    const uint32_t units = units_of(rq);
    if (units <= 1u) return;
    const uint64_t w = units_before(a, a.n_seqs, tid & 63u) * a.n_kv_heads;
    const uint64_t begin = units_before(a, s, tid & 63u) * a.n_kv_heads + (uint64_t)kvh * units;
    const uint32_t n = (uint32_t)min((uint64_t)waves, w);
    const uint32_t g0 = part_of(begin, w, n), g1 = part_of(begin + units - 1u, w, n);
    if (g0 == g1) return;
    for (uint32_t e = tid; e < rq.rows * G * (D / 4u); e += 256u) {
        const uint32_t x = e / (D / 4u), d = 4u * (e % (D / 4u));
        f32x4 v;
        const bool sees = join_row(
            g0, g1, a.scale_log2,
            [&](uint32_t g) { return scratch + (size_t)(2u * g + (g == g0 ? 1u : 0u)) * part_floats<D, NR>(); }, 16u * NR, D,
            x, d, v);
        uint16_t* const dst = (uint16_t*)a.out + (size_t)(rq.first + x / G) * a.out_stride + (kvh * G + x % G) * D + d;
        *(u32x2*)dst = sees ? u32x2{pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)} : u32x2{0u, 0u};
    }
}

}  // namespace
}  // namespace seqattn
}  // namespace llmr
