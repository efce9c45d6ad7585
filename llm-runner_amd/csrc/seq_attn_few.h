// seq_attn_few.h - attention over a paged cache for requests of few new tokens
// (seq_attn.hip): at most 16 NR rows (new tokens x query heads of a group) a
// key/value head. Every key and value is read once for few products, so the
// kernel is a stream of the cache's pages; what it has to do is to keep enough
// of them in flight on every CU whatever the requests' lengths are.
//
// One wave a workgroup, four, three or two a CU (up to 16, 32, 64 rows: what the LDS of
// head_dim 128 lets reside), each with a ring of two units (32 keys, their
// values, and where a pair begins its queries) in its own LDS, sent for by DMA two
// units ahead, over the ends of pairs; no wave waits for another. (As built, the
// block table's entries are vector loads, and waiting for one waits for the DMAs in
// flight too, four times a unit: it is the other waves' units that keep the memory
// busy meanwhile.) The keys of all
// (request, key/value head) pairs, cut into units of 32, make one line of W units;
// wave g of N <= W takes the units [g W / N, (g + 1) W / N) of it. A pair that one
// wave takes whole is written to `out` by it; the parts of the others go to
// `scratch` (f32 rows, their maximum and sum), at most two a wave (its first part,
// where the pair began before it, and its last), and a second launch joins them,
// by a record that the wave of a pair's first part leaves. So any mix of lengths
// fills the card to within one unit a wave, the scratch depends on no length, and
// the order of every sum is fixed.
//
// S^T = K Q^T by 16x16x32 MFMAs (16 keys x 16 rows), O^T += V^T P^T with P^T
// straight from the score registers: a lane's eight weights of a tile are the keys
// 4g .. 4g+3 and 16+4g .. of its row (g = lane / 16), and the transposing reads of V
// give the same keys.
//
// Memory bounds it where enough is in flight, single tokens at head_dim 128: 4 x 85000
// keys of 32/8 heads (1.39 GB) 270 us and 6 for the join, 5.1 TB/s, which is what a large
// copy reaches; 64 ragged contexts of 100 to 12000 keys, 30/6 heads, fp16 (0.47 GB) 109 and
// 5, with pages of 16, 64 and 256 alike. Queries by ordinary loads at a pair's beginning, a wave
// waiting for its own, and a join that searched for its parts: 320 and 141. Head_dim 64
// has half the bytes in flight: 213 us for the 4 x 85000 keys (3.3 TB/s). More rows take
// longer than the bytes: 8 and 16 new tokens (32 and 64 rows) 366 and 687 us at 128, 296
// and 493 at 64, where paged_attn_tiles takes 284 and 285, 145 and 153; the 64 rows of 128
// do not fit the registers (200 bytes a lane go to scratch memory, within the loop too).
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

// Wave g of n takes the units [part_begin(g), part_begin(g + 1)) of w; the wave that has
// unit x. (w < 2^38 units x 1024 heads, n < 2^14.)
__device__ __forceinline__ uint64_t part_begin(uint64_t g, uint64_t w, uint32_t n) { return g * w / n; }
__device__ __forceinline__ uint32_t part_of(uint64_t x, uint64_t w, uint32_t n) {
    return (uint32_t)(((x + 1u) * n + w - 1u) / w - 1u);
}

// What a worker leaves about the rows whose first part it has and not the last (last = 0
// otherwise): parts of the workers it .. last, of rows `row0` .. + n of a request's rows
// (token, head in group) that starts at token `first`, of key/value head kvh.
struct JoinRecord {
    uint32_t last, first, row0, n, kvh, pad[3];
};

// The requests of a call, 64 at a time in the lanes of a wave, and the units before them.
struct RequestWindow {
    PagedRequest mine;  // request s0 + lane
    uint32_t s0;
    __device__ __forceinline__ void load(const SeqAttnArgs& a, uint32_t from, uint32_t lane) {
        s0 = from;
        mine = from + lane < a.n_seqs ? paged_request(a, from + lane) : PagedRequest{0, 0, 0, 0};
    }
    __device__ __forceinline__ PagedRequest get(uint32_t s) const {
        const int l = (int)(s - s0);
        return {(uint32_t)__builtin_amdgcn_readlane((int)mine.first, l), (uint32_t)__builtin_amdgcn_readlane((int)mine.rows, l),
                __builtin_amdgcn_readlane(mine.pos0, l), (uint32_t)__builtin_amdgcn_readlane((int)mine.keys, l)};
    }
};

// The sum of cost(request) over the batch, and the window (loaded where one is not enough)
// moved to the request of unit x (heads * cost units each): it, and the units before it.
template <typename Cost>
__device__ __forceinline__ uint64_t batch_cost(const SeqAttnArgs& a, RequestWindow& win, uint32_t lane, const Cost& cost) {
    uint64_t sum = 0;
    for (uint32_t s0 = 0; s0 < a.n_seqs; s0 += 64u) {
        win.load(a, s0, lane);
        sum += cost(win.mine);
    }
    return uniform64(shfl64(wave_scan(sum, lane), 63));
}
template <typename Cost>
__device__ __forceinline__ uint32_t find_request(const SeqAttnArgs& a, RequestWindow& win, uint32_t lane, const Cost& cost,
                                                 uint32_t heads, uint64_t x, uint64_t& base) {
    base = 0;
    for (uint32_t s0 = 0; s0 < a.n_seqs; s0 += 64u) {
        if (a.n_seqs > 64u) win.load(a, s0, lane);
        const uint64_t u = cost(win.mine) * heads, inc = wave_scan(u, lane);
        const uint64_t here = __builtin_amdgcn_ballot_w64(base + inc > x);
        if (here != 0) {
            const int l = __builtin_ctzll(here);
            base += uniform64(shfl64(inc - u, l));
            return s0 + (uint32_t)l;
        }
        base += uniform64(shfl64(inc, 63));
    }
    return a.n_seqs;
}

// Adds a part's O, m, l to (o, m, l); l = -1: no key seen.
__device__ __forceinline__ void join_part(f32x4& o, float& m, float& l, f32x4 po, float pm, float pl, float c) {
    if (pl == -1.0f) return;
    const float mx = fmaxf(m, pm);
    // (a part whose scores are all -inf has m = -inf and sums of 0 or NaN)
    const float fo = l == -1.0f || m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mx) * c);
    const float fp = pm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((pm - mx) * c);
    const bool both = l != -1.0f;
    o = both ? o * fo + po * fp : po * fp;
    l = both ? l * fo + pl * fp : pl * fp;
    m = mx;
}

// A part of a pair in scratch: O[16 NR][D], then m[16 NR], l[16 NR] (l = -1: the row
// sees no key of this part). The records come first.
template <uint32_t D, uint32_t NR>
constexpr uint32_t part_floats() { return 16u * NR * (D + 2u); }

// A unit of 32 keys of a pair.
struct FewUnit {
    PagedRequest rq;
    uint32_t s, kvh, u, units;
    bool first;  // of this wave's part of the pair: its queries come with it
};

template <uint32_t T, uint32_t D, uint32_t NR>
__device__ __forceinline__ void few_rows(const SeqAttnArgs& a, uint8_t* lds, JoinRecord* __restrict__ records,
                                         float* __restrict__ parts) {
    constexpr uint32_t ROW = D * 2u, RPI = 1024u / ROW, CPR = ROW / 16u;
    constexpr uint32_t IPG = 16u / RPI;        // DMA instructions per 16 rows
    constexpr uint32_t TILE = kUnit * ROW;     // bytes of a K or V tile; lds: two of K, two of V, two of Q
    constexpr uint32_t QT = 16u * NR * ROW;    // bytes of Q
    constexpr int DMAS = 4 * (int)IPG;         // per unit: K and V, two groups of 16 keys each
    constexpr int QI = (int)(NR * IPG);        // and Q
    constexpr int CH = D / 32, DT = D / 16;
    constexpr float OFF = T == kGgmlF16 ? 7.0f : 0.0f;
    const uint32_t lane = threadIdx.x, n16 = lane & 15u, g = lane >> 4;
    const uint32_t G = a.n_heads / a.n_kv_heads;
    const float c = a.scale_log2, grow_by = 8.0f / c;
    const auto cost = [](const PagedRequest& r) { return (uint64_t)units_of(r); };

    // this wave's units
    RequestWindow win;
    const uint64_t w = batch_cost(a, win, lane, cost) * a.n_kv_heads;
    const uint32_t n = (uint32_t)min((uint64_t)gridDim.x, w);  // every wave has a unit
    JoinRecord rec{};
    if (blockIdx.x >= n) {
        if (lane == 0) records[blockIdx.x].last = 0;
        return;
    }
    const uint64_t at = part_begin(blockIdx.x, w, n);
    uint64_t left = part_begin(blockIdx.x + 1u, w, n) - at;  // units to send for

    // DMA lane offsets within 16 rows; fragment addresses within a tile
    uint32_t kvo[IPG], vvo[IPG], qvo[NR * IPG];
#pragma unroll
    for (uint32_t i = 0; i < IPG; i++) {
        const uint32_t r = RPI * i + lane / CPR, p = lane % CPR;
        kvo[i] = r * ROW + ((p ^ kswz<D>(r)) << 4);
        vvo[i] = r * ROW + ((p ^ fswz<D>(r)) << 4);
#pragma unroll
        for (uint32_t b = 0; b < NR; b++) {  // row x = (token x / G, head of the group x % G)
            const uint32_t x = 16u * b + r;
            qvo[b * IPG + i] = (x / G * a.q_stride + x % G * a.q_head_stride) * 2u + ((p ^ kswz<D>(r)) << 4);
        }
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

    // 16 keys from key k0 on: their page (negative: none)
    auto page_at = [&](const FewUnit& x, uint32_t k0) -> int32_t {
        if (k0 >= x.rq.keys) return -1;
        const int32_t p = a.table[(size_t)x.s * a.max_pages + (k0 >> a.page_log2)];
        return p >= 0 && (uint32_t)p < a.n_pages ? p : -1;
    };
    auto dma = [&](const FewUnit& x, uint32_t slot) {
        if (x.first) {
            // the rows there are end before offset rows * q_stride, the first one there is not
            const uint32_t bytes = ((x.rq.rows - 1u) * a.q_stride + (G - 1u) * a.q_head_stride + D) * 2u;
            const rsrc_t qr = __builtin_amdgcn_make_buffer_rsrc(
                (uint8_t*)const_cast<void*>(a.q) +
                    2u * ((uint64_t)x.rq.first * a.q_stride + (uint64_t)x.kvh * G * a.q_head_stride),
                (short)0, (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
            uint8_t* const qd = lds + 4u * TILE + slot * QT;
#pragma unroll
            for (int i = 0; i < QI; i++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(qr, (lds_void*)(qd + 1024u * i), 16, qvo[i], 0, 0, 0);
        }
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
            const uint32_t k0 = x.u * kUnit + 16u * h;
            const int32_t p = page_at(x, k0);
            const uint64_t off = ((((uint64_t)(uint32_t)max(p, 0) * a.n_kv_heads + x.kvh) << a.page_log2) +
                                  (k0 & ((1u << a.page_log2) - 1u))) * ROW;
            const uint32_t keys = p < 0 ? 0u : min(__builtin_elementwise_sub_sat(x.rq.keys, k0), 16u);
            const int bytes = (int)__builtin_amdgcn_readfirstlane(keys * ROW);
            const rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)const_cast<void*>(a.k) + off, (short)0, bytes,
                                                                0x00020000);
            const rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)const_cast<void*>(a.v) + off, (short)0, bytes,
                                                                0x00020000);
            uint8_t* const kd = lds + slot * TILE + h * 16u * ROW;
#pragma unroll
            for (uint32_t i = 0; i < IPG; i++) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void*)(kd + 1024u * i), 16, kvo[i], 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void*)(kd + 2u * TILE + 1024u * i), 16, vvo[i], 0, 0, 0);
            }
        }
    };
    // the unit behind x on the line
    auto next_of = [&](const FewUnit& x) -> FewUnit {
        FewUnit y = x;
        y.u++;
        y.first = false;
        if (y.u == y.units) {
            y.u = 0;
            y.first = true;
            if (++y.kvh == a.n_kv_heads) {
                y.kvh = 0;
                do {  // (units are left, so there is a request that has some)
                    y.s++;
                    if (y.s - win.s0 >= 64u) win.load(a, y.s, lane);
                    y.rq = win.get(y.s);
                    y.units = units_of(y.rq);
                } while (y.units == 0 && y.s + 1u < a.n_seqs);
            }
        }
        return y;
    };

    FewUnit cur, next{};
    {
        uint64_t base;
        cur.s = find_request(a, win, lane, cost, a.n_kv_heads, at, base);
        cur.rq = win.get(cur.s);
        cur.units = units_of(cur.rq);
        cur.kvh = (uint32_t)((at - base) / cur.units);
        cur.u = (uint32_t)((at - base) % cur.units);
        cur.first = true;
        dma(cur, 0);
        left--;
        if (left) {
            next = next_of(cur);
            dma(next, 1);
        }
    }
    bool begun = cur.u == 0;  // this wave has the first part of the pair it is at

    s16x8 qf[NR][CH];
    int32_t hi[NR], hi_min = 0;  // last key the row sees
    f32x4 o[NR][DT];
    float m_ref[NR], l_i[NR];
    uint32_t fresh = 0, sees = 0, u0 = 0;  // per row block: no maximum yet; a key seen; the part's first unit
    bool bad = false;                      // a masked tile's V has an infinity or NaN
    // a row's weights of a tile are 0 where it does not see the key, and 0 times an
    // infinity or NaN is NaN: in masked tiles V's are set to 0, and the rows that do see
    // them, with a weight above 0, get them from memory after the part's last tile
    auto clean_v = [&](uint32_t slot) {
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
    auto add_bad = [&]() {
        for (uint32_t u = u0; u <= cur.u; u++) {
            const uint32_t j = u * kUnit + (lane & 31u);
            const int32_t p = page_at(cur, j & ~15u);
            if ((int32_t)(u * kUnit + kUnit - 1u) <= hi_min && __builtin_amdgcn_ballot_w64(p < 0) == 0) continue;
            const uint8_t* const vr =
                (const uint8_t*)a.v + ((((uint64_t)(uint32_t)max(p, 0) * a.n_kv_heads + cur.kvh) << a.page_log2) +
                                       (j & ((1u << a.page_log2) - 1u))) * ROW;
            bool nf = false;
            if (p >= 0 && j < cur.rq.keys)
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
    };
    // the part that ends with unit cur
    auto finish = [&]() {
        const bool last = cur.u + 1u == cur.units, whole = begun && last;
        const uint32_t rows = cur.rq.rows * G;
        float* const part = parts + (size_t)(2u * blockIdx.x + (begun ? 1u : 0u)) * part_floats<D, NR>();
        if (begun && !last) {  // (the wave's last part: the record is its one)
            const uint64_t end = part_begin(blockIdx.x + 1u, w, n) + (cur.units - 1u - cur.u);  // of the pair
            rec = JoinRecord{part_of(end - 1u, w, n), cur.rq.first, 0, rows, cur.kvh, {}};
        }
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
                uint16_t* const dst = (uint16_t*)a.out + (size_t)(cur.rq.first + x / G) * a.out_stride +
                                      (cur.kvh * G + x % G) * D + 4u * g;
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
    };

    for (uint32_t slot = 0;; slot ^= 1u) {
        // this unit's data have landed; at most the next one's are on their way
        asm volatile("" ::: "memory");
        if (left == 0) {
            LLMR_WAIT_VMCNT(0);
        } else if (next.first) {
            LLMR_WAIT_VMCNT(DMAS + QI);
        } else {
            LLMR_WAIT_VMCNT(DMAS);
        }
        asm volatile("" ::: "memory");
        if (cur.first) {
            const uint32_t rows = cur.rq.rows * G;
            u0 = cur.u;
            fresh = (1u << NR) - 1u;
            sees = 0;
            bad = false;
            hi_min = 0x7fffffff;
#pragma unroll
            for (int r = 0; r < (int)NR; r++) {
                const uint32_t x = 16u * r + n16;
                hi[r] = x < rows ? cur.rq.pos0 + (int32_t)(x / G) : -1;
                if (x < rows) hi_min = min(hi_min, hi[r]);
                m_ref[r] = l_i[r] = 0.0f;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[r][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ch = 0; ch < CH; ch++)
                    qf[r][ch] = *(const lds_s16x8*)(uintptr_t)(kfo[ch] + 4u * TILE + slot * QT + (uint32_t)r * 16u * ROW);
            }
            // (the first token's rows see least)
            hi_min = __builtin_amdgcn_readfirstlane(hi_min);
        }
        // keys past the last one, on no page, or unseen by a row: masked
        const bool v0 = page_at(cur, cur.u * kUnit) >= 0, v1 = page_at(cur, cur.u * kUnit + 16u) >= 0;
        const bool masked = !v0 || !v1 || (int32_t)(cur.u * kUnit + kUnit - 1u) > hi_min;
        if (masked) clean_v(slot);
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
                const int32_t k0 = (int32_t)(cur.u * kUnit + 4u * g);
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
                // (only rows whose own maximum calls for it)
                const float d = fr ? (mx > -INFINITY ? mx : 0.0f) : (mx > grow_by ? mx : 0.0f);
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
        // every read of this slot has arrived before its next unit is sent for
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
        asm volatile("" ::: "memory");
        if (left == 0) break;
        FewUnit after{};
        const bool more = --left != 0;
        if (more) {
            after = next_of(next);
            dma(after, slot);
        }
        if (next.first) {
            if (bad) add_bad();
            finish();
            begun = true;
        }
        cur = next;
        next = after;
    }
    if (bad) add_bad();
    finish();
    if (lane == 0) records[blockIdx.x] = rec;
}

template <uint32_t T, uint32_t D, uint32_t NR>
__global__ void __launch_bounds__(64, 1)
paged_attn_few(SeqAttnArgs a, JoinRecord* __restrict__ records, float* __restrict__ parts) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[(4u * kUnit + 32u * NR) * D * 2u];
    few_rows<T, D, NR>(a, lds, records, parts);
}

// Joins the parts that worker blockIdx.y's record names, in their order: 16 rows a workgroup
// (blockIdx.x; side by side, so that a record's rows go to all XCDs: 512 new tokens behind
// 30000, every fourth worker with a record, 21.6 -> 12.0 us), as many of them at a time as the
// threads hold, or fewer with their parts shared by several groups of D / 4 threads, so that no
// row takes more than a few rounds of loads (35 parts of four rows: 21.8 -> 6.0). PR: rows of a
// part.
// Parts of 16 rows come from many waves (138 of five rows where one of 20306 keys is the
// longest of five): 16 rows or shares at a time, eight parts' loads in flight a thread; 56 ->
// 42 us for that call, 14.0 -> 12.6 for one request of 1100 keys. Larger parts are fewer and
// have rows enough: with as many threads 24 mixed requests took 43 us for 39. Eight loads in
// flight are worth it for parts of 32 rows too, us: 16 x 4 tokens of 28 heads over a 4-bit cache
// 32.3 -> 31.5; over a 16-bit one, with the kernel before it, one request of 1100 keys with 8 tokens
// of four heads 27.8 -> 25.0, 8 x 5 tokens 25.8 -> 24.4, four of 40000 to 131000 keys 363 -> 360, 64 x 5
// tokens 159 both, 16 x 4 tokens of 28/4 heads of 64 81.6 -> 83.7 (the join itself 11.4 -> 9.5 there).
template <uint32_t D, uint32_t PR>
constexpr uint32_t join_threads() { return PR == 16u ? 4u * D : 256u; }

template <uint32_t T, uint32_t D, uint32_t PR>
__global__ void __launch_bounds__((join_threads<D, PR>()))
paged_attn_join(SeqAttnArgs a, const JoinRecord* __restrict__ records, const float* __restrict__ parts) {
    constexpr uint32_t LPR = D / 4u, GROUPS = join_threads<D, PR>() / LPR;  // threads of a row, rows or shares at a time
    constexpr uint32_t LOADS = PR <= 32u ? 8u : 4u;  // parts of a thread in flight
    __shared__ f32x4 so[GROUPS][LPR];
    __shared__ float sm[GROUPS], sl[GROUPS];
    const uint32_t worker = blockIdx.y, x0 = 16u * blockIdx.x;
    const JoinRecord rec = records[worker];
    if (rec.last == 0 || x0 >= rec.n) return;
    const uint32_t rows = min(rec.n - x0, 16u), n_parts = rec.last - worker + 1u;
    // shares of a row's parts: GROUPS / (rows rounded up to a power of two)
    uint32_t shares = GROUPS;
    while (shares > 1u && shares * rows > GROUPS) shares /= 2u;
    const uint32_t at_once = GROUPS / shares;
    const uint32_t grp = threadIdx.x / LPR, d = 4u * (threadIdx.x % LPR), share = grp % shares;
    for (uint32_t r0 = 0; r0 < rows; r0 += at_once) {
        const uint32_t x = x0 + r0 + grp / shares;
        const bool live = r0 + grp / shares < rows;
        f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = -1.0f;  // l = -1: no key seen
        if (live) {
            for (uint32_t i0 = share; i0 < n_parts; i0 += LOADS * shares) {
                float pm[LOADS], pl[LOADS];
                f32x4 po[LOADS];
#pragma unroll
                for (int k = 0; k < (int)LOADS; k++) {
                    const uint32_t i = min(i0 + (uint32_t)k * shares, n_parts - 1u);
                    // a worker's second part where it is the rows' first
                    const float* const p = parts + (size_t)(2u * (worker + i) + (i == 0 ? 1u : 0u)) * (PR * (D + 2u));
                    pm[k] = p[PR * D + x];
                    pl[k] = i0 + (uint32_t)k * shares < n_parts ? p[PR * (D + 1u) + x] : -1.0f;
                    po[k] = *(const f32x4*)(p + x * D + d);
                }
#pragma unroll
                for (int k = 0; k < (int)LOADS; k++) join_part(o, m, l, po[k], pm[k], pl[k], a.scale_log2);
            }
        }
        if (shares > 1u) {
            so[grp][threadIdx.x % LPR] = o;
            if (threadIdx.x % LPR == 0) {
                sm[grp] = m;
                sl[grp] = l;
            }
            __syncthreads();
            if (share == 0)
                for (uint32_t k = 1; k < shares; k++)
                    join_part(o, m, l, so[grp + k][threadIdx.x % LPR], sm[grp + k], sl[grp + k], a.scale_log2);
            __syncthreads();
        }
        if (live && share == 0) {
            const uint32_t r = rec.row0 + x, G = a.n_heads / a.n_kv_heads;
            const f32x4 v = o * (1.0f / l);
            uint16_t* const dst = (uint16_t*)a.out + (size_t)(rec.first + r / G) * a.out_stride +
                                  (rec.kvh * G + r % G) * D + d;
            *(u32x2*)dst = l != -1.0f ? u32x2{pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)} : u32x2{0u, 0u};
        }
    }
}

}  // namespace
}  // namespace seqattn
}  // namespace llmr
