// mx4_attn_few.h - attention over a paged cache in 4 bits for requests of few new tokens
// (mx4_attn.hip): at most 16 NR rows (new tokens x query heads of a group) a key/value head.
//
// As paged_attn_few, a stream of the cache: the keys of all (request, key/value head) pairs, cut
// into units of 32, make one line that the workers share evenly; a worker has at most two parts of
// pairs, which paged_attn_join joins. What differs follows from the rows being short (64 bytes of
// numbers and 4 of powers of two at head_dim 128):
//  - a worker is a workgroup of four waves that take its units in turn and add up their rows in
//    LDS at a pair's end. With a wave a worker, as many waves as the short rows need would leave
//    four times the parts to join;
//  - keys and values come into registers, two units on their way, each register asked for again as
//    soon as it is free (4 x 131000..40000 keys 88 -> 80 us), past the caches: a step reads a cache
//    once. The rows' addresses are made for 32 units at once, a half of a unit a lane;
//  - a lane has a quarter of a key's row (a block of 32, at head_dim 128), which is what its
//    products with the queries take if the dims are dealt out so (lane group g: dims D/4 g ..; the
//    queries alike), so that keys need no LDS. Values pass through LDS in any case: four lanes side
//    by side have one row, a quarter of the addresses to look up (4 x 131000..40000 keys at head_dim
//    64 54 -> 48 us; the keys alike, by a way through LDS of their own: 49);
//  - v_cvt_scalef32_pk_{bf16,f16}_fp4 turns two numbers and their power of two into 16-bit values,
//    exactly, at the rate of an f32 fma: a unit's 8192 elements are 64 instructions a wave. The
//    values are written to LDS as 16-bit rows and read transposed.
// S^T = K Q^T and O^T += V^T P^T by 16x16x32 MFMAs, the softmax and the treatment of masked keys
// as in paged_attn_few: scores, maxima, sums and O are f32; P is rounded to the values' type for
// its product, as the MFMA takes it.
// Measured in a graph, us, floors by bytes: 4 x 131000..40000 keys of 8 heads of 128, one token
// each 78 (71.6 at a large copy's rate: 4.7 TB/s), eight 98; 64 x 100..12000 keys of 6 heads 37
// (24.3); one of 1100 keys 10.7 (two launches and a pair's start). Bound by HBM at long contexts,
// at short ones by the workers' starts, the last of them, and the join. (Counters, of a wave's
// cycles: waits 41 to 49%, for its turn to issue 16 to 28%, VALU 17 to 24%.)
#pragma once

#include "seq_attn_few.h"

namespace llmr {
namespace mx4attn {
namespace {

using namespace seqattn;

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

constexpr uint32_t kWaves = 4;         // of a worker
constexpr uint32_t kTopPower = 127 + 13;  // of what llmr_qkv_tokens_mx4 writes; above it values may be infinite, at 255 NaN
// A pair's units on the line: those of its keys, the first of them kPairStart units more, for what a
// pair costs a worker (its pages, queries and first rows waited for, its rows added up).
constexpr uint32_t kPairStart = 12;

struct Mx4Args {
    SeqAttnArgs a;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
};

// A lane's share of a unit's keys or values: of keys n16 and 16 + n16, dims D/4 g .. + D/4 - 1.
template <uint32_t D>
struct Half4 {
    uint32_t n[2][D / 32], power[2];
};
template <uint32_t D>
struct Mx4Unit {
    Half4<D> k, v;
    uint64_t row[2];  // (uniform) the cache's rows where its halves begin
    bool on[2];       // (uniform) the halves have a page
};

template <uint32_t D, uint32_t NR>
constexpr uint32_t few_lds_bytes() { return kWaves * (32u * D * 2u) + kWaves * 16u * 2u * 4u; }

template <uint32_t T, uint32_t D, uint32_t NR>
__device__ __forceinline__ void few_rows(const Mx4Args& m4, uint8_t* lds, JoinRecord* __restrict__ records,
                                         float* __restrict__ parts) {
    const SeqAttnArgs& a = m4.a;
    constexpr uint32_t ROW4 = D / 2u, CB = D / 8u, SROW = D / 32u;  // bytes: a row's numbers, a lane's, a row's powers
    constexpr uint32_t ROW = D * 2u, TILE = 32u * ROW;              // of 16-bit values: a row, a wave's tile of V
    constexpr int ND = D / 32, DT = D / 16;
    constexpr float OFF = T == kGgmlF16 ? 7.0f : 0.0f;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n16 = lane & 15u, g = lane >> 4;
    const uint32_t vrow = lane >> 2, vg = lane & 3u;  // of V's loads
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t G = a.n_heads / a.n_kv_heads;
    const float c = a.scale_log2, grow_by = 8.0f / c;
    const auto cost = [](const PagedRequest& r) { return r.rows ? (uint64_t)units_of(r) + kPairStart : 0ull; };

    RequestWindow win;
    const uint64_t w = batch_cost(a, win, lane, cost) * a.n_kv_heads;
    // a unit a wave at least, while there are few
    const uint32_t n = (uint32_t)min((uint64_t)gridDim.x, (w + kWaves - 1u) / kWaves);
    JoinRecord rec{};
    if (blockIdx.x >= n) {
        if (tid == 0) records[blockIdx.x].last = 0;
        return;
    }
    uint64_t at = part_begin(blockIdx.x, w, n);
    const uint64_t end = part_begin(blockIdx.x + 1u, w, n);

    const uint32_t ko = n16 * ROW4 + g * CB, kso = n16 * SROW + (D == 128u ? g : g >> 1);
    const uint32_t vo = vrow * ROW4 + vg * CB, vso = vrow * SROW + (D == 128u ? vg : vg >> 1);
    uint8_t* const vt = lds + wave * TILE;
    const uint32_t vt0 = (uint32_t)(uintptr_t)(lds_void*)vt;
    // V's tile: chunk q of key r at q ^ fswz(r), fswz even: chunk 2 dt + x of a row is at A ^ 32 dt, and chunk ND g + e
    // at B ^ 16 e
    const uint32_t vr0 = 4u * g + (n16 >> 2);
    uint32_t va = vr0 * ROW + ((((n16 & 3u) >> 1) ^ fswz<D>(vr0)) << 4) + 8u * (n16 & 1u);
    uint32_t vb = vrow * ROW + (((ND * vg) ^ fswz<D>(vrow)) << 4);

    uint64_t base;
    uint32_t s = find_request(a, win, lane, cost, a.n_kv_heads, at, base);
    PagedRequest rq = win.get(s);
    uint32_t units = units_of(rq), kvh = (uint32_t)((at - base) / (units + kPairStart));
    uint32_t x0 = (uint32_t)((at - base) % (units + kPairStart));

    while (true) {
        // [x0, x1) of the pair on the line: its units [u0, u1)
        const uint32_t x1 = (uint32_t)min((uint64_t)units + kPairStart, x0 + (end - at));
        const uint32_t u0 = x0 > kPairStart ? x0 - kPairStart : 0u, u1 = x1 > kPairStart ? x1 - kPairStart : 0u;
        at += x1 - x0;
        if (u0 != u1) {
        const uint32_t rows = rq.rows * G;
        const uint32_t count = u1 - u0 > wave ? (u1 - u0 - wave + kWaves - 1u) / kWaves : 0u;  // of them this wave's
        const int32_t hi_min = rq.pos0;  // (the first token's rows see least)
        s16x8 qf[NR][ND];
        int32_t hi[NR];  // last key the row sees
        f32x4 o[NR][DT], nm[NR];  // O^T; minus the row's reference maximum, four times: the scores start from it
        float l_i[NR];
        uint32_t fresh = (1u << NR) - 1u, sees = 0;  // per row block: no maximum yet; a key seen
        const uint8_t* const q0 = (const uint8_t*)a.q + 2u * ((uint64_t)rq.first * a.q_stride + (uint64_t)kvh * G * a.q_head_stride);
#pragma unroll
        for (int r = 0; r < (int)NR; r++) {
            // row x: token x / G, head of the group x % G
            const uint32_t x = 16u * r + n16 < rows ? 16u * r + n16 : 0u;
            hi[r] = 16u * r + n16 < rows ? rq.pos0 + (int32_t)(x / G) : -1;
            const uint8_t* const qr = q0 + 2u * (x / G * a.q_stride + x % G * a.q_head_stride + D / 4u * g);
#pragma unroll
            for (int ch = 0; ch < ND; ch++) qf[r][ch] = *(const s16x8*)(qr + 16 * ch);
            nm[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            l_i[r] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[r][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // the cache's rows where the halves of this wave's units i0 .. i0 + 31 begin, a half a lane (-1: no
        // page): the vector ALU makes them for 32 units at once, and a unit takes its two into scalars
        int64_t rows0 = -1;
        auto window = [&](uint32_t i0) {
            const uint32_t k0 = (u0 + wave + kWaves * (i0 + (lane >> 1))) * kUnit + 16u * (lane & 1u);
            rows0 = -1;
            if (i0 + (lane >> 1) < count && k0 < rq.keys) {
                const uint32_t p = (uint32_t)a.table[(size_t)s * a.max_pages + (k0 >> a.page_log2)];
                if (p < a.n_pages)
                    rows0 = (int64_t)((((uint64_t)p * a.n_kv_heads + kvh) << a.page_log2) + (k0 & ((1u << a.page_log2) - 1u)));
            }
        };
        // A half's 16 rows are one page's, so all of them are the cache's to read, those of keys past the last
        // one too; for a half of no page, the cache's first rows are read. step() sets such values to 0.
        auto place = [&](Mx4Unit<D>& x, uint32_t i) {
            if ((i & 31u) == 0) window(i);
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                const int l = (int)(2u * (i & 31u) + h);
                const int32_t hi32 = __builtin_amdgcn_readlane((int32_t)(rows0 >> 32), l);
                const uint32_t lo32 = (uint32_t)__builtin_amdgcn_readlane((int32_t)rows0, l);
                x.on[h] = hi32 >= 0;
                x.row[h] = hi32 >= 0 ? (uint64_t)(uint32_t)hi32 << 32 | lo32 : 0ull;
            }
        };
        auto load = [&](Half4<D>& x, const Mx4Unit<D>& at, const void* base, const uint8_t* scales, uint32_t kvo, uint32_t so) {
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                const uint8_t* const p = (const uint8_t*)base + at.row[h] * ROW4;
                if constexpr (D == 128u) {
                    const u32x4 n = __builtin_nontemporal_load((const u32x4*)(p + kvo));
#pragma unroll
                    for (int e = 0; e < 4; e++) x.n[h][e] = n[e];
                } else {
                    const u32x2 n = __builtin_nontemporal_load((const u32x2*)(p + kvo));
#pragma unroll
                    for (int e = 0; e < 2; e++) x.n[h][e] = n[e];
                }
                x.power[h] = *(scales + at.row[h] * SROW + so);
            }
        };
        bool any_far = false;  // (uniform)
        // unit i, in x; each of its registers is asked for again, for unit i + 2, as soon as it is free
        auto step = [&](Mx4Unit<D>& x, uint32_t i) {
            const uint32_t u = u0 + wave + kWaves * i;
            // keys past the last one, on no page, or unseen by a row: masked
            const bool on[2] = {x.on[0], x.on[1]};
            const bool masked = !on[0] || !on[1] || (int32_t)(u * kUnit + kUnit - 1u) > hi_min;
            bool far = false;  // V's blocks may hold infinities or NaN
            if (masked) {
                // a row's weight of a key it does not see is 0, and 0 times an infinity or NaN is NaN: V's rows
                // of keys that there are not are set to 0 here, and what is not finite in others below; the rows
                // that do see it get it after the part's last unit
                const uint32_t last = rq.keys - u * kUnit;  // (of keys; this unit has some, or the part has none at all)
#pragma unroll
                for (uint32_t h = 0; h < 2u; h++) {
                    const bool is = on[h] && 16u * h + vrow < last;
                    far = far || __builtin_amdgcn_ballot_w64(is && x.v.power[h] > kTopPower) != 0;
                    if (!is) {
                        x.v.power[h] = 0;
#pragma unroll
                        for (int e = 0; e < ND; e++) x.v.n[h][e] = 0;
                    }
                }
            }
            // (the addresses are made anew in each unit: hipcc would keep all of them in registers)
            asm volatile("" : "+v"(va), "+v"(vb));
#pragma unroll
            for (uint32_t e = 0; e < (uint32_t)ND; e++) {
                const uint32_t at = vt0 + (vb ^ (e << 4));
#pragma unroll
                for (uint32_t h = 0; h < 2u; h++)
                    *(lds_u32x4*)(uintptr_t)(at + h * 16u * ROW) = values8<T>(x.v.n[h][e], power4(x.v.power[h]));
            }
            if (far) {
                any_far = true;
                uint32_t lo = 0xffffu;  // (opaque: hipcc would keep the masks in registers from the beginning on)
                asm volatile("" : "+s"(lo));
#pragma unroll 1
                for (uint32_t e = 16u * lane; e < TILE; e += 1024u) {
                    lds_u32x4* const at = (lds_u32x4*)(uintptr_t)(vt0 + e);
                    u32x4 w = *at;
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = finite2<T>(w[k], lo);
                    *at = w;
                }
            }
            const bool more = i + 2u < count;
            if (more) {
                place(x, i + 2u);
                load(x.v, x, a.v, m4.v_scales, vo, vso);
            }
            f32x4 sc[NR][2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                const float sk = power4(x.k.power[kb]);
#pragma unroll
                for (int ch = 0; ch < ND; ch++) {
                    const s16x8 k = __builtin_bit_cast(s16x8, values8<T>(x.k.n[kb][ch], sk));
#pragma unroll
                    for (int r = 0; r < (int)NR; r++)
                        sc[r][kb] = mfma16<T>(k, qf[r][ch], ch == 0 ? nm[r] : sc[r][kb]);
                }
            }
            if (more) load(x.k, x, a.k, m4.k_scales, ko, kso);
            s16x8 pf[NR];
#pragma unroll
            for (int r = 0; r < (int)NR; r++) {
                if (masked) {
                    const int32_t k0 = (int32_t)(u * kUnit + 4u * g);
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool a0 = on[0] && k0 + e <= hi[r], a1 = on[1] && k0 + 16 + e <= hi[r];
                        sc[r][0][e] = a0 ? sc[r][0][e] : -INFINITY;
                        sc[r][1][e] = a1 ? sc[r][1][e] : -INFINITY;
                        any = any || a0 || a1;
                    }
                    if (any) sees |= 1u << r;
                } else {
                    sees |= 1u << r;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; e++) mx = fmaxf(fmaxf(mx, sc[r][0][e]), sc[r][1][e]);
                // (the lanes' own maxima say whether some row's reference has to rise; its four lanes are asked
                // only then)
                const bool fr = (fresh >> r) & 1u;
                if (__builtin_amdgcn_ballot_w64(mx > grow_by || (fr && mx > -INFINITY)) != 0) {
                    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                    // (only rows whose own maximum calls for it)
                    const float d = fr ? (mx > -INFINITY ? mx : 0.0f) : (mx > grow_by ? mx : 0.0f);
                    const float alpha = fr ? 0.0f : __builtin_amdgcn_exp2f(-d * c);
                    nm[r] -= d;
                    l_i[r] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[r][dt] *= alpha;
                    sc[r][0] -= d;
                    sc[r][1] -= d;
                    if (mx > -INFINITY) fresh &= ~(1u << r);
                }
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    p[e] = __builtin_amdgcn_exp2f(fmaf(sc[r][e >> 2][e & 3], c, OFF));
                    l_i[r] += p[e];
                }
                pf[r] = __builtin_bit_cast(s16x8, u32x4{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]), pack2<T>(p[4], p[5]),
                                                       pack2<T>(p[6], p[7])});
            }
            asm volatile("" ::: "memory");  // (a wave's LDS accesses run in order: the reads follow its own writes)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const uint32_t at = vt0 + (va ^ (32u * dt));
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)at);
                const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(at + 16u * ROW));
                const s16x8 v = s16x8{lo.x, lo.y, lo.z, lo.w, up.x, up.y, up.z, up.w};
#pragma unroll
                for (int r = 0; r < (int)NR; r++) o[r][dt] = mfma16<T>(v, pf[r], o[r][dt]);
            }
            asm volatile("" ::: "memory");
        };
        if (count != 0) {
            Mx4Unit<D> x, y;
            auto first = [&](Mx4Unit<D>& z, uint32_t i) {
                place(z, i);
                load(z.v, z, a.v, m4.v_scales, vo, vso);
                load(z.k, z, a.k, m4.k_scales, ko, kso);
            };
            first(x, 0);
            if (count > 1u) first(y, 1u);
            for (uint32_t i = 0; i < count; i += 2u) {
                step(x, i);
                if (i + 1u < count) step(y, i + 1u);
            }
        }

        // the four waves' rows: through LDS, 16 of them at a time
        const bool begun = u0 == 0, last = u1 == units;
        float* const part = parts + (size_t)(2u * blockIdx.x + (begun ? 1u : 0u)) * part_floats<D, NR>();
        float* const ml = (float*)(lds + kWaves * TILE);  // [kWaves][2][16]: m, l
        if (begun && !last)  // (the worker's last part: the record is its one)
            rec = JoinRecord{part_of(at + (units - u1) - 1u, w, n), rq.first, 0, rows, kvh, {}};
#pragma unroll
        for (int r = 0; r < (int)NR; r++) {
            if (16u * r >= rows) break;
            float l = l_i[r];
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            // a row's four lanes have seen different keys of a masked unit
            uint32_t sn = (sees >> r) & 1u;
            sn |= (uint32_t)__shfl_xor((int)sn, 16, 64);
            sn |= (uint32_t)__shfl_xor((int)sn, 32, 64);
            f32x4* const ow = (f32x4*)vt;  // [16][D / 4], chunk q of row x at q ^ x
#pragma unroll
            for (int dt = 0; dt < DT; dt++) ow[n16 * (D / 4u) + ((4u * dt + g) ^ n16)] = o[r][dt];
            if (any_far) {  // what masked units hold that is not finite, to the rows that see it
                uint32_t so = vso;  // (opaque, as above)
                float inf = INFINITY;
                asm volatile("" : "+v"(so), "+s"(inf));
                Mx4Unit<D> z;
#pragma unroll 1
                for (uint32_t i = 0; i < count; i++) {
                    place(z, i);
                    const uint32_t k0 = (u0 + wave + kWaves * i) * kUnit;
                    if (z.on[0] && z.on[1] && (int32_t)(k0 + kUnit - 1u) <= hi_min) continue;  // not masked
#pragma unroll
                    for (uint32_t h = 0; h < 2u; h++) {
                        const bool is = z.on[h] && k0 + 16u * h + vrow < rq.keys;
                        uint64_t b = __builtin_amdgcn_ballot_w64(is && m4.v_scales[z.row[h] * SROW + so] > kTopPower);
#pragma unroll 1
                        for (; b != 0; b &= b - 1u) {
                            const uint32_t l = (uint32_t)__builtin_ctzll(b), d0 = D / 4u * (l & 3u);
                            const uint64_t row = z.row[h] + (l >> 2);
                            const float s = power4(m4.v_scales[row * SROW + d0 / 32u]);
                            if ((int32_t)(k0 + 16u * h + (l >> 2)) > hi[r]) continue;
#pragma unroll 1
                            for (uint32_t d = d0 + 4u * g; d < d0 + D / 4u; d += 16u) {
                                const u32x4 w = values8<T>(*(const uint16_t*)((const uint8_t*)a.v + row * ROW4 + d / 2u), s);
                                f32x4 v{lo_f32<T>(w.x), hi_f32<T>(w.x), lo_f32<T>(w.y), hi_f32<T>(w.y)};
#pragma unroll
                                for (int e = 0; e < 4; e++) v[e] = !(fabsf(v[e]) < inf) ? v[e] : 0.0f;
                                ow[n16 * (D / 4u) + (d / 4u ^ n16)] += v;
                            }
                        }
                    }
                }
            }
            if (g == 0) {
                ml[wave * 32u + n16] = (fresh >> r) & 1u ? -INFINITY : -nm[r].x;
                ml[wave * 32u + 16u + n16] = sn ? l : -1.0f;
            }
            __syncthreads();
            const uint32_t here = min(rows - 16u * r, 16u);
            for (uint32_t it = tid; it < here * (D / 4u); it += 64u * kWaves) {
                const uint32_t x = it / (D / 4u), q = it % (D / 4u);
                f32x4 oj{0.0f, 0.0f, 0.0f, 0.0f};
                float mj = -INFINITY, lj = -1.0f;
#pragma unroll
                for (uint32_t v = 0; v < kWaves; v++)
                    join_part(oj, mj, lj, ((const f32x4*)(lds + v * TILE))[x * (D / 4u) + (q ^ x)], ml[v * 32u + x],
                              ml[v * 32u + 16u + x], c);
                const uint32_t row = 16u * r + x;
                if (begun && last) {
                    uint16_t* const dst = (uint16_t*)a.out + (size_t)(rq.first + row / G) * a.out_stride +
                                          (kvh * G + row % G) * D + 4u * q;
                    const f32x4 v = oj * (1.0f / lj);
                    *(u32x2*)dst = lj != -1.0f ? u32x2{pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)} : u32x2{0u, 0u};
                } else {
                    *(f32x4*)(part + row * D + 4u * q) = oj;
                    if (q == 0) {
                        part[16u * NR * D + row] = mj;
                        part[16u * NR * (D + 1u) + row] = lj;
                    }
                }
            }
            __syncthreads();
        }
        }
        if (at >= end) break;
        // the next pair (units are left, so there is a request that has some)
        x0 = 0;
        if (++kvh == a.n_kv_heads) {
            kvh = 0;
            do {
                s++;
                if (s - win.s0 >= 64u) win.load(a, s, lane);
                rq = win.get(s);
                units = units_of(rq);
            } while (units == 0 && s + 1u < a.n_seqs);
        }
    }
    if (tid == 0) records[blockIdx.x] = rec;
}

// Waves a SIMD: what the registers let reside. (At head_dim 64 one more would fit: four contexts of 40000 to
// 131000 keys 50 -> 52 us, with eight tokens each 65 -> 64, 64 ragged ones 30.5 -> 31.5.)
template <uint32_t NR>
constexpr uint32_t few_waves() { return 4u - NR; }

template <uint32_t T, uint32_t D, uint32_t NR>
__global__ void __launch_bounds__(64 * kWaves, few_waves<NR>())
mx4_attn_few(Mx4Args m4, JoinRecord* __restrict__ records, float* __restrict__ parts) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[few_lds_bytes<D, NR>()];
    few_rows<T, D, NR>(m4, lds, records, parts);
}

}  // namespace
}  // namespace mx4attn
}  // namespace llmr
