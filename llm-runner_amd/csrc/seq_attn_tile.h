// seq_attn_tile.h - the matrix-core body of causal attention over packed rows
// (seq_attn.hip): 32 * NW rows of one key/value head per workgroup.
//
// A row is one query head of one token: the G query heads of a key/value head
// lie side by side (row = token * G + head in group), so a workgroup's 256 rows
// are 64 tokens at G = 4 and one tile of keys serves all of a group's heads;
// with heads apart a workgroup would reach over 256 tokens and pass four
// diagonal tiles of keys, half of each hidden, instead of one. Rows are numbered
// through the whole batch: a workgroup that reaches over the end of one request
// into the next takes the keys of both and masks each row to its own request, so
// short prompts share workgroups instead of leaving them part-filled.
//
// S^T = K Q^T (32 keys x 32 rows an MFMA; Q in registers as the B operand), then
// O^T += V^T P^T with P^T straight from the score registers. K and V tiles of 64
// keys come by DMA into LDS rings of four slots each, K sent for four tiles ahead and V
// three; V lies row-major and is read by transposing reads. (As hipcc builds the
// prompts' kernel, it takes those reads for dependent on every DMA in flight and waits
// for all of them, vmcnt(0), before a tile's first one: what was sent for in the same
// tile has the time of its score products to land, and the tile pays the rest. The
// kernel over pages has no such wait in its loop.) The scores start from
// -m_ref (a row's reference maximum), so that p = exp2(c (s - m_ref)) is one
// multiplication and one exp2; m_ref is raised lazily, when the row's maximum exceeds
// it by more than 2^8 in p. Scores, maxima, sums and O are f32; P is rounded to the input
// type for its MFMA (bf16 or fp16, half a step 2^-8 or 2^-11 of each weight).
//
// A wave whose 32 rows see nothing of a tile only moves its share of the DMA and
// waits; masks are applied for the side (a request's beginning, the diagonal) that
// cuts through a tile. What bounds long prompts is the matrix cores at the clock the
// power limit leaves: 16384 tokens, bf16, 32/8 heads of 128 take 1890-2060 us, 1070 to
// 1160 TFLOP/s, where a library product of 8192^3 reaches 1236. Short ones are latency:
// 20 tokens 8 us (launch and the search for the request 3, the first tiles landed 3,
// one tile's exponentials and products, the rows' end), a further tile 1.3, and a block's
// tiles are one after another: 1000 tokens 27-29 us, 2048 62. 24 packed prompts of 13 to
// 414 tokens, fp16, 24/8 heads of 64: 23-24.5 us.
//
// fp16 weights carry a factor 2^7, which the division takes out again: weights
// below 2^-14 of the reference would lose bits, now below 2^-21, and the lazy
// maximum's 2^8 above it is 2^15, within fp16.
#pragma once

#include "llmr_device.h"
#include "llmr_internal.h"

namespace llmr {
namespace seqattn {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;
typedef __attribute__((address_space(3))) uint8_t lds_u8;

template <uint32_t T>
__device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
    if constexpr (T == kGgmlBF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}
template <uint32_t T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (T == kGgmlBF16) return pack_bf16x2(a, b);
    else return pack_f16x2(a, b);
}
// The two halves of a dword as f32.
template <uint32_t T>
__device__ __forceinline__ float lo_f32(uint32_t w) {
    if constexpr (T == kGgmlBF16) return __uint_as_float(w << 16);
    else return (float)__builtin_bit_cast(f16x2, w).x;
}
template <uint32_t T>
__device__ __forceinline__ float hi_f32(uint32_t w) {
    if constexpr (T == kGgmlBF16) return __uint_as_float(w & 0xffff0000u);
    else return (float)__builtin_bit_cast(f16x2, w).y;
}
// A dword's halves with 0 in the place of infinities and NaN.
template <uint32_t T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
    constexpr uint32_t E = T == kGgmlBF16 ? 0x7f80u : 0x7c00u;
    return w & (((w & E) == E ? 0u : 0xffffu) | ((w & (E << 16)) == (E << 16) ? 0u : 0xffff0000u));
}
// Whether either half of a dword is an infinity or NaN.
template <uint32_t T>
__device__ __forceinline__ bool nonfinite2(uint32_t w) {
    constexpr uint32_t E = T == kGgmlBF16 ? 0x7f80u : 0x7c00u;
    return (w & E) == E || (w & (E << 16)) == (E << 16);
}

template <uint32_t T>
__device__ __forceinline__ bool nonfinite4(u32x4 w) {
    return nonfinite2<T>(w.x) || nonfinite2<T>(w.y) || nonfinite2<T>(w.z) || nonfinite2<T>(w.w);
}
template <uint32_t T>
__device__ __forceinline__ u32x4 finite4(u32x4 w) {
    return u32x4{finite2<T>(w.x), finite2<T>(w.y), finite2<T>(w.z), finite2<T>(w.w)};
}

__device__ __forceinline__ float xhalf_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xhalf_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Where a 16-byte chunk of key r lies within its row in an LDS slot: chunk c at
// c ^ swizzle(r). K: a fragment read's 16 lanes (16 keys, one chunk) touch 16
// distinct places of the 256 bytes the banks cover (a row of 256 bytes, or two
// rows of 128). V: a transposing read's 8 keys x 4 chunks lie evenly, two a place.
template <uint32_t D>
__device__ __forceinline__ uint32_t kswz(uint32_t r) {
    return D == 128u ? r & 15u : (r >> 1) & 7u;
}
template <uint32_t D>
__device__ __forceinline__ uint32_t vswz(uint32_t r) {
    return D == 128u ? ((r & 3u) << 2) | ((r >> 2) & 1u) : (((r >> 1) & 1u) << 2) | ((r >> 2) & 1u);
}

constexpr uint32_t kKeys = 64;  // keys of a tile

template <uint32_t D>
constexpr uint32_t tile_bytes() { return kKeys * D * 2u; }
// LDS of a workgroup: four K and four V slots, then three words of its own; the
// epilogue stages 32 rows a wave in the rings.
template <uint32_t D>
constexpr uint32_t lds_bytes() { return 8u * tile_bytes<D>() + 16u; }

// A lane's row. Keys are counted from the first one the workgroup takes; the row sees the
// keys lo .. hi (hi < lo: none); neither falls from row to row of a wave.
struct RowOfLane {
    int lo, hi;
    const uint8_t* q;  // the row's first byte (some row's, for a lane that has none)
    bool live;         // the lane has a row
};

// One workgroup: its rows over n_keys keys, into `out`, or, where part is given, as a part
// to be joined with others: O[32 NW][D] f32, then m, then l (l = -1: the row sees no key of
// the part). Source: where keys come from,
//   uint32_t stage(t, n): tiles [t, its result) of n are made ready; kStages: a barrier and
//     staged() come before the first is asked for;
//   uint32_t page(t): of the wave's keys of tile t (read where lgkmcnt(0) is waited for);
//   rsrc_t tile(base, t, page): the wave's keys of tile t; keys past n_keys, on no page or of
//     no tile that is staged read as zero, or as whatever LDS held;
//   uint32_t voffset(r, chunk): byte offset of a chunk of the tile's key r in it;
//   bool holes(): some staged page is none; uint32_t groups(t): bit i: the keys 16 i .. of
//     tile t have a page;
//   const uint8_t* row(base, j): key j < n_keys's row (null: on no page).
// out_at(): element offset of the lane's row in `out`.
template <uint32_t T, uint32_t D, uint32_t NW, typename Source, typename OutAt>
__device__ __forceinline__ void tile_rows(const SeqAttnArgs& a, uint8_t* lds, Source& src, uint32_t n_keys,
                                          const RowOfLane& row, float* part, const OutAt& out_at) {
    constexpr uint32_t ROW = D * 2u, TILE = tile_bytes<D>();
    constexpr int NF = D / 8;                       // K fragments of a tile, and V fragments
    constexpr int CH = D / 32;                      // 32-dim blocks of a row
    constexpr uint32_t RPI = 1024u / ROW;           // keys a DMA instruction fills (64 lanes x 16 bytes)
    constexpr uint32_t DI = kKeys / RPI / NW;       // DMA instructions per tile and wave
    constexpr uint32_t CPR = ROW / 16u;             // 16-byte chunks of a key row
    constexpr float OFF = T == kGgmlF16 ? 7.0f : 0.0f;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t l32 = lane & 31u, kh = lane >> 5;
    const float c = a.scale_log2, grow_by = 8.0f / c;
    int* const wave_lohi = (int*)(lds + 8u * TILE);         // the workgroup's largest lo, smallest hi
    uint32_t* const any_bad = (uint32_t*)(wave_lohi + 2);  // a masked tile's V has an infinity or NaN

    // Q fragments (B operand): row l32, dims 32 ch + 16 kh + 8 st ..
    s16x8 qf[CH][2];
#pragma unroll
    for (int ch = 0; ch < CH; ch++)
#pragma unroll
        for (int st = 0; st < 2; st++) qf[ch][st] = *(const s16x8*)(row.q + 64u * ch + 32u * kh + 16u * st);

    if (tid == 0) {
        wave_lohi[0] = 0;
        wave_lohi[1] = 0x7ffffffe;
        *any_bad = 0;
    }

    // instruction i of wave w fills the keys RPI (DI w + i) + lane / CPR of a slot,
    // the lane's chunk landing at lane % CPR of its key's row
    uint32_t kvo[DI], vvo[DI];
#pragma unroll
    for (int i = 0; i < (int)DI; i++) {
        const uint32_t r = RPI * (DI * wave + i) + lane / CPR, p = lane % CPR;
        kvo[i] = src.voffset(r, p ^ kswz<D>(r));
        vvo[i] = src.voffset(r, p ^ vswz<D>(r));
    }
    auto dma = [&](const void* base, const uint32_t (&vo)[DI], uint32_t t, uint32_t page, uint32_t slot) {
        const rsrc_t r = src.tile(base, t, page);
        uint8_t* dst = lds + slot * TILE + wave * (DI * 1024u);
#pragma unroll
        for (int i = 0; i < (int)DI; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(dst + 1024u * i), 16, vo[i], 0, 0, 0);
    };

    // K fragment: keys 32 kb + l32, chunk 4 ch + 2 kh + st. V^T fragment (transposing
    // reads): lane (group g, index j) addresses key 4 (g / 2) + j / 4 (+ R), dims
    // 32 dt + 16 (g % 2) + 4 (j % 4) .. + 3.
    uint32_t kfo[CH][2], vto[CH];
    {
        const uint32_t g = lane >> 4, j = lane & 15u, kr = 4u * (g >> 1) + (j >> 2);
        const uint32_t x = 2u * (g & 1u) + ((j & 3u) >> 1), half = j & 1u;
#pragma unroll
        for (int ch = 0; ch < CH; ch++) {
#pragma unroll
            for (int st = 0; st < 2; st++)
                kfo[ch][st] = l32 * ROW + (((4u * ch + 2u * kh + st) ^ kswz<D>(l32)) << 4);
            vto[ch] = kr * ROW + (((4u * ch + x) ^ vswz<D>(kr)) << 4) + 8u * half;
        }
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds;
    // fragment addresses in registers of their own: every read of a tile is then one of
    // them plus an immediate
    auto kaddr = [&](uint32_t slot, uint32_t (&ka)[CH][2]) {
#pragma unroll
        for (int ch = 0; ch < CH; ch++)
#pragma unroll
            for (int st = 0; st < 2; st++) {
                ka[ch][st] = lds0 + slot * TILE + kfo[ch][st];
                asm("" : "+v"(ka[ch][st]));
            }
    };
    auto vaddr = [&](uint32_t slot, uint32_t (&va)[CH]) {
#pragma unroll
        for (int dt = 0; dt < CH; dt++) {
            va[dt] = lds0 + (4u + slot) * TILE + vto[dt];
            asm("" : "+v"(va[dt]));
        }
    };
    auto kfrag = [&](const uint32_t (&ka)[CH][2], int f) -> s16x8 {
        const int k = f % (NF / 2);
        return *(const lds_s16x8*)(uintptr_t)(ka[k / 2][k % 2] + 32u * (uint32_t)(f / (NF / 2)) * ROW);
    };
    auto vfrag = [&](const uint32_t (&va)[CH], int f) -> s16x8 {
        const uint32_t R = 32u * (uint32_t)(f / (NF / 2)) + 16u * (uint32_t)((f % (NF / 2)) / CH);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(va[f % CH] + R * ROW));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(va[f % CH] + (R + 8u) * ROW));
        return s16x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    };

    f32x16 o[CH];
#pragma unroll
    for (int dt = 0; dt < CH; dt++) o[dt] = f32x16{};
    float m_ref = 0.0f, l_i = 0.0f;
    uint64_t seen = 0;  // lanes whose m_ref is a maximum of theirs

    const uint32_t n_tiles = (n_keys + kKeys - 1u) / kKeys;
    // over the wave's rows that see a key: tiles [see0, see1) are seen by some, tiles [full0,
    // full1) whole by every. lo and hi do not fall from row to row, so the first and the last of
    // them say it.
    uint32_t see0 = ~0u, see1 = 0, full0 = 0, full1 = ~0u;
    int lo_max = 0, hi_min = 0x7ffffffe;
    const uint64_t some = __builtin_amdgcn_ballot_w64(row.live && row.hi >= row.lo);
    if (some != 0) {
        const uint32_t a0 = (uint32_t)__builtin_ctzll(some), a1 = 63u - (uint32_t)__builtin_clzll(some);
        see0 = (uint32_t)__builtin_amdgcn_readlane(row.lo, (int)(a0 & 31u)) / kKeys;
        see1 = (uint32_t)__builtin_amdgcn_readlane(row.hi, (int)a1) / kKeys + 1u;
        lo_max = __builtin_amdgcn_readlane(row.lo, (int)a1);
        hi_min = __builtin_amdgcn_readlane(row.hi, (int)(a0 & 31u));
        full0 = ((uint32_t)lo_max + kKeys - 1u) / kKeys;
        full1 = ((uint32_t)hi_min + 1u) / kKeys;
    }
    bool sees = false;  // a key

    // scores of the keys a row does not see to -inf: a compare with a constant and a select
    // a score, for each side that the tile needs
    auto mask = [&](f32x16& h0, f32x16& h1, uint32_t t) {
        int k0 = (int)(t * kKeys + 4u * kh);
        // (without it the 64 compares of the first tile seen, the same all the time, are made ahead
        // of everything, into scalars that spill)
        asm volatile("" : "+v"(k0));
        const bool holes = src.holes();
        if (t >= full1 || holes) {
            const int d = row.hi - k0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                h0[i] = 8 * (i >> 2) + (i & 3) <= d ? h0[i] : -INFINITY;
                h1[i] = 8 * (i >> 2) + (i & 3) + 32 <= d ? h1[i] : -INFINITY;
            }
        }
        if (t < full0 || holes) {
            const int d = row.lo - k0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                h0[i] = 8 * (i >> 2) + (i & 3) >= d ? h0[i] : -INFINITY;
                h1[i] = 8 * (i >> 2) + (i & 3) + 32 >= d ? h1[i] : -INFINITY;
            }
        }
        if (holes) {
            const uint32_t on = src.groups(t);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int k = k0 + 8 * (i >> 2) + (i & 3);
                const bool p0 = (on >> (i >> 3)) & 1u, p1 = (on >> (2 + (i >> 3))) & 1u;
                h0[i] = p0 ? h0[i] : -INFINITY;
                h1[i] = p1 ? h1[i] : -INFINITY;
                sees = sees || (p0 && k >= row.lo && k <= row.hi) || (p1 && k + 32 >= row.lo && k + 32 <= row.hi);
            }
        }
    };
    auto masked = [&](uint32_t t) { return t < full0 || t >= full1 || src.holes(); };
    auto rescale = [&](uint64_t grow, float mx, f32x16& n0, f32x16& n1) {
        if (grow != 0) {
            const bool fresh = ((seen >> lane) & 1u) == 0;
            // only rows whose own maximum calls for it: what another row of the wave sees changes no
            // bit of this one (0 leaves everything as it is)
            const float d = fresh ? (mx > -INFINITY ? mx : 0.0f) : (mx > grow_by ? mx : 0.0f);
            const float alpha = fresh ? 0.0f : __builtin_amdgcn_exp2f(-d * c);
            m_ref += d;
            l_i *= alpha;
#pragma unroll
            for (int dt = 0; dt < CH; dt++) o[dt] *= alpha;
            n0 -= d;
            n1 -= d;
        }
    };
    // P of score pair `item` (keys 2 (item % 8), + 1 of half h) into dword item of p
    auto exp_pair = [&](const f32x16& h, int item, uint32_t (&p)[16], float& rs) {
        const int i = 2 * (item % 8);
        const float e0 = __builtin_amdgcn_exp2f(fmaf(h[i], c, OFF));
        const float e1 = __builtin_amdgcn_exp2f(fmaf(h[i + 1], c, OFF));
        p[item] = pack2<T>(e0, e1);
        rs += e0 + e1;
    };
    auto pfrag = [&](const uint32_t (&p)[16], int kb, int cc) -> s16x8 {
        const int b = 8 * kb + 4 * cc;
        return __builtin_bit_cast(s16x8, u32x4{p[b], p[b + 1], p[b + 2], p[b + 3]});
    };

    // Infinities and NaN in V rows that some row of the workgroup does not see: its
    // weight there is 0, and 0 times them is NaN. Where a tile is masked they are set to 0
    // in LDS a tile before anyone reads it; the rows that do see them, with a weight above 0,
    // get them from memory after the last tile.
    uint32_t wg_full0 = 0, wg_full1 = 0;
    auto wg_masked = [&](uint32_t t) { return t < wg_full0 || t >= wg_full1 || src.holes(); };
    auto clean_v = [&](uint32_t t) {
        uint8_t* const vt = lds + (4u + (t & 3u)) * TILE;
#pragma unroll
        for (uint32_t b = 0; b < TILE / (NW * 1024u); b++) {
            u32x4* const at = (u32x4*)(vt + (b * NW + wave) * 1024u + lane * 16u);
            const u32x4 w = *at;
            const bool n = nonfinite4<T>(w);
            if (__builtin_amdgcn_ballot_w64(n) != 0) {
                if (n) {
                    // (past the last key: whatever LDS held)
                    if (t * kKeys + (b * NW + wave) * RPI + lane / CPR < n_keys) *any_bad = 1u;
                    *at = finite4<T>(w);
                }
            }
        }
    };
    auto add_bad = [&](uint32_t t) {
        const uint32_t j = t * kKeys + lane;
        bool n = false;
        if (j < n_keys) {
            const uint8_t* const vr = src.row(a.v, j);
            for (uint32_t b = 0; vr && b < CPR; b++) {
                const u32x4 w = *(const u32x4*)(vr + 16u * b);
                n = n || nonfinite4<T>(w);
            }
        }
        for (uint64_t bad = __builtin_amdgcn_ballot_w64(n); bad != 0; bad &= bad - 1u) {
            const uint32_t key = t * kKeys + (uint32_t)__builtin_ctzll(bad);  // < n_keys: a lane found it there
            const bool in = (int)key >= row.lo && (int)key <= row.hi;
            const uint8_t* const vr = src.row(a.v, key);
#pragma unroll
            for (int dt = 0; dt < CH; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const u32x2 v = *(const u32x2*)(vr + 64u * dt + 16u * g + 8u * kh);
                    const float x[4] = {lo_f32<T>(v.x), hi_f32<T>(v.x), lo_f32<T>(v.y), hi_f32<T>(v.y)};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[dt][4 * g + e] += (int)in & (int)!(fabsf(x[e]) < INFINITY) ? x[e] : 0.0f;
                }
        }
    };

    constexpr int PF = 3;  // fragments in flight ahead of their MFMAs
    uint32_t ka[CH][2];    // K(t+1)'s fragment addresses
    s16x8 kf[PF + 1];      // its fragments in flight: the first PF are read before the tile starts
    f32x16 h0, h1, h2;
    uint32_t p3 = 0, p4 = 0, p5 = 0;  // pages of the wave's keys of tiles t + 3, t + 4 and t + 5
    uint32_t seg = 0;                 // tiles below it are ready

    // S(t) by itself, into (n0, n1), and its maximum
    auto scores = [&](f32x16& n0, f32x16& n1, uint32_t t) {
        uint32_t kt[CH][2];
        kaddr(t & 3u, kt);
        static_for<0, NF>([&](auto F) {
            constexpr int f = F, kb = f / (NF / 2), k = f % (NF / 2);
            f32x16& s = kb == 0 ? n0 : n1;
            s = mfma32<T>(kfrag(kt, f), qf[k / 2][k % 2], k == 0 ? f32x16{} - m_ref : s);
        });
        if (masked(t)) mask(n0, n1, t);
        float mx = n0[0];
#pragma unroll
        for (int i = 0; i < 16; i++) mx = fmaxf(fmaxf(mx, n0[i]), n1[i]);
        mx = xhalf_max(mx);
        const uint64_t any = __builtin_amdgcn_ballot_w64(mx > -INFINITY);
        rescale(__builtin_amdgcn_ballot_w64(mx > grow_by) | (any & ~seen), mx, n0, n1);
        seen |= any;
    };
    // the first fragments of K(t), which the tile before it expects
    auto first_frags = [&](uint32_t t) {
        kaddr(t & 3u, ka);
        static_for<0, PF>([&](auto F) { kf[F] = kfrag(ka, F); });
    };
    // O += P(t) V(t) by itself, S(t) in (c0, c1)
    auto accumulate = [&](const f32x16& c0, const f32x16& c1, uint32_t t) {
        uint32_t va[CH], p[16];
        float rs = 0.0f;
        static_for<0, 8>([&](auto I) { exp_pair(c0, I, p, rs); });
        static_for<8, 16>([&](auto I) { exp_pair(c1, I, p, rs); });
        l_i += rs;
        vaddr(t & 3u, va);
        static_for<0, NF>([&](auto F) {
            constexpr int f = F, kb = f / (NF / 2), cc = (f % (NF / 2)) / CH, dt = f % CH;
            o[dt] = mfma32<T>(vfrag(va, f), pfrag(p, kb, cc), o[dt]);
        });
    };
    // What every wave does in tile t, whatever it sees of it: K(t+4) to K slot t % 4, V(t+3) to
    // V slot (t+3) % 4 (both last read in tile t - 1), V(t+1) looked through where it is masked.
    auto send = [&](uint32_t t) {
        dma(a.k, kvo, t + 4u, p4, t & 3u);
        dma(a.v, vvo, t + 3u, p3, 4u + ((t + 3u) & 3u));
        p5 = src.page(t + 5u);
        if (t + 1u < seg && wg_masked(t + 1u)) clean_v(t + 1u);
    };
    auto sent = [&]() {
        LLMR_STAGE_BARRIER(2 * DI);
        p3 = p4;
        p4 = (uint32_t)__builtin_amdgcn_readfirstlane(p5);
    };

    // One tile t: S(t) in (c0, c1), S(t+1) = K(t+1) Q^T to (n0, c0). The MFMAs are issued in a
    // fixed order with the vector work spread between them: the exponentials of S(t)'s first
    // half before c0 is written again, those of the second half by the time its accumulation
    // starts, the maximum of S(t+1) under the first accumulations, the first fragment reads of
    // K(t+2) under the last ones.
    auto tile = [&](f32x16& c0, f32x16& c1, f32x16& n0, uint32_t t) {
        send(t);
        const bool mask_next = masked(t + 1u);
        uint32_t va[CH], p[16];
        vaddr(t & 3u, va);
        s16x8 vf[PF + 1];
        float rs = 0.0f, mt = -INFINITY, mx = 0.0f;
        uint64_t grow = 0, any = 0;
        static_for<0, 2 * NF>([&](auto J) {
            constexpr int j = J;
            if constexpr (j < NF) {
                constexpr int f = j, kb = f / (NF / 2), k = f % (NF / 2);
                if constexpr (f + PF < NF) kf[(f + PF) % (PF + 1)] = kfrag(ka, f + PF);
                f32x16& s = kb == 0 ? n0 : c0;
                s = mfma32<T>(kf[f % (PF + 1)], qf[k / 2][k % 2], k == 0 ? f32x16{} - m_ref : s);
            } else {
                constexpr int f = j - NF, kb = f / (NF / 2), cc = (f % (NF / 2)) / CH, dt = f % CH;
                if constexpr (f + PF < NF) vf[(f + PF) % (PF + 1)] = vfrag(va, f + PF);
                o[dt] = mfma32<T>(vf[f % (PF + 1)], pfrag(p, kb, cc), o[dt]);
            }
            if constexpr (j >= NF - PF && j < NF) vf[j - (NF - PF)] = vfrag(va, j - (NF - PF));
            // first half: 8 pairs over NF / 2 steps; second half: 8 over the next NF
            if constexpr (j < NF / 2)
                static_for<0, 16 / NF>([&](auto E) { exp_pair(c0, j * (16 / NF) + E, p, rs); });
            if constexpr (j >= NF / 2 && j < NF + NF / 2 && (NF == 8 || j % 2 == 0))
                exp_pair(c1, 8 + (j - NF / 2) / (NF / 8), p, rs);
            if constexpr (j == NF - 1) {
                if (mask_next) mask(n0, c0, t + 1u);
            }
            if constexpr (j >= NF && j < NF + NF / 2)
                static_for<0, 16 / NF>([&](auto E) {  // 4 scores of 32 at a time
                    constexpr int k = (j - NF) * (16 / NF) + E, i = 4 * (k % 4);
                    const f32x16& s = k < 4 ? n0 : c0;
                    mt = fmaxf(fmaxf(mt, s[i]), s[i + 1]);
                    mt = fmaxf(fmaxf(mt, s[i + 2]), s[i + 3]);
                });
            if constexpr (j == NF + NF / 2) mx = xhalf_max(mt);
            if constexpr (j == NF + NF / 2 + 1) {
                any = __builtin_amdgcn_ballot_w64(mx > -INFINITY);
                grow = __builtin_amdgcn_ballot_w64(mx > grow_by) | (any & ~seen);
            }
            if constexpr (j == NF + NF / 2 + 2) kaddr((t + 2u) & 3u, ka);
            // K(t+2): this tile's successor starts with it
            if constexpr (NF == 16 && j >= NF + NF / 2 + 3 && j < NF + NF / 2 + 3 + PF)
                kf[j - (NF + NF / 2 + 3)] = kfrag(ka, j - (NF + NF / 2 + 3));
            if constexpr (NF == 8 && j == 2 * NF - 1) static_for<0, PF>([&](auto F) { kf[F] = kfrag(ka, F); });
            __builtin_amdgcn_sched_barrier(0);
        });
        l_i += rs;
        rescale(grow, mx, n0, c0);
        seen |= any;
        sent();
    };

    uint32_t t = 0;
    for (bool first = true; first || (Source::kStages && t < n_tiles); first = false) {
        if (Source::kStages && n_tiles == 0) break;
        // (the rings' slots go on by t: a source stages a multiple of four tiles, or the rest)
        seg = src.stage(t, n_tiles);
        if constexpr (Source::kStages) {
            __syncthreads();
            src.staged();
        }
        if (!src.holes()) sees = sees || (row.hi >= row.lo && row.hi >= (int)(t * kKeys));
        {
            uint32_t pg[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) pg[i] = (uint32_t)__builtin_amdgcn_readfirstlane(src.page(t + i));
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {  // K(t) V(t) K(t+1) V(t+1) K(t+2) V(t+2) K(t+3) in flight
                dma(a.k, kvo, t + i, pg[i], i);
                if (i < 3u) dma(a.v, vvo, t + i, pg[i], 4u + i);
            }
            p3 = pg[3];
            p4 = (uint32_t)__builtin_amdgcn_readfirstlane(src.page(t + 4u));
        }
        // the wave's tiles of this segment: [see0, end)
        const uint32_t end = min(see1, seg);
        LLMR_STAGE_BARRIER(6 * DI);  // K(t) has landed
        if (first && lane == 0) {
            atomicMax(&wave_lohi[0], lo_max);
            atomicMin(&wave_lohi[1], hi_min);
        }
        if (see0 <= t && t < end) scores(h0, h1, t);
        LLMR_STAGE_BARRIER(2 * DI);  // K(t+1), V(t), K(t+2), V(t+1) have landed
        if (first) {
            wg_full0 = (uint32_t)(__builtin_amdgcn_readfirstlane(wave_lohi[0]) + (int)kKeys - 1) / kKeys;
            wg_full1 = (uint32_t)(__builtin_amdgcn_readfirstlane(wave_lohi[1]) + 1) / kKeys;
        }
        if (wg_masked(t)) {
            clean_v(t);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0), the DMAs go on
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        // Before the wave's first tile it sees nothing, then come its scores; S(t+1) is computed
        // beside P(t) V(t), the score halves rotating with period 3 (S(t) in (h0, h1), (h2, h0),
        // (h1, h2)); then its last P V, and nothing again.
        while (t < seg) {
            if (t >= see0 && t + 1u < end) {
                first_frags(t + 1u);
                while (t + 4u <= end) {
                    tile(h0, h1, h2, t);
                    tile(h2, h0, h1, t + 1u);
                    tile(h1, h2, h0, t + 2u);
                    t += 3u;
                }
                while (t + 1u < end) {
                    tile(h0, h1, h2, t);
                    h1 = h0;
                    h0 = h2;
                    t++;
                }
            }
            send(t);
            if (t >= see0 && t + 1u == end) accumulate(h0, h1, t);
            if (t + 1u == see0 && see0 < end) scores(h0, h1, see0);
            sent();
            t++;
        }
        LLMR_WAIT_VMCNT(0);  // no DMA may still be writing LDS when something else goes there
        __syncthreads();
    }
    if (n_tiles != 0 && __builtin_amdgcn_readfirstlane(*any_bad) != 0)
        for (t = 0; t < n_tiles; t++)
            if (wg_masked(t)) add_bad(t);

    const float l_sum = xhalf_sum(l_i);
    // the row's other lane has seen the keys between its own (asked by every lane: behind a `||` the
    // lanes that have seen some would not take part, and the others would read nothing from them)
    const int other = __shfl_xor((int)sees, 32, 64);
    sees = sees || other != 0;
    if (part != nullptr) {
        float* const po = part + (size_t)(wave * 32u + l32) * D;
        if (row.live) {
#pragma unroll
            for (int dt = 0; dt < CH; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *(f32x4*)(po + 32 * dt + 8 * g + 4u * kh) =
                        f32x4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
            if (kh == 0) {
                float* const pm = part + 32u * NW * D + wave * 32u + l32;
                pm[0] = (seen >> lane) & 1u ? m_ref : -INFINITY;
                pm[32u * NW] = sees ? l_sum : -1.0f;
            }
        }
        return;
    }

    // O = O^T / l through LDS, so that a store writes whole rows: lane l32 holds the dims
    // 32 dt + 8 g + 4 kh .. + 3 of its row; row r's chunk q lies at q ^ (r % CPR)
    uint8_t* const ot = lds + wave * (32u * ROW);
    const float inv_l = 1.0f / l_sum;
#pragma unroll
    for (int dt = 0; dt < CH; dt++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const u32x2 w{pack2<T>(o[dt][4 * g] * inv_l, o[dt][4 * g + 1] * inv_l),
                          pack2<T>(o[dt][4 * g + 2] * inv_l, o[dt][4 * g + 3] * inv_l)};
            *(u32x2*)(ot + l32 * ROW + (((4u * dt + g) ^ (l32 % CPR)) << 4) + 8u * kh) = sees ? w : u32x2{0u, 0u};
        }
    const uint64_t my_out = out_at();
    // the wave reads back only what it wrote: its LDS operations run in order
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (uint32_t i = 0; i < 32u / RPI; i++) {
        const uint32_t r = RPI * i + lane / CPR, q = lane % CPR;
        const u32x4 v = *(const u32x4*)(ot + r * ROW + ((q ^ (r % CPR)) << 4));
        const uint64_t at = ((uint64_t)(uint32_t)__shfl((int)(my_out >> 32), (int)r, 64) << 32) |
                            (uint32_t)__shfl((int)(uint32_t)my_out, (int)r, 64);
        if (__shfl((int)row.live, (int)r, 64)) *(u32x4*)((uint16_t*)a.out + at + 8u * q) = v;
    }
}

}  // namespace seqattn
}  // namespace llmr
