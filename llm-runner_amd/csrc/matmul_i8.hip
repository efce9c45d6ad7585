// matmul_i8.hip - the product of 8-bit rows and 8-bit weights (llmr_matmul_i8):
//
//   out[m, n] = x_scales[m] w_scales[n] sum_k x[m, k] w[n, k]
//
// The sum is exact in int32, in any order and any split of K, so every kernel gives
// the same bits.
//
//  - matmul_i8_few, few tokens, or few outputs with long rows: a stream of the weights.
//    A workgroup has 16 or 32 channels and up to 64 tokens; its eight waves share K and
//    add up in LDS.
//  - matmul_i8_small: tiles of 64 or 128 tokens x 128 channels, one a workgroup.
//  - matmul_i8_tiles: persistent tiles of 64 to 256 tokens x 256 channels, 128 bytes of
//    K a stage, both operands by DMA into LDS rings.
// The MFMAs take the weights as A and the tokens as B, so that a lane's results are
// consecutive channels of one token.
#include "gemm_q_common.h"
#include "llmr_device.h"
#include "llmr_internal.h"

// every rounding that the definition names is one
#pragma clang fp contract(off)

namespace llmr {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// A sum to the product, rounded to f32 after each factor. (The empty asm keeps the last product apart
// from a conversion to f16 behind it: hipcc makes one v_fma_mixlo_f16 of the two, contraction or not,
// which rounds once where the definition rounds twice.)
__device__ __forceinline__ float scaled(int acc, float xs, float ws) {
    float y = (float)acc * xs * ws;
    asm("" : "+v"(y));
    return y;
}
template <uint32_t OT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return OT == kGgmlF16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
}
template <uint32_t OT>
constexpr uint32_t out_size() { return OT == kGgmlF32 ? 4u : 2u; }

// 16 bytes and 8 of output rows, which are aligned to their elements only (any stride): global stores
// take any alignment.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_s4 __attribute__((ext_vector_type(4), aligned(4)));

// Four consecutive channels c .. of one token (those below N), from their sums.
template <uint32_t OT>
__device__ __forceinline__ void store4(const MatmulI8Args& a, uint32_t m, uint32_t c, i32x4 acc, float xs, const float (&ws)[4]) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = scaled(acc[i], xs, ws[i]);
    uint8_t* const dst = (uint8_t*)a.out + ((uint64_t)m * a.out_stride + c) * out_size<OT>();
    if (c + 4u <= a.N) {
        if constexpr (OT == kGgmlF32)
            *(u32x4_s4*)dst = u32x4_s4{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])};
        else *(u32x2_a2*)dst = u32x2_a2{pack2<OT>(y[0], y[1]), pack2<OT>(y[2], y[3])};
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++)
        if (c + i < a.N) {
            if constexpr (OT == kGgmlF32) ((float*)dst)[i] = y[i];
            else ((uint16_t*)dst)[i] = (uint16_t)pack2<OT>(y[i], 0.0f);
        }
}

// ---- few tokens ----------------------------------------------------------------------
//
// A workgroup has 16 CT channels of 16 MT tokens; its waves share K. A wave's step is 128 bytes of K, step s of a
// workgroup its wave s % 8's, as two halves of 64 bytes for a 16x16x64 MFMA each; U steps' rows are on their way while
// one is worked on. A load has lanes 4 r .. 4 r + 3 at four pieces of 16 bytes of row r: four lanes side by side that
// are on four rows, as the MFMA has them, take about four times as long (64 x 4096 x 4096 12.4 us, 1 x 4096 x 6144 8.7;
// this way 9.4 and 7.4, of which the pieces' way to the MFMA's lanes, over LDS, is 1.4 and 0.4). Which k a piece is does
// not matter as long as both operands agree.
// Measured, weights from HBM, us: 1 x 4096 x 6144 7.4 (3.4 TB/s), 1 x 4096 x 20480 18.1 (4.6), 64 x 4096 x 4096 9.4,
// 64 x 14336 x 4096 25.5: the CU's loads of the tokens' rows (64 for 16 channels), at one token the start and the end.
constexpr uint32_t kFewWaves = 8;

template <uint32_t OT, uint32_t MT, uint32_t CT>
__global__ void __launch_bounds__(64 * kFewWaves) matmul_i8_few(MatmulI8Args a) {
    constexpr uint32_t U = MT == 1u ? 6u / CT : MT == 2u ? 4u : 3u;
    // each wave's halves of CT + MT row blocks: piece p of row r in column p ^ (r / 4) % 4
    __shared__ u32x4 turn[kFewWaves][CT + MT][64];
    __shared__ i32x4 red[kFewWaves][CT * MT][64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, row = lane >> 2, piece = lane & 3u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n0 = blockIdx.x * 16u * CT, m0 = blockIdx.y * 16u * MT;
    // rows past the last one, and pieces past K, read as zero: past the descriptors' ends
    const uint32_t wrows = min(a.N - n0, 16u * CT), xrows = min(a.M - m0, 16u * MT);
    const rsrc_t wr = make_rsrc(a.w + (uint64_t)n0 * a.w_stride, (uint64_t)(wrows - 1u) * a.w_stride + a.K);
    const rsrc_t xr = make_rsrc(a.x + (uint64_t)m0 * a.x_stride, (uint64_t)(xrows - 1u) * a.x_stride + a.K);
    const uint32_t steps = (a.K + 127u) / 128u;
    uint32_t wo[CT], xo[MT];
#pragma unroll
    for (uint32_t c = 0; c < CT; c++) wo[c] = 16u * c + row < wrows ? (16u * c + row) * a.w_stride + 16u * piece : ~0u;
#pragma unroll
    for (uint32_t t = 0; t < MT; t++) xo[t] = 16u * t + row < xrows ? (16u * t + row) * a.x_stride + 16u * piece : ~0u;
    i32x4 acc[CT][MT];
#pragma unroll
    for (uint32_t c = 0; c < CT; c++)
#pragma unroll
        for (uint32_t t = 0; t < MT; t++) acc[c][t] = i32x4{0, 0, 0, 0};
    u32x4 wf[U][CT][2], xf[U][MT][2];
    auto send = [&](auto B, uint32_t s) {  // step s into buffer B; a row's halves one after the other: one line
        constexpr int u = decltype(B)::value;
        const uint32_t k = s * 128u;  // (past K for every lane: nothing is read)
        const bool in[2] = {k + 16u * piece < a.K, k + 16u * piece + 64u < a.K};
#pragma unroll
        for (uint32_t c = 0; c < CT; c++)
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) wf[u][c][h] = bload16(wr, in[h] && wo[c] != ~0u ? wo[c] + k + 64u * h : ~0u, 0u);
#pragma unroll
        for (uint32_t t = 0; t < MT; t++)
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) xf[u][t][h] = bload16(xr, in[h] && xo[t] != ~0u ? xo[t] + k + 64u * h : ~0u, 0u);
    };
    // (an MFMA's lane has row lane % 16, piece lane / 16)
    const uint32_t to = 4u * row + (piece ^ (row >> 2)), from = 4u * (lane & 15u) + ((lane >> 4) ^ (lane >> 2 & 3u));
    static_for<0, (int)U>([&](auto B) { send(B, wave + (uint32_t)decltype(B)::value * kFewWaves); });
    for (uint32_t s0 = wave; s0 < steps; s0 += U * kFewWaves) {
        static_for<0, (int)U>([&](auto B) {
            constexpr int u = decltype(B)::value;
            const uint32_t s = s0 + (uint32_t)u * kFewWaves;
            if (s < steps) {
#pragma unroll
                for (uint32_t h = 0; h < 2u; h++) {
                    i32x4 w[CT], x[MT];
#pragma unroll
                    for (uint32_t c = 0; c < CT; c++) turn[wave][c][to] = wf[u][c][h];
#pragma unroll
                    for (uint32_t t = 0; t < MT; t++) turn[wave][CT + t][to] = xf[u][t][h];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (a wave's LDS accesses run in order)
#pragma unroll
                    for (uint32_t c = 0; c < CT; c++) w[c] = __builtin_bit_cast(i32x4, turn[wave][c][from]);
#pragma unroll
                    for (uint32_t t = 0; t < MT; t++) x[t] = __builtin_bit_cast(i32x4, turn[wave][CT + t][from]);
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                    for (uint32_t t = 0; t < MT; t++)
#pragma unroll
                        for (uint32_t c = 0; c < CT; c++) acc[c][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[c], x[t], acc[c][t], 0, 0, 0);
                }
                if (s + U * kFewWaves < steps) send(B, s + U * kFewWaves);
            }
        });
    }
#pragma unroll
    for (uint32_t c = 0; c < CT; c++)
#pragma unroll
        for (uint32_t t = 0; t < MT; t++) red[wave][c * MT + t][lane] = acc[c][t];
    __syncthreads();
    for (uint32_t i = tid; i < CT * MT * 64u; i += 64u * kFewWaves) {
        const uint32_t f = i >> 6, l = i & 63u, m = m0 + 16u * (f % MT) + (l & 15u), c = n0 + 16u * (f / MT) + 4u * (l >> 4);
        i32x4 s = red[0][f][l];
#pragma unroll
        for (uint32_t v = 1; v < kFewWaves; v++) s += red[v][f][l];
        if (m < a.M && c < a.N) {
            float ws[4];
#pragma unroll
            for (uint32_t e = 0; e < 4u; e++) ws[e] = a.w_scales[min(c + e, a.N - 1u)];
            store4<OT>(a, m, c, s, a.x_scales[m], ws);
        }
    }
}

// ---- tiles ---------------------------------------------------------------------------
//
// The structure of the two-pass 16-bit GEMM's second pass (gemm_w16_persist: five LDS slots, the
// tokens sent for two stages ahead and the weights one, fragments a 16-byte chunk of a row, a stage
// in four steps with the next step's fragments read beside its MFMAs), on bytes: a stage is 128 of K
// instead of 64, the same bytes and matrix-core cycles for twice the products. Four waves in 2 x 2, each 32 MB tokens
// x 128 channels as 32x32x32 MFMAs; MB: 1 to 4, a tile of 64 MB tokens x 256 channels.
constexpr uint32_t kRow = 128;             // bytes of K a stage
constexpr uint32_t kWSlot = 256u * kRow;   // LDS bytes of a stage's weights

template <uint32_t MB>
struct FragsI8 {
    i32x4 x[MB], w[4];
};

// 64 lanes' 16 bytes to dst .. + 1023. (A function of its own: in a kernel's body, where dst depends on a
// template argument, hipcc's host pass drops the kernel for this cast, without an error.)
__device__ __forceinline__ void dma16(rsrc_t r, uint8_t* dst, uint32_t voffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 16, voffset, 0, 0, 0);
}

#define LLMR8_STEP_SCHEDULE                                                                    \
    LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1); LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1);           \
    LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1); LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1);           \
    LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1); LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1);           \
    LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1); LLMR_SGB(0x008, 1); LLMR_SGB(0x100, 1);           \
    LLMR_SGB(0x008, 1); LLMR_SGB(0x020, 1); LLMR_SGB(0x008, 1); LLMR_SGB(0x020, 1);           \
    LLMR_SGB(0x008, 1); LLMR_SGB(0x020, 1); LLMR_SGB(0x008, 1); LLMR_SGB(0x020, 1);           \
    LLMR_SGB(0x008, 4)

template <uint32_t OT, uint32_t MB>
__global__ void __launch_bounds__(256, 1) matmul_i8_tiles(MatmulI8Args a, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr uint32_t BM = 64u * MB, XSLOT = BM * kRow;
    constexpr int XD = 2 * MB, WD = 8;  // 1 KiB DMAs (8 rows) a wave and stage: of the tokens, of the weights
    __shared__ __attribute__((aligned(16))) uint8_t X0[XSLOT];
    __shared__ __attribute__((aligned(16))) uint8_t X1[XSLOT];
    __shared__ __attribute__((aligned(16))) uint8_t X2[XSLOT];
    __shared__ __attribute__((aligned(16))) uint8_t W0[kWSlot];
    __shared__ __attribute__((aligned(16))) uint8_t W1[kWSlot];

    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t l32 = lane & 31u, kh = lane >> 5;
    const uint32_t wm = wave & 1u, wn = wave >> 1;
    const uint32_t G = gridDim.x, total = tiles_m * tiles_n;
    const uint32_t n_tiles = w16_n_tiles(blockIdx.x, G, total);
    if (n_tiles == 0) return;
    const uint32_t S = (a.K + kRow - 1u) / kRow, SP = (S + 5u) / 6u * 6u;

    // DMA i of wave w: rows 16 MB w + 8 i + lane / 8 (tokens), 64 w + 8 i + lane / 8 (weights), physical
    // chunk lane % 8, logical chunk (lane % 8) ^ lds_swz(row); 16 MB w is a multiple of 16, so that swz is (lane / 8) ^ (i & 1)
    uint32_t xvoff[XD], wvoff[WD];
    const uint32_t c0 = (lane & 7u) ^ (lane >> 3);  // of even i; odd i: ^ 1
#pragma unroll
    for (int i = 0; i < XD; i++) xvoff[i] = (16u * MB * wave + 8u * i + (lane >> 3)) * a.x_stride + ((c0 ^ (i & 1)) << 4);
#pragma unroll
    for (int i = 0; i < WD; i++) wvoff[i] = (64u * wave + 8u * i + (lane >> 3)) * a.w_stride + ((c0 ^ (i & 1)) << 4);
    uint32_t xoff[4], woff[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint32_t ch = 4u * (t >> 1) + 2u * kh + (t & 1);
        xoff[t] = lds_off(wm * 32u * MB + l32, ch);
        woff[t] = lds_off(wn * 128u + l32, ch);
    }

    struct Cursor {
        uint32_t s;           // stage within the tile
        const int8_t* base;   // the tile's first row
        uint32_t size;        // bytes of its rows (0 past the last tile)
    };
    auto tile_origin = [&](uint32_t k, uint32_t& m0, uint32_t& n0) {
        uint32_t tm, tn;
        w16_tile(blockIdx.x, k, G, tiles_m, tiles_n, tm, tn);
        m0 = tm * BM;
        n0 = tn * 256u;
    };
    // (at most 2^31 bytes: an offset of 2^31 and more is past them)
    auto x_tile = [&](Cursor& c, uint32_t k) {
        uint32_t m0, n0;
        tile_origin(k, m0, n0);
        c = Cursor{0, a.x + (uint64_t)m0 * a.x_stride, k < n_tiles ? (a.M - m0 < BM ? a.M - m0 : BM) * a.x_stride : 0u};
    };
    auto w_tile = [&](Cursor& c, uint32_t k) {
        uint32_t m0, n0;
        tile_origin(k, m0, n0);
        c = Cursor{0, a.w + (uint64_t)n0 * a.w_stride, k < n_tiles ? (a.N - n0 < 256u ? a.N - n0 : 256u) * a.w_stride : 0u};
    };
    Cursor cx, cw, nx, nw;
    auto advance = [&](Cursor& c, const Cursor& next) {
        if (++c.s == SP) c = next;
    };
    auto rsrc = [&](const Cursor& c) { return make_rsrc(c.base + (uint64_t)c.s * kRow, c.s < S ? c.size : 0u); };
    // 2^31 for a lane whose chunk of stage s is past K (even i, odd i)
    auto past = [&](uint32_t s, uint32_t odd) {
        return s * kRow + ((c0 ^ odd) << 4) < a.K ? 0u : 0x80000000u;
    };
    auto xdma = [&](rsrc_t r, uint8_t* Xs, int i, uint32_t add) {
        dma16(r, Xs + wave * (16u * MB * kRow) + 1024u * i, xvoff[i] + add);
    };
    auto wdma = [&](rsrc_t r, uint8_t* Ws, int i, uint32_t add) {
        dma16(r, Ws + wave * (64u * kRow) + 1024u * i, wvoff[i] + add);
    };
    // part p of four of a stage's loads: the weights of the next stage, then the tokens two stages ahead
    constexpr int PER = (WD + XD + 3) / 4;
    auto issue_part = [&](auto PART, rsrc_t wr, const uint32_t (&wp)[2], uint8_t* Wd, rsrc_t xr, const uint32_t (&xp)[2], uint8_t* Xd) {
        constexpr int p = decltype(PART)::value;
        static_for<PER * p, (PER * p + PER < WD + XD ? PER * p + PER : WD + XD)>([&](auto I) {
            constexpr int i = decltype(I)::value;
            if constexpr (i < WD) wdma(wr, Wd, i, wp[i & 1]);
            else xdma(xr, Xd, i - WD, xp[(i - WD) & 1]);
        });
    };

    i32x16 acc[4][MB];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (uint32_t b = 0; b < MB; b++) acc[i][b] = i32x16{};
    auto read_frags = [&](FragsI8<MB>& f, const uint8_t* Xs, const uint8_t* Ws, int t) {
#pragma unroll
        for (uint32_t b = 0; b < MB; b++) f.x[b] = *(const i32x4*)(Xs + b * 32u * kRow + xoff[t]);
#pragma unroll
        for (int i = 0; i < 4; i++) f.w[i] = *(const i32x4*)(Ws + i * 32 * (int)kRow + woff[t]);
    };
    auto mfma_step = [&](const FragsI8<MB>& f) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (uint32_t b = 0; b < MB; b++) acc[i][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[i], f.x[b], acc[i][b], 0, 0, 0);
    };

    // A wave's results: token 32 b + l32, channels 32 i + 8 g + 4 kh + 0..3. Through LDS (its own
    // quarter of W1, which its own DMAs alone write next), 32 tokens x 256 bytes at a time, so that a store
    // instruction writes four whole rows of it.
    const rsrc_t wsr = make_rsrc(a.w_scales, (uint64_t)a.N * 4u);
    auto store_tile = [&](uint32_t k) {
        uint32_t m0, n0;
        tile_origin(k, m0, n0);
        uint8_t* const st = W1 + wave * 8192u;
        constexpr int HALVES = OT == kGgmlF32 ? 2 : 1, PERH = 4 / HALVES;  // 32-channel blocks a row of 256 bytes
        constexpr uint32_t EPC = 16u / out_size<OT>();                     // elements a 16-byte chunk
        const uint32_t nw0 = n0 + wn * 128u, mw0 = m0 + wm * 32u * MB;
        const uint32_t cc = lane & 15u, rq = lane >> 4;
        float xs[MB];
#pragma unroll
        for (uint32_t b = 0; b < MB; b++) xs[b] = a.x_scales[min(mw0 + 32u * b + l32, a.M - 1u)];
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            f32x4 ws[PERH][4];
#pragma unroll
            for (int i = 0; i < PERH; i++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    ws[i][g] = __builtin_bit_cast(f32x4, bload16(wsr, (nw0 + 32u * (PERH * h + i) + 8u * g + 4u * kh) * 4u, 0u));
#pragma unroll
            for (uint32_t b = 0; b < MB; b++) {
#pragma unroll
                for (int i = 0; i < PERH; i++) {
                    i32x16& s = acc[PERH * h + i][b];
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        float y[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] = scaled(s[4 * g + e], xs[b], ws[i][g][e]);
                        if constexpr (OT == kGgmlF32)
                            *(f32x4*)(st + l32 * 256u + (((8u * i + 2u * g + kh) ^ (l32 & 15u)) << 4)) = f32x4{y[0], y[1], y[2], y[3]};
                        else
                            *(u32x2*)(st + l32 * 256u + (((4u * i + g) ^ (l32 & 15u)) << 4) + 8u * kh) =
                                u32x2{pack2<OT>(y[0], y[1]), pack2<OT>(y[2], y[3])};
                    }
                    s = i32x16{};
                }
                u32x4 v[8];  // all eight reads before the stores
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t r = 4u * i + rq;
                    v[i] = *(const u32x4*)(st + r * 256u + ((cc ^ (r & 15u)) << 4));
                }
                const uint32_t n = nw0 + 64u * h + EPC * cc;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t m = mw0 + 32u * b + 4u * i + rq;
                    if (m >= a.M || n >= a.N) continue;
                    uint8_t* const dst = (uint8_t*)a.out + ((uint64_t)m * a.out_stride + n) * out_size<OT>();
                    if (n + EPC <= a.N) {
                        if constexpr (OT == kGgmlF32) *(u32x4_s4*)dst = v[i];
                        else *(u32x4_a2*)dst = v[i];
                    } else {
#pragma unroll
                        for (uint32_t e = 0; e < EPC; e++)
                            if (n + e < a.N) {
                                if constexpr (OT == kGgmlF32) ((uint32_t*)dst)[e] = v[i][e];
                                else ((uint16_t*)dst)[e] = (uint16_t)(v[i][e / 2u] >> (16u * (e & 1u)));
                            }
                    }
                }
            }
        }
    };

    // W(0) -> W0, X(0) -> X0, X(1) -> X1; stage 0's operands have landed once at most X(1)'s are in flight
    x_tile(cx, 0);
    w_tile(cw, 0);
    x_tile(nx, 1);
    w_tile(nw, 1);
    {
        const uint32_t wp[2] = {past(cw.s, 0), past(cw.s, 1)};
        const rsrc_t wr = rsrc(cw);
#pragma unroll
        for (int i = 0; i < WD; i++) wdma(wr, W0, i, wp[i & 1]);
        advance(cw, nw);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t xp[2] = {past(cx.s, 0), past(cx.s, 1)};
            const rsrc_t xr = rsrc(cx);
#pragma unroll
            for (int i = 0; i < XD; i++) xdma(xr, j == 0 ? X0 : X1, i, xp[i & 1]);
            advance(cx, nx);
        }
    }
    LLMR_STAGE_BARRIER(XD);

    FragsI8<MB> F0, F1;
    // Stage g reads X[g%3], W[g%2] and sends for W(g+1) -> W[(g+1)%2] and X(g+2) -> X[(g+2)%3] (both slots were
    // last read in stage g-1). The barrier at its end waits until at most X(g+2)'s DMAs are in flight.
    // A tile's stages are made a multiple of six, so that every slot is a fixed one; those past K only go
    // on with the loads.
#define LLMR8_STEP(P, FR, FM, XC, WC, XDST, WDST)                                             \
    issue_part(std::integral_constant<int, P>{}, wr_, wp_, WDST, xr_, xp_, XDST);             \
    read_frags(FR, XC, WC, P);                                                                \
    mfma_step(FM);                                                                            \
    if constexpr (MB == 4u) {                                                                 \
        LLMR8_STEP_SCHEDULE;                                                                  \
    }                                                                                         \
    __builtin_amdgcn_sched_barrier(0)
#define LLMR8_STAGE(I, XC, WC, XDST, WDST)                                                    \
    {                                                                                         \
        const rsrc_t wr_ = rsrc(cw), xr_ = rsrc(cx);                                          \
        const uint32_t wp_[2] = {past(cw.s, 0), past(cw.s, 1)};                               \
        const uint32_t xp_[2] = {past(cx.s, 0), past(cx.s, 1)};                               \
        if (s0 + I < S) {                                                                     \
            LLMR8_STEP(0, F0, F1, XC, WC, XDST, WDST);                                        \
            LLMR8_STEP(1, F1, F0, XC, WC, XDST, WDST);                                        \
            LLMR8_STEP(2, F0, F1, XC, WC, XDST, WDST);                                        \
            LLMR8_STEP(3, F1, F0, XC, WC, XDST, WDST);                                        \
        } else {                                                                              \
            issue_part(std::integral_constant<int, 0>{}, wr_, wp_, WDST, xr_, xp_, XDST);     \
            issue_part(std::integral_constant<int, 1>{}, wr_, wp_, WDST, xr_, xp_, XDST);     \
            issue_part(std::integral_constant<int, 2>{}, wr_, wp_, WDST, xr_, xp_, XDST);     \
            issue_part(std::integral_constant<int, 3>{}, wr_, wp_, WDST, xr_, xp_, XDST);     \
        }                                                                                     \
        advance(cw, nw);                                                                      \
        advance(cx, nx);                                                                      \
        LLMR_STAGE_BARRIER(XD);                                                               \
    }
    for (uint32_t k = 0; k < n_tiles; k++) {
        if (k > 0) {  // the load cursors have moved on to tile k: prepare tile k+1
            x_tile(nx, k + 1u);
            w_tile(nw, k + 1u);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            if (i < MB) F1.x[i % MB] = i32x4{0, 0, 0, 0};
            F1.w[i] = i32x4{0, 0, 0, 0};
        }
        for (uint32_t s0 = 0; s0 < SP; s0 += 6u) {
            LLMR8_STAGE(0, X0, W0, X2, W1)
            LLMR8_STAGE(1, X1, W1, X0, W0)
            LLMR8_STAGE(2, X2, W0, X1, W1)
            LLMR8_STAGE(3, X0, W1, X2, W0)
            LLMR8_STAGE(4, X1, W0, X0, W1)
            LLMR8_STAGE(5, X2, W1, X1, W0)
        }
        mfma_step(F1);
        store_tile(k);
    }
#undef LLMR8_STAGE
#undef LLMR8_STEP
    LLMR_WAIT_VMCNT(0);  // no DMA may still be writing this workgroup's LDS when it exits
}

// ---- small tiles -----------------------------------------------------------------------
//
// Tiles of 64 MB tokens x 128 channels, one a workgroup, for launches that large tiles leave most CUs without: four
// waves in 2 x 2 of 32 MB x 64, stages of 128 bytes of K in four LDS slots, sent for three stages ahead (a stage
// takes less than its loads' way from L2 and memory).

template <uint32_t OT, uint32_t MB>
__global__ void __launch_bounds__(256, 1) matmul_i8_small(MatmulI8Args a, uint32_t tiles_m) {
    constexpr uint32_t BM = 64u * MB, BN = 128u, SLOT = (BM + BN) * kRow;
    constexpr int XD = 2 * MB, WD = 4;
    __shared__ __attribute__((aligned(16))) uint8_t L0[SLOT];
    __shared__ __attribute__((aligned(16))) uint8_t L1[SLOT];
    __shared__ __attribute__((aligned(16))) uint8_t L2[SLOT];
    __shared__ __attribute__((aligned(16))) uint8_t L3[SLOT];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t l32 = lane & 31u, kh = lane >> 5, wm = wave & 1u, wn = wave >> 1;
    // an XCD has a run of channel tiles with all their token tiles
    const uint32_t L = xcd_linear(blockIdx.x, gridDim.x), m0 = (L % tiles_m) * BM, n0 = (L / tiles_m) * BN;
    const uint32_t S = (a.K + kRow - 1u) / kRow;
    const int8_t* const xb = a.x + (uint64_t)m0 * a.x_stride;
    const int8_t* const wb = a.w + (uint64_t)n0 * a.w_stride;
    const uint32_t xsize = (a.M - m0 < BM ? a.M - m0 : BM) * a.x_stride, wsize = (a.N - n0 < BN ? a.N - n0 : BN) * a.w_stride;
    uint32_t xvoff[XD], wvoff[WD];
    const uint32_t c0 = (lane & 7u) ^ (lane >> 3);  // of even i; odd i: ^ 1
#pragma unroll
    for (int i = 0; i < XD; i++) xvoff[i] = (16u * MB * wave + 8u * i + (lane >> 3)) * a.x_stride + ((c0 ^ (i & 1)) << 4);
#pragma unroll
    for (int i = 0; i < WD; i++) wvoff[i] = (32u * wave + 8u * i + (lane >> 3)) * a.w_stride + ((c0 ^ (i & 1)) << 4);
    uint32_t xoff[4], woff[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint32_t ch = 4u * (t >> 1) + 2u * kh + (t & 1);
        xoff[t] = lds_off(wm * 32u * MB + l32, ch);
        woff[t] = BM * kRow + lds_off(wn * 64u + l32, ch);
    }
    auto send = [&](uint32_t s, uint8_t* slot) {  // (a stage past the last: nothing is read, zeros arrive)
        const auto xr = make_rsrc(xb + (uint64_t)s * kRow, s < S ? xsize : 0u), wr = make_rsrc(wb + (uint64_t)s * kRow, s < S ? wsize : 0u);
        const uint32_t past[2] = {s * kRow + (c0 << 4) < a.K ? 0u : 0x80000000u, s * kRow + ((c0 ^ 1u) << 4) < a.K ? 0u : 0x80000000u};
#pragma unroll
        for (int i = 0; i < WD; i++) dma16(wr, slot + BM * kRow + wave * (32u * kRow) + 1024u * i, wvoff[i] + past[i & 1]);
#pragma unroll
        for (int i = 0; i < XD; i++) dma16(xr, slot + wave * (16u * MB * kRow) + 1024u * i, xvoff[i] + past[i & 1]);
    };
    i32x16 acc[2][MB];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (uint32_t b = 0; b < MB; b++) acc[i][b] = i32x16{};
    auto work = [&](const uint8_t* slot) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            i32x4 xf[MB], wf[2];
#pragma unroll
            for (uint32_t b = 0; b < MB; b++) xf[b] = *(const i32x4*)(slot + b * 32u * kRow + xoff[t]);
#pragma unroll
            for (int i = 0; i < 2; i++) wf[i] = *(const i32x4*)(slot + i * 32 * (int)kRow + woff[t]);
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (uint32_t b = 0; b < MB; b++) acc[i][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[i], xf[b], acc[i][b], 0, 0, 0);
        }
    };
    send(0, L0);
    send(1, L1);
    send(2, L2);
    LLMR_STAGE_BARRIER(2 * (XD + WD));
    // Stage s reads slot s % 4 and sends for stage s + 3 into the slot that stage s - 1 read; its end waits until at
    // most the stages s + 2 and s + 3 are on their way.
    for (uint32_t s = 0;;) {
#define LLMR8_SMALL(CUR, DST)            \
    send(s + 3u, DST);                   \
    work(CUR);                           \
    LLMR_STAGE_BARRIER(2 * (XD + WD));   \
    if (++s == S) break
        LLMR8_SMALL(L0, L3);
        LLMR8_SMALL(L1, L0);
        LLMR8_SMALL(L2, L1);
        LLMR8_SMALL(L3, L2);
#undef LLMR8_SMALL
    }
    LLMR_WAIT_VMCNT(0);  // no DMA may still be writing this workgroup's LDS when it exits
#pragma unroll
    for (uint32_t b = 0; b < MB; b++) {
        const uint32_t m = m0 + wm * 32u * MB + 32u * b + l32;
        const float xs = a.x_scales[m < a.M ? m : a.M - 1u];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (uint32_t g = 0; g < 4u; g++) {
                const uint32_t c = n0 + wn * 64u + 32u * i + 8u * g + 4u * kh;
                float ws[4];
#pragma unroll
                for (uint32_t e = 0; e < 4u; e++) ws[e] = a.w_scales[c + e < a.N ? c + e : a.N - 1u];
                if (m < a.M && c < a.N)
                    store4<OT>(a, m, c, i32x4{acc[i][b][4 * g], acc[i][b][4 * g + 1], acc[i][b][4 * g + 2], acc[i][b][4 * g + 3]}, xs, ws);
            }
    }
}

template <uint32_t OT, uint32_t MB>
hipError_t launch_small(const MatmulI8Args& a, hipStream_t st) {
    const uint32_t tm = (a.M + 64u * MB - 1u) / (64u * MB), tn = (a.N + 127u) / 128u;
    hipLaunchKernelGGL((matmul_i8_small<OT, MB>), dim3(tm * tn), dim3(256), 0, st, a, tm);
    return hipGetLastError();
}

template <uint32_t OT, uint32_t MB>
hipError_t launch_tiles(const MatmulI8Args& a, int num_cus, hipStream_t st) {
    hipLaunchKernelGGL((matmul_i8_tiles<OT, MB>), dim3(num_cus), dim3(256), 0, st, a, (a.M + 64u * MB - 1u) / (64u * MB),
                       (a.N + 255u) / 256u);
    return hipGetLastError();
}

template <uint32_t OT, uint32_t MT, uint32_t CT>
hipError_t launch_few(const MatmulI8Args& a, hipStream_t st) {
    const dim3 grid((a.N + 16u * CT - 1u) / (16u * CT), (a.M + 16u * MT - 1u) / (16u * MT));
    hipLaunchKernelGGL((matmul_i8_few<OT, MT, CT>), grid, dim3(64 * kFewWaves), 0, st, a);
    return hipGetLastError();
}

template <uint32_t OT>
hipError_t launch_matmul(const MatmulI8Args& a, int num_cus, hipStream_t st) {
    const uint32_t cus = (uint32_t)num_cus;
    // Up to 16 tokens the weight stream, 32 channels a workgroup where that leaves two a CU (N 20480, K 4096, us: 18.1 to
    // 19.7, of 16 channels 19.2 to 22, small tiles 24.5 to 26; K 1024: 7.5, 11, 8.6); up to 64 where N or K makes it faster
    // than small tiles (32 tokens, K 1024, N 6144, 10240, 20480: 6.2, 8.3, 12.9 and 7.7, 7.9, 9.0; K 4096: 9.1, 11.9, 27.2
    // and 15.2, 15.8, 25.6; 64 tokens, K 4096: 14.9, 21.3, 32.0 and 16.1, 23.1, 28.4).
    if (a.M <= 16u && a.N < (1u << 27))  // (under 2^32 threads)
        return a.N / 32u >= 2u * cus ? launch_few<OT, 1, 2>(a, st) : launch_few<OT, 1, 1>(a, st);
    if (a.M <= 64u && (a.N <= 24u * cus || (a.N <= 40u * cus && a.K >= 2048u)))
        return a.M <= 32u ? launch_few<OT, 2, 1>(a, st) : launch_few<OT, 4, 1>(a, st);
    // The tiles whose rounds take least, in ns: a stage of 128 bytes of K, and what a round has besides. Fitted to one
    // round each (S stages of 256 x N, 512 x 4096, 128 x 1024 and so on: within 15%), the largest to full rounds. The last
    // is the weight stream's, for few tiles of long rows (300 x 16000 x 600: 21 us, in small tiles 44; 100 x 14336 x 1000: 18, 40).
    struct Kind {
        uint32_t m, n, stage, round;
    };
    static const Kind kinds[] = {{64, 128, 410, 1800}, {128, 128, 580, 3000}, {64, 256, 600, 3100},
                                 {128, 256, 820, 5000}, {192, 256, 1150, 6000}, {256, 256, 1450, 7000}, {64, 16, 195, 2200}};
    const uint64_t S = (a.K + kRow - 1u) / kRow;
    uint32_t best = 0;
    uint64_t least = ~0ull;
    for (uint32_t i = 0; i < 7u; i++) {
        const Kind& k = kinds[i];
        const uint64_t tiles = (uint64_t)((a.M + k.m - 1u) / k.m) * ((a.N + k.n - 1u) / k.n);
        const uint64_t cost = (tiles + (uint64_t)num_cus - 1u) / (uint64_t)num_cus * (S * k.stage + k.round);
        // (a launch has under 2^32 threads and 2^16 blocks along y)
        const bool fits = i < 2u ? tiles < (1u << 24) : i < 6u || (tiles < (1u << 23) && a.M <= 64u * 65535u);
        if (cost < least && fits) {
            least = cost;
            best = i;
        }
    }
    switch (best) {
        case 0: return launch_small<OT, 1>(a, st);
        case 1: return launch_small<OT, 2>(a, st);
        case 2: return launch_tiles<OT, 1>(a, num_cus, st);
        case 3: return launch_tiles<OT, 2>(a, num_cus, st);
        case 4: return launch_tiles<OT, 3>(a, num_cus, st);
        case 5: return launch_tiles<OT, 4>(a, num_cus, st);
        default: return launch_few<OT, 4, 1>(a, st);
    }
}

}  // namespace

hipError_t launch_matmul_i8(const MatmulI8Args& a, uint32_t otype, int num_cus, hipStream_t st) {
    if (otype == kGgmlF32) return launch_matmul<kGgmlF32>(a, num_cus, st);
    return otype == kGgmlF16 ? launch_matmul<kGgmlF16>(a, num_cus, st) : launch_matmul<kGgmlBF16>(a, num_cus, st);
}

}  // namespace llmr
