// mx4.hip - what fills and reads back the paged key/value cache in 4 bits: the QKV
// projection's rows into query rows and cache slots (llmr_qkv_tokens_mx4), and cached
// rows as 16-bit rows (llmr_mx4_rows).
//
// 32 elements x of a row become x / 2^e rounded to E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6),
// e + 2 the exponent of the largest |x| rounded to two significant bits: the largest is
// then 3.5 to 7 times 2^e, as far from 6 as rounding to a neighbour would put it. With
// e + 2 its plain exponent it would be up to 8 and lose a quarter.
//
// Bound by memory: 8192 tokens of 32/8 heads of 128 with norms and rotation 55 us (272 MB:
// 4.9 TB/s), as many rows read back 10.5; 64 tokens 3.6 and 2.5, a launch each.
#include "llmr_device.h"
#include "llmr_internal.h"
#include "mx4_values.h"

// products and sums round where the formulas write them, as in the other glue
#pragma clang fp contract(off)

namespace llmr {
namespace {

constexpr uint32_t kMaxGridRows = 1u << 23;

template <uint32_t OT>
__device__ __forceinline__ uint32_t pack16(float x, float y) {
    return OT == kGgmlF16 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
}

// A double as a float that lies on the same side of every number of 22 bits or fewer (the
// borders between E2M1 numbers, and between powers of two): the nearer to zero, its last bit set
// where bits are lost.
__device__ __forceinline__ float to_odd(double d) {
    const float f = (float)d;
    uint32_t b = __float_as_uint(f);
    if ((double)f != d) {
        b -= fabs((double)f) > fabs(d) ? 1u : 0u;
        b |= 1u;
    }
    return __uint_as_float(b);
}

__device__ __forceinline__ uint32_t top_bits(f32x4 x) {
    auto m = [](float a) { return __float_as_uint(a) & 0x7fffffffu; };  // (NaN above everything)
    return max(max(m(x.x), m(x.y)), max(m(x.z), m(x.w)));
}

// The biased exponent of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t block_exponent(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    const int e = (int)((top + (1u << 21)) >> 23) - 2;
    return (uint32_t)min(max(e, 127 - 23), 127 + 13);
}
// Four elements as 16 bits of codes.
__device__ __forceinline__ uint32_t codes4(f32x4 x, uint32_t e) {
    const float s = __uint_as_float(e << 23);
    // v_cvt_scalef32_pk_fp4_f32: x / s, to nearest even, ends at 6
    const uint32_t lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x.x, x.y, s, 0);
    return e == 255u ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, x.z, x.w, s, 1) & 0xffffu;
}

// The threads of qkv_tokens_kernel: D / 8 lanes a head, two vectors of four elements a lane (of the
// two halves, or one behind the other: the pairs of the rotation). A block is eight lanes' vectors
// of one half, or both vectors of four lanes. Keys are normed and rotated in 64 bits (one head in
// six, where 32/8 heads are; the vector ALU does 64-bit fmas at the 32-bit rate).
template <uint32_t QT, uint32_t D, bool HALVES>
__global__ void __launch_bounds__(256) qkv_tokens_mx4_kernel(QkvTokensArgs a, uint8_t* k_scales, uint8_t* v_scales) {
    constexpr uint32_t L = D / 8u;  // lanes of a head
    const uint32_t l = threadIdx.x % L, h = blockIdx.y * (256u / L) + threadIdx.x / L;
    const uint32_t r = blockIdx.z * kMaxGridRows + blockIdx.x;
    if (r >= a.n_tokens || h >= a.n_heads + 2u * a.n_kv_heads) return;  // (whole heads: the reductions stay within one)
    const uint32_t e0 = HALVES ? 4u * l : 8u * l, e1 = HALVES ? e0 + D / 2u : e0 + 4u;
    const float* src = a.qkv + (size_t)r * a.qkv_stride + (size_t)h * D;
    f32x4 x0 = *(const f32x4*)(src + e0), x1 = *(const f32x4*)(src + e1);
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv_heads;
    const int32_t slot = is_q ? 0 : a.slots[r];
    const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    f32x4 w0{1.0f, 1.0f, 1.0f, 1.0f}, w1 = w0, c{1.0f, 1.0f, 1.0f, 1.0f}, sn{};
    if (w) {
        w0 = *(const f32x4*)(w + e0);
        w1 = *(const f32x4*)(w + e1);
    }
    if (a.rope_cos && !is_v) {
        const uint32_t pos = a.positions ? (uint32_t)min(max(a.positions[r], 0), (int32_t)(a.n_positions - 1u)) : r;
        const size_t at = (size_t)pos * (D / 2u) + 4u * l;
        c = *(const f32x4*)(a.rope_cos + at);
        sn = *(const f32x4*)(a.rope_sin + at);
    }
    if (is_q) {  // llmr_qkv_tokens' arithmetic
        if (w) {
            const f32x4 q = x0 * x0 + x1 * x1;
            float ss = (q.x + q.y) + (q.z + q.w);
#pragma unroll
            for (uint32_t o = L / 2u; o > 0; o >>= 1) ss += __shfl_xor(ss, (int)o, 64);
            const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
            x0 = x0 * inv * w0;
            x1 = x1 * inv * w1;
        }
        if (a.rope_cos) {
            const f32x4 u = HALVES ? x0 : f32x4{x0.x, x0.z, x1.x, x1.z}, v = HALVES ? x1 : f32x4{x0.y, x0.w, x1.y, x1.w};
            const f32x4 y0 = u * c - v * sn, y1 = u * sn + v * c;
            x0 = HALVES ? y0 : f32x4{y0.x, y1.x, y0.y, y1.y};
            x1 = HALVES ? y1 : f32x4{y0.z, y1.z, y0.w, y1.w};
        }
        uint16_t* const dst = (uint16_t*)a.q + (size_t)r * a.q_stride + (size_t)h * D;
        *(u32x2*)(dst + e0) = u32x2{pack16<QT>(x0.x, x0.y), pack16<QT>(x0.z, x0.w)};
        *(u32x2*)(dst + e1) = u32x2{pack16<QT>(x1.x, x1.y), pack16<QT>(x1.z, x1.w)};
        return;
    }
    if (!is_v && (w || a.rope_cos)) {
        double y0[4], y1[4], inv = 1.0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y0[i] = x0[i];
            y1[i] = x1[i];
        }
        if (w) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 4; i++) ss += y0[i] * y0[i] + y1[i] * y1[i];
#pragma unroll
            for (uint32_t o = L / 2u; o > 0; o >>= 1) ss += __shfl_xor(ss, (int)o, 64);
            inv = 1.0 / sqrt(ss / (double)D + (double)a.eps);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                y0[i] = y0[i] * inv * (double)w0[i];
                y1[i] = y1[i] * inv * (double)w1[i];
            }
        }
        if (a.rope_cos) {
#pragma unroll
            for (int i = 0; i < 4; i++) {  // pair i of the lane, in place
                double& u = HALVES ? y0[i] : i < 2 ? y0[2 * i] : y1[2 * i - 4];
                double& v = HALVES ? y1[i] : i < 2 ? y0[2 * i + 1] : y1[2 * i - 3];
                const double cc = c[i], ss = sn[i], t = u * cc - v * ss;
                v = u * ss + v * cc;
                u = t;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x0[i] = to_odd(y0[i]);
            x1[i] = to_odd(y1[i]);
        }
    }
    uint32_t t0 = top_bits(x0), t1 = top_bits(x1);
    if (!HALVES) t0 = max(t0, t1);
#pragma unroll
    for (uint32_t o = (HALVES ? 8u : 4u) / 2u; o > 0; o >>= 1) {
        t0 = max(t0, (uint32_t)__shfl_xor((int)t0, (int)o, 64));
        if (HALVES) t1 = max(t1, (uint32_t)__shfl_xor((int)t1, (int)o, 64));
    }
    const uint32_t b0 = block_exponent(t0), b1 = HALVES ? block_exponent(t1) : b0;
    const uint32_t page = (uint32_t)slot >> a.page_log2;
    if (slot < 0 || page >= a.n_pages) return;
    const uint32_t kh = h - a.n_heads - (is_v ? a.n_kv_heads : 0u);
    const size_t row = (((size_t)page * a.n_kv_heads + kh) << a.page_log2) + ((uint32_t)slot & ((1u << a.page_log2) - 1u));
    uint8_t* const dst = (uint8_t*)(is_v ? a.v : a.k) + row * (D / 2u);
    uint8_t* const sc = (is_v ? v_scales : k_scales) + row * (D / 32u);
    const uint32_t c0 = codes4(x0, b0), c1 = codes4(x1, b1);
    if (HALVES) {
        *(uint16_t*)(dst + e0 / 2u) = (uint16_t)c0;
        *(uint16_t*)(dst + e1 / 2u) = (uint16_t)c1;
        if (l % 8u == 0) {
            sc[e0 / 32u] = (uint8_t)b0;
            sc[e1 / 32u] = (uint8_t)b1;
        }
    } else {
        *(uint32_t*)(dst + e0 / 2u) = c0 | c1 << 16;
        if (l % 4u == 0) sc[e0 / 32u] = (uint8_t)b0;
    }
}

// Eight elements a thread: four bytes and a scale in, 16 bytes out.
template <uint32_t OT, uint32_t D>
__global__ void __launch_bounds__(256) mx4_rows_kernel(Mx4RowsArgs a) {
    constexpr uint32_t L = D / 8u;
    const uint32_t l = threadIdx.x % L, h = blockIdx.y * (256u / L) + threadIdx.x / L;
    const uint32_t r = blockIdx.z * kMaxGridRows + blockIdx.x;
    if (r >= a.n_rows || h >= 2u * a.n_kv_heads) return;
    const int32_t slot = a.slots[r];
    const uint32_t page = (uint32_t)slot >> a.page_log2;
    if (slot < 0 || page >= a.n_pages) return;
    const bool is_v = h >= a.n_kv_heads;
    const uint32_t kh = h - (is_v ? a.n_kv_heads : 0u);
    const Mx4Pages& c = is_v ? a.v : a.k;
    const size_t row = (((size_t)page * a.n_kv_heads + kh) << a.page_log2) + ((uint32_t)slot & ((1u << a.page_log2) - 1u));
    const uint32_t w = *(const uint32_t*)(c.data + row * (D / 2u) + 4u * l);
    const u32x4 o = values8<OT>(w, power4(c.scales[row * (D / 32u) + l / 4u]));
    *(u32x4*)((uint16_t*)(is_v ? a.v_out : a.k_out) + (size_t)r * a.out_stride + (size_t)kh * D + 8u * l) = o;
}

// Workgroups: a row each along x (its 256 threads a row stay under 2^32), going on in z; heads along y.
dim3 row_grid(uint32_t rows, uint32_t heads, uint32_t dim) {
    const uint32_t per = 256u / (dim / 8u), x = rows < kMaxGridRows ? rows : kMaxGridRows;
    return dim3(x, (heads + per - 1u) / per, (rows + x - 1u) / x);
}

}  // namespace

hipError_t launch_qkv_tokens_mx4(const QkvTokensArgs& a, uint8_t* k_scales, uint8_t* v_scales, uint32_t dim,
                                 uint32_t qtype, bool halves, hipStream_t st) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, row_grid(a.n_tokens, a.n_heads + 2u * a.n_kv_heads, dim), dim3(256), 0, st, a, k_scales,
                           v_scales);
    };
    if (qtype == kGgmlBF16) {
        if (dim == 128u) halves ? go(qkv_tokens_mx4_kernel<kGgmlBF16, 128, true>) : go(qkv_tokens_mx4_kernel<kGgmlBF16, 128, false>);
        else halves ? go(qkv_tokens_mx4_kernel<kGgmlBF16, 64, true>) : go(qkv_tokens_mx4_kernel<kGgmlBF16, 64, false>);
    } else {
        if (dim == 128u) halves ? go(qkv_tokens_mx4_kernel<kGgmlF16, 128, true>) : go(qkv_tokens_mx4_kernel<kGgmlF16, 128, false>);
        else halves ? go(qkv_tokens_mx4_kernel<kGgmlF16, 64, true>) : go(qkv_tokens_mx4_kernel<kGgmlF16, 64, false>);
    }
    return hipGetLastError();
}

hipError_t launch_mx4_rows(const Mx4RowsArgs& a, uint32_t dim, uint32_t otype, hipStream_t st) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, row_grid(a.n_rows, 2u * a.n_kv_heads, dim), dim3(256), 0, st, a);
    };
    if (otype == kGgmlBF16) dim == 128u ? go(mx4_rows_kernel<kGgmlBF16, 128>) : go(mx4_rows_kernel<kGgmlBF16, 64>);
    else dim == 128u ? go(mx4_rows_kernel<kGgmlF16, 128>) : go(mx4_rows_kernel<kGgmlF16, 64>);
    return hipGetLastError();
}

}  // namespace llmr
