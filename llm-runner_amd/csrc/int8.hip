// int8.hip - rows to 8-bit integers with a scale each (llmr_quantize_rows_i8):
//
//   y = x * norm, a = max |y|, q = 127 y / a to nearest even, scale = a / 127 [/ rms(x)]
//
// A row is read once and held in registers, as it lies, from its sums to the rounding;
// rows past 16384 elements are read twice. The definition is in 64 bits, so that q does
// not depend on an order or a contraction; f32 rounds where it provably gives the same
// (round8). Bound by memory, a wave's loads waited for (76% of its cycles at 8192 x 3840). Over
// inputs past the memory-side cache, us: 8192 x 3840 bf16 27.4 (3.4 TB/s), 8192 x 4096 f32 with
// the norm 39 (4.3), 8192 x 10240 f32 with the norm 100 (4.2: 16 waves a CU, whose sums and
// roundings do not hide all of their loads); with an input that it holds 26, 34, 103. Rows past
// 16384: 2048 x 28672 bf16 59 (3.0; a large copy's rate would be 34), 8192 x 28672 190 (3.7),
// 64 x 28672 22, one of 28672 13, one of 131056 55: 256 threads a row, each step waits for its
// own load. One row of 4096 3.0 to 4.1, a launch and two dependent loads.
#include "llmr_device.h"
#include "llmr_internal.h"

// every rounding that the definitions name is one
#pragma clang fp contract(off)

namespace llmr {
namespace {

// Eight elements as they lie, and as f32.
template <uint32_t XT>
struct Eight {
    u32x4 w[XT == kGgmlF32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* x) {
        w[0] = *(const u32x4*)x;
        if constexpr (XT == kGgmlF32) w[1] = *((const u32x4*)x + 1);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < (XT == kGgmlF32 ? 8 : 4); i++) {
            const uint32_t u = w[i / 4][i % 4];
            if constexpr (XT == kGgmlF32) {
                v[i] = __uint_as_float(u);
            } else if constexpr (XT == kGgmlBF16) {
                v[2 * i] = __uint_as_float(u << 16);
                v[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
            } else {
                const f16x2 h = __builtin_bit_cast(f16x2, u);
                v[2 * i] = (float)h.x;
                v[2 * i + 1] = (float)h.y;
            }
        }
    }
};

constexpr uint32_t kRowThreads = 256;

// 127 y / a to the nearest whole number, ties to even; r = 127 / a. Where y r is next to a half, the
// half is compared with exactly: d is the sign of 254 |y| - (2 k + 1) a. a is a product of up to 48 bits
// and (2 k + 1) a has up to 56, so its low part is kept; the differences are small and whole multiples
// of y's last bit, so both are exact. (Rows have such elements: half of the largest one is 63.5.)
__device__ __forceinline__ int round127(double y, double r, double a) {
    const double v = y * r, q = rint(v);
    int n = (int)q;
    if (fabs(fabs(v - q) - 0.5) < 1e-9) {
        const double k = floor(fabs(v)), h = 2.0 * k + 1.0, p = h * a;
        const double d = fma(254.0, fabs(y), -p) - fma(h, a, -p);
        const int lo = (int)k;
        const int m = d > 0.0 ? lo + 1 : d < 0.0 ? lo : lo + (lo & 1);
        n = v < 0.0 ? -m : m;
    }
    return n;
}

// A row's sums over the TPR threads that have it (a wave, or a workgroup).
struct RowSums {
    double top, ss;  // largest |y|, sum of x^2
    uint32_t bad;    // an infinity or NaN
};
template <uint32_t TPR>
__device__ __forceinline__ RowSums row_sums(RowSums s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        s.top = fmax(s.top, __shfl_xor(s.top, o, 64));
        s.ss += __shfl_xor(s.ss, o, 64);
    }
    s.bad = __builtin_amdgcn_ballot_w64(s.bad != 0) != 0 ? 1u : 0u;
    if constexpr (TPR > 64u) {
        __shared__ RowSums part[TPR / 64u];
        if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        s = part[0];
#pragma unroll
        for (uint32_t i = 1; i < TPR / 64u; i++) {
            s.top = fmax(s.top, part[i].top);
            s.ss += part[i].ss;
            s.bad |= part[i].bad;
        }
        __syncthreads();
    }
    return s;
}

// Eight elements of a row into its sums.
template <bool NORM>
__device__ __forceinline__ void add8(RowSums& s, const float (&v)[8], const float (&w)[8]) {
    if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const double y = (double)v[i] * (double)w[i];  // exact
            s.top = fmax(s.top, fabs(y));
            if (!(fabs(y) < (double)INFINITY)) s.bad = 1u;
            s.ss += (double)v[i] * (double)v[i];
        }
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);  // (NaN above everything)
        if (m >= 0x7f800000u) s.bad = 1u;
        else s.top = fmax(s.top, (double)__uint_as_float(m));
    }
}

// What rounding a row's elements needs.
struct RowScale {
    double r, top;
    float r32;
    bool zero, exact;  // no rounding at all; f32 has not the range for it
};
template <bool NORM>
__device__ __forceinline__ RowScale row_scale(const QuantizeRowsArgs& a, const RowSums& s, uint32_t row, bool writes) {
    RowScale k;
    k.zero = s.bad != 0 || s.top == 0.0;
    k.top = s.top;
    k.r = k.zero ? 0.0 : 127.0 / s.top;
    k.r32 = (float)k.r;
    k.exact = s.top < 1e-30 || s.top > 1e30;
    if (writes) {
        double f = s.top / 127.0;
        if (NORM) f /= sqrt(s.ss / (double)a.dim + (double)a.eps);
        a.scales[row] = s.bad ? __uint_as_float(0x7fc00000u) : s.top == 0.0 ? 0.0f : (float)f;
    }
    return k;
}

// Eight elements to integers. In f32, y, r and their product are each off by 2^-24 of them: 2.3e-5 of a step
// at 127 steps, so that the nearest whole number is the one of 64 bits unless a half is within 5e-5.
template <bool NORM>
__device__ __forceinline__ u32x2 round8(const RowScale& k, const float (&v)[8], const float (&w)[8]) {
    u32x2 o{0u, 0u};
    if (k.zero) return o;
    int n[8];
    bool near = k.exact;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = (NORM ? v[i] * w[i] : v[i]) * k.r32, q = rintf(t);
        near = near || fabsf(fabsf(t - q) - 0.5f) < 5e-5f;
        n[i] = (int)q;
    }
    if (near) {
#pragma unroll
        for (int i = 0; i < 8; i++) n[i] = round127(NORM ? (double)v[i] * (double)w[i] : (double)v[i], k.r, k.top);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) o[i / 4] |= ((uint32_t)n[i] & 0xffu) << (8 * (i % 4));
    return o;
}

// TPR threads a row, eight elements a thread and piece, NV pieces held from the sums to the rounding.
template <uint32_t TPR>
constexpr uint32_t row_threads() { return TPR > kRowThreads ? TPR : kRowThreads; }
template <uint32_t XT, bool NORM, uint32_t TPR, uint32_t NV>
__global__ void __launch_bounds__(row_threads<TPR>()) quantize_rows_kernel(QuantizeRowsArgs a) {
    constexpr uint32_t XS = XT == kGgmlF32 ? 4u : 2u, PER = row_threads<TPR>() / TPR;
    const uint32_t t = threadIdx.x % TPR;
    for (uint64_t row = (uint64_t)blockIdx.x * PER + threadIdx.x / TPR; row < a.rows; row += (uint64_t)gridDim.x * PER) {
        const uint8_t* const x = (const uint8_t*)a.x + row * a.x_stride * XS;
        Eight<XT> e[NV];
        float v[8], w[8];
        RowSums s{0.0, 0.0, 0u};
        // the norm's weights are held where that leaves rows enough on their way, and read twice, from L2, where
        // the pieces are more (8192 x 4096 f32: held 31.4 us, read twice 33.4; one row 4.0, 4.15)
        constexpr bool HELD = NORM && NV <= 2u;
        Eight<kGgmlF32> held[HELD ? NV : 1u];
        auto weights = [&](uint32_t c, uint32_t k) {
            if constexpr (HELD) {
                held[c].values(w);
            } else if constexpr (NORM) {
                Eight<kGgmlF32> n;
                n.load(a.norm + k);
                n.values(w);
            }
        };
#pragma unroll
        for (uint32_t c = 0; c < NV; c++) {
            const uint32_t k = 8u * (t + TPR * c);
            if (k < a.dim) {
                e[c].load(x + (uint64_t)k * XS);
                if constexpr (HELD) held[c].load(a.norm + k);
            }
        }
#pragma unroll
        for (uint32_t c = 0; c < NV; c++) {
            const uint32_t k = 8u * (t + TPR * c);
            if (k < a.dim) {
                weights(c, k);
                e[c].values(v);
                add8<NORM>(s, v, w);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        s = row_sums<TPR>(s);
        const RowScale sc = row_scale<NORM>(a, s, (uint32_t)row, t == 0);
        int8_t* const q = a.q + row * a.q_stride;
#pragma unroll
        for (uint32_t c = 0; c < NV; c++) {
            const uint32_t k = 8u * (t + TPR * c);
            if (k < a.dim) {
                weights(c, k);
                e[c].values(v);
                *(u32x2*)(q + k) = round8<NORM>(sc, v, w);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// Rows too long for the registers: read twice, a workgroup a row.
template <uint32_t XT, bool NORM>
__global__ void __launch_bounds__(kRowThreads) quantize_long_rows_kernel(QuantizeRowsArgs a) {
    constexpr uint32_t XS = XT == kGgmlF32 ? 4u : 2u;
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint8_t* const x = (const uint8_t*)a.x + (uint64_t)row * a.x_stride * XS;
        RowSums s{0.0, 0.0, 0u};
        float v[8], w[8];
        auto at = [&](uint32_t k) {
            Eight<XT> e;
            e.load(x + (uint64_t)k * XS);
            e.values(v);
            if constexpr (NORM) {
                Eight<kGgmlF32> n;
                n.load(a.norm + k);
                n.values(w);
            }
        };
        for (uint32_t k = 8u * threadIdx.x; k < a.dim; k += 8u * kRowThreads) {
            at(k);
            add8<NORM>(s, v, w);
        }
        s = row_sums<kRowThreads>(s);
        const RowScale sc = row_scale<NORM>(a, s, row, threadIdx.x == 0);
        int8_t* const q = a.q + (uint64_t)row * a.q_stride;
        for (uint32_t k = 8u * threadIdx.x; k < a.dim; k += 8u * kRowThreads) {
            at(k);
            *(u32x2*)(q + k) = round8<NORM>(sc, v, w);
        }
    }
}

template <uint32_t XT, bool NORM>
hipError_t launch_rows(const QuantizeRowsArgs& a, int num_cus, hipStream_t st) {
    const uint32_t most = (uint32_t)num_cus * 8u;
    auto go = [&](auto kernel, uint32_t per, uint32_t threads = kRowThreads) {
        const uint32_t wgs = (a.rows + per - 1u) / per;
        hipLaunchKernelGGL(kernel, dim3(wgs < most ? wgs : most), dim3(threads), 0, st, a);
        return hipGetLastError();
    };
    if (a.dim <= 512u) return go(quantize_rows_kernel<XT, NORM, 64, 1>, 4);
    if (a.dim <= 1024u) return go(quantize_rows_kernel<XT, NORM, 64, 2>, 4);
    if (a.dim <= 2048u) return go(quantize_rows_kernel<XT, NORM, 256, 1>, 1);
    if (a.dim <= 4096u) return go(quantize_rows_kernel<XT, NORM, 256, 2>, 1);
    if (a.dim <= 8192u) return go(quantize_rows_kernel<XT, NORM, 256, 4>, 1);
    if (a.dim <= 16384u) return go(quantize_rows_kernel<XT, NORM, 512, 4>, 1, 512);
    return go(quantize_long_rows_kernel<XT, NORM>, 1);
}

}  // namespace

hipError_t launch_quantize_rows_i8(const QuantizeRowsArgs& a, uint32_t xtype, int num_cus, hipStream_t st) {
    if (xtype == kGgmlF32) return a.norm ? launch_rows<kGgmlF32, true>(a, num_cus, st) : launch_rows<kGgmlF32, false>(a, num_cus, st);
    if (xtype == kGgmlF16) return a.norm ? launch_rows<kGgmlF16, true>(a, num_cus, st) : launch_rows<kGgmlF16, false>(a, num_cus, st);
    return a.norm ? launch_rows<kGgmlBF16, true>(a, num_cus, st) : launch_rows<kGgmlBF16, false>(a, num_cus, st);
}

}  // namespace llmr
