// int8.hip - rows to 8-bit integers with a scale each (llmr_quantize_rows_i8).
#include "llmr_device.h"
#include "llmr_internal.h"

// every rounding that the definitions name is one
#pragma clang fp contract(off)

namespace llmr {
namespace {

// Eight elements from x on, as f32.
template <uint32_t XT>
__device__ __forceinline__ void load8(const uint8_t* x, float (&v)[8]) {
    if constexpr (XT == kGgmlF32) {
        const f32x4 a = *(const f32x4*)x, b = *(const f32x4*)(x + 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    } else {
        const u32x4 w = *(const u32x4*)x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t u = w[i];
            if constexpr (XT == kGgmlBF16) {
                v[2 * i] = __uint_as_float(u << 16);
                v[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
            } else {
                const f16x2 h = __builtin_bit_cast(f16x2, u);
                v[2 * i] = (float)h.x;
                v[2 * i + 1] = (float)h.y;
            }
        }
    }
}

constexpr uint32_t kRowThreads = 256;

// 127 y / a to the nearest whole number, ties to even; r = 127 / a. Where y r is next to a half, the
// half is compared with exactly (f16 and bf16 rows do have elements there).
__device__ __forceinline__ int round127(double y, double r, double a) {
    const double v = y * r, q = rint(v);
    int n = (int)q;
    if (fabs(fabs(v - q) - 0.5) < 1e-9) {
        const double k = floor(fabs(v)), d = fma(254.0, fabs(y), -(2.0 * k + 1.0) * a);
        const int lo = (int)k;
        const int m = d > 0.0 ? lo + 1 : d < 0.0 ? lo : lo + (lo & 1);
        n = v < 0.0 ? -m : m;
    }
    return n;
}

// One row a workgroup at a time, eight elements a thread.
template <uint32_t XT, bool NORM>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(QuantizeRowsArgs a) {
    constexpr uint32_t XS = XT == kGgmlF32 ? 4u : 2u;
    __shared__ double red[2][kRowThreads / 64];
    __shared__ uint32_t red_bad[kRowThreads / 64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint8_t* const x = (const uint8_t*)a.x + (uint64_t)row * a.x_stride * XS;
        double top = 0.0, ss = 0.0;
        uint32_t bad = 0;
        for (uint32_t k = 8u * tid; k < a.dim; k += 8u * kRowThreads) {
            float v[8], w[8];
            load8<XT>(x + (uint64_t)k * XS, v);
            if (NORM) load8<kGgmlF32>((const uint8_t*)(a.norm + k), w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const double y = NORM ? (double)v[i] * (double)w[i] : (double)v[i];
                top = fmax(top, fabs(y));
                if (!(fabs(y) < (double)INFINITY)) bad = 1u;
                if (NORM) ss += (double)v[i] * (double)v[i];
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            top = fmax(top, __shfl_xor(top, o, 64));
            if (NORM) ss += __shfl_xor(ss, o, 64);
        }
        bad = __builtin_amdgcn_ballot_w64(bad != 0) != 0 ? 1u : 0u;
        if (lane == 0) {
            red[0][wave] = top;
            red[1][wave] = ss;
            red_bad[wave] = bad;
        }
        __syncthreads();
        top = fmax(fmax(red[0][0], red[0][1]), fmax(red[0][2], red[0][3]));
        ss = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
        bad = red_bad[0] | red_bad[1] | red_bad[2] | red_bad[3];
        __syncthreads();
        const bool zero = bad != 0 || top == 0.0;
        const double r = zero ? 0.0 : 127.0 / top;
        if (tid == 0) {
            double s = top / 127.0;
            if (NORM) s /= sqrt(ss / (double)a.dim + (double)a.eps);
            a.scales[row] = bad ? __uint_as_float(0x7fc00000u) : top == 0.0 ? 0.0f : (float)s;
        }
        int8_t* const q = a.q + (uint64_t)row * a.q_stride;
        for (uint32_t k = 8u * tid; k < a.dim; k += 8u * kRowThreads) {
            float v[8], w[8];
            load8<XT>(x + (uint64_t)k * XS, v);
            if (NORM) load8<kGgmlF32>((const uint8_t*)(a.norm + k), w);
            u32x2 o{0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const double y = NORM ? (double)v[i] * (double)w[i] : (double)v[i];
                const int n = zero ? 0 : round127(y, r, top);
                o[i / 4] |= ((uint32_t)n & 0xffu) << (8 * (i % 4));
            }
            *(u32x2*)(q + k) = o;
        }
    }
}

}  // namespace

hipError_t launch_quantize_rows_i8(const QuantizeRowsArgs& a, uint32_t xtype, int num_cus, hipStream_t st) {
    const uint32_t grid = a.rows < (uint32_t)num_cus * 8u ? a.rows : (uint32_t)num_cus * 8u;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(kRowThreads), 0, st, a); };
    if (xtype == kGgmlF32) a.norm ? go(quantize_rows_kernel<kGgmlF32, true>) : go(quantize_rows_kernel<kGgmlF32, false>);
    else if (xtype == kGgmlF16) a.norm ? go(quantize_rows_kernel<kGgmlF16, true>) : go(quantize_rows_kernel<kGgmlF16, false>);
    else a.norm ? go(quantize_rows_kernel<kGgmlBF16, true>) : go(quantize_rows_kernel<kGgmlBF16, false>);
    return hipGetLastError();
}

}  // namespace llmr
