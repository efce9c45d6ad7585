// mx4_values.h - the 16-bit values of a cache in 4 bits: E2M1 numbers times their block's power of two.
#pragma once

#include "llmr_device.h"
#include "llmr_internal.h"

namespace llmr {

// A block's power of two from its byte (255: NaN comes out of values8).
__device__ __forceinline__ float power4(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight numbers (a dword) times a power of two, as 16-bit values: exact where the type has them.
template <uint32_t T>
__device__ __forceinline__ u32x4 values8(uint32_t w, float s) {
    u32x4 o;
    if constexpr (T == kGgmlBF16) {
        o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
        o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
        o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
        o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    } else {
        o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
        o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
        o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
        o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
    }
    return o;
}

}  // namespace llmr
