// Quantised KV rows: what a code stands for, and how it becomes a matrix
// instruction's operand.
//
// A row of D values is held as D 8-bit codes and one fp32 scale:
//   amax  = max(max |x|, 2^-100)
//   scale = amax / Q,  code = nearest-even(x * (Q / amax)),  value = code * scale
// with Q = 448 (e4m3, its largest value) or 127 (int8, symmetric).  Both
// quotients are IEEE divisions and the product is one fp32 multiply, so the
// codes are a pure function of the row.  The floor 2^-100 keeps Q / amax
// finite and makes an all-zero row codes 0 at a finite scale.  A row that
// holds an infinity or a NaN has no amax: it is stored as codes 0 with scale
// NaN and reads back as NaN in every element, so the damage stays visible.
#pragma once

#include <cuda_fp8.h>

#include "qf_common.cuh"

namespace qf {

template <int FMT>
__device__ __forceinline__ float code_top() {
    return FMT == QF_CACHE_E4M3 ? 448.f : 127.f;
}

// Four codes (a 32-bit word) as two fp16x2 registers, exact: {c0, c1}, {c2, c3}.
// int8: the byte c + 128 under the high byte 0x64 is the fp16 number
// 1024 + (c + 128); subtracting 1152 leaves c.
template <int FMT>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (FMT == QF_CACHE_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        lo = Packed<__half>::sub(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u);
        hi = Packed<__half>::sub(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u);
    }
}

// Four codes as floats.
template <int FMT>
__device__ __forceinline__ void codes_to_float(uint32_t w, float* f) {
    uint32_t lo, hi;
    codes_to_f16<FMT>(w, lo, hi);
    f[0] = Packed<__half>::lo(lo);
    f[1] = Packed<__half>::hi(lo);
    f[2] = Packed<__half>::lo(hi);
    f[3] = Packed<__half>::hi(hi);
}

template <int FMT>
__device__ __forceinline__ float code_to_float(uint8_t c) {
    float f[4];
    codes_to_float<FMT>(c, f);
    return f[0];
}

// The codes of four already scaled values, in one word (value 0 lowest).
template <int FMT>
__device__ __forceinline__ uint32_t float_to_codes(float a, float b, float c, float d) {
    if constexpr (FMT == QF_CACHE_E4M3) {
        uint16_t lo, hi;  // saturating: a product one rounding above 448 stays 448
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)lo | ((uint32_t)hi << 16);
    } else {
        const int i0 = __float2int_rn(a), i1 = __float2int_rn(b), i2 = __float2int_rn(c),
                  i3 = __float2int_rn(d);
        return (uint32_t)(i0 & 255) | ((uint32_t)(i1 & 255) << 8) | ((uint32_t)(i2 & 255) << 16) |
               ((uint32_t)(i3 & 255) << 24);
    }
}

// A row's scale and the factor its values are multiplied by, from the largest
// |x| as fp32 bits (an unsigned maximum, in which a NaN is above an infinity
// and both are above every finite value).
template <int FMT>
__device__ __forceinline__ void row_scale(uint32_t amax_bits, float& scale, float& factor) {
    if (amax_bits >= 0x7f800000u) {
        scale = __int_as_float(0x7fc00000);
        factor = 0.f;  // the codes are zeroed by the caller (0 * inf is NaN)
        return;
    }
    const float amax = fmaxf(__uint_as_float(amax_bits), 7.888609052210118e-31f);  // 2^-100
    scale = __fdiv_rn(amax, code_top<FMT>());
    factor = __fdiv_rn(code_top<FMT>(), amax);
}

}  // namespace qf
