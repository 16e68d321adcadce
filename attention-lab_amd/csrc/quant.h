// The 8-bit K/V cache's element format, shared by the kernels that write it (quant.hip) and read it (range_attend.hip,
// range_prefill.hip): e4m3 codes (1 sign, 4 exponent, 3 mantissa bits; largest 448, smallest step 2^-9, 0x7f / 0xff NaN) and
// one scale 2^(x - 127) per block of positions, KV head and tensor, kept as the byte x.
//
// A scale that is a power of two keeps every conversion exact: x * 2^-e and code * 2^e round nothing in fp32 or bf16
// (a code has 4 significant bits, a bf16 8), and moving a code to a larger scale only rounds what falls below 2^-6. In
// a floating code it costs no precision either: the scale only decides which values lie among the subnormals.
#pragma once

#include "common.h"

namespace attnlab {

typedef __bf16 qbf16x2_t __attribute__((ext_vector_type(2)));
typedef float qf32x2_t __attribute__((ext_vector_type(2)));

constexpr int kQuantMinExp = 127 - 110;       // smallest scale 2^-110: the code 1 times it is a normal bf16
constexpr float kQuantLargest = 0x1.ep127f;   // larger finite values saturate here: their code times the scale is finite

__device__ __forceinline__ float scale_of(uint32_t x) { return __uint_as_float(x << 23); }          // 2^(x - 127)

// The smallest scale byte x with top <= 448 * 2^(x - 127) (448 = 1.75 * 2^8), top >= 0 finite.
__device__ __forceinline__ uint32_t scale_for(float top) {
    const uint32_t u = __float_as_uint(top);
    const int x = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(x, kQuantMinExp);
}

// Two codes (the low half of w, or its high half) times `scale` as a packed bf16 pair: exact for a power of two.
template <bool HIGH>
__device__ __forceinline__ uint32_t e4m3_to_bf16x2(uint32_t w, float scale) {
    const qbf16x2_t v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH);
    return __builtin_bit_cast(uint32_t, v);
}

// Two codes of w as floats, unscaled.
template <bool HIGH>
__device__ __forceinline__ qf32x2_t e4m3_to_f32x2(uint32_t w) { return __builtin_amdgcn_cvt_pk_f32_fp8(w, HIGH); }

// Four floats of magnitude <= 448 as four codes, round to nearest even; NaN and infinities become NaN codes.
__device__ __forceinline__ uint32_t f32_to_e4m3x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

}  // namespace attnlab
