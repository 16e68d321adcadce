// What the matrix-core attention kernels share (prefill.hip, range_prefill.hip, range_attend.hip): operand types, packed
// bf16 rounding, copies from memory into LDS and the transposing LDS read.
#pragma once

#include "common.h"

namespace attnlab {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2v_t __attribute__((ext_vector_type(2)));

// two fp32 -> packed bf16 pair, round to nearest even (gfx950 converts in hardware: v_cvt_pk_bf16_f32)
typedef __bf16 bf16x2v_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16x2(float x, float y) {
    const bf16x2v_t v = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, v);
}

// 16 bytes per lane from global memory straight into LDS: the wave's 64 lanes fill the 1 KB at `lds` in lane order.
__device__ __forceinline__ void load_lds16(const uint16_t* src, uint16_t* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// The same from a buffer of `bytes` bytes at `base` (wave-uniform), lane l from byte offset `off`; zeros past the end.
__device__ __forceinline__ void load_lds16_buf(const uint16_t* base, uint32_t bytes, uint32_t off, uint16_t* lds) {
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, (int)bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, (int)off, 0, 0, 0);
}

// the larger of x over lanes l and l ^ 32 (v_permlane32_swap, no LDS round trip)
__device__ __forceinline__ float max_xor32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// the larger of x over lanes l and l ^ 16
__device__ __forceinline__ float max_xor16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Transposing LDS read (ds_read_b64_tr_b16): each 16 lanes read a 4 x 16 matrix of 16-bit elements, lane 4 e + j the
// elements 4 j .. 4 j + 3 of row e; lane i receives column i.
typedef short s16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2v_t read_tr16(const char* lds) {
    return __builtin_bit_cast(u32x2v_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                            (__attribute__((address_space(3))) s16x4_t*)lds));
}

// The same of 8-bit elements (ds_read_b64_tr_b8): each 16 lanes read an 8 x 16 matrix of bytes, lane 2 e + j the bytes
// 8 j .. 8 j + 7 of row e; lane i receives column i.
typedef int s32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2v_t read_tr8(const char* lds) {
    return __builtin_bit_cast(u32x2v_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                            (__attribute__((address_space(3))) s32x2_t*)lds));
}

}  // namespace attnlab
