// MXFP4 values in registers, shared by the kernels that read them (mxfp4.hip states the format).
#pragma once
#include "mma.h"

namespace lumen {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// the factor 2^(s - 127) of scale byte s as the scaled conversions take it: they read the exponent field alone, 0 as 2^-127, 255
// as NaN
__device__ __forceinline__ float mx_scale(unsigned s) { return __uint_as_float(s << 23); }

// the same of one of four scale bytes, which turning `by` = 9 + 8 x its number to the right takes there; the other bytes go
// where nothing is read
__device__ __forceinline__ float mx_scale_of(unsigned s4, int by) { return __uint_as_float(__builtin_amdgcn_alignbit(s4, s4, by)); }

// the 16-bit values of 8 codes: exact in bf16; in fp16 as rounded to it (from 2^-24 on exact, infinite beyond 65504)
template <typename T> __device__ __forceinline__ uint4 unfold(unsigned c, float scale);
template <> __device__ __forceinline__ uint4 unfold<bf16>(unsigned c, float scale) {
  return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3)));
}
template <> __device__ __forceinline__ uint4 unfold<fp16>(unsigned c, float scale) {
  return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3)));
}

}  // namespace lumen
