// Microscaled 4-bit floating point (MXFP4): rows -> codes and scales, and back.
//
// A block is 32 values of a row (the last one of a row the values that are left).  Its scale is 2^e, e = floor(log2(max |x|)) - 2, kept as the byte e + 127; a value is the nearest
// of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} to x / 2^e, ties to the even code, 6 beyond.  Two values share a byte, the first in its low
// half.  Blocks that hold an infinity or a NaN get the scale byte 255, which stands for NaN; blocks of zeros the byte 0.
//  * floor(log2) is the exponent field of the largest magnitude (bit patterns of one sign compare like the numbers, NaN above all):
//    no logarithm, no rounding that could cross a power of two;
//  * x / 2^e and its rounding are the hardware's scaled conversions; over all 65536 patterns of both 16-bit types and scales from the
//    smallest to the largest they round as said above, denormals included.
// A matrix lies in panels of 128 values of its rows, the last one padded with codes and scales of zero: codes [panel][row][64 bytes],
// scales [panel][row][4 bytes].  Whatever a product reads of consecutive rows is then one run of memory, and needs no bounds in k.
#include "mx.h"

using namespace lumen;

namespace {

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));

// max |x| of 8 values as the bits of an fp32, 0x7f800000 and above where one is no finite number
template <typename T> __device__ __forceinline__ unsigned top8(const uint4 (&v)[sizeof(T) / 2]) {
  const unsigned w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
  unsigned lo = 0, hi = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo = max(lo, w[i] & 0x7fffu);
    hi = max(hi, w[i] & 0x7fff0000u);
  }
  const unsigned top = max(lo, hi >> 16);
  if constexpr (__is_same(T, bf16)) return top << 16;
  if (top >= 0x7c00u) return 0x7f800000u;
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top))));
}
template <> __device__ __forceinline__ unsigned top8<float>(const uint4 (&v)[2]) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top = max(top, max(max(v[i].x & 0x7fffffffu, v[i].y & 0x7fffffffu), max(v[i].z & 0x7fffffffu, v[i].w & 0x7fffffffu)));
  }
  return top;
}

// 8 values -> 8 codes
template <typename T> __device__ __forceinline__ unsigned codes8(const uint4 (&v)[sizeof(T) / 2], float scale) {
  unsigned c = 0;
  if constexpr (__is_same(T, float)) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[0].x), __uint_as_float(v[0].y), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[0].z), __uint_as_float(v[0].w), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[1].x), __uint_as_float(v[1].y), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[1].z), __uint_as_float(v[1].w), scale, 3);
  } else if constexpr (__is_same(T, bf16)) {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v[0].x), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v[0].y), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v[0].z), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, v[0].w), scale, 3);
  } else {
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(lumen_f16x2, v[0].x), scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(lumen_f16x2, v[0].y), scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(lumen_f16x2, v[0].z), scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(lumen_f16x2, v[0].w), scale, 3);
  }
  return c;
}

// Bound by memory.  A workgroup: 16 rows by kPan panels, 16 lanes a row of a panel, four a block; a wave writes whole lines of four rows.
template <typename T, int kPan>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, long long ldx, unsigned* __restrict__ codes,
                                                       unsigned char* __restrict__ scales, int R, int K, int panels) {
  const int r = blockIdx.x * 16 + (threadIdx.x >> 4), u = threadIdx.x & 15, p0 = blockIdx.y * kPan;
  if (r >= R) return;
  uint4 v[kPan][sizeof(T) / 2];
#pragma unroll
  for (int p = 0; p < kPan; ++p) {
    const int k = 128 * (p0 + p) + 8 * u;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      v[p][i] = k < K ? reinterpret_cast<const uint4*>(x + r * ldx + k)[i] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int p = 0; p < kPan; ++p) {
    unsigned top = top8<T>(v[p]);
    top = max(top, (unsigned)__shfl_xor((int)top, 1));
    top = max(top, (unsigned)__shfl_xor((int)top, 2));
    const bool bad = top >= 0x7f800000u;
    const int s = bad ? 255 : max((int)(top >> 23) - 2, 0);
    const unsigned c = codes8<T>(v[p], mx_scale(s));
    if (p0 + p < panels) {
      const long long row = (long long)(p0 + p) * R + r;
      codes[row * 16 + u] = bad ? 0u : c;
      if ((u & 3) == 0) scales[row * 4 + (u >> 2)] = (unsigned char)s;
    }
  }
}

template <typename T> __device__ __forceinline__ void values8(unsigned c, float scale, T* y) {
  if constexpr (__is_same(T, float)) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
    const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
    reinterpret_cast<float4*>(y)[0] = make_float4(a[0], a[1], b[0], b[1]);
    reinterpret_cast<float4*>(y)[1] = make_float4(d[0], d[1], e[0], e[1]);
  } else {
    *reinterpret_cast<uint4*>(y) = unfold<T>(c, scale);
  }
}

template <typename T, int kPan>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                         T* __restrict__ y, int R, int K, int panels) {
  const int r = blockIdx.x * 16 + (threadIdx.x >> 4), u = threadIdx.x & 15, p0 = blockIdx.y * kPan;
  if (r >= R) return;
  unsigned c[kPan], s[kPan];
#pragma unroll
  for (int p = 0; p < kPan; ++p) {
    const long long row = (long long)min(p0 + p, panels - 1) * R + r;
    c[p] = codes[row * 16 + u];
    s[p] = scales[row * 4 + (u >> 2)];
  }
#pragma unroll
  for (int p = 0; p < kPan; ++p) {
    const int k = 128 * (p0 + p) + 8 * u;
    if (k < K) values8<T>(c[p], mx_scale(s[p]), y + (long long)r * K + k);
  }
}

// workgroups for R rows, `pan` panels each
inline dim3 grid_of(int R, int panels, int pan) { return dim3((R + 15) / 16, (panels + pan - 1) / pan); }
// Panels a workgroup takes: one of few values, whose loads then start at once everywhere, two of many, where half the workgroups come
// and go (us, 1 / 2 / 4 panels: quantised 8 x 4096 2.0 / 2.0 / 2.2, 509 x 5632 3.4 / 3.6 / 4.0, 1021 x 5632 5.6 / 5.4 / 5.8, 22016 x 4096 50.0 /
// 45.5 / 47.2 = 5.0 TB/s; back to 16 bits 2.0, 3.2 / 3.4 / 3.5, 5.2 / 4.9 / 5.1, 51.0 / 48.4 / 49.6).
inline bool few(int R, int K) { return (long long)R * K <= (4 << 20); }

}  // namespace

extern "C" {

// codes [panels, R, 64], scales [panels, R, 4] of x [R, K] at ldx; K % 8 == 0, panels of 128 values, rows of x at 16-byte addresses
hipError_t sm_mx_quantize(int dt, const void* x, long long ldx, void* codes, void* scales, int R, int K, hipStream_t st) {
  const int P = (K + 127) / 128;
  if (R < 1 || R > (1 << 24) || K < 8 || K % 8 || K > (1 << 23) || ldx < K || ldx % (dt == kF32 ? 4 : 8) || (uintptr_t)x % 16 ||
      (uintptr_t)codes % 16 || (uintptr_t)scales % 4 || (dt != kF16 && dt != kBF16 && dt != kF32))
    return hipErrorInvalidValue;
  unsigned* c = (unsigned*)codes;
  unsigned char* s = (unsigned char*)scales;
#define GO(PAN)                                                                                                                     \
  if (dt == kF32) quantize_kernel<float, PAN><<<grid_of(R, P, PAN), 256, 0, st>>>((const float*)x, ldx, c, s, R, K, P);             \
  else if (dt == kBF16) quantize_kernel<bf16, PAN><<<grid_of(R, P, PAN), 256, 0, st>>>((const bf16*)x, ldx, c, s, R, K, P);         \
  else quantize_kernel<fp16, PAN><<<grid_of(R, P, PAN), 256, 0, st>>>((const fp16*)x, ldx, c, s, R, K, P);
  if (few(R, K)) { GO(1) } else { GO(2) }
#undef GO
  return hipGetLastError();
}

// y [R, K] of such codes and scales
hipError_t sm_mx_dequantize(int dt, const void* codes, const void* scales, void* y, int R, int K, hipStream_t st) {
  const int P = (K + 127) / 128;
  if (R < 1 || R > (1 << 24) || K < 8 || K % 8 || K > (1 << 23) || (uintptr_t)y % 16 || (uintptr_t)codes % 16 || (uintptr_t)scales % 4 ||
      (dt != kF16 && dt != kBF16 && dt != kF32))
    return hipErrorInvalidValue;
  const unsigned* c = (const unsigned*)codes;
  const unsigned char* s = (const unsigned char*)scales;
#define GO(PAN)                                                                                                                     \
  if (dt == kF32) dequantize_kernel<float, PAN><<<grid_of(R, P, PAN), 256, 0, st>>>(c, s, (float*)y, R, K, P);                      \
  else if (dt == kBF16) dequantize_kernel<bf16, PAN><<<grid_of(R, P, PAN), 256, 0, st>>>(c, s, (bf16*)y, R, K, P);                  \
  else dequantize_kernel<fp16, PAN><<<grid_of(R, P, PAN), 256, 0, st>>>(c, s, (fp16*)y, R, K, P);
  if (few(R, K)) { GO(1) } else { GO(2) }
#undef GO
  return hipGetLastError();
}

}  // extern "C"
