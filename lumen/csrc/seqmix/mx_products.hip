// Products with MXFP4 weights, a wave per 16 x 16 tile, operands straight from memory.
#include "mx.h"

using namespace lumen;

namespace {

struct MxArgs {
  const void* x; long long ldx;          // 16-bit rows, or codes of the rows
  const unsigned char* xs;               // their scales
  const unsigned char *codes, *scales;   // of the weight [N, Kp]
  const void* bias;
  void* y;
  int M, N, K, Kp;
};

// y [M, N] = x [M, K] w^T + bias
template <typename T>
__global__ void __launch_bounds__(64) linear_kernel(const MxArgs a) {
  const int lane = threadIdx.x, lr = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const long long n = min(n0 + lr, a.N - 1), m = min(m0 + lr, a.M - 1);
  const T* x = (const T*)a.x + m * a.ldx;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.K; k += 32) {
    const unsigned c = *reinterpret_cast<const unsigned*>(a.codes + n * (a.Kp / 2) + k / 2 + 4 * lg);
    const uint4 w = unfold<T>(c, mx_scale(a.scales[n * (a.Kp / 32) + k / 32]));
    acc = Mfma<T>::run(w, *reinterpret_cast<const uint4*>(x + k + 8 * lg), acc);
  }
  if (m0 + lr >= a.M) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = n0 + 4 * lg + e;
    if (c < a.N) ((T*)a.y)[m * a.N + c] = from_f32<T>(acc[e] + (a.bias ? to_f32(((const T*)a.bias)[c]) : 0.f));
  }
}

// dx [M, K] = dy [M, N] w; x: dy
template <typename T>
__global__ void __launch_bounds__(64) grad_kernel(const MxArgs a) {
  const int lane = threadIdx.x, lr = lane & 15, lg = lane >> 4;
  const int k0 = blockIdx.x * 16, m0 = blockIdx.y * 16, k = k0 + lr;   // (K % 32 == 0)
  const long long m = min(m0 + lr, a.M - 1);
  const T* dy = (const T*)a.x + m * a.ldx;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int n0 = 0; n0 < a.N; n0 += 32) {
    unsigned short w[8], d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = n0 + 8 * lg + j;
      w[j] = d[j] = 0;
      if (n < a.N) {
        const unsigned c = a.codes[(long long)n * (a.Kp / 2) + k / 2] >> (4 * (k & 1));
        w[j] = (unsigned short)unfold<T>(c, mx_scale(a.scales[(long long)n * (a.Kp / 32) + k / 32])).x;
        d[j] = __builtin_bit_cast(unsigned short, dy[n]);
      }
    }
    uint4 wv, dv;
    __builtin_memcpy(&wv, w, 16);
    __builtin_memcpy(&dv, d, 16);
    acc = Mfma<T>::run(wv, dv, acc);
  }
  if (m0 + lr >= a.M) return;
  *reinterpret_cast<uint2*>((T*)a.y + m * a.K + k0 + 4 * lg) = make_uint2(pk2<T>(acc[0], acc[1]), pk2<T>(acc[2], acc[3]));
}

// y [M, N] = x w^T + bias of two MXFP4 operands
template <typename T>
__global__ void __launch_bounds__(64) matmul_kernel(const MxArgs a) {
  const int lane = threadIdx.x, lr = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const long long n = min(n0 + lr, a.N - 1), m = min(m0 + lr, a.M - 1);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < a.Kp; k += 128) {
    const uint4 w = *reinterpret_cast<const uint4*>(a.codes + n * (a.Kp / 2) + k / 2 + 16 * lg);
    const uint4 x = *reinterpret_cast<const uint4*>((const unsigned char*)a.x + m * (a.Kp / 2) + k / 2 + 16 * lg);
    const int sw = a.scales[n * (a.Kp / 32) + k / 32 + lg], sx = a.xs[m * (a.Kp / 32) + k / 32 + lg];
    const i32x8 A = {(int)w.x, (int)w.y, (int)w.z, (int)w.w}, B = {(int)x.x, (int)x.y, (int)x.z, (int)x.w};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc, 4, 4, 0, sw, 0, sx);
  }
  if (m0 + lr >= a.M) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = n0 + 4 * lg + e;
    if (c < a.N) ((T*)a.y)[m * a.N + c] = from_f32<T>(acc[e] + (a.bias ? to_f32(((const T*)a.bias)[c]) : 0.f));
  }
}

bool sizes_ok(int M, int N, int K) {
  return M >= 1 && N >= 1 && K >= 32 && K % 32 == 0 && K <= (1 << 23) && (M + 15) / 16 <= 65535;
}

}  // namespace

extern "C" {

hipError_t sm_mx_linear(int dt, const void* x, long long ldx, const void* codes, const void* scales, const void* bias, void* y,
                        int M, int N, int K, hipStream_t st) {
  if (!sizes_ok(M, N, K) || ldx < K || ldx % 8 || ((uintptr_t)x | (uintptr_t)codes) % 16 || (dt != kF16 && dt != kBF16))
    return hipErrorInvalidValue;
  const MxArgs a{x, ldx, nullptr, (const unsigned char*)codes, (const unsigned char*)scales, bias, y, M, N, K, (K + 127) / 128 * 128};
  const dim3 grid((N + 15) / 16, (M + 15) / 16);
  if (dt == kBF16) linear_kernel<bf16><<<grid, 64, 0, st>>>(a);
  else linear_kernel<fp16><<<grid, 64, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t sm_mx_grad(int dt, const void* dy, long long ldy, const void* codes, const void* scales, void* dx, int M, int N, int K,
                      hipStream_t st) {
  if (!sizes_ok(M, N, K) || ldy < N || ((uintptr_t)dx | (uintptr_t)codes) % 16 || (dt != kF16 && dt != kBF16)) return hipErrorInvalidValue;
  const MxArgs a{dy, ldy, nullptr, (const unsigned char*)codes, (const unsigned char*)scales, nullptr, dx, M, N, K, (K + 127) / 128 * 128};
  const dim3 grid(K / 16, (M + 15) / 16);
  if (dt == kBF16) grad_kernel<bf16><<<grid, 64, 0, st>>>(a);
  else grad_kernel<fp16><<<grid, 64, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t sm_mx_matmul(int dt, const void* xc, const void* xs, const void* codes, const void* scales, const void* bias, void* y,
                        int M, int N, int K, hipStream_t st) {
  if (!sizes_ok(M, N, K) || ((uintptr_t)xc | (uintptr_t)codes) % 16 || (dt != kF16 && dt != kBF16 && dt != kF32))
    return hipErrorInvalidValue;
  const MxArgs a{xc, 0, (const unsigned char*)xs, (const unsigned char*)codes, (const unsigned char*)scales, bias, y, M, N, K,
                 (K + 127) / 128 * 128};
  const dim3 grid((N + 15) / 16, (M + 15) / 16);
  if (dt == kBF16) matmul_kernel<bf16><<<grid, 64, 0, st>>>(a);
  else if (dt == kF16) matmul_kernel<fp16><<<grid, 64, 0, st>>>(a);
  else matmul_kernel<float><<<grid, 64, 0, st>>>(a);
  return hipGetLastError();
}

}  // extern "C"
