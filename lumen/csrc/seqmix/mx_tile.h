// Arguments, stores and checks that the products with MXFP4 weights on tiles share (mx_loop.h).
#pragma once
#include "mx_loop.h"

namespace lumen {
namespace mx {

struct TileArgs {
  const void* x; long long ldx;          // rows (in MXFP4: codes)
  const void* xs;                        // scales of rows in MXFP4
  const void *codes, *scales;            // of the weight [N, K]
  const void* bias;
  void* y;
  int M, N, K, Nx;                       // Nx: columns of dy that can be read (N up to a multiple of 8, zeros behind N)
  int tiles_m, tiles_n, group, wide;     // wide: values a store can take, 8, 4 or 1
};

// columns n .. n + 3 (u) and n + 4 .. n + 7 (v, `two`) of row m
template <typename T>
__device__ __forceinline__ void put(const TileArgs& a, int m, int n, bool two, const f32x4& u, const f32x4& v) {
  T* p = (T*)a.y + (long long)m * a.N + n;
  float r[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = u[e], r[4 + e] = v[e];
  if (a.bias) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < (two ? 8 : 4)) r[e] += to_f32(((const T*)a.bias)[min(n + e, a.N - 1)]);
  }
  if constexpr (sizeof(T) == 2) {
    if (a.wide == 8 && two && n + 8 <= a.N) {
      store8(p, r);
      return;
    }
    if (a.wide >= 4) {
      if (n < a.N) *reinterpret_cast<uint2*>(p) = make_uint2(pk2<T>(r[0], r[1]), pk2<T>(r[2], r[3]));
      if (two && n + 4 < a.N) *reinterpret_cast<uint2*>(p + 4) = make_uint2(pk2<T>(r[4], r[5]), pk2<T>(r[6], r[7]));
      return;
    }
  } else if (a.wide >= 4) {
    if (n < a.N) *reinterpret_cast<float4*>(p) = make_float4(r[0], r[1], r[2], r[3]);
    if (two && n + 4 < a.N) *reinterpret_cast<float4*>(p + 4) = make_float4(r[4], r[5], r[6], r[7]);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < (two ? 8 : 4) && n + e < a.N) p[e] = from_f32<T>(r[e]);
}

// the results of a wave, whose fragments of w stand for columns as tile::colperm says
template <typename T, int NI, int MJ>
__device__ __forceinline__ void put_all(const TileArgs& a, f32x4 (&acc)[NI][MJ], int m0, int n0) {
  static_assert(NI % 2 == 0, "columns in pairs of fragments");
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const int m = m0 + 16 * j + lr;
#pragma unroll
    for (int i = 0; i < NI; i += 2) {
      hold<kNamed<NI, MJ>>(acc[i][j]);
      hold<kNamed<NI, MJ>>(acc[i + 1][j]);
      if (m < a.M) put<T>(a, m, n0 + 16 * i + 8 * lg, true, acc[i][j], acc[i + 1][j]);
    }
  }
}

// the sums of NW waves that split k, 16 MT rows by 16 RT columns each, meet in LDS in the waves' order: the same bits every time
template <typename T, int RT, int MT, int NW>
__device__ __forceinline__ void sum_waves(const TileArgs& a, char* lds, f32x4 (&acc)[RT][MT], int m0, int n0) {
  constexpr int PART = RT * MT * 1024;
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  tile::done_reading();                                  // (every wave's ring: the sums lie over them)
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(lds + wid * PART + (i * MT + j) * 1024 + lane * 16) = acc[i][j];
  __syncthreads();
  for (int q = wid; q < RT * MT; q += NW) {
    f32x4 v = *reinterpret_cast<const f32x4*>(lds + q * 1024 + lane * 16);
#pragma unroll
    for (int w = 1; w < NW; ++w) v += *reinterpret_cast<const f32x4*>(lds + w * PART + q * 1024 + lane * 16);
    const int i = q / MT, m = m0 + 16 * (q - i * MT) + lr;
    if (m < a.M) put<T>(a, m, n0 + 16 * i + 4 * lg, false, v, v);
  }
}

inline bool sizes_ok(int M, int N, int K) {
  return M >= 1 && N >= 1 && M <= (1 << 24) && N <= (1 << 24) && K >= 8 && K % 8 == 0 && K <= (1 << 23);
}

// Grid of BM x BN tiles over M x C results; false: too many.  Tiles go to an XCD by `most` groups of rows or, where there are more, by 4
// (64 x 64 and 64 x 128 results: 1021 x 1024 x 4096 14.1 -> 12.0 us, 1021 x 4096 x 4096 38.5 -> 37.3; 5 groups by 4 rather 35.2 -> 36.3).
inline bool plan(TileArgs& a, int C, int BM, int BN, int& grid, int most = 4) {
  const long long tm = (a.M + BM - 1LL) / BM, tn = (C + BN - 1LL) / BN;
  if (tm * tn >= (1LL << 24)) return false;
  a.tiles_m = (int)tm, a.tiles_n = (int)tn, a.group = (int)(tm <= most ? tm : 4);
  grid = (int)(tm * tn);
  return true;
}

inline int store_width(const void* y, int N, int size) { return N % 8 == 0 && (uintptr_t)y % 16 == 0 ? 8 : N % 4 == 0 && (uintptr_t)y % (4 * size) == 0 ? 4 : 1; }

}  // namespace mx
}  // namespace lumen
