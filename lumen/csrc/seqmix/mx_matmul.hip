// y = x w^T + bias, both in MXFP4, on tiles (mx_loop.h).
#include "mx_tile.h"

using namespace lumen;
using mx::TileArgs;

namespace {

template <typename T, int NI, int MJ, int WN>
__global__ void __launch_bounds__(256, 1) matmul_kernel(const TileArgs a) {
  using S = mx::Shape4<NI, MJ, WN>;
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  tile::tile_at(tile::unit_of(blockIdx.x, gridDim.x), a.tiles_m, a.tiles_n, a.group, tm, tn);
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  auto column = [&](int r) { return (unsigned)min(n0 + r / (16 * NI) * (16 * NI) + tile::colperm<NI>(r % (16 * NI)), a.N - 1); };
  auto row = [&](int r) { return (unsigned)min(m0 + r, a.M - 1); };
  unsigned offx[S::PX], offw[S::PW];
#pragma unroll
  for (int q = 0; q < S::PX; ++q) offx[q] = row((wid + 4 * q) % S::NX * 16 + (lane >> 2)) * 64u + 16 * (lane & 3);
#pragma unroll
  for (int q = 0; q < S::PW; ++q) offw[q] = column((wid + 4 * q) % S::NW * 16 + (lane >> 2)) * 64u + 16 * (lane & 3);
  const mx::Walk4 walk{(const char*)a.x, (const char*)a.xs, (const char*)a.codes, (const char*)a.scales, (long long)a.M * 64,
                       (long long)a.M * 4, (long long)a.N * 64, (long long)a.N * 4, (a.K + 127) / 128};
  f32x4 acc[NI][MJ];
  mx::products4<NI, MJ, WN>(lds, walk, offx, row(min(64 * wid + lane, S::BM - 1)) * 4u, offw, column(min(64 * wid + lane, S::BN - 1)) * 4u, acc);
  mx::put_all<T, NI, MJ>(a, acc, m0 + 16 * MJ * (wid / WN), n0 + 16 * NI * (wid % WN));
}

}  // namespace

extern "C" {

// y [M, N] = x w^T + bias, x [M, K] and w [N, K] in MXFP4, y 16-bit or fp32; tiles of 32 mj x 32 ni
hipError_t sm_mx_matmul(int dt, const void* xc, const void* xs, const void* codes, const void* scales, const void* bias, void* y,
                        int M, int N, int K, int mj, int ni, hipStream_t st) {
  if (!mx::sizes_ok(M, N, K) || ((uintptr_t)xc | (uintptr_t)xs | (uintptr_t)codes | (uintptr_t)scales) % 16 ||
      (dt != kF16 && dt != kBF16 && dt != kF32))
    return hipErrorInvalidValue;
  TileArgs a{xc, 0, xs, codes, scales, bias, y, M, N, K, 0, 0, 0, 0, mx::store_width(y, N, dt == kF32 ? 4 : 2)};
  int grid;
  if (!mx::plan(a, N, 32 * mj, 32 * ni, grid)) return hipErrorInvalidValue;
  switch (10 * mj + ni) {
#define GO(MJ, NI)                                                                     \
  case 10 * MJ + NI:                                                                   \
    if (dt == kBF16) matmul_kernel<bf16, NI, MJ, 2><<<grid, 256, 0, st>>>(a);          \
    else if (dt == kF16) matmul_kernel<fp16, NI, MJ, 2><<<grid, 256, 0, st>>>(a);      \
    else matmul_kernel<float, NI, MJ, 2><<<grid, 256, 0, st>>>(a);                     \
    break;
    GO(1, 1) GO(1, 2) GO(1, 4) GO(1, 8) GO(2, 1) GO(2, 2) GO(2, 4) GO(2, 8) GO(4, 2) GO(4, 4) GO(4, 8) GO(8, 4) GO(8, 8)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // extern "C"
