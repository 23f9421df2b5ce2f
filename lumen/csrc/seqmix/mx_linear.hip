// y = x w^T + bias of 16-bit rows and an MXFP4 weight, on tiles (mx_loop.h): y[m][n] = sum over k of x[m][k] c[n][k] 2^e[n][k / 32].
//
// The weight's values are made in x's type (exact in bf16; in fp16 rounded once: what lies below 2^-24 is lost, above 65504 infinite) and
// multiplied by the 16-bit matrix instructions with fp32 sums, so those bound it.  A stage of 64 k of the 256 x 256 tile is, for each of
// the four waves, 128 products of 16 cycles and between them 40 LDS reads, 64 conversions, 16 turned scales and 11 DMA pieces; alone on
// the chip it takes 1.07 us, 0.85 being the products', on all CUs, whose clock falls with their power, 1.25 - 1.34.
// The larger a tile, the less its products wait (columns: 128 x 128 0.48 us a stage, 256 x 128 0.77, 256 x 256 1.29 with all CUs at work),
// but whole rounds of 256 workgroups come and go, so there are six (us, 128 x 128 / 128 x 192 / 192 x 128 / 256 x 128 / 256 x 192 / 256 x 256: 2048 x
// 2048 x 5632 46 / 57 / 54 / 64 / 84 / 104, 509 x 12288 x 4096 66 / 50 / 80 / 50 / 64 / 79, 1021 x 5120 x 5120 79 / 53 / 55 / 59 / 77 / 96, 4096 x 12288 x
// 4096 - / - / - / 320 / 290 / 269).
// 4096 x 12288 x 4096 bf16: 269 us = 1.53 PFLOP/s; the library's 16-bit product of 8192^3 runs at 1.36 on the same card.
#include "mx_tile.h"

using namespace lumen;
using mx::TileArgs;

namespace {

template <typename T, int NI, int MJ, int WN>
__global__ void __launch_bounds__(256, 1) linear_kernel(const TileArgs a) {
  using S = mx::Shape<NI, MJ, WN, false>;
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  tile::tile_at(tile::unit_of(blockIdx.x, gridDim.x), a.tiles_m, a.tiles_n, a.group, tm, tn);
  const int m0 = tm * S::BM, n0 = tn * S::BN;
  auto column = [&](int r) { return min(n0 + r / (16 * NI) * (16 * NI) + tile::colperm<NI>(r % (16 * NI)), a.N - 1); };
  unsigned offx[S::PX], offw[S::PW], offs[1];
#pragma unroll
  for (int q = 0; q < S::PX; ++q) {                      // (rows past the edge read the last row: never stored)
    const int r = 8 * (wid + 4 * q) + (lane >> 3);
    offx[q] = (unsigned)min(r, a.M - m0 - 1) * (unsigned)(2 * a.ldx) + 16 * ((lane & 7) ^ tile::swz(r));
  }
#pragma unroll
  for (int q = 0; q < S::PW; ++q)
    offw[q] = (unsigned)column((wid + 4 * q) % S::NW * 32 + (lane >> 1)) * 64u + 16 * ((lane ^ lane >> 4) & 1);
  offs[0] = (unsigned)column(min(64 * wid + lane, S::BN - 1)) * 4u;
  const int nk = (a.K + 63) / 64;
  const mx::Walk walk{(const char*)a.x + (long long)m0 * a.ldx * 2, (const char*)a.codes, (const char*)a.scales, (long long)a.N * 64,
                      (long long)a.N * 4, nk, a.K - 64 * (nk - 1), 64, 0};
  f32x4 acc[NI][MJ];
  mx::products<T, NI, MJ, WN, false>(lds, walk, offx, offw, offs, offw, offs, acc);
  mx::put_all<T, NI, MJ>(a, acc, m0 + 16 * MJ * (wid / WN), n0 + 16 * NI * (wid % WN));
}

}  // namespace

extern "C" {

// y [M, N] = x [M, K] w^T + bias (or null), x 16-bit at ldx, 16-byte aligned rows; tiles of 32 mj x 32 ni
hipError_t sm_mx_linear(int dt, const void* x, long long ldx, const void* codes, const void* scales, const void* bias, void* y,
                        int M, int N, int K, int mj, int ni, hipStream_t st) {
  if (!mx::sizes_ok(M, N, K) || ldx < K || ldx % 8 || ldx > (1 << 22) || ((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) % 16 ||
      (dt != kF16 && dt != kBF16))
    return hipErrorInvalidValue;
  TileArgs a{x, ldx, nullptr, codes, scales, bias, y, M, N, K, 0, 0, 0, 0, mx::store_width(y, N, 2)};
  int grid;
  if (!mx::plan(a, N, 32 * mj, 32 * ni, grid)) return hipErrorInvalidValue;
  switch (10 * mj + ni) {
#define GO(MJ, NI)                                                                     \
  case 10 * MJ + NI:                                                                   \
    if (dt == kBF16) linear_kernel<bf16, NI, MJ, 2><<<grid, 256, 0, st>>>(a);          \
    else linear_kernel<fp16, NI, MJ, 2><<<grid, 256, 0, st>>>(a);                      \
    break;
    GO(4, 4) GO(4, 6) GO(6, 4) GO(8, 4) GO(8, 6) GO(8, 8)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // extern "C"
