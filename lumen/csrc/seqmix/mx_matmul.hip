// y = x w^T + bias, both in MXFP4: y[m][n] = sum over blocks b of 2^(e[m][b] + f[n][b]) sum over k in b of c[m][k] d[n][k], on the scaled
// matrix instructions, which take a block of 32 codes and its scale byte from every lane: 16 x 16 x 128 a product, exact but for the fp32 sums.
//
// On tiles (mx_loop.h) a stage is a panel.  256 x 256: 64 products of 16 cycles a wave between 32 LDS reads, 16 shifts and 10 DMA pieces; a
// stage alone on the chip takes 0.61 us, 0.43 being the products' and 0.39 its 34 KB of DMA, on all CUs 0.80 (products alone, with random
// codes: 6.4 PFLOP/s, with zeros 9.8: power).  Six tiles by rounds, as in mx_linear.hip (us, 256 x 128 / 256 x 192 / 256 x 256:
// 1021 x 12288 x 4096 48 / 32 / 33, 4096 x 22016 x 4096 268 / 229 / 210 = 3.52 PFLOP/s; 128 x 128 / 128 x 192 / 256 x 128: 2048 x 2048 x 5632 22 / 26 / 31,
// 509 x 12288 x 4096 31 / 23 / 26).
// Few results: below.
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

// Few results: a workgroup takes XR rows and 16 RT columns, its four waves split k, each in a ring of its own (seqmix/mx_rows.hip); a
// stage is a panel.  Bound by bytes: a CU takes 97 B/ns from L2, and 64 x 128 results are 13 KB a panel for 32 products.  The interleaved
// loop of the tiles brings nothing here (64 x 22016 x 4096 13.9 -> 14.6 us, 1021 x 2048 x 5632 12.6 -> 12.7).  1 x 4096 x 4096 4.4 us, 48 x
// 12288 x 4096 9.4 = 2.8 TB/s of weight; against tiles 509 x 4096 x 4096 11 (256 x 128: 23), 1021 x 2048 x 5632 12.9 (30).
template <int XR, int RT, int D>
struct Ring {
  static constexpr int NW = 4, MT = XR / 16, XB = MT * 1024, WB = RT * 1024, SX = (MT + 3) / 4, SW = (RT + 3) / 4;
  static constexpr int SB = XB + WB + (SX + SW) * 256, G = MT + RT + SX + SW, PART = RT * MT * 1024;
  static constexpr int LDS = NW * D * SB > NW * PART ? NW * D * SB : NW * PART;
  static_assert(XR % 16 == 0 && LDS <= mx::kLds && D >= 2 && G * (D - 1) < 64, "ring");
};

template <typename T, int XR, int RT, int D>
__global__ void __launch_bounds__(256, 1) rows_matmul_kernel(const TileArgs a) {
  using S = Ring<XR, RT, D>;
  constexpr int NW = S::NW, MT = S::MT, SX = S::SX, SW = S::SW, XB = S::XB, WB = S::WB, G = S::G;
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;                                            // (the row groups of a column tile share an XCD)
  tile::tile_at(tile::unit_of(blockIdx.x, gridDim.x), a.tiles_m, a.tiles_n, a.group, tm, tn);
  const int m0 = tm * XR, n0 = tn * 16 * RT;
  char* ring = lds + wid * D * S::SB;
  const unsigned ring0 = __builtin_amdgcn_readfirstlane(mx::lds_addr(ring));
  const int steps = (a.K + 127) / 128, t0 = steps * wid / NW, nk = steps * (wid + 1) / NW - t0;
  const long long xp = (long long)a.M * 64, xsp = (long long)a.M * 4, wp = (long long)a.N * 64, sp = (long long)a.N * 4;
  auto row = [&](int r) { return (unsigned)min(m0 + r, a.M - 1); };
  auto column = [&](int r) { return (unsigned)min(n0 + r, a.N - 1); };
  unsigned offx[MT], offw[RT], offxs[SX], offs[SW];
#pragma unroll
  for (int q = 0; q < MT; ++q) offx[q] = row(16 * q + (lane >> 2)) * 64u + 16 * (lane & 3);
#pragma unroll
  for (int q = 0; q < RT; ++q) offw[q] = column(16 * q + (lane >> 2)) * 64u + 16 * (lane & 3);
#pragma unroll
  for (int q = 0; q < SX; ++q) offxs[q] = row(64 * q + lane) * 4u;
#pragma unroll
  for (int q = 0; q < SW; ++q) offs[q] = column(64 * q + lane) * 4u;
  auto issue = [&](int i) __attribute__((always_inline)) {
    const int t = t0 + i;
    const unsigned d = ring0 + i % D * S::SB;
#pragma unroll
    for (int q = 0; q < RT; ++q) tile::dma16((const char*)a.codes + t * wp, offw[q], __builtin_amdgcn_readfirstlane(d + XB + q * 1024));
#pragma unroll
    for (int q = 0; q < SW; ++q) mx::dma4((const char*)a.scales + t * sp, offs[q], __builtin_amdgcn_readfirstlane(d + XB + WB + (SX + q) * 256));
#pragma unroll
    for (int q = 0; q < SX; ++q) mx::dma4((const char*)a.xs + t * xsp, offxs[q], __builtin_amdgcn_readfirstlane(d + XB + WB + q * 256));
#pragma unroll
    for (int q = 0; q < MT; ++q) tile::dma16((const char*)a.x + t * xp, offx[q], __builtin_amdgcn_readfirstlane(d + q * 1024));
  };
  f32x4 acc[RT][MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D - 1; ++i)
    if (i < nk) issue(i);
  for (int i = 0; i < nk; ++i) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the fragments of stage i - 1 have been read: its slot may be filled again)
    if (i + D - 1 < nk) issue(i + D - 1);
    tile::wait_stages<D - 1, G>(nk - 1 - i);             // stage i has arrived
    asm volatile("" ::: "memory");
    const char* img = ring + i % D * S::SB;
    uint4 x[MT];
    unsigned sx[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      x[j] = *reinterpret_cast<const uint4*>(img + (16 * j + lr) * 64 + lg * 16);
      sx[j] = *reinterpret_cast<const unsigned*>(img + XB + WB + (16 * j + lr) * 4) >> (8 * lg);
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const uint4 w = *reinterpret_cast<const uint4*>(img + XB + (16 * u + lr) * 64 + lg * 16);
      const unsigned sw = *reinterpret_cast<const unsigned*>(img + XB + WB + SX * 256 + (16 * u + lr) * 4) >> (8 * lg);
#pragma unroll
      for (int j = 0; j < MT; ++j) mx::mfma4<false>(acc[u][j], w, x[j], sw, sx[j]);
    }
  }
  mx::sum_waves<T, RT, MT, NW>(a, lds, acc, m0, n0);
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
    GO(4, 4) GO(4, 6) GO(6, 4) GO(8, 4) GO(8, 6) GO(8, 8)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

// the same of few results: xr rows x 16 rt columns a workgroup
hipError_t sm_mx_rows_matmul(int dt, const void* xc, const void* xs, const void* codes, const void* scales, const void* bias, void* y,
                             int M, int N, int K, int xr, int rt, hipStream_t st) {
  if (!mx::sizes_ok(M, N, K) || ((uintptr_t)xc | (uintptr_t)xs | (uintptr_t)codes | (uintptr_t)scales) % 16 ||
      (dt != kF16 && dt != kBF16 && dt != kF32))
    return hipErrorInvalidValue;
  TileArgs a{xc, 0, xs, codes, scales, bias, y, M, N, K, 0, 0, 0, 0, mx::store_width(y, N, dt == kF32 ? 4 : 2)};
  int grid;
  if (!mx::plan(a, N, xr, 16 * rt, grid, 8)) return hipErrorInvalidValue;
  switch (10 * xr + rt) {
#define GO(XR, RT, D)                                                                  \
  case 10 * XR + RT:                                                                   \
    if (dt == kBF16) rows_matmul_kernel<bf16, XR, RT, D><<<grid, 256, 0, st>>>(a);     \
    else if (dt == kF16) rows_matmul_kernel<fp16, XR, RT, D><<<grid, 256, 0, st>>>(a); \
    else rows_matmul_kernel<float, XR, RT, D><<<grid, 256, 0, st>>>(a);                \
    break;
    GO(16, 1, 8) GO(16, 2, 8) GO(16, 4, 6) GO(16, 6, 5) GO(16, 8, 4)
    GO(32, 1, 8) GO(32, 2, 8) GO(32, 4, 6) GO(32, 6, 4) GO(32, 8, 3)
    GO(64, 1, 6) GO(64, 2, 5) GO(64, 3, 5) GO(64, 4, 4) GO(64, 6, 3) GO(64, 8, 3)
    GO(128, 4, 3)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // extern "C"
