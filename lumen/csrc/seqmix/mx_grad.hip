// dx = dy w of 16-bit rows and an MXFP4 weight (mx_loop.h): dx[m][k] = sum over n of dy[m][n] c[n][k] 2^e[n][k / 32], the weight's
// values in dy's type, as the forward product has them.
//
// The sum runs over the weight's rows, which the codes do not lie along: a matrix instruction wants 8 rows' values of one column in a
// lane.  A lane takes four bytes of 8 rows, makes pairs of neighbouring columns and exchanges halves between two rows (v_perm): 4
// conversions and 4 exchanges for 8 values of two rows, where a transposed copy of the weight would cost its memory again.
// On tiles of 128, 192 or 256 rows x two panels: a stage (64 of the weight's rows) of 256 x 256 takes 1.40 us on all CUs, the vector unit's 16
// units a half beside 1.29 of the forward product.  4096 rows, weight 4096 x 11008: 282 us = 1.31 PFLOP/s on 256 rows, 305 on 192, 351 on 128;
// 2048 rows, 4096 x 4096: 63 on 128, 90 on 256.
#include "mx_tile.h"

using namespace lumen;
using mx::TileArgs;

namespace {

template <typename T, int MJ>
__global__ void __launch_bounds__(256, 1) grad_kernel(const TileArgs a) {
  constexpr int WN = 2;
  using S = mx::Shape<8, MJ, WN, true>;
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  tile::tile_at(tile::unit_of(blockIdx.x, gridDim.x), a.tiles_m, a.tiles_n, a.group, tm, tn);
  const int m0 = tm * S::BM, panel = tn * WN, panels = (a.K + 127) / 128;
  const int nk = (a.N + 63) / 64, left = a.N - 64 * (nk - 1);
  const long long wp = (long long)a.N * 64, sp = (long long)a.N * 4;
  unsigned offx[S::PX], offw[S::PW], lastw[S::PW];
#pragma unroll
  for (int q = 0; q < S::PX; ++q) {
    const int r = 8 * (wid + 4 * q) + (lane >> 3);
    offx[q] = (unsigned)min(r, a.M - m0 - 1) * (unsigned)(2 * a.ldx) + 16 * ((lane & 7) ^ tile::swz(r));
  }
#pragma unroll
  for (int q = 0; q < S::PW; ++q) {
    const int pc = (wid + 4 * q) % S::NW, pos = 16 * (pc & 1) + (lane >> 2);
    const int n = 32 * ((pc >> 1) & 1) + ((pos & 3) << 3 | pos >> 2);
    const unsigned at = (unsigned)min(pc >> 2, panels - 1 - panel) * (unsigned)wp + 16 * (lane & 3);
    offw[q] = at + 64 * n;
    lastw[q] = at + 64 * min(n, left - 1);
  }
  const unsigned as = (unsigned)min(wid % WN, panels - 1 - panel) * (unsigned)sp;
  const mx::Walk walk{(const char*)a.x + (long long)m0 * a.ldx * 2, (const char*)a.codes + panel * wp, (const char*)a.scales + panel * sp,
                      wp, sp, nk, a.Nx - 64 * (nk - 1), left, 0};
  const unsigned offs[1] = {as + 4 * lane}, lasts[1] = {as + 4 * min(lane, left - 1)};
  f32x4 acc[8][MJ];
  mx::products<T, 8, MJ, WN, true>(lds, walk, offx, offw, offs, lastw, lasts, acc);
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const int m = m0 + 16 * MJ * (wid / WN) + 16 * j + lr;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx::hold<mx::kNamed<8, MJ>>(acc[i][j]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {                        // row 4 lg + e of fragment i: column 8 (4 lg + e) + i
      const int k = 128 * (panel + wid % WN) + 32 * lg + 8 * e;
      const float r[8] = {acc[0][j][e], acc[1][j][e], acc[2][j][e], acc[3][j][e], acc[4][j][e], acc[5][j][e], acc[6][j][e], acc[7][j][e]};
      if (m < a.M && k < a.K) store8((T*)a.y + (long long)m * a.K + k, r);
    }
  }
}

// Few results: a workgroup takes 16 MT rows of dy and one panel of columns, its NW waves split the sum over w's rows, each in a ring of its
// own.  16 rows leave a SIMD room for two waves.  Us: 17 rows, 4096 x 4096 11.6 on 16 (14.7 on 32), 200 rows 16.1 on 32 (19.7 on 64), 509 rows
// 21.6 on 64 (29.3 on 32, on tiles of 128 x 256 57) = 0.79 PFLOP/s.  The sum is not split among workgroups, so few rows leave CUs idle: 17
// rows x 4096 columns are 64 workgroups, and up to some 300 rows a call takes 3 - 6 times what its bytes do.
template <typename T, int MT, int NW>
__global__ void __launch_bounds__(64 * NW, 1) rows_grad_kernel(const TileArgs a) {
  using S = mx::Shape<8, MT, -NW, true>;
  constexpr int XR = 16 * MT, PART = 8 * MT * 1024;
  __shared__ __attribute__((aligned(16))) char lds[NW * (S::LDS > PART ? S::LDS : PART)];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, panel;
  tile::tile_at(tile::unit_of(blockIdx.x, gridDim.x), a.tiles_m, a.tiles_n, a.group, tm, panel);
  const int m0 = tm * XR;
  const int steps = (a.N + 63) / 64, t0 = steps * wid / NW, nk = steps * (wid + 1) / NW - t0;
  f32x4 acc[8][MT];
  if (nk > 0) {
    const bool last = t0 + nk == steps;
    const int tail = last ? a.Nx - 64 * (steps - 1) : 64, left = last ? a.N - 64 * (steps - 1) : 64;
    unsigned offx[S::PX], offw[4], lastw[4];
#pragma unroll
    for (int q = 0; q < S::PX; ++q) {
      const int r = 8 * q + (lane >> 3);
      offx[q] = (unsigned)min(r, a.M - m0 - 1) * (unsigned)(2 * a.ldx) + 16 * ((lane & 7) ^ tile::swz(r));
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int pos = 16 * (q & 1) + (lane >> 2), n = 32 * (q >> 1) + ((pos & 3) << 3 | pos >> 2);
      offw[q] = 64 * n + 16 * (lane & 3);
      lastw[q] = 64 * min(n, left - 1) + 16 * (lane & 3);
    }
    const unsigned offs[1] = {4u * lane}, lasts[1] = {4u * min(lane, left - 1)};
    const mx::Walk walk{(const char*)a.x + (long long)m0 * a.ldx * 2 + (long long)t0 * 128, (const char*)a.codes + (long long)panel * a.N * 64 + (long long)t0 * 4096,
                        (const char*)a.scales + (long long)panel * a.N * 4 + (long long)t0 * 256, 0, 0, nk, tail, left, 0};
    mx::products<T, 8, MT, -NW, true>(lds + wid * S::LDS, walk, offx, offw, offs, lastw, lasts, acc);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // the waves' sums, over the rings
  tile::done_reading();
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(lds + wid * PART + (i * MT + j) * 1024 + lane * 16) = acc[i][j];
  __syncthreads();
  for (int q = wid; q < 4 * MT; q += NW) {               // row 4 lg + e of fragment i: column 8 (4 lg + e) + i
    const int j = q >> 2, e = q & 3, m = m0 + 16 * j + lr, k = 128 * panel + 32 * lg + 8 * e;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[i] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) r[i] += *reinterpret_cast<const float*>(lds + w * PART + (i * MT + j) * 1024 + lane * 16 + 4 * e);
    }
    if (m < a.M && k < a.K) store8((T*)a.y + (long long)m * a.K + k, r);
  }
}

}  // namespace

extern "C" {

// dx [M, K] = dy [M, N] w; dy 16-bit at ldy, its rows readable (and zero) up to a multiple of 8 values; tiles of 32 mj x 256
hipError_t sm_mx_grad(int dt, const void* dy, long long ldy, const void* codes, const void* scales, void* dx, int M, int N, int K, int mj,
                      hipStream_t st) {
  const int Nx = (N + 7) / 8 * 8;
  if (!mx::sizes_ok(M, N, K) || ldy < Nx || ldy % 8 || ldy > (1 << 22) || ((uintptr_t)dx | (uintptr_t)dy | (uintptr_t)codes | (uintptr_t)scales) % 16 ||
      (dt != kF16 && dt != kBF16))
    return hipErrorInvalidValue;
  TileArgs a{dy, ldy, nullptr, codes, scales, nullptr, dx, M, N, K, Nx, 0, 0, 0, 8};
  int grid;
  if (!mx::plan(a, K, 32 * mj, 256, grid)) return hipErrorInvalidValue;
  switch (mj) {
#define GO(MJ)                                                                         \
  case MJ:                                                                             \
    if (dt == kBF16) grad_kernel<bf16, MJ><<<grid, 256, 0, st>>>(a);                   \
    else grad_kernel<fp16, MJ><<<grid, 256, 0, st>>>(a);                               \
    break;
    GO(4) GO(6) GO(8)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

// the same of few results: xr rows x 128 columns a workgroup
hipError_t sm_mx_rows_grad(int dt, const void* dy, long long ldy, const void* codes, const void* scales, void* dx, int M, int N, int K,
                           int xr, hipStream_t st) {
  const int Nx = (N + 7) / 8 * 8;
  if (!mx::sizes_ok(M, N, K) || ldy < Nx || ldy % 8 || ldy > (1 << 22) ||
      ((uintptr_t)dx | (uintptr_t)dy | (uintptr_t)codes | (uintptr_t)scales) % 16 || (dt != kF16 && dt != kBF16))
    return hipErrorInvalidValue;
  TileArgs a{dy, ldy, nullptr, codes, scales, nullptr, dx, M, N, K, Nx, 0, 0, 0, 8};
  int grid;
  if (!mx::plan(a, K, xr, 128, grid, 8)) return hipErrorInvalidValue;
  switch (xr) {
#define GO(XR, NW)                                                                             \
  case XR:                                                                                     \
    if (dt == kBF16) rows_grad_kernel<bf16, XR / 16, NW><<<grid, 64 * NW, 0, st>>>(a);         \
    else rows_grad_kernel<fp16, XR / 16, NW><<<grid, 64 * NW, 0, st>>>(a);                     \
    break;
    GO(16, 8) GO(32, 4) GO(64, 4)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // extern "C"
