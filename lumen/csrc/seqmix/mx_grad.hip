// dx = dy w of 16-bit rows and an MXFP4 weight, on tiles (mx_loop.h).
#include "mx_tile.h"

using namespace lumen;
using mx::TileArgs;

namespace {

template <typename T, int MJ, int WN>
__global__ void __launch_bounds__(256, 1) grad_kernel(const TileArgs a) {
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
                      wp, sp, nk, a.Nx - 64 * (nk - 1), left};
  f32x4 acc[8][MJ];
  mx::products<T, 8, MJ, WN, true>(lds, walk, offx, offw, as + 4 * lane, lastw, as + 4 * min(lane, left - 1), acc);
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

// Few results: a workgroup takes XR rows of dy and one panel of columns, its NW waves split the sum over w's rows (seqmix/mx_rows.hip has
// the ring); a wave's stage is 64 of them.
template <int XR, int NW, int D>
struct Ring {
  static constexpr int MT = XR / 16, XB = XR * 128, XP = XB / 1024, SB = XB + 4096 + 256, G = XP + 5, PART = 8 * MT * 1024;
  static constexpr int LDS = NW * D * SB > NW * PART ? NW * D * SB : NW * PART;
  static_assert(XR % 16 == 0 && LDS <= mx::kLds && D >= 2 && G * (D - 1) < 64, "ring");
};

template <typename T, int XR, int NW, int D>
__global__ void __launch_bounds__(64 * NW, 1) rows_grad_kernel(const TileArgs a) {
  using S = Ring<XR, NW, D>;
  constexpr int MT = S::MT, XP = S::XP, XB = S::XB, G = S::G;
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = tile::unit_of(blockIdx.x, gridDim.x);
  const int tm = tile % a.tiles_m, panel = tile / a.tiles_m;
  const int m0 = tm * XR;
  char* ring = lds + wid * D * S::SB;
  const unsigned ring0 = __builtin_amdgcn_readfirstlane(mx::lds_addr(ring));
  const int steps = (a.N + 63) / 64, t0 = steps * wid / NW, nk = steps * (wid + 1) / NW - t0;
  const int tail = a.Nx - 64 * (steps - 1), left = a.N - 64 * (steps - 1);
  const char* xb = (const char*)a.x + (long long)m0 * a.ldx * 2;
  const char* wb = (const char*)a.codes + (long long)panel * a.N * 64;
  const char* sb = (const char*)a.scales + (long long)panel * a.N * 4;
  unsigned offx[XP], offw[4], lastw[4];
#pragma unroll
  for (int q = 0; q < XP; ++q) {
    const int r = 8 * q + (lane >> 3);
    offx[q] = (unsigned)min(r, a.M - m0 - 1) * (unsigned)(2 * a.ldx) + 16 * ((lane & 7) ^ tile::swz(r));
  }
  auto row = [&](int q) {                                // of w, that the lane brings with piece q: rows 8 apart lie side by side
    const int pos = 16 * (q & 1) + (lane >> 2);
    return 32 * (q >> 1) + ((pos & 3) << 3 | pos >> 2);
  };
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    offw[q] = 64 * row(q) + 16 * (lane & 3);
    lastw[q] = 64 * min(row(q), left - 1) + 16 * (lane & 3);
  }
  auto issue = [&](int i) __attribute__((always_inline)) {
    const int t = t0 + i;
    const bool last = t == steps - 1;
    const unsigned d = ring0 + i % D * S::SB;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      tile::dma16(wb + (long long)t * 4096, last ? lastw[q] : offw[q], __builtin_amdgcn_readfirstlane(d + XB + q * 1024));
    mx::dma4(sb + (long long)t * 256, 4 * (last ? min(lane, left - 1) : lane), __builtin_amdgcn_readfirstlane(d + XB + 4096));
#pragma unroll
    for (int q = 0; q < XP; ++q) {
      const int c = (lane & 7) ^ tile::swz(8 * q + (lane >> 3));
      tile::dma16(xb + (long long)t * 128, offx[q] - (last && 8 * c >= tail ? 16 * c : 0), __builtin_amdgcn_readfirstlane(d + q * 1024));
    }
  };
  f32x4 acc[8][MT];
#pragma unroll
  for (int i = 0; i < 8; ++i)
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
    char* img = ring + i % D * S::SB;
    if (t0 + i == steps - 1 && left < 64) {              // what lies beyond w's rows: zeros
#pragma unroll
      for (int q = 0; q < XP; ++q)
        if (8 * ((lane & 7) ^ tile::swz(8 * q + (lane >> 3))) >= tail) *reinterpret_cast<uint4*>(img + q * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (row(q) >= left) *reinterpret_cast<uint4*>(img + XB + q * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
      if (lane >= left) *reinterpret_cast<unsigned*>(img + XB + 4096 + lane * 4) = 0;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned raw[8], fw[8][4];
      float sc[8];
      uint4 fx[MT];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        raw[r] = *reinterpret_cast<const unsigned*>(img + XB + h * 2048 + (4 * r + lg) * 64 + lr * 4);
        sc[r] = mx_scale(*reinterpret_cast<const unsigned char*>(img + XB + 4096 + (32 * h + 8 * lg + r) * 4 + (lr >> 2)));
      }
#pragma unroll
      for (int j = 0; j < MT; ++j)
        fx[j] = *reinterpret_cast<const uint4*>(img + (16 * j + lr) * 128 + (((4 * h + lg) ^ tile::swz(lr)) << 4));
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint2 v0 = mx::columns<T, 0>(raw[2 * u], raw[2 * u + 1], sc[2 * u], sc[2 * u + 1]);
        const uint2 v1 = mx::columns<T, 1>(raw[2 * u], raw[2 * u + 1], sc[2 * u], sc[2 * u + 1]);
        const uint2 v2 = mx::columns<T, 2>(raw[2 * u], raw[2 * u + 1], sc[2 * u], sc[2 * u + 1]);
        const uint2 v3 = mx::columns<T, 3>(raw[2 * u], raw[2 * u + 1], sc[2 * u], sc[2 * u + 1]);
        fw[0][u] = v0.x, fw[1][u] = v0.y, fw[2][u] = v1.x, fw[3][u] = v1.y;
        fw[4][u] = v2.x, fw[5][u] = v2.y, fw[6][u] = v3.x, fw[7][u] = v3.y;
      }
      mx::ready();
#pragma unroll
      for (int i8 = 0; i8 < 8; ++i8) {
        const uint4 w = make_uint4(fw[i8][0], fw[i8][1], fw[i8][2], fw[i8][3]);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i8][j] = Mfma<T>::run(w, fx[j], acc[i8][j]);
      }
    }
  }
  // the waves' sums, over the rings
  tile::done_reading();
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(lds + wid * S::PART + (i * MT + j) * 1024 + lane * 16) = acc[i][j];
  __syncthreads();
  for (int q = wid; q < 4 * MT; q += NW) {               // row 4 lg + e of fragment i: column 8 (4 lg + e) + i
    const int j = q >> 2, e = q & 3, m = m0 + 16 * j + lr, k = 128 * panel + 32 * lg + 8 * e;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[i] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) r[i] += *reinterpret_cast<const float*>(lds + w * S::PART + (i * MT + j) * 1024 + lane * 16 + 4 * e);
    }
    if (m < a.M && k < a.K) store8((T*)a.y + (long long)m * a.K + k, r);
  }
}

}  // namespace

extern "C" {

// dx [M, K] = dy [M, N] w; dy 16-bit at ldy, its rows readable (and zero) up to a multiple of 8 values; tiles of 64 mj / wn x 128 wn
hipError_t sm_mx_grad(int dt, const void* dy, long long ldy, const void* codes, const void* scales, void* dx, int M, int N, int K, int mj,
                      int wn, hipStream_t st) {
  const int Nx = (N + 7) / 8 * 8;
  if (!mx::sizes_ok(M, N, K) || ldy < Nx || ldy % 8 || ldy > (1 << 22) || ((uintptr_t)dx | (uintptr_t)dy | (uintptr_t)codes | (uintptr_t)scales) % 16 ||
      (dt != kF16 && dt != kBF16))
    return hipErrorInvalidValue;
  TileArgs a{dy, ldy, nullptr, codes, scales, nullptr, dx, M, N, K, Nx, 0, 0, 0, 8};
  int grid;
  if (!mx::plan(a, K, 64 * mj / wn, 128 * wn, grid)) return hipErrorInvalidValue;
  switch (10 * mj + wn) {
#define GO(MJ, WN)                                                                     \
  case 10 * MJ + WN:                                                                   \
    if (dt == kBF16) grad_kernel<bf16, MJ, WN><<<grid, 256, 0, st>>>(a);               \
    else grad_kernel<fp16, MJ, WN><<<grid, 256, 0, st>>>(a);                           \
    break;
    GO(4, 2) GO(8, 2)
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
  if (!mx::plan(a, K, xr, 128, grid)) return hipErrorInvalidValue;
  switch (xr) {
#define GO(XR, NW, D)                                                                          \
  case XR:                                                                                     \
    if (dt == kBF16) rows_grad_kernel<bf16, XR, NW, D><<<grid, 64 * NW, 0, st>>>(a);           \
    else rows_grad_kernel<fp16, XR, NW, D><<<grid, 64 * NW, 0, st>>>(a);                       \
    break;
    GO(16, 8, 3) GO(32, 4, 4) GO(64, 4, 3)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // extern "C"
