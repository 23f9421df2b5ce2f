// y = x w^T + bias of few 16-bit rows and an MXFP4 weight [N, K]: a stream of the weight.
//
// A workgroup takes XR rows of x and 16 RT columns; its waves split k and every wave streams its share of both through a ring of its own
// in LDS, filled by LDS-DMA.  No barrier stands in the loop: a wave waits for its own stages by a counted vmcnt.  The waves' sums
// meet in LDS at the end, in wave order.  The weight's codes become 16-bit fragments in registers, by the scaled conversions.
//  * Up to 32 rows it is bound by the weight's bytes and by the launch: stages of 128 k, whole lines of the weight, reads in a row
//    before the products (us: 1 x 4096 x 4096 4.9, 8 x 22016 x 4096 12.0 = 4.0 TB/s of weight, 17 x 32000 x 2048 12.8).
//  * 64 rows, and 32 with 128 columns, are bound by the matrix core, the DMA and what a wave issues in turn: the tiles' loop, where each
//    stands between products, 64 k a stage (509 x 4096 x 4096 23.9 -> 20.4 us = 0.84 PFLOP/s, 64 x 22016 x 4096 22.2 -> 20.1; 32 x 12288 x
//    4096 with 48 columns rather 11.1 -> 12.4).
//  * x comes from L2 once per workgroup, 4 to 16 times the weight's bytes, so the columns of a workgroup are as many as make one
//    round of workgroups (64 x 22016 x 4096: 32 columns 33.6, 96 22.0, 128 25.0 of the first form).
//  * Where one round of such workgroups (64 x 128 results on each of 256 CUs) holds all results they beat tiles, which then leave CUs idle;
//    from the second round on tiles of 128 rows win (us, 64 x 128 here / the best tiles: 509 x 4096 x 4096 20.4 / 33.9, 800 x 4096 x 4096
//    35.6 / 34.8, 1021 x 4096 x 4096 37.9 / 35.0, 509 x 12288 x 4096 59.6 / 49.5).
#include "mx_tile.h"

using namespace lumen;
using mx::TileArgs;

namespace {

template <int XR, int RT, int NW, int D>
struct Ring {
  static constexpr int MT = XR / 16;                     // fragments of x
  static constexpr int XB = XR * 256, XP = XB / 1024;    // bytes and DMA pieces of x in a stage
  static constexpr int SP = (RT + 3) / 4, WB = RT * 1024, SB = XB + WB + SP * 256, G = XP + RT + SP;
  static constexpr int PART = RT * MT * 1024;            // a wave's sums
  static constexpr int LDS = NW * D * SB > NW * PART ? NW * D * SB : NW * PART;
  static_assert(XB % 1024 == 0 && LDS <= mx::kLds && D >= 2 && G * (D - 1) < 64, "ring");
};

template <typename T, int XR, int RT, int NW, int D>
__global__ void __launch_bounds__(64 * NW, 1) rows_kernel(const TileArgs a) {
  using S = Ring<XR, RT, NW, D>;
  constexpr int MT = S::MT, XP = S::XP, SP = S::SP, XB = S::XB, WB = S::WB, G = S::G;
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;                                            // (the row groups of a column tile share an XCD)
  tile::tile_at(tile::unit_of(blockIdx.x, gridDim.x), a.tiles_m, a.tiles_n, a.group, tm, tn);
  const int m0 = tm * XR, n0 = tn * 16 * RT;
  char* ring = lds + wid * D * S::SB;
  const unsigned ring0 = __builtin_amdgcn_readfirstlane(mx::lds_addr(ring));
  const int steps = (a.K + 127) / 128, t0 = steps * wid / NW, nk = steps * (wid + 1) / NW - t0;
  const char* xb = (const char*)a.x + (long long)m0 * a.ldx * 2;
  const long long wp = (long long)a.N * 64, sp = (long long)a.N * 4;
  // a lane's place in the pieces; chunk c of row r of x lies at c ^ (r & 15)
  unsigned offx[XP], offw[RT], offs[SP];
  auto chunk = [&](int q) { return (lane & 15) ^ ((4 * q + (lane >> 4)) & 15); };        // of x, that the lane brings with piece q
#pragma unroll
  for (int q = 0; q < XP; ++q) offx[q] = (unsigned)min(4 * q + (lane >> 4), a.M - m0 - 1) * (unsigned)(2 * a.ldx) + 16 * chunk(q);
#pragma unroll
  for (int q = 0; q < RT; ++q) offw[q] = (unsigned)min(n0 + 16 * q + (lane >> 2), a.N - 1) * 64u + 16 * (lane & 3);
#pragma unroll
  for (int q = 0; q < SP; ++q) offs[q] = (unsigned)min(n0 + 64 * q + lane, a.N - 1) * 4u;
  const int tail = a.K - 128 * (steps - 1);               // values of x in the last stage
  auto issue = [&](int i) __attribute__((always_inline)) {               // the wave's stage i
    const int t = t0 + i;
    const bool last = t == steps - 1;
    const unsigned d = ring0 + i % D * S::SB;
    const char *xs = xb + (long long)t * 256, *ws = (const char*)a.codes + t * wp, *ss = (const char*)a.scales + t * sp;
#pragma unroll
    for (int q = 0; q < RT; ++q) tile::dma16(ws, offw[q], __builtin_amdgcn_readfirstlane(d + XB + q * 1024));
#pragma unroll
    for (int q = 0; q < SP; ++q) mx::dma4(ss, offs[q], __builtin_amdgcn_readfirstlane(d + XB + WB + q * 256));
#pragma unroll
    for (int q = 0; q < XP; ++q)
      tile::dma16(xs, offx[q] - (last && 8 * chunk(q) >= tail ? 16 * chunk(q) : 0), __builtin_amdgcn_readfirstlane(d + q * 1024));
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
    // (the fragments of stage i - 1 have been read: its slot may be filled again)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (i + D - 1 < nk) issue(i + D - 1);
    tile::wait_stages<D - 1, G>(nk - 1 - i);             // stage i has arrived
    asm volatile("" ::: "memory");
    char* img = ring + i % D * S::SB;
    const int t = t0 + i;
    if (t == steps - 1 && tail < 128) {                  // what lies beyond k: zeros
#pragma unroll
      for (int q = 0; q < XP; ++q)
        if (8 * chunk(q) >= tail) *reinterpret_cast<uint4*>(img + q * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
    }
    float sc[RT];
    uint4 raw[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) {                       // block lg of the lane's row and its scale
      sc[u] = mx_scale_of(*reinterpret_cast<const unsigned*>(img + XB + WB + (16 * u + lr) * 4), 9 + 8 * lg);
      raw[u] = *reinterpret_cast<const uint4*>(img + XB + u * 1024 + lr * 64 + lg * 16);
    }
    // lane (lr, lg) multiplies k 32 lg + 8 h .. + 7 in step h
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      uint4 b[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        b[j] = *reinterpret_cast<const uint4*>(img + (16 * j + lr) * 256 + (((4 * lg + h) ^ lr) << 4));
      }
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        const uint4 w = unfold<T>(h == 0 ? raw[u].x : h == 1 ? raw[u].y : h == 2 ? raw[u].z : raw[u].w, sc[u]);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[u][j] = Mfma<T>::run(w, b[j], acc[u][j]);
      }
    }
  }
  mx::sum_waves<T, RT, MT, NW>(a, lds, acc, m0, n0);
}

// the same on the loop of the tiles (mx_loop.h), a stage 64 k
template <typename T, int RT, int MT>
__global__ void __launch_bounds__(256, 1) rows_loop_kernel(const TileArgs a) {
  using S = mx::Shape<RT, MT, -4, false>;
  constexpr int NW = 4, XR = 16 * MT, PART = RT * MT * 1024;
  __shared__ __attribute__((aligned(16))) char lds[NW * (S::LDS > PART ? S::LDS : PART)];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;                                            // (the row groups of a column tile share an XCD)
  tile::tile_at(tile::unit_of(blockIdx.x, gridDim.x), a.tiles_m, a.tiles_n, a.group, tm, tn);
  const int m0 = tm * XR, n0 = tn * 16 * RT;
  const int steps = (a.K + 63) / 64, t0 = steps * wid / NW, nk = steps * (wid + 1) / NW - t0;
  const long long wp = (long long)a.N * 64, sp = (long long)a.N * 4;
  f32x4 acc[RT][MT];
  if (nk > 0) {
    unsigned offx[S::PX], offw[S::PW], offs[S::PS];
#pragma unroll
    for (int q = 0; q < S::PX; ++q) {
      const int r = 8 * q + (lane >> 3);
      offx[q] = (unsigned)min(r, a.M - m0 - 1) * (unsigned)(2 * a.ldx) + 16 * ((lane & 7) ^ tile::swz(r));
    }
#pragma unroll
    for (int q = 0; q < S::PW; ++q) offw[q] = (unsigned)min(n0 + 32 * q + (lane >> 1), a.N - 1) * 64u + 16 * ((lane ^ lane >> 4) & 1);
#pragma unroll
    for (int q = 0; q < S::PS; ++q) offs[q] = (unsigned)min(n0 + 64 * q + lane, a.N - 1) * 4u;
    const mx::Walk walk{(const char*)a.x + (long long)m0 * a.ldx * 2 + (long long)t0 * 128, (const char*)a.codes + (t0 >> 1) * wp + (t0 & 1) * 32,
                        (const char*)a.scales + (t0 >> 1) * sp, wp, sp, nk, t0 + nk == steps ? a.K - 64 * (steps - 1) : 64, 64, t0 & 1};
    mx::products<T, RT, MT, -4, false>(lds + wid * S::LDS, walk, offx, offw, offs, offw, offs, acc);
  } else {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  mx::sum_waves<T, RT, MT, NW>(a, lds, acc, m0, n0);
}

}  // namespace

extern "C" {

// y [M, N] = x [M, K] w^T + bias (or null), x 16-bit at ldx, 16-byte aligned rows; xr rows x 16 rt columns a workgroup
hipError_t sm_mx_rows(int dt, const void* x, long long ldx, const void* codes, const void* scales, const void* bias, void* y,
                      int M, int N, int K, int xr, int rt, hipStream_t st) {
  if (!mx::sizes_ok(M, N, K) || ldx < K || ldx % 8 || ldx > (1 << 22) || ((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) % 16 ||
      (dt != kF16 && dt != kBF16))
    return hipErrorInvalidValue;
  TileArgs a{x, ldx, nullptr, codes, scales, bias, y, M, N, K, 0, 0, 0, 0, mx::store_width(y, N, 2)};
  int grid;
  if (!mx::plan(a, N, xr, 16 * rt, grid, 8)) return hipErrorInvalidValue;
  switch (10 * xr + rt) {
#define GO(XR, RT, NW, D)                                                                \
  case 10 * XR + RT:                                                                     \
    if (dt == kBF16) rows_kernel<bf16, XR, RT, NW, D><<<grid, 64 * NW, 0, st>>>(a);      \
    else rows_kernel<fp16, XR, RT, NW, D><<<grid, 64 * NW, 0, st>>>(a);                  \
    break;
    GO(16, 1, 8, 3) GO(16, 2, 8, 3) GO(16, 3, 8, 2) GO(16, 4, 8, 2) GO(16, 6, 4, 3) GO(16, 8, 4, 3)
    GO(32, 1, 4, 4) GO(32, 2, 4, 3) GO(32, 3, 4, 3) GO(32, 4, 4, 3) GO(32, 6, 4, 2)
#undef GO
#define GO(XR, RT)                                                                       \
  case 10 * XR + RT:                                                                     \
    if (dt == kBF16) rows_loop_kernel<bf16, RT, XR / 16><<<grid, 256, 0, st>>>(a);       \
    else rows_loop_kernel<fp16, RT, XR / 16><<<grid, 256, 0, st>>>(a);                   \
    break;
    GO(32, 8) GO(64, 2) GO(64, 3) GO(64, 4) GO(64, 6) GO(64, 8)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // extern "C"
