// y = x w^T + bias of few 16-bit rows and an MXFP4 weight [N, K]: a stream of the weight.
//
// A workgroup takes XR rows of x and 16 RT columns; its NW waves split k and every wave streams its share of both through a
// ring of its own in LDS, D stages of KS k, filled by LDS-DMA.  No barrier stands in the loop: a wave waits for its own stages by a
// counted vmcnt.  The waves' sums meet in LDS at the end, in wave order.
//  * The weight's 4-bit rows become 16-bit fragments in registers, by the scaled conversions, between the reads and the products.
//  * x comes from L2 once per workgroup, 4 to 16 times the weight's bytes: the columns of a workgroup are as many as make one round
//    of workgroups.
#include "mx_tile.h"

using namespace lumen;
using mx::TileArgs;

namespace {

template <int XR, int RT, int NW, int D, int KS>
struct Ring {
  static constexpr int MT = XR < 16 ? 1 : XR / 16;       // fragments of x (of fewer than 16 rows: read again, never stored)
  static constexpr int NH = KS / 32;                     // products along a stage
  static constexpr int XB = XR * KS * 2, XP = XB / 1024; // bytes and DMA pieces of x in a stage
  static constexpr int WP = KS == 128 ? RT : (RT + 1) / 2, WB = WP * 1024;
  static constexpr int SP = (RT + 3) / 4, SB = XB + WB + SP * 256, G = XP + WP + SP;
  static constexpr int PART = RT * MT * 1024;            // a wave's sums
  static constexpr int LDS = NW * D * SB > NW * PART ? NW * D * SB : NW * PART;
  static_assert(XB % 1024 == 0 && LDS <= mx::kLds && D >= 2 && G * (D - 1) < 64, "ring");
};

template <typename T, int XR, int RT, int NW, int D, int KS>
__global__ void __launch_bounds__(64 * NW, 1) rows_kernel(const TileArgs a) {
  using S = Ring<XR, RT, NW, D, KS>;
  constexpr int MT = S::MT, XP = S::XP, WP = S::WP, SP = S::SP, NH = S::NH, XB = S::XB, WB = S::WB, G = S::G;
  constexpr int CH = KS / 8, RP = 64 / CH;               // 16-byte chunks of a row of x in a stage; rows of a piece
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = tile::unit_of(blockIdx.x, gridDim.x);
  const int tm = tile % a.tiles_m, tn = tile / a.tiles_m;                // the row groups of a column tile share an XCD
  const int m0 = tm * XR, n0 = tn * 16 * RT;
  char* ring = lds + wid * D * S::SB;
  const unsigned ring0 = __builtin_amdgcn_readfirstlane(mx::lds_addr(ring));
  const int steps = (a.K + KS - 1) / KS, t0 = steps * wid / NW, nk = steps * (wid + 1) / NW - t0;
  const char* xb = (const char*)a.x + (long long)m0 * a.ldx * 2;
  const long long wp = (long long)a.N * 64, sp = (long long)a.N * 4;
  // a lane's place in the pieces; chunk c of row r of x lies at c ^ (r & 15) (KS 64: c ^ (r / 2 & 7))
  unsigned offx[XP], offw[WP], offs[SP];
  const int cx = KS == 128 ? (lane & 15) : (lane & 7), rx = lane / CH;
  auto swz = [](int r) { return KS == 128 ? r & 15 : (r >> 1) & 7; };
#pragma unroll
  for (int q = 0; q < XP; ++q) {
    const int r = RP * q + rx;
    offx[q] = (unsigned)min(r, a.M - m0 - 1) * (unsigned)(2 * a.ldx) + 16 * (cx ^ swz(r));
  }
#pragma unroll
  for (int q = 0; q < WP; ++q)
    offw[q] = KS == 128 ? (unsigned)min(n0 + 16 * q + (lane >> 2), a.N - 1) * 64u + 16 * (lane & 3)
                        : (unsigned)min(n0 + 32 * q + (lane >> 1), a.N - 1) * 64u + 16 * ((lane ^ lane >> 4) & 1);
#pragma unroll
  for (int q = 0; q < SP; ++q) offs[q] = (unsigned)min(n0 + 64 * q + lane, a.N - 1) * 4u;
  const int tail = a.K - KS * (steps - 1);               // values of x in the last stage
  auto issue = [&](int i) __attribute__((always_inline)) {               // the wave's stage i
    const int t = t0 + i;
    const bool last = t == steps - 1;
    const unsigned d = ring0 + i % D * S::SB;
    const char* xs = xb + (long long)t * (2 * KS);
    const char* ws = KS == 128 ? (const char*)a.codes + t * wp : (const char*)a.codes + (t >> 1) * wp + (t & 1) * 32;
    const char* ss = (const char*)a.scales + (KS == 128 ? t : t >> 1) * sp;
#pragma unroll
    for (int q = 0; q < WP; ++q) tile::dma16(ws, offw[q], __builtin_amdgcn_readfirstlane(d + XB + q * 1024));
#pragma unroll
    for (int q = 0; q < SP; ++q) mx::dma4(ss, offs[q], __builtin_amdgcn_readfirstlane(d + XB + WB + q * 256));
#pragma unroll
    for (int q = 0; q < XP; ++q) {
      const int c = cx ^ swz(RP * q + rx);
      tile::dma16(xs, offx[q] - (last && 8 * c >= tail ? 16 * c : 0), __builtin_amdgcn_readfirstlane(d + q * 1024));
    }
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
    if (t == steps - 1 && tail < KS) {                   // what lies beyond k: zeros
#pragma unroll
      for (int q = 0; q < XP; ++q)
        if (8 * (cx ^ swz(RP * q + rx)) >= tail) *reinterpret_cast<uint4*>(img + q * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
    }
    unsigned sc[RT], raw[RT][NH];
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      sc[u] = *reinterpret_cast<const unsigned*>(img + XB + WB + (16 * u + lr) * 4);
      if constexpr (KS == 128) {                         // block lg of the lane's row
        const uint4 v = *reinterpret_cast<const uint4*>(img + XB + u * 1024 + lr * 64 + lg * 16);
        raw[u][0] = v.x, raw[u][1] = v.y, raw[u][NH - 2] = v.z, raw[u][NH - 1] = v.w;
      } else {
#pragma unroll
        for (int h = 0; h < NH; ++h)
          raw[u][h] = *reinterpret_cast<const unsigned*>(img + XB + u * 512 + lr * 32 + (((h ^ lr >> 3) & 1) << 4) + lg * 4);
      }
    }
    // KS 128: lane (lr, lg) multiplies k 32 lg + 8 h .. + 7 in step h; 64: k 32 h + 8 lg ..
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      uint4 b[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int r = (16 * j + lr) & (XR - 1), c = KS == 128 ? 4 * lg + h : 4 * h + lg;
        b[j] = *reinterpret_cast<const uint4*>(img + r * (2 * KS) + ((c ^ swz(r)) << 4));
      }
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        const int byte = KS == 128 ? lg : 2 * (t & 1) + h;
        const uint4 w = unfold<T>(raw[u][h], mx_scale((sc[u] >> (8 * byte)) & 255u));
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[u][j] = Mfma<T>::run(w, b[j], acc[u][j]);
      }
    }
  }
  // the waves' sums, over the rings
  tile::done_reading();
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(lds + wid * S::PART + (i * MT + j) * 1024 + lane * 16) = acc[i][j];
  __syncthreads();
  for (int q = wid; q < RT * MT; q += NW) {
    f32x4 v = *reinterpret_cast<const f32x4*>(lds + q * 1024 + lane * 16);
#pragma unroll
    for (int w = 1; w < NW; ++w) v += *reinterpret_cast<const f32x4*>(lds + w * S::PART + q * 1024 + lane * 16);
    const int i = q / MT, r = 16 * (q - i * MT) + lr, m = m0 + r;
    if (r < XR && m < a.M) mx::put<T>(a, m, n0 + 16 * i + 4 * lg, false, v, v);
  }
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
  if (!mx::plan(a, N, xr, 16 * rt, grid)) return hipErrorInvalidValue;
  switch (10 * xr + rt) {
#define GO(XR, RT, NW, D, KS)                                                                  \
  case 10 * XR + RT:                                                                           \
    if (dt == kBF16) rows_kernel<bf16, XR, RT, NW, D, KS><<<grid, 64 * NW, 0, st>>>(a);        \
    else rows_kernel<fp16, XR, RT, NW, D, KS><<<grid, 64 * NW, 0, st>>>(a);                    \
    break;
    GO(4, 1, 8, 8, 128) GO(4, 2, 8, 6, 128) GO(4, 3, 8, 4, 128) GO(4, 4, 8, 3, 128) GO(4, 6, 8, 2, 128) GO(4, 8, 4, 4, 128)
    GO(16, 1, 8, 3, 128) GO(16, 2, 8, 3, 128) GO(16, 3, 8, 2, 128) GO(16, 4, 8, 2, 128) GO(16, 6, 4, 3, 128) GO(16, 8, 4, 3, 128)
    GO(32, 1, 4, 4, 128) GO(32, 2, 4, 3, 128) GO(32, 3, 4, 3, 128) GO(32, 4, 4, 3, 128) GO(32, 6, 4, 2, 128) GO(32, 8, 4, 4, 64)
    GO(64, 1, 4, 4, 64) GO(64, 2, 4, 4, 64) GO(64, 3, 4, 3, 64) GO(64, 4, 4, 3, 64) GO(64, 6, 4, 3, 64) GO(64, 8, 4, 3, 64)
#undef GO
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // extern "C"
