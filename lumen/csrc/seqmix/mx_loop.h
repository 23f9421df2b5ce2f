// Main loops of products with MXFP4 weights, one workgroup per CU: four waves on a tile, or waves that split the sum.
//
// Rows in MXFP4 lie in panels of 128 k: codes [K / 128][rows][64 bytes], scales [K / 128][rows][4 bytes] (mxfp4.hip), so that a stage
// of a tile is one run of memory whichever product reads it.
//  * Operands come by LDS-DMA, as many stages ahead as fit into 160 KiB, under counted waits; one barrier a stage.
//  * While the matrix core multiplies one set of fragments, the next set is read and made: between two products stands at most a
//    read, a DMA or a few instructions of the vector unit, which the matrix core's 16 cycles cover.  A wave's instructions leave in
//    order, one in four cycles or more, so each one too many there is time lost: addresses move once a stage, the last stage is
//    sent for again rather than asked about, and a scale is turned into place by one instruction.
//  * 192 and more accumulators are named as accumulation registers in the products' assembly: the compiler, left to place them, moves
//    them to and fro.  It knows nothing of such products' latency, so nothing may read or move an accumulator before settle(): the
//    loops have one way round and settle before they are left.  Fewer are the compiler's.
#pragma once
#include "mx.h"
#include "../kernels/tile_loop.h"

namespace lumen {
namespace mx {

constexpr int kLds = 160 * 1024;
template <int NI, int MJ> constexpr bool kNamed = NI * MJ >= 48;

// c += a b, 16 x 16 x 32
template <typename T, bool NAMED>
__device__ __forceinline__ void mfma(f32x4& c, uint4 a, uint4 b) {
  if constexpr (NAMED) tile::mfma<T>(c, a, b);
  else c = Mfma<T>::run(a, b, c);
}
// the last products have left the matrix core
template <bool NAMED> __device__ __forceinline__ void settle() { if constexpr (NAMED) tile::settle(); }
template <bool NAMED> __device__ __forceinline__ void hold(f32x4& c) { if constexpr (NAMED) tile::hold(c); }

// LDS-DMA of 16 and 4 bytes per lane to lds + AT: three instructions, as they stand between products, where each costs its issue (with a
// stage's addresses worked out for every piece of it a tile of 256 x 256 x 11008 of 4-bit operands took 87 us, so 61)
template <int AT>
__device__ __forceinline__ void dma16(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(lds), "n"(AT) : "memory", "m0", "scc");
}
template <int AT>
__device__ __forceinline__ void dma4(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" :: "v"(off), "s"(base), "s"(lds), "n"(AT) : "memory", "m0", "scc");
}
// LDS-DMA of 4 bytes per lane
__device__ __forceinline__ void dma4(const void* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

__device__ __forceinline__ unsigned lds_addr(const char* p) {
  return (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p);
}

// f(0) ... f(N - 1), each with its number as a constant (a loop's bounds and choices by it cost the unroller too much)
template <int N> struct Int { static constexpr int value = N; };
template <int A, int B, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (A < B) {
    f(Int<A>{});
    each<A + 1, B>(f);
  }
}

// two 16-bit values of byte W of eight codes, in the place where it is written: a product may follow two instructions later
template <typename T, int W>
__device__ __forceinline__ unsigned pair(unsigned c, float scale) {
  unsigned r;
  if constexpr (__is_same(T, bf16)) {
    if constexpr (W == 0) asm volatile("v_cvt_scalef32_pk_bf16_fp4 %0, %1, %2" : "=v"(r) : "v"(c), "v"(scale));
    if constexpr (W == 1) asm volatile("v_cvt_scalef32_pk_bf16_fp4 %0, %1, %2 op_sel:[1,0,0]" : "=v"(r) : "v"(c), "v"(scale));
    if constexpr (W == 2) asm volatile("v_cvt_scalef32_pk_bf16_fp4 %0, %1, %2 op_sel:[0,1,0]" : "=v"(r) : "v"(c), "v"(scale));
    if constexpr (W == 3) asm volatile("v_cvt_scalef32_pk_bf16_fp4 %0, %1, %2 op_sel:[1,1,0]" : "=v"(r) : "v"(c), "v"(scale));
  } else {
    if constexpr (W == 0) asm volatile("v_cvt_scalef32_pk_f16_fp4 %0, %1, %2" : "=v"(r) : "v"(c), "v"(scale));
    if constexpr (W == 1) asm volatile("v_cvt_scalef32_pk_f16_fp4 %0, %1, %2 op_sel:[1,0,0]" : "=v"(r) : "v"(c), "v"(scale));
    if constexpr (W == 2) asm volatile("v_cvt_scalef32_pk_f16_fp4 %0, %1, %2 op_sel:[0,1,0]" : "=v"(r) : "v"(c), "v"(scale));
    if constexpr (W == 3) asm volatile("v_cvt_scalef32_pk_f16_fp4 %0, %1, %2 op_sel:[1,1,0]" : "=v"(r) : "v"(c), "v"(scale));
  }
  return r;
}

// what the vector unit wrote is there for the matrix core
__device__ __forceinline__ void ready() { asm volatile("s_nop 1" ::: "memory"); }

// values of byte W of two rows' codes c0 and c1, regrouped by column: x the pair (row 0, row 1) of the even column, y of the odd one
template <typename T, int W>
__device__ __forceinline__ uint2 columns(unsigned c0, unsigned c1, float s0, float s1) {
  const unsigned p = pair<T, W>(c0, s0), q = pair<T, W>(c1, s1);
  unsigned even, odd;
  asm volatile("v_perm_b32 %0, %1, %2, %3" : "=v"(even) : "v"(q), "v"(p), "s"(0x05040100u));
  asm volatile("v_perm_b32 %0, %1, %2, %3" : "=v"(odd) : "v"(q), "v"(p), "s"(0x07060302u));
  return make_uint2(even, odd);
}

// ---- 16-bit rows against 4-bit weights -------------------------------------------------------------
//
// Tiles of 16 MJ WM rows of x and 16 NI WN columns, WM x WN = 4 waves, a wave 16 MJ x 16 NI.  A stage is 64 of the summed index.
//  * GRAD false: y = x w^T.  A fragment of w is 16 of its rows by 32 k, one block a row: a lane reads four bytes, its 8 codes.
//  * GRAD true: dx = dy w, the sum runs over w's rows.  A lane takes 8 rows' codes of the 8 columns it stands for; two rows' pairs
//    are regrouped by column (v_perm), which gives 8 fragments, of columns 8 a + j for j = 0 .. 7 (a: row of the fragment).
// WN = -4 or -8: one wave's 16 MJ x 16 NI, in a ring of its own among the 4 or 8 waves of a workgroup that split the sum: no barriers.
template <int NI, int MJ, int WN, bool GRAD>
struct Shape {
  static constexpr bool OWN = WN < 0;
  static constexpr int WM = OWN ? 1 : 4 / WN, BM = 16 * MJ * WM, BN = 16 * NI * (OWN ? 1 : WN);
  static constexpr int NW = OWN ? (GRAD ? 4 : (NI + 1) / 2) : BN / 32;        // KiB of codes in a stage
  // a wave's pieces of x, codes and scales, and what lies between two of them
  static constexpr int PX = OWN ? BM / 8 : BM / 32, PW = OWN ? NW : (NW + 3) / 4, PS = OWN && !GRAD ? (NI + 3) / 4 : 1;
  static constexpr int STEP = OWN ? 1024 : 4096, PIECES = PX + PW + PS;
  static constexpr int XB = BM * 128, WB = NW * 1024, SB = XB + WB + (OWN ? 256 * PS : 1024);      // a stage: x, codes, scales
  static constexpr int FIT = kLds / ((OWN ? -WN : 1) * SB), NST = FIT < 6 ? FIT : 6, LDS = NST * SB;
  static_assert((OWN || (BM % 32 == 0 && BN % 32 == 0 && BN <= 256)) && NST >= 3 && (NST - 1) * PIECES < 64, "tile");
  static_assert(!GRAD || NI == 8, "a panel a wave");
};

struct Walk {
  const char* x;              // first row of the tile, 2-byte elements, 128 bytes a stage
  const char *w, *s;          // codes and scales: of the first stage and row 0 (GRAD: of the tile's first panel)
  long long wp, sp;           // bytes from panel to panel
  int nk, tail, tailw;        // stages; values of x in the last one (a multiple of 8); GRAD: rows of w in it
  int odd;                    // 1: the first stage is the second half of a panel
};

// acc[i][j] += products of fragments i of w and j of x.  offx[q], offw[q], offs[q]: the lane's byte offsets of its pieces; lastw, lasts: of
// those of the last stage (GRAD), whose rows from `tail` on are not w's own.
template <typename T, int NI, int MJ, int WN, bool GRAD>
__device__ __forceinline__ void products(char* lds, const Walk& a, const unsigned (&offx)[Shape<NI, MJ, WN, GRAD>::PX],
                                         const unsigned (&offw)[Shape<NI, MJ, WN, GRAD>::PW],
                                         const unsigned (&offs)[Shape<NI, MJ, WN, GRAD>::PS],
                                         const unsigned (&lastw)[Shape<NI, MJ, WN, GRAD>::PW],
                                         const unsigned (&lasts)[Shape<NI, MJ, WN, GRAD>::PS], f32x4 (&acc)[NI][MJ]) {
  using S = Shape<NI, MJ, WN, GRAD>;
  constexpr bool NAMED = kNamed<NI, MJ>, OWN = S::OWN;
  constexpr int PX = S::PX, PW = S::PW, PS = S::PS, NW = S::NW, P = S::PIECES, NST = S::NST, SB = S::SB, XB = S::XB, WB = S::WB;
  constexpr int STEP = S::STEP, P1 = (P + 1) / 2;
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = OWN ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = OWN ? 0 : wid / (OWN ? 1 : WN), wn = OWN ? 0 : wid % (OWN ? 1 : WN);
  const unsigned lds0 = lds_addr(lds);
  auto chunk = [&](int q) { return (lane & 7) ^ ((4 * (OWN ? q : wid) + (lane >> 4)) & 7); };            // of x, that the lane brings
  // the next stage to send for: its addresses and number; from the last on the same one again, into slots that nobody reads
  const char *xs = a.x, *ws = a.w, *ss = a.s;
  int sent = 0;
  unsigned ox[PX], ow[PW], os[PS];
#pragma unroll
  for (int q = 0; q < PX; ++q) ox[q] = offx[q];
#pragma unroll
  for (int q = 0; q < PW; ++q) ow[q] = offw[q];
#pragma unroll
  for (int q = 0; q < PS; ++q) os[q] = offs[q];
  auto begin = [&] __attribute__((always_inline)) {
    if (sent != a.nk - 1) return;
#pragma unroll
    for (int q = 0; q < PX; ++q) ox[q] -= 8 * chunk(q) >= a.tail ? 16 * chunk(q) : 0;
    if constexpr (GRAD) {
#pragma unroll
      for (int q = 0; q < PW; ++q) ow[q] = lastw[q];
#pragma unroll
      for (int q = 0; q < PS; ++q) os[q] = lasts[q];
    }
  };
  auto piece = [&](auto num, unsigned d) __attribute__((always_inline)) {      // d: the wave's first KiB in the slot
    constexpr int q = decltype(num)::value;
    if constexpr (q < PX) dma16<q * STEP>(xs, ox[q], d);
    else if constexpr (q < PX + PW) {
      constexpr int u = q - PX;
      if constexpr (OWN || NW % 4 == 0) dma16<XB + u * STEP>(ws, ow[u], d);
      else dma16<XB>(ws, ow[u], d + ((wid + 4 * u) % NW - wid) * 1024);
    } else {
      dma4<XB + WB + (q - PX - PW) * 256>(ss, os[q - PX - PW], d - wid * 768);
    }
  };
  auto end = [&] __attribute__((always_inline)) {
    const bool more = ++sent < a.nk, odd = (sent + a.odd) & 1;
    xs += more ? 128 : 0;
    if constexpr (GRAD) ws += more ? 4096 : 0, ss += more ? 256 : 0;
    else ws += more ? (odd ? 32 : a.wp - 32) : 0, ss += more && !odd ? a.sp : 0;
  };
  // what a last stage holds beyond the sum's end becomes zero; each wave mends the pieces that it sent for
  auto mend = [&](int slot) __attribute__((always_inline)) {
    if (a.tail == 64 && (!GRAD || a.tailw == 64)) return;
    char* d = lds + slot * SB;
#pragma unroll
    for (int q = 0; q < PX; ++q)
      if (8 * chunk(q) >= a.tail) *reinterpret_cast<uint4*>(d + wid * 1024 + q * STEP + lane * 16) = make_uint4(0, 0, 0, 0);
    if constexpr (GRAD) {
#pragma unroll
      for (int u = 0; u < PW; ++u) {
        const int pc = OWN ? u : (wid + 4 * u) % NW, pos = 16 * (pc & 1) + (lane >> 2);
        if (32 * ((pc >> 1) & 1) + ((pos & 3) << 3 | pos >> 2) >= a.tailw)
          *reinterpret_cast<uint4*>(d + XB + pc * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
      }
      if (lane >= a.tailw) *reinterpret_cast<unsigned*>(d + XB + WB + wid * 256 + lane * 4) = 0;
    }
  };
  // the wave's reads have arrived, and (not OWN) every wave's
  auto done = [&] __attribute__((always_inline)) {
    if constexpr (OWN) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    else tile::done_reading();
  };
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f}, hold<NAMED>(acc[i][j]);
  settle<NAMED>();
  constexpr int RW = GRAD ? 8 : NI;                      // reads of codes of a half
  uint4 fx[2][MJ];
  unsigned fw[2][NI][4], raw[RW], sc[RW];
  float fs[GRAD ? 2 : 1];
  const int xrow = (16 * MJ * wm + lr) * 128;
  const int wrow = 16 * NI * wn + lr;
  const int by = 9 + 8 * (lr >> 2);                      // GRAD: to the byte of the lane's columns
  // read n of half h of a stage: codes, scales (a row's four, once a stage; GRAD: those of four rows), fragments of x
  constexpr int RS = GRAD ? 2 : RW, READS = RW + RS + MJ;
  auto read = [&](int h, int slot, int n) __attribute__((always_inline)) {
    const char* d = lds + slot * SB;
    if (n < RW) {
      if constexpr (GRAD) {
        raw[n] = *reinterpret_cast<const unsigned*>(d + XB + wn * 4096 + h * 2048 + (4 * n + lg) * 64 + lr * 4);
      } else {
        const int r = wrow + 16 * n;
        raw[n] = *reinterpret_cast<const unsigned*>(d + XB + r * 32 + (((h ^ lr >> 3) & 1) << 4) + lg * 4);
      }
    } else if (n < RW + RS) {
      const int u = n - RW;
      if constexpr (GRAD) {
        const uint4 v = *reinterpret_cast<const uint4*>(d + XB + WB + wn * 256 + (32 * h + 8 * lg + 4 * u) * 4);
        sc[4 * u] = v.x, sc[4 * u + 1] = v.y, sc[4 * u + 2] = v.z, sc[4 * u + 3] = v.w;
      } else if (h == 0) sc[u] = *reinterpret_cast<const unsigned*>(d + XB + WB + (wrow + 16 * u) * 4);
    } else {
      const int u = n - RW - RS;
      fx[h][u] = *reinterpret_cast<const uint4*>(d + xrow + u * 2048 + (((4 * h + lg) ^ tile::swz(16 * MJ * wm + lr)) << 4));
    }
  };
  // unit n of the making of half h's fragments of w; t: their stage
  constexpr int UNITS = GRAD ? 16 : 4 * NI;
  auto make = [&](int h, int t, auto num) __attribute__((always_inline)) {
    constexpr int n = decltype(num)::value, w = n & 3, u = n >> 2;
    if constexpr (GRAD) {                                // rows 2 u and 2 u + 1, columns 2 w and 2 w + 1
      if constexpr (w == 0) fs[0] = mx_scale_of(sc[2 * u], by), fs[1] = mx_scale_of(sc[2 * u + 1], by);
      const uint2 v = columns<T, w>(raw[2 * u], raw[2 * u + 1], fs[0], fs[1]);
      fw[h][2 * w][u] = v.x, fw[h][2 * w + 1][u] = v.y;
    } else {
      if constexpr (w == 0) fs[0] = mx_scale_of(sc[u], (9 + 8 * h + 16 * ((t + a.odd) & 1)) & 31);
      fw[h][u][w] = pair<T, w>(raw[u], fs[0]);
    }
  };
  // the products of half h, between them reads and making of the other half, of stage t2 in `slot`, and pieces A .. B - 1 of a stage to d
  auto half = [&](int h, int t2, int slot, auto from, auto to, unsigned d) __attribute__((always_inline)) {
    constexpr int U = NI * MJ, UR = (U * 3 + 7) / 8, UV = U < 48 ? U / 2 : U / 4;        // reads in products 0 .. UR - 1, making from UV on
    constexpr int A = decltype(from)::value, N = decltype(to)::value - A;
    ready();
    each<0, U>([&](auto num) __attribute__((always_inline)) {
      constexpr int n = decltype(num)::value, i = n % NI, j = n / NI;
      mfma<T, NAMED>(acc[i][j], make_uint4(fw[h][i][0], fw[h][i][1], fw[h][i][2], fw[h][i][3]), fx[h][j]);
      constexpr int r0 = (n * READS + UR - 1) / UR, r1 = ((n + 1) * READS + UR - 1) / UR;
      each<(r0 < READS ? r0 : READS), (r1 < READS ? r1 : READS)>([&](auto r) __attribute__((always_inline)) { read(1 - h, slot, r.value); });
      if constexpr (n >= UV)
        each<(n - UV) * UNITS / (U - UV), (n - UV + 1) * UNITS / (U - UV)>([&](auto r) __attribute__((always_inline)) { make(1 - h, t2, r); });
      each<A + n * N / U, A + (n + 1) * N / U>([&](auto q) __attribute__((always_inline)) { piece(q, d); });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  const int nk = a.nk;
  const unsigned d0 = __builtin_amdgcn_readfirstlane(lds0 + wid * 1024);
  each<0, NST>([&](auto slot) __attribute__((always_inline)) {
    constexpr int u = decltype(slot)::value;
    begin();
    each<0, (u < NST - 1 ? P : P1)>([&](auto q) __attribute__((always_inline)) { piece(q, d0 + u * SB); });
    if constexpr (u < NST - 1) end();
  });
  // stage 0 has arrived
  tile::wait_vm<(NST - 2) * P + P1>();
  if (nk == 1) mend(0);
  done();
#pragma unroll
  for (int r = 0; r < READS; ++r) read(0, 0, r);
  each<0, UNITS>([&](auto r) __attribute__((always_inline)) { make(0, 0, r); });
  // slots of stages t and t + 1; half of a stage's pieces go with either half's products
  unsigned dp = d0 + (NST - 1) * SB;
  for (int t = 0, s0 = 0, s1 = 1;;) {
    half(0, t, s0, Int<P1>{}, Int<P>{}, dp);
    end();
    tile::wait_vm<(NST - 2) * P>();                      // stage t + 1 has arrived
    if (t + 2 == nk) mend(s1);
    done();
    begin();
    dp = __builtin_amdgcn_readfirstlane(d0 + s0 * SB);
    half(1, t + 1, s1, Int<0>{}, Int<P1>{}, dp);
    s0 = s1, s1 = s1 == NST - 1 ? 0 : s1 + 1;            // (the last step reads a slot that holds an earlier stage, or none: unused)
    if (++t == nk) break;
  }
  tile::wait_vm<0>();                                    // (nothing of this workgroup is under way when its LDS is another's)
  settle<NAMED>();
}

// ---- both operands in 4 bits ---------------------------------------------------------------------------
//
// Tiles as above; a stage is a panel, 128 k: one scaled product of 16 x 16 x 128 per pair of fragments, which takes a block and its scale
// byte from every lane.
template <int NI, int MJ, int WN>
struct Shape4 {
  static constexpr int WM = 4 / WN, BM = 16 * MJ * WM, BN = 16 * NI * WN;
  static constexpr int XB = BM * 64, WB = BN * 64, SB = XB + WB + 2048;
  static constexpr int NX = BM / 16, NW = BN / 16, PX = (NX + 3) / 4, PW = (NW + 3) / 4, PIECES = PX + PW + 2;
  static constexpr int FIT = kLds / SB, NST = FIT < 6 ? FIT : 6, LDS = NST * SB;
  static_assert(BM <= 256 && BM % 64 == 0 && BN <= 256 && NST >= 3 && (NST - 1) * PIECES < 64, "tile");
};

struct Walk4 {
  const char *x, *xs, *w, *s;  // codes and scales of both
  long long xp, xsp, wp, sp;   // bytes from panel to panel
  int nk;
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <bool NAMED>
__device__ __forceinline__ void mfma4(f32x4& c, uint4 a, uint4 b, unsigned sa, unsigned sb) {
  if constexpr (NAMED)
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                 : "+a"(c) : "v"(__builtin_bit_cast(u32x4, a)), "v"(__builtin_bit_cast(u32x4, b)), "v"(sa), "v"(sb));
  else
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w},
                                                         i32x8{(int)b.x, (int)b.y, (int)b.z, (int)b.w}, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

template <int NI, int MJ, int WN>
__device__ __forceinline__ void products4(char* lds, const Walk4& a, const unsigned (&offx)[Shape4<NI, MJ, WN>::PX], unsigned offxs,
                                          const unsigned (&offw)[Shape4<NI, MJ, WN>::PW], unsigned offs, f32x4 (&acc)[NI][MJ]) {
  using S = Shape4<NI, MJ, WN>;
  constexpr bool NAMED = kNamed<NI, MJ>;
  constexpr int PX = S::PX, PW = S::PW, NW = S::NW, P = S::PIECES, NST = S::NST, SB = S::SB, XB = S::XB, WB = S::WB;
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wid / WN, wn = wid % WN;
  const unsigned lds0 = lds_addr(lds);
  const char *px = a.x, *pxs = a.xs, *pw = a.w, *ps = a.s;               // the next panel to send for, from the last on that one again
  int sent = 0;
  auto piece = [&](auto num, unsigned d) __attribute__((always_inline)) {      // d: the wave's first KiB in the slot
    constexpr int q = decltype(num)::value;
    if constexpr (q < PX) dma16<q * 4096>(px, offx[q], d);
    else if constexpr (q < PX + PW) {
      constexpr int u = q - PX;
      if constexpr (NW % 4 == 0) dma16<XB + u * 4096>(pw, offw[u], d);
      else dma16<XB>(pw, offw[u], d + ((wid + 4 * u) % NW - wid) * 1024);
    } else if constexpr (q == PX + PW) dma4<XB + WB>(pxs, offxs, d - wid * 768);
    else dma4<XB + WB + 1024>(ps, offs, d - wid * 768);
  };
  auto end = [&] __attribute__((always_inline)) {
    const bool more = ++sent < a.nk;
    px += more ? a.xp : 0, pxs += more ? a.xsp : 0, pw += more ? a.wp : 0, ps += more ? a.sp : 0;
  };
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f}, hold<NAMED>(acc[i][j]);
  settle<NAMED>();
  uint4 fx[2][MJ], fw[2][NI];
  unsigned sx[2][MJ], sw[2][NI];
  const int xrow = 16 * MJ * wm + lr, wrow = 16 * NI * wn + lr;
  constexpr int READS = 2 * (NI + MJ), UNITS = NI + MJ;
  auto read = [&](int h, int slot, int n) __attribute__((always_inline)) {
    const char* d = lds + slot * SB;
    if (n < NI) sw[h][n] = *reinterpret_cast<const unsigned*>(d + XB + WB + 1024 + (wrow + 16 * n) * 4);
    else if (n < NI + MJ) sx[h][n - NI] = *reinterpret_cast<const unsigned*>(d + XB + WB + (xrow + 16 * (n - NI)) * 4);
    else if (n < 2 * NI + MJ) fw[h][n - NI - MJ] = *reinterpret_cast<const uint4*>(d + XB + (wrow + 16 * (n - NI - MJ)) * 64 + lg * 16);
    else fx[h][n - 2 * NI - MJ] = *reinterpret_cast<const uint4*>(d + (xrow + 16 * (n - 2 * NI - MJ)) * 64 + lg * 16);
  };
  auto make = [&](int h, int n) __attribute__((always_inline)) {         // a lane's byte of its row's four
    if (n < NI) asm volatile("v_lshrrev_b32 %0, %1, %0" : "+v"(sw[h][n]) : "v"(8 * lg));
    else asm volatile("v_lshrrev_b32 %0, %1, %0" : "+v"(sx[h][n - NI]) : "v"(8 * lg));
  };
  auto step = [&](int h, int slot, unsigned d) __attribute__((always_inline)) {
    constexpr int U = NI * MJ, UR = (U * 5 + 7) / 8, UV = U / 2;
    ready();
    each<0, U>([&](auto num) __attribute__((always_inline)) {
      constexpr int n = decltype(num)::value, i = n % NI, j = n / NI;
      mfma4<NAMED>(acc[i][j], fw[h][i], fx[h][j], sw[h][i], sx[h][j]);
      constexpr int r0 = (n * READS + UR - 1) / UR, r1 = ((n + 1) * READS + UR - 1) / UR;
      each<(r0 < READS ? r0 : READS), (r1 < READS ? r1 : READS)>([&](auto r) __attribute__((always_inline)) { read(1 - h, slot, r.value); });
      if constexpr (n >= UV)
        each<(n - UV) * UNITS / (U - UV), (n - UV + 1) * UNITS / (U - UV)>([&](auto r) __attribute__((always_inline)) { make(1 - h, r.value); });
      each<n * P / U, (n + 1) * P / U>([&](auto q) __attribute__((always_inline)) { piece(q, d); });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // two panels a way round, the second one zeros where there is none: the loop has one way out (accumulators, above)
  const int nk = (a.nk + 1) & ~1;
  const unsigned d0 = __builtin_amdgcn_readfirstlane(lds0 + wid * 1024);
#pragma unroll
  for (int u = 0; u < NST; ++u) {
    each<0, P>([&](auto q) __attribute__((always_inline)) { piece(q, d0 + u * SB); });
    end();
  }
  tile::wait_vm<(NST - 1) * P>();
  tile::done_reading();
#pragma unroll
  for (int r = 0; r < READS; ++r) read(0, 0, r);
#pragma unroll
  for (int r = 0; r < UNITS; ++r) make(0, r);
  int t = 0, s0 = 0, s1 = 1;
  auto next = [&](int h) __attribute__((always_inline)) {
    tile::wait_vm<(NST - 2) * P>();                      // panel t + 1 has arrived
    if (t + 1 == a.nk) {                                 // (each wave clears what it sent for)
#pragma unroll
      for (int q = 0; q < PX; ++q) *reinterpret_cast<uint4*>(lds + s1 * SB + (wid + 4 * q) * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
    }
    tile::done_reading();
    step(h, s1, __builtin_amdgcn_readfirstlane(d0 + s0 * SB));
    end();
    s0 = s1, s1 = s1 == NST - 1 ? 0 : s1 + 1, ++t;
  };
  do next(0), next(1);
  while (t < nk);
  tile::wait_vm<0>();                                    // (nothing of this workgroup is under way when its LDS is another's)
  settle<NAMED>();
}

}  // namespace mx
}  // namespace lumen
