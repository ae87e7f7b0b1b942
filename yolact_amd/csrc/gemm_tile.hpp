// Matrix-core tile engine of the prediction-head operators (gfx950).
//
//   C[j][i] = sum_k A[i][k] * B[j][k]        i < I (contiguous in the output), j < J
//
// Both operands are rows of K contiguous elements, so a step of k is always 128 BYTES of a row - 64 bf16 / f16, 32 f32 or
// 128 int8, a whole cache line - and one body serves every type: the global loads, the LDS image and the fragment
// addresses only know bytes.  K is a multiple of 128 bytes (callers pad with zeros), rows start on 16-byte boundaries.
//
// LDS image: two buffers, one step each.  Row r of a buffer is 8 chunks of 16 bytes; chunk c sits at slot c ^ (r & 7), so
// that the 8 rows a fragment read touches at a time fall into different banks (no conflicts counted).  It is filled by
// direct global -> LDS loads (16 bytes a lane, 8 rows a wave instruction), whose LDS side is fixed to lane order: the
// exclusive-or is applied to the global side.
//
// A lane of a 16 x 16 fragment holds row (lane & 15) and 16 bytes of k at chunk (lane >> 4) (+ 4 for the second half
// of the step); f32 feeds its 4 elements to 4 matrix instructions - which k goes to which instruction does not
// matter as long as A and B agree.  The result of lane l is j = l & 15, i = (l >> 4) * 4 + {0..3}: a lane owns four
// consecutive outputs of one row, and a row's sum over i (softmax) is mostly inside the lane.
#pragma once

#include "common.hpp"

enum { YP_T_F32 = YP_F32, YP_T_BF16 = YP_BF16, YP_T_F16 = YP_F16, YP_T_I8 = 3 };

typedef float yp_f4 __attribute__((ext_vector_type(4)));
typedef int yp_i4 __attribute__((ext_vector_type(4)));
typedef __bf16 yp_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 yp_h8 __attribute__((ext_vector_type(8)));

template <int TYPE> struct yp_type;
template <> struct yp_type<YP_T_F32> { typedef float elem; typedef yp_f4 frag; typedef yp_f4 acc; static constexpr int bytes = 4; };
template <> struct yp_type<YP_T_BF16> { typedef __bf16 elem; typedef yp_bf8 frag; typedef yp_f4 acc; static constexpr int bytes = 2; };
template <> struct yp_type<YP_T_F16> { typedef _Float16 elem; typedef yp_h8 frag; typedef yp_f4 acc; static constexpr int bytes = 2; };
template <> struct yp_type<YP_T_I8> { typedef signed char elem; typedef yp_i4 frag; typedef yp_i4 acc; static constexpr int bytes = 1; };

#define YP_TILE_KB 128   // bytes of k per step

static inline int64_t yp_pad_k(int64_t k, int bytes) { return (k * bytes + YP_TILE_KB - 1) / YP_TILE_KB * YP_TILE_KB; }   // in bytes

struct yp_gemm {
  const char* a;      // [I] rows of lda bytes
  const char* b;      // [J] rows of ldb bytes
  int64_t lda, ldb;
  int I, J;           // rows of a / b that exist (tiles past them read the last row again)
  int steps;          // K / YP_TILE_KB
  int splits;         // the steps are dealt to this many workgroups per tile (epilogues that take a split only)
  int tiles_i, tiles_j;
};

#ifdef __HIPCC__
template <int V> struct yp_const { static constexpr int value = V; };

template <int TYPE>
__device__ __forceinline__ typename yp_type<TYPE>::acc yp_mma(const typename yp_type<TYPE>::frag& a, const typename yp_type<TYPE>::frag& b,
                                                              typename yp_type<TYPE>::acc c) {
  if constexpr (TYPE == YP_T_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else if constexpr (TYPE == YP_T_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  else if constexpr (TYPE == YP_T_I8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  else {
#pragma unroll
    for (int u = 0; u < 4; ++u) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u], b[u], c, 0, 0, 0);
    return c;
  }
}

// The same in place, for the tile whose accumulators fill all 256 accumulation registers: given the builtin, the register
// allocator has no room to turn and moves every accumulator once per step (873 against 1 3xx TFLOP/s).  The compiler
// does not know that this is a matrix instruction: yp_settle stands between these and any other use of the result.
template <int TYPE, int U>
__device__ __forceinline__ void yp_mma_inplace(const typename yp_type<TYPE>::frag& a, const typename yp_type<TYPE>::frag& b, typename yp_type<TYPE>::acc& c) {
  if constexpr (TYPE == YP_T_BF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else if constexpr (TYPE == YP_T_F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else if constexpr (TYPE == YP_T_I8) asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_16x16x4_f32 %0, %1, %2, %0" : "+a"(c) : "v"(a[U]), "v"(b[U]));
}
// Nothing passes this: the accumulators are written by vector instructions before it and by matrix instructions after it,
// or the other way round, and the longest of either (16 passes) has finished.
template <int MI, int NJ, class Acc>
__device__ __forceinline__ void yp_settle(Acc (&acc)[MI][NJ]) {
  asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[0][0]));
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) asm volatile("" : "+a"(acc[m][n]));
  __builtin_amdgcn_sched_barrier(0);
}

// 64 lanes x 16 bytes from base + off (per lane) to LDS at `lds` (uniform) + lane * 16.  Written as assembly because the
// compiler would wait for it before every later LDS read that it cannot tell apart; the kernel below waits itself
// (yp_arrive).  It writes no register.
__device__ __forceinline__ void yp_load_lds16(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
// All but the last N of this wave's loads have landed and its LDS reads are done; then everybody's.
template <int N>
__device__ __forceinline__ void yp_arrive() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Where fragment m of a wave's M starts in a tile side of SIDE rows, relative to its fragment 0: half of them lie in each
// half of the side.  A wave's fragment 0 starts at wave * SIDE / 2 / waves.
template <int SIDE, int M>
__device__ __forceinline__ constexpr int yp_frag_at(int m) { return m / (M / 2) * (SIDE / 2) + m % (M / 2) * 16; }

// Which tile a workgroup takes.  Workgroup ids go round the 8 XCDs: every XCD gets a contiguous run of the tile order,
// and that order walks bands of 8 tiles in j, so that the tiles one XCD works on at a time share rows of both operands
// in its L2.
__device__ __forceinline__ void yp_tile_of(const yp_gemm& g, int wg, int nwg, int& ti, int& tj, int& split) {
  const int q = nwg >> 3, r = nwg & 7, x = wg & 7;
  int p = x * q + min(x, r) + (wg >> 3);
  const int tiles = g.tiles_i * g.tiles_j;
  split = p / tiles;
  p -= split * tiles;
  const int band = 8 * g.tiles_i;
  const int j0 = p / band * 8;
  const int h = min(8, g.tiles_j - j0);
  p -= (j0 >> 3) * band;
  ti = p / h;
  tj = j0 + p - ti * h;
}

// BM x BN tile, WI x WJ waves, each (BM / WI) x (BN / WJ).
//
// A wave's share is four quadrants, A0 and A1 by B0 and B1, half of its rows in each half of the tile.  A step is four
// phases of products, and each phase reads from LDS the fragments of the next:
//   p0  A0 B0, reads B1     p1  A0 B1, reads A1     p2  A1 B0, reads A0 of the next step     p3  A1 B1, reads its B0
// so every fragment has one set of registers, and half of a buffer is free half a step before the other: the loads of
// step s + 2 go into the buffer of step s in two groups, A0 B0 in p0 and p1 of s, B1 A1 in p2 and p3, each group a step
// and a half before it is read.  (With the whole buffer loaded at once, half a step to a step before: 1057 TFLOP/s.  With
// more stages of 64 bytes of k, every cache line fetched twice: 985.  bf16, 16384 x 8192 x 4096.)
template <int TYPE, int BM, int BN, int WI, int WJ, int WAVES_PER_SIMD, class Epi>
__global__ __launch_bounds__(WI * WJ * 64, WAVES_PER_SIMD) void yp_gemm_kernel(const yp_gemm g, const Epi epi) {
  typedef typename yp_type<TYPE>::frag frag;
  typedef typename yp_type<TYPE>::acc accv;
  constexpr int WAVES = WI * WJ, MI = BM / WI / 16, NJ = BN / WJ / 16, MH = MI / 2, NH = NJ / 2;
  constexpr int PA = BM / 16 / WAVES, PB = BN / 16 / WAVES;   // a wave's loads of half of A, of half of B (8 rows each)
  static_assert(PA * WAVES * 16 == BM && PB * WAVES * 16 == BN, "every wave issues as many loads: the waits count them");
  constexpr int BUF = (BM + BN) * YP_TILE_KB;
  constexpr bool INPLACE = MI * NJ * 4 == 256;
  __shared__ __align__(1024) char lds[2 * BUF];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int ti, tj, split;
  yp_tile_of(g, (int)blockIdx.x, (int)gridDim.x, ti, tj, split);
  const int i0 = ti * BM, j0 = tj * BN;
  const int k0 = (int)((int64_t)g.steps * split / g.splits), k1 = (int)((int64_t)g.steps * (split + 1) / g.splits);

  // this lane's source offsets (rows past the end read the last row: in bounds, and their results are dropped; a tile
  // may lie past the end altogether)
  const int ifirst = min(i0, g.I - 1), jfirst = min(j0, g.J - 1);
  const char* const abase = g.a + (int64_t)ifirst * g.lda;
  const char* const bbase = g.b + (int64_t)jfirst * g.ldb;
  const uint32_t col = (uint32_t)(((lane & 7) ^ (lane >> 3)) * 16);
  uint32_t aoff[2][PA], boff[2][PB];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int u = 0; u < PA; ++u)
      aoff[x][u] = (uint32_t)min(x * (BM / 2) + (wave * PA + u) * 8 + (lane >> 3), g.I - 1 - ifirst) * (uint32_t)g.lda + col;
#pragma unroll
    for (int u = 0; u < PB; ++u)
      boff[x][u] = (uint32_t)min(x * (BN / 2) + (wave * PB + u) * 8 + (lane >> 3), g.J - 1 - jfirst) * (uint32_t)g.ldb + col;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  auto load_a = [&](int buf, int k, int x, int u) {
    yp_load_lds16(abase + (int64_t)k * YP_TILE_KB, aoff[x][u], lds0 + (uint32_t)(buf * BUF + (x * (BM / 2) + (wave * PA + u) * 8) * YP_TILE_KB));
  };
  auto load_b = [&](int buf, int k, int x, int u) {
    yp_load_lds16(bbase + (int64_t)k * YP_TILE_KB, boff[x][u], lds0 + (uint32_t)(buf * BUF + (BM + x * (BN / 2) + (wave * PB + u) * 8) * YP_TILE_KB));
  };

  const int wi = wave % WI, wj = wave / WI;
  accv acc[MI][NJ];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[m][n] = accv{0, 0, 0, 0};
  if constexpr (INPLACE) yp_settle<MI, NJ>(acc);

  const int fo = (lane & 15) * YP_TILE_KB + (((lane >> 4) ^ (lane & 7)) * 16);
  const int fa = wi * (BM / 2 / WI) * YP_TILE_KB + fo, fb = (BM + wj * (BN / 2 / WJ)) * YP_TILE_KB + fo;
  frag a[2][MH][2], b[2][NH][2];          // [half][fragment][half step]
  auto read_a = [&](int buf, int x, int q) {
    a[x][q >> 1][q & 1] = *reinterpret_cast<const frag*>(lds + buf * BUF + ((fa ^ ((q & 1) * 64)) + (x * (BM / 2) + (q >> 1) * 16) * YP_TILE_KB));
  };
  auto read_b = [&](int buf, int x, int q) {
    b[x][q >> 1][q & 1] = *reinterpret_cast<const frag*>(lds + buf * BUF + ((fb ^ ((q & 1) * 64)) + (x * (BN / 2) + (q >> 1) * 16) * YP_TILE_KB));
  };
  typedef yp_const<0> E0; typedef yp_const<1> E1; typedef yp_const<2> E2;

  // products of half X of A and half Y of B; meanwhile reads half RX of A (RD = 1) or of B (RD = 2) in rbuf, and loads
  // half LX of A (LD = 1) or of B (LD = 2) of step lk into lbuf.  2 MH groups of NH products, the reads first in each.
  auto phase = [&](auto X, auto Y, auto RD, auto RX, int rbuf, auto LD, auto LX, int lbuf, int lk) {
    constexpr int x = decltype(X)::value, y = decltype(Y)::value, rdk = decltype(RD)::value, rx = decltype(RX)::value;
    constexpr int ldk = decltype(LD)::value, lx = decltype(LX)::value;
    constexpr int G = 2 * MH, RN = rdk == 1 ? 2 * MH : rdk == 2 ? 2 * NH : 0, LN = ldk == 1 ? PA : ldk == 2 ? PB : 0;
    int rd = 0, ld = 0;
#pragma unroll
    for (int gi = 0; gi < G; ++gi) {
      const int q = gi & 1, m = gi >> 1;
#pragma unroll
      for (; rd * G < (gi + 1) * RN; ++rd) {
        if constexpr (rdk == 1) read_a(rbuf, rx, rd);
        else if constexpr (rdk == 2) read_b(rbuf, rx, rd);
      }
#pragma unroll
      for (; ld * G < (gi + 1) * LN; ++ld) {
        if constexpr (ldk == 1) load_a(lbuf, lk, lx, ld);
        else if constexpr (ldk == 2) load_b(lbuf, lk, lx, ld);
      }
      if constexpr (INPLACE) {
#pragma unroll
        for (int n = 0; n < NH; ++n) yp_mma_inplace<TYPE, 0>(a[x][m][q], b[y][n][q], acc[x * MH + m][y * NH + n]);
        if constexpr (TYPE == YP_T_F32) {      // (the same accumulator again after NH others)
#pragma unroll
          for (int n = 0; n < NH; ++n) yp_mma_inplace<TYPE, 1>(a[x][m][q], b[y][n][q], acc[x * MH + m][y * NH + n]);
#pragma unroll
          for (int n = 0; n < NH; ++n) yp_mma_inplace<TYPE, 2>(a[x][m][q], b[y][n][q], acc[x * MH + m][y * NH + n]);
#pragma unroll
          for (int n = 0; n < NH; ++n) yp_mma_inplace<TYPE, 3>(a[x][m][q], b[y][n][q], acc[x * MH + m][y * NH + n]);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NH; ++n) acc[x * MH + m][y * NH + n] = yp_mma<TYPE>(a[x][m][q], b[y][n][q], acc[x * MH + m][y * NH + n]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (k0 < k1) {
    const int last = k1 - 1;
    // past the last step the last one is loaded again: the number of loads in flight, which the waits count, is always
    // the same
    constexpr int GROUP = PA + PB;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int u = 0; u < PA; ++u) load_a(s, min(k0 + s, last), 0, u);
#pragma unroll
      for (int u = 0; u < PB; ++u) load_b(s, min(k0 + s, last), 0, u);
#pragma unroll
      for (int u = 0; u < PB; ++u) load_b(s, min(k0 + s, last), 1, u);
#pragma unroll
      for (int u = 0; u < PA; ++u) load_a(s, min(k0 + s, last), 1, u);
    }
    yp_arrive<3 * GROUP>();
#pragma unroll
    for (int q = 0; q < 2 * MH; ++q) read_a(0, 0, q);
#pragma unroll
    for (int q = 0; q < 2 * NH; ++q) read_b(0, 0, q);
    yp_arrive<2 * GROUP>();
    int buf = 0;
    for (int k = k0; k < last; ++k, buf ^= 1) {
      const int lk = min(k + 2, last);
      phase(E0{}, E0{}, E2{}, E1{}, buf, E1{}, E0{}, buf, lk);
      phase(E0{}, E1{}, E1{}, E1{}, buf, E2{}, E0{}, buf, lk);
      yp_arrive<2 * GROUP>();
      phase(E1{}, E0{}, E1{}, E0{}, buf ^ 1, E2{}, E1{}, buf, lk);
      phase(E1{}, E1{}, E2{}, E0{}, buf ^ 1, E1{}, E1{}, buf, lk);
      yp_arrive<2 * GROUP>();
    }
    phase(E0{}, E0{}, E2{}, E1{}, buf, E0{}, E0{}, 0, 0);
    phase(E0{}, E1{}, E1{}, E1{}, buf, E0{}, E0{}, 0, 0);
    phase(E1{}, E0{}, E0{}, E0{}, 0, E0{}, E0{}, 0, 0);
    phase(E1{}, E1{}, E0{}, E0{}, 0, E0{}, E0{}, 0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the surplus loads: nothing may arrive in LDS after the workgroup has left it
  }
  if constexpr (INPLACE) yp_settle<MI, NJ>(acc);
  epi.template apply<TYPE, BM, BN, WI, WJ, MI, NJ>(g, acc, ti, tj, split, wi, wj, lane);
}
#endif  // __HIPCC__
