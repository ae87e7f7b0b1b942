// Matrix-core tile engine of the prediction-head operators (gfx950).
//
//   C[j][i] = sum_k A(i, k) * B(j, k)        i < I (contiguous in the output), j < J
//
// An operand is either rows of K contiguous elements ("by rows": [I][K]) or K rows of its elements ("by k": [K][I]),
// chosen at compile time, so that the gradient products read what the other products read and wrote, without transposed
// copies.  A step of k is always 128 BYTES of elements - 64 bf16 / f16, 32 f32 or 128 int8 - and the loads and the LDS
// image only know bytes.  By rows, K is a multiple of 128 bytes (callers pad with zeros); by k, rows of k past the end
// read the last one again, and the other operand is zero there.  Rows start on 16-byte boundaries.
//
// LDS image: two buffers of one step; the halves of each side lie apart.  By rows, a row is 8 chunks of 16 bytes and chunk
// c sits at slot c ^ (r & 7), so that the 8 rows a fragment read touches at a time fall into different banks (no conflicts
// counted).  By k, a row of k is the half side's elements; its chunks are exclusive-ored by a function of k that spreads
// the rows of k one transposing read (16 bit) or four word reads (f32) touch.  The image is filled by direct global -> LDS
// loads (16 bytes a lane, 1024 a wave instruction), whose LDS side is fixed to lane order: the exclusive-or is applied to
// the global side.
//
// A lane of a 16 x 16 fragment holds row (lane & 15) and 16 bytes of k at chunk (lane >> 4) (+ 4 for the second half
// of the step); f32 feeds its 4 elements to 4 matrix instructions - which k goes to which instruction does not
// matter as long as A and B agree.  The result of lane l is j = l & 15, i = (l >> 4) * 4 + {0..3}: a lane owns four
// consecutive outputs of one row, and a row's sum over i (softmax) is mostly inside the lane.
#pragma once

#include "common.hpp"

enum { YP_TILE_L = 0, YP_TILE_M = 1, YP_TILE_T = 2 };
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
  const char* a;
  const char* b;
  int64_t lda, ldb;   // bytes between rows (of I / J elements' k, or of k)
  int I, J;           // rows of the result's axes that exist (tiles past them read the last one again)
  int K;              // by k: rows of k that exist
  int steps;          // steps of 128 bytes of k
  int splits;         // the steps are dealt to this many workgroups per tile (epilogues that take a split only)
  int tiles_i, tiles_j;
  int64_t aplane, bplane;   // bytes between the planes
};

// SEGS > 1: operands as the sum of two planes of their type, and the products of planes one after the other along a k
// axis SEGS times as long:
//   2  B has two planes: twice its precision
//   3  f32 operands, scaled by a power of two, as two f16 planes each (22 bits, to 2^-39 of the largest element); of the
//      four products of planes the three whose terms are not below 2^-24 of the result.  The f16 matrix instructions are
//      16 times as fast as the f32 ones: three of them for one.  Sums are f32 as ever.
#define YP_SEGMENT_A(s) ((s) == 2)
#define YP_SEGMENT_B(s) ((s) == 1)

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
// allocator has no room to turn and moves every accumulator once per step (883 TFLOP/s against 1057, bf16, 16384 x 8192 x 4096).  The compiler
// does not know that this is a matrix instruction: yp_settle stands between these and any other use of the result.
template <int TYPE>
__device__ __forceinline__ void yp_mma_inplace(const typename yp_type<TYPE>::frag& a, const typename yp_type<TYPE>::frag& b, typename yp_type<TYPE>::acc& c) {
  if constexpr (TYPE == YP_T_BF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else if constexpr (TYPE == YP_T_F16) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
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

// (the compiler does not always see that a value is the same in all lanes)
__device__ __forceinline__ int64_t yp_uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// 64 lanes x 16 bytes from base + off (per lane) to LDS at `lds` (uniform) + lane * 16.  Written as assembly because the
// compiler would wait for it before every later LDS read that it cannot tell apart; the kernel below waits itself
// (yp_arrive).  It writes no register but m0, and says so: nothing of the compiler's may stand between its own write of m0 and
// the use.  (That it restores nothing is what the compiler would warn of at every use; nobody expects m0 to last.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void yp_load_lds16(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
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

// One operand of a tile: SIDE rows (of I or J), shared by WAVES waves for the loads and by W of them for the fragments.
template <int TYPE, int SIDE, int WAVES, int W, bool BY_K>
struct yp_side {
  typedef typename yp_type<TYPE>::frag frag;
  static constexpr int B = yp_type<TYPE>::bytes;
  static constexpr int P = SIDE / 16 / WAVES;          // a wave's loads of one half
  static constexpr int FH = SIDE / 32 / W;             // a wave's fragments in one half
  static constexpr int HALF = SIDE * (YP_TILE_KB / 2); // bytes of a half in LDS
  static constexpr int KR = YP_TILE_KB / B;            // elements of k per step
  static constexpr int HB = SIDE / 2 * B;              // by k: bytes of a row of k
  static constexpr int CH = HB / 16;                   //       its chunks
  static_assert(P * WAVES * 16 == SIDE, "every wave issues as many loads: the waits count them");

  const char* base;
  int64_t stride;          // bytes from step to step
  uint32_t off[2][P];      // this lane's source offsets
  uint32_t ld, colmax;     // by k
  int K;
  uint32_t lds;            // LDS address of the first half's first load of this wave
  int fbase;               // this lane's first fragment, relative to the half

  static __device__ __forceinline__ int swizzle(int k) {
    if (B == 4) return HB >= 256 ? 4 * ((k >> 2) & 3) : 4 * ((k >> 2) & 1);
    if (HB == 256) return 2 * ((k & 3) | ((k >> 3) & 1) << 2);
    if (HB == 128) return 2 * (((k >> 1) & 1) | ((k >> 3) & 1) << 1);
    return 2 * ((k >> 3) & 1);
  }
  // rows past the end read the last row: in bounds, and their results are dropped (a tile may lie past the end altogether)
  __device__ __forceinline__ void init(const char* p, int64_t row_bytes, int first, int count, int krows, uint32_t lds_at, int wave, int w, int lane) {
    lds = lds_at + (uint32_t)(wave * P) * 1024u;
    if constexpr (!BY_K) {
      const int f = min(first, count - 1);
      base = p + (int64_t)f * row_bytes;
      stride = YP_TILE_KB;
      const uint32_t col = (uint32_t)(((lane & 7) ^ (lane >> 3)) * 16);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int u = 0; u < P; ++u)
          off[x][u] = (uint32_t)min(x * (SIDE / 2) + (wave * P + u) * 8 + (lane >> 3), count - 1 - f) * (uint32_t)row_bytes + col;
      fbase = (w * (SIDE / 2 / W) + (lane & 15)) * YP_TILE_KB + (((lane >> 4) ^ (lane & 7)) * 16);
    } else {
      const int64_t c0 = min((int64_t)first * B, row_bytes - 16);
      base = p + c0;
      stride = (int64_t)KR * row_bytes;
      ld = (uint32_t)row_bytes;
      K = krows;
      colmax = (uint32_t)min(row_bytes - 16 - c0, (int64_t)SIDE * B);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int u = 0; u < P; ++u) {
          const int k = (wave * P + u) * (64 / CH) + lane / CH;
          off[x][u] = (uint32_t)k * ld + min((uint32_t)(x * HB + ((lane % CH) ^ swizzle(k)) * 16), colmax);
        }
      const int t = lane & 15, g = lane >> 4;
      if (B == 4) fbase = g * 4 * HB + (((w * (HB / W / 16) + (t >> 2)) ^ swizzle(g * 4)) * 16) + (t & 3) * 4;
      else fbase = (g * 8 + (t >> 2)) * HB + (((w * (HB / W / 16) + ((t & 3) >> 1)) ^ swizzle(g * 8 + (t >> 2))) * 16) + (t & 1) * 8;
    }
  }
  // load u of half x of step k, which begins `from` bytes after the base, into a buffer `at` bytes into the LDS
  __device__ __forceinline__ void load(int at, int64_t from, int k, int x, int u) const {
    const uint32_t to = lds + (uint32_t)(at + x * HALF + u * 1024);
    if constexpr (!BY_K) yp_load_lds16(base + from, off[x][u], to);
    else yp_load_lds16(base + from, min(off[x][u], (uint32_t)(min(K - k * KR, KR) - 1) * ld + colmax), to);
  }
  // fragment f of half x, half step q
  __device__ __forceinline__ frag read(const char* buf, int x, int f, int q) const {
    if constexpr (!BY_K) {
      return *reinterpret_cast<const frag*>(buf + x * HALF + ((fbase ^ (q * 64)) + f * 16 * YP_TILE_KB));
    } else if constexpr (B == 4) {
      const char* const p = buf + x * HALF + (fbase ^ (f * 64)) + q * 16 * HB;
      frag r;
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = *reinterpret_cast<const float*>(p + u * HB);
      return r;
    } else {
      // 16 lanes read 4 rows of k x 16 elements and get them transposed: 4 consecutive k of one element each
      typedef short s4 __attribute__((ext_vector_type(4)));
      const char* const p = buf + x * HALF + (fbase ^ (f * 32)) + q * 32 * HB;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 4 * HB));
      return __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// The tile shapes: BM x BN by WI x WJ waves, each (BM / WI) x (BN / WJ).
template <int SHAPE> struct yp_shape;
template <> struct yp_shape<YP_TILE_L> { static constexpr int BM = 256, BN = 256, WI = 2, WJ = 2, WPS = 1; };
template <> struct yp_shape<YP_TILE_M> { static constexpr int BM = 128, BN = 128, WI = 2, WJ = 2, WPS = 2; };
template <> struct yp_shape<YP_TILE_T> { static constexpr int BM = 64, BN = 64, WI = 2, WJ = 2, WPS = 4; };
template <int SHAPE> constexpr int yp_lds_bytes = 2 * (yp_shape<SHAPE>::BM + yp_shape<SHAPE>::BN) * YP_TILE_KB;

// What an epilogue knows about its place.
struct yp_place {
  int ti, tj, split;   // tile, part of the k axis
  int wi, wj, lane;
  char* lds;           // all of the tile's LDS, after yp_arrive<0>
};

// A wave's share is four quadrants, A0 and A1 by B0 and B1, half of its rows in each half of the tile.  A step is four
// phases of products, and each phase reads from LDS the fragments of the next:
//   p0  A0 B0, reads B1     p1  A0 B1, reads A1     p2  A1 B0, reads A0 of the next step     p3  A1 B1, reads its B0
// so every fragment has one set of registers, and half of a buffer is free half a step before the other: the loads of
// step s + 2 go into the buffer of step s in two groups, A0 B0 in p0 and p1 of s, B1 A1 in p2 and p3, each group a step
// and a half before it is read.  (With the whole buffer loaded at once, half a step to a step before: 1057 TFLOP/s.  With
// more stages of 64 bytes of k, every cache line fetched twice: 985.  This: 1257.  bf16, 16384 x 8192 x 4096.)
template <int TYPE, int SHAPE, bool A_BY_K, bool B_BY_K, int SEGS, class Epi>
__device__ __forceinline__ void yp_gemm_tile(const yp_gemm& g, const Epi& epi, int wg, int nwg, char* lds) {
  typedef typename yp_type<TYPE>::frag frag;
  typedef typename yp_type<TYPE>::acc accv;
  typedef yp_shape<SHAPE> S;
  constexpr int BM = S::BM, BN = S::BN, WI = S::WI, WJ = S::WJ, WAVES = WI * WJ;
  constexpr int MI = BM / WI / 16, NJ = BN / WJ / 16, MH = MI / 2, NH = NJ / 2;
  constexpr int BUF = (BM + BN) * YP_TILE_KB;
  constexpr bool INPLACE = MI * NJ * 4 == 256;
  static_assert(!(INPLACE && TYPE == YP_T_F32), "f32 as it is runs on the smaller tiles: it keeps two sums");
  yp_place at;
  at.lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  yp_tile_of(g, wg, nwg, at.ti, at.tj, at.split);
  at.wi = wave % WI; at.wj = wave / WI;
  at.lds = lds;
  const int steps = g.steps * SEGS;
  const int k0 = (int)((int64_t)steps * at.split / g.splits), k1 = (int)((int64_t)steps * (at.split + 1) / g.splits);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  typedef yp_side<TYPE, BM, WAVES, WI, A_BY_K> SA;
  typedef yp_side<TYPE, BN, WAVES, WJ, B_BY_K> SB;
  SA sa;
  SB sb;
  sa.init(g.a, g.lda, at.ti * BM, g.I, g.K, lds0, wave, at.wi, at.lane);
  sb.init(g.b, g.ldb, at.tj * BN, g.J, g.K, lds0 + BM * YP_TILE_KB, wave, at.wj, at.lane);

  accv acc[MI][NJ];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[m][n] = accv{0, 0, 0, 0};
  if constexpr (INPLACE) yp_settle<MI, NJ>(acc);
  // the f32 matrix instruction rounds after every k: sums of 256 are added up apart, or thousands of roundings in a row show
  constexpr bool CHUNKS = TYPE == YP_T_F32;
  accv total[MI][NJ];
  if constexpr (CHUNKS) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NJ; ++n) total[m][n] = accv{0, 0, 0, 0};
  }

  frag a[2][MH][2], b[2][NH][2];          // [half][fragment][half step]
  auto read_a = [&](int buf, int x, int q) { a[x][q >> 1][q & 1] = sa.read(lds + buf * BUF, x, q >> 1, q & 1); };
  auto read_b = [&](int buf, int x, int q) { b[x][q >> 1][q & 1] = sb.read(lds + buf * BUF + BM * YP_TILE_KB, x, q >> 1, q & 1); };
  typedef yp_const<0> E0; typedef yp_const<1> E1; typedef yp_const<2> E2;

  // the step to load: k, and where it begins in a and b
  int lk = 0, ls = 0, todo = 0;
  int64_t from_a = 0, from_b = 0;
  auto place = [&]() {
    from_a = lk * sa.stride;
    from_b = lk * sb.stride;
    if (SEGS > 1) {
      from_a = yp_uniform(from_a + (YP_SEGMENT_A(ls) ? g.aplane : 0));
      from_b = yp_uniform(from_b + (YP_SEGMENT_B(ls) ? g.bplane : 0));
    }
  };
  // past the last step the last one is loaded again: the number of loads in flight, which the waits count, is always the
  // same
  auto advance = [&]() {
    if (todo > 0) {
      --todo;
      if (SEGS > 1 && lk + 1 == g.steps) { lk = 0; ++ls; } else ++lk;
      place();
    }
  };

  // products of half X of A and half Y of B; meanwhile reads half RX of A (RD = 1) or of B (RD = 2) in rbuf, and loads
  // half LX of A (LD = 1) or of B (LD = 2) of the step to load into lbuf.  2 MH groups of NH products, the reads first in each.
  auto phase = [&](auto X, auto Y, auto RD, auto RX, int rbuf, auto LD, auto LX, int lbuf) {
    constexpr int x = decltype(X)::value, y = decltype(Y)::value, rdk = decltype(RD)::value, rx = decltype(RX)::value;
    constexpr int ldk = decltype(LD)::value, lx = decltype(LX)::value;
    constexpr int G = 2 * MH, RN = rdk == 1 ? 2 * MH : rdk == 2 ? 2 * NH : 0, LN = ldk == 1 ? SA::P : ldk == 2 ? SB::P : 0;
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
        if constexpr (ldk == 1) sa.load(lbuf * BUF, from_a, lk, lx, ld);
        else if constexpr (ldk == 2) sb.load(lbuf * BUF, from_b, lk, lx, ld);
      }
      if constexpr (INPLACE) {
#pragma unroll
        for (int n = 0; n < NH; ++n) yp_mma_inplace<TYPE>(a[x][m][q], b[y][n][q], acc[x * MH + m][y * NH + n]);
      } else {
#pragma unroll
        for (int n = 0; n < NH; ++n) acc[x * MH + m][y * NH + n] = yp_mma<TYPE>(a[x][m][q], b[y][n][q], acc[x * MH + m][y * NH + n]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (k0 < k1) {
    ls = SEGS > 1 ? k0 / g.steps : 0;
    lk = k0 - ls * g.steps;
    todo = k1 - 1 - k0;
    place();
    constexpr int GROUP = SA::P + SB::P;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int u = 0; u < SA::P; ++u) sa.load(s * BUF, from_a, lk, 0, u);
#pragma unroll
      for (int u = 0; u < SB::P; ++u) sb.load(s * BUF, from_b, lk, 0, u);
#pragma unroll
      for (int u = 0; u < SB::P; ++u) sb.load(s * BUF, from_b, lk, 1, u);
#pragma unroll
      for (int u = 0; u < SA::P; ++u) sa.load(s * BUF, from_a, lk, 1, u);
      advance();
    }
    yp_arrive<3 * GROUP>();
#pragma unroll
    for (int q = 0; q < 2 * MH; ++q) read_a(0, 0, q);
#pragma unroll
    for (int q = 0; q < 2 * NH; ++q) read_b(0, 0, q);
    yp_arrive<2 * GROUP>();
    int buf = 0;
    for (int k = k0; k < k1 - 1; ++k, buf ^= 1) {
      if (CHUNKS && k > k0 && ((k - k0) & 7) == 0) {
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
          for (int n = 0; n < NJ; ++n) { total[m][n] = total[m][n] + acc[m][n]; acc[m][n] = accv{0, 0, 0, 0}; }
      }
      phase(E0{}, E0{}, E2{}, E1{}, buf, E1{}, E0{}, buf);
      phase(E0{}, E1{}, E1{}, E1{}, buf, E2{}, E0{}, buf);
      yp_arrive<2 * GROUP>();
      phase(E1{}, E0{}, E1{}, E0{}, buf ^ 1, E2{}, E1{}, buf);
      phase(E1{}, E1{}, E2{}, E0{}, buf ^ 1, E1{}, E1{}, buf);
      advance();
      yp_arrive<2 * GROUP>();
    }
    phase(E0{}, E0{}, E2{}, E1{}, buf, E0{}, E0{}, 0);
    phase(E0{}, E1{}, E1{}, E1{}, buf, E0{}, E0{}, 0);
    phase(E1{}, E0{}, E0{}, E0{}, 0, E0{}, E0{}, 0);
    phase(E1{}, E1{}, E0{}, E0{}, 0, E0{}, E0{}, 0);
  }
  if constexpr (INPLACE) yp_settle<MI, NJ>(acc);
  if constexpr (CHUNKS) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NJ; ++n) acc[m][n] = total[m][n] + acc[m][n];
  }
  yp_arrive<0>();    // the surplus loads of every wave have landed: the LDS is the epilogue's
  epi.template apply<TYPE, SHAPE, MI, NJ>(g, acc, at);
}

template <int TYPE, int SHAPE, int SEGS, class Epi>
__global__ __launch_bounds__(256, yp_shape<SHAPE>::WPS) void yp_gemm_kernel(const yp_gemm g, const Epi epi) {
  __shared__ __align__(1024) char lds[yp_lds_bytes<SHAPE>];
  yp_gemm_tile<TYPE, SHAPE, false, false, SEGS>(g, epi, (int)blockIdx.x, (int)gridDim.x, lds);
}

// The two gradient products, of one tile shape, in one launch: the first reads both operands by k, the second A by k and B by
// rows; n1 and n2 workgroups, with `second_first` the second one's first.  Workgroups past them take `extra(i, lds)`.
template <int TYPE, int SHAPE, int SEGS, class Epi, class Extra>
__global__ __launch_bounds__(256, yp_shape<SHAPE>::WPS) void yp_two_gemms_kernel(const yp_gemm g1, const Epi e1, int n1, const yp_gemm g2, const Epi e2, int n2,
                                                                                 int second_first, const Extra extra) {
  __shared__ __align__(1024) char lds[yp_lds_bytes<SHAPE>];
  const int wg = (int)blockIdx.x;
  if (wg >= n1 + n2) { extra(wg - n1 - n2, lds); return; }
  const bool first = second_first ? wg >= n2 : wg < n1;
  if (first) yp_gemm_tile<TYPE, SHAPE, true, true, SEGS>(g1, e1, second_first ? wg - n2 : wg, n1, lds);
  else yp_gemm_tile<TYPE, SHAPE, true, false, SEGS>(g2, e2, second_first ? wg : wg - n1, n2, lds);
}

// Where an epilogue's fragment (0, 0), element 0 lies: i and j of this lane.
template <int SHAPE>
__device__ __forceinline__ void yp_origin(const yp_place& at, int& i, int& j) {
  typedef yp_shape<SHAPE> S;
  i = at.ti * S::BM + at.wi * (S::BM / 2 / S::WI) + (at.lane >> 4) * 4;
  j = at.tj * S::BN + at.wj * (S::BN / 2 / S::WJ) + (at.lane & 15);
}

// Stores a tile, val(m, n) = the four values of a lane's fragment, as rows of out ([j][i], `ld` elements apart, i < I,
// j < J), or adds them to what is there: through LDS, so that the stores are whole lines.  Stored from the fragments
// directly - 16 rows of 32 bytes an instruction - 134 MB took 60 us, with this 26 (8192 x 8192 bf16).
// vec: out and ld are multiples of 16 bytes.
template <int OUT, int SHAPE, bool ADD, int MI, int NJ, class Val>
__device__ __forceinline__ void yp_put_tile(const yp_place& at, void* out, int64_t ld, int I, int J, bool vec, const Val& val) {
  typedef yp_shape<SHAPE> S;
  typedef typename yp_type<OUT>::elem elem;
  constexpr int OB = yp_type<OUT>::bytes, E = 16 / OB, CPR = S::BM / E;      // elements per chunk, chunks per row
  constexpr int SW = (CPR < 16 ? CPR : 16) - 1;                             // chunk c of row r sits at slot c ^ (r & SW)
  constexpr int PASSES = S::BM * S::BN * OB > yp_lds_bytes<SHAPE> ? 2 : 1;
  typedef elem e4 __attribute__((ext_vector_type(4)));
  typedef elem eE __attribute__((ext_vector_type(E)));
  const int tid = (int)threadIdx.x;
  const int iw = at.wi * (S::BM / 2 / S::WI) + (at.lane >> 4) * 4;
#pragma unroll
  for (int pass = 0; pass < PASSES; ++pass) {
    if (pass) yp_arrive<0>();
#pragma unroll
    for (int n = pass * NJ / PASSES; n < (pass + 1) * NJ / PASSES; ++n) {
      const int jl = at.wj * (S::BN / 2 / S::WJ) + (at.lane & 15) + yp_frag_at<S::BN, NJ>(n) - pass * (S::BN / 2);
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int byte = (iw + yp_frag_at<S::BM, MI>(m)) * OB;
        const yp_f4 v = val(m, n);
        *reinterpret_cast<e4*>(at.lds + jl * (S::BM * OB) + (((byte >> 4) ^ (at.lane & SW)) << 4) + (byte & 15)) =
            e4{(elem)v.x, (elem)v.y, (elem)v.z, (elem)v.w};
      }
    }
    yp_arrive<0>();
    constexpr int ROWS = S::BN / PASSES;
    const int j0 = at.tj * S::BN + pass * ROWS, i0 = at.ti * S::BM;
    if (vec) {
      const int c = tid % CPR, i = i0 + c * E;
      for (int r = tid / CPR; r < ROWS && j0 + r < J; r += 256 / CPR) {
        if (i >= I) break;
        eE v = *reinterpret_cast<const eE*>(at.lds + r * (S::BM * OB) + ((c ^ (r & SW)) << 4));
        elem* const to = reinterpret_cast<elem*>(out) + (int64_t)(j0 + r) * ld + i;
        if (i + E <= I) {
          if (ADD) v = v + *reinterpret_cast<const eE*>(to);
          *reinterpret_cast<eE*>(to) = v;
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) if (i + e < I) to[e] = ADD ? (elem)(v[e] + to[e]) : v[e];
        }
      }
    } else {   // odd rows: element by element, consecutive lanes to consecutive elements
      const int c = tid % S::BM, i = i0 + c;
      if (i < I)
        for (int r = tid / S::BM; r < ROWS && j0 + r < J; r += 256 / S::BM) {
          const elem v = *reinterpret_cast<const elem*>(at.lds + r * (S::BM * OB) + (((c / E) ^ (r & SW)) << 4) + (c % E) * OB);
          elem* const to = reinterpret_cast<elem*>(out) + (int64_t)(j0 + r) * ld + i;
          *to = ADD ? (elem)(v + *to) : v;
        }
    }
  }
}
#endif  // __HIPCC__
