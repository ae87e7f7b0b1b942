// Matrix-core tile engine of the prediction-head operators (gfx950).
//
//   C[j][i] = sum_k A[i][k] * B[j][k]        i < I (contiguous in the output), j < J
//
// Both operands are rows of K contiguous elements, so a tile row is always 128 BYTES of k - 64 bf16 / f16, 32 f32 or
// 128 int8 - and one body serves every type: the global loads, the LDS image and the fragment addresses only know
// bytes.  K is a multiple of 128 bytes (callers pad with zeros), rows start on 16-byte boundaries.
//
// LDS image: row r of a tile is 8 chunks of 16 bytes; chunk c of the row sits at slot c ^ (r & 7), so that the 8 rows
// a fragment read touches at a time fall into 8 different slots.  The image is filled by direct global -> LDS loads
// (16 bytes a lane, 8 rows a wave instruction), whose LDS side is fixed to lane order: the exclusive-or is applied to
// the global side.  Two LDS buffers, as two arrays, so that the compiler knows the fragment reads of one apart from
// the loads into the other and does not wait for them.
//
// A lane of a 16 x 16 fragment holds row (lane & 15) and 16 bytes of k at chunk (lane >> 4) (+ 4 for the second half
// of the tile row); f32 feeds its 4 elements to 4 matrix instructions - which k goes to which instruction does not
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

#define YP_TILE_KB 128   // bytes of k per tile row

static inline int64_t yp_pad_k(int64_t k, int bytes) { return (k * bytes + YP_TILE_KB - 1) / YP_TILE_KB * YP_TILE_KB; }   // in bytes

struct yp_gemm {
  const char* a;      // [I] rows of lda bytes
  const char* b;      // [J] rows of ldb bytes
  int64_t lda, ldb;
  int I, J;           // rows of a / b that exist (tiles past them read the last row again)
  int steps;          // K / 128 bytes
  int splits;         // the steps are dealt to this many workgroups per tile (epilogues that take a split only)
  int tiles_i, tiles_j;
};

#ifdef __HIPCC__
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

__device__ __forceinline__ void yp_load_lds16(const char* src, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

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
template <int TYPE, int BM, int BN, int WI, int WJ, class Epi>
__global__ __launch_bounds__(WI * WJ * 64, (BM * BN >= 256 * 256 ? 2 : (WI * WJ == 4 ? 2 : 1)))
void yp_gemm_kernel(const yp_gemm g, const Epi epi) {
  typedef typename yp_type<TYPE>::frag frag;
  typedef typename yp_type<TYPE>::acc accv;
  constexpr int WAVES = WI * WJ, MI = BM / WI / 16, NJ = BN / WJ / 16;
  constexpr int NA = BM / 8, NL = (BM + BN) / 8;            // wave instructions that load A, and all
  constexpr int PER = (NL + WAVES - 1) / WAVES;
  __shared__ __align__(1024) char lds0[(BM + BN) * YP_TILE_KB];
  __shared__ __align__(1024) char lds1[(BM + BN) * YP_TILE_KB];
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
  uint32_t off[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int n = u * WAVES + wave;
    const bool isa = n < NA;
    const int row = (isa ? n : n - NA) * 8 + (lane >> 3);
    const int last = isa ? g.I - 1 - ifirst : g.J - 1 - jfirst;
    off[u] = (uint32_t)min(row, last) * (uint32_t)(isa ? g.lda : g.ldb) + (uint32_t)(((lane & 7) ^ (lane >> 3)) * 16);
  }
  auto load = [&](char* lds, int k) {
    const char* const ak = abase + (int64_t)k * YP_TILE_KB;
    const char* const bk = bbase + (int64_t)k * YP_TILE_KB;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int n = u * WAVES + wave;
      if (NL % WAVES != 0 && n >= NL) break;
      yp_load_lds16((n < NA ? ak : bk) + off[u], lds + n * 1024);
    }
  };

  const int wi = wave % WI, wj = wave / WI;
  accv acc[MI][NJ];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[m][n] = accv{0, 0, 0, 0};

  const int fo = (lane & 15) * YP_TILE_KB + (((lane >> 4) ^ (lane & 7)) * 16);
  const int fa = wi * (BM / WI) * YP_TILE_KB + fo, fb = (BM + wj * (BN / WJ)) * YP_TILE_KB + fo;
  auto compute = [&](const char* lds) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      frag a[MI], b[NJ];
#pragma unroll
      for (int n = 0; n < NJ; ++n) b[n] = *reinterpret_cast<const frag*>(lds + ((fb ^ (h * 64)) + n * 16 * YP_TILE_KB));
#pragma unroll
      for (int m = 0; m < MI; ++m) a[m] = *reinterpret_cast<const frag*>(lds + ((fa ^ (h * 64)) + m * 16 * YP_TILE_KB));
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] = yp_mma<TYPE>(a[m], b[n], acc[m][n]);
    }
  };
  auto arrive = [&]() {   // this wave's loads have landed and its reads are done; then everybody's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (k0 < k1) {
    load(lds0, k0);
    arrive();
    for (int k = k0; k < k1; k += 2) {
      if (k + 1 < k1) load(lds1, k + 1);
      compute(lds0);
      arrive();
      if (k + 1 >= k1) break;
      if (k + 2 < k1) load(lds0, k + 2);
      compute(lds1);
      arrive();
    }
  }
  epi.template apply<TYPE, BM, BN, WI, WJ, MI, NJ>(g, acc, lds0, ti, tj, split, wi, wj, lane);
}
#endif  // __HIPCC__
