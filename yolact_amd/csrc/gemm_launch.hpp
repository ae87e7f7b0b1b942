// Host side of the tile engine: which tile shape a product gets and over how many workgroups its k axis is split,
// and the epilogue that stores a plain product.
#pragma once

#include "gemm_tile.hpp"

enum { YP_TILE_L = 0, YP_TILE_M = 1, YP_TILE_S = 2 };

struct yp_tile_plan {
  int shape;      // YP_TILE_*
  int bi, bj;     // its tile
  int tiles_i, tiles_j, splits;
};

// L 256 x 256 (4 waves of 128 x 128: 256 rows of fragments read for 128 x 128 results, half of what M reads),
// M 128 x 128 (4 waves of 64 x 64, two workgroups a CU), S 128 x 64 (4 waves of 32 x 64, three workgroups a CU) for few
// rows, where only streaming A counts.  L needs about a full round of tiles; below that M's finer cut wins.
static inline yp_tile_plan yp_plan_tiles(int64_t I, int64_t J, int64_t steps, bool may_split) {
  const int cus = 256;   // MI355X
  yp_tile_plan p;
  const int64_t tl = ((I + 255) / 256) * ((J + 255) / 256);
  p.shape = J <= 64 ? YP_TILE_S : (tl * 4 >= (int64_t)cus * 3 ? YP_TILE_L : YP_TILE_M);
  p.bi = p.shape == YP_TILE_L ? 256 : 128;
  p.bj = p.shape == YP_TILE_L ? 256 : (p.shape == YP_TILE_M ? 128 : 64);
  p.tiles_i = (int)((I + p.bi - 1) / p.bi);
  p.tiles_j = (int)((J + p.bj - 1) / p.bj);
  p.splits = 1;
  const int64_t tiles = (int64_t)p.tiles_i * p.tiles_j;
  if (may_split && tiles < cus) {   // few tiles: deal the k axis to more workgroups, at least 4 steps each
    int64_t s = (2 * cus + tiles - 1) / tiles;
    if (s > steps / 4) s = steps / 4;
    p.splits = s < 1 ? 1 : (int)s;
  }
  return p;
}

#ifdef __HIPCC__
template <int TYPE, class Epi>
static hipError_t yp_launch_gemm(const yp_tile_plan& p, yp_gemm g, const Epi& epi, hipStream_t st) {
  g.tiles_i = p.tiles_i; g.tiles_j = p.tiles_j; g.splits = p.splits;
  const dim3 grid((unsigned)((int64_t)p.tiles_i * p.tiles_j * p.splits));
  if (p.shape == YP_TILE_L) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, 256, 256, 2, 2, 1, Epi>), grid, dim3(256), 0, st, g, epi);
  else if (p.shape == YP_TILE_M) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, 128, 128, 2, 2, 2, Epi>), grid, dim3(256), 0, st, g, epi);
  else hipLaunchKernelGGL((yp_gemm_kernel<TYPE, 128, 64, 4, 1, 3, Epi>), grid, dim3(256), 0, st, g, epi);
  return hipGetLastError();
}

__device__ __forceinline__ float yp_load_as_float(const void* p, int64_t i, int type) {
  return type == YP_F32 ? reinterpret_cast<const float*>(p)[i]
       : type == YP_BF16 ? (float)reinterpret_cast<const __bf16*>(p)[i] : (float)reinterpret_cast<const _Float16*>(p)[i];
}
// four consecutive values at element i of p, the first `n` of them; VEC: the address is aligned to the four of them
template <int TYPE, bool VEC>
__device__ __forceinline__ void yp_store4(void* p, int64_t i, const yp_f4 v, int n) {
  typedef typename yp_type<TYPE>::elem elem;
  typedef elem e4 __attribute__((ext_vector_type(4)));
  elem* const at = reinterpret_cast<elem*>(p) + i;
  if (VEC && n >= 4) {
    *reinterpret_cast<e4*>(at) = e4{(elem)v.x, (elem)v.y, (elem)v.z, (elem)v.w};
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) if (r < n) at[r] = (elem)v[r];
  }
}

// out[j][i] = scale * C, in the operands' type; or, with `part`, the f32 sums of this split for a later join
// (part[split][j][i], added to what is there if `add`).
struct yp_epi_store {
  void* out;
  int64_t ld;             // elements
  int vec;                // ld (for part: I) and out are aligned to four elements
  const float* scale;     // device scalar, null = 1
  float* part;
  int add;
  template <int TYPE, int BM, int BN, bool VEC, bool PART, int MI, int NJ, class Acc>
  __device__ __forceinline__ void put(Acc (&acc)[MI][NJ], void* to, int64_t ldo, int I, int J, int ib, int jb, float sc) const {
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      if (jb + yp_frag_at<BN, NJ>(n) < J) {
        const int64_t row = (int64_t)(jb + yp_frag_at<BN, NJ>(n)) * ldo + ib;
#pragma unroll
        for (int m = 0; m < MI; ++m) {
          const int di = yp_frag_at<BM, MI>(m), left = I - ib - di;
          if (left > 0) {
            yp_f4 v = acc[m][n];
            if (PART) {
              if (add) {
                const float* const at = reinterpret_cast<const float*>(to) + row + di;
                if (VEC && left >= 4) v = v + *reinterpret_cast<const yp_f4*>(at);
                else
#pragma unroll
                  for (int r = 0; r < 4; ++r) if (r < left) v[r] += at[r];
              }
              yp_store4<YP_T_F32, VEC>(to, row + di, v, left);
            } else {
              yp_store4<TYPE, VEC>(to, row + di, v * sc, left);
            }
          }
        }
      }
    }
  }
  template <int TYPE, int BM, int BN, int WI, int WJ, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], int ti, int tj, int split, int wi, int wj, int lane) const {
    const int ib = ti * BM + wi * (BM / 2 / WI) + (lane >> 4) * 4, jb = tj * BN + wj * (BN / 2 / WJ) + (lane & 15);
    if (part) {
      float* const to = part + (int64_t)split * g.J * g.I;
      if (vec) put<TYPE, BM, BN, true, true>(acc, to, g.I, g.I, g.J, ib, jb, 1.0f);
      else put<TYPE, BM, BN, false, true>(acc, to, g.I, g.I, g.J, ib, jb, 1.0f);
    } else {
      const float sc = scale ? *scale : 1.0f;
      if (vec) put<TYPE, BM, BN, true, false>(acc, out, ld, g.I, g.J, ib, jb, sc);
      else put<TYPE, BM, BN, false, false>(acc, out, ld, g.I, g.J, ib, jb, sc);
    }
  }
};
#endif
