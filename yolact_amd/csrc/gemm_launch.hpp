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

// L 256 x 256 (8 waves of 128 x 64: 192 rows of fragments read for 128 x 64 results - the shape the LDS can feed),
// M 128 x 128 (4 waves of 64 x 64, two workgroups a CU), S 128 x 32 (4 waves of 32 x 32, four workgroups a CU) for few
// rows, where only streaming A counts.  L needs about a full round of tiles; below that M's finer cut wins.
static inline yp_tile_plan yp_plan_tiles(int64_t I, int64_t J, int64_t steps, bool may_split) {
  const int cus = 256;   // MI355X
  yp_tile_plan p;
  const int64_t tl = ((I + 255) / 256) * ((J + 255) / 256);
  p.shape = J <= 32 ? YP_TILE_S : (tl * 4 >= (int64_t)cus * 3 ? YP_TILE_L : YP_TILE_M);
  p.bi = p.shape == YP_TILE_L ? 256 : 128;
  p.bj = p.shape == YP_TILE_L ? 256 : (p.shape == YP_TILE_M ? 128 : 32);
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
  if (p.shape == YP_TILE_L) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, 256, 256, 2, 4, Epi>), grid, dim3(512), 0, st, g, epi);
  else if (p.shape == YP_TILE_M) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, 128, 128, 2, 2, Epi>), grid, dim3(256), 0, st, g, epi);
  else hipLaunchKernelGGL((yp_gemm_kernel<TYPE, 128, 32, 4, 1, Epi>), grid, dim3(256), 0, st, g, epi);
  return hipGetLastError();
}

__device__ __forceinline__ float yp_load_as_float(const void* p, int64_t i, int type) {
  return type == YP_F32 ? reinterpret_cast<const float*>(p)[i]
       : type == YP_BF16 ? (float)reinterpret_cast<const __bf16*>(p)[i] : (float)reinterpret_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void yp_store_from_float(void* p, int64_t i, int type, float v) {
  if (type == YP_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (type == YP_BF16) reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
  else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}
// four consecutive values, the first `n` of them; `vec`: the address is aligned to the four of them
__device__ __forceinline__ void yp_store4(void* p, int64_t i, int type, const yp_f4 v, int n, bool vec) {
  if (vec && n >= 4) {
    if (type == YP_F32) { *reinterpret_cast<yp_f4*>(reinterpret_cast<float*>(p) + i) = v; return; }
    if (type == YP_BF16) {
      typedef __bf16 b4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<b4*>(reinterpret_cast<__bf16*>(p) + i) = b4{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
      return;
    }
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4*>(reinterpret_cast<_Float16*>(p) + i) = h4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) if (r < n) yp_store_from_float(p, i + r, type, v[r]);
}

// out[j][i] = scale * C, in out_type; or, with `part`, the f32 sums of this split for a later join
// (part[split][j][i], added to what is there if `add`).
struct yp_epi_store {
  void* out;
  int64_t ld;             // elements
  int out_type;
  int vec;                // ld and out are aligned to four elements
  const float* scale;     // device scalar, null = 1
  float* part;
  int add;
  template <int TYPE, int BM, int BN, int WI, int WJ, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], char*, int ti, int tj, int split, int wi, int wj, int lane) const {
    const int ib = ti * BM + wi * (BM / WI) + (lane >> 4) * 4, jb = tj * BN + wj * (BN / WJ) + (lane & 15);
    const float sc = scale ? *scale : 1.0f;
    float* const ps = part ? part + (int64_t)split * g.J * g.I : nullptr;
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int j = jb + n * 16;
      if (j >= g.J) continue;
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int i = ib + m * 16, left = g.I - i;
        if (left <= 0) continue;
        if (ps) {
          float* const at = ps + (int64_t)j * g.I + i;
          if (vec && left >= 4) {
            yp_f4 v = acc[m][n];
            if (add) v = v + *reinterpret_cast<const yp_f4*>(at);
            *reinterpret_cast<yp_f4*>(at) = v;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) if (r < left) at[r] = add ? at[r] + acc[m][n][r] : acc[m][n][r];
          }
        } else {
          yp_store4(out, (int64_t)j * ld + i, out_type, acc[m][n] * sc, left, vec != 0);
        }
      }
    }
  }
};
#endif
