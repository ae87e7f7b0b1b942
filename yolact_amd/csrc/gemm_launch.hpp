// Host side of the tile engine: which tile shape a product gets and over how many workgroups its k axis is split,
// and the epilogue that stores a plain product.
#pragma once

#include "gemm_tile.hpp"

struct yp_tile_plan {
  int shape;      // YP_TILE_*
  int bi, bj;     // its tile
  int tiles_i, tiles_j, splits;
};

// L 256 x 256 (4 waves of 128 x 128: 256 rows of fragments read for 128 x 128 results), M 128 x 128 (4 waves of 64 x 64,
// two workgroups a CU), T 64 x 64 (4 waves of 32 x 32, four a CU): the larger, the faster per result once the card is
// full - 1315, 1088 and about 600 TFLOP/s, bf16 - but a small product leaves most of the card idle with it.
static inline yp_tile_plan yp_plan_shape(int shape, int64_t I, int64_t J) {
  yp_tile_plan p;
  p.shape = shape;
  p.bi = p.bj = shape == YP_TILE_L ? 256 : shape == YP_TILE_M ? 128 : 64;
  p.tiles_i = (int)((I + p.bi - 1) / p.bi);
  p.tiles_j = (int)((J + p.bj - 1) / p.bj);
  p.splits = 1;
  return p;
}
// Time of `tiles` tiles of a shape, in units of a 64 x 64 tile at the large shape's rate: rounds of what is resident at a
// time (256 CUs), each as long as the CU's share of them takes.
static inline int64_t yp_plan_cost(int shape, int64_t tiles) {
  if (shape == YP_TILE_L) return (tiles + 255) / 256 * 16;
  if (shape == YP_TILE_M) return tiles <= 256 ? 6 : (tiles + 511) / 512 * 10;
  return tiles <= 256 ? 2 : tiles <= 512 ? 4 : (tiles + 1023) / 1024 * 8;
}
static inline int yp_plan_best(int64_t I1, int64_t J1, int64_t I2, int64_t J2) {   // (J2 = 0: one product)
  int best = YP_TILE_L;
  int64_t least = INT64_MAX;
  for (int s = YP_TILE_L; s <= YP_TILE_T; ++s) {
    const int64_t e = s == YP_TILE_L ? 256 : s == YP_TILE_M ? 128 : 64;
    const int64_t c = yp_plan_cost(s, (I1 + e - 1) / e * ((J1 + e - 1) / e) + (I2 + e - 1) / e * ((J2 + e - 1) / e));
    if (c < least) { least = c; best = s; }
  }
  return best;
}
static inline yp_tile_plan yp_plan_tiles(int64_t I, int64_t J) { return yp_plan_shape(yp_plan_best(I, J, 0, 0), I, J); }
static inline int yp_plan_waves_i(const yp_tile_plan&) { return 2; }

// Few tiles: deal the k axis to more workgroups, until half of the card is busy or a workgroup has 8 steps left.
static inline void yp_plan_splits(yp_tile_plan* p, int64_t steps) {
  const int64_t tiles = (int64_t)p->tiles_i * p->tiles_j, fill = p->shape == YP_TILE_L ? 128 : p->shape == YP_TILE_M ? 256 : 512;
  if (tiles >= fill) return;
  int64_t s = fill / tiles;
  if (s > steps / 8) s = steps / 8;
  p->splits = s < 1 ? 1 : (int)s;
}
// Two products that share a launch, and so a shape.
static inline void yp_plan_two(int64_t I1, int64_t J1, int64_t steps1, int64_t I2, int64_t J2, int64_t steps2, yp_tile_plan* p1, yp_tile_plan* p2) {
  const int shape = yp_plan_best(I1, J1, I2, J2);
  *p1 = yp_plan_shape(shape, I1, J1);
  *p2 = yp_plan_shape(shape, I2, J2);
  yp_plan_splits(p1, steps1);
  yp_plan_splits(p2, steps2);
}

#ifdef __HIPCC__
#define YP_MAX_WORKGROUPS (1 << 24)   // of 256 threads: a launch's work items are counted in 32 bits
static inline yp_gemm yp_with_plan(yp_gemm g, const yp_tile_plan& p) { g.tiles_i = p.tiles_i; g.tiles_j = p.tiles_j; g.splits = p.splits; return g; }
static inline int64_t yp_plan_workgroups(const yp_tile_plan& p) { return (int64_t)p.tiles_i * p.tiles_j * p.splits; }

template <int TYPE, bool SPLIT = false, class Epi>
static hipError_t yp_launch_gemm(const yp_tile_plan& p, const yp_gemm& g0, const Epi& epi, hipStream_t st) {
  const yp_gemm g = yp_with_plan(g0, p);
  if (yp_plan_workgroups(p) >= YP_MAX_WORKGROUPS) return hipErrorInvalidValue;
  const dim3 grid((unsigned)yp_plan_workgroups(p));
  if (p.shape == YP_TILE_L) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, YP_TILE_L, SPLIT, Epi>), grid, dim3(256), 0, st, g, epi);
  else if (p.shape == YP_TILE_M) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, YP_TILE_M, SPLIT, Epi>), grid, dim3(256), 0, st, g, epi);
  else hipLaunchKernelGGL((yp_gemm_kernel<TYPE, YP_TILE_T, SPLIT, Epi>), grid, dim3(256), 0, st, g, epi);
  return hipGetLastError();
}

// (either of the two may be left out: no output)
template <int TYPE, bool SPLIT, class Epi, class Extra>
static hipError_t yp_launch_two(const yp_tile_plan& p1, const yp_gemm& g1, const Epi& e1, const yp_tile_plan& p2, const yp_gemm& g2, const Epi& e2,
                                const Extra& extra, int extras, hipStream_t st) {
  const yp_gemm a = yp_with_plan(g1, p1), b = yp_with_plan(g2, p2);
  if (yp_plan_workgroups(p1) + yp_plan_workgroups(p2) + extras >= YP_MAX_WORKGROUPS) return hipErrorInvalidValue;
  const int n1 = e1.out ? (int)yp_plan_workgroups(p1) : 0, n2 = e2.out ? (int)yp_plan_workgroups(p2) : 0;
  if (n1 + n2 + extras == 0) return hipSuccess;
  const int second_first = b.steps / b.splits > a.steps / a.splits;   // the longer ones first: the short ones fill up the end
  const dim3 grid((unsigned)(n1 + n2 + extras));
  if (p1.shape == YP_TILE_L) hipLaunchKernelGGL((yp_two_gemms_kernel<TYPE, YP_TILE_L, SPLIT, Epi, Extra>), grid, dim3(256), 0, st, a, e1, n1, b, e2, n2, second_first, extra);
  else if (p1.shape == YP_TILE_M) hipLaunchKernelGGL((yp_two_gemms_kernel<TYPE, YP_TILE_M, SPLIT, Epi, Extra>), grid, dim3(256), 0, st, a, e1, n1, b, e2, n2, second_first, extra);
  else hipLaunchKernelGGL((yp_two_gemms_kernel<TYPE, YP_TILE_T, SPLIT, Epi, Extra>), grid, dim3(256), 0, st, a, e1, n1, b, e2, n2, second_first, extra);
  return hipGetLastError();
}

__device__ __forceinline__ float yp_load_as_float(const void* p, int64_t i, int type) {
  return type == YP_F32 ? reinterpret_cast<const float*>(p)[i]
       : type == YP_BF16 ? (float)reinterpret_cast<const __bf16*>(p)[i] : (float)reinterpret_cast<const _Float16*>(p)[i];
}
// A factor that lies on the device: by * (a ? *a : 1) / (count ? max(*count, 1) : 1).
struct yp_scale {
  const float* a;
  const float* count;
  float by;
  __device__ __forceinline__ float get() const { return (a ? *a : 1.0f) * by / (count ? fmaxf(*count, 1.0f) : 1.0f); }
};
// (what is exactly zero stays so, whatever the factor)
__device__ __forceinline__ float yp_times(float v, float scale) { return v == 0.0f ? 0.0f : v * scale; }

// out[j][i] = scale * C, in type OUT; or, with `part`, the f32 sums of this split for a later join
// (part[split][j][i], added to what is there if `add`).
template <int OUT>
struct yp_epi_store {
  void* out;
  int64_t ld;             // elements
  int vec, part_vec;      // rows of out / of part are multiples of 16 bytes
  yp_scale scale;
  float* part;
  int add;
  template <int TYPE, int SHAPE, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], const yp_place& at) const {
    if (part) {
      float* const to = part + (int64_t)at.split * g.J * g.I;
      auto val = [&](int m, int n) { return acc[m][n]; };
      if (add) yp_put_tile<YP_T_F32, SHAPE, true, MI, NJ>(at, to, g.I, g.I, g.J, part_vec != 0, val);
      else yp_put_tile<YP_T_F32, SHAPE, false, MI, NJ>(at, to, g.I, g.I, g.J, part_vec != 0, val);
    } else {
      const float sc = scale.get();
      yp_put_tile<OUT, SHAPE, false, MI, NJ>(at, out, ld, g.I, g.J, vec != 0, [&](int m, int n) {
        yp_f4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = yp_times(acc[m][n][r], sc);
        return v;
      });
    }
  }
};
#endif
