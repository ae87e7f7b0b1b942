// Host side of the tile engine: which tile shape a product gets and over how many workgroups its k axis is split,
// and the epilogue that stores a plain product.
#pragma once

#include <math.h>

#include "gemm_tile.hpp"

struct yp_tile_plan {
  int shape;      // YP_TILE_*
  int bi, bj;     // its tile
  int tiles_i, tiles_j, splits;
};

// L 256 x 256 (4 waves of 128 x 128: 256 rows of fragments read for 128 x 128 results), M 128 x 128 (4 waves of 64 x 64,
// two workgroups a CU), T 64 x 64 (4 waves of 32 x 32, five a CU): the larger, the faster per result once the card is
// full - 1315, 1088 and 650 TFLOP/s, bf16 - but a small product leaves most of the card idle with it, and the more
// workgroups share a CU, the better one's epilogue hides behind another's products.
static inline yp_tile_plan yp_plan_shape(int shape, int64_t I, int64_t J) {
  yp_tile_plan p;
  p.shape = shape;
  p.bi = p.bj = shape == YP_TILE_L ? 256 : shape == YP_TILE_M ? 128 : 64;
  p.tiles_i = (int)((I + p.bi - 1) / p.bi);
  p.tiles_j = (int)((J + p.bj - 1) / p.bj);
  p.splits = 1;
  return p;
}
// Microseconds that `wgs` workgroups of `steps` steps each take, fitted to bf16 products from 256 x 256 to 8192 x 8192 with 4
// to 64 steps (within 15 %).  Only the order of the shapes matters, and it holds for int8 and for f32 in planes too: of 14
// products with each shape forced the choice is the fastest of the three, once 3 % behind it - int8 (L, M, T us) 512 x 1024 x
// 1024 20, 9.2, 9.4; 1024 x 1024 x 8192 81, 30, 22; 4096 x 4096 x 4096 69, 75, 106; 8192 x 16384 x 4096 465, 581, 755;
// planes, forward, 1024 x 4096 x 1024 90, 51, 62; 4096 x 32000 x 1024 747, 826, 1198.
static inline double yp_plan_cost(int shape, double wgs, double steps) {
  if (shape == YP_TILE_L) return ceil(wgs / 256) * (steps * (wgs > 128 ? 1.57 : 1.2) + 12);
  if (shape == YP_TILE_M) return wgs <= 256 ? steps * 0.49 + 5 : wgs <= 512 ? steps * 0.79 + 6 : steps * 0.93 * ceil(wgs / 256) / 2 + 6 * ceil(wgs / 512);
  return wgs <= 256 ? steps * 0.28 + 3 : wgs <= 512 ? steps * 0.45 + 3 : wgs <= 1280 ? steps * 0.75 + 4 : steps * 0.92 * wgs / 1280 + 4 * ceil(wgs / 1280);
}
#define YP_MAX_WORKGROUPS (1 << 24)   // of 256 threads: a launch's work items are counted in 32 bits
// `largest`: YP_TILE_M for f32 as it is, else YP_TILE_L.  Smaller shapes only where their workgroups fit a launch.
static inline yp_tile_plan yp_plan_tiles(int64_t I, int64_t J, int64_t steps, int largest) {
  yp_tile_plan best = {};
  double least = 1e30;
  for (int s = largest; s <= YP_TILE_T; ++s) {
    const yp_tile_plan p = yp_plan_shape(s, I, J);
    if (s != largest && (int64_t)p.tiles_i * p.tiles_j >= YP_MAX_WORKGROUPS) continue;
    const double c = yp_plan_cost(s, (double)p.tiles_i * p.tiles_j, (double)steps);
    if (c < least) { least = c; best = p; }
  }
  return best;
}
// Two products that share a launch, and so a shape, each with its k axis dealt to as many workgroups as pays: their
// f32 sums are written and read once more (5 TB/s), by another launch.  A workgroup keeps 8 steps at least.
static inline void yp_plan_two(int64_t I1, int64_t J1, int64_t steps1, int64_t I2, int64_t J2, int64_t steps2, int largest, yp_tile_plan* p1, yp_tile_plan* p2) {
  double least = 1e30;
  for (int shape = largest; shape <= YP_TILE_T; ++shape) {
    yp_tile_plan a = yp_plan_shape(shape, I1, J1), b = yp_plan_shape(shape, I2, J2);
    const double ta = (double)a.tiles_i * a.tiles_j, tb = (double)b.tiles_i * b.tiles_j;
    if (shape != largest && ta + tb >= YP_MAX_WORKGROUPS - (1 << 16)) continue;      // (room for what else the launch does)
    const double alone = shape == YP_TILE_L ? 1.57 : shape == YP_TILE_M ? 0.79 : 0.45;
    for (int64_t sa = 1; sa == 1 || (sa <= steps1 / 8 && ta * sa <= 1024); sa *= 2)
      for (int64_t sb = 1; sb == 1 || (sb <= steps2 / 8 && tb * sb <= 1024); sb *= 2) {
        const double qa = (double)steps1 / sa, qb = (double)steps2 / sb, wgs = ta * sa + tb * sb;
        const double longest = (qa > qb ? qa : qb) * alone + 5;
        // (by k, T reads LDS twice as often as it can: 310 TFLOP/s with the card full)
        double c = (shape == YP_TILE_T && wgs > 512 ? 2.0 : 1.0) * yp_plan_cost(shape, wgs, (ta * sa * qa + tb * sb * qb) / wgs);
        if (c < longest) c = longest;
        if (sa > 1 || sb > 1) c += 6 + ((sa > 1 ? (double)I1 * J1 * sa : 0) + (sb > 1 ? (double)I2 * J2 * sb : 0)) * 8 / 5e6;
        if (c < least) {
          least = c;
          *p1 = a; p1->splits = (int)sa;
          *p2 = b; p2->splits = (int)sb;
        }
      }
  }
}

#ifdef __HIPCC__
static inline yp_gemm yp_with_plan(yp_gemm g, const yp_tile_plan& p) { g.tiles_i = p.tiles_i; g.tiles_j = p.tiles_j; g.splits = p.splits; return g; }
static inline int64_t yp_plan_workgroups(const yp_tile_plan& p) { return (int64_t)p.tiles_i * p.tiles_j * p.splits; }

template <int TYPE, int SEGS = 1, class Epi>
static hipError_t yp_launch_gemm(const yp_tile_plan& p, const yp_gemm& g0, const Epi& epi, hipStream_t st) {
  const yp_gemm g = yp_with_plan(g0, p);
  if (yp_plan_workgroups(p) >= YP_MAX_WORKGROUPS) return hipErrorInvalidValue;
  const dim3 grid((unsigned)yp_plan_workgroups(p));
  if constexpr (TYPE != YP_T_F32) {
    if (p.shape == YP_TILE_L) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, YP_TILE_L, SEGS, Epi>), grid, dim3(256), 0, st, g, epi);
  }
  if (p.shape == YP_TILE_M) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, YP_TILE_M, SEGS, Epi>), grid, dim3(256), 0, st, g, epi);
  if (p.shape == YP_TILE_T) hipLaunchKernelGGL((yp_gemm_kernel<TYPE, YP_TILE_T, SEGS, Epi>), grid, dim3(256), 0, st, g, epi);
  return hipGetLastError();
}

// (either of the two may be left out: no output)
template <int TYPE, int SEGS, class Epi, class Extra>
static hipError_t yp_launch_two(const yp_tile_plan& p1, const yp_gemm& g1, const Epi& e1, const yp_tile_plan& p2, const yp_gemm& g2, const Epi& e2,
                                const Extra& extra, int extras, hipStream_t st) {
  const yp_gemm a = yp_with_plan(g1, p1), b = yp_with_plan(g2, p2);
  if (yp_plan_workgroups(p1) + yp_plan_workgroups(p2) + extras >= YP_MAX_WORKGROUPS) return hipErrorInvalidValue;
  const int n1 = e1.out ? (int)yp_plan_workgroups(p1) : 0, n2 = e2.out ? (int)yp_plan_workgroups(p2) : 0;
  if (n1 + n2 + extras == 0) return hipSuccess;
  const int second_first = b.steps / b.splits > a.steps / a.splits;   // the longer ones first: the short ones fill up the end
  const dim3 grid((unsigned)(n1 + n2 + extras));
  if constexpr (TYPE != YP_T_F32) {
    if (p1.shape == YP_TILE_L) hipLaunchKernelGGL((yp_two_gemms_kernel<TYPE, YP_TILE_L, SEGS, Epi, Extra>), grid, dim3(256), 0, st, a, e1, n1, b, e2, n2, second_first, extra);
  }
  if (p1.shape == YP_TILE_M) hipLaunchKernelGGL((yp_two_gemms_kernel<TYPE, YP_TILE_M, SEGS, Epi, Extra>), grid, dim3(256), 0, st, a, e1, n1, b, e2, n2, second_first, extra);
  if (p1.shape == YP_TILE_T) hipLaunchKernelGGL((yp_two_gemms_kernel<TYPE, YP_TILE_T, SEGS, Epi, Extra>), grid, dim3(256), 0, st, a, e1, n1, b, e2, n2, second_first, extra);
  return hipGetLastError();
}

__device__ __forceinline__ float yp_load_as_float(const void* p, int64_t i, int type) {
  return type == YP_F32 ? reinterpret_cast<const float*>(p)[i]
       : type == YP_BF16 ? (float)reinterpret_cast<const __bf16*>(p)[i] : (float)reinterpret_cast<const _Float16*>(p)[i];
}
// A factor that lies on the device, 2^by * (a ? *a : 1) / (count ? max(*count, 1) : 1) * (more ? 2^*more : 1), as m 2^e with m in
// [1, 2): the factor itself may be outside f32's range where the products that it gives are not.
struct yp_factor { float m; int e; };
__device__ __forceinline__ yp_factor yp_factor_of(float v, int e) {      // v 2^e (0, infinities and NaN stay in m)
  return {2.0f * __builtin_amdgcn_frexp_mantf(v), e + __builtin_amdgcn_frexp_expf(v) - 1};
}
struct yp_scale {
  const float* a;
  const float* count;
  int by;
  const int* more;
  __device__ __forceinline__ yp_factor get() const {
    yp_factor f = yp_factor_of(a ? *a : 1.0f, by + (more ? *more : 0));
    return count ? yp_factor_of(f.m / fmaxf(*count, 1.0f), f.e) : f;
  }
};
__device__ __forceinline__ yp_factor yp_with(const yp_factor& f, float v) {
  const yp_factor x = yp_factor_of(v, f.e);
  return {x.m * f.m, x.e};
}
// (what is exactly zero stays so, whatever the factor)
__device__ __forceinline__ float yp_times(float v, const yp_factor& f) { return v == 0.0f ? 0.0f : __builtin_amdgcn_ldexpf(v * f.m, f.e); }

// out[j][i] = scale * (C + before[j][i]), in type OUT; or, with `part`, the f32 sums of this split for a later join
// (part[split][j][i], added to what is there if `add`).
template <int OUT>
struct yp_epi_store {
  void* out;
  int64_t ld;             // elements
  int vec, part_vec;      // rows of out / of part are multiples of 16 bytes
  yp_scale scale;
  const float* row;       // null, or another factor for every row j (f32 in f16 planes only)
  const float* before;    // null: nothing (16-bit types only: those of f32 lose more to the registers it takes)
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
      const yp_factor sc = scale.get();
      if constexpr (TYPE == YP_T_F16 && OUT == YP_T_F32) {
        if (row) {
          typedef yp_shape<SHAPE> S;
          int i0, j0;
          yp_origin<SHAPE>(at, i0, j0);
          yp_factor f[NJ];
#pragma unroll
          for (int n = 0; n < NJ; ++n) { const int j = j0 + yp_frag_at<S::BN, NJ>(n); f[n] = yp_with(sc, j < g.J ? row[j] : 0.0f); }
          yp_put_tile<OUT, SHAPE, false, MI, NJ>(at, out, ld, g.I, g.J, vec != 0, [&](int m, int n) {
            yp_f4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = yp_times(acc[m][n][r], f[n]);
            return v;
          });
          return;
        }
      }
      if (OUT != YP_T_F32 && before) {
        typedef yp_shape<SHAPE> S;
        int i0, j0;
        yp_origin<SHAPE>(at, i0, j0);
#pragma unroll
        for (int n = 0; n < NJ; ++n)
#pragma unroll
          for (int m = 0; m < MI; ++m) {
            const int i = i0 + yp_frag_at<S::BM, MI>(m), j = j0 + yp_frag_at<S::BN, NJ>(n);
            if (j < g.J && i < g.I) {
              const float* const b = before + (int64_t)j * g.I + i;
              if (part_vec) acc[m][n] = acc[m][n] + *reinterpret_cast<const yp_f4*>(b);      // (I is a multiple of four)
              else
#pragma unroll
                for (int r = 0; r < 4; ++r) if (i + r < g.I) acc[m][n][r] += b[r];
            }
          }
      }
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
