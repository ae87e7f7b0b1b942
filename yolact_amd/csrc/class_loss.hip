// Class loss: softmax cross entropy of features h [N,D] against a class matrix w [V,D] (and a bias [V]), for a large V,
// without ever holding the logits, and its gradients.
//
//   z = h w^T + b      lse_n = log sum_v exp z_nv      loss_n = lse_n - z[n, label_n]
//   dz = g_n (exp(z - lse_n) - onehot(label_n))        dh = dz w     dw = dz^T h     db = sum_n dz
//
// A row whose label is the ignored value takes no part: loss 0, no gradient, its features are never multiplied.
// A class whose bias is -inf takes no part either: probability 0, no gradient, its row of w is never multiplied.
// A row whose label is outside [0, V) has loss NaN and no gradient.
//
// Forward: one product on the tile engine whose epilogue reduces a wave's part of the vocabulary to (max, sum exp) per
// row; a second kernel joins the parts.  2 N V D operations, h and w are read, 8 bytes per row and half tile of classes written.
// Backward, per piece of the vocabulary (so that a piece of dz stays in the Infinity Cache): the product again, with an
// epilogue that turns z into dz [row][class]; then both gradient products in one launch, which read dz, h and w as they
// lie ("by k", gemm_tile.hpp): dw's piece is complete, dh adds up over the pieces in f32.
// dz is rounded to the features' type - the matrix instruction takes nothing wider beside h and w; each dz is off by
// half a step of that type, like the gradients themselves.  It is held relative to the largest |g| - one g for all rows
// is taken out altogether -, which the results get back in f32: with g inside, every row's -g would be rounded the same
// way, and sums over rows be off by as much as one of them.  f16 with 2^13 more, so that probabilities down to 2^-38 are
// kept; in the planes of f32 (below) g stays outside altogether: dh's rows get theirs at the end, dw's product
// reads g h instead of h, so that a row of far smaller g keeps its bits.  Where rows are few, their roundings do not average out, and dz has two planes (twice the precision).
// f32 of any size worth it runs on the f16 matrix instructions, as two f16 planes per operand (SPLIT; gemm_tile.hpp): 22 bits
// of a value, or 2^-39 of the largest one where that is more - a value below 2^-17 of the largest has fewer bits than f32,
// its share of a sum over both is as good.  In z, whose sums run along the rows, the largest is the row's own, of h and of w
// alike: each row has an exponent of its own, which its results get back, so no row's logits depend on another row, ignored
// or not.  The gradient products add up over the rows of h, and of w: those have one scale each, another two planes.
// What takes no part has dz = 0, but 0 times NaN is NaN: the gradient products read a copy of h in which ignored rows are
// zero (and of w, if a bias may mask classes).
// All sums are f32 in a fixed order: no float atomics, the same call gives the same bits.
#include "gemm_launch.hpp"

#define YP_CL_THREADS 256
// f32 products of as many multiplications go through f16 planes; below, the exponents and copies cost more.  Forward and backward
// through planes and through the f32 instruction: 1024 x 1024 x 1024 33 + 74 and 29 + 71 us, 76992 x 81 x 256 76 + 182 and
// 55 + 181; 2048 x 1024 x 1024 37 + 97 and 43 + 131, 2048 x 8192 x 1024 112 + 343 and 254 + 772.
#define YP_CL_SPLIT_FROM (1ll << 31)
// Up to as many rows, or as many multiplications, dz has two planes: 12 instead of 8 N V D operations where reading w,
// writing dw or the launches are a good part of the time.  The backward pass in bf16, with two planes and with one: 19248 x 81 x
// 256 46 and 42 us, 1024 x 1024 x 1024 38 and 30, 128 x 32000 x 2048 141 and 109, 512 x 32000 x 2048 380 and 228; past
// the limits 2048 x 1024 x 1024 59 and 40, 1024 x 32000 x 2048 656 and 418.
#define YP_CL_FINE_ROWS 512
#define YP_CL_FINE_WORK (1ll << 30)
#define YP_CL_PIECE_MAX (1 << 17)
#define YP_CL_PIECE_BYTES (256ll << 20)   // of dz: the Infinity Cache (128 MB and 512 MB: up to 10 % slower)

__device__ __forceinline__ int64_t yp_label_at(const void* labels, int64_t n, int bytes) {
  return bytes == 8 ? reinterpret_cast<const int64_t*>(labels)[n] : (int64_t)reinterpret_cast<const int32_t*>(labels)[n];
}

#define YP_LOG2E 1.44269504088896341f
__device__ __forceinline__ float yp_exp_hw(float x) { return __builtin_amdgcn_exp2f(x * YP_LOG2E); }

struct yp_softmax_part { float m, s; };
__device__ __forceinline__ void yp_join(float& m, float& s, float m2, float s2) {
  const float t = fmaxf(m, m2);
  const float ref = t == -INFINITY ? 0.0f : t;
  s = s * yp_exp_hw(m - ref) + s2 * yp_exp_hw(m2 - ref);
  m = t;
}

// what is left of an f32 beside its first plane: exact (nothing beside an infinity or NaN)
template <class E>
__device__ __forceinline__ float yp_plane_rest(float x) {
  const float h = (float)(E)x;
  return fabsf(h) < INFINITY ? x - h : 0.0f;
}

// Of the two planes' rows: a row of f32 whose largest finite magnitude lies in [2^(e-1), 2^e) is held times 2^(15-e), e = 0 for
// one of zeros.  (The integer exponents undo it: products of two float scales would leave f32's range.)
struct yp_row_exponents {
  const int *i, *j;            // [V], of the piece, and [N]; both padded to 256, which is as far as a tile reaches
  template <int SHAPE, int MI, int NJ, class Acc>
  __device__ __forceinline__ void give_back(Acc (&acc)[MI][NJ], int ib, int jb) const {
    typedef yp_shape<SHAPE> S;
    int ej[NJ];
#pragma unroll
    for (int n = 0; n < NJ; ++n) ej[n] = j[jb + yp_frag_at<S::BN, NJ>(n)] - 30;
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      const yp_i4 ei = *reinterpret_cast<const yp_i4*>(i + ib + yp_frag_at<S::BM, MI>(m));
#pragma unroll
      for (int n = 0; n < NJ; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[m][n][r] = __builtin_amdgcn_ldexpf(acc[m][n][r], ei[r] + ej[n]);
    }
  }
};

struct yp_labels {
  const void* labels;
  int bytes;
  int64_t ignore_index;
  int V;
  __device__ __forceinline__ int64_t at(int64_t n) const { return yp_label_at(labels, n, bytes); }
  // the class, or -1: ignored or outside the vocabulary
  __device__ __forceinline__ int counted(int64_t n) const {
    const int64_t l = at(n);
    return l == ignore_index || l < 0 || l >= V ? -1 : (int)l;
  }
};

// ---- epilogue of the forward product: i = class, j = row ----------------------------------------------------------
template <int ELEM, bool SPLIT>
struct yp_epi_stats {
  const void* bias;            // of the tensors' type ELEM, may be null; of the piece
  yp_labels labels;
  int first;                   // first class of the piece
  yp_softmax_part* part;       // [tiles_i * WI][N] of the piece
  float* picked;               // [N] z of the label
  yp_row_exponents exponents;  // SPLIT
  template <int TYPE, int SHAPE, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], const yp_place& at) const {
    typedef yp_shape<SHAPE> S;
    int ib, jb;
    yp_origin<SHAPE>(at, ib, jb);
    if constexpr (SPLIT) exponents.give_back<SHAPE>(acc, ib, jb);
    if (bias || (at.ti + 1) * S::BM > g.I) {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = ib + yp_frag_at<S::BM, MI>(m) + r;
          const float b = i >= g.I ? -INFINITY : (bias ? yp_load_as_float(bias, i, ELEM) : 0.0f);
#pragma unroll
          for (int n = 0; n < NJ; ++n) acc[m][n][r] = b == -INFINITY ? -INFINITY : acc[m][n][r] + b;
        }
    }
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int j = jb + yp_frag_at<S::BN, NJ>(n);
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[m][n][r]);
      // (c finite: -inf, a class that takes no part, stays -inf also beside logits of the lowest value)
      const float ref = top == -INFINITY ? 0.0f : top, c = fminf(-ref * YP_LOG2E, 0x1.fffffep127f);
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[m][n][r], YP_LOG2E, c));
      // between 1 and the number of terms, whatever the rounding of c makes of it (2^-24 of ref: for 10^9, anything)
      if (top != -INFINITY) sum = sum < 1.0f ? 1.0f : sum > MI * 4.0f ? MI * 4.0f : sum;
      const int64_t l = j < g.J ? labels.at(j) - first - ib : -1;
      const bool mine = l >= 0 && l < S::BM;
      if (__builtin_amdgcn_ballot_w64(mine)) {      // (mostly no lane of the wave)
        const int at_l = mine ? (int)l : -1;
        float z = 0.0f;
        bool found = false;
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool is = at_l == yp_frag_at<S::BM, MI>(m) + r;
            z = is ? acc[m][n][r] : z;
            found |= is;
          }
        if (found) picked[j] = z;
      }
#pragma unroll
      for (int x = 16; x < 64; x <<= 1) yp_join(top, sum, __shfl_xor(top, x), __shfl_xor(sum, x));
      if (j < g.J && at.lane < 16) part[(int64_t)(at.ti * S::WI + at.wi) * g.J + j] = yp_softmax_part{top, sum};
    }
  }
};

// ---- epilogue of the backward product -----------------------------------------------------------------------------
// What g is held by, relative to the largest |g| = m 2^e, m in [1, 2), of the rows that take part (and whose g is finite: what an
// infinity gives is no matter of scale): g 2^-e (2^up / m), and the results get m 2^-up 2^e back.
struct yp_relative { float by, back; int e; };
template <int ELEM, bool SPLIT, int PLANES>
struct yp_epi_dz {
  const void* bias;            // of the tensors' type ELEM; of the piece
  const float* lse;
  yp_labels labels;
  const float* grad;           // of every row, as `relative` says (if there is one); null: `up` for all of them.  SPLIT: `up`
                               // for all of them in dz, `grad` in the bias gradient only
  const yp_relative* relative;
  float up;
  yp_scale scale;              // what the bias gradient gets back
  yp_row_exponents exponents;  // SPLIT
  int first;                   // first class of the piece
  void* dz;                    // [kn][kv], zero in [N, kn) and [V, kv); or PLANES of it
  int64_t plane;               // bytes of one
  int kv, kn;
  void* bias_out;              // of the piece; null without bias
  float* bias_part;            // [tiles_j][classes of the piece] if there is more than one tile in j, else null
  template <int TYPE, int SHAPE, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], const yp_place& at) const {
    typedef yp_shape<SHAPE> S;
    typedef typename yp_type<ELEM>::elem elem;
    int ib, jb;
    yp_origin<SHAPE>(at, ib, jb);
    const yp_relative held = relative ? *relative : yp_relative{1.0f, 1.0f, 0};
    float own[NJ];
    if constexpr (SPLIT) exponents.give_back<SHAPE>(acc, ib, jb);
    if (bias || (at.ti + 1) * S::BM > g.I) {      // a class that takes no part, or does not exist: z = -inf
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = ib + yp_frag_at<S::BM, MI>(m) + r;
          const float b = i >= g.I ? -INFINITY : (bias ? yp_load_as_float(bias, i, ELEM) : 0.0f);
#pragma unroll
          for (int n = 0; n < NJ; ++n) acc[m][n][r] = b == -INFINITY ? -INFINITY : acc[m][n][r] + b;
        }
    }
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int j = jb + yp_frag_at<S::BN, NJ>(n);
      const int label = j < g.J ? labels.counted(j) : -1;
      const float l = label >= 0 ? lse[j] : INFINITY;
      // exp(z - lse) = 2^min(z log2e + c, 0) - rounding may bring z above lse, by any amount where large products cancel -; a
      // row that takes no part, or has no class left: 2^-inf = 0; one with NaN among its z has it in lse, and here in gr
      const float gr = label < 0 ? 0.0f : l != l ? l : grad && !SPLIT ? __builtin_amdgcn_ldexpf(grad[j], -held.e) * held.by : up;
      own[n] = SPLIT && grad && label >= 0 ? grad[j] : 1.0f;
      const float c = fabsf(l) == INFINITY ? -INFINITY : __builtin_amdgcn_fmed3f(-l * YP_LOG2E, -0x1.fffffep127f, 0x1.fffffep127f);
      const int hit = label < 0 ? -1 : label - first - ib;
      if (__builtin_amdgcn_ballot_w64(hit >= 0 && hit < S::BM)) {      // (mostly no lane of the wave)
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float z = acc[m][n][r], p = __builtin_amdgcn_exp2f(fminf(__builtin_fmaf(z, YP_LOG2E, c), 0.0f));
            acc[m][n][r] = (hit == yp_frag_at<S::BM, MI>(m) + r && z != -INFINITY ? p - 1.0f : p) * gr;
          }
      } else {
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[m][n][r] = __builtin_amdgcn_exp2f(fminf(__builtin_fmaf(acc[m][n][r], YP_LOG2E, c), 0.0f)) * gr;
      }
    }
    if (bias_out) {   // sums over the tile's rows: 16 lanes, then the waves that share the classes
      float* const lds = reinterpret_cast<float*>(at.lds);
      const int il = at.wi * (S::BM / 2 / S::WI) + (at.lane >> 4) * 4;
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float col = 0.0f;
#pragma unroll
          for (int n = 0; n < NJ; ++n) col += SPLIT ? acc[m][n][r] * own[n] : acc[m][n][r];
#pragma unroll
          for (int x = 1; x < 16; x <<= 1) col += __shfl_xor(col, x);
          if ((at.lane & 15) == 0) lds[at.wj * S::BM + il + yp_frag_at<S::BM, MI>(m) + r] = col;
        }
      yp_arrive<0>();
      for (int t = (int)threadIdx.x; t < S::BM; t += 256) {
        const int i = at.ti * S::BM + t;
        float col = 0.0f;
#pragma unroll
        for (int w = 0; w < S::WJ; ++w) col += lds[w * S::BM + t];
        if (i < g.I) {
          if (bias_part) bias_part[(int64_t)at.tj * g.I + i] = col;
          else reinterpret_cast<elem*>(bias_out)[i] = (elem)yp_times(col, scale.get());
        }
      }
      yp_arrive<0>();
    }
    yp_put_tile<TYPE, SHAPE, false, MI, NJ>(at, dz, kv, kv, kn, true, [&](int m, int n) { return acc[m][n]; });
    if constexpr (PLANES == 2) {
      yp_arrive<0>();
      yp_put_tile<TYPE, SHAPE, false, MI, NJ>(at, (char*)dz + plane, kv, kv, kn, true, [&](int m, int n) {
        yp_f4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = yp_plane_rest<typename yp_type<TYPE>::elem>(acc[m][n][r]);
        return v;
      });
    }
  }
};

// ---- the small kernels around the products ------------------------------------------------------------------------
// Up to two matrices copied to rows of `kb` bytes with a zero tail, and to `rows_out` rows with zero rows at the end.  A
// row that takes no part - its label is ignored, its bias -inf - is written as zeros: whatever it holds, it meets only
// zeros in a product.
struct yp_copy_job {
  const char* src;
  char* dst;
  int64_t row_bytes, kb, rows, rows_out;
  int vec;                // rows of src are multiples of 16 bytes and so is their address
  int by_label;
  const void* bias;
  int64_t plane;          // 0, or: f32 rows to two f16 planes, this many bytes apart (row_bytes, kb: of a plane's row),
  const int* exponent;    //   each held by its own exponent (yp_row_exponents)
  char* common;           //   and, unless null, to two more, times 2^-*back: for products that add up over the rows;
  const int* back;
  const float* grad;      //   and times this of its row, unless null
};
struct yp_copy_args {
  yp_copy_job job[2];
  int64_t chunks0;        // 16-byte chunks of the first job
  int64_t chunks;         // of both
  yp_labels labels;
  int type;
};
// (PLANES apart: the few rows of 16-bit copies that a thread takes waited for its registers and arguments, 22 -> 38 us, 30011 x 1000)
template <bool PLANES>
__global__ __launch_bounds__(YP_CL_THREADS) void yp_copy_rows_kernel(const yp_copy_args a) {
  for (int64_t e = (int64_t)blockIdx.x * YP_CL_THREADS + threadIdx.x; e < a.chunks; e += (int64_t)gridDim.x * YP_CL_THREADS) {
    const bool second = e >= a.chunks0;
    const yp_copy_job& j = a.job[second];
    const int64_t c = second ? e - a.chunks0 : e;
    const int per = (int)(j.kb / 16);
    const int64_t r = c / per;
    const int at = (int)(c - r * per) * 16;
    bool in = r < j.rows;
    if (in && j.by_label) in = a.labels.counted(r) >= 0;
    if (in && j.bias) in = yp_load_as_float(j.bias, r, a.type) != -INFINITY;
    if constexpr (PLANES) {        // 8 elements
      const int up = in ? 15 - j.exponent[r] : 0;
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = 0.0f;
      if (in) {
        const char* const s = j.src + (r * j.row_bytes + at) * 2;
        if (j.vec && at + 16 <= j.row_bytes) {
          const yp_f4 lo = reinterpret_cast<const yp_f4*>(s)[0], hi = reinterpret_cast<const yp_f4*>(s)[1];
#pragma unroll
          for (int u = 0; u < 4; ++u) { x[u] = lo[u]; x[4 + u] = hi[u]; }
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u) if (at + 2 * u < j.row_bytes) x[u] = reinterpret_cast<const float*>(s)[u];
        }
      }
      auto put = [&](char* dst, auto val) {
        float y[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = val(x[u]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          yp_h8 o;
#pragma unroll
          for (int u = 0; u < 8; ++u) { o[u] = (_Float16)y[u]; y[u] = yp_plane_rest<_Float16>(y[u]); }
          *reinterpret_cast<yp_h8*>(dst + q * j.plane + r * j.kb + at) = o;
        }
      };
      put(j.dst, [&](float v) { return __builtin_amdgcn_ldexpf(v, up); });
      if (j.common) {
        // (the product of the row as it is held and the gradient's mantissa: neither leaves f32's range on the way)
        const float gr = j.grad && in ? j.grad[r] : 1.0f, gm = __builtin_amdgcn_frexp_mantf(gr);
        const int by = __builtin_amdgcn_frexp_expf(gr) - up - *j.back;
        put(j.common, [&](float v) { return __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(v, up) * gm, by); });
      }
      continue;
    }
    yp_i4 v = {0, 0, 0, 0};
    if (in) {
      const char* const s = j.src + r * j.row_bytes + at;
      if (j.vec && at + 16 <= j.row_bytes) v = *reinterpret_cast<const yp_i4*>(s);
      else if (a.type == YP_F32) {
#pragma unroll
        for (int u = 0; u < 4; ++u) if (at + 4 * u < j.row_bytes) v[u] = *reinterpret_cast<const int*>(s + 4 * u);
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (at + 2 * u < j.row_bytes) v[u >> 1] |= (int)((uint32_t) * reinterpret_cast<const uint16_t*>(s + 2 * u) << (16 * (u & 1)));
      }
    }
    *reinterpret_cast<yp_i4*>(j.dst + r * j.kb + at) = v;
  }
}

// The exponents of all rows of features and weight (yp_row_exponents), a wave a row; and, unless `part` is null, the largest of
// either among the rows that take part, a part per workgroup, for back[0] and [1]: times 2^-back, those rows' largest finite
// magnitude (times its row's `grad`, if there is one) lies in [2^14, 2^15).
#define YP_NO_EXPONENT (-100000)
struct yp_peak_args {
  const float* src[2];
  int64_t rows[2];
  int d, vec;
  yp_labels labels;            // of the first
  const float* bias;           // of the second, may be null
  const float* grad;           // of the first, may be null
  int* exponent[2];
  int* part;                   // [2][YP_PEAK_BLOCKS], may be null; YP_NO_EXPONENT: only zeros
};
#define YP_PEAK_BLOCKS 2048
__global__ __launch_bounds__(YP_CL_THREADS) void yp_peak_kernel(const yp_peak_args a) {
  __shared__ int red[YP_CL_THREADS / 64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int most = YP_NO_EXPONENT;
    for (int64_t r = (int64_t)blockIdx.x * (YP_CL_THREADS / 64) + wave; r < a.rows[j]; r += YP_PEAK_BLOCKS * (YP_CL_THREADS / 64)) {
      const float* const p = a.src[j] + r * a.d;
      float top = 0.0f;
      auto see = [&](float v) { v = fabsf(v); top = fmaxf(top, v < INFINITY ? v : 0.0f); };
      int c = lane * 4;
      if (a.vec) {
        for (; c + 768 < a.d; c += 1024) {      // four loads in flight
          yp_f4 v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const yp_f4*>(p + c + u * 256);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) see(v[u][e]);
        }
        for (; c < a.d; c += 256) {
          const yp_f4 v = *reinterpret_cast<const yp_f4*>(p + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) see(v[e]);
        }
      } else {
        for (c = lane; c + 448 < a.d; c += 512) {
          float v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = p[c + u * 64];
#pragma unroll
          for (int u = 0; u < 8; ++u) see(v[u]);
        }
        for (; c < a.d; c += 64) see(p[c]);
      }
#pragma unroll
      for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
      const int e = __builtin_amdgcn_frexp_expf(top);      // (0 of 0)
      if (lane == 0) a.exponent[j][r] = e;
      if (a.part && top > 0.0f && (j == 0 ? a.labels.counted(r) >= 0 : !a.bias || a.bias[r] != -INFINITY)) {
        const float g = j == 0 && a.grad ? fabsf(a.grad[r]) : 1.0f;
        if (g > 0.0f && g < INFINITY)       // the product's exponent, without the product: f32's range may be too small for it
          most = max(most, e + __builtin_amdgcn_frexp_expf(g) + __builtin_amdgcn_frexp_expf(__builtin_amdgcn_frexp_mantf(top) * __builtin_amdgcn_frexp_mantf(g)));
      }
    }
    if (!a.part) continue;
    __syncthreads();
    if (lane == 0) red[wave] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < YP_CL_THREADS / 64; ++w) most = max(most, red[w]);
      a.part[j * YP_PEAK_BLOCKS + blockIdx.x] = most;
    }
  }
}
// (a wave each, its loads all in flight: one after the other they took 10 us)
__global__ __launch_bounds__(128) void yp_back_kernel(const int* part, int* back) {
  const int lane = (int)threadIdx.x & 63, j = (int)threadIdx.x >> 6;
  yp_i4 v[YP_PEAK_BLOCKS / 256];
#pragma unroll
  for (int i = 0; i < YP_PEAK_BLOCKS / 256; ++i) v[i] = reinterpret_cast<const yp_i4*>(part + j * YP_PEAK_BLOCKS)[i * 64 + lane];
  int most = YP_NO_EXPONENT;
#pragma unroll
  for (int i = 0; i < YP_PEAK_BLOCKS / 256; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) most = max(most, v[i][e]);
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) most = max(most, __shfl_xor(most, x));
  if (lane == 0) back[j] = most == YP_NO_EXPONENT ? 0 : most - 15;
}

__device__ __forceinline__ double yp_block_sum(double v, double* lds) {   // fixed order; result in thread 0
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) v += __shfl_xor(v, x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x == 0) for (int w = 0; w < (int)blockDim.x / 64; ++w) t += lds[w];
  return t;
}

struct yp_reduced {
  float *sum, *mean, *count;     // any may be null
  __host__ __device__ bool wanted() const { return sum || mean || count; }
  __device__ __forceinline__ void put(double s, double c) const {
    if (sum) *sum = (float)s;
    if (mean) *mean = c > 0.0 ? (float)(s / c) : 0.0f;
    if (count) *count = (float)c;
  }
};

struct yp_join_args {
  const yp_softmax_part* part;
  int parts;
  const float* picked;
  yp_labels labels;
  int N;
  float *losses, *lse;
  yp_reduced reduced;
  double* block_part;       // [blocks][2]
};
// Joins the parts of the rows, and the sum of their losses if it is asked for.
template <int RPB>   // rows per workgroup and turn; YP_CL_THREADS / RPB threads a row
__global__ __launch_bounds__(YP_CL_THREADS) void yp_join_kernel(const yp_join_args a) {
  constexpr int TPR = YP_CL_THREADS / RPB;
  __shared__ float lm[TPR][RPB], ls[TPR][RPB];
  __shared__ double red[YP_CL_THREADS / 64];
  const int x = (int)threadIdx.x % RPB, y = (int)threadIdx.x / RPB;
  double loss = 0.0, count = 0.0;
  for (int n0 = (int)blockIdx.x * RPB; n0 < a.N; n0 += (int)gridDim.x * RPB) {
    const int n = n0 + x;
    float m = -INFINITY, s = 0.0f;
    if (n < a.N) {
      const yp_softmax_part* const col = a.part + n;
      int p = y;
      for (; p + 3 * TPR < a.parts; p += 4 * TPR) {     // four loads in flight
        yp_softmax_part v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = col[(int64_t)(p + u * TPR) * a.N];
#pragma unroll
        for (int u = 0; u < 4; ++u) yp_join(m, s, v[u].m, v[u].s);
      }
      for (; p < a.parts; p += TPR) {
        const yp_softmax_part v = col[(int64_t)p * a.N];
        yp_join(m, s, v.m, v.s);
      }
    }
    __syncthreads();
    lm[y][x] = m; ls[y][x] = s;
    if constexpr (TPR > 8) {                            // 8 threads gather the others'
      __syncthreads();
      if (y < 8) {
        for (int u = y + 8; u < TPR; u += 8) yp_join(m, s, lm[u][x], ls[u][x]);
        lm[y][x] = m; ls[y][x] = s;
      }
    }
    __syncthreads();
    if (y == 0 && n < a.N) {
      for (int u = 1; u < 8; ++u) yp_join(m, s, lm[u][x], ls[u][x]);
      const float l = m + logf(s);
      const int64_t lab = a.labels.at(n);
      float v = 0.0f;
      if (lab != a.labels.ignore_index) {
        const float p = lab < 0 || lab >= a.labels.V ? NAN : a.picked[n];
        v = p == -INFINITY ? INFINITY : l - p;
        loss += v;
        count += 1.0;
      }
      a.lse[n] = l;
      if (a.losses) a.losses[n] = v;
    }
  }
  if (!a.reduced.wanted()) return;
  const double ts = yp_block_sum(loss, red), tc = yp_block_sum(count, red);
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) a.reduced.put(ts, tc);
    else { a.block_part[2 * blockIdx.x] = ts; a.block_part[2 * blockIdx.x + 1] = tc; }
  }
}
__global__ __launch_bounds__(YP_CL_THREADS) void yp_reduce_kernel(const double* block_part, int blocks, const yp_reduced reduced) {
  __shared__ double red[YP_CL_THREADS / 64];
  double s = 0.0, c = 0.0;
  for (int i = (int)threadIdx.x; i < blocks; i += YP_CL_THREADS) { s += block_part[2 * i]; c += block_part[2 * i + 1]; }
  const double ts = yp_block_sum(s, red), tc = yp_block_sum(c, red);
  if (threadIdx.x == 0) reduced.put(ts, tc);
}

__global__ __launch_bounds__(1024) void yp_relative_kernel(const float* grad, const yp_labels labels, int64_t n, int up, yp_relative* out) {
  __shared__ float red[16];
  float top = 0.0f;
  auto see = [&](float v, int label) {
    v = fabsf(v);
    top = fmaxf(top, label >= 0 && v < INFINITY ? v : 0.0f);
  };
  int64_t i = threadIdx.x;
  for (; i + 3 * 1024 < n; i += 4 * 1024) {
    float v[4];
    int l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) { v[u] = grad[i + u * 1024]; l[u] = labels.counted(i + u * 1024); }
#pragma unroll
    for (int u = 0; u < 4; ++u) see(v[u], l[u]);
  }
  for (; i < n; i += 1024) see(grad[i], labels.counted(i));
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) top = fmaxf(top, red[w]);
    const yp_factor f = yp_factor_of(top > 0.0f ? top : 1.0f, 0);      // (1: nothing to go by)
    *out = {__builtin_amdgcn_ldexpf(1.0f, up) / f.m, __builtin_amdgcn_ldexpf(f.m, -up), f.e};
  }
}

// The bias gradient: the tiles' column sums added up, 32 classes of 8 threads in workgroup i of those that follow the gradient
// products (one thread a class waited 40 us for its 151 loads, 19248 rows).
struct yp_bias_sum {
  static constexpr int CLASSES = 32, GROUPS = 256 / CLASSES;
  const float* part;   // [parts][total]
  int parts, total, type;
  yp_scale scale;
  void* out;
  __device__ __forceinline__ void operator()(int i, char* lds) const {
    float(*const red)[CLASSES] = reinterpret_cast<float(*)[CLASSES]>(lds);
    const int x = (int)threadIdx.x % CLASSES, y = (int)threadIdx.x / CLASSES, e = i * CLASSES + x;
    float s = 0.0f;
    if (e < total) {
      int p = y;
      for (; p + 3 * GROUPS < parts; p += 4 * GROUPS) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = part[(int64_t)(p + u * GROUPS) * total + e];
#pragma unroll
        for (int u = 0; u < 4; ++u) s += v[u];
      }
      for (; p < parts; p += GROUPS) s += part[(int64_t)p * total + e];
    }
    red[y][x] = s;
    __syncthreads();
    if (y == 0 && e < total) {
      for (int u = 1; u < GROUPS; ++u) s += red[u][x];
      s = yp_times(s, scale.get());
      if (type == YP_F32) reinterpret_cast<float*>(out)[e] = s;
      else if (type == YP_BF16) reinterpret_cast<__bf16*>(out)[e] = (__bf16)s;
      else reinterpret_cast<_Float16*>(out)[e] = (_Float16)s;
    }
  }
};

// Up to two arrays, each out[e] = its scale * sum over its parts.  64 elements and 4 waves a workgroup: wave w adds parts
// w, w + 4, ... in their order, then the four sums are added in theirs.
struct yp_sum_job {
  const float* part; int parts; int64_t total; void* out; yp_scale scale;
  const float* row; int cols;      // null, or another factor for every row of as many elements
};
struct yp_sum_args { yp_sum_job job[2]; int jobs, out_type; };
__global__ __launch_bounds__(YP_CL_THREADS) void yp_sum_parts_kernel(const yp_sum_args a) {
  __shared__ float red[YP_CL_THREADS / 64][64];
  const int x = (int)threadIdx.x & 63, y = (int)threadIdx.x >> 6;
  for (int j = 0; j < a.jobs; ++j) {
    const yp_sum_job& b = a.job[j];
    const yp_factor sc = b.scale.get();
    auto put = [&](int64_t e, float s) {
      s = yp_times(s, b.row ? yp_with(sc, b.row[e / b.cols]) : sc);
      if (a.out_type == YP_F32) reinterpret_cast<float*>(b.out)[e] = s;
      else if (a.out_type == YP_BF16) reinterpret_cast<__bf16*>(b.out)[e] = (__bf16)s;
      else reinterpret_cast<_Float16*>(b.out)[e] = (_Float16)s;
    };
    if (b.parts < 4) {   // (or none: zeros) a thread an element
      for (int64_t e = (int64_t)blockIdx.x * YP_CL_THREADS + threadIdx.x; e < b.total; e += (int64_t)gridDim.x * YP_CL_THREADS) {
        float s = 0.0f;
        for (int p = 0; p < b.parts; ++p) s += b.part[(int64_t)p * b.total + e];
        put(e, s);
      }
      continue;
    }
    for (int64_t e0 = (int64_t)blockIdx.x * 64; e0 < b.total; e0 += (int64_t)gridDim.x * 64) {
      const int64_t e = e0 + x;
      float s = 0.0f;
      if (e < b.total) {
        int p = y;
        for (; p + 12 < b.parts; p += 16) {
          float v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = b.part[(int64_t)(p + 4 * u) * b.total + e];
#pragma unroll
          for (int u = 0; u < 4; ++u) s += v[u];
        }
        for (; p < b.parts; p += 4) s += b.part[(int64_t)p * b.total + e];
      }
      __syncthreads();
      red[y][x] = s;
      __syncthreads();
      if (y == 0 && e < b.total) put(e, ((red[0][x] + red[1][x]) + red[2][x]) + red[3][x]);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------
static inline int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
static inline int type_bytes(int t) { return t == YP_F32 ? 4 : 2; }
static inline unsigned blocks_for(int64_t n, int per, int64_t most) { const int64_t b = (n + per - 1) / per; return (unsigned)(b < 1 ? 1 : b > most ? most : b); }

static hipError_t sum_parts(const yp_sum_args& a, hipStream_t st) {
  int64_t most = 0;
  for (int j = 0; j < a.jobs; ++j) {
    const int64_t b = (a.job[j].total + 63) / 64 / (a.job[j].parts < 4 ? 4 : 1);
    most = b > most ? b : most;
  }
  if (a.jobs == 0) return hipSuccess;
  hipLaunchKernelGGL(yp_sum_parts_kernel, dim3(blocks_for(most, 1, 8192)), dim3(YP_CL_THREADS), 0, st, a);
  return hipGetLastError();
}
static void add_sum(yp_sum_args& a, const float* part, int parts, int64_t total, void* out, const yp_scale& scale, const float* row, int cols) {
  a.job[a.jobs++] = yp_sum_job{part, parts, total, out, scale, row, cols};
}
static hipError_t zero(void* out, int64_t n, int type, hipStream_t st) {   // (a kernel, not a memset: the call may be captured)
  yp_sum_args a = {};
  a.out_type = type;
  add_sum(a, nullptr, 0, n, out, yp_scale{nullptr, nullptr, 0, nullptr}, nullptr, 1);
  return sum_parts(a, st);
}

// The launch plan of a call, from its sizes alone: the same for yp_class_loss_workspace and for the call.
struct ClassLossPlan {
  bool split;                  // f32 in two f16 planes
  int b, planes;               // bytes of an element of what the products read, and its planes
  int dzplanes, segs;          // planes of dz, segments of the gradient products
  int64_t kd;                  // bytes of a padded feature row
  int fwd_pieces, fwd_piece;   // forward: pieces of the vocabulary if w is copied, else one
  yp_tile_plan fwd;            // of a whole piece
  int parts;                   // per piece
  int pieces, piece;           // backward: pieces of the vocabulary and their width
  int64_t kn, kv;              // rows of dz padded to a step, elements; bytes of a row
  yp_tile_plan dzp, dwp, dhp;
  // workspace offsets
  int64_t o_eh, o_ew;          // both passes
  int64_t o_back, o_peaks;   // backward
  int64_t o_h, o_w, o_part, o_picked, o_block, fwd_total;
  int64_t o_relative, o_hc, o_wc, o_hs, o_ws, o_dz, o_bp, o_dwpart, o_dhpart, bwd_total;
};

static void cut_pieces(int64_t V, int64_t most, int* pieces, int* piece) {   // equal pieces, multiples of 256
  most = most / 256 * 256;
  if (most < 256) most = 256;
  if (most > YP_CL_PIECE_MAX) most = YP_CL_PIECE_MAX;
  int64_t n = (V + most - 1) / most, w = V;
  if (n > 1) { w = ((V + n - 1) / n + 255) / 256 * 256; n = (V + w - 1) / w; }
  *pieces = (int)n;
  *piece = (int)w;
}

static ClassLossPlan plan_class_loss(int64_t N, int64_t V, int64_t D, int type, bool has_bias, bool copy_fwd) {
  ClassLossPlan p;
  p.split = type == YP_F32 && N * V >= YP_CL_SPLIT_FROM / D;
  const int b = p.split ? 2 : type_bytes(type), planes = p.split ? 2 : 1;
  p.b = b;
  p.planes = planes;
  p.dzplanes = p.split || (type != YP_F32 && (N <= YP_CL_FINE_ROWS || N * V <= YP_CL_FINE_WORK / D)) ? 2 : 1;
  p.segs = p.split ? 3 : p.dzplanes;
  copy_fwd = copy_fwd || p.split;
  p.kd = yp_pad_k(D, b);
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = up256(off + bytes); return o; };
  p.o_eh = take(p.split ? up256(N) * 4 : 0);
  p.o_ew = take(p.split ? up256(V) * 4 : 0);
  const int64_t both = off;
  if (copy_fwd) cut_pieces(V, YP_CL_PIECE_BYTES / (p.kd * planes), &p.fwd_pieces, &p.fwd_piece);
  else { p.fwd_pieces = 1; p.fwd_piece = (int)V; }
  const int largest = type == YP_F32 && !p.split ? YP_TILE_M : YP_TILE_L;
  const int64_t dsteps = p.kd / YP_TILE_KB * (p.split ? 3 : 1);
  p.fwd = yp_plan_tiles(p.fwd_piece, N, dsteps, largest);
  p.parts = p.fwd.tiles_i * 2;
  p.o_h = take(copy_fwd ? N * p.kd * planes : 0);
  p.o_w = take(copy_fwd ? p.fwd_piece * p.kd * planes : 0);
  p.o_part = take((int64_t)p.fwd_pieces * p.parts * N * sizeof(yp_softmax_part));
  p.o_picked = take(N * 4);
  p.o_block = take((N <= 1024 ? (N + 1) / 2 : N <= 4096 ? (N + 7) / 8 : (N + 31) / 32) * 16);
  p.fwd_total = off;

  off = both;
  const int kr = YP_TILE_KB / b;
  p.kn = (N + kr - 1) / kr * kr;
  int64_t most = YP_CL_PIECE_BYTES / (p.kn * b * p.dzplanes);
  if (most > YP_CL_PIECE_BYTES / (p.kd * planes)) most = YP_CL_PIECE_BYTES / (p.kd * planes);
  cut_pieces(V, most, &p.pieces, &p.piece);
  p.kv = yp_pad_k(p.piece, b);
  // (two planes of dz to write: M's epilogues hide better.  The backward pass, 2048 x 8192 x 1024: 347 us, with L 355;
  // 4096 x 32000 x 1024: 2300 and 2323; the same where the plan takes M anyway)
  p.dzp = p.split ? yp_plan_shape(YP_TILE_M, p.piece, p.kn) : yp_plan_tiles(p.piece, p.kn, dsteps, largest);
  // the two gradient products share a launch and so a tile shape
  yp_plan_two(D, p.piece, p.kn / kr * p.segs, D, N, p.kv / YP_TILE_KB * p.segs, largest, &p.dwp, &p.dhp);
  p.o_back = take(p.split ? 8 : 0);
  p.o_peaks = take(p.split ? 2 * YP_PEAK_BLOCKS * 4 : 0);
  p.o_relative = take(sizeof(yp_relative));
  p.o_hc = take(p.kn * p.kd * planes);
  p.o_wc = take(p.piece * p.kd * planes);
  p.o_hs = take(p.split ? p.kn * p.kd * planes : 0);
  p.o_ws = take(p.split ? p.piece * p.kd * planes : 0);
  p.o_dz = take(p.kn * p.kv * p.dzplanes);
  p.o_bp = take(has_bias && p.dzp.tiles_j > 1 ? (int64_t)p.dzp.tiles_j * p.piece * 4 : 0);
  p.o_dwpart = take(p.dwp.splits > 1 ? (int64_t)p.dwp.splits * p.piece * D * 4 : 0);
  p.o_dhpart = take(p.dhp.splits > 1 || p.pieces > 1 ? (int64_t)p.dhp.splits * N * D * 4 : 0);
  p.bwd_total = off;
  return p;
}

int64_t yp_class_loss_bytes(int64_t n, int64_t v, int64_t d, int type, int has_bias, int backward) {
  const ClassLossPlan a = plan_class_loss(n, v, d, type, has_bias != 0, false);
  if (backward) return a.bwd_total;
  const ClassLossPlan c = plan_class_loss(n, v, d, type, has_bias != 0, true);   // (rows that need a copy: known at the call)
  return a.fwd_total > c.fwd_total ? a.fwd_total : c.fwd_total;
}

#define CL_TRY(...) do { const hipError_t e_ = (__VA_ARGS__); if (e_ != hipSuccess) return e_; } while (0)

static yp_copy_job copy_job(const void* src, char* dst, int64_t d, const ClassLossPlan& p, int64_t rows, int64_t rows_out) {
  const int64_t row_bytes = d * p.b, kb = p.kd;
  yp_copy_job j = {};
  if (p.split) j.plane = rows_out * kb;
  j.src = (const char*)src; j.dst = dst; j.row_bytes = row_bytes; j.kb = kb; j.rows = rows; j.rows_out = rows_out;
  j.vec = row_bytes % 16 == 0 && ((uintptr_t)src & 15) == 0;
  return j;
}
// the rows' exponents; and back[0], [1], of the features and of the weight, for the backward pass
static hipError_t find_exponents(const yp_class_loss_args& a, const yp_labels& labels, char* ws, const ClassLossPlan& p, bool backward, hipStream_t st) {
  yp_peak_args k;
  k.src[0] = (const float*)a.features; k.src[1] = (const float*)a.weight;
  k.rows[0] = a.n; k.rows[1] = a.v; k.d = a.d;
  k.vec = a.d % 4 == 0 && (((uintptr_t)a.features | (uintptr_t)a.weight) & 15) == 0;
  k.labels = labels; k.bias = (const float*)a.bias; k.grad = backward && a.grad_stride ? a.grad : nullptr; k.part = backward ? (int*)(ws + p.o_peaks) : nullptr;
  k.exponent[0] = (int*)(ws + p.o_eh); k.exponent[1] = (int*)(ws + p.o_ew);
  hipLaunchKernelGGL(yp_peak_kernel, dim3(YP_PEAK_BLOCKS), dim3(YP_CL_THREADS), 0, st, k);
  if (backward) hipLaunchKernelGGL(yp_back_kernel, dim3(1), dim3(128), 0, st, (const int*)k.part, (int*)(ws + p.o_back));
  return hipGetLastError();
}
static hipError_t copy_rows(yp_copy_args a, hipStream_t st) {
  a.chunks0 = a.job[0].rows_out * (a.job[0].kb / 16);
  a.chunks = a.chunks0 + (a.job[1].src ? a.job[1].rows_out * (a.job[1].kb / 16) : 0);
  const dim3 grid(blocks_for(a.chunks, YP_CL_THREADS, 8192));
  if (a.job[0].plane) hipLaunchKernelGGL(yp_copy_rows_kernel<true>, grid, dim3(YP_CL_THREADS), 0, st, a);
  else hipLaunchKernelGGL(yp_copy_rows_kernel<false>, grid, dim3(YP_CL_THREADS), 0, st, a);
  return hipGetLastError();
}

// TYPE: the matrix instructions'; ELEM: the tensors'.  SPLIT: f32 by two f16 planes.
template <int TYPE, int ELEM, bool SPLIT>
static hipError_t forward_t(const yp_class_loss_args& a, hipStream_t st) {
  constexpr int b = yp_type<ELEM>::bytes;
  const int64_t row = (int64_t)a.d * b;
  const bool copy = SPLIT || row % YP_TILE_KB != 0 || (((uintptr_t)a.features | (uintptr_t)a.weight) & 15) != 0;
  const ClassLossPlan p = plan_class_loss(a.n, a.v, a.d, ELEM, a.bias != nullptr, copy);
  char* const ws = (char*)a.workspace;
  const yp_labels labels = {a.labels, a.label_bytes, a.ignore_index, a.v};
  const int *const eh = (const int*)(ws + p.o_eh), *const ew = (const int*)(ws + p.o_ew);     // SPLIT
  if (SPLIT) CL_TRY(find_exponents(a, labels, ws, p, false, st));
  yp_softmax_part* const part = (yp_softmax_part*)(ws + p.o_part);
  int parts = 0;
  for (int s = 0; s < p.fwd_pieces; ++s) {
    const int v0 = s * p.fwd_piece, nv = a.v - v0 < p.fwd_piece ? a.v - v0 : p.fwd_piece;
    yp_gemm g = {};
    g.a = (const char*)a.weight; g.b = (const char*)a.features;
    if (copy) {
      yp_copy_args c = {};
      c.type = ELEM;
      c.job[0] = copy_job(g.a + v0 * row, ws + p.o_w, a.d, p, nv, nv);
      if (s == 0) c.job[1] = copy_job(g.b, ws + p.o_h, a.d, p, a.n, a.n);
      c.labels = labels;
      if (SPLIT) { c.job[0].exponent = ew + v0; c.job[1].exponent = eh; }
      g.aplane = nv * p.kd; g.bplane = a.n * p.kd;
      CL_TRY(copy_rows(c, st));
      g.a = ws + p.o_w; g.b = ws + p.o_h;
    }
    g.lda = g.ldb = p.kd;
    g.I = nv; g.J = a.n; g.steps = (int)(p.kd / YP_TILE_KB);
    yp_tile_plan tp = p.fwd;
    tp.tiles_i = (nv + tp.bi - 1) / tp.bi;
    yp_epi_stats<ELEM, SPLIT> e;
    e.exponents = yp_row_exponents{ew + v0, eh};
    e.bias = a.bias ? (const char*)a.bias + (int64_t)v0 * b : nullptr;
    e.labels = labels; e.first = v0; e.part = part + (int64_t)parts * a.n; e.picked = (float*)(ws + p.o_picked);
    CL_TRY(yp_launch_gemm<TYPE, SPLIT ? 3 : 1>(tp, g, e, st));
    parts += tp.tiles_i * 2;
  }
  yp_join_args j;
  j.part = part; j.parts = parts; j.picked = (const float*)(ws + p.o_picked); j.labels = labels;
  j.N = a.n; j.losses = a.losses; j.lse = a.lse; j.reduced = yp_reduced{a.sum, a.mean, a.counted}; j.block_part = (double*)(ws + p.o_block);
  // few rows of many parts: 128 threads a row, or 32; else 8.  A few rows of few parts are one workgroup's, which sums their losses
  // itself: a launch less.
  int blocks;
  if (a.n <= 1024 && parts > 64) {
    blocks = (a.n + 1) / 2;
    hipLaunchKernelGGL(yp_join_kernel<2>, dim3(blocks), dim3(YP_CL_THREADS), 0, st, j);
  } else if (a.n <= 4096 && parts > 64) {
    blocks = (a.n + 7) / 8;
    hipLaunchKernelGGL(yp_join_kernel<8>, dim3(blocks), dim3(YP_CL_THREADS), 0, st, j);
  } else {
    blocks = a.n <= 256 ? 1 : (a.n + 31) / 32;
    hipLaunchKernelGGL(yp_join_kernel<32>, dim3(blocks), dim3(YP_CL_THREADS), 0, st, j);
  }
  if (j.reduced.wanted() && blocks > 1) hipLaunchKernelGGL(yp_reduce_kernel, dim3(1), dim3(YP_CL_THREADS), 0, st, (const double*)j.block_part, blocks, j.reduced);
  return hipGetLastError();
}

template <int TYPE, int ELEM, bool SPLIT, int PLANES>
static hipError_t backward_t(const yp_class_loss_args& a, hipStream_t st) {
  constexpr int b = yp_type<ELEM>::bytes, tb = yp_type<TYPE>::bytes;
  const int64_t row = (int64_t)a.d * b;
  const ClassLossPlan p = plan_class_loss(a.n, a.v, a.d, ELEM, a.bias != nullptr, false);
  const bool copy_w = SPLIT || a.bias || row % YP_TILE_KB != 0 || ((uintptr_t)a.weight & 15) != 0;
  char* const ws = (char*)a.workspace;
  const yp_labels labels = {a.labels, a.label_bytes, a.ignore_index, a.v};
  const int *const re_h = (const int*)(ws + p.o_eh), *const re_w = (const int*)(ws + p.o_ew);   // SPLIT
  const int* const common = SPLIT ? (const int*)(ws + p.o_back) : nullptr;
  if (SPLIT) CL_TRY(find_exponents(a, labels, ws, p, true, st));
  const int up = TYPE == YP_T_F16 ? 13 : 0;                 // dz is held times 2^up
  yp_relative* relative = nullptr;
  yp_scale back = {a.grad, a.count, -up, nullptr};          // one g for all rows
  if (a.grad_stride) {
    back = yp_scale{nullptr, a.count, SPLIT ? -up : 0, nullptr};
    if (!SPLIT && TYPE != YP_T_F32) {                       // (f32 as it is: dz is not rounded)
      relative = (yp_relative*)(ws + p.o_relative);
      hipLaunchKernelGGL(yp_relative_kernel, dim3(1), dim3(1024), 0, st, a.grad, labels, (int64_t)a.n, up, relative);
      CL_TRY(hipGetLastError());
      back.a = &relative->back;
      back.more = &relative->e;
    }
  }
  float* const dhpart = (float*)(ws + p.o_dhpart);
  float* const biaspart = a.grad_bias && p.dzp.tiles_j > 1 ? (float*)(ws + p.o_bp) : nullptr;
  yp_scale back_w = back, back_h = back;                    // of grad_weight, which has the features' exponent, and the other way round
  if (SPLIT) { back_w.more = common; back_h.more = common + 1; }
  yp_sum_args sums = {};
  sums.out_type = ELEM;
  for (int s = 0; s < p.pieces; ++s) {
    const int v0 = s * p.piece, nv = a.v - v0 < p.piece ? a.v - v0 : p.piece;
    const char* const bias = a.bias ? (const char*)a.bias + (int64_t)v0 * b : nullptr;
    const char* w = (const char*)a.weight + v0 * row;
    if (s == 0 || copy_w) {
      yp_copy_args c = {};
      c.type = ELEM;
      c.labels = labels;
      int n = 0;
      if (s == 0) {
        yp_copy_job& j = c.job[n++];
        j = copy_job(a.features, ws + p.o_hc, a.d, p, a.n, p.kn);
        j.by_label = 1;
        if (SPLIT) { j.exponent = re_h; j.common = ws + p.o_hs; j.back = common; j.grad = a.grad_stride ? a.grad : nullptr; }
      }
      if (copy_w) {
        yp_copy_job& j = c.job[n++];
        j = copy_job(w, ws + p.o_wc, a.d, p, nv, nv);
        j.bias = bias;
        if (SPLIT) { j.exponent = re_w + v0; j.common = ws + p.o_ws; j.back = common + 1; }
        w = ws + p.o_wc;
      }
      CL_TRY(copy_rows(c, st));
    }
    const int kv = (int)(yp_pad_k(nv, tb) / tb);
    const int64_t hplane = p.kn * p.kd, wplane = nv * p.kd, dzplane = p.kn * kv * tb;
    // dz of the piece
    yp_gemm g = {};
    g.a = w; g.b = ws + p.o_hc; g.lda = g.ldb = p.kd;
    g.aplane = wplane; g.bplane = hplane;
    g.I = nv; g.J = a.n; g.steps = (int)(p.kd / YP_TILE_KB);
    yp_epi_dz<ELEM, SPLIT, PLANES> e;
    e.plane = dzplane;
    e.exponents = yp_row_exponents{re_w + v0, re_h};
    e.bias = bias; e.lse = a.lse; e.labels = labels; e.grad = a.grad_stride ? a.grad : nullptr; e.relative = relative; e.up = ldexpf(1.0f, up); e.scale = back;
    e.first = v0; e.dz = ws + p.o_dz; e.kv = kv; e.kn = (int)p.kn;
    e.bias_out = a.grad_bias ? (char*)a.grad_bias + (int64_t)v0 * b : nullptr;
    e.bias_part = biaspart;
    yp_tile_plan tp = p.dzp;
    tp.tiles_i = (nv + tp.bi - 1) / tp.bi;
    CL_TRY(yp_launch_gemm<TYPE, SPLIT ? 3 : 1>(tp, g, e, st));
    // dw[v][d] = sum_n dz[n][v] h[n][d]
    yp_gemm gw = {};
    gw.a = ws + (SPLIT ? p.o_hs : p.o_hc); gw.lda = p.kd; gw.I = a.d; gw.aplane = hplane; gw.bplane = dzplane;
    gw.b = ws + p.o_dz; gw.ldb = (int64_t)kv * tb; gw.J = nv;
    gw.K = (int)p.kn; gw.steps = (int)(p.kn * tb / YP_TILE_KB);
    char* const gwo = a.grad_weight ? (char*)a.grad_weight + v0 * row : nullptr;
    yp_epi_store<ELEM> ew = {};
    ew.out = gwo; ew.ld = a.d; ew.scale = back_w;
    ew.vec = row % 16 == 0 && ((uintptr_t)a.grad_weight & 15) == 0;
    ew.part_vec = a.d % 4 == 0;
    ew.part = gwo && p.dwp.splits > 1 ? (float*)(ws + p.o_dwpart) : nullptr;
    yp_tile_plan twp = p.dwp;
    twp.tiles_j = (nv + twp.bj - 1) / twp.bj;
    // dh[n][d] (+)= sum_v dz[n][v] w[v][d]
    yp_gemm gh = {};
    gh.a = SPLIT ? ws + p.o_ws : w; gh.lda = copy_w ? p.kd : row; gh.I = a.d; gh.aplane = wplane; gh.bplane = dzplane;
    gh.b = ws + p.o_dz; gh.ldb = (int64_t)kv * tb; gh.J = a.n;
    gh.K = nv; gh.steps = (int)((int64_t)kv * tb / YP_TILE_KB);
    yp_epi_store<ELEM> eh = {};
    eh.out = a.grad_features; eh.ld = a.d; eh.scale = back_h; eh.row = SPLIT && a.grad_stride ? a.grad : nullptr;
    eh.vec = row % 16 == 0 && ((uintptr_t)a.grad_features & 15) == 0;
    eh.part_vec = a.d % 4 == 0;
    // (over pieces dh adds up in f32; for 16-bit types without a split the last one adds what lies there and rounds,
    // 700 us for 200 x 128000 x 1024, joined by a kernel after it 722)
    const bool dh_last = p.dhp.splits == 1 && (p.pieces == 1 || (s == p.pieces - 1 && ELEM != YP_F32));
    eh.part = dh_last ? nullptr : dhpart;
    eh.before = dh_last && s > 0 ? dhpart : nullptr;
    eh.add = s > 0;
    yp_bias_sum bs = {};
    bs.part = biaspart; bs.parts = p.dzp.tiles_j; bs.total = nv; bs.type = ELEM; bs.scale = back; bs.out = e.bias_out;
    CL_TRY(yp_launch_two<TYPE, SPLIT ? 3 : PLANES>(twp, gw, ew, p.dhp, gh, eh, bs, biaspart ? (nv + yp_bias_sum::CLASSES - 1) / yp_bias_sum::CLASSES : 0, st));
    if (ew.part) add_sum(sums, ew.part, p.dwp.splits, (int64_t)nv * a.d, gwo, back_w, nullptr, a.d);
    if (s == p.pieces - 1 && eh.part && a.grad_features) add_sum(sums, dhpart, p.dhp.splits, (int64_t)a.n * a.d, a.grad_features, back_h, eh.row, a.d);
    CL_TRY(sum_parts(sums, st));
    sums.jobs = 0;
  }
  return hipSuccess;
}

hipError_t yp_launch_class_loss(const yp_class_loss_args& a, hipStream_t st) {
  if (a.n == 0) {
    for (float* one : {a.sum, a.mean, a.counted}) if (one) CL_TRY(zero(one, 1, YP_F32, st));
    return hipSuccess;
  }
  const bool split = plan_class_loss(a.n, a.v, a.d, a.type, false, false).split;
  return a.type == YP_BF16 ? forward_t<YP_T_BF16, YP_T_BF16, false>(a, st) : a.type == YP_F16 ? forward_t<YP_T_F16, YP_T_F16, false>(a, st)
       : split ? forward_t<YP_T_F16, YP_T_F32, true>(a, st) : forward_t<YP_T_F32, YP_T_F32, false>(a, st);
}
hipError_t yp_launch_class_loss_backward(const yp_class_loss_args& a, hipStream_t st) {
  if (a.n == 0) {
    if (a.grad_weight) CL_TRY(zero(a.grad_weight, (int64_t)a.v * a.d, a.type, st));
    return a.grad_bias ? zero(a.grad_bias, a.v, a.type, st) : hipSuccess;
  }
  const ClassLossPlan p = plan_class_loss(a.n, a.v, a.d, a.type, false, false);
  if (a.type == YP_F32) return p.split ? backward_t<YP_T_F16, YP_T_F32, true, 2>(a, st) : backward_t<YP_T_F32, YP_T_F32, false, 1>(a, st);
  if (a.type == YP_BF16) return p.dzplanes == 2 ? backward_t<YP_T_BF16, YP_T_BF16, false, 2>(a, st) : backward_t<YP_T_BF16, YP_T_BF16, false, 1>(a, st);
  return p.dzplanes == 2 ? backward_t<YP_T_F16, YP_T_F16, false, 2>(a, st) : backward_t<YP_T_F16, YP_T_F16, false, 1>(a, st);
}
