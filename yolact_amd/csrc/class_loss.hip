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
// row; a second kernel joins the parts.  2 N V D operations, h and w are read, 8 bytes per row and 128 classes written.
// Backward, per piece of the vocabulary (so that a piece of dz stays near the Infinity Cache): the product again, with
// an epilogue that turns z into dz, written in both orders ([row][class] and [class][row]) so that the two gradient
// products find k contiguous in both operands; dw's piece is complete then, dh adds up over the pieces in f32.
// dz is rounded to the features' type - the matrix instruction takes nothing wider beside h and w; each dz is off by
// half a step of that type, like the gradients themselves - f16 with a power-of-two factor that brings the largest
// |g| to [2^13, 2^14), so that probabilities down to 2^-38 of it are kept, taken out again in f32 at the end.
// All sums are f32 in a fixed order: no float atomics, the same call gives the same bits.
#include "gemm_launch.hpp"

#define YP_CL_THREADS 256
#define YP_CL_PIECE_MAX (1 << 17)
#define YP_CL_PIECE_BYTES (128ll << 20)   // dz in one order: with the other order it fills the 256 MB Infinity Cache

__device__ __forceinline__ int64_t yp_label_at(const void* labels, int64_t n, int bytes) {
  return bytes == 8 ? reinterpret_cast<const int64_t*>(labels)[n] : (int64_t)reinterpret_cast<const int32_t*>(labels)[n];
}

__device__ __forceinline__ float yp_exp_hw(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

struct yp_softmax_part { float m, s; };
__device__ __forceinline__ void yp_join(float& m, float& s, float m2, float s2) {
  const float t = fmaxf(m, m2);
  const float ref = t == -INFINITY ? 0.0f : t;
  s = s * yp_exp_hw(m - ref) + s2 * yp_exp_hw(m2 - ref);
  m = t;
}

// ---- epilogue of the forward product: i = class, j = row ----------------------------------------------------------
struct yp_epi_stats {
  const void* bias;            // elements of the features' type, may be null
  const void* labels;
  int label_bytes;
  int V;
  yp_softmax_part* part;       // [tiles_i * WI][N]
  float* picked;               // [N] z of the label
  template <int TYPE, int BM, int BN, int WI, int WJ, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], int ti, int tj, int, int wi, int wj, int lane) const {
    const int ib = ti * BM + wi * (BM / 2 / WI) + (lane >> 4) * 4, jb = tj * BN + wj * (BN / 2 / WJ) + (lane & 15);
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = ib + yp_frag_at<BM, MI>(m) + r;
        const float b = i >= V ? -INFINITY : (bias ? yp_load_as_float(bias, i, TYPE) : 0.0f);
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n][r] = b == -INFINITY ? -INFINITY : acc[m][n][r] + b;
      }
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int j = jb + yp_frag_at<BN, NJ>(n);
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[m][n][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += yp_exp_hw(acc[m][n][r] - ref);
      if (j < g.J) {
        const int64_t at = yp_label_at(labels, j, label_bytes) - ib;
        if (at >= 0 && at < BM) {
#pragma unroll
          for (int m = 0; m < MI; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) if (at == yp_frag_at<BM, MI>(m) + r) picked[j] = acc[m][n][r];
        }
      }
#pragma unroll
      for (int x = 16; x < 64; x <<= 1) yp_join(top, sum, __shfl_xor(top, x), __shfl_xor(sum, x));
      if (j < g.J && lane < 16) part[(int64_t)(ti * WI + wi) * g.J + j] = yp_softmax_part{top, sum};
    }
  }
};

// ---- epilogue of the backward product -----------------------------------------------------------------------------
struct yp_epi_dz {
  const void* bias;            // of the piece
  const float* lse;
  const float* row_grad;       // [N] g, already times the f16 factor
  const int32_t* row_label;    // [N] label relative to class 0, -1 = the row takes no part
  int first;                   // first class of the piece
  int V;                       // classes in the piece
  char* dz;                    // [N][kv]
  char* dzt;                   // [V][kn]
  int kv, kn;                  // elements, padded: dz is zero in [V, kv), dzt in [N, kn)
  float* bias_part;            // [tiles_j * WJ][V], null without bias
  template <int TYPE, int BM, int BN, int WI, int WJ, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], int ti, int tj, int, int wi, int wj, int lane) const {
    typedef typename yp_type<TYPE>::elem elem;
    typedef elem e4 __attribute__((ext_vector_type(4)));
    const int ib = ti * BM + wi * (BM / 2 / WI) + (lane >> 4) * 4, jb = tj * BN + wj * (BN / 2 / WJ) + (lane & 15);
    elem* const z0 = reinterpret_cast<elem*>(dz);
    elem* const zt = reinterpret_cast<elem*>(dzt);
    float l[NJ], gr[NJ];
    int lab[NJ];
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int j = jb + yp_frag_at<BN, NJ>(n);
      const bool in = j < g.J;
      l[n] = in ? lse[j] : 0.0f;
      gr[n] = in ? row_grad[j] : 0.0f;
      const int t = in ? row_label[j] : -1;
      lab[n] = t < 0 ? -1 : (t >= first && t - first < V ? t - first : 0x7fffffff);   // 0x7fffffff: counted, label elsewhere
    }
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      const int i = ib + yp_frag_at<BM, MI>(m);
      float col[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      float b[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) b[r] = i + r >= V ? -INFINITY : (bias ? yp_load_as_float(bias, i + r, TYPE) : 0.0f);
#pragma unroll
      for (int n = 0; n < NJ; ++n) {
        const int j = jb + yp_frag_at<BN, NJ>(n);
        e4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float z = acc[m][n][r] + b[r];
          float p = l[n] == -INFINITY ? 0.0f : yp_exp_hw(z - l[n]);
          if (lab[n] == i + r) p -= 1.0f;
          const float d = lab[n] < 0 || b[r] == -INFINITY ? 0.0f : p * gr[n];
          col[r] += d;
          o[r] = (elem)d;
        }
        if (j < g.J && i < kv) *reinterpret_cast<e4*>(z0 + (int64_t)j * kv + i) = o;
        if (j < kn) {
#pragma unroll
          for (int r = 0; r < 4; ++r) if (i + r < V) zt[(int64_t)(i + r) * kn + j] = o[r];
        }
      }
      if (bias_part) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int x = 1; x < 16; x <<= 1) col[r] += __shfl_xor(col[r], x);
          if ((lane & 15) == 0 && i + r < V) bias_part[(int64_t)(tj * WJ + wj) * V + i + r] = col[r];
        }
      }
    }
  }
};

// ---- the small kernels around the products ------------------------------------------------------------------------
// rows of `cols` elements copied to rows of `kb` bytes, the tail zero
__global__ __launch_bounds__(YP_CL_THREADS) void yp_pack_rows_kernel(const char* src, char* dst, int64_t rows, int64_t row_bytes, int64_t kb, int elem) {
  const int64_t per = kb / elem, total = rows * per;
  for (int64_t e = (int64_t)blockIdx.x * YP_CL_THREADS + threadIdx.x; e < total; e += (int64_t)gridDim.x * YP_CL_THREADS) {
    const int64_t r = e / per, c = (e - r * per) * elem;
    if (elem == 4) *reinterpret_cast<uint32_t*>(dst + r * kb + c) = c < row_bytes ? *reinterpret_cast<const uint32_t*>(src + r * row_bytes + c) : 0u;
    else *reinterpret_cast<uint16_t*>(dst + r * kb + c) = c < row_bytes ? *reinterpret_cast<const uint16_t*>(src + r * row_bytes + c) : (uint16_t)0;
  }
}

// src [R][C] -> dst [C][kr], kr >= R elements, the tail zero.  A row of src that takes no part - its label is < 0 or
// its bias -inf - is written as zeros: whatever it holds, it meets only zeros in the product.
template <class E>
__global__ __launch_bounds__(YP_CL_THREADS) void yp_transpose_kernel(const E* src, E* dst, int R, int C, int kr, const int32_t* row_label,
                                                                     const void* row_bias, int bias_type) {
  __shared__ E t[64][65];
  const int r0 = (int)blockIdx.x * 64, c0 = (int)blockIdx.y * 64;
  const int x = (int)threadIdx.x & 63, y = (int)threadIdx.x >> 6;
  for (int u = y; u < 64; u += YP_CL_THREADS / 64) {
    const int r = r0 + u;
    bool in = r < R && c0 + x < C;
    if (in && row_label && row_label[r] < 0) in = false;
    if (in && row_bias && yp_load_as_float(row_bias, r, bias_type) == -INFINITY) in = false;
    t[u][x] = in ? src[(int64_t)r * C + c0 + x] : (E)0;
  }
  __syncthreads();
  for (int u = y; u < 64; u += YP_CL_THREADS / 64)
    if (c0 + u < C && r0 + x < kr) dst[(int64_t)(c0 + u) * kr + r0 + x] = t[x][u];
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

__device__ __forceinline__ void yp_write_reduced(float* reduced, double sum, double count) {
  reduced[0] = (float)sum;
  reduced[1] = count > 0.0 ? (float)(sum / count) : 0.0f;
  reduced[2] = (float)count;
}

// Joins the parts of 32 rows per workgroup (8 threads a row), and the rows' losses if they are asked for.
struct yp_join_args {
  const yp_softmax_part* part;
  int parts;
  const float* picked;
  const void* labels;
  int label_bytes;
  int64_t ignore_index;
  int N, V;
  float *losses, *lse;
  float* reduced;           // [3], may be null
  double* block_part;       // [blocks][2]
};
__global__ __launch_bounds__(YP_CL_THREADS) void yp_join_kernel(const yp_join_args a) {
  __shared__ float lm[8][32], ls[8][32];
  __shared__ double red[YP_CL_THREADS / 64];
  const int x = (int)threadIdx.x & 31, y = (int)threadIdx.x >> 5;
  const int n = (int)blockIdx.x * 32 + x;
  float m = -INFINITY, s = 0.0f;
  if (n < a.N)
    for (int p = y; p < a.parts; p += 8) {
      const yp_softmax_part v = a.part[(int64_t)p * a.N + n];
      yp_join(m, s, v.m, v.s);
    }
  lm[y][x] = m; ls[y][x] = s;
  __syncthreads();
  double loss = 0.0, count = 0.0;
  if (y == 0 && n < a.N) {
    for (int u = 1; u < 8; ++u) yp_join(m, s, lm[u][x], ls[u][x]);
    const float l = m + logf(s);
    const int64_t lab = yp_label_at(a.labels, n, a.label_bytes);
    float v;
    if (lab == a.ignore_index) v = 0.0f;
    else if (lab < 0 || lab >= a.V) { v = NAN; count = 1.0; }
    else {
      const float p = a.picked[n];
      v = p == -INFINITY ? INFINITY : l - p;
      count = 1.0;
    }
    a.lse[n] = l;
    a.losses[n] = v;
    loss = v;
  }
  if (!a.reduced) return;
  const double ts = yp_block_sum(loss, red), tc = yp_block_sum(count, red);
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) yp_write_reduced(a.reduced, ts, tc);
    else { a.block_part[2 * blockIdx.x] = ts; a.block_part[2 * blockIdx.x + 1] = tc; }
  }
}
__global__ __launch_bounds__(YP_CL_THREADS) void yp_reduce_kernel(const double* block_part, int blocks, float* reduced) {
  __shared__ double red[YP_CL_THREADS / 64];
  double s = 0.0, c = 0.0;
  for (int i = (int)threadIdx.x; i < blocks; i += YP_CL_THREADS) { s += block_part[2 * i]; c += block_part[2 * i + 1]; }
  const double ts = yp_block_sum(s, red), tc = yp_block_sum(c, red);
  if (threadIdx.x == 0) yp_write_reduced(reduced, ts, tc);
}

// g and label of every row as the backward product wants them, and the f16 factor.
struct yp_rows_args {
  const void* labels;
  int label_bytes;
  int64_t ignore_index;
  int N, V;
  const float* grad;
  int grad_stride;
  const float* count;      // null: grads are the rows' own; else divided by max(count, 1)
  float* row_grad;
  int32_t* row_label;
  const float* factor;     // [2] {2^e, 2^-e} or null
};
__device__ __forceinline__ float yp_row_grad(const yp_rows_args& a, int64_t n) {
  const float g = a.grad[n * a.grad_stride];
  return a.count ? g / fmaxf(*a.count, 1.0f) : g;
}
__global__ __launch_bounds__(YP_CL_THREADS) void yp_rows_kernel(const yp_rows_args a) {
  const int n = (int)blockIdx.x * YP_CL_THREADS + (int)threadIdx.x;
  if (n >= a.N) return;
  const int64_t lab = yp_label_at(a.labels, n, a.label_bytes);
  const bool counted = lab != a.ignore_index && lab >= 0 && lab < a.V;
  a.row_label[n] = counted ? (int32_t)lab : -1;
  a.row_grad[n] = counted ? yp_row_grad(a, n) * (a.factor ? a.factor[0] : 1.0f) : 0.0f;
}
__global__ __launch_bounds__(1024) void yp_factor_kernel(const yp_rows_args a, float* factor) {
  __shared__ float red[16];
  float top = 0.0f;
  const int64_t n1 = a.grad_stride ? a.N : (a.N > 0 ? 1 : 0);
  for (int64_t n = threadIdx.x; n < n1; n += 1024) top = fmaxf(top, fabsf(yp_row_grad(a, n)));
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) top = fmaxf(top, red[w]);
    int e = 0;
    if (top > 0.0f && top < INFINITY) e = 13 - ilogbf(top);
    e = min(max(e, -100), 100);
    factor[0] = ldexpf(1.0f, e);
    factor[1] = ldexpf(1.0f, -e);
  }
}

// out[e] = scale * sum over the parts, in the order of the parts
__global__ __launch_bounds__(YP_CL_THREADS) void yp_sum_parts_kernel(const float* part, int parts, int64_t stride, int64_t total, void* out,
                                                                     int out_type, const float* scale) {
  const float sc = scale ? *scale : 1.0f;
  for (int64_t e = (int64_t)blockIdx.x * YP_CL_THREADS + threadIdx.x; e < total; e += (int64_t)gridDim.x * YP_CL_THREADS) {
    float s = 0.0f;
    for (int p = 0; p < parts; ++p) s += part[(int64_t)p * stride + e];
    if (out_type == YP_F32) reinterpret_cast<float*>(out)[e] = s * sc;
    else if (out_type == YP_BF16) reinterpret_cast<__bf16*>(out)[e] = (__bf16)(s * sc);
    else reinterpret_cast<_Float16*>(out)[e] = (_Float16)(s * sc);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------
static inline int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
static inline int type_bytes(int t) { return t == YP_F32 ? 4 : 2; }
static inline unsigned blocks_for(int64_t n, int per, int64_t most) { const int64_t b = (n + per - 1) / per; return (unsigned)(b < 1 ? 1 : b > most ? most : b); }

struct ClassLossPlan {
  int64_t kd;                  // bytes of a padded feature row
  bool pack_h, pack_w;         // copied to padded rows first
  yp_tile_plan fwd;
  int parts;
  int pieces, piece;           // backward: vocabulary pieces and their width (a multiple of 256 unless there is one)
  int64_t kn, kv;              // bytes of a padded row of [.][N] and [.][piece]
  yp_tile_plan dzp, dwp, dhp;
  int bias_parts;
  // workspace offsets
  int64_t o_h, o_w, o_part, o_picked, o_block, fwd_total;
  int64_t o_rg, o_rl, o_factor, o_dz, o_dzt, o_ht, o_wt, o_bp, o_dwpart, o_dhpart, bwd_total;
};

// `aligned`: both matrices start on 16 bytes
static ClassLossPlan plan_class_loss(int64_t N, int64_t V, int64_t D, int type, bool has_bias, bool aligned) {
  ClassLossPlan p;
  const int b = type_bytes(type);
  p.kd = yp_pad_k(D, b);
  p.pack_h = p.pack_w = p.kd != D * b || !aligned;
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = up256(off + bytes); return o; };
  p.o_h = take(p.pack_h ? N * p.kd : 0);
  p.o_w = take(p.pack_w ? V * p.kd : 0);
  const int64_t common = off;
  p.fwd = yp_plan_tiles(V, N, p.kd / YP_TILE_KB, false);
  p.parts = p.fwd.tiles_i * (p.fwd.shape == YP_TILE_S ? 4 : 2);
  p.o_part = take((int64_t)p.parts * N * sizeof(yp_softmax_part));
  p.o_picked = take(N * 4);
  p.o_block = take((N + 31) / 32 * 16);
  p.fwd_total = off;

  off = common;
  p.kn = yp_pad_k(N, b);
  int64_t piece = YP_CL_PIECE_BYTES / ((N > D ? N : D) * b) / 256 * 256;   // (the piece of w is transposed into [D][piece])
  if (piece < 256) piece = 256;
  if (piece > YP_CL_PIECE_MAX) piece = YP_CL_PIECE_MAX;
  p.pieces = (int)((V + piece - 1) / piece);
  if (p.pieces == 1) piece = V;
  else {   // equal pieces
    piece = ((V + p.pieces - 1) / p.pieces + 255) / 256 * 256;
    p.pieces = (int)((V + piece - 1) / piece);
  }
  p.piece = (int)piece;
  p.kv = yp_pad_k(piece, b);
  p.dzp = yp_plan_tiles(piece, p.kn / b, p.kd / YP_TILE_KB, false);   // (the padded rows too: their columns of dzt are zeros)
  p.dwp = yp_plan_tiles(D, piece, p.kn / YP_TILE_KB, true);
  p.dhp = yp_plan_tiles(D, N, p.kv / YP_TILE_KB, true);
  p.bias_parts = p.dzp.tiles_j * (p.dzp.shape == YP_TILE_S ? 1 : 2);
  p.o_rg = take(N * 4);
  p.o_rl = take(N * 4);
  p.o_factor = take(8);
  p.o_dz = take(N * p.kv);
  p.o_dzt = take(piece * p.kn);
  p.o_ht = take(D * p.kn);
  p.o_wt = take(D * p.kv);
  p.o_bp = take(has_bias ? (int64_t)p.bias_parts * piece * 4 : 0);
  p.o_dwpart = take(p.dwp.splits > 1 ? (int64_t)p.dwp.splits * piece * D * 4 : 0);
  p.o_dhpart = take(p.dhp.splits > 1 || p.pieces > 1 ? (int64_t)p.dhp.splits * N * D * 4 : 0);
  p.bwd_total = off;
  return p;
}

int64_t yp_class_loss_bytes(int64_t n, int64_t v, int64_t d, int type, int has_bias, int backward) {
  // (alignment is not known here: room for the packed copies either way)
  const ClassLossPlan a = plan_class_loss(n, v, d, type, has_bias != 0, false);
  return backward ? a.bwd_total : a.fwd_total;
}

#define CL_TRY(call) do { const hipError_t e_ = (call); if (e_ != hipSuccess) return e_; } while (0)

static hipError_t zero(void* out, int64_t n, int type, hipStream_t st) {   // (a kernel, not a memset: the call may be captured)
  hipLaunchKernelGGL(yp_sum_parts_kernel, dim3(blocks_for(n, YP_CL_THREADS, 8192)), dim3(YP_CL_THREADS), 0, st, (const float*)nullptr, 0, (int64_t)0, n, out, type,
                     (const float*)nullptr);
  return hipGetLastError();
}

static hipError_t pack(const ClassLossPlan& p, const yp_class_loss_args& a, char* ws, const char** h, const char** w, hipStream_t st) {
  const int b = type_bytes(a.type);
  *h = (const char*)a.features;
  *w = (const char*)a.weight;
  if (!p.pack_h) return hipSuccess;
  hipLaunchKernelGGL(yp_pack_rows_kernel, dim3(blocks_for(a.n * p.kd / b, 4 * YP_CL_THREADS, 4096)), dim3(YP_CL_THREADS), 0, st, *h, ws + p.o_h,
                     (int64_t)a.n, (int64_t)a.d * b, p.kd, b);
  hipLaunchKernelGGL(yp_pack_rows_kernel, dim3(blocks_for(a.v * p.kd / b, 4 * YP_CL_THREADS, 4096)), dim3(YP_CL_THREADS), 0, st, *w, ws + p.o_w,
                     (int64_t)a.v, (int64_t)a.d * b, p.kd, b);
  *h = ws + p.o_h;
  *w = ws + p.o_w;
  return hipGetLastError();
}

template <int TYPE>
static hipError_t forward_t(const yp_class_loss_args& a, hipStream_t st) {
  const bool aligned = (((uintptr_t)a.features | (uintptr_t)a.weight) & 15) == 0;
  const ClassLossPlan p = plan_class_loss(a.n, a.v, a.d, TYPE, a.bias != nullptr, aligned);
  char* const ws = (char*)a.workspace;
  yp_gemm g = {};
  CL_TRY(pack(p, a, ws, &g.b, &g.a, st));
  g.lda = g.ldb = p.kd;
  g.I = a.v; g.J = a.n; g.steps = (int)(p.kd / YP_TILE_KB);
  yp_epi_stats e;
  e.bias = a.bias; e.labels = a.labels; e.label_bytes = a.label_bytes; e.V = a.v;
  e.part = (yp_softmax_part*)(ws + p.o_part); e.picked = (float*)(ws + p.o_picked);
  CL_TRY(yp_launch_gemm<TYPE>(p.fwd, g, e, st));
  yp_join_args j;
  j.part = e.part; j.parts = p.parts; j.picked = e.picked; j.labels = a.labels; j.label_bytes = a.label_bytes;
  j.ignore_index = a.ignore_index; j.N = a.n; j.V = a.v; j.losses = a.losses; j.lse = a.lse; j.reduced = a.reduced;
  j.block_part = (double*)(ws + p.o_block);
  const int blocks = (a.n + 31) / 32;
  hipLaunchKernelGGL(yp_join_kernel, dim3(blocks), dim3(YP_CL_THREADS), 0, st, j);
  if (a.reduced && blocks > 1) hipLaunchKernelGGL(yp_reduce_kernel, dim3(1), dim3(YP_CL_THREADS), 0, st, (const double*)j.block_part, blocks, a.reduced);
  return hipGetLastError();
}

template <int TYPE>
static hipError_t transpose(const void* src, char* dst, int R, int C, int64_t kr_bytes, const int32_t* row_label, const void* row_bias, hipStream_t st) {
  typedef typename yp_type<TYPE>::elem elem;
  const int kr = (int)(kr_bytes / (int)sizeof(elem));
  hipLaunchKernelGGL(yp_transpose_kernel<elem>, dim3((kr + 63) / 64, (C + 63) / 64), dim3(YP_CL_THREADS), 0, st, (const elem*)src, (elem*)dst, R, C, kr,
                     row_label, row_bias, TYPE);
  return hipGetLastError();
}

template <int TYPE>
static hipError_t backward_t(const yp_class_loss_args& a, hipStream_t st) {
  constexpr int b = yp_type<TYPE>::bytes;
  const bool aligned = (((uintptr_t)a.features | (uintptr_t)a.weight) & 15) == 0;
  const ClassLossPlan p = plan_class_loss(a.n, a.v, a.d, TYPE, a.bias != nullptr, aligned);
  char* const ws = (char*)a.workspace;
  const char *h, *w;
  CL_TRY(pack(p, a, ws, &h, &w, st));
  yp_rows_args r;
  r.labels = a.labels; r.label_bytes = a.label_bytes; r.ignore_index = a.ignore_index; r.N = a.n; r.V = a.v;
  r.grad = a.grad; r.grad_stride = a.grad_stride; r.count = a.count;
  r.row_grad = (float*)(ws + p.o_rg); r.row_label = (int32_t*)(ws + p.o_rl);
  float* const factor = TYPE == YP_T_F16 ? (float*)(ws + p.o_factor) : nullptr;
  r.factor = factor;
  if (factor) hipLaunchKernelGGL(yp_factor_kernel, dim3(1), dim3(1024), 0, st, r, factor);
  hipLaunchKernelGGL(yp_rows_kernel, dim3((a.n + YP_CL_THREADS - 1) / YP_CL_THREADS), dim3(YP_CL_THREADS), 0, st, r);
  CL_TRY(hipGetLastError());
  const float* const back = factor ? factor + 1 : nullptr;
  CL_TRY(transpose<TYPE>(a.features, ws + p.o_ht, a.n, a.d, p.kn, r.row_label, nullptr, st));

  float* const dhpart = (float*)(ws + p.o_dhpart);
  const bool dh_joined = p.dhp.splits > 1 || p.pieces > 1;
  for (int s = 0; s < p.pieces; ++s) {
    const int v0 = s * p.piece, nv = a.v - v0 < p.piece ? a.v - v0 : p.piece;
    const char* const bias = a.bias ? (const char*)a.bias + (int64_t)v0 * b : nullptr;
    // dz of the piece, both orders
    yp_gemm g = {};
    g.a = w + (int64_t)v0 * p.kd; g.b = h; g.lda = g.ldb = p.kd;
    g.I = nv; g.J = a.n; g.steps = (int)(p.kd / YP_TILE_KB);
    yp_epi_dz e;
    e.bias = bias; e.lse = a.lse; e.row_grad = r.row_grad; e.row_label = r.row_label; e.first = v0; e.V = nv;
    e.dz = ws + p.o_dz; e.dzt = ws + p.o_dzt; e.kv = (int)(yp_pad_k(nv, b) / b); e.kn = (int)(p.kn / b);
    e.bias_part = a.bias ? (float*)(ws + p.o_bp) : nullptr;
    yp_tile_plan tp = p.dzp;
    tp.tiles_i = (nv + tp.bi - 1) / tp.bi;
    CL_TRY(yp_launch_gemm<TYPE>(tp, g, e, st));
    if (a.bias) {
      hipLaunchKernelGGL(yp_sum_parts_kernel, dim3(blocks_for(nv, YP_CL_THREADS, 4096)), dim3(YP_CL_THREADS), 0, st, (const float*)e.bias_part, p.bias_parts,
                         (int64_t)nv, (int64_t)nv, (void*)((char*)a.grad_bias + (int64_t)v0 * b), TYPE, back);
      CL_TRY(hipGetLastError());
    }
    CL_TRY(transpose<TYPE>((const char*)a.weight + (int64_t)v0 * a.d * b, ws + p.o_wt, nv, a.d, (int64_t)e.kv * b, nullptr, bias, st));
    // dw[v][d] = sum_n dz[n][v] h[n][d]
    yp_gemm gw = {};
    gw.a = ws + p.o_ht; gw.lda = p.kn; gw.I = a.d;
    gw.b = ws + p.o_dzt; gw.ldb = p.kn; gw.J = nv;
    gw.steps = (int)(p.kn / YP_TILE_KB);
    char* const gwo = (char*)a.grad_weight + (int64_t)v0 * a.d * b;
    yp_epi_store ew = {};
    ew.out = gwo; ew.ld = a.d; ew.scale = back;
    ew.vec = a.d % 4 == 0 && ((uintptr_t)a.grad_weight & 15) == 0;
    ew.part = p.dwp.splits > 1 ? (float*)(ws + p.o_dwpart) : nullptr;
    yp_tile_plan twp = p.dwp;
    twp.tiles_j = (nv + twp.bj - 1) / twp.bj;
    CL_TRY(yp_launch_gemm<TYPE>(twp, gw, ew, st));
    if (ew.part) {
      hipLaunchKernelGGL(yp_sum_parts_kernel, dim3(blocks_for((int64_t)nv * a.d, YP_CL_THREADS, 8192)), dim3(YP_CL_THREADS), 0, st, (const float*)ew.part, p.dwp.splits,
                         (int64_t)nv * a.d, (int64_t)nv * a.d, (void*)gwo, TYPE, back);
      CL_TRY(hipGetLastError());
    }
    // dh[n][d] (+)= sum_v dz[n][v] w[v][d]
    yp_gemm gh = {};
    gh.a = ws + p.o_wt; gh.lda = (int64_t)e.kv * b; gh.I = a.d;
    gh.b = ws + p.o_dz; gh.ldb = (int64_t)e.kv * b; gh.J = a.n;
    gh.steps = (int)((int64_t)e.kv * b / YP_TILE_KB);
    yp_epi_store eh = {};
    eh.out = a.grad_features; eh.ld = a.d; eh.scale = back;
    eh.vec = a.d % 4 == 0 && ((uintptr_t)a.grad_features & 15) == 0;
    eh.part = dh_joined ? dhpart : nullptr;
    eh.add = s > 0;
    CL_TRY(yp_launch_gemm<TYPE>(p.dhp, gh, eh, st));
  }
  if (dh_joined) {
    hipLaunchKernelGGL(yp_sum_parts_kernel, dim3(blocks_for((int64_t)a.n * a.d, YP_CL_THREADS, 8192)), dim3(YP_CL_THREADS), 0, st, (const float*)dhpart, p.dhp.splits,
                       (int64_t)a.n * a.d, (int64_t)a.n * a.d, a.grad_features, TYPE, back);
  }
  return hipGetLastError();
}

hipError_t yp_launch_class_loss(const yp_class_loss_args& a, hipStream_t st) {
  if (a.n == 0) return a.reduced ? zero(a.reduced, 3, YP_F32, st) : hipSuccess;
  return a.type == YP_F32 ? forward_t<YP_T_F32>(a, st) : a.type == YP_BF16 ? forward_t<YP_T_BF16>(a, st) : forward_t<YP_T_F16>(a, st);
}
hipError_t yp_launch_class_loss_backward(const yp_class_loss_args& a, hipStream_t st) {
  if (a.n == 0) {
    CL_TRY(zero(a.grad_weight, (int64_t)a.v * a.d, a.type, st));
    return a.bias ? zero(a.grad_bias, a.v, a.type, st) : hipSuccess;
  }
  return a.type == YP_F32 ? backward_t<YP_T_F32>(a, st) : a.type == YP_BF16 ? backward_t<YP_T_BF16>(a, st) : backward_t<YP_T_F16>(a, st);
}
