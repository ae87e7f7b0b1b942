// Quantized linear: out = (xq wq^T) x_scale w_scale + bias with 8-bit integers and one scale per row of either operand.
//
//   scale = max|x| / 127 (f32)      q = x / scale to the nearest integer, ties to even
//
// q is the rounding of the exact quotient: r = rint(x * (1 / scale)) is at most one off (only next to a half), and
// x - r scale is exact in one fused multiply-add (|r| <= 127, |x - r scale| <= scale), so comparing it with half a
// scale settles the case.  A reciprocal per row and no division per element.
// The integer sums are exact (k <= 131072: 127 * 127 * k < 2^31); the only roundings are the sum's conversion to f32,
// the two scales, the bias, and the output type.
#include "gemm_launch.hpp"

#define YP_QR_THREADS 256

int64_t yp_qrow_bytes(int64_t k) { return yp_pad_k(k, 1); }

struct yp_row_scale { float scale, unit, inv, half; float pre; };

// scale of a row from the bits of its largest magnitude (NaN and infinities have the largest bits of all)
__device__ __forceinline__ yp_row_scale yp_make_scale(uint32_t top) {
  yp_row_scale r;
  if (top >= 0x7f800000u) { r.scale = NAN; r.unit = r.inv = r.half = r.pre = 0.0f; return r; }
  const float amax = __builtin_bit_cast(float, top);
  r.scale = amax / 127.0f;
  r.pre = amax < 0x1p-60f ? 0x1p64f : 1.0f;          // keeps the reciprocal of a tiny scale finite; exact
  r.unit = r.scale * r.pre;
  r.inv = r.unit > 0.0f ? 1.0f / r.unit : 0.0f;
  r.half = 0.5f * r.unit;
  return r;
}
__device__ __forceinline__ int yp_quantize(float x, const yp_row_scale& s) {
  const float v = x * s.pre;
  float r = rintf(v * s.inv);
  r = fminf(fmaxf(r, -127.0f), 127.0f);
  const float rem = __builtin_fmaf(-r, s.unit, v);
  const bool odd = ((int)r & 1) != 0;
  if (rem > s.half || (rem == s.half && odd && s.unit > 0.0f)) r += 1.0f;
  else if (rem < -s.half || (rem == -s.half && odd && s.unit > 0.0f)) r -= 1.0f;
  return (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

// LANES threads per row; a thread takes 16-byte chunks of the row.
template <int TYPE, int LANES>
__global__ __launch_bounds__(YP_QR_THREADS) void yp_quantize_rows_kernel(const void* x, int64_t rows, int k, int kp, char* q, float* scale, int vec) {
  typedef typename yp_type<TYPE>::elem elem;
  constexpr int E = 16 / (int)sizeof(elem);
  typedef elem ev __attribute__((ext_vector_type(E)));
  __shared__ uint32_t red[YP_QR_THREADS / 64];
  const int lane = (int)threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * (YP_QR_THREADS / LANES) + (int)threadIdx.x / LANES;
  const bool live = row < rows;
  const elem* const src = reinterpret_cast<const elem*>(x) + (live ? row : 0) * k;
  auto get = [&](int c, float (&v)[E]) {
    if (vec && c + E <= k) {
      const ev t = *reinterpret_cast<const ev*>(src + c);
#pragma unroll
      for (int u = 0; u < E; ++u) v[u] = (float)t[u];
    } else {
#pragma unroll
      for (int u = 0; u < E; ++u) v[u] = c + u < k ? (float)src[c + u] : 0.0f;
    }
  };
  uint32_t top = 0;
  if (live)
    for (int c = lane * E; c < k; c += LANES * E) {
      float v[E];
      get(c, v);
#pragma unroll
      for (int u = 0; u < E; ++u) top = max(top, __builtin_bit_cast(uint32_t, v[u]) & 0x7fffffffu);
    }
#pragma unroll
  for (int s = (LANES < 64 ? LANES : 64) / 2; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) top = max(top, red[(threadIdx.x / LANES) * (LANES / 64) + w]);
  }
  if (!live) return;
  const yp_row_scale s = yp_make_scale(top);
  if (lane == 0) scale[row] = s.scale;
  char* const dst = q + row * kp;
  for (int c = lane * E; c < kp; c += LANES * E) {
    float v[E];
    get(c, v);
    uint32_t word[E / 4];
#pragma unroll
    for (int w = 0; w < E / 4; ++w) {
      word[w] = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) word[w] |= ((uint32_t)yp_quantize(v[w * 4 + u], s) & 0xffu) << (8 * u);
      reinterpret_cast<uint32_t*>(dst + c)[w] = word[w];
    }
  }
}

template <int TYPE>
static hipError_t quantize_t(int64_t rows, int k, const void* x, void* q, float* scale, hipStream_t st) {
  const int kp = (int)yp_qrow_bytes(k);
  const int vec = ((int64_t)k * yp_type<TYPE>::bytes) % 16 == 0 && ((uintptr_t)x & 15) == 0;
  if (k <= 2048)
    hipLaunchKernelGGL((yp_quantize_rows_kernel<TYPE, 64>), dim3((unsigned)((rows + 3) / 4)), dim3(YP_QR_THREADS), 0, st, x, rows, k, kp, (char*)q, scale, vec);
  else
    hipLaunchKernelGGL((yp_quantize_rows_kernel<TYPE, 256>), dim3((unsigned)rows), dim3(YP_QR_THREADS), 0, st, x, rows, k, kp, (char*)q, scale, vec);
  return hipGetLastError();
}

hipError_t yp_launch_quantize_rows(int64_t rows, int k, int type, const void* x, void* q, float* scale, hipStream_t st) {
  return type == YP_F32 ? quantize_t<YP_T_F32>(rows, k, x, q, scale, st)
       : type == YP_BF16 ? quantize_t<YP_T_BF16>(rows, k, x, q, scale, st) : quantize_t<YP_T_F16>(rows, k, x, q, scale, st);
}

template <int OUT>
struct yp_epi_scaled {
  const float *x_scale, *w_scale, *bias;
  void* out;
  int vec;
  template <int TYPE, int SHAPE, int MI, int NJ, class Acc>
  __device__ __forceinline__ void apply(const yp_gemm& g, Acc (&acc)[MI][NJ], const yp_place& at) const {
    typedef yp_shape<SHAPE> S;
    int i0, j0;
    yp_origin<SHAPE>(at, i0, j0);
    float sx[NJ];
#pragma unroll
    for (int n = 0; n < NJ; ++n) { const int j = j0 + yp_frag_at<S::BN, NJ>(n); sx[n] = j < g.J ? x_scale[j] : 0.0f; }
    yp_f4 sw[MI], b[MI];
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + yp_frag_at<S::BM, MI>(m) + r;
        sw[m][r] = i < g.I ? w_scale[i] : 0.0f;
        b[m][r] = bias && i < g.I ? bias[i] : 0.0f;
      }
    yp_put_tile<OUT, SHAPE, false, MI, NJ>(at, out, g.I, g.I, g.J, vec != 0, [&](int m, int n) {
      yp_f4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = __builtin_fmaf((float)acc[m][n][r] * sx[n], sw[m][r], b[m][r]);
      return y;
    });
  }
};

template <int OUT>
static hipError_t linear_t(const yp_gemm& g, const float* x_scale, const float* w_scale, const float* bias, void* out, hipStream_t st) {
  yp_epi_scaled<OUT> e;
  e.x_scale = x_scale; e.w_scale = w_scale; e.bias = bias; e.out = out;
  e.vec = (int64_t)g.I * yp_type<OUT>::bytes % 16 == 0 && ((uintptr_t)out & 15) == 0;
  return yp_launch_gemm<YP_T_I8>(yp_plan_tiles(g.I, g.J, g.steps, false), g, e, st);
}

hipError_t yp_launch_quantized_linear(int rows, int v, int k, const void* xq, const float* x_scale, const void* wq, const float* w_scale,
                                      const float* bias, void* out, int out_type, hipStream_t st) {
  yp_gemm g = {};
  g.lda = g.ldb = yp_qrow_bytes(k);
  g.a = (const char*)wq; g.b = (const char*)xq;
  g.I = v; g.J = rows; g.steps = (int)(g.lda / YP_TILE_KB);
  return out_type == YP_F32 ? linear_t<YP_T_F32>(g, x_scale, w_scale, bias, out, st)
       : out_type == YP_BF16 ? linear_t<YP_T_BF16>(g, x_scale, w_scale, bias, out, st) : linear_t<YP_T_F16>(g, x_scale, w_scale, bias, out, st);
}
