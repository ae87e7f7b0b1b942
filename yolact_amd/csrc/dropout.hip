// Dropout with its mask computed again wherever it is needed: element i is kept if word i % 4 of Philox4x32-10 (Salmon,
// Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter state[1] + i / 4 under the key
// state[0] is at least floor(p 2^32).  A thread takes 16 bytes: one counter's four words for four f32, two counters' for
// eight 16-bit elements.  Bound by memory: one read and one write; 5 products of 32 x 32 -> 64 bits per element beside
// them.
#include "gemm_launch.hpp"

#define YP_DO_THREADS 256

__device__ __forceinline__ void yp_philox(uint64_t key, uint64_t counter, uint32_t (&w)[4]) {
  uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

template <int TYPE>
__global__ __launch_bounds__(YP_DO_THREADS) void yp_dropout_kernel(const void* xp, void* yp, int64_t count, uint64_t least, float scale,
                                                                   const int64_t* state, int vec) {
  typedef typename yp_type<TYPE>::elem elem;
  constexpr int E = 16 / yp_type<TYPE>::bytes;
  typedef elem eE __attribute__((ext_vector_type(E)));
  const uint64_t key = (uint64_t)state[0], first = (uint64_t)state[1];
  for (int64_t i = ((int64_t)blockIdx.x * YP_DO_THREADS + threadIdx.x) * E; i < count; i += (int64_t)gridDim.x * YP_DO_THREADS * E) {
    const elem* const x = reinterpret_cast<const elem*>(xp) + i;
    elem* const y = reinterpret_cast<elem*>(yp) + i;
    const bool whole = vec && i + E <= count;
    eE v;
    if (whole) v = *reinterpret_cast<const eE*>(x);
    else
#pragma unroll
      for (int u = 0; u < E; ++u) v[u] = i + u < count ? x[u] : (elem)0;
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      uint32_t w[4];
      yp_philox(key, first + (uint64_t)(i / 4 + q), w);
#pragma unroll
      for (int u = 0; u < 4; ++u) v[q * 4 + u] = (uint64_t)w[u] >= least ? (elem)((float)v[q * 4 + u] * scale) : (elem)0;
    }
    if (whole) *reinterpret_cast<eE*>(y) = v;
    else
#pragma unroll
      for (int u = 0; u < E; ++u) if (i + u < count) y[u] = v[u];
  }
}

template <int TYPE>
static hipError_t dropout_t(int64_t count, double p, const int64_t* state, const void* x, void* y, hipStream_t st) {
  const uint64_t least = (uint64_t)floor(p * 4294967296.0);     // (p = 1: 2^32, which no word reaches)
  const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  const int64_t per = (int64_t)YP_DO_THREADS * (16 / yp_type<TYPE>::bytes), blocks = (count + per - 1) / per;
  const int vec = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
  hipLaunchKernelGGL(yp_dropout_kernel<TYPE>, dim3((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22))), dim3(YP_DO_THREADS), 0, st, x, y, count, least, scale, state, vec);
  return hipGetLastError();
}

hipError_t yp_launch_dropout(int64_t count, int type, double p, const int64_t* state, const void* x, void* y, hipStream_t st) {
  return type == YP_F32 ? dropout_t<YP_T_F32>(count, p, state, x, y, st)
       : type == YP_BF16 ? dropout_t<YP_T_BF16>(count, p, state, x, y, st) : dropout_t<YP_T_F16>(count, p, state, x, y, st);
}
