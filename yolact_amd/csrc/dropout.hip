// Dropout with its mask computed again wherever it is needed: element i is kept if word i % 4 of Philox4x32-10 (Salmon,
// Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter state[1] + i / 4 under the key
// state[0] is at least floor(p 2^32).  A thread computes one counter's four words for four consecutive elements.
// Bound by memory: one read and one write; 20 32 x 32 -> 64-bit products per 4 elements beside them.
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
  typedef elem e4 __attribute__((ext_vector_type(4)));
  const elem* const x = reinterpret_cast<const elem*>(xp);
  const uint64_t key = (uint64_t)state[0], first = (uint64_t)state[1];
  const int64_t quads = (count + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * YP_DO_THREADS + threadIdx.x; i < quads; i += (int64_t)gridDim.x * YP_DO_THREADS) {
    uint32_t w[4];
    yp_philox(key, first + (uint64_t)i, w);
    const int n = count - i * 4 < 4 ? (int)(count - i * 4) : 4;
    yp_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (vec && n == 4) {
      const e4 t = *reinterpret_cast<const e4*>(x + i * 4);
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = (float)t[u];
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) if (u < n) v[u] = (float)x[i * 4 + u];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = (uint64_t)w[u] >= least ? v[u] * scale : 0.0f;
    if (vec) yp_store4<TYPE, true>(yp, i * 4, v, n);
    else yp_store4<TYPE, false>(yp, i * 4, v, n);
  }
}

template <int TYPE>
static hipError_t dropout_t(int64_t count, double p, const int64_t* state, const void* x, void* y, hipStream_t st) {
  const uint64_t least = (uint64_t)floor(p * 4294967296.0);     // (p = 1: 2^32, which no word reaches)
  const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  const int64_t blocks = ((count + 3) / 4 + YP_DO_THREADS - 1) / YP_DO_THREADS;
  const int vec = (((uintptr_t)x | (uintptr_t)y) & (4 * sizeof(typename yp_type<TYPE>::elem) - 1)) == 0;
  hipLaunchKernelGGL(yp_dropout_kernel<TYPE>, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(YP_DO_THREADS), 0, st, x, y, count, least, scale, state, vec);
  return hipGetLastError();
}

hipError_t yp_launch_dropout(int64_t count, int type, double p, const int64_t* state, const void* x, void* y, hipStream_t st) {
  return type == YP_F32 ? dropout_t<YP_T_F32>(count, p, state, x, y, st)
       : type == YP_BF16 ? dropout_t<YP_T_BF16>(count, p, state, x, y, st) : dropout_t<YP_T_F16>(count, p, state, x, y, st);
}
