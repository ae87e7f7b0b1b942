// Quantized linear: out = (xq wq^T) x_scale w_scale + bias with 8-bit integers and one scale per row of either operand.
//
//   scale = max|x| / 127 (f32)      q = x / scale to the nearest integer, ties to even
//
// q is the rounding of the exact quotient: r = x * (1 / scale) rounded to a whole number is at most one off, and only next
// to a half; x - r scale is exact in one fused multiply-add (|r| <= 127, |x - r scale| <= scale), so comparing it with half
// a scale settles the case.  A reciprocal per row and no division per element; the comparison is one maximum per element,
// and only where some element of the thread's lies within 2^-12 of a half (1 in 2000 chunks) is each looked at.
// The integer sums are exact (k <= 131072: 127 * 127 * k < 2^31); the only roundings are the sum's conversion to f32,
// the two scales, the bias, and the output type.
#include "gemm_launch.hpp"

#define YP_QR_THREADS 256

int64_t yp_qrow_bytes(int64_t k) { return yp_pad_k(k, 1); }

struct yp_row_scale { float scale, unit, inv, half, near; };

// scale of a row from the bits of its largest magnitude (NaN and infinities have the largest bits of all)
__device__ __forceinline__ yp_row_scale yp_make_scale(uint32_t top) {
  yp_row_scale r;
  if (top >= 0x7f800000u) { r.scale = NAN; r.unit = r.inv = r.half = 0.0f; r.near = -1.0f; return r; }
  const float amax = __builtin_bit_cast(float, top);
  r.scale = amax / 127.0f;
  const bool tiny = amax < 0x1p-60f;                // near = -1: every element the careful way, scaled up by 2^64 (exact)
  r.unit = r.scale * (tiny ? 0x1p64f : 1.0f);
  r.inv = r.unit > 0.0f ? 1.0f / r.unit : 0.0f;
  r.half = 0.5f * r.unit;
  r.near = tiny ? -1.0f : r.half * (1.0f - 0x1p-12f);
  return r;
}
static __device__ __attribute__((noinline)) uint32_t yp_quantize_carefully(float x, const yp_row_scale s) {
  const float v = s.near < 0.0f ? x * 0x1p64f : x;
  float r = fminf(fmaxf(rintf(v * s.inv), -127.0f), 127.0f);
  const float rem = __builtin_fmaf(-r, s.unit, v);
  const bool odd = ((int)r & 1) != 0 && s.unit > 0.0f;
  if (rem > s.half || (rem == s.half && odd)) r += 1.0f;
  else if (rem < -s.half || (rem == -s.half && odd)) r -= 1.0f;
  return s.unit > 0.0f ? (uint32_t)(int)fminf(fmaxf(r, -127.0f), 127.0f) & 0xffu : 0u;
}
// N elements to N bytes
template <int N>
__device__ __forceinline__ void yp_quantize(const float (&x)[N], const yp_row_scale& s, uint32_t (&word)[N / 4]) {
  uint32_t bits[N];
  float far = 0.0f;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const float m = __builtin_fmaf(x[u], s.inv, 12582912.0f);        // 1.5 * 2^23: the sum's low byte is the whole number
    far = fmaxf(far, fabsf(__builtin_fmaf(-(m - 12582912.0f), s.unit, x[u])));
    bits[u] = __builtin_bit_cast(uint32_t, m);
  }
  if (far > s.near) {
#pragma unroll
    for (int u = 0; u < N; ++u) bits[u] = yp_quantize_carefully(x[u], s);
  }
#pragma unroll
  for (int w = 0; w < N / 4; ++w) {
    const uint32_t lo = __builtin_amdgcn_perm(bits[w * 4 + 1], bits[w * 4], 0x0c0c0400u), hi = __builtin_amdgcn_perm(bits[w * 4 + 3], bits[w * 4 + 2], 0x0c0c0400u);
    word[w] = lo | hi << 16;
  }
}

// A row's elements in 16-byte chunks: chunk c as floats, zeros past the end.
template <int TYPE>
struct yp_row_reader {
  typedef typename yp_type<TYPE>::elem elem;
  static constexpr int E = 16 / (int)sizeof(elem);
  typedef elem ev __attribute__((ext_vector_type(E)));
  const elem* src;
  int k, vec;              // vec: the row starts on 16 bytes
  __device__ __forceinline__ ev get(int c) const {
    const int e = c * E;
    if (vec && e + E <= k) return *reinterpret_cast<const ev*>(src + e);
    ev t;
#pragma unroll
    for (int u = 0; u < E; ++u) t[u] = e + u < k ? src[e + u] : (elem)0;
    return t;
  }
  static __device__ __forceinline__ uint32_t top(const ev& t, uint32_t m) {
#pragma unroll
    for (int u = 0; u < E; ++u) m = max(m, __builtin_bit_cast(uint32_t, (float)t[u]) & 0x7fffffffu);
    return m;
  }
  static __device__ __forceinline__ void quantize(const ev& t, const yp_row_scale& s, uint32_t (&word)[E / 4]) {
    float x[E];
#pragma unroll
    for (int u = 0; u < E; ++u) x[u] = (float)t[u];
    yp_quantize<E>(x, s, word);
  }
  static __device__ __forceinline__ void put(char* dst, int c, const ev& t, const yp_row_scale& s) {
    uint32_t word[E / 4];
    quantize(t, s, word);
#pragma unroll
    for (int w = 0; w < E / 4; ++w) reinterpret_cast<uint32_t*>(dst + c * E)[w] = word[w];
  }
};

// LANES threads per row, a thread takes chunks LANES apart and keeps the first YP_QR_KEEP of them in registers between the
// two passes (maximum, quotients); a longer row's are read again, out of the caches.
#define YP_QR_KEEP 4
template <int TYPE, int LANES>
__global__ __launch_bounds__(YP_QR_THREADS) void yp_quantize_rows_kernel(const void* x, int64_t rows, int k, int kp, char* q, float* scale, int vec) {
  typedef yp_row_reader<TYPE> R;
  constexpr int PER = YP_QR_THREADS / LANES;
  __shared__ uint32_t red[2][YP_QR_THREADS / 64];
  const int lane = (int)threadIdx.x % LANES, chunks = kp / R::E;
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * PER; first < rows; first += (int64_t)gridDim.x * PER, turn ^= 1) {
    const int64_t row = first + (int)threadIdx.x / LANES;
    const bool live = row < rows;
    const R r = {reinterpret_cast<const typename R::elem*>(x) + (live ? row : 0) * k, k, vec};
    typename R::ev keep[YP_QR_KEEP];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < YP_QR_KEEP; ++u) if (lane + u * LANES < chunks) keep[u] = r.get(lane + u * LANES);
#pragma unroll
    for (int u = 0; u < YP_QR_KEEP; ++u) if (lane + u * LANES < chunks) top = R::top(keep[u], top);
    for (int c = lane + YP_QR_KEEP * LANES; c < chunks; c += LANES) top = R::top(r.get(c), top);
#pragma unroll
    for (int s = (LANES < 64 ? LANES : 64) / 2; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if constexpr (LANES > 64) {
      if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < LANES / 64; ++w) top = max(top, red[turn][(int)threadIdx.x / LANES * (LANES / 64) + w]);
    }
    if (!live) continue;
    const yp_row_scale s = yp_make_scale(top);
    if (lane == 0) scale[row] = s.scale;
    char* const dst = q + row * kp;
#pragma unroll
    for (int u = 0; u < YP_QR_KEEP; ++u) if (lane + u * LANES < chunks) R::put(dst, lane + u * LANES, keep[u], s);
    for (int c = lane + YP_QR_KEEP * LANES; c < chunks; c += LANES) R::put(dst, c, r.get(c), s);
  }
}

template <int TYPE>
static int row_vec(int k, const void* x) { return (int64_t)k * yp_type<TYPE>::bytes % 16 == 0 && ((uintptr_t)x & 15) == 0; }

template <int TYPE, int LANES>
static hipError_t quantize_l(int64_t rows, int k, const void* x, void* q, float* scale, hipStream_t st) {
  const int64_t blocks = (rows * LANES + YP_QR_THREADS - 1) / YP_QR_THREADS;
  hipLaunchKernelGGL((yp_quantize_rows_kernel<TYPE, LANES>), dim3((unsigned)(blocks < (1 << 22) ? blocks : (1 << 22))), dim3(YP_QR_THREADS), 0, st, x, rows, k,
                     (int)yp_qrow_bytes(k), (char*)q, scale, row_vec<TYPE>(k, x));
  return hipGetLastError();
}
// as many threads to a row as keep it in registers
template <int TYPE>
static hipError_t quantize_t(int64_t rows, int k, const void* x, void* q, float* scale, hipStream_t st) {
  const int64_t chunks = yp_qrow_bytes(k) * yp_type<TYPE>::bytes / 16;
  return chunks <= 16 * YP_QR_KEEP ? quantize_l<TYPE, 16>(rows, k, x, q, scale, st)
       : chunks <= 64 * YP_QR_KEEP ? quantize_l<TYPE, 64>(rows, k, x, q, scale, st)
       : chunks <= 128 * YP_QR_KEEP ? quantize_l<TYPE, 128>(rows, k, x, q, scale, st) : quantize_l<TYPE, 256>(rows, k, x, q, scale, st);
}

hipError_t yp_launch_quantize_rows(int64_t rows, int k, int type, const void* x, void* q, float* scale, hipStream_t st) {
  return type == YP_F32 ? quantize_t<YP_T_F32>(rows, k, x, q, scale, st)
       : type == YP_BF16 ? quantize_t<YP_T_BF16>(rows, k, x, q, scale, st) : quantize_t<YP_T_F16>(rows, k, x, q, scale, st);
}

// ---- one row: the weight is read once and that is all there is -----------------------------------------------------
// A workgroup holds the row in LDS, quantized by itself - 8 KB from L2 cost less than another launch - and its waves walk
// over rows of the weight, YP_OR_W at a time: a lane reads 16 bytes of k of each.  The matrix instruction takes lane l's 16
// bytes as quarter l >> 4 of row and column l & 15, of the weight and of x alike: its diagonal holds the sums of four lanes'
// products, which the wave adds up at the end.  YP_OR_C chunks of each are on their way at a time - 16 KB a wave -, the first ones while x is
// quantized.  26 us for 32000 x 4096 (131 MB: 5.0 TB/s); from two rows on the tile engine is faster (30 us; a kernel of this kind,
// with dot products, took 43 for two rows and 100 for eight).
#define YP_OR_W 4
#define YP_OR_C 4
#define YP_OR_LDS 61440

template <int XTYPE, int OUT>
__global__ __launch_bounds__(YP_QR_THREADS, 4) void yp_one_row_kernel(const void* x, const float* x_scale, int v, int k, int kp, const char* wq, const float* w_scale,
                                                                   const float* bias, void* out, int vec) {
  typedef typename yp_type<OUT>::elem oelem;
  extern __shared__ __align__(16) char xl[];      // [kp]
  __shared__ uint32_t red[YP_QR_THREADS / 64];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = (int)blockIdx.x * (YP_QR_THREADS / 64) + (tid >> 6), waves = (int)gridDim.x * (YP_QR_THREADS / 64);
  const int chunks = kp / 16;
  yp_i4 w[YP_OR_C][YP_OR_W];
  auto get_w = [&](int j0, int c0) {              // (zeros past the row)
#pragma unroll
    for (int c = 0; c < YP_OR_C; ++c)
#pragma unroll
      for (int u = 0; u < YP_OR_W; ++u)
        w[c][u] = c0 + c * 64 < chunks ? *reinterpret_cast<const yp_i4*>(wq + (int64_t)min(j0 + u, v - 1) * kp + (c0 + c * 64) * 16) : yp_i4{0, 0, 0, 0};
  };
  int64_t j0 = (int64_t)wave * YP_OR_W;
  if (j0 < v) get_w((int)j0, lane);
  float sx;
  if constexpr (XTYPE == YP_T_I8) {
    for (int c = tid; c < chunks; c += YP_QR_THREADS) reinterpret_cast<yp_i4*>(xl)[c] = reinterpret_cast<const yp_i4*>(x)[c];
    sx = x_scale[0];
  } else {
    typedef yp_row_reader<XTYPE> R;
    const int ec = kp / R::E;
    const R rr = {reinterpret_cast<const typename R::elem*>(x), k, vec};
    uint32_t top = 0;
    for (int c = tid; c < ec; c += YP_QR_THREADS) top = R::top(rr.get(c), top);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
    if (lane == 0) red[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < YP_QR_THREADS / 64; ++u) top = max(top, red[u]);
    const yp_row_scale s = yp_make_scale(top);
    sx = s.scale;
    for (int c = tid; c < ec; c += YP_QR_THREADS) R::put(xl, c, rr.get(c), s);
  }
  __syncthreads();
  for (; j0 < v; j0 += (int64_t)waves * YP_OR_W) {
    yp_i4 acc[YP_OR_W];
#pragma unroll
    for (int u = 0; u < YP_OR_W; ++u) acc[u] = yp_i4{0, 0, 0, 0};
    for (int c0 = lane; c0 - lane < chunks; c0 += YP_OR_C * 64) {
      if (c0 != lane) get_w((int)j0, c0);
#pragma unroll
      for (int c = 0; c < YP_OR_C; ++c) {
        if (c0 - lane + c * 64 < chunks) {              // (for the whole wave: a lane past the row has zeros)
          const yp_i4 xv = *reinterpret_cast<const yp_i4*>(xl + min(c0 + c * 64, chunks - 1) * 16);
#pragma unroll
          for (int u = 0; u < YP_OR_W; ++u) acc[u] = yp_mma<YP_T_I8>(w[c][u], xv, acc[u]);
        }
      }
    }
    if (j0 + (int64_t)waves * YP_OR_W < v) get_w((int)j0 + waves * YP_OR_W, lane);
#pragma unroll
    for (int u = 0; u < YP_OR_W; ++u) {
      const int r = (lane & 15) - (lane >> 4) * 4;      // C[i][i]: lane i + 16 (i / 4), register i % 4
      int t = r == 0 ? acc[u][0] : r == 1 ? acc[u][1] : r == 2 ? acc[u][2] : r == 3 ? acc[u][3] : 0;
#pragma unroll
      for (int s = 32; s > 0; s >>= 1) t += __shfl_xor(t, s);
      const int64_t j = j0 + u;
      if (lane == u && j < v) reinterpret_cast<oelem*>(out)[j] = (oelem)__builtin_fmaf((float)t * sx, w_scale[j], bias ? bias[j] : 0.0f);
    }
  }
}

template <int XTYPE, int OUT>
static hipError_t one_row_t(int v, int k, const void* x, const float* x_scale, const void* wq, const float* w_scale, const float* bias, void* out, hipStream_t st) {
  const int kp = (int)yp_qrow_bytes(k);
  const int per = YP_OR_W * (YP_QR_THREADS / 64);                 // rows of the weight per workgroup and turn
  const int64_t turns = ((int64_t)v + per - 1) / per;
  int64_t resident = 163840 / (kp + 256);                         // workgroups a CU's LDS holds; more would only quantize x again
  if (resident > 4) resident = 4;                                 // (and its registers: 4)
  const unsigned blocks = (unsigned)(turns < 256 * resident ? turns : 256 * resident);
  int vec = 0;
  if constexpr (XTYPE != YP_T_I8) vec = row_vec<XTYPE>(k, x);
  hipLaunchKernelGGL((yp_one_row_kernel<XTYPE, OUT>), dim3(blocks), dim3(YP_QR_THREADS), (size_t)kp, st, x, x_scale, v, k, kp, (const char*)wq, w_scale, bias, out, vec);
  return hipGetLastError();
}
template <int XTYPE>
static hipError_t one_row_x(int v, int k, const void* x, const float* x_scale, const void* wq, const float* w_scale, const float* bias, void* out, int out_type, hipStream_t st) {
  return out_type == YP_F32 ? one_row_t<XTYPE, YP_T_F32>(v, k, x, x_scale, wq, w_scale, bias, out, st)
       : out_type == YP_BF16 ? one_row_t<XTYPE, YP_T_BF16>(v, k, x, x_scale, wq, w_scale, bias, out, st)
                             : one_row_t<XTYPE, YP_T_F16>(v, k, x, x_scale, wq, w_scale, bias, out, st);
}

// ---- a small weight: the head over anchors ---------------------------------------------------------------------------
// x is read once, and that is most of it: 25.4 us for 76992 x 256 float32 against 81 rows (105 MB: 4.1 TB/s; quantizing
// and the tile engine apart 52 us).  From two rows on: the device takes 0 to 2 us longer below 4096 than with the two
// kernels, a caller launches one less (9.7 us a call against 11.5).  A wave takes 16 rows and keeps them in registers in the order of the matrix
// instruction - lane l holds row l & 15, and of every 64 k those that 16-byte loads bring to quarter l >> 4 (which k they
// are does not matter as long as the weight has the same order: it is laid out so in LDS, once per workgroup) -, so the
// row's maximum is two shuffles and the quotients never leave the lane.  The results go through LDS, 16 rows at a time,
// and out as one run of 16-byte stores: 16 rows are a multiple of 16 bytes whatever v is.
#define YP_SW_LDS 81920

template <int XTYPE, int OUT, int STEPS>   // STEPS: 64 k each, at most
__global__ __launch_bounds__(YP_QR_THREADS) void yp_small_weight_kernel(const void* x, const float* x_scale, int rows, int v, int k, int kp, const char* wq,
                                                                const float* w_scale, const float* bias, void* out, int vec, int out_vec) {
  typedef typename yp_type<OUT>::elem oelem;
  constexpr int XB = yp_type<XTYPE>::bytes, E = 16 / XB, LOADS = 4 * XB / 4;   // loads per 64 k: 4 (f32), 2, 1
  extern __shared__ __align__(16) char lds[];          // [v padded to 16][kp] weight | [2][v padded] scales, biases | per wave [16][v] results
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, row = lane & 15, g = lane >> 4;
  const int vt = (v + 15) / 16, steps = kp / 64;
  // chunk c of a weight row (16 k): its 64 k's quarter-chunks, reordered; slot exclusive-ored by the row against bank conflicts
  for (int c = tid; c < vt * 16 * (kp / 16); c += YP_QR_THREADS) {
    const int i = c / (kp / 16), q = c - i * (kp / 16), s = q >> 2, qg = q & 3;
    yp_i4 w = {0, 0, 0, 0};
    if (i < v) {
      const char* const src = wq + (int64_t)i * kp + s * 64;
#pragma unroll
      for (int e = 0; e < LOADS; ++e)
#pragma unroll
        for (int u = 0; u < E / 4; ++u) w[e * (E / 4) + u] = *reinterpret_cast<const int*>(src + e * 4 * E + qg * E + u * 4);
    }
    *reinterpret_cast<yp_i4*>(lds + i * kp + ((q ^ (i & 7)) * 16)) = w;
  }
  float* const sw = reinterpret_cast<float*>(lds + vt * 16 * kp);
  for (int i = tid; i < vt * 16; i += YP_QR_THREADS) { sw[i] = i < v ? w_scale[i] : 0.0f; sw[vt * 16 + i] = bias && i < v ? bias[i] : 0.0f; }
  oelem* const stage = reinterpret_cast<oelem*>(lds + vt * 16 * (kp + 8)) + wave * 16 * v;
  __syncthreads();
  for (int64_t r0 = ((int64_t)blockIdx.x * 4 + wave) * 16; r0 < rows; r0 += (int64_t)gridDim.x * 64) {
    const int64_t r = r0 + row < rows ? r0 + row : rows - 1;
    yp_i4 f[STEPS];
    float sx;
    if constexpr (XTYPE == YP_T_I8) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        f[s] = s < steps ? *reinterpret_cast<const yp_i4*>(reinterpret_cast<const char*>(x) + r * kp + s * 64 + g * 16) : yp_i4{0, 0, 0, 0};
      sx = x_scale[r];
    } else {
      typedef yp_row_reader<XTYPE> R;
      const R rr = {reinterpret_cast<const typename R::elem*>(x) + r * k, k, vec};
      typename R::ev t[STEPS][LOADS];
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (s < steps)
#pragma unroll
          for (int e = 0; e < LOADS; ++e) t[s][e] = rr.get(s * (64 / E) + e * 4 + g);
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (s < steps)
#pragma unroll
          for (int e = 0; e < LOADS; ++e) top = R::top(t[s][e], top);
      top = max(top, (uint32_t)__shfl_xor((int)top, 16));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32));
      const yp_row_scale sc = yp_make_scale(top);
      sx = sc.scale;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        f[s] = yp_i4{0, 0, 0, 0};
        if (s < steps)
#pragma unroll
          for (int e = 0; e < LOADS; ++e) {
            uint32_t word[E / 4];
            R::quantize(t[s][e], sc, word);
#pragma unroll
            for (int u = 0; u < E / 4; ++u) f[s][e * (E / 4) + u] = (int)word[u];
          }
      }
    }
    for (int it = 0; it < vt; ++it) {
      yp_i4 acc = {0, 0, 0, 0};
      const int i = it * 16 + row;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (s < steps) acc = yp_mma<YP_T_I8>(*reinterpret_cast<const yp_i4*>(lds + i * kp + (((s * 4 + g) ^ (i & 7)) * 16)), f[s], acc);
      const yp_f4 ws = *reinterpret_cast<const yp_f4*>(sw + it * 16 + g * 4), b = *reinterpret_cast<const yp_f4*>(sw + vt * 16 + it * 16 + g * 4);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int o = it * 16 + g * 4 + u;
        if (o < v) stage[row * v + o] = (oelem)__builtin_fmaf((float)acc[u] * sx, ws[u], b[u]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the wave's own rows: no other wave to wait for)
    const int total = (int)(rows - r0 < 16 ? rows - r0 : 16) * v, per = 16 / (int)sizeof(oelem);
    oelem* const to = reinterpret_cast<oelem*>(out) + r0 * v;
    if (out_vec) {
      for (int c = lane; c < total / per; c += 64) reinterpret_cast<yp_i4*>(to)[c] = reinterpret_cast<const yp_i4*>(stage)[c];
      for (int c = total / per * per + lane; c < total; c += 64) to[c] = stage[c];
    } else {
      for (int c = lane; c < total; c += 64) to[c] = stage[c];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

static bool small_weight(int v, int64_t kp, int out_bytes) {
  return kp <= 512 && (int64_t)(v + 15) / 16 * 16 * (kp + 8) + (int64_t)64 * v * out_bytes <= YP_SW_LDS;
}
template <int XTYPE, int OUT>
static hipError_t small_weight_t(int rows, int v, int k, const void* x, const float* x_scale, const void* wq, const float* w_scale, const float* bias, void* out, hipStream_t st) {
  const int kp = (int)yp_qrow_bytes(k);
  const size_t lds = (size_t)(v + 15) / 16 * 16 * (kp + 8) + (size_t)64 * v * yp_type<OUT>::bytes;
  int64_t blocks = ((int64_t)rows + 63) / 64, resident = 256 * (163840 / (int64_t)lds < 4 ? 163840 / (int64_t)lds : 4);
  if (blocks > resident) blocks = resident;
  int vec = 0;
  if constexpr (XTYPE != YP_T_I8) vec = row_vec<XTYPE>(k, x);
  const int out_vec = ((uintptr_t)out & 15) == 0;
  const void* const fn = kp <= 256 ? reinterpret_cast<const void*>(&yp_small_weight_kernel<XTYPE, OUT, 4>) : reinterpret_cast<const void*>(&yp_small_weight_kernel<XTYPE, OUT, 8>);
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, YP_SW_LDS);
    if (e != hipSuccess) return e;
  }
  if (kp <= 256)
    hipLaunchKernelGGL((yp_small_weight_kernel<XTYPE, OUT, 4>), dim3((unsigned)blocks), dim3(YP_QR_THREADS), lds, st, x, x_scale, rows, v, k, kp, (const char*)wq, w_scale, bias, out, vec, out_vec);
  else
    hipLaunchKernelGGL((yp_small_weight_kernel<XTYPE, OUT, 8>), dim3((unsigned)blocks), dim3(YP_QR_THREADS), lds, st, x, x_scale, rows, v, k, kp, (const char*)wq, w_scale, bias, out, vec, out_vec);
  return hipGetLastError();
}
template <int XTYPE>
static hipError_t small_weight_x(int rows, int v, int k, const void* x, const float* x_scale, const void* wq, const float* w_scale, const float* bias, void* out, int out_type,
                         hipStream_t st) {
  return out_type == YP_F32 ? small_weight_t<XTYPE, YP_T_F32>(rows, v, k, x, x_scale, wq, w_scale, bias, out, st)
       : out_type == YP_BF16 ? small_weight_t<XTYPE, YP_T_BF16>(rows, v, k, x, x_scale, wq, w_scale, bias, out, st)
                             : small_weight_t<XTYPE, YP_T_F16>(rows, v, k, x, x_scale, wq, w_scale, bias, out, st);
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
  return yp_launch_gemm<YP_T_I8>(yp_plan_tiles(g.I, g.J, g.steps, YP_TILE_L), g, e, st);
}

hipError_t yp_launch_quantized_linear(int rows, int v, int k, int x_type, const void* x, const float* x_scale, const void* wq, const float* w_scale,
                                      const float* bias, void* workspace, void* out, int out_type, hipStream_t st) {
  const int64_t kp = yp_qrow_bytes(k);
  if (rows == 1 && kp <= YP_OR_LDS)
    return x_type == YP_INT8 ? one_row_x<YP_T_I8>(v, k, x, x_scale, wq, w_scale, bias, out, out_type, st)
         : x_type == YP_F32 ? one_row_x<YP_T_F32>(v, k, x, x_scale, wq, w_scale, bias, out, out_type, st)
         : x_type == YP_BF16 ? one_row_x<YP_T_BF16>(v, k, x, x_scale, wq, w_scale, bias, out, out_type, st)
                             : one_row_x<YP_T_F16>(v, k, x, x_scale, wq, w_scale, bias, out, out_type, st);
  if (small_weight(v, kp, out_type == YP_F32 ? 4 : 2))
    return x_type == YP_INT8 ? small_weight_x<YP_T_I8>(rows, v, k, x, x_scale, wq, w_scale, bias, out, out_type, st)
         : x_type == YP_F32 ? small_weight_x<YP_T_F32>(rows, v, k, x, x_scale, wq, w_scale, bias, out, out_type, st)
         : x_type == YP_BF16 ? small_weight_x<YP_T_BF16>(rows, v, k, x, x_scale, wq, w_scale, bias, out, out_type, st)
                             : small_weight_x<YP_T_F16>(rows, v, k, x, x_scale, wq, w_scale, bias, out, out_type, st);
  if (x_type != YP_INT8) {
    float* const s = (float*)((char*)workspace + rows * kp);
    const hipError_t e = yp_launch_quantize_rows(rows, k, x_type, x, workspace, s, st);
    if (e != hipSuccess) return e;
    x = workspace;
    x_scale = s;
  }
  yp_gemm g = {};
  g.lda = g.ldb = kp;
  g.a = (const char*)wq; g.b = (const char*)x;
  g.I = v; g.J = rows; g.steps = (int)(kp / YP_TILE_KB);
  return out_type == YP_F32 ? linear_t<YP_T_F32>(g, x_scale, w_scale, bias, out, st)
       : out_type == YP_BF16 ? linear_t<YP_T_BF16>(g, x_scale, w_scale, bias, out, st) : linear_t<YP_T_F16>(g, x_scale, w_scale, bias, out, st);
}
