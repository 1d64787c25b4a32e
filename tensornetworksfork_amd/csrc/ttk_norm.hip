// ttk_norm.hip -- gfx950 kernels between raw rows and a model's inputs: layer norm (forward, backward with the
// column sums of the weight's and bias' gradient) and dropout from a counter-based generator.
//
// Element types: float64, float32, bfloat16, float16 in memory; statistics, products and sums are float32 (float64 for
// float64 rows), and one rounding to the element type ends each output.
//
// Dropout.  Element number e = offset + index is kept iff word e mod 4 of Philox4x32-10 (J. Salmon, M. Moraes, R. Dror,
// D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with key = seed and counter = (e div 4, 0, 0) is at
// least T = min(round(p 2^32), 2^32 - 1); kept elements are divided by 1 - p.  The mask is a function of (seed, e): it is
// recomputed wherever it is needed and never stored, and a shard that passes the element number of its first row as
// offset draws the mask of the whole set.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ttk.h"

namespace {

template <typename X>
struct Acc {
  typedef float type;
};
template <>
struct Acc<double> {
  typedef double type;
};

// 16 bytes of elements as one unaligned global access: rows of odd length start anywhere.
typedef uint32_t raw_t __attribute__((ext_vector_type(4), aligned(2)));

template <typename X>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(X);
  union {
    uint32_t u[4];
    X e[N];
  };
  __device__ __forceinline__ void load(const X* p) {
    raw_t r = *reinterpret_cast<const raw_t*>(p);
    u[0] = r.x, u[1] = r.y, u[2] = r.z, u[3] = r.w;
  }
  __device__ __forceinline__ void store(X* p) const {
    raw_t r;
    r.x = u[0], r.y = u[1], r.z = u[2], r.w = u[3];
    *reinterpret_cast<raw_t*>(p) = r;
  }
  // the first n (< N) elements one by one, the rest zero
  __device__ __forceinline__ void load_some(const X* p, int n) {
    u[0] = u[1] = u[2] = u[3] = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) e[j] = p[j];
  }
  __device__ __forceinline__ void store_some(X* p, int n) const {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p[j] = e[j];
  }
};

// ---------------------------------------------------------------------------------------
// Counter-based mask
// ---------------------------------------------------------------------------------------
struct Drop {
  uint32_t k0, k1, threshold;
  int mode;                 // 0: keep everything, 1: mask, 2: drop everything (p = 1)
  int64_t offset;
  const int64_t* offset_dev;  // added when not null
  double scale;             // 1 / (1 - p)
};

__device__ __forceinline__ uint64_t drop_base(const Drop& d) {
  return (uint64_t)d.offset + (d.offset_dev ? (uint64_t)*d.offset_dev : 0ull);
}

// bit i = element 4 block + i is kept
__device__ __forceinline__ uint32_t philox_keep4(const Drop& d, uint64_t block) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = 0, c3 = 0, k0 = d.k0, k1 = d.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t t = d.threshold;
  return (uint32_t)(c0 >= t) | ((uint32_t)(c1 >= t) << 1) | ((uint32_t)(c2 >= t) << 2) | ((uint32_t)(c3 >= t) << 3);
}

// bits of the N elements e, e + 1, ...
template <int N>
__device__ __forceinline__ uint32_t keep_bits(const Drop& d, uint64_t e) {
  if (d.mode == 0) return ~0u;
  if (d.mode == 2) return 0u;
  const uint64_t b = e >> 2;
  const int s = (int)(e & 3);
  uint32_t bits = philox_keep4(d, b);
#pragma unroll
  for (int i = 1; i < (N + 3) / 4; ++i) bits |= philox_keep4(d, b + i) << (4 * i);
  if (s + N > 4 * ((N + 3) / 4)) bits |= philox_keep4(d, b + (N + 3) / 4) << (4 * ((N + 3) / 4));
  return bits >> s;
}

// ---------------------------------------------------------------------------------------
// Sums
// ---------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_mov(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp_mov(double v) {
  const int64_t b = __double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xf, 0xf, true);
  return __longlong_as_double((int64_t)(((uint64_t)hi << 32) | lo));
}

// Sum over groups of LANES (16 or 64) consecutive lanes, the same bits in every lane.
template <int LANES, typename A>
__device__ __forceinline__ A lane_sum(A v) {
  v += dpp_mov<0xB1>(v);    // quad_perm 1 0 3 2
  v += dpp_mov<0x4E>(v);    // quad_perm 2 3 0 1
  v += dpp_mov<0x141>(v);   // mirror within 8
  v += dpp_mov<0x140>(v);   // mirror within 16
  if (LANES == 64) {
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
  }
  return v;
}

// Sum of two values over a workgroup of WAVES waves; `buf` holds 2 * WAVES values and may be written again after the
// next barrier that follows.
template <int WAVES, typename A>
__device__ __forceinline__ void block_sum2(A& a, A& b, A* buf) {
  a = lane_sum<64>(a);
  b = lane_sum<64>(b);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = a, buf[WAVES + (threadIdx.x >> 6)] = b;
  __syncthreads();
  a = b = A(0);
#pragma unroll
  for (int i = 0; i < WAVES; ++i) a += buf[i], b += buf[WAVES + i];
}

// ---------------------------------------------------------------------------------------
// Layer norm, any row length: one workgroup walks a row as often as it needs it.
// ---------------------------------------------------------------------------------------
constexpr int LONG_THREADS = 1024;

template <typename X, typename W>
__global__ __launch_bounds__(LONG_THREADS) void ln_fwd_long_kernel(const X* __restrict__ x, int64_t ldx, const W* __restrict__ w,
                                                                   const W* __restrict__ b, X* __restrict__ y,
                                                                   typename Acc<X>::type* __restrict__ mean_out,
                                                                   typename Acc<X>::type* __restrict__ rstd_out, int64_t rows,
                                                                   int cols, double eps, Drop drop) {
  typedef typename Acc<X>::type A;
  __shared__ A buf[2][2 * (LONG_THREADS / 64)];
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const X* xr = x + row * ldx;
    A s = 0, unused = 0;
    for (int c = threadIdx.x; c < cols; c += LONG_THREADS) s += (A)xr[c];
    block_sum2<LONG_THREADS / 64>(s, unused, buf[0]);
    const A mean = s / (A)cols;
    A q = 0;
    for (int c = threadIdx.x; c < cols; c += LONG_THREADS) {
      const A d = (A)xr[c] - mean;
      q += d * d;
    }
    unused = 0;
    block_sum2<LONG_THREADS / 64>(q, unused, buf[1]);
    const A rstd = A(1) / sqrt(q / (A)cols + (A)eps);
    for (int c = threadIdx.x; c < cols; c += LONG_THREADS) {
      A v = ((A)xr[c] - mean) * rstd;
      if (w) v *= (A)w[c];
      if (b) v += (A)b[c];
      if (drop.mode) v = (keep_bits<1>(drop, e0 + (uint64_t)row * cols + c) & 1) ? v * scale : A(0);
      y[row * cols + c] = (X)v;
    }
    if (threadIdx.x == 0) mean_out[row] = mean, rstd_out[row] = rstd;
  }
}

template <typename X, typename W>
__global__ __launch_bounds__(LONG_THREADS) void ln_bwd_long_kernel(const X* __restrict__ dy, int64_t lddy, const X* __restrict__ x,
                                                                   int64_t ldx, const W* __restrict__ w,
                                                                   const typename Acc<X>::type* __restrict__ mean_in,
                                                                   const typename Acc<X>::type* __restrict__ rstd_in,
                                                                   X* __restrict__ dx, int64_t rows, int cols, Drop drop) {
  typedef typename Acc<X>::type A;
  __shared__ A buf[2][2 * (LONG_THREADS / 64)];
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const X *xr = x + row * ldx, *dr = dy + row * lddy;
    const A mean = mean_in[row], rstd = rstd_in[row];
    A s1 = 0, s2 = 0;
    for (int c = threadIdx.x; c < cols; c += LONG_THREADS) {
      A g = (A)dr[c];
      if (drop.mode) g = (keep_bits<1>(drop, e0 + (uint64_t)row * cols + c) & 1) ? g * scale : A(0);
      const A a = w ? g * (A)w[c] : g;
      s1 += a;
      s2 += a * (((A)xr[c] - mean) * rstd);
    }
    block_sum2<LONG_THREADS / 64>(s1, s2, buf[turn]);
    s1 /= (A)cols;
    s2 /= (A)cols;
    for (int c = threadIdx.x; c < cols; c += LONG_THREADS) {
      A g = (A)dr[c];
      if (drop.mode) g = (keep_bits<1>(drop, e0 + (uint64_t)row * cols + c) & 1) ? g * scale : A(0);
      const A a = w ? g * (A)w[c] : g;
      const A h = ((A)xr[c] - mean) * rstd;
      dx[row * cols + c] = (X)(rstd * (a - s1 - h * s2));
    }
  }
}

// Partial column sums of a range of rows: part[split][0][c] = sum dy h, part[split][1][c] = sum dy.
template <typename X>
__global__ __launch_bounds__(256) void ln_cols_kernel(const X* __restrict__ dy, int64_t lddy, const X* __restrict__ x, int64_t ldx,
                                                      const typename Acc<X>::type* __restrict__ mean_in,
                                                      const typename Acc<X>::type* __restrict__ rstd_in,
                                                      typename Acc<X>::type* __restrict__ part, int64_t rows, int cols,
                                                      int64_t rows_per_split, Drop drop) {
  typedef typename Acc<X>::type A;
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per_split, r1 = min(rows, r0 + rows_per_split);
  double sw = 0, sb = 0;      // (a range may hold thousands of rows)
  for (int64_t row = r0; row < r1; ++row) {
    A g = (A)dy[row * lddy + c];
    if (drop.mode) g = (keep_bits<1>(drop, e0 + (uint64_t)row * cols + c) & 1) ? g * scale : A(0);
    sw += g * (((A)x[row * ldx + c] - mean_in[row]) * rstd_in[row]);
    sb += g;
  }
  A* p = part + (int64_t)blockIdx.y * 2 * cols;
  p[c] = (A)sw;
  p[cols + c] = (A)sb;
}

// Partials added in a fixed order, in 64 bits.
template <typename A, typename W>
__global__ __launch_bounds__(1024) void ln_cols_sum_kernel(const A* __restrict__ part, int nparts, int cols, W* __restrict__ dw,
                                                           W* __restrict__ db) {
  __shared__ double red[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), ty = threadIdx.x >> 6;
  W* out = blockIdx.y ? db : dw;
  const A* p = part + (int64_t)blockIdx.y * cols;
  double s = 0;
  if (c < cols)
    for (int g = ty; g < nparts; g += 16) s += (double)p[(int64_t)g * 2 * cols + c];
  red[ty][threadIdx.x & 63] = s;
  __syncthreads();
  if (ty == 0 && c < cols && out) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x & 63];
    out[c] = (W)s;
  }
}

// ---------------------------------------------------------------------------------------
// Dropout of a contiguous array
// ---------------------------------------------------------------------------------------
template <typename X>
__global__ __launch_bounds__(256) void dropout_kernel(const X* x, X* y, int64_t n, Drop drop) {
  typedef typename Acc<X>::type A;
  constexpr int N = Vec<X>::N;
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  const int64_t step = (int64_t)gridDim.x * 256 * N;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N; i < n; i += step) {
    Vec<X> v;
    const int m = (int)min((int64_t)N, n - i);
    if (m == N)
      v.load(x + i);
    else
      v.load_some(x + i, m);
    const uint32_t bits = keep_bits<N>(drop, e0 + (uint64_t)i);
#pragma unroll
    for (int j = 0; j < N; ++j) v.e[j] = (bits >> j & 1) ? (X)((A)v.e[j] * scale) : (X)A(0);
    if (m == N)
      v.store(y + i);
    else
      v.store_some(y + i, m);
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
inline int status() { return hipGetLastError() == hipSuccess ? TTK_OK : TTK_ELAUNCH; }

constexpr int CUS = 256;

bool make_drop(Drop& d, double p, uint64_t seed, int64_t offset, const int64_t* offset_dev) {
  if (!(p >= 0.0 && p <= 1.0) || offset < 0) return false;
  d.k0 = (uint32_t)seed;
  d.k1 = (uint32_t)(seed >> 32);
  const double t = p * 4294967296.0;
  d.threshold = t >= 4294967295.0 ? 0xFFFFFFFFu : (uint32_t)__builtin_rint(t);
  d.mode = p == 0.0 ? 0 : p == 1.0 ? 2 : 1;
  d.offset = offset;
  d.offset_dev = offset_dev;
  d.scale = p < 1.0 ? 1.0 / (1.0 - p) : 0.0;
  return true;
}

bool types_ok(int dtype, int wdtype) {
  return dtype == wdtype ? dtype >= 0 && dtype <= 3 : (dtype == 2 || dtype == 3) && wdtype == 1;
}

// how the column sums of a backward pass are split over the rows
struct ColsPlan {
  int splits;
  int64_t rows_per_split;
};
ColsPlan cols_plan(int64_t rows, int cols) {
  const int64_t tiles = (cols + 255) / 256;
  int64_t s = min((int64_t)1024, max((int64_t)1, 8 * CUS / tiles));
  s = min(s, (rows + 15) / 16);
  ColsPlan p;
  p.rows_per_split = (rows + s - 1) / s;
  p.splits = (int)((rows + p.rows_per_split - 1) / p.rows_per_split);
  return p;
}

template <typename X, typename W>
int ln_fwd(const void* x, int64_t ldx, const void* w, const void* b, void* y, void* mean, void* rstd, int64_t rows, int cols,
           double eps, const Drop& d, hipStream_t st) {
  typedef typename Acc<X>::type A;
  hipLaunchKernelGGL((ln_fwd_long_kernel<X, W>), dim3((unsigned)min(rows, (int64_t)(4 * CUS))), dim3(LONG_THREADS), 0, st,
                     (const X*)x, ldx, (const W*)w, (const W*)b, (X*)y, (A*)mean, (A*)rstd, rows, cols, eps, d);
  return status();
}

template <typename X, typename W>
int ln_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const void* mean, const void* rstd, void* dx,
           void* dw, void* db, int64_t rows, int cols, const Drop& d, void* ws, int64_t ws_bytes, hipStream_t st) {
  typedef typename Acc<X>::type A;
  const ColsPlan cp = cols_plan(rows, cols);
  if ((dw || db) && (!ws || ws_bytes < (int64_t)cp.splits * 2 * cols * (int64_t)sizeof(A))) return TTK_EWORKSPACE;
  if (dx)
    hipLaunchKernelGGL((ln_bwd_long_kernel<X, W>), dim3((unsigned)min(rows, (int64_t)(4 * CUS))), dim3(LONG_THREADS), 0, st,
                       (const X*)dy, lddy, (const X*)x, ldx, (const W*)w, (const A*)mean, (const A*)rstd, (X*)dx, rows, cols, d);
  if (dw || db) {
    hipLaunchKernelGGL((ln_cols_kernel<X>), dim3((unsigned)((cols + 255) / 256), (unsigned)cp.splits), dim3(256), 0, st,
                       (const X*)dy, lddy, (const X*)x, ldx, (const A*)mean, (const A*)rstd, (A*)ws, rows, cols,
                       cp.rows_per_split, d);
    hipLaunchKernelGGL((ln_cols_sum_kernel<A, W>), dim3((unsigned)((cols + 63) / 64), 2), dim3(1024), 0, st, (const A*)ws,
                       cp.splits, cols, (W*)dw, (W*)db);
  }
  return status();
}

}  // namespace

// one call of F<X, W> for a pair of type codes (0 float64, 1 float32, 2 bfloat16, 3 float16)
#define TTK_BY_TYPES(F, ...)                                                              \
  switch (dtype * 4 + wdtype) {                                                           \
    case 0: return F<double, double>(__VA_ARGS__);                                        \
    case 5: return F<float, float>(__VA_ARGS__);                                          \
    case 9: return F<__bf16, float>(__VA_ARGS__);                                         \
    case 10: return F<__bf16, __bf16>(__VA_ARGS__);                                       \
    case 13: return F<_Float16, float>(__VA_ARGS__);                                      \
    case 15: return F<_Float16, _Float16>(__VA_ARGS__);                                   \
  }                                                                                       \
  return TTK_EINVAL

extern "C" {

int ttk_layer_norm(int dtype, int wdtype, const void* x, int64_t ldx, const void* w, const void* b, void* y, void* mean, void* rstd,
                   int64_t rows, int cols, double eps, double p, uint64_t seed, int64_t offset, const int64_t* offset_dev,
                   void* stream) {
  Drop d;
  if (!x || !y || !mean || !rstd || rows < 1 || cols < 1 || ldx < 0 || !(eps >= 0.0) || !types_ok(dtype, wdtype) ||
      !make_drop(d, p, seed, offset, offset_dev))
    return TTK_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  TTK_BY_TYPES(ln_fwd, x, ldx, w, b, y, mean, rstd, rows, cols, eps, d, st);
}

int64_t ttk_layer_norm_backward_ws_bytes(int dtype, int64_t rows, int cols) {
  if (dtype < 0 || dtype > 3 || rows < 1 || cols < 1) return TTK_EINVAL;
  return (int64_t)cols_plan(rows, cols).splits * 2 * cols * (dtype == 0 ? 8 : 4);
}

int ttk_layer_norm_backward(int dtype, int wdtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w,
                            const void* mean, const void* rstd, void* dx, void* dw, void* db, int64_t rows, int cols, double p,
                            uint64_t seed, int64_t offset, const int64_t* offset_dev, void* ws, int64_t ws_bytes, void* stream) {
  Drop d;
  if (!dy || !x || !mean || !rstd || rows < 1 || cols < 1 || lddy < 0 || ldx < 0 || !types_ok(dtype, wdtype) ||
      !make_drop(d, p, seed, offset, offset_dev))
    return TTK_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  TTK_BY_TYPES(ln_bwd, dy, lddy, x, ldx, w, mean, rstd, dx, dw, db, rows, cols, d, ws, ws_bytes, st);
}

int ttk_dropout(int dtype, const void* x, void* y, int64_t n, double p, uint64_t seed, int64_t offset, const int64_t* offset_dev,
                void* stream) {
  Drop d;
  if (!x || !y || n < 1 || dtype < 0 || dtype > 3 || !make_drop(d, p, seed, offset, offset_dev)) return TTK_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  const int per = 256 * (dtype == 0 ? 2 : dtype == 1 ? 4 : 8);
  const dim3 grid((unsigned)min((n + per - 1) / per, (int64_t)(16 * CUS)));
  switch (dtype) {
    case 0: hipLaunchKernelGGL((dropout_kernel<double>), grid, dim3(256), 0, st, (const double*)x, (double*)y, n, d); break;
    case 1: hipLaunchKernelGGL((dropout_kernel<float>), grid, dim3(256), 0, st, (const float*)x, (float*)y, n, d); break;
    case 2: hipLaunchKernelGGL((dropout_kernel<__bf16>), grid, dim3(256), 0, st, (const __bf16*)x, (__bf16*)y, n, d); break;
    case 3: hipLaunchKernelGGL((dropout_kernel<_Float16>), grid, dim3(256), 0, st, (const _Float16*)x, (_Float16*)y, n, d); break;
  }
  return status();
}

}  // extern "C"
