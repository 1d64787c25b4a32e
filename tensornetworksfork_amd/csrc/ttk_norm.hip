// ttk_norm.hip -- gfx950 kernels between raw rows and a model's inputs: layer norm (forward, backward with the
// column sums of the weight's and bias' gradient) and dropout from a counter-based generator.
//
// Element types: float64, float32, bfloat16, float16 in memory; statistics, products and sums are float32 (float64 for
// float64 rows, and in the sums of rows that the registers do not hold), and one rounding to the element type ends each output.
//
// Dropout.  Element number e = offset + index is kept iff word e mod 4 of Philox4x32-10 (J. Salmon, M. Moraes, R. Dror,
// D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with key = seed and counter = (e div 4, 0, 0) is at
// least T = min(round(p 2^32), 2^32 - 1); kept elements are divided by 1 - p.  The mask is a function of (seed, e): it is
// recomputed wherever it is needed and never stored, and a shard that passes the element number of its first row as
// offset draws the mask of the whole set.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

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
typedef uint32_t half_t __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t word_t __attribute__((aligned(2)));

// Held as four words (elements of their own would take a register each).
template <typename X>
struct Vec {
  typedef typename Acc<X>::type A;
  static constexpr int N = 16 / (int)sizeof(X);
  uint32_t u[4];
  __device__ __forceinline__ void load(const X* p) {
    const raw_t r = *reinterpret_cast<const raw_t*>(p);
    u[0] = r.x, u[1] = r.y, u[2] = r.z, u[3] = r.w;
  }
  __device__ __forceinline__ void store(X* p) const {
    raw_t r;
    r.x = u[0], r.y = u[1], r.z = u[2], r.w = u[3];
    *reinterpret_cast<raw_t*>(p) = r;
  }
  __device__ __forceinline__ void clear() { u[0] = u[1] = u[2] = u[3] = 0; }
  // the first n (< N) elements one by one, the rest zero
  __device__ __forceinline__ void load_some(const X* p, int n) {
    clear();
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) put(j, p[j]);
  }
  // the first n (0 < n < N) elements, in pieces of 8, 4 and 2 bytes
  __device__ __forceinline__ void store_some(X* p, int n) const {
    uint32_t a = u[0], b = u[1];
    const int bytes = n * (int)sizeof(X);
    char* q = reinterpret_cast<char*>(p);
    if (bytes & 8) {
      half_t r;
      r.x = a, r.y = b;
      *reinterpret_cast<half_t*>(q) = r;
      q += 8, a = u[2], b = u[3];
    }
    if (sizeof(X) <= 4 && bytes & 4) {
      *reinterpret_cast<word_t*>(q) = a;
      q += 4, a = b;
    }
    if (sizeof(X) == 2 && bytes & 2) *reinterpret_cast<uint16_t*>(q) = (uint16_t)a;
  }
  // drops the first k (< N) elements: the others move down, zeros behind them
  __device__ __forceinline__ void drop_first(int k) {
    const int bytes = k * (int)sizeof(X);
    if (sizeof(X) == 2 && bytes & 2) {
      u[0] = u[0] >> 16 | u[1] << 16;
      u[1] = u[1] >> 16 | u[2] << 16;
      u[2] = u[2] >> 16 | u[3] << 16;
      u[3] >>= 16;
    }
    if (sizeof(X) <= 4 && bytes & 4) u[0] = u[1], u[1] = u[2], u[2] = u[3], u[3] = 0;
    if (bytes & 8) u[0] = u[2], u[1] = u[3], u[2] = u[3] = 0;
  }
  // Forgets what was computed from the elements: without it the compiler keeps every element's float beside the element
  // across the phases of a row, which are twice to three times the registers.
  __device__ __forceinline__ void forget() { asm volatile("" : "+v"(u[0]), "+v"(u[1]), "+v"(u[2]), "+v"(u[3])); }

  __device__ __forceinline__ X element(int j) const {
    if constexpr (sizeof(X) == 2)
      return __builtin_bit_cast(X, (uint16_t)(u[j / 2] >> (16 * (j % 2))));
    else if constexpr (sizeof(X) == 4)
      return __builtin_bit_cast(X, u[j]);
    else
      return __builtin_bit_cast(X, (uint64_t)u[2 * j + 1] << 32 | u[2 * j]);
  }
  __device__ __forceinline__ void put(int j, X e) {      // into a zero
    if constexpr (sizeof(X) == 2) {
      u[j / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, e) << (16 * (j % 2));
    } else if constexpr (sizeof(X) == 4) {
      u[j] = __builtin_bit_cast(uint32_t, e);
    } else {
      const uint64_t b = __builtin_bit_cast(uint64_t, e);
      u[2 * j] = (uint32_t)b, u[2 * j + 1] = (uint32_t)(b >> 32);
    }
  }
  __device__ __forceinline__ A get(int j) const {
    if constexpr (__is_same(X, __bf16))
      return __builtin_bit_cast(float, j % 2 ? u[j / 2] & 0xFFFF0000u : u[j / 2] << 16);
    else
      return (A)element(j);
  }
  __device__ __forceinline__ void set(const A (&h)[N]) {      // rounded to the element type
    u[0] = u[1] = u[2] = u[3] = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) put(j, (X)h[j]);
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

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);      // (the compiler keeps two xors by itself)
}

__device__ __forceinline__ void philox(const Drop& d, uint64_t block, uint32_t (&out)[4]) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = 0, c3 = 0, k0 = d.k0, k1 = d.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(p1 >> 32), c1, k0);
    c1 = (uint32_t)p1;
    c2 = xor3((uint32_t)(p0 >> 32), c3, k1);
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0, out[1] = c1, out[2] = c2, out[3] = c3;
}

// bit i = element 4 block + i is kept
__device__ __forceinline__ uint32_t philox_keep4(const Drop& d, uint64_t block) {
  uint32_t w[4];
  philox(d, block, w);
  const uint32_t t = d.threshold;
  return (uint32_t)(w[0] >= t) | ((uint32_t)(w[1] >= t) << 1) | ((uint32_t)(w[2] >= t) << 2) | ((uint32_t)(w[3] >= t) << 3);
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

// Bits of the N elements from e on where the next lane has those from e + N on (N a multiple of 4, e mod 4 the same in the
// wave): a block that reaches into the next lane's elements comes from there, and behind the wave's last lane from the scalar
// unit.
template <int N>
__device__ __forceinline__ uint32_t keep_bits_wave(const Drop& d, uint64_t e) {
  if (d.mode == 0) return ~0u;
  if (d.mode == 2) return 0u;
  constexpr int NB = N / 4;
  const uint64_t b = e >> 2;
  uint32_t bits = philox_keep4(d, b);
#pragma unroll
  for (int i = 1; i < NB; ++i) bits |= philox_keep4(d, b + i) << (4 * i);
  const int s = __builtin_amdgcn_readfirstlane((int)(e & 3));
  if (s) {
    const uint64_t b0 = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 |
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    const uint64_t end = b0 + 64 * NB;      // (the first lane is lane 0)
    uint32_t c0 = (uint32_t)end, c1 = (uint32_t)(end >> 32), c2 = 0, c3 = 0, k0 = d.k0, k1 = d.k1;
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
    const uint32_t last = (uint32_t)(c0 >= t) | ((uint32_t)(c1 >= t) << 1) | ((uint32_t)(c2 >= t) << 2) | ((uint32_t)(c3 >= t) << 3);
    const uint32_t next = (uint32_t)__builtin_amdgcn_update_dpp((int)last, (int)bits, 0x130, 0xf, 0xf, false);      // lane + 1
    bits |= (next & 0xF) << N;
  }
  return bits >> s;
}

// Bits of a lane's N elements of a row that LANES lanes share.
template <int N, int LANES>
__device__ __forceinline__ uint32_t keep_bits_row(const Drop& d, uint64_t e) {
  if constexpr (LANES >= 64 && N % 4 == 0)
    return keep_bits_wave<N>(d, e);
  else
    return keep_bits<N>(d, e);
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

// Sum over groups of LANES (8 to 64) consecutive lanes, the same bits in every lane.
template <int LANES, typename A>
__device__ __forceinline__ A lane_sum(A v) {
  v += dpp_mov<0xB1>(v);    // quad_perm 1 0 3 2
  v += dpp_mov<0x4E>(v);    // quad_perm 2 3 0 1
  v += dpp_mov<0x141>(v);   // mirror within 8
  if (LANES >= 16) v += dpp_mov<0x140>(v);   // mirror within 16
  if (LANES >= 32) v += __shfl_xor(v, 16);
  if (LANES >= 64) v += __shfl_xor(v, 32);
  return v;
}

// Sums over a workgroup of WAVES (at most 16) waves, the same bits in every lane; `buf` holds 16 values a sum and may be
// written again after the next barrier that follows.
template <int WAVES, typename A>
__device__ __forceinline__ A block_sum(A a, A* buf) {
  const int lane = threadIdx.x & 63;
  a = lane_sum<64>(a);
  if (lane == 0) buf[threadIdx.x >> 6] = a;
  __syncthreads();
  return lane_sum<16>((lane & 15) < WAVES ? buf[lane & 15] : A(0));
}
template <int WAVES, typename A>
__device__ __forceinline__ void block_sum2(A& a, A& b, A* buf) {
  const int lane = threadIdx.x & 63;
  a = lane_sum<64>(a);
  b = lane_sum<64>(b);
  if (lane == 0) buf[threadIdx.x >> 6] = a, buf[16 + (threadIdx.x >> 6)] = b;
  __syncthreads();
  const bool is = (lane & 15) < WAVES;
  a = lane_sum<16>(is ? buf[lane & 15] : A(0));
  b = lane_sum<16>(is ? buf[16 + (lane & 15)] : A(0));
}

// ---------------------------------------------------------------------------------------
// Layer norm, any row length: one workgroup walks a row as often as it needs it (forward: sum, centred squares, output;
// backward: the two sums, dx; the column sums in a pass of their own).  Rows longer than the registers of a workgroup hold
// (16384 elements; float64 8192).  Bound by one element a lane and load and by the second and third pass, which L2 serves:
// 4096 rows of 30000 float32 columns 398 us forward (2.5 TB/s of traffic counted once), 417 us for dx (3.5) and 199 us for the
// column sums; bfloat16 328, 448 and 242 us.  Few rows of millions of columns leave most of the machine idle (22 rows of 3 million
// float32: 3.7 ms forward, 3.3 ms for dx, 0.1 and 0.2 TB/s).  Sums over a row are float64 whatever its type (a lane adds cols / 1024
// terms one after the other; 3 % of the forward pass).  Rows may have up to 2^31 - 1 columns, which are counted in 64 bits.
// ---------------------------------------------------------------------------------------
constexpr int LONG_THREADS = 1024;

template <typename X, typename W>
__global__ __launch_bounds__(LONG_THREADS) void ln_fwd_long_kernel(const X* __restrict__ x, int64_t ldx, const W* __restrict__ w,
                                                                   const W* __restrict__ b, X* __restrict__ y,
                                                                   typename Acc<X>::type* __restrict__ mean_out,
                                                                   typename Acc<X>::type* __restrict__ rstd_out, int64_t rows,
                                                                   int cols, double eps, Drop drop) {
  typedef typename Acc<X>::type A;
  __shared__ double buf[2][32];
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const X* xr = x + row * ldx;
    double s = 0;      // (a lane adds cols / 1024 terms one after the other)
    for (int64_t c = threadIdx.x; c < cols; c += LONG_THREADS) s += (A)xr[c];
    const A mean = (A)(block_sum<LONG_THREADS / 64>(s, buf[0]) / (double)cols);
    double q = 0;
    for (int64_t c = threadIdx.x; c < cols; c += LONG_THREADS) {
      const A d = (A)xr[c] - mean;
      q += d * d;
    }
    const A rstd = A(1) / sqrt((A)(block_sum<LONG_THREADS / 64>(q, buf[1]) / (double)cols) + (A)eps);
    for (int64_t c = threadIdx.x; c < cols; c += LONG_THREADS) {
      A v = ((A)xr[c] - mean) * rstd;
      if (w) v *= (A)w[c];
      if (b) v += (A)b[c];
      if (drop.mode) v = (keep_bits<1>(drop, e0 + (uint64_t)row * cols + c) & 1) ? v * scale : A(0);
      y[row * cols + c] = (X)v;
    }
    if (threadIdx.x == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
  }
}

template <typename X, typename W>
__global__ __launch_bounds__(LONG_THREADS) void ln_bwd_long_kernel(const X* __restrict__ dy, int64_t lddy, const X* __restrict__ x,
                                                                   int64_t ldx, const W* __restrict__ w,
                                                                   const typename Acc<X>::type* __restrict__ mean_in,
                                                                   const typename Acc<X>::type* __restrict__ rstd_in,
                                                                   X* __restrict__ dx, int64_t rows, int cols, Drop drop) {
  typedef typename Acc<X>::type A;
  __shared__ double buf[2][32];
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const X *xr = x + row * ldx, *dr = dy + row * lddy;
    const A mean = mean_in[row], rstd = rstd_in[row];
    double sum1 = 0, sum2 = 0;
    for (int64_t c = threadIdx.x; c < cols; c += LONG_THREADS) {
      A g = (A)dr[c];
      if (drop.mode) g = (keep_bits<1>(drop, e0 + (uint64_t)row * cols + c) & 1) ? g * scale : A(0);
      const A a = w ? g * (A)w[c] : g;
      sum1 += a;
      sum2 += a * (((A)xr[c] - mean) * rstd);
    }
    block_sum2<LONG_THREADS / 64>(sum1, sum2, buf[turn]);
    const A s1 = (A)(sum1 / (double)cols), s2 = (A)(sum2 / (double)cols);
    for (int64_t c = threadIdx.x; c < cols; c += LONG_THREADS) {
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
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
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

// Partials added in a fixed order, in 64 bits.  The launch has SUM_GROUPS workgroups at most, each walks its share of the columns
// (a launch counts its threads in 32 bits; one of more runs a part of its workgroups without an error).
constexpr int SUM_GROUPS = 1 << 16;
template <typename A, typename W>
__global__ __launch_bounds__(1024) void ln_cols_sum_kernel(const A* __restrict__ part, int nparts, int cols, W* __restrict__ dw,
                                                           W* __restrict__ db) {
  __shared__ double red[16][64];
  const int ty = threadIdx.x >> 6;
  W* out = blockIdx.y ? db : dw;
  const A* p = part + (int64_t)blockIdx.y * cols;
  for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < cols; c0 += (int64_t)gridDim.x * 64) {
    const int64_t c = c0 + (threadIdx.x & 63);
    double s = 0;
    if (c < cols) {
      int g = ty;
      for (; g + 7 * 16 < nparts; g += 8 * 16) {      // eight loads under way
        A v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = p[(int64_t)(g + 16 * k) * 2 * cols + c];
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)v[k];
      }
      for (; g < nparts; g += 16) s += (double)p[(int64_t)g * 2 * cols + c];
    }
    red[ty][threadIdx.x & 63] = s;
    __syncthreads();
    if (ty == 0 && c < cols && out) {
#pragma unroll
      for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x & 63];
      out[c] = (W)s;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// Layer norm, rows held in registers: LANES lanes own a row, NV vectors of 16 bytes each (vector v of lane l starts at
// column (v LANES + l) N).  One pass over memory: both statistics come from the registers, the variance from the centred
// values.  LANES 8 to 64: several rows a workgroup, no barrier; 256 and more: a workgroup a row.  The next row's loads are
// under way while a row is worked on.
//
// The backward pass walks many rows a workgroup and keeps each lane's columns of dw and db in registers; they leave as one
// partial row per workgroup (`part`: [workgroup][dw | db][cols]), so the rows are read once and no atomic orders the sums.  In
// the registers they are the rows' arithmetic type, float32 for 16- and 32-bit rows: float64 would take twice the registers of
// kernels that registers bound.  A lane adds 480 rows at most before its partial is added in float64 (see row_groups).
//
// Bound by HBM (a copy reaches 5.1 to 5.4 TB/s) up to the mask of 16-bit rows, whose counter blocks cost as much as their
// bytes.  Measured: float32 54000 x 784 with dropout, forward 60 us (339 MB, 5.7 TB/s with the 256 MB cache's help), backward
// 110 us (508 MB, 4.6 TB/s); bfloat16 16384 x 8192 backward 155 us (805 MB, 5.2 TB/s); float16 1021 x 10007 with dropout 29 and
// 54 us (4 rows a workgroup: latency of a row's barriers, up to 6 counter blocks a lane and row, and backward 54 spilled registers).
// ---------------------------------------------------------------------------------------
// RAGGED: the row's length is no multiple of a vector's.  The vector that reaches behind the row is then loaded from where it
// ends with the row (no load an element, no wait before the values are used) and put right by settle_row.
template <bool RAGGED, typename X, int LANES, int NV>
__device__ __forceinline__ void load_row(Vec<X> (&v)[NV], const X* p, int lane, int cols, bool live) {
  constexpr int N = Vec<X>::N;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * N;
    if (RAGGED && cols < N) {
      v[i].load_some(p + c, live ? cols - c : 0);
    } else {
      v[i].clear();
      if (live && c < cols) v[i].load(p + (RAGGED ? min(c, cols - N) : c));
    }
  }
}
template <bool RAGGED, typename X, int LANES, int NV>
__device__ __forceinline__ void settle_row(Vec<X> (&v)[NV], int lane, int cols) {
  constexpr int N = Vec<X>::N;
  if (!RAGGED || cols < N) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * N;
    if (c < cols && c + N > cols) v[i].drop_first(c + N - cols);
  }
}

template <bool RAGGED, typename X, int LANES, int NV>
__device__ __forceinline__ void store_row(const Vec<X> (&v)[NV], X* p, int lane, int cols) {
  constexpr int N = Vec<X>::N;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * N;
    if (RAGGED ? c + N <= cols : c < cols)
      v[i].store(p + c);
    else if (RAGGED && c < cols)
      v[i].store_some(p + c, cols - c);
  }
}

// N weights from column c on (missing ones 0)
template <bool RAGGED, typename A, typename W, int N>
__device__ __forceinline__ void load_weights(A (&out)[N], const W* w, int c, int cols) {
  constexpr int M = Vec<W>::N;
  if (N >= M && c < cols && (!RAGGED || cols >= N)) {
    const int at = RAGGED ? min(c, cols - N) : c, k = c - at;
#pragma unroll
    for (int t = 0; t < N / M; ++t) {
      Vec<W> v;
      v.load(w + at + t * M);
#pragma unroll
      for (int j = 0; j < M; ++j) out[t * M + j] = (A)v.get(j);
    }
    if (RAGGED && k) {      // the row's last, incomplete vector
#pragma unroll
      for (int b = 1; b < N; b *= 2)
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = k & b ? (j + b < N ? out[j + b] : A(0)) : out[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = c + j < cols ? (A)w[c + j] : A(0);
  }
}

// sums over the LANES lanes of a row, in every lane
template <int LANES, typename A>
__device__ __forceinline__ void row_sum2(A& a, A& b, A* buf) {
  if constexpr (LANES <= 64) {
    a = lane_sum<LANES>(a);
    b = lane_sum<LANES>(b);
  } else {
    block_sum2<LANES / 64>(a, b, buf);
  }
}
template <int LANES, typename A>
__device__ __forceinline__ A row_sum(A a, A* buf) {
  if constexpr (LANES <= 64)
    return lane_sum<LANES>(a);
  else
    return block_sum<LANES / 64>(a, buf);
}

constexpr int group_threads(int lanes) { return lanes < 256 ? 256 : lanes; }

// The same value, of which the compiler knows nothing: what is computed or loaded from it in a loop stays there instead of
// taking a register for the whole kernel.
template <typename T>
__device__ __forceinline__ T in_loop(T v) {
  asm volatile("" : "+v"(v));
  return v;
}
template <typename T>
__device__ __forceinline__ const T* in_loop_uniform(const T* p) {
  asm volatile("" : "+s"(p));
  return p;
}

// Keeps the instructions of a lane's vectors apart where there are many: interleaved they need every vector's temporaries at
// once.
template <int NV>
__device__ __forceinline__ void one_by_one() {
  if constexpr (NV > 2) __builtin_amdgcn_sched_barrier(0);
}

// weights of a lane's columns; absent ones act as `none`
template <bool RAGGED, typename A, typename W, int N>
__device__ __forceinline__ void load_weights_or(A (&out)[N], const W* w, int c, int cols, A none) {
  if (w) {
    load_weights<RAGGED, A, W, N>(out, w, c, cols);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) out[j] = none;
  }
}
template <bool RAGGED, typename A, typename W, int LANES, int NV, int N>
__device__ __forceinline__ void lane_weights(A (&out)[NV][N], const W* w, int lane, int cols, A none) {
#pragma unroll
  for (int i = 0; i < NV; ++i) load_weights_or<RAGGED, A, W, N>(out[i], w, (i * LANES + lane) * N, cols, none);
}

template <typename X, typename W, int LANES, int NV, bool RAGGED>
__global__ __launch_bounds__(group_threads(LANES), NV <= 2 || LANES >= 512 ? 4 : 3) void ln_fwd_group_kernel(
    const X* __restrict__ x, int64_t ldx, const W* __restrict__ w, const W* __restrict__ b, X* __restrict__ y,
    typename Acc<X>::type* __restrict__ mean_out, typename Acc<X>::type* __restrict__ rstd_out, int64_t rows, int cols, double eps,
    Drop drop) {
  typedef typename Acc<X>::type A;
  constexpr int N = Vec<X>::N, RPB = group_threads(LANES) / LANES;
  constexpr bool HOLD = NV * N <= 16, WIDE = NV * N > 16;      // weights stay in registers; many elements a lane
  __shared__ A buf[2][LANES > 64 ? 16 : 1];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  A wv[NV][N], bv[NV][N];
  if constexpr (HOLD) {
    lane_weights<RAGGED, A, W, LANES, NV, N>(wv, w, lane, cols, A(1));
    lane_weights<RAGGED, A, W, LANES, NV, N>(bv, b, lane, cols, A(0));
  }
  const int64_t step = (int64_t)gridDim.x * RPB;
  Vec<X> next[NV];
  load_row<RAGGED, X, LANES, NV>(next, x + ((int64_t)blockIdx.x * RPB + sub) * ldx, lane, cols, (int64_t)blockIdx.x * RPB + sub < rows);
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += step) {
    const int64_t row = r0 + sub;
    const bool live = row < rows;
    Vec<X> v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = next[i];
    settle_row<RAGGED, X, LANES, NV>(v, lane, cols);
    if (r0 + step < rows) load_row<RAGGED, X, LANES, NV>(next, x + (row + step) * ldx, lane, cols, row + step < rows);
    A s = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) s += v[i].get(j);
    const A mean = row_sum<LANES>(s, buf[0]) / (A)cols;      // (times 1 / cols the mean of a constant row misses it)
    if constexpr (WIDE)
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i].forget();
    A q = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const A d = (i * LANES + lane) * N + j < cols ? v[i].get(j) - mean : A(0);
        q += d * d;
      }
    const A rstd = A(1) / sqrt(row_sum<LANES>(q, buf[1]) / (A)cols + (A)eps);
    if (!live) continue;
    if constexpr (WIDE)
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i].forget();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (!HOLD) {
        load_weights_or<RAGGED, A, W, N>(wv[i], in_loop_uniform(w), (i * LANES + lane) * N, cols, A(1));
        load_weights_or<RAGGED, A, W, N>(bv[i], in_loop_uniform(b), (i * LANES + lane) * N, cols, A(0));
      }
      A h[N];
#pragma unroll
      for (int j = 0; j < N; ++j) h[j] = (v[i].get(j) - mean) * rstd * wv[i][j] + bv[i][j];
      if (drop.mode) {
        const uint32_t bits = keep_bits_row<N, LANES>(drop, e0 + (uint64_t)row * cols + (i * LANES + lane) * N);
#pragma unroll
        for (int j = 0; j < N; ++j) h[j] = (bits >> j & 1) ? h[j] * scale : A(0);
      }
      v[i].set(h);
      one_by_one<NV>();
    }
    store_row<RAGGED, X, LANES, NV>(v, y + row * cols, lane, cols);
    if (lane == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
  }
}

template <typename X, typename W, int LANES, int NV, bool RAGGED>
__global__ __launch_bounds__(group_threads(LANES)) void ln_bwd_group_kernel(
    const X* __restrict__ dy, int64_t lddy, const X* __restrict__ x, int64_t ldx, const W* __restrict__ w,
    const typename Acc<X>::type* __restrict__ mean_in, const typename Acc<X>::type* __restrict__ rstd_in, X* __restrict__ dx,
    typename Acc<X>::type* __restrict__ part, int64_t rows, int cols, Drop drop) {
  typedef typename Acc<X>::type A;
  constexpr int N = Vec<X>::N, RPB = group_threads(LANES) / LANES;
  // a row's a and h stay in registers between its two halves; the next row's loads are under way meanwhile
  constexpr bool HOLD = NV * N * (int)sizeof(A) <= 32, AHEAD = NV * N * (int)sizeof(A) + NV * 32 <= (LANES >= 1024 ? 128 : 256);
  __shared__ A buf[2][LANES > 64 ? 32 : 1];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  A aw[NV][N], ab[NV][N], wv[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) aw[i][j] = ab[i][j] = A(0);
  if constexpr (AHEAD) lane_weights<RAGGED, A, W, LANES, NV, N>(wv, w, lane, cols, A(1));
  const int64_t step = (int64_t)gridDim.x * RPB;
  Vec<X> nx[NV], ng[NV];
  A nmean = 0, nrstd = 0;
  auto fetch = [&](int64_t row) {
    const bool live = row < rows;
    load_row<RAGGED, X, LANES, NV>(nx, x + row * ldx, lane, cols, live);
    load_row<RAGGED, X, LANES, NV>(ng, dy + row * lddy, lane, cols, live);
    nmean = live ? mean_in[row] : A(0);
    nrstd = live ? rstd_in[row] : A(0);
  };
  if (AHEAD) fetch((int64_t)blockIdx.x * RPB + sub);
  int turn = 0;
#pragma unroll 1
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += step, turn ^= 1) {
    const int64_t row = r0 + sub;
    const bool live = row < rows;
    Vec<X> xv[NV], gv[NV];
    if (!AHEAD) fetch(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) xv[i] = nx[i], gv[i] = ng[i];
    settle_row<RAGGED, X, LANES, NV>(xv, lane, cols);
    settle_row<RAGGED, X, LANES, NV>(gv, lane, cols);
    const A mean = nmean, rstd = nrstd;
    if (AHEAD && r0 + step < rows) fetch(row + step);
    A s1 = 0, s2 = 0, ha[HOLD ? NV : 1][N], aa[HOLD ? NV : 1][N];
    uint32_t bits[NV];
    // Columns behind the row have dy = 0 and add nothing.  Their h is 0 as well: (0 - mean) rstd may lie beyond the type's range,
    // and 0 times that is no number.
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LANES + lane) * N;
      const A mid = c < cols ? mean : A(0);
      if constexpr (!AHEAD) load_weights_or<RAGGED, A, W, N>(wv[i], in_loop_uniform(w), c, cols, A(1));
      if (drop.mode) bits[i] = live ? keep_bits_row<N, NV == 1 ? LANES : 1>(drop, e0 + (uint64_t)row * cols + c) : 0u;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        A g = gv[i].get(j);
        if (drop.mode) g = (bits[i] >> j & 1) ? g * scale : A(0);
        const A d = xv[i].get(j) - mid, h = (RAGGED && c + j >= cols ? A(0) : d) * rstd, a = g * wv[i][j];
        s1 += a;
        s2 += a * h;
        aw[i][j] += g * h;
        ab[i][j] += g;
        if constexpr (HOLD) ha[i][j] = h, aa[i][j] = a;
      }
      one_by_one<NV>();
    }
    if (!dx) continue;
    row_sum2<LANES>(s1, s2, buf[turn]);
    s1 /= (A)cols;
    s2 /= (A)cols;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (!HOLD) xv[i].forget(), gv[i].forget();
      if constexpr (!AHEAD) load_weights_or<RAGGED, A, W, N>(wv[i], in_loop_uniform(w), (i * LANES + lane) * N, cols, A(1));
      A out[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        A h, a;
        if constexpr (HOLD) {
          h = ha[i][j], a = aa[i][j];
        } else {
          A g = gv[i].get(j);
          if (drop.mode) g = (bits[i] >> j & 1) ? g * scale : A(0);
          h = (xv[i].get(j) - mean) * rstd;
          a = g * wv[i][j];
        }
        out[j] = rstd * (a - s1 - h * s2);
      }
      gv[i].set(out);
      one_by_one<NV>();
    }
    store_row<RAGGED, X, LANES, NV>(gv, dx + row * cols, lane, cols);
  }
  if (!part) return;
  A* p = part + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = (i * LANES + lane) * N + j;
        if (c < cols) p[c] = aw[i][j], p[cols + c] = ab[i][j];
      }
  } else {      // the workgroup's row groups, one after the other
    __shared__ A col[2][LANES * NV * N];
    for (int g = 0; g < RPB; ++g) {
      if (sub == g)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const int c = (i * LANES + lane) * N + j;
            col[0][c] = g ? col[0][c] + aw[i][j] : aw[i][j];
            col[1][c] = g ? col[1][c] + ab[i][j] : ab[i][j];
          }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += 256) p[c] = col[0][c], p[cols + c] = col[1][c];
  }
}

// ---------------------------------------------------------------------------------------
// Layer norm of short dense rows: a wave takes 64 rows at once.  The tile (one contiguous piece of memory) goes through
// the wave's own LDS with 16-byte accesses to memory, then each lane owns one row in registers and needs no other lane;
// rows lie an odd number of words apart in LDS.  No barrier: a wave's LDS accesses stay in order.  (Lanes that share such a
// row stay partly empty: 17 float32 fill 5 of 8 vectors, and every row needs its own sums across lanes.)
//
// Bound by HBM; backward also by its 216 registers, two waves a SIMD.  Measured at float32 2700000 x 17: forward 83 us (378 MB,
// 4.5 TB/s), backward 131 us (572 MB, 4.4 TB/s).  Every column's work is done whether the row has it or not: with a branch a
// column each load of a value or a weight was waited for by itself (98 and 212 us).
// ---------------------------------------------------------------------------------------
constexpr int SHORT_WAVES = 4;

// LDS position of flat element i of the tile: one word of padding a row when the row length is even (inv = 65536 / cols
// rounded up: exact for the tile's i < 2048)
__device__ __forceinline__ int short_pos(int i, int pad, int inv) { return pad ? i + (int)((uint32_t)i * (uint32_t)inv >> 16) : i; }

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A tile in registers: n elements from p on, 16 bytes a lane and turn.
template <typename X, int NC>
struct Tile {
  static constexpr int N = Vec<X>::N, IT = NC / N;
  Vec<X> v[IT];
  __device__ __forceinline__ void load(const X* p, int n, int lane) {
#pragma unroll
    for (int t = 0; t < IT; ++t) {
      const int i = (t * 64 + lane) * N;
      if (i + N <= n)
        v[t].load(p + i);
      else if (i < n)
        v[t].load_some(p + i, n - i);
    }
  }
};
// N values to or from consecutive places (pad: with a gap after every row) of a tile in LDS; what lies behind n stays unused
template <typename A, int N>
__device__ __forceinline__ void short_put(A* lds, const A (&h)[N], int i, int pad, int inv) {
  if (!pad) {
    struct alignas(16) Piece { A e[16 / sizeof(A)]; };
#pragma unroll
    for (int k = 0; k < N; k += 16 / (int)sizeof(A)) {
      Piece q;
#pragma unroll
      for (int j = 0; j < 16 / (int)sizeof(A); ++j) q.e[j] = h[k + j];
      *reinterpret_cast<Piece*>(lds + i + k) = q;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) lds[short_pos(i + j, pad, inv)] = h[j];
  }
}
template <typename A, int N>
__device__ __forceinline__ void short_get(const A* lds, A (&h)[N], int i, int pad, int inv) {
  if (!pad) {
    struct alignas(16) Piece { A e[16 / sizeof(A)]; };
#pragma unroll
    for (int k = 0; k < N; k += 16 / (int)sizeof(A)) {
      const Piece q = *reinterpret_cast<const Piece*>(lds + i + k);
#pragma unroll
      for (int j = 0; j < 16 / (int)sizeof(A); ++j) h[k + j] = q.e[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) h[j] = lds[short_pos(i + j, pad, inv)];
  }
}

// A tile of LDS: 64 rows and room for the last 16 bytes.
template <typename A, int NC>
constexpr int short_words() {
  return 64 * (NC | 1) + 64;
}

template <typename X, typename W, int NC>
__global__ __launch_bounds__(64 * SHORT_WAVES, 4) void ln_fwd_short_kernel(
    const X* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b, X* __restrict__ y,
    typename Acc<X>::type* __restrict__ mean_out, typename Acc<X>::type* __restrict__ rstd_out, int64_t rows, int cols, double eps,
    Drop drop) {
  typedef typename Acc<X>::type A;
  constexpr int N = Vec<X>::N, IT = Tile<X, NC>::IT;
  __shared__ alignas(16) A tile[SHORT_WAVES][short_words<A, NC>()];
  const int wave = threadIdx.x >> 6;
  A* lds = tile[wave];
  const int pad = cols % 2 == 0, pitch = cols | 1, inv = (65536 + cols - 1) / cols;
  __shared__ alignas(16) A weights[2][NC];      // 0 behind the row
  if (threadIdx.x < NC) {
    weights[0][threadIdx.x] = threadIdx.x < cols ? (w ? (A)w[threadIdx.x] : A(1)) : A(0);
    weights[1][threadIdx.x] = threadIdx.x < cols && b ? (A)b[threadIdx.x] : A(0);
  }
  __syncthreads();
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  const int64_t tiles = (rows + 63) / 64, step = (int64_t)gridDim.x * SHORT_WAVES;
  auto elements = [&](int64_t t) { return (int)min((int64_t)64, rows - t * 64) * cols; };
#pragma unroll 1
  for (int64_t t = (int64_t)blockIdx.x * SHORT_WAVES + wave; t < tiles; t += step) {
    const int64_t row0 = t * 64;
    const int n = elements(t), lane = in_loop((int)(threadIdx.x & 63));
    Tile<X, NC> in;
    in.load(x + row0 * cols, n, lane);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int i = (k * 64 + lane) * N;
      A h[N];
#pragma unroll
      for (int j = 0; j < N; ++j) h[j] = in.v[k].get(j);
      if (i < n) short_put<A, N>(lds, h, i, pad, inv);
    }
    wave_lds_fence();
    A v[NC], s = 0, q = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) v[c] = lds[lane * pitch + c];
#pragma unroll
    for (int c = 0; c < NC; ++c) s += c < cols ? v[c] : A(0);
    const A mean = s / (A)cols;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      v[c] = c < cols ? v[c] - mean : A(0);
      q += v[c] * v[c];
    }
    const A rstd = A(1) / sqrt(q / (A)cols + (A)eps);
    if (lane * cols < n) {
#pragma unroll
      for (int k = 0; k < NC; k += 8) {
        A wv[8], bv[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) wv[c] = weights[0][k + c], bv[c] = weights[1][k + c];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (k + c < cols) lds[lane * pitch + k + c] = v[k + c] * rstd * wv[c] + bv[c];
        __builtin_amdgcn_sched_barrier(0);
      }
      if (mean_out) mean_out[row0 + lane] = mean, rstd_out[row0 + lane] = rstd;
    }
    wave_lds_fence();
    X* out = y + row0 * cols;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int i = (k * 64 + lane) * N;
      if (i < n) {
        A h[N];
        short_get<A, N>(lds, h, i, pad, inv);
        if (drop.mode) {
          const uint32_t bits = keep_bits<N>(drop, e0 + (uint64_t)row0 * cols + i);
#pragma unroll
          for (int j = 0; j < N; ++j) h[j] = (bits >> j & 1) ? h[j] * scale : A(0);
        }
        Vec<X> v;
        v.set(h);
        if (i + N <= n)
          v.store(out + i);
        else
          v.store_some(out + i, n - i);
      }
    }
    wave_lds_fence();
  }
}

template <typename X, typename W, int NC>
__global__ __launch_bounds__(64 * SHORT_WAVES, 2) void ln_bwd_short_kernel(
    const X* __restrict__ dy, const X* __restrict__ x, const W* __restrict__ w, const typename Acc<X>::type* __restrict__ mean_in,
    const typename Acc<X>::type* __restrict__ rstd_in, X* __restrict__ dx, typename Acc<X>::type* __restrict__ part, int64_t rows,
    int cols, Drop drop) {
  typedef typename Acc<X>::type A;
  constexpr int N = Vec<X>::N, IT = Tile<X, NC>::IT;
  __shared__ alignas(16) A tile[SHORT_WAVES][short_words<A, NC>()];
  const int wave = threadIdx.x >> 6;
  A* lds = tile[wave];
  const int pad = cols % 2 == 0, pitch = cols | 1, inv = (65536 + cols - 1) / cols;
  __shared__ alignas(16) A weights[1][NC];      // 0 behind the row
  if (threadIdx.x < NC) {
    weights[0][threadIdx.x] = threadIdx.x < cols ? (w ? (A)w[threadIdx.x] : A(1)) : A(0);
  }
  __syncthreads();
  const uint64_t e0 = drop_base(drop);
  const A scale = (A)drop.scale;
  A aw[NC], ab[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) aw[c] = ab[c] = A(0);
  const int64_t tiles = (rows + 63) / 64, step = (int64_t)gridDim.x * SHORT_WAVES;
  auto elements = [&](int64_t t) { return (int)min((int64_t)64, rows - t * 64) * cols; };
#pragma unroll 1
  for (int64_t t = (int64_t)blockIdx.x * SHORT_WAVES + wave; t < tiles; t += step) {
    const int64_t row0 = t * 64;
    const int n = elements(t);
    int lane = in_loop((int)(threadIdx.x & 63));
    const bool live = lane * cols < n;
    Tile<X, NC> nx, ng;
    nx.load(x + row0 * cols, n, lane);
    ng.load(dy + row0 * cols, n, lane);
    const A mean = live ? mean_in[row0 + lane] : A(0), rstd = live ? rstd_in[row0 + lane] : A(0);
    A h[NC], g[NC], s1 = 0, s2 = 0;
    // both tiles change hands in the same piece of LDS: x, then dy, then dx
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int i = (k * 64 + lane) * N;
      A f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = nx.v[k].get(j);
      if (i < n) short_put<A, N>(lds, f, i, pad, inv);
    }
    wave_lds_fence();
#pragma unroll
    for (int c = 0; c < NC; ++c) h[c] = lds[lane * pitch + c];
#pragma unroll
    for (int c = 0; c < NC; ++c) h[c] = c < cols && live ? (h[c] - mean) * rstd : A(0);
    wave_lds_fence();
    lane = in_loop(lane);      // (places in LDS are not kept from one turn to the next: a register an element)
#pragma unroll
    for (int k = 0; k < IT; ++k) {
      const int i = (k * 64 + lane) * N;
      A f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = ng.v[k].get(j);
      if (drop.mode) {
        const uint32_t bits = keep_bits<N>(drop, e0 + (uint64_t)row0 * cols + i);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = (bits >> j & 1) ? f[j] * scale : A(0);
      }
      if (i < n) short_put<A, N>(lds, f, i, pad, inv);
      __builtin_amdgcn_sched_barrier(0);
    }
    wave_lds_fence();
#pragma unroll
    for (int k = 0; k < NC; k += 8) {
      A wv[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) g[k + c] = lds[lane * pitch + k + c], wv[c] = weights[0][k + c];
#pragma unroll
      for (int c = k; c < k + 8; ++c) {
        g[c] = c < cols && live ? g[c] : A(0);
        aw[c] += g[c] * h[c];
        ab[c] += g[c];
        g[c] *= wv[c - k];
        s1 += g[c];
        s2 += g[c] * h[c];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    wave_lds_fence();
    if (dx) {
      s1 /= (A)cols;
      s2 /= (A)cols;
      if (live)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (c < cols) lds[lane * pitch + c] = rstd * (g[c] - s1 - h[c] * s2);
      wave_lds_fence();
      lane = in_loop(lane);
      X* out = dx + row0 * cols;
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int i = (k * 64 + lane) * N;
        if (i < n) {
          A f[N];
          short_get<A, N>(lds, f, i, pad, inv);
          Vec<X> v;
          v.set(f);
          if (i + N <= n)
            v.store(out + i);
          else
            v.store_some(out + i, n - i);
        }
      }
      wave_lds_fence();
    }
  }
  if (!part) return;
  const int lane = threadIdx.x & 63;
  __shared__ A red[SHORT_WAVES][2][NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (c < cols) {
      const A a = lane_sum<64>(aw[c]), g = lane_sum<64>(ab[c]);
      if (lane == 0) red[wave][0][c] = a, red[wave][1][c] = g;
    }
  __syncthreads();
  A* p = part + (int64_t)blockIdx.x * 2 * cols;
  for (int c = threadIdx.x; c < 2 * cols; c += 64 * SHORT_WAVES) {
    const int k = c >= cols, cc = c - k * cols;
    A s = red[0][k][cc];
#pragma unroll
    for (int i = 1; i < SHORT_WAVES; ++i) s += red[i][k][cc];
    p[c] = s;
  }
}

// ---------------------------------------------------------------------------------------
// Dropout of a contiguous array
// ---------------------------------------------------------------------------------------
// Threads own whole counter blocks: a thread's elements start where e is a multiple of 4 (memory alignment does not
// matter, see Vec), so no block is computed twice; the first and the last vector of the array may be partial.
// Bound by HBM and, in 16 bits, nearly as much by the ten rounds of 32 x 32 -> 64 products a block: 2^27 bfloat16 111 us
// (537 MB, 4.8 TB/s; a copy of them 104 us).
template <typename X>
struct DropChunk {
  static constexpr int E = sizeof(X) == 2 ? 8 : 4;         // elements a thread takes at once
};

template <typename X>
__global__ __launch_bounds__(256) void dropout_kernel(const X* x, X* y, int64_t n, Drop drop) {
  typedef typename Acc<X>::type A;
  constexpr int N = Vec<X>::N, E = DropChunk<X>::E, V = E / N;
  const uint64_t e0 = drop_base(drop);
  const int s = (int)(e0 & 3);
  const uint64_t b0 = e0 >> 2;
  const A scale = (A)drop.scale;
  const int64_t step = (int64_t)gridDim.x * 256 * E;
  for (int64_t a = ((int64_t)blockIdx.x * 256 + threadIdx.x) * E; a - s < n; a += step) {
    const int64_t i = a - s;                                // a thread's elements are i .. i + E - 1
    const bool whole = i >= 0 && i + E <= n;
    Vec<X> v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (whole) {
        v[k].load(x + i + k * N);
      } else {
        v[k].u[0] = v[k].u[1] = v[k].u[2] = v[k].u[3] = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (i + k * N + j >= 0 && i + k * N + j < n) v[k].put(j, x[i + k * N + j]);
      }
    }
    if (drop.mode) {
      uint32_t w[E / 4][4];
      if (drop.mode == 1)
#pragma unroll
        for (int q = 0; q < E / 4; ++q) philox(drop, b0 + (uint64_t)(a >> 2) + q, w[q]);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        A h[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int at = k * N + j;
          h[j] = drop.mode == 1 && w[at / 4][at % 4] >= drop.threshold ? v[k].get(j) * scale : A(0);
        }
        v[k].set(h);
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (whole) {
        v[k].store(y + i + k * N);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (i + k * N + j >= 0 && i + k * N + j < n) y[i + k * N + j] = v[k].element(j);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
// (sizes on the host: std::min, the min of hip_runtime.h takes ints there)
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

// Which lanes own a row.
struct Layout {
  int lanes, nv;     // lanes 1: short dense rows, nv columns at most; lanes 0: longer than the registers hold
};
// Forward: few lanes with many elements each (rows of a workgroup of 256 run beside each other).  Backward: two sums stay
// beside every element, so wide rows take more lanes.  Both sides of the borders, TB/s of the rows' traffic:
//   16-bit, 64 columns: 8 lanes 4.9 forward, 4.6 backward; 16 lanes 3.1, 2.5.  16-bit, 200 columns: 32 lanes 4.7, 64 lanes 2.5
//   float32, 32 columns, backward: 8 lanes 4.9; a lane a row 3.3 (its registers spill); 24 columns: a lane a row 4.7
//   float64, 16 columns, backward: 8 lanes 4.7; a lane a row 3.6
//   bfloat16, 8192 columns, forward: 512 lanes of 2 vectors 5.5; 256 of 4 3.7.  16384 columns: 1024 of 2 5.5; 512 of 4 4.5
//   float32, 16384 columns, backward: 1024 lanes of 4 vectors 3.0; 512 of 8 2.2
// float64 (1 GiB of rows), as lanes x vectors, the one taken first: 128 columns 64x1 4.4 forward, 4.5 backward, 64x2 4.3, 4.7; 256
// columns 64x2 4.5, 4.5, 64x4 4.6, 5.4; 512 columns 64x4 5.2, 5.1, 256x2 4.0, 4.5; 1024 columns 256x2 4.8, 4.6, 512x4 3.9 forward,
// 512x2 4.7 backward; 2048 columns 256x4 5.2 forward, 512x4 5.3, 512x2 5.1 backward, 1024x2 5.6; 4096 columns 512x4 5.2 forward,
// 1024x4 5.7, 1024x2 5.2 backward, 1024x4 2.5; 8192 columns 1024x4 5.6, 3.6.
// float32 (512 MB), the same: 512 columns 64x2 6.2, 4.8, 256x2 3.6, 3.7; 1024 columns 64x4 6.0, 4.8, 256x2 5.0, 4.9; 2048 columns 256x2
// 6.1, 4.7, 512x2 5.0 backward, 512x4 4.6 forward; 4096 columns 256x4 6.3 forward, 512x4 6.3, 512x2 4.8 backward, 1024x2 5.0; 8192
// columns 512x4 6.4 forward, 1024x4 5.9, 1024x2 4.6 backward, 1024x4 2.7.
// The backward kernels of 1024 lanes and 2 or 4 vectors spill: 19 to 81 registers of 16-bit rows, 21 (64 where the last vector is
// incomplete) of float32, 39 (95) of float64 ones.
Layout row_layout(int dtype, int cols, bool dense, bool backward) {
  if (dense && cols <= (dtype == 0 ? 8 : dtype == 1 ? 24 : 32)) return {1, (cols + 7) / 8 * 8};
  const int n = dtype == 0 ? 2 : dtype == 1 ? 4 : 8;         // elements of a 16-byte vector
  const int64_t nvec = ((int64_t)cols + n - 1) / n;
  const bool half = n == 8;
  if (nvec <= 8) return {8, 1};
  if (nvec <= 16) return {16, 1};
  if (nvec <= 32) return half ? Layout{32, 1} : Layout{16, 2};
  if (nvec <= 64) return {64, 1};
  if (nvec <= 128) return {64, 2};
  if (nvec <= 256) return half ? Layout{256, 1} : Layout{64, 4};
  if (nvec <= 512) return half && backward ? Layout{512, 1} : Layout{256, 2};
  if (nvec <= 1024) return half ? (backward ? Layout{1024, 1} : Layout{512, 2}) : backward ? Layout{512, 2} : Layout{256, 4};
  if (nvec <= 2048) return backward || half ? Layout{1024, 2} : Layout{512, 4};
  if (nvec <= 4096 && !half) return Layout{1024, 4};
  return {0, 0};
}

// Workgroups of a launch: as many as are resident at a time, each walks its share of the rows (the backward pass leaves
// one partial row of column sums per workgroup).  Backward, a lane adds LANE_ROWS rows at most in its registers' float32: the
// partials are added in 64 bits (2^22 rows of one value: 16384 in a row were off by 800 to 2700 half steps, 480 are by 30).
// PART_BYTES of partials are enough for that with any rows and gradients that 288 GB hold (16-bit ones: 288 GB 2 / 480); of one row
// broadcast to more, a lane adds more.  A launch counts its threads in 32 bits.
constexpr int64_t LANE_ROWS = 480, PART_BYTES = 5ll << 28;

int row_groups(const Layout& l, int64_t rows, int cols, int acc_bytes, bool backward) {
  const int64_t rpb = l.lanes == 1 ? 64 * SHORT_WAVES : std::max(1, 256 / l.lanes);
  const int per_cu = l.lanes <= 256 ? (backward ? 4 : l.nv >= 4 ? 4 : 8) : l.lanes == 512 ? (backward ? (l.nv >= 4 ? 1 : 2) : 4)
                                                                                         : (backward ? 1 : 2);
  const int64_t turns = (rows + rpb - 1) / rpb, resident = per_cu * CUS;
  if (!backward) return (int)std::min(turns, resident);
  const int64_t most = std::min(PART_BYTES / (2ll * cols * acc_bytes), (1ll << 31) / (l.lanes == 1 ? 64 * SHORT_WAVES : group_threads(l.lanes)));
  return (int)std::min(turns, std::max(resident, std::min(most, (turns + LANE_ROWS - 1) / LANE_ROWS)));
}

// column sums of rows the registers do not hold: a thread a column over a range of rows
struct ColsPlan {
  int splits;
  int64_t rows_per_split;
};
ColsPlan cols_plan(int64_t rows, int cols) {
  const int64_t tiles = ((int64_t)cols + 255) / 256;
  int64_t s = std::min((int64_t)1024, std::max((int64_t)1, 8 * CUS / tiles));
  s = std::min(s, (rows + 15) / 16);
  ColsPlan p;
  p.rows_per_split = (rows + s - 1) / s;
  p.splits = (int)((rows + p.rows_per_split - 1) / p.rows_per_split);
  return p;
}

int bwd_parts(const Layout& l, int64_t rows, int cols, int acc_bytes) {
  return l.lanes ? row_groups(l, rows, cols, acc_bytes, true) : cols_plan(rows, cols).splits;
}

template <typename X>
constexpr int type_code() {
  return sizeof(X) == 8 ? 0 : sizeof(X) == 4 ? 1 : 2;      // (layouts depend on the size alone)
}

// S(NC) of short rows; K(LANES, NV) of the layouts forward and backward share
#define TTK_SHORT(S)                                        \
  switch (l.nv) {                                           \
    case 8: S(8); break;                                    \
    case 16:                                                \
      if constexpr (sizeof(X) < 8) { S(16); }               \
      break;                                                \
    case 24:                                                \
      if constexpr (sizeof(X) < 8) { S(24); }               \
      break;                                                \
    case 32:                                                \
      if constexpr (sizeof(X) == 2) { S(32); }              \
      break;                                                \
  }
#define TTK_LAYOUT(L, V, K) \
  case L * 16 + V: K(L, V); break
#define TTK_FWD_LAYOUTS(K)                                                                             \
  if constexpr (sizeof(X) == 2) {                                                                      \
    switch (l.lanes * 16 + l.nv) {                                                                     \
      TTK_LAYOUT(8, 1, K); TTK_LAYOUT(16, 1, K); TTK_LAYOUT(32, 1, K); TTK_LAYOUT(64, 1, K);           \
      TTK_LAYOUT(64, 2, K); TTK_LAYOUT(256, 1, K); TTK_LAYOUT(256, 2, K); TTK_LAYOUT(512, 2, K);       \
      TTK_LAYOUT(1024, 2, K);                            \
    }                                                                                                  \
  } else {                                                                                             \
    switch (l.lanes * 16 + l.nv) {                                                                     \
      TTK_LAYOUT(8, 1, K); TTK_LAYOUT(16, 1, K); TTK_LAYOUT(16, 2, K); TTK_LAYOUT(64, 1, K); TTK_LAYOUT(64, 2, K);          \
      TTK_LAYOUT(64, 4, K); TTK_LAYOUT(256, 2, K); TTK_LAYOUT(256, 4, K); TTK_LAYOUT(512, 4, K);       \
      TTK_LAYOUT(1024, 4, K);                                                                          \
    }                                                                                                  \
  }
#define TTK_BWD_LAYOUTS(K)                                                                             \
  if constexpr (sizeof(X) == 2) {                                                                      \
    switch (l.lanes * 16 + l.nv) {                                                                     \
      TTK_LAYOUT(8, 1, K); TTK_LAYOUT(16, 1, K); TTK_LAYOUT(32, 1, K); TTK_LAYOUT(64, 1, K);           \
      TTK_LAYOUT(64, 2, K); TTK_LAYOUT(256, 1, K); TTK_LAYOUT(512, 1, K); TTK_LAYOUT(1024, 1, K); TTK_LAYOUT(1024, 2, K);                           \
    }                                                                                                  \
  } else {                                                                                             \
    switch (l.lanes * 16 + l.nv) {                                                                     \
      TTK_LAYOUT(8, 1, K); TTK_LAYOUT(16, 1, K); TTK_LAYOUT(16, 2, K); TTK_LAYOUT(64, 1, K); TTK_LAYOUT(64, 2, K);          \
      TTK_LAYOUT(64, 4, K); TTK_LAYOUT(256, 2, K); TTK_LAYOUT(512, 2, K); TTK_LAYOUT(1024, 2, K);      \
      TTK_LAYOUT(1024, 4, K);                                                                          \
    }                                                                                                  \
  }

template <typename X, typename W>
int ln_fwd(const void* x, int64_t ldx, const void* w, const void* b, void* y, void* mean, void* rstd, int64_t rows, int cols,
           double eps, const Drop& d, hipStream_t st) {
  typedef typename Acc<X>::type A;
  const Layout l = row_layout(type_code<X>(), cols, ldx == cols || rows == 1, false);
  if (!l.lanes) {
    hipLaunchKernelGGL((ln_fwd_long_kernel<X, W>), dim3((unsigned)std::min(rows, (int64_t)(4 * CUS))), dim3(LONG_THREADS), 0, st,
                       (const X*)x, ldx, (const W*)w, (const W*)b, (X*)y, (A*)mean, (A*)rstd, rows, cols, eps, d);
    return status();
  }
  const dim3 grid((unsigned)row_groups(l, rows, cols, (int)sizeof(A), false));
#define KR(LANES, NV, R)                                                                                                  \
  hipLaunchKernelGGL((ln_fwd_group_kernel<X, W, LANES, NV, R>), grid, dim3(group_threads(LANES)), 0, st, (const X*)x, ldx,    \
                     (const W*)w, (const W*)b, (X*)y, (A*)mean, (A*)rstd, rows, cols, eps, d)
#define K(LANES, NV) if (cols % Vec<X>::N) KR(LANES, NV, true); else KR(LANES, NV, false)
#define S(NC)                                                                                                             \
  hipLaunchKernelGGL((ln_fwd_short_kernel<X, W, NC>), grid, dim3(64 * SHORT_WAVES), 0, st, (const X*)x, (const W*)w,       \
                     (const W*)b, (X*)y, (A*)mean, (A*)rstd, rows, cols, eps, d)
  if (l.lanes == 1)
    TTK_SHORT(S)
  else
    TTK_FWD_LAYOUTS(K)
#undef K
#undef KR
#undef S
  return status();
}

template <typename X, typename W>
int ln_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const void* mean, const void* rstd, void* dx,
           void* dw, void* db, int64_t rows, int cols, const Drop& d, void* ws, int64_t ws_bytes, hipStream_t st) {
  typedef typename Acc<X>::type A;
  const Layout l = row_layout(type_code<X>(), cols, (ldx == cols && lddy == cols) || rows == 1, true);
  const int parts = bwd_parts(l, rows, cols, (int)sizeof(A));
  const bool sums = dw || db;
  if (sums && (!ws || ws_bytes < (int64_t)parts * 2 * cols * (int64_t)sizeof(A))) return TTK_EWORKSPACE;
  if (sums && (uintptr_t)ws % 8) return TTK_EINVAL;
  if (l.lanes && (dx || sums)) {
    A* part = sums ? (A*)ws : (A*)nullptr;
#define KR(LANES, NV, R)                                                                                                  \
  hipLaunchKernelGGL((ln_bwd_group_kernel<X, W, LANES, NV, R>), dim3((unsigned)parts), dim3(group_threads(LANES)), 0, st,     \
                     (const X*)dy, lddy, (const X*)x, ldx, (const W*)w, (const A*)mean, (const A*)rstd, (X*)dx, part,      \
                     rows, cols, d)
#define K(LANES, NV) if (cols % Vec<X>::N) KR(LANES, NV, true); else KR(LANES, NV, false)
#define S(NC)                                                                                                             \
  hipLaunchKernelGGL((ln_bwd_short_kernel<X, W, NC>), dim3((unsigned)parts), dim3(64 * SHORT_WAVES), 0, st, (const X*)dy,  \
                     (const X*)x, (const W*)w, (const A*)mean, (const A*)rstd, (X*)dx, part, rows, cols, d)
    if (l.lanes == 1)
      TTK_SHORT(S)
    else
      TTK_BWD_LAYOUTS(K)
#undef K
#undef KR
#undef S
  } else if (!l.lanes) {
    if (dx)
      hipLaunchKernelGGL((ln_bwd_long_kernel<X, W>), dim3((unsigned)std::min(rows, (int64_t)(4 * CUS))), dim3(LONG_THREADS), 0, st,
                         (const X*)dy, lddy, (const X*)x, ldx, (const W*)w, (const A*)mean, (const A*)rstd, (X*)dx, rows, cols, d);
    if (sums)
      hipLaunchKernelGGL((ln_cols_kernel<X>), dim3((unsigned)(((int64_t)cols + 255) / 256), (unsigned)parts), dim3(256), 0, st,
                         (const X*)dy, lddy, (const X*)x, ldx, (const A*)mean, (const A*)rstd, (A*)ws, rows, cols,
                         cols_plan(rows, cols).rows_per_split, d);
  }
  if (sums)
    hipLaunchKernelGGL((ln_cols_sum_kernel<A, W>), dim3((unsigned)std::min(((int64_t)cols + 63) / 64, (int64_t)SUM_GROUPS), 2), dim3(1024), 0, st,
                       (const A*)ws, parts, cols, (W*)dw, (W*)db);
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
  if (!x || !y || !mean != !rstd || rows < 1 || cols < 1 || ldx < 0 || !(eps >= 0.0) || !types_ok(dtype, wdtype) ||
      !make_drop(d, p, seed, offset, offset_dev))
    return TTK_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  TTK_BY_TYPES(ln_fwd, x, ldx, w, b, y, mean, rstd, rows, cols, eps, d, st);
}

int64_t ttk_layer_norm_backward_ws_bytes(int dtype, int64_t rows, int cols) {
  if (dtype < 0 || dtype > 3 || rows < 1 || cols < 1) return TTK_EINVAL;
  const int size = dtype == 0 ? 8 : 4;
  const int parts = std::max(bwd_parts(row_layout(dtype, cols, true, true), rows, cols, size),
                             bwd_parts(row_layout(dtype, cols, false, true), rows, cols, size));
  return (int64_t)parts * 2 * cols * size;
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
  const int per = 256 * (dtype < 2 ? 4 : 8);
  const dim3 grid((unsigned)std::min((n + 3 + per - 1) / per, (int64_t)(16 * CUS)));
  switch (dtype) {
    case 0: hipLaunchKernelGGL((dropout_kernel<double>), grid, dim3(256), 0, st, (const double*)x, (double*)y, n, d); break;
    case 1: hipLaunchKernelGGL((dropout_kernel<float>), grid, dim3(256), 0, st, (const float*)x, (float*)y, n, d); break;
    case 2: hipLaunchKernelGGL((dropout_kernel<__bf16>), grid, dim3(256), 0, st, (const __bf16*)x, (__bf16*)y, n, d); break;
    case 3: hipLaunchKernelGGL((dropout_kernel<_Float16>), grid, dim3(256), 0, st, (const _Float16*)x, (_Float16*)y, n, d); break;
  }
  return status();
}

}  // extern "C"
