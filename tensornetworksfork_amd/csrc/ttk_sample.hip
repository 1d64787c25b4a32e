// ttk_sample.hip -- gfx950 kernels that draw a label from a row of logits and a given random number.
//
// With m the row's largest logit: weights w_i = exp((z_i - m) / T) in float64 (1 where z_i == m, 0 where z_i = -inf; NaN
// counts as -inf).  Elements are ordered by descending logit, ties by ascending index.  top-k keeps the first k; top-p
// keeps the elements whose exclusive cumulative weight is below top_p times the weight top-k kept; min-p keeps w_i >= min_p
// (the largest weight is 1).  The label is the first index, in index order, whose cumulative kept weight exceeds u times
// the total.  T <= 0 answers with the lowest index of the maximum, a row without a logit above -inf with -1.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ttk.h"

namespace {

struct SampleArgs {
  const void *u, *temperature, *top_p, *min_p;   // one value a row (float64 when f64, else float32); parameters may be null
  const int32_t* top_k;
  double temperature_all, top_p_all, min_p_all;  // used where the row's own value is missing
  int32_t top_k_all;
  int f64;
};

struct RowArgs {
  double u, T, P, M;
  int k;
};

__device__ __forceinline__ double row_value(const void* p, double all, int f64, int64_t row) {
  return !p ? all : f64 ? reinterpret_cast<const double*>(p)[row] : (double)reinterpret_cast<const float*>(p)[row];
}

__device__ __forceinline__ RowArgs row_args(const SampleArgs& a, int64_t row, int V) {
  RowArgs r;
  r.u = row_value(a.u, 0.0, a.f64, row);
  if (!(r.u > 0.0)) r.u = 0.0;
  r.T = row_value(a.temperature, a.temperature_all, a.f64, row);
  r.P = row_value(a.top_p, a.top_p_all, a.f64, row);
  if (!(r.P < 1.0)) r.P = 1.0;
  r.M = row_value(a.min_p, a.min_p_all, a.f64, row);
  if (!(r.M > 0.0)) r.M = 0.0;
  if (r.M > 1.0) r.M = 1.0;
  r.k = a.top_k ? a.top_k[row] : a.top_k_all;
  if (!(r.P > 0.0)) r.P = 1.0, r.k = 1;      // nothing but the first element
  if (r.k <= 0 || r.k >= V) r.k = 0;
  return r;
}

// Unsigned integers in the order of the logits they stand for; -0 and +0 are one key, NaN is -inf.
template <typename Z>
struct Key {
  typedef uint32_t type;
  typedef float val_t;
  static __device__ __forceinline__ float value(Z z) {
    const float f = (float)z;
    return f != f ? -__builtin_inff() : f + 0.0f;
  }
  static __device__ __forceinline__ uint32_t of(float f) {
    const uint32_t b = __float_as_uint(f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  }
};
template <>
struct Key<double> {
  typedef uint64_t type;
  typedef double val_t;
  static __device__ __forceinline__ double value(double z) { return z != z ? -__builtin_inf() : z + 0.0; }
  static __device__ __forceinline__ uint64_t of(double f) {
    const uint64_t b = (uint64_t)__double_as_longlong(f);
    return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
  }
};

template <typename T>
__device__ __forceinline__ double weight(T z, T m, double temperature) {
  return z == m ? 1.0 : exp(((double)z - (double)m) / temperature);
}

constexpr int ROW_THREADS = 256;

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* buf) {
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  v = buf[0];
#pragma unroll
  for (int i = 1; i < ROW_THREADS / 64; ++i) v += buf[i];
  return v;
}

// index of the n-th (from 1) element of the row with key t
template <typename Z>
__device__ int nth_tie(const Z* z, int c0, int c1, typename Key<Z>::type t, int n, int* counts, int* found) {
  int mine = 0;
  for (int c = c0; c < c1; ++c) mine += Key<Z>::of(Key<Z>::value(z[c])) == t;
  __syncthreads();
  counts[threadIdx.x] = mine;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < (int)threadIdx.x; ++i) before += counts[i];
  if (before < n && before + mine >= n)
    for (int c = c0; c < c1; ++c)
      if (Key<Z>::of(Key<Z>::value(z[c])) == t && ++before == n) *found = c;
  __syncthreads();
  return *found;
}

// One workgroup a row.  Thresholds are found bit by bit: the largest key t with enough elements (or weight) at or above it.
template <typename Z>
__global__ __launch_bounds__(ROW_THREADS) void sample_row_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args,
                                                                 int64_t* __restrict__ label, int64_t rows, int V) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  __shared__ double dbuf[ROW_THREADS];
  __shared__ int ibuf[ROW_THREADS];
  __shared__ F fbuf[ROW_THREADS / 64];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63;
  const int chunk = (V + ROW_THREADS - 1) / ROW_THREADS;
  const int c0 = min(V, tid * chunk), c1 = min(V, c0 + chunk);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const Z* z = logits + row * ld;
    const RowArgs a = row_args(args, row, V);
    F m = -__builtin_inff();
    int at = V;
    for (int c = c0; c < c1; ++c) {
      const F f = Key<Z>::value(z[c]);
      if (f > m) m = f, at = c;
    }
    const F mine = m;
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = max(m, (F)__shfl_xor(m, s));
    __syncthreads();
    if (lane == 0) fbuf[tid >> 6] = m;
    ibuf[tid] = mine == m ? at : V;
    __syncthreads();
    for (int i = 0; i < ROW_THREADS / 64; ++i) m = max(m, fbuf[i]);
    if (!(m > -__builtin_inff()) || !(a.T > 0.0)) {
      if (tid == 0) {
        int first = V;
        for (int i = 0; i < ROW_THREADS; ++i)
          if (fbuf[i >> 6] == m) first = min(first, ibuf[i]);
        label[row] = m > -__builtin_inff() ? first : -1;
      }
      __syncthreads();
      continue;
    }
    K cut = 0;        // kept: key > cut, or key == cut and index <= icut
    int icut = V;
    if (a.k) {
      for (int bit = 8 * (int)sizeof(K) - 1; bit >= 0; --bit) {
        const K cand = cut | ((K)1 << bit);
        int n = 0;
        for (int c = c0; c < c1; ++c) n += Key<Z>::of(Key<Z>::value(z[c])) >= cand;
        if (block_sum(n, ibuf) >= a.k) cut = cand;
      }
      int above = 0;
      for (int c = c0; c < c1; ++c) above += Key<Z>::of(Key<Z>::value(z[c])) > cut;
      above = block_sum(above, ibuf);
      icut = nth_tie<Z>(z, c0, c1, cut, a.k - above, ibuf, &found);
    }
    if (a.P < 1.0) {
      K cut2 = 0;
      double target = 0;
      for (int bit = 8 * (int)sizeof(K); bit >= 0; --bit) {
        const K cand = bit == 8 * (int)sizeof(K) ? (K)0 : cut2 | ((K)1 << bit);   // the first turn sums everything kept
        double s = 0;
        for (int c = c0; c < c1; ++c) {
          const F f = Key<Z>::value(z[c]);
          const K key = Key<Z>::of(f);
          if (key >= cand && (key > cut || (key == cut && c <= icut))) s += weight(f, m, a.T);
        }
        s = block_sum(s, dbuf);
        if (bit == 8 * (int)sizeof(K))
          target = a.P * s;
        else if (s >= target)
          cut2 = cand;
      }
      double s = 0, wt = 0;
      int ties = 0;
      for (int c = c0; c < c1; ++c) {
        const F f = Key<Z>::value(z[c]);
        const K key = Key<Z>::of(f);
        if (key > cut2) s += weight(f, m, a.T);
        if (key == cut2 && (key > cut || c <= icut)) ++ties, wt = weight(f, m, a.T);
      }
      s = block_sum(s, dbuf);
      ties = block_sum(ties, ibuf);
#pragma unroll
      for (int i = 32; i > 0; i >>= 1) wt = max(wt, __shfl_xor(wt, i));
      __syncthreads();
      if (lane == 0) dbuf[tid >> 6] = wt;
      __syncthreads();
      for (int i = 0; i < ROW_THREADS / 64; ++i) wt = max(wt, dbuf[i]);
      const double need = wt > 0 ? ceil((target - s) / wt) : 1.0;
      const int n = need < 1.0 ? 1 : need > (double)ties ? ties : (int)need;
      const int i2 = nth_tie<Z>(z, c0, c1, cut2, n, ibuf, &found);
      cut = cut2;
      icut = i2;
    }
    double s = 0;
    for (int c = c0; c < c1; ++c) {
      const F f = Key<Z>::value(z[c]);
      const K key = Key<Z>::of(f);
      if (key > cut || (key == cut && c <= icut)) {
        const double w = weight(f, m, a.T);
        if (w >= a.M) s += w;
      }
    }
    __syncthreads();
    dbuf[tid] = s;
    if (tid == 0) found = -1;
    __syncthreads();
    double before = 0, total = 0;
    for (int i = 0; i < ROW_THREADS; ++i) {
      if (i == tid) before = total;
      total += dbuf[i];
    }
    const double target = a.u * total;
    const bool last = !(target < total);  // u >= 1, or rounded up to it: the last kept element
    if (s > 0 && (last ? before + s >= total : (before <= target && before + s > target))) {
      int pick = -1;
      double c = before;
      for (int i = c0; i < c1; ++i) {
        const F f = Key<Z>::value(z[i]);
        const K key = Key<Z>::of(f);
        if (!(key > cut || (key == cut && i <= icut))) continue;
        const double w = weight(f, m, a.T);
        if (!(w >= a.M) || !(w > 0)) continue;
        pick = i;
        c += w;
        if (!last && c > target) break;
      }
      found = pick;
    }
    __syncthreads();
    if (tid == 0) label[row] = found;
    __syncthreads();
  }
}

template <typename Z>
int launch(const void* logits, int64_t ld, const SampleArgs& a, int64_t* label, int64_t rows, int V, hipStream_t st) {
  hipLaunchKernelGGL((sample_row_kernel<Z>), dim3((unsigned)min(rows, (int64_t)65536)), dim3(ROW_THREADS), 0, st,
                     (const Z*)logits, ld, a, label, rows, V);
  return hipGetLastError() == hipSuccess ? TTK_OK : TTK_ELAUNCH;
}

}  // namespace

extern "C" {

int ttk_sample(int dtype, const void* logits, int64_t ld, const void* u, int f64, const void* temperature, double temperature_all,
               const int32_t* top_k, int top_k_all, const void* top_p, double top_p_all, const void* min_p, double min_p_all,
               int64_t* label, int64_t rows, int V, void* stream) {
  if (!logits || !u || !label || rows < 1 || V < 1 || ld < 0) return TTK_EINVAL;
  const SampleArgs a = {u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, f64};
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case 0: return launch<double>(logits, ld, a, label, rows, V, st);
    case 1: return launch<float>(logits, ld, a, label, rows, V, st);
    case 2: return launch<__bf16>(logits, ld, a, label, rows, V, st);
    case 3: return launch<_Float16>(logits, ld, a, label, rows, V, st);
  }
  return TTK_EINVAL;
}

}  // extern "C"
