// ttk_sample.hip -- gfx950 kernels that draw a label from a row of logits and a given random number.
//
// With m the row's largest logit: weights w_i = exp((z_i - m) / T) in float64 (1 where z_i == m, 0 where z_i = -inf; NaN
// counts as -inf).  Elements are ordered by descending logit, ties by ascending index.  top-k keeps the first k; top-p
// keeps the elements whose exclusive cumulative weight is below top_p times the weight top-k kept; min-p keeps w_i >= min_p
// (the largest weight is 1).  The label is the first index, in index order, whose cumulative kept weight exceeds u times
// the total.  T <= 0 answers with the lowest index of the maximum (temperatures between 0 and 1e-306 act as 1e-306, an
// infinite one as the largest number: all weigh the same), a row without a logit above -inf with -1.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

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
  if (r.T > 0.0 && r.T < 1e-306) r.T = 1e-306;      // 32 log2(e) / T stays finite
  if (r.T > 0x1.fffffffffffffp1023) r.T = 0x1.fffffffffffffp1023;      // (infinite times log(1) would be no number)
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
// LOW: that many low bits of a 16-bit logit's key are all 0 or all 1 (bits a float32 has and the logit has not).
template <typename Z>
struct Key {
  typedef uint32_t type;
  typedef float val_t;
  static constexpr int LOW = sizeof(Z) == 4 ? 0 : __is_same(Z, __bf16) ? 16 : 13;
  static __device__ __forceinline__ float value(Z z) { return fmaxf((float)z, -__builtin_inff()); }
  static __device__ __forceinline__ uint32_t of(float f) {
    const uint32_t b = __float_as_uint(f + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  }
};
template <>
struct Key<double> {
  typedef uint64_t type;
  typedef double val_t;
  static constexpr int LOW = 0;
  static __device__ __forceinline__ double value(double z) { return fmax(z, -__builtin_inf()); }
  static __device__ __forceinline__ uint64_t of(double f) {
    const uint64_t b = (uint64_t)__double_as_longlong(f + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
  }
};

// Weights relative to the row's largest logit: 2^((z - m) log2(e) / T) as 2^n times the Taylor polynomial of 2^f, |f| <= 1/2
// (terms up to (f ln 2)^12 / 12!: relative error below 2e-16).  z == m gives exactly 1, -inf exactly 0.
template <typename F>
struct Weight {
  F m;
  double c;        // log2(e) / T
  __device__ __forceinline__ Weight(F m_, double T) : m(m_), c(1.4426950408889634074 / T) {}
  __device__ __forceinline__ double operator()(F z) const {
    double t = ((double)z - (double)m) * c;
    t = z == m ? 0.0 : t > -1100.0 ? t : -1100.0;
    const double n = rint(t), f = t - n;
    double p = 2.56784359934881958e-11;
    p = fma(p, f, 4.44553827187081007e-10);
    p = fma(p, f, 7.05491162080112088e-09);
    p = fma(p, f, 1.01780860092396960e-07);
    p = fma(p, f, 1.32154867901443053e-06);
    p = fma(p, f, 1.52527338040598377e-05);
    p = fma(p, f, 1.54035303933816061e-04);
    p = fma(p, f, 1.33335581464284411e-03);
    p = fma(p, f, 9.61812910762847688e-03);
    p = fma(p, f, 5.55041086648215762e-02);
    p = fma(p, f, 2.40226506959100694e-01);
    p = fma(p, f, 6.93147180559945286e-01);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
  }
};

// The row with an infinite maximum is the row of its +inf elements alone, all alike.
template <typename F>
__device__ __forceinline__ F finite(F z, bool top_inf) {
  return top_inf ? (z == __builtin_inff() ? F(0) : F(-__builtin_inff())) : z;
}

// One step of a scan over the wave: v + (v of the lane CTRL names, 0 where there is none), in the rows of ROWS.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T scan_step(T v) {
  union {
    T t;
    int u[sizeof(T) / 4];
  } a, b;
  a.t = v;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 4; ++i) b.u[i] = __builtin_amdgcn_update_dpp(0, a.u[i], CTRL, ROWS, 0xf, ROWS == 0xf);
  return v + b.t;
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {      // inclusive
  v = scan_step<0x111, 0xf>(v);      // 1, 2, 4, 8 lanes back within 16
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);      // lane 15 to the next 16 lanes
  return scan_step<0x143, 0xc>(v);   // lane 31 to the upper 32
}
template <typename T>
__device__ __forceinline__ T from_lane(T v, int lane) {      // lane: the same in every lane
  union {
    T t;
    int u[sizeof(T) / 4];
  } a;
  a.t = v;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 4; ++i) a.u[i] = __builtin_amdgcn_readlane(a.u[i], lane);
  return a.t;
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
  return from_lane(wave_scan(v), 63);
}
template <typename T>
__device__ __forceinline__ T wave_max(T v) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const T o = __shfl_xor(v, s);
    v = o > v ? o : v;
  }
  return v;
}

// ---------------------------------------------------------------------------------------
// Few classes: a thread a row, everything in registers; an element's place in the order is counted against all others.
// Bound by the launch: 60000 float64 rows of 10 take 6 us (5 MB).
// ---------------------------------------------------------------------------------------
constexpr int FEW = 16;

template <typename Z>
__global__ __launch_bounds__(64) void sample_few_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args,
                                                        int64_t* __restrict__ label, int64_t rows, int V) {
  typedef typename Key<Z>::val_t F;
  const int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (row >= rows) return;
  const Z* p = logits + row * ld;
  F z[FEW], m = -__builtin_inff();
  int first = -1;
#pragma unroll
  for (int i = 0; i < FEW; ++i) z[i] = i < V ? Key<Z>::value(p[i]) : F(-__builtin_inff());
#pragma unroll
  for (int i = 0; i < FEW; ++i)
    if (z[i] > m) m = z[i], first = i;
  const RowArgs a = row_args(args, row, V);
  if (first < 0 || !(a.T > 0.0)) {
    label[row] = first;
    return;
  }
  const bool inf = m == __builtin_inff();
  if (inf) m = 0;
  const Weight<F> weight(m, a.T);
  double w[FEW];
#pragma unroll
  for (int i = 0; i < FEW; ++i) {
    z[i] = finite(z[i], inf);
    w[i] = i < V ? weight(z[i]) : 0.0;
  }
  if (a.k || a.P < 1.0) {
    uint32_t kept = 0;
    double total = 0;
#pragma unroll
    for (int i = 0; i < FEW; ++i) {
      int rank = 0;
#pragma unroll
      for (int j = 0; j < FEW; ++j)
        if (j != i) rank += j < i ? z[j] >= z[i] : z[j] > z[i];
      if (!a.k || rank < a.k) kept |= 1u << i, total += w[i];
    }
    if (a.P < 1.0) {
      const double target = a.P * total;
      uint32_t nucleus = 0;
#pragma unroll
      for (int i = 0; i < FEW; ++i) {
        double before = 0;
#pragma unroll
        for (int j = 0; j < FEW; ++j)
          if (j != i && (j < i ? z[j] >= z[i] : z[j] > z[i])) before += w[j];
        if (before < target) nucleus |= 1u << i;
      }
      kept &= nucleus;
    }
#pragma unroll
    for (int i = 0; i < FEW; ++i)
      if (!(kept >> i & 1)) w[i] = 0;
  }
  double total = 0;
#pragma unroll
  for (int i = 0; i < FEW; ++i) {
    if (!(w[i] >= a.M)) w[i] = 0;
    total += w[i];
  }
  const double target = a.u * total;
  double c = 0;
  int pick = -1;
  bool done = false;
#pragma unroll
  for (int i = 0; i < FEW; ++i) {
    c += w[i];
    if (!done && w[i] > 0) pick = i, done = c > target;
  }
  label[row] = pick;
}

// ---------------------------------------------------------------------------------------
// Up to 64 E W classes: W waves a row, E consecutive elements a lane at most.  Cuts are found bit by bit: the largest key t
// with enough elements (or weight) at or above it.  A search ends as soon as one element more or less is all that is open.
//
// A row is read once; the time goes into the searches (an instruction or two an element and bit) and the float64 weights.
// Measured for 16.7 million float32 logits (a copy: 13 us), 1000 and 6000 classes a row: greedy 19 and 20 us, plain 35 and
// 49, top-k 50 52 and 87, top-p 0.9 85 and 160.  The launches that longer rows take need 954 us for top-k 50 on rows of 1025.
// ---------------------------------------------------------------------------------------
typedef uint32_t raw_t __attribute__((ext_vector_type(4), aligned(2)));

// What the waves of a row agree on.  Every call writes the other half of `buf`, so one barrier a call is enough.
template <int W>
struct RowWaves {
  struct Part {
    double s;
    int n;
  };
  Part* buf;      // [2][W]
  int wave, turn;
  __device__ __forceinline__ RowWaves(Part* buf_) : buf(buf_), wave(W > 1 ? threadIdx.x >> 6 : 0), turn(0) {}
  __device__ __forceinline__ const Part* share(double s, int n) {
    Part* p = buf + turn * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) p[wave] = Part{s, n};
    __syncthreads();
    return p;
  }
  // sums over the row's waves, and over the waves in front of this one
  __device__ __forceinline__ void sum(int& n) {
    if constexpr (W > 1) {
      const Part* p = share(0.0, n);
      n = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) n += p[i].n;
      n = __builtin_amdgcn_readfirstlane(n);
    }
  }
  __device__ __forceinline__ void sum(double& s, int& n) {
    if constexpr (W > 1) {
      const Part* p = share(s, n);
      s = 0, n = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) s += p[i].s, n += p[i].n;
    }
  }
  __device__ __forceinline__ int in_front(int n) {
    int before = 0;
    if constexpr (W > 1) {
      const Part* p = share(0.0, n);
#pragma unroll
      for (int i = 0; i < W - 1; ++i) before += i < wave ? p[i].n : 0;
    }
    return before;
  }
  __device__ __forceinline__ double in_front(double s, double& total) {
    double before = 0;
    total = s;
    if constexpr (W > 1) {
      const Part* p = share(s, 0);
      total = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        before += i < wave ? p[i].s : 0.0;
        total += p[i].s;
      }
    }
    return before;
  }
  __device__ __forceinline__ double largest(double s) {
    if constexpr (W > 1) {
      const Part* p = share(s, 0);
#pragma unroll
      for (int i = 0; i < W; ++i) s = p[i].s > s ? p[i].s : s;
    }
    return s;
  }
  // the row's largest and the first index that has it
  __device__ __forceinline__ void largest(double& s, int& at) {
    if constexpr (W > 1) {
      const Part* p = share(s, at);
      s = p[0].s, at = p[0].n;
#pragma unroll
      for (int i = 1; i < W; ++i)
        if (p[i].s > s) s = p[i].s, at = p[i].n;
    }
  }
  // bit i: what wave i says
  __device__ __forceinline__ uint32_t votes(bool b) {
    uint32_t v = b;
    if constexpr (W > 1) {
      const Part* p = share(0.0, b);
      v = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) v |= (uint32_t)p[i].n << i;
    }
    return v;
  }
};

template <typename Z, int E, int W>
__global__ __launch_bounds__(W > 1 ? 64 * W : 256) void sample_wave_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args,
                                                                          int64_t* __restrict__ label, int64_t rows, int V) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  constexpr int N = 16 / (int)sizeof(Z);      // elements of a 16-byte load (any alignment)
  __shared__ typename RowWaves<W>::Part parts[2 * W];
  RowWaves<W> waves(parts);
  const int lane = threadIdx.x & 63;
  const int64_t row = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const Z* p = logits + row * ld;
  int e = (V + 64 * W - 1) / (64 * W);
  if (E >= N) e = (e + N - 1) / N * N;
  const int c0 = (waves.wave * 64 + lane) * e;      // this lane's elements: c0 .. c0 + e - 1
  F z[E], m = -__builtin_inff();
  int first = 0x7FFFFFFF;
  if constexpr (E >= N) {
    struct Elements {
      Z z[N];
    };
#pragma unroll
    for (int i = 0; i < E; i += N) {
      if (i < e && c0 + i + N <= V) {
        const Elements v = __builtin_bit_cast(Elements, *reinterpret_cast<const raw_t*>(p + c0 + i));
#pragma unroll
        for (int j = 0; j < N; ++j) z[i + j] = Key<Z>::value(v.z[j]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) z[i + j] = i < e && c0 + i + j < V ? Key<Z>::value(p[c0 + i + j]) : F(-__builtin_inff());
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) z[i] = i < e && c0 + i < V ? Key<Z>::value(p[c0 + i]) : F(-__builtin_inff());
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (z[i] > m) m = z[i], first = c0 + i;
  const F mine = m;
  m = wave_max(m);
  int at_m = __builtin_amdgcn_readlane(first, (int)__builtin_ctzll(__ballot(mine == m)));
  if constexpr (W > 1) {
    double s = (double)m;
    waves.largest(s, at_m);
    m = (F)s;
  }
  const RowArgs a = row_args(args, row, V);
  if (!(m > -__builtin_inff()) || !(a.T > 0.0)) {
    if (lane == 0 && waves.wave == 0) label[row] = m > -__builtin_inff() ? at_m : -1;
    return;
  }
  const bool inf = m == __builtin_inff();
  if (inf) m = 0;
  const Weight<F> weight(m, a.T);
  K key[E];
  double w[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    z[i] = finite(z[i], inf);
    w[i] = weight(z[i]);
    key[i] = w[i] > 0 ? Key<Z>::of(z[i]) : K(0);      // (key 0: dropped; no element that is left has it)
  }
  constexpr int BITS = 8 * (int)sizeof(K), LOW = Key<Z>::LOW;
  // keeps, of the elements with w > 0, those in front of the cut: key above t, or the first `ties` of those with key t
  auto cut_at = [&](K t, int ties) {
    int before = 0;
    const K low = LOW ? (K)((1ull << LOW) - 1) : (K)0;
    t |= low;
#pragma unroll
    for (int i = 0; i < E; ++i) before += w[i] > 0 && (K)(key[i] | low) == t;
    const int upto = wave_scan(before);
    before = upto - before + waves.in_front(__builtin_amdgcn_readlane(upto, 63));
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const K k = key[i] | low;
      if (k < t || (k == t && w[i] > 0 && before++ >= ties)) w[i] = 0, key[i] = 0;
    }
  };
  auto cut_below = [&](K t) {      // keeps what is not below t
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (key[i] < t) w[i] = 0, key[i] = 0;
  };
  if (a.k) {
    K t = 0;
    int above = 0, all = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) all += __popcll(__ballot(key[i] > 0));
    waves.sum(all);
    if (all > a.k) {
      bool exact = false;
      for (int bit = BITS - 1; bit >= LOW && !exact; --bit) {
        const K cand = t | ((K)1 << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) n += __popcll(__ballot(key[i] >= cand));
        waves.sum(n);
        if (n >= a.k)
          t = cand, exact = n == a.k;
        else
          above = n;      // the last candidate with too few is the next key above the final t: what lies above t
      }
      if (exact)
        cut_below(t);
      else
        cut_at(t, a.k - above);
    }
  }
  if (a.P < 1.0) {
    double total = 0;
    int kept = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) total += w[i], kept += __popcll(__ballot(key[i] > 0));
    total = wave_sum(total);
    waves.sum(total, kept);
    const double target = a.P * total;
    K t = 0;
    double above = 0;
    int n_above = 0;                             // elements (w > 0) that `above` sums, and those at or above t
    bool one = kept == 1;
    for (int bit = BITS - 1; bit >= LOW && !one; --bit) {
      const K cand = t | ((K)1 << bit);
      double s = 0;
      int n = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const bool in = key[i] >= cand;
        s += in ? w[i] : 0.0;
        n += __popcll(__ballot(in));
      }
      s = wave_sum(s);
      waves.sum(s, n);
      if (s >= target)
        t = cand, kept = n;
      else
        above = s, n_above = n;
      one = kept - n_above == 1;                 // the element that takes the sum to the target
    }
    if (one) {
      cut_below(t);
    } else {
      double wt = 0;
      const K low = LOW ? (K)((1ull << LOW) - 1) : (K)0;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if ((K)(key[i] | low) == (K)(t | low) && w[i] > 0) wt = w[i];
      wt = waves.largest(wave_max(wt));
      const double need = wt > 0 ? ceil((target - above) / wt) : 1.0;
      cut_at(t, need < 1.0 ? 1 : need > (double)V ? V : (int)need);
    }
  }
  double s = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (!(w[i] >= a.M)) w[i] = 0;
    s += w[i];
  }
  double upto = wave_scan(s), total;
  upto += waves.in_front(from_lane(upto, 63), total);
  const double target = a.u * total;
  uint64_t who = __ballot(s > 0 && upto > target);
  uint32_t where = waves.votes(who != 0);
  const bool last = where == 0;                     // u >= 1, or rounded up to it: the last kept element
  if (last) who = __ballot(s > 0), where = waves.votes(who != 0);
  if (waves.wave != (last ? 31 - (int)__builtin_clz(where) : (int)__builtin_ctz(where))) return;
  const int at = last ? 63 - (int)__builtin_clzll(who) : (int)__builtin_ctzll(who);
  if (lane == at) {
    double c = upto - s;
    int pick = -1;
    bool done = false;
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (!done && w[i] > 0) c += w[i], pick = c0 + i, done = !last && c > target;
    label[row] = pick;
  }
}

// ---------------------------------------------------------------------------------------
// Many classes: a few launches over all rows, a row split over workgroups where rows are few.
//
//   maxima    the largest logit of each of up to 4096 groups of a row's elements (their largest is m; the k-th largest bounds
//             the k-th largest element from below)
//   collect   top-k: the elements at or above that bound, a few more than k, into the row's list
//   counts    top-p, and top-k where the list would not hold it: the number of elements in each of 4096 bins below m and the
//             sum of their places within the bin.  The bin's weight follows to second order in its width (relative 1e-5), so
//             the cumulative weight is bounded from both sides, and
//   window    the border of top-p lies in a window of a few bins, that of top-k in one
//   sums      every weight once: float64 sums of the kept ones per segment of the row, and of the rest; the window's elements
//             go into the row's list
//   finish    a workgroup a row: the cut, by histograms of the list refined until few elements share the border's bin, whose
//             order is then counted (or, up to 512, sorted) in LDS; what the cut keeps of the list joins the segment sums; the
//             segment where their running sum passes u times the total, and the element in it.  A top-k list of at most 256
//             elements is drawn from by itself
//   slow      the rows whose list does not hold what it should (thousands of equal logits) and those that both top-p and a
//             top-k above what the groups bound cut: the same by histograms over the whole row
//
// Elements of -inf do not exist for any of this, nor do weights that are 0 in 64 bits; min-p is a bound on the value,
// m + T ln(min_p).  Sums are added in a fixed order in float64, counts are whole numbers, lists are sorted: the label does not
// depend on the order in which workgroups run.  Where LDS atomics add up weights these are whole numbers too: of 2^-48 of the
// largest for the (at most 8192) elements of a list, two words each for the elements of a whole row.
//
// Measured for 512 rows of 131072 bfloat16 (134 MB, read in 26 us at a copy's rate), top-p 0.95, us: maxima 14 (HBM), counts
// 49 (one 64-bit LDS atomic an element), sums 82 (about 22 instructions an element, 14 of them float64, and a dozen more
// for the window), finish 20 and slow 4 (latency of one workgroup a row).  One row alone, top-k 50: 19, four launches of
// which each waits for the one before.  256 rows of 100003 float32 with cuts of their own: 19 + 29 + 22 + 33 + 21 + 4.
// ---------------------------------------------------------------------------------------
constexpr int BINS = 2048, COUNTS = 4096, SEGS = 1024, FEW_GROUPS = 1024, GROUPS = 4096, LIST_CAP = 8192;
constexpr int TB = 256, TW = TB / 64;      // threads and waves of the passes and of `finish`
constexpr int RT = 1024, RW = RT / 64;     // of `counts`, `window` and `slow`

template <typename Z>
struct Chunk {
  static constexpr int N = 16 / (int)sizeof(Z);
  typedef uint32_t raw_t __attribute__((ext_vector_type(4), aligned(2)));
  union {
    uint32_t u[4];
    Z e[N];
  };
};

// A row as a wave sees it: steps of 64 x 16 bytes, R steps a segment; the wave owns segments first, first + stride, ...
template <typename Z>
struct RowView {
  const Z* p;
  int V, steps, R, first, stride;
  bool inf;        // the maximum is +inf
};

// The 16 bytes of this lane in step t.  Behind the row's end the last 16 bytes are read again (a row has more than that).
template <typename Z>
__device__ __forceinline__ int chunk_base(const RowView<Z>& row, int t) {
  const int64_t at = ((int64_t)t * 64 + (int)(threadIdx.x & 63)) * Chunk<Z>::N;
  return (int)min(at, (int64_t)(row.V - Chunk<Z>::N));
}
template <typename Z>
__device__ __forceinline__ void load_chunk(Chunk<Z>& c, const RowView<Z>& row, int t) {
  const typename Chunk<Z>::raw_t r = *reinterpret_cast<const typename Chunk<Z>::raw_t*>(row.p + chunk_base(row, t));
  c.u[0] = r.x, c.u[1] = r.y, c.u[2] = r.z, c.u[3] = r.w;
}
// Its values; those another lane has already are -inf.  NaN stays: every comparison below is false for it, which is what
// -inf would get.
template <typename Z>
__device__ __forceinline__ void chunk_values(typename Key<Z>::val_t (&v)[Chunk<Z>::N], const Chunk<Z>& c, const RowView<Z>& row,
                                             int t) {
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = (F)c.e[j];
  if (t == row.steps - 1) {
    const int64_t again = ((int64_t)t * 64 + (int)(threadIdx.x & 63)) * N - chunk_base(row, t);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < again) v[j] = -__builtin_inff();
  }
  if (row.inf)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = finite(v[j], true);
}

// Calls f(values, first index) for every 16 bytes of the wave's part of the row and end(segment) after its last step of a
// segment.  The next three steps are under way while one is worked on.
template <typename Z, typename Fn, typename End>
__device__ __forceinline__ void walk(const RowView<Z>& row, Fn f, End end) {
  constexpr int N = Chunk<Z>::N;
  int s = row.first, r = 0, ls = s, lr = 0;      // the step at work, the step to load next
  Chunk<Z> q[4];
  auto load = [&](Chunk<Z>& c) {
    load_chunk<Z>(c, row, ls * row.R + lr);
    if (++lr == row.R) lr = 0, ls += row.stride;
  };
  load(q[0]);
  load(q[1]);
  load(q[2]);
#pragma unroll 1
  for (int t = s * row.R; t < row.steps;) {
    load(q[3]);
    typename Key<Z>::val_t v[N];
    chunk_values<Z>(v, q[0], row, t);
    f(v, chunk_base(row, t));
    q[0] = q[1], q[1] = q[2], q[2] = q[3];
    const bool full = ++r == row.R;
    if (full || t + 1 >= row.steps) end(s);
    if (full) r = 0, s += row.stride;
    t = s * row.R + r;
  }
}
struct NoEnd {
  __device__ __forceinline__ void operator()(int) const {}
};

// LDS of a workgroup of T threads that cuts a row and draws from it.
template <typename Z, int T>
struct RowShared {
  typedef typename Key<Z>::type K;
  static constexpr int CAP = 2 * T;
  union {
    unsigned long long hist[BINS];
    struct {
      uint64_t key[CAP];                                     // 32-bit keys: key << 32 | ~index
      uint32_t nidx[sizeof(K) == 8 ? CAP : 1];               // 64-bit keys: ~index
    } list;
    int count[SEGS];
  };
  double seg[SEGS];
  double pow2[32];
  double wave_d[T / 64], seg_before;
  unsigned long long wave_u[T / 64];
  K wave_lo[T / 64], wave_hi[T / 64];
  int n, at, which, last;
  unsigned long long above, above_l;
  unsigned long long hist_l[T > 256 ? BINS : 1];             // second words (whole rows)
  K cut_key;
  int cut_idx;
};

__device__ __forceinline__ void fill_pow2(double* pow2) {
  if (threadIdx.x < 32) pow2[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
}

// The weight of Weight, with 2^(n / 32) from a table: 2^((z - m) log2(e) / T) = 2^(n div 32) pow2[n mod 32] 2^(f / 32),
// |f| <= 1/2, the last factor by its Taylor polynomial (relative error below 3e-15).  The 32 doubles lie in 64 different
// LDS banks.  m is finite; an element that is not kept weighs 0, one that is lies at most 1075 / log2(e) T below m.
template <typename F>
struct RowWeight {
  double m, c;
  const double* pow2;
  __device__ __forceinline__ RowWeight(F m_, double T, const double* table)
      : m((double)m_), c(32 * 1.4426950408889634074 / T), pow2(table) {}
  __device__ __forceinline__ double operator()(F z, bool keep) const {
    const int64_t b = __double_as_longlong(((double)z - m) * c);
    const int hi = keep ? (int)(b >> 32) : (int)0xC0E13000;      // -35200: 2^-1100, which is 0
    const double t = __longlong_as_double((int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)b));
    const double s = t + 0x1.8p52, f = t - (s - 0x1.8p52);
    const int n = (int)(uint32_t)__double_as_longlong(s);
    double p = 3.97370998454941544e-11;
    p = fma(p, f, 9.17256270182464302e-09);
    p = fma(p, f, 1.69385097243718189e-06);
    p = fma(p, f, 2.34596198202246772e-04);
    p = fma(p, f, 2.16608493924982902e-02);
    p = fma(p, f, 1.0);
    return ldexp(p * pow2[n & 31], n >> 5);
  }
};

// Weights of a list's elements as whole numbers of 2^-48: sums that do not depend on an order.  The sum of LIST_CAP = 2^13 of them
// stays below 2^62; each is off by half a unit at most, a list by 2^-36 of the largest weight.
struct Whole {
  static constexpr double FIXED = 0x1p48;
  __device__ __forceinline__ unsigned long long operator()(double w) const {      // w <= 1, rounded
    return (unsigned long long)__double_as_longlong(w * FIXED + 0x1p52) - 0x4330000000000000ull;
  }
};

// Weights of a whole row's elements in two such words: h 2^-S + l 2^-2S with S = 61 - log2 V, rounded down.  V of either stay
// below 2^62, and V times the half unit that each weight is off by is 2^-33 of the largest weight at V = 2^30, 2^-72 at 2^17.
struct Mass {
  unsigned long long h, l;
  __device__ __forceinline__ Mass operator+(const Mass& o) const { return {h + o.h, l + o.l}; }
};
struct TwoWords {
  double fixed;      // 2^S <= 2^48
  __device__ __forceinline__ explicit TwoWords(int V) : fixed(ldexp(1.0, 30 + (int)__builtin_clz(V))) {}
  __device__ __forceinline__ Mass operator()(double w) const {      // w <= 1
    const double x = w * fixed, h = fmax(x - 0.5, 0.0) + 0x1p52;   // 2^52 + the whole part of x, or one less where x is whole
    const double l = (x - (h - 0x1p52)) * fixed + 0x1p52;          // 2^52 + the rest, 0 to 1, in units of 2^-S
    constexpr unsigned long long ZERO = 0x4330000000000000ull;
    return {(unsigned long long)__double_as_longlong(h) - ZERO, (unsigned long long)__double_as_longlong(l) - ZERO};
  }
  __device__ __forceinline__ double value(const Mass& m) const { return (double)m.h / fixed + (double)m.l / (fixed * fixed); }
};

template <int T, typename A>
__device__ __forceinline__ A block_scan(A v, A* buf, A& total) {      // inclusive; buf: T / 64 values
  const int wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) buf[wave] = v;
  __syncthreads();
  A before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) {
    if (i < wave) before += buf[i];
    total += buf[i];
  }
  return v + before;
}

template <int T, typename K>
__device__ __forceinline__ void block_range(K& lo, K& hi, K* buf_lo, K* buf_hi) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const K a = __shfl_xor(lo, s), b = __shfl_xor(hi, s);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf_lo[threadIdx.x >> 6] = lo, buf_hi[threadIdx.x >> 6] = hi;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < T / 64; ++i) {
    lo = buf_lo[i] < lo ? buf_lo[i] : lo;
    hi = buf_hi[i] > hi ? buf_hi[i] : hi;
  }
}

// ---- the LDS list: at most 2 T elements; what comes first sorts higher -------------------------------------------

template <typename Z>
struct Item {
  typedef typename Key<Z>::type K;
  K k;
  uint32_t n;        // ~index
};
template <typename Z>
__device__ __forceinline__ bool in_front(const Item<Z>& a, const Item<Z>& b) {
  if constexpr (sizeof(a.k) == 4)
    return ((uint64_t)a.k << 32 | a.n) > ((uint64_t)b.k << 32 | b.n);
  else
    return a.k > b.k || (a.k == b.k && a.n > b.n);
}
template <typename Z, int T>
__device__ __forceinline__ void list_put(RowShared<Z, T>& sh, int i, const Item<Z>& e) {
  if constexpr (sizeof(e.k) == 4) {
    sh.list.key[i] = (uint64_t)e.k << 32 | e.n;
  } else {
    sh.list.key[i] = e.k;
    sh.list.nidx[i] = e.n;
  }
}
template <typename Z, int T>
__device__ __forceinline__ Item<Z> list_get(const RowShared<Z, T>& sh, int i) {
  if constexpr (sizeof(typename Key<Z>::type) == 4)
    return {(uint32_t)(sh.list.key[i] >> 32), (uint32_t)sh.list.key[i]};
  else
    return {sh.list.key[i], sh.list.nidx[i]};
}

// Bitonic sort of the first n elements (n <= 2 T), the first in front.  Wave w holds elements 128 w + lane and 128 w + 64 +
// lane in registers; distances up to 64 are exchanged there, longer ones through LDS.
template <typename Z, int T>
__device__ __forceinline__ void list_sort(RowShared<Z, T>& sh, int n) {
  int n2 = 128;
  while (n2 < n) n2 <<= 1;
  const int lane = threadIdx.x & 63, i0 = (threadIdx.x >> 6) * 128 + lane;
  const bool mine = i0 - lane < n2;      // (the same in a wave)
  Item<Z> e[2];
  __syncthreads();
  if (mine)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Item<Z> none = {0, 0};       // sorts last
      e[h] = i0 + 64 * h < n ? list_get<Z, T>(sh, i0 + 64 * h) : none;
    }
#pragma unroll 1
  for (int size = 2; size <= n2; size <<= 1) {
    if (size > 128) {
      __syncthreads();
      if (mine) {
        list_put<Z, T>(sh, i0, e[0]);
        list_put<Z, T>(sh, i0 + 64, e[1]);
      }
#pragma unroll 1
      for (int d = size >> 1; d > 64; d >>= 1) {
        __syncthreads();
        const int t = threadIdx.x;
        if (t < n2 / 2) {
          const int i = 2 * t - (t & (d - 1)), j = i + d;
          const Item<Z> a = list_get<Z, T>(sh, i), b = list_get<Z, T>(sh, j);
          if ((i & size) ? in_front<Z>(a, b) : in_front<Z>(b, a)) {
            list_put<Z, T>(sh, i, b);
            list_put<Z, T>(sh, j, a);
          }
        }
      }
      __syncthreads();
      if (mine) {
        e[0] = list_get<Z, T>(sh, i0);
        e[1] = list_get<Z, T>(sh, i0 + 64);
      }
    }
    if (mine) {
      if (size >= 128) {
        const bool swap = (i0 & size) ? in_front<Z>(e[0], e[1]) : in_front<Z>(e[1], e[0]);
        const Item<Z> x = e[0];
        e[0] = swap ? e[1] : e[0];
        e[1] = swap ? x : e[1];
      }
#pragma unroll 1
      for (int d = min(size >> 1, 32); d > 0; d >>= 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = i0 + 64 * h;
          Item<Z> o;
          o.k = __shfl_xor(e[h].k, d);
          o.n = __shfl_xor(e[h].n, d);
          const bool first = ((i & d) == 0) == ((i & size) == 0);      // takes the one in front
          if (first ? in_front<Z>(o, e[h]) : in_front<Z>(e[h], o)) e[h] = o;
        }
      }
    }
  }
  __syncthreads();
  if (mine) {
    list_put<Z, T>(sh, i0, e[0]);
    list_put<Z, T>(sh, i0 + 64, e[1]);
  }
  __syncthreads();
}

// ---- cuts ---------------------------------------------------------------------------------------------------------

template <typename F>
__device__ __forceinline__ F next_up(F v) {      // v not NaN, not +inf
  if constexpr (sizeof(F) == 4) {
    const uint32_t b = __float_as_uint(v);
    return v == 0 ? __uint_as_float(1u) : __uint_as_float(b >> 31 ? b - 1 : b + 1);
  } else {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return v == 0 ? __longlong_as_double(1) : __longlong_as_double((int64_t)(b >> 63 ? b - 1 : b + 1));
  }
}
template <typename F>
__device__ __forceinline__ F round_up(double x) {      // the smallest finite F not below x
  F f = (F)x;
  if ((double)f < x || f == -__builtin_inff()) f = next_up(f);
  return f;
}

template <typename Z>
__device__ __forceinline__ typename Key<Z>::val_t value_of(typename Key<Z>::type k) {
  if constexpr (sizeof(k) == 4)
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
  else
    return __longlong_as_double((int64_t)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}

// What one row's largest logit and parameters say about its elements.
template <typename Z>
struct RowScale {
  typedef typename Key<Z>::val_t F;
  F m;
  bool inf;
  F floor, least;      // up to `floor` weights are 0 in 64 bits (finite: -inf is below it); below `least` min-p drops
  __device__ __forceinline__ RowScale(typename Key<Z>::type key, const RowArgs& a) {
    m = value_of<Z>(key);
    inf = m == __builtin_inff();
    if (inf) m = 0;
    // 2^-1075, which rounds to 0; and float64 logits whose difference overflows, which weigh exp(-inf)
    floor = round_up<F>((double)m - fmin(745.1332191019412 * a.T, 0x1.fffffffffffffp1023));
    // (a weight of at least 1: one that rounds to 1 in 64 bits, as in the kernels that compare weights)
    least = a.M > 0 ? round_up<F>((double)m + a.T * (a.M < 1.0 ? log(a.M) : -0x1p-54)) : floor;
    if (least < floor) least = floor;
  }
};

// What is kept: the elements that do not come behind (v, idx) in the order.
template <typename F>
struct Cut {
  F v;
  int idx;
  __device__ __forceinline__ bool keeps(F z, int i) const { return z > v || (z == v && i <= idx); }
};

// The same, of elements not below `floor`, as one comparison an element: z is kept iff z >= the limit of its 16 bytes, but
// for the 16 bytes that the index splits.
template <typename F>
struct Limit {
  F with, without;      // limits where elements that equal v are kept, and where they are not
  int idx;
  __device__ __forceinline__ Limit(const Cut<F>& c, F floor) : idx(c.idx) {
    const F up = next_up(c.v);
    without = up > floor ? up : floor;
    with = c.idx < 0 || c.v < floor ? without : c.v;
  }
  template <int N>
  __device__ __forceinline__ F of(F (&z)[N], int base) const {
    const bool split = base <= idx && base + N - 1 > idx;
    if (__any(split)) {
      if (split)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (base + j > idx && z[j] < without) z[j] = -__builtin_inff();
    }
    return base > idx ? without : with;
  }
};

// ---- one row by one workgroup of T threads ------------------------------------------------------------------------

template <typename Z, int T>
struct RowSampler {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  static constexpr int N = Chunk<Z>::N, CAP = RowShared<Z, T>::CAP, PB = BINS / T, PS = SEGS / T;
  RowShared<Z, T>& sh;
  RowView<Z> row;
  RowScale<Z> sc;
  RowWeight<F> weight;
  Whole whole;

  // The bin (of the histogram in LDS) where the running sum, which starts at `above`, first reaches the target (or, share, the
  // target times the sum of all), and in sh.above what lies in front of it; -1 if there is none.
  __device__ __forceinline__ int border_bin(unsigned long long above, double& target, bool share) {
    unsigned long long v[PB], mine = 0, total;
#pragma unroll
    for (int e = 0; e < PB; ++e) v[e] = sh.hist[PB * threadIdx.x + e], mine += v[e];
    if (threadIdx.x == 0) sh.which = -1;
    unsigned long long from = above + block_scan<T>(mine, sh.wave_u, total) - mine;
    if (share) target *= (double)(above + total);
#pragma unroll
    for (int e = 0; e < PB; ++e) {
      // (the very first element is kept whatever the target)
      if (v[e] && ((double)from < target || from == above) && (double)(from + v[e]) >= target)
        sh.which = PB * threadIdx.x + e, sh.above = from;
      from += v[e];
    }
    __syncthreads();
    return sh.which;
  }

  // The same for weights in two words; sh.above and sh.above_l hold what the sum starts at.
  __device__ __forceinline__ int border_bin(const TwoWords& two, double& target, bool share) {
    const Mass above = {sh.above, sh.above_l};
    Mass v[PB], mine = {0, 0}, total, from;
#pragma unroll
    for (int e = 0; e < PB; ++e) v[e] = {sh.hist[PB * threadIdx.x + e], sh.hist_l[PB * threadIdx.x + e]}, mine = mine + v[e];
    if (threadIdx.x == 0) sh.which = -1;
    from.h = above.h + block_scan<T>(mine.h, sh.wave_u, total.h) - mine.h;
    from.l = above.l + block_scan<T>(mine.l, sh.wave_u, total.l) - mine.l;
    if (share) target *= two.value(above + total);
#pragma unroll
    for (int e = 0; e < PB; ++e) {
      const Mass to = from + v[e];
      const bool first = from.h == above.h && from.l == above.l;
      if ((v[e].h | v[e].l) && (two.value(from) < target || first) && two.value(to) >= target)
        sh.which = PB * threadIdx.x + e, sh.above = from.h, sh.above_l = from.l;
      from = to;
    }
    __syncthreads();
    return sh.which;
  }

  // The cut behind the last of the n sorted elements of the LDS list with less than the target in front of it.
  template <bool MASS>
  __device__ __forceinline__ Cut<F> sorted_cut(int n, double target, unsigned long long above) {
    Item<Z> e[2];
    unsigned long long q[2] = {0, 0}, sum;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (2 * (int)threadIdx.x + h < n) {
        e[h] = list_get<Z, T>(sh, 2 * threadIdx.x + h);
        q[h] = MASS ? whole(weight(value_of<Z>(e[h].k), true)) : 1ull;
      }
    unsigned long long before = above + block_scan<T>(q[0] + q[1], sh.wave_u, sum) - q[0] - q[1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = 2 * threadIdx.x + h;
      if (i < n && ((double)before < target || i == 0) && (i == n - 1 || (double)(before + q[h]) >= target))
        sh.cut_key = e[h].k, sh.cut_idx = (int)~e[h].n;
      before += q[h];
    }
    __syncthreads();
    const Cut<F> cut = {value_of<Z>(sh.cut_key), sh.cut_idx};
    __syncthreads();
    return cut;
  }

  // The place, by index, where the running sum of the kept weights passes u times the total; sh.seg holds their sums.
  __device__ __forceinline__ int draw(const Cut<F>& cut, double u) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    double v[PS], mine = 0, total;
#pragma unroll
    for (int e = 0; e < PS; ++e) v[e] = sh.seg[PS * threadIdx.x + e], mine += v[e];
    if (threadIdx.x == 0) sh.which = SEGS, sh.last = -1, sh.at = -1, sh.n = -1;
    const double from = block_scan<T>(mine, sh.wave_d, total) - mine, target = u * total;
    double upto = from;
    int first = SEGS, last = -1;
#pragma unroll
    for (int e = 0; e < PS; ++e) {
      upto += v[e];
      if (v[e] > 0) {
        if (upto > target) first = min(first, PS * (int)threadIdx.x + e);
        last = PS * threadIdx.x + e;
      }
    }
    const uint64_t over = __ballot(first < SEGS), any = __ballot(last >= 0);
    if (over && lane == (int)__builtin_ctzll(over)) atomicMin(&sh.which, first);
    if (any && lane == 63 - (int)__builtin_clzll(any)) atomicMax(&sh.last, last);
    __syncthreads();
    const bool to_end = sh.which == SEGS;               // u >= 1, or rounded up to it: the last kept element
    const int s = to_end ? sh.last : sh.which;
    if (s < 0) return -1;                               // nothing is kept (the first element always is)
    if ((int)threadIdx.x == s / PS) {
      upto = from;
#pragma unroll
      for (int e = 0; e < PS; ++e)
        if (e < s % PS) upto += v[e];
      sh.seg_before = upto;
    }
    __syncthreads();
    double before = sh.seg_before;
    const Limit<F> limit(cut, sc.least);
#pragma unroll 1
    for (int r0 = 0; r0 < row.R; r0 += T / 64) {        // a step a wave
      const int r = r0 + wave, step = s * row.R + r;
      const bool in = r < row.R && step < row.steps;
      const int base = in ? chunk_base(row, step) : 0;
      double w[N], t = 0, all;
      int end = -1;                                     // the last kept element so far
      if (in) {
        Chunk<Z> q;
        F z[N];
        load_chunk<Z>(q, row, step);
        chunk_values<Z>(z, q, row, step);
        const F lim = limit.template of<N>(z, base);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          w[j] = weight(z[j], z[j] >= lim);
          if (w[j] > 0) end = base + j;
          t += w[j];
        }
      }
      const double upto = before + block_scan<T>(t, sh.wave_d, all);
      const uint64_t who = to_end ? 0 : __ballot(t > 0 && upto > target);
      if (who && lane == (int)__builtin_ctzll(who)) {
        double c = upto - t;
        int pick = -1;
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (w[j] > 0 && !(pick >= 0 && c > target)) c += w[j], pick = base + j;
        atomicMin((unsigned int*)&sh.at, (unsigned int)pick);      // (-1 is the largest)
      }
      const uint64_t some = __ballot(end >= 0);
      if (some && lane == 63 - (int)__builtin_clzll(some)) atomicMax(&sh.n, end);
      __syncthreads();
      if (sh.at >= 0) break;
      before += all;
    }
    return sh.at >= 0 ? sh.at : sh.n;
  }
};

// ---- launches -----------------------------------------------------------------------------------------------------

struct Geometry {
  int V, steps, R, segs, per_seg;      // per_seg: groups a segment (a power of two)
  int most, alone;                     // top-k up to this many is taken from the list: with top-p, by itself
};

template <typename Z>
Geometry geometry(int V, int64_t rows, const SampleArgs& a) {
  constexpr int N = Chunk<Z>::N;
  Geometry g;
  g.V = V;
  g.steps = (int)(((int64_t)V + 64 * N - 1) / (64 * N));
  // segments of up to 4 steps where the machine has work enough without shorter ones
  g.R = std::max((g.steps + SEGS - 1) / SEGS, rows * g.steps >= 16384 ? std::max(1, std::min(4, g.steps / 64)) : 1);
  g.segs = (g.steps + g.R - 1) / g.R;
  // few groups while they do (every workgroup reads them: 1 row of 131072 bfloat16, top-k 50: 24 us with 1024, 32 with 4096;
  // but 104 us where 1024 do not bound k)
  for (int limit = FEW_GROUPS; limit <= GROUPS; limit += GROUPS - FEW_GROUPS) {
    g.per_seg = 64;
    while (g.per_seg * g.segs > limit) g.per_seg /= 2;
    // the k-th largest of n groups' maxima has about -n ln(1 - k / n) elements at or above it
    const int groups = g.per_seg * g.segs;
    g.most = std::min(groups - groups / 128, (int)(groups * (1.0 - exp(-0.92 * LIST_CAP / groups))));
    const bool windows = !a.top_p && a.top_p_all >= 1.0 && (rows <= 64 || a.top_k_all > FEW_GROUPS);      // do without the list
    if (!a.top_k && (a.top_k_all >= V || a.top_k_all <= g.most || windows)) break;
  }
  // few rows, top-k alone: a list that is not short keeps the row's one workgroup busy longer than the windows' launches take (1
  // row of 131072 float32, top-k 900: 39 us against 25, top-k 190: 28 against 25; 128 rows, top-k 900: 58 us against 70)
  g.alone = rows <= 64 ? std::min(g.most, 128) : g.most;
  return g;
}

// A row's part of the workspace.
template <typename Z>
struct RowWork {
  typedef typename Key<Z>::type K;
  K maxima[GROUPS];
  unsigned long long counts[COUNTS];              // number << 33 + sum of the places within the bin
  double seg[SEGS], above[SEGS], total[SEGS];     // what is kept for certain; that before min-p; all
  K key[LIST_CAP];
  uint32_t idx[LIST_CAP];
  K top;                                          // the largest logit (rows that are listed or summed)
  int n;                                          // elements that asked for a place in the list
  int first, last;                                // window: bins; first > last: none was found
  int before;                                     // top-k: elements in front of the window
};

enum Path { BY_MAX, LIST, WINDOW, PLAIN, SLOW };

__device__ __forceinline__ Path row_path(const RowArgs& a, const Geometry& g) {
  if (!(a.T > 0.0)) return BY_MAX;
  if (a.k) return a.k <= (a.P < 1.0 ? g.most : g.alone) ? LIST : a.P < 1.0 ? SLOW : WINDOW;
  return a.P < 1.0 ? WINDOW : PLAIN;
}

// the part of a row that wave number `wave` of `waves` owns
template <typename Z>
__device__ __forceinline__ RowView<Z> row_part(const Z* p, const Geometry& g, int wave, int waves, bool inf) {
  return {p, g.V, g.steps, g.R, wave, waves, inf};
}

// a thread's PER of the n keys of the groups' maxima, all loads under way at a time; 0 behind them
template <int T, int PER, typename K>
__device__ __forceinline__ void load_maxima(K (&key)[PER], const K* maxima, int n) {
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = maxima[min(i * T + (int)threadIdx.x, n - 1)];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = i * T + (int)threadIdx.x < n ? key[i] : (K)0;
}
template <int PER, typename K>
__device__ __forceinline__ K largest_of(const K (&key)[PER]) {
  K m = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) m = key[i] > m ? key[i] : m;
  return m;
}

// the largest key of the groups' maxima, in every thread of a workgroup of T threads
template <int T, typename K>
__device__ __forceinline__ K largest(const K* maxima, int n, K* buf) {
  K m;
  if (n <= FEW_GROUPS) {
    K key[FEW_GROUPS / T];
    load_maxima<T>(key, maxima, n);
    m = largest_of(key);
  } else {
    K key[GROUPS / T];
    load_maxima<T>(key, maxima, n);
    m = largest_of(key);
  }
  m = wave_max(m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = m;
  __syncthreads();
  m = buf[0];
#pragma unroll
  for (int i = 1; i < T / 64; ++i) m = buf[i] > m ? buf[i] : m;
  return m;
}

template <typename Z>
__global__ __launch_bounds__(TB) void row_maxima_kernel(const Z* __restrict__ logits, int64_t ld, Geometry g,
                                                        RowWork<Z>* __restrict__ work) {
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  RowWork<Z>& w = work[blockIdx.y];
  const int lane = threadIdx.x & 63, wide = 64 / g.per_seg;
  if (blockIdx.x == 0 && threadIdx.x == 0) w.n = 0, w.first = 1, w.last = 0;
  for (int i = blockIdx.x * TB + threadIdx.x; i < COUNTS; i += gridDim.x * TB) w.counts[i] = 0;
  F mine = -__builtin_inff();
  walk<Z>(row_part(logits + (int64_t)blockIdx.y * ld, g, blockIdx.x * TW + (threadIdx.x >> 6), gridDim.x * TW, false),
          [&](F(&v)[N], int) {
#pragma unroll
            for (int j = 0; j < N; ++j) mine = v[j] > mine ? v[j] : mine;
          },
          [&](int s) {
            for (int d = 1; d < wide; d <<= 1) {
              const F o = __shfl_xor(mine, d);
              mine = o > mine ? o : mine;
            }
            if (lane % wide == 0) w.maxima[s * g.per_seg + lane / wide] = Key<Z>::of(mine);
            mine = -__builtin_inff();
          });
}

// Elements of a wave on their way into the row's list: gathered in LDS, so that the list's counter, which every wave of the
// row adds to, is asked once a wave and not once a step of its walk.
template <typename Z>
struct WaveList {
  typedef typename Key<Z>::type K;
  static constexpr int N = Chunk<Z>::N, CAP = 64 * N;      // a step's at most
  struct Room {
    K key[TW][CAP];
    uint32_t idx[TW][CAP];
  };
  Room& room;
  RowWork<Z>& w;
  int n;
  __device__ __forceinline__ WaveList(Room& r, RowWork<Z>& work) : room(r), w(work), n(0) {}

  // the `mask`ed ones of the lanes' 16 bytes
  __device__ __forceinline__ void add(const typename Key<Z>::val_t (&v)[N], int base, uint32_t mask) {
    const int c = __popc(mask), upto = wave_scan(c), all = from_lane(upto, 63), wave = threadIdx.x >> 6;
    if (n + all > CAP) flush();
    int at = n + upto - c;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (mask >> j & 1) room.key[wave][at] = Key<Z>::of(v[j]), room.idx[wave][at++] = (uint32_t)(base + j);
    n += all;
  }
  __device__ __forceinline__ void flush() {
    if (n == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int at = 0;
    if (lane == 0) at = atomicAdd(&w.n, n);
    at = from_lane(at, 0);
    for (int i = lane; i < n; i += 64)
      if (at + i < LIST_CAP) w.key[at + i] = room.key[wave][i], w.idx[at + i] = room.idx[wave][i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    n = 0;
  }
};

template <typename Z>
__global__ __launch_bounds__(TB) void row_collect_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args, Geometry g,
                                                         RowWork<Z>* __restrict__ work, int64_t row0) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  __shared__ K buf[TW];
  __shared__ uint64_t counts[2][TW];
  __shared__ typename WaveList<Z>::Room room;
  RowWork<Z>& w = work[blockIdx.y];
  const RowArgs a = row_args(args, row0 + blockIdx.y, g.V);
  if (row_path(a, g) != LIST) return;
  const int groups = g.segs * g.per_seg;
  const K top = largest<TB>(w.maxima, groups, buf);
  if (blockIdx.x == 0 && threadIdx.x == 0) w.top = top;
  const RowScale<Z> sc(top, a);
  K bound = 0;
  if (a.k <= groups) {      // the k-th largest of the maxima, its upper 16 (64-bit keys: 24) bits, two at a time
    constexpr int PER = GROUPS / TB, LEAST = FEW_GROUPS / TB;
    int per = LEAST;                 // a thread's keys
    K key[PER];
    if (groups <= FEW_GROUPS) {
      K few[LEAST];
      load_maxima<TB>(few, w.maxima, groups);
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = i < LEAST ? few[i] : (K)0;
    } else {
      // where few are asked for, groups are joined to as many as bound k to a few elements more
      load_maxima<TB>(key, w.maxima, groups);
      per = PER;
#pragma unroll
      for (int h = PER / 2; h >= LEAST; h /= 2)
        if (6 * a.k <= h * TB) {
          per = h;
#pragma unroll
          for (int i = 0; i < h; ++i) key[i] = key[i + h] > key[i] ? key[i + h] : key[i];
        }
    }
    if (sc.inf)
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = Key<Z>::of(finite(value_of<Z>(key[i]), true));
    constexpr int BITS = 8 * (int)sizeof(K), END = BITS - (BITS == 64 ? 24 : 16);
    int turn = 0;
#pragma unroll 1
    for (int bit = BITS - 2; bit >= END; bit -= 2, turn ^= 1) {
      uint32_t c[3] = {0, 0, 0};
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < per)
#pragma unroll
          for (int j = 0; j < 3; ++j) c[j] += __popcll(__ballot(key[i] >= (bound | (K)(j + 1) << bit)));
      if ((threadIdx.x & 63) == 0) counts[turn][threadIdx.x >> 6] = c[0] | (uint64_t)c[1] << 20 | (uint64_t)c[2] << 40;
      __syncthreads();
      uint64_t all = 0;
#pragma unroll
      for (int i = 0; i < TW; ++i) all += counts[turn][i];
      K digit = 0;
#pragma unroll
      for (int j = 0; j < 3; ++j) digit += (int)(all >> (20 * j) & 0xFFFFF) >= a.k;
      bound |= digit << bit;
    }
  }
  const F lim = bound > Key<Z>::of(sc.floor) ? value_of<Z>(bound) : sc.floor;
  WaveList<Z> list(room, w);
  walk<Z>(row_part(logits + (int64_t)blockIdx.y * ld, g, blockIdx.x * TW + (threadIdx.x >> 6), gridDim.x * TW, sc.inf),
          [&](F(&v)[N], int base) {
            uint32_t mask = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) mask |= (uint32_t)(v[j] >= lim) << j;
            if (__any(mask != 0)) list.add(v, base, mask);
          },
          NoEnd());
  list.flush();
}

// Bins over what matters of a row cut by top-p: what lies further below the maximum than ln(V / (1 - P)) weighs less than
// 1 - P of the total, and five units more make what lies behind the bins weigh nothing against a bin.  Top-k alone: bins down
// to what weighs 1e-9 / V of the total, where the k-th element mostly is.
template <typename F>
__device__ __forceinline__ F bin_slope(const RowArgs& a, int V) {
  return (F)fmin((double)COUNTS / (a.T * (log((double)V / (a.k ? 1e-9 : 1.0 - a.P)) + 5.0)), 1e38);
}
// Places within a bin are counted in units of 2^-place_bits: V of them stay below 2^33.
__device__ __forceinline__ int place_bits(int V) { return min(10, 1 + (int)__builtin_clz(V)); }

// The bins the border of top-p must lie in.  With step = width of a bin in units of T, an element at place f of bin b weighs
// e^(-(b + f) step), and e^(-y) lies between 1 - y and 1 - y + y^2 / 2; places are known to their unit and to the roundings of
// the bin number (below 4096 2^-22 of a bin).
__device__ __forceinline__ void find_window(const unsigned long long* counts, int beyond, double slope, const RowArgs& a, int V,
                                            double* buf, int* found) {
  constexpr int PER = COUNTS / RT;
  const double step = 1.0 / (slope * a.T), unit = ldexp(1.0, -place_bits(V));
  double least[PER], most[PER], sl = 0, sm = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int bin = PER * threadIdx.x + i;
    const double n = (double)(counts[bin] >> 33), f = (double)(counts[bin] & 0x1FFFFFFFFull) * unit;
    const double low = fmax(f - 0.001 * n, 0.0), high = f + (unit + 0.001) * n, e = exp(-(double)bin * step);
    least[i] = e * fmax(n - step * high, 0.0);
    most[i] = e * (n - step * low + 0.5 * step * step * high);
    sl += least[i];
    sm += most[i];
  }
  double total_least, total_most;
  double ul = block_scan<RT>(sl, buf, total_least) - sl;
  double um = block_scan<RT>(sm, buf, total_most) - sm;
  total_most += (double)beyond * exp(-((double)COUNTS - 0.001) * step);
  if (threadIdx.x == 0) found[0] = found[1] = COUNTS;
  __syncthreads();
  const double early = a.P * total_least * (1 - 1e-9), late = a.P * total_most * (1 + 1e-9);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (um < early && um + most[i] >= early) atomicMin(&found[0], PER * (int)threadIdx.x + i);
    if (ul < late && ul + least[i] >= late) atomicMin(&found[1], PER * (int)threadIdx.x + i);
    ul += least[i];
    um += most[i];
  }
  __syncthreads();
}

// The bin of the k-th element, and the number of elements in front of it.
__device__ __forceinline__ void find_kth(const unsigned long long* counts, int k, double* buf, int* found) {
  constexpr int PER = COUNTS / RT;
  int n[PER], mine = 0;
  double total;
#pragma unroll
  for (int i = 0; i < PER; ++i) n[i] = (int)(counts[PER * threadIdx.x + i] >> 33), mine += n[i];
  int before = (int)(block_scan<RT>((double)mine, buf, total)) - mine;
  if (threadIdx.x == 0) found[0] = found[1] = COUNTS, found[2] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before < k && before + n[i] >= k) found[0] = found[1] = PER * threadIdx.x + i, found[2] = before;
    before += n[i];
  }
  __syncthreads();
}

// counts; where a row has one workgroup, its window too (`n` of the row's work holds, meanwhile, the elements behind the bins)
template <typename Z>
__global__ __launch_bounds__(RT) void row_counts_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args, Geometry g,
                                                        RowWork<Z>* __restrict__ work, int64_t row0) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  __shared__ unsigned long long counts[COUNTS + 64];      // the last 64: elements that are not counted
  __shared__ K buf[RW];
  __shared__ double dbuf[RW];
  __shared__ int beyond, found[3];
  RowWork<Z>& w = work[blockIdx.y];
  const RowArgs a = row_args(args, row0 + blockIdx.y, g.V);
  if (row_path(a, g) != WINDOW) return;
  for (int i = threadIdx.x; i < COUNTS; i += RT) counts[i] = 0;
  if (threadIdx.x == 0) beyond = 0;
  const K top = largest<RT>(w.maxima, g.segs * g.per_seg, buf);      // (its barriers cover the zeros)
  if (blockIdx.x == 0 && threadIdx.x == 0) w.top = top;
  const RowScale<Z> sc(top, a);
  const F slope = bin_slope<F>(a, g.V), units = (F)(1 << place_bits(g.V));
  int behind = 0;
  const int none = COUNTS + (int)(threadIdx.x & 63);
  walk<Z>(row_part(logits + (int64_t)blockIdx.y * ld, g, blockIdx.x * RW + (threadIdx.x >> 6), gridDim.x * RW, sc.inf),
          [&](F(&v)[N], int) {
            int bin[N];
            uint32_t place[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {      // without branches: the chains overlap
              const F x = (sc.m - v[j]) * slope;
              const bool in = x < F(COUNTS), is = v[j] >= sc.floor;
              const int b = (int)x;
              place[j] = (uint32_t)((x - (F)b) * units);
              bin[j] = in && is ? b : none;
              behind += is && !in;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) atomicAdd(&counts[bin[j]], (1ull << 33) | place[j]);
          },
          NoEnd());
  behind = wave_sum(behind);
  if ((threadIdx.x & 63) == 0 && behind) atomicAdd(&beyond, behind);
  __syncthreads();
  if (gridDim.x == 1) {
    if (a.k)
      find_kth(counts, a.k, dbuf, found);
    else
      find_window(counts, beyond, (double)slope, a, g.V, dbuf, found);
    if (threadIdx.x == 0) w.first = found[0], w.last = found[1] < COUNTS ? found[1] : -1, w.before = a.k ? found[2] : 0;
    return;
  }
  for (int i = threadIdx.x; i < COUNTS; i += RT)
    if (counts[i]) atomicAdd(&w.counts[i], counts[i]);
  if (threadIdx.x == 0 && beyond) atomicAdd(&w.n, beyond);
}

template <typename Z>
__global__ __launch_bounds__(RT) void row_window_kernel(SampleArgs args, Geometry g, RowWork<Z>* __restrict__ work, int64_t row0) {
  typedef typename Key<Z>::val_t F;
  __shared__ double dbuf[RW];
  __shared__ int found[3];
  RowWork<Z>& w = work[blockIdx.x];
  const RowArgs a = row_args(args, row0 + blockIdx.x, g.V);
  if (row_path(a, g) != WINDOW) return;
  if (a.k)
    find_kth(w.counts, a.k, dbuf, found);
  else
    find_window(w.counts, w.n, (double)bin_slope<F>(a, g.V), a, g.V, dbuf, found);
  if (threadIdx.x == 0)
    w.first = found[0], w.last = found[1] < COUNTS ? found[1] : -1, w.before = a.k ? found[2] : 0, w.n = 0;
}

// The sums of a row that top-p cuts: MIN_P where the elements min-p drops are summed apart.
template <typename Z, bool MIN_P>
__device__ __forceinline__ void window_sums(const RowView<Z>& row, const RowScale<Z>& sc, const RowArgs& a,
                                            const RowWeight<typename Key<Z>::val_t>& weight, RowWork<Z>& w,
                                            typename WaveList<Z>::Room& room) {
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  const F slope = bin_slope<F>(a, row.V), top = F(w.first), bottom = F(w.last + 1);
  double sum = 0, above = 0, total = 0;
  WaveList<Z> list(room, w);
  walk<Z>(row,
          [&](F(&v)[N], int base) {
            uint32_t mask = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const F x = (sc.m - v[j]) * slope;
              const bool is = v[j] >= sc.floor;
              const double t = weight(v[j], is), c = x < top ? t : 0.0;
              total += t;
              above += c;
              if (MIN_P) sum += v[j] >= sc.least ? c : 0.0;
              mask |= (uint32_t)(is && x >= top && x < bottom) << j;
            }
            if (__any(mask != 0)) list.add(v, base, mask);
          },
          [&](int s) {
            total = wave_sum(total);
            above = wave_sum(above);
            if (MIN_P) sum = wave_sum(sum);
            if ((threadIdx.x & 63) == 0) w.seg[s] = MIN_P ? sum : above, w.above[s] = above, w.total[s] = total;
            sum = above = total = 0;
          });
  list.flush();
}

template <typename Z>
__global__ __launch_bounds__(TB) void row_sums_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args, Geometry g,
                                                      RowWork<Z>* __restrict__ work, int64_t row0) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  __shared__ K buf[TW];
  __shared__ double pow2[32];
  __shared__ typename WaveList<Z>::Room room;
  RowWork<Z>& w = work[blockIdx.y];
  const RowArgs a = row_args(args, row0 + blockIdx.y, g.V);
  const Path path = row_path(a, g);
  if ((path != PLAIN && path != WINDOW) || (path == WINDOW && w.first > w.last)) return;
  fill_pow2(pow2);
  // (a barrier covers pow2 either way)
  const K top = path == WINDOW ? w.top : largest<TB>(w.maxima, g.segs * g.per_seg, buf);
  if (path == WINDOW)
    __syncthreads();
  else if (blockIdx.x == 0 && threadIdx.x == 0)
    w.top = top;
  const RowScale<Z> sc(top, a);
  const RowWeight<F> weight(sc.m, a.T, pow2);
  const RowView<Z> row = row_part(logits + (int64_t)blockIdx.y * ld, g, blockIdx.x * TW + (threadIdx.x >> 6), gridDim.x * TW, sc.inf);
  if (path == PLAIN) {
    double sum = 0;
    walk<Z>(row,
            [&](F(&v)[N], int) {
#pragma unroll
              for (int j = 0; j < N; ++j) sum += weight(v[j], v[j] >= sc.least);
            },
            [&](int s) {
              sum = wave_sum(sum);
              if ((threadIdx.x & 63) == 0) w.seg[s] = sum;
              sum = 0;
            });
  } else if (a.M > 0) {
    window_sums<Z, true>(row, sc, a, weight, w, room);
  } else {
    window_sums<Z, false>(row, sc, a, weight, w, room);
  }
}

// Cuts of a row from its list of c <= LIST_CAP elements (in the workspace).
template <typename Z>
struct ListCut : RowSampler<Z, TB> {
  typedef RowSampler<Z, TB> Base;
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  using Base::sh;
  using Base::weight;
  using Base::whole;
  static constexpr int SIDE = 1024;      // histogram words from here on lie behind the list
  const RowWork<Z>& w;
  int c;
  __device__ __forceinline__ ListCut(const Base& b, const RowWork<Z>& work) : Base(b), w(work), c(work.n) {}

  // f(key, index) of a thread's share of the list, eight elements under way at a time
  template <typename Fn>
  __device__ __forceinline__ void each(Fn f) {
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < c; i0 += 8 * TB) {
      K k[8];
      uint32_t at[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = min(i0 + j * TB, c - 1);
        k[j] = w.key[i], at[j] = w.idx[i];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j * TB < c) f(k[j], at[j]);
    }
  }

  // f(element, what it counts for) of the n (at most TB) elements in LDS, in every thread, eight under way at a time (they are
  // filled up to a multiple of eight with elements that sort last and count for nothing)
  template <typename Fn>
  __device__ __forceinline__ void all(int n, Fn f) {
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += 8) {
      Item<Z> o[8];
      unsigned long long q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = list_get<Z, TB>(sh, j0 + j), q[j] = sh.hist[SIDE + j0 + j];
#pragma unroll
      for (int j = 0; j < 8; ++j) f(o[j], q[j]);
    }
  }
  static __device__ __forceinline__ bool fills(int i, int n) { return i < ((n + 7) & ~7); }

  // The last of the n elements in LDS, a thread an element (in: this thread has one), that has less than `target` in front of
  // it, or the first of them where `first` says so; false where there is none.
  __device__ __forceinline__ bool last_kept(Cut<F>& cut, const Item<Z>& e, bool in, int n, double target, unsigned long long above,
                                            bool first) {
    int rank = 0;
    unsigned long long before = above, kept;
    all(n, [&](const Item<Z>& o, unsigned long long q) {
      const bool front = in_front<Z>(o, e);
      rank += front;
      before += front ? q : 0;
    });
    const bool keep = in && ((double)before < target || (rank == 0 && first));
    block_scan<TB>((unsigned long long)keep, sh.wave_u, kept);
    if (keep && rank == (int)kept - 1) sh.cut_key = e.k, sh.cut_idx = (int)~e.n;
    __syncthreads();
    if (kept == 0) return false;
    cut = {value_of<Z>(sh.cut_key), sh.cut_idx};
    __syncthreads();
    return true;
  }

  // cut_at of a list of at most TB elements, a thread an element: what lies in front of it is counted over all others.
  template <bool MASS>
  __device__ __forceinline__ bool cut_few(Cut<F>& cut, double target, bool share, unsigned long long above, bool first) {
    static_assert(sizeof(sh.list) <= SIDE * sizeof(sh.hist[0]) && SIDE + TB <= BINS, "the list and what its elements count for");
    const int i = threadIdx.x;
    Item<Z> e = {0, 0};
    unsigned long long q = 0, sum;
    bool in = false;
    if (i < c) {
      e = {w.key[i], ~w.idx[i]};
      in = cut.keeps(value_of<Z>(e.k), (int)~e.n);
    }
    __syncthreads();
    if (in) q = MASS ? whole(weight(value_of<Z>(e.k), true)) : 1ull;
    if (fills(i, c)) list_put<Z, TB>(sh, i, in ? e : Item<Z>{0, 0}), sh.hist[SIDE + i] = q;
    block_scan<TB>(q, sh.wave_u, sum);               // (its barriers cover the list)
    if (share) target *= (double)(above + sum);
    // (the very first element is kept whatever the target)
    return last_kept(cut, e, in, c, target, above, first) && (double)(above + sum) >= target;
  }

  // The cut behind the last element with less than `target` in front of it, of the list's elements that `cut` keeps: in
  // number, of which `above` lie in front of all of them, or, MASS, in weight (units of 2^-48; share: target is a share of
  // theirs).  first: nothing lies in front of the list, so that its first element is kept whatever the target.  False where
  // the list does not hold it.
  template <bool MASS>
  __device__ __forceinline__ bool cut_at(Cut<F>& cut, double target, bool share, unsigned long long above, bool first) {
    if (!first && !((double)above < target)) return false;
    if (c <= TB) return cut_few<MASS>(cut, target, share, above, first);
    K lo = ~(K)0, hi = 0;
    each([&](K k, uint32_t at) {
      if (cut.keeps(value_of<Z>(k), (int)at)) lo = k < lo ? k : lo, hi = k > hi ? k : hi;
    });
    block_range<TB>(lo, hi, sh.wave_lo, sh.wave_hi);
#pragma unroll 1
    for (;;) {
      __syncthreads();
      for (int i = threadIdx.x; i < BINS; i += TB) sh.hist[i] = 0;
      if (threadIdx.x == 0) sh.n = 0;
      __syncthreads();
      int shift = 0;
      while (((hi - lo) >> shift) >= (K)BINS) ++shift;
      each([&](K k, uint32_t at) {
        if (k >= lo && k <= hi && cut.keeps(value_of<Z>(k), (int)at))
          atomicAdd(&sh.hist[(int)((hi - k) >> shift)], MASS ? whole(weight(value_of<Z>(k), true)) : 1ull);
      });
      __syncthreads();
      const int bin = this->border_bin(above, target, share);
      share = false;
      if (bin < 0) return false;
      above = sh.above;
      const K top = hi - ((K)bin << shift), span = ((K)1 << shift) - 1, bottom = top - lo > span ? top - span : lo;
      __syncthreads();
      K l = ~(K)0, h = 0;
      each([&](K k, uint32_t at) {
        if (k >= bottom && k <= top && cut.keeps(value_of<Z>(k), (int)at)) {
          const int place = atomicAdd(&sh.n, 1);
          if (place < Base::CAP) list_put<Z, TB>(sh, place, {k, ~at});
          l = k < l ? k : l;
          h = k > h ? k : h;
        }
      });
      block_range<TB>(l, h, sh.wave_lo, sh.wave_hi);
      if (sh.n <= Base::CAP) break;
      if (l == h) return false;
      lo = l, hi = h;
    }
    const int n = sh.n, i = threadIdx.x;
    if (n <= TB) {
      Item<Z> e = {0, 0};
      if (i < n) e = list_get<Z, TB>(sh, i);
      if (fills(i, n)) {
        sh.hist[SIDE + i] = i >= n ? 0 : MASS ? whole(weight(value_of<Z>(e.k), true)) : 1ull;
        if (i >= n) list_put<Z, TB>(sh, i, e);
      }
      __syncthreads();
      return last_kept(cut, e, i < n, n, target, above, true);
    }
    list_sort<Z, TB>(sh, n);
    cut = this->template sorted_cut<MASS>(n, target, above);
    return true;
  }

  // The label of a list of at most TB elements that holds the k first, a thread an element: its place in the order, and then
  // its place by index, is counted against all others (one row, top-k 50: a sort and the segments' sums take as long as the
  // whole of this).
  __device__ __forceinline__ int draw_few(const RowArgs& a) {
    const int i = threadIdx.x;
    Item<Z> e = {0, 0};
    double wt = 0;
    unsigned long long q = 0, sum;
    if (i == 0) sh.which = 0x7FFFFFFF, sh.last = -1;
    if (i < c) e = {w.key[i], ~w.idx[i]};
    __syncthreads();                                 // (covers the weights' table)
    if (i < c) {
      wt = weight(value_of<Z>(e.k), true);
      q = whole(wt);
    }
    if (fills(i, c)) list_put<Z, TB>(sh, i, e), sh.hist[SIDE + i] = q;
    __syncthreads();
    int rank = 0;
    unsigned long long before = 0, upto = 0, total = 0;
    all(c, [&](const Item<Z>& o, unsigned long long n) {
      const bool front = in_front<Z>(o, e);
      rank += front;
      before += front ? n : 0;
    });
    bool keep = i < c && rank < a.k;
    if (a.P < 1.0) {
      block_scan<TB>(keep ? q : 0, sh.wave_u, sum);
      keep = keep && (rank == 0 || (double)before < a.P * (double)sum);
    }
    keep = keep && value_of<Z>(e.k) >= this->sc.least;
    __syncthreads();
    if (fills(i, c)) sh.hist[SIDE + i] = keep ? q : 0;
    __syncthreads();
    const int mine = (int)~e.n;
    all(c, [&](const Item<Z>& o, unsigned long long n) {
      total += n;
      upto += (int)~o.n <= mine ? n : 0;
    });
    const double target = a.u * (double)total;
    if (keep && wt > 0) {
      if ((double)upto > target || !(target > 0)) atomicMin(&sh.which, mine);
      atomicMax(&sh.last, mine);
    }
    __syncthreads();
    return sh.which == 0x7FFFFFFF ? sh.last : sh.which;
  }

  // top-k and top-p of a list that holds the k first elements.  A list of just k needs its cut as well: the draw reads the row
  // again, where the elements that are not listed stand too (a list of fewer holds everything that weighs anything).
  __device__ __forceinline__ bool top_cut(Cut<F>& cut, const RowArgs& a) {
    if (c >= a.k && !cut_at<false>(cut, (double)a.k, false, 0, true)) return false;
    return !(a.P < 1.0) || cut_at<true>(cut, a.P, true, 0, true);
  }

  // the list's elements that `cut` and min-p keep join their segments' sums
  __device__ __forceinline__ void join_segments(const Cut<F>& cut) {
    const int span = this->row.R * 64 * Base::N;
    __syncthreads();
    for (int i = threadIdx.x; i < SEGS; i += TB) sh.hist[i] = 0;
    __syncthreads();
    each([&](K k, uint32_t at) {
      const F v = value_of<Z>(k);
      if (v >= this->sc.least && cut.keeps(v, (int)at)) {
        // (u = 0 draws the first element that weighs anything: its segment must not look empty)
        const double wt = weight(v, true);
        const unsigned long long q = whole(wt);
        if (wt > 0) atomicAdd(&sh.hist[at / (uint32_t)span], q ? q : 1);
      }
    });
    __syncthreads();
    for (int i = threadIdx.x; i < SEGS; i += TB) sh.seg[i] += (double)sh.hist[i] / Whole::FIXED;
  }
};

constexpr int64_t NOT_YET = -2;      // the label of a row that `slow` has to do

template <typename Z>
__global__ __launch_bounds__(TB) void row_finish_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args, Geometry g,
                                                        RowWork<Z>* __restrict__ work, int64_t* __restrict__ label, int64_t row0) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  __shared__ RowShared<Z, TB> sh;
  const int64_t i = row0 + blockIdx.x;
  const RowWork<Z>& w = work[blockIdx.x];
  const RowArgs a = row_args(args, i, g.V);
  const Path path = row_path(a, g);
  const Z* p = logits + (int64_t)blockIdx.x * ld;
  fill_pow2(sh.pow2);
  for (int s = threadIdx.x; s < SEGS; s += TB) sh.seg[s] = (path == PLAIN || path == WINDOW) && s < g.segs ? w.seg[s] : 0.0;
  const int groups = g.segs * g.per_seg;
  const K top = path == BY_MAX || path == SLOW ? largest<TB>(w.maxima, groups, sh.wave_hi) : w.top;
  if (!(value_of<Z>(top) > -__builtin_inff())) {
    if (threadIdx.x == 0) label[i] = -1;
    return;
  }
  int64_t pick = NOT_YET;
  if (path == BY_MAX) {
    // the first segment with the maximum, by one wave
    if (threadIdx.x == 0) sh.which = groups, sh.at = g.V;
    __syncthreads();
    for (int j = threadIdx.x; j < groups; j += TB)
      if (w.maxima[j] == top) atomicMin(&sh.which, j);
    __syncthreads();
    const int s = sh.which / g.per_seg;
    const F m = value_of<Z>(top);
    const RowView<Z> row = row_part(p, g, 0, 1, false);
    if (threadIdx.x < 64)
#pragma unroll 1
      for (int r = 0; r < g.R && s * g.R + r < g.steps; ++r) {
        Chunk<Z> q;
        F v[N];
        load_chunk<Z>(q, row, s * g.R + r);
        chunk_values<Z>(v, q, row, s * g.R + r);
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (v[j] == m) atomicMin(&sh.at, chunk_base(row, s * g.R + r) + j);
      }
    __syncthreads();
    pick = sh.at;
  } else if (path != SLOW) {
    const RowScale<Z> sc(top, a);
    const RowSampler<Z, TB> sampler = {sh, row_part(p, g, 0, 1, sc.inf), sc, RowWeight<F>(sc.m, a.T, sh.pow2), Whole()};
    ListCut<Z> row(sampler, w);
    Cut<F> cut = {-__builtin_inff(), -1};
    bool good = path == PLAIN;
    if (path == LIST && row.c > 0 && row.c <= TB) {
      pick = row.draw_few(a);
    } else if (row.c > 0 && row.c <= LIST_CAP) {
      if (path == LIST) good = row.top_cut(cut, a);
      if (path == WINDOW && w.first <= w.last && a.k) {
        good = row.template cut_at<false>(cut, (double)a.k, false, (unsigned long long)w.before, w.before == 0);
      } else if (path == WINDOW && w.first <= w.last) {
        double above = 0, total = 0, all_above, all;
        for (int s = threadIdx.x; s < g.segs; s += TB) above += w.above[s], total += w.total[s];
        block_scan<TB>(above, sh.wave_d, all_above);
        block_scan<TB>(total, sh.wave_d, all);
        good = row.template cut_at<true>(cut, (a.P * all - all_above) * Whole::FIXED, false, 0, all_above == 0);
      }
    }
    if (good) {
      if (path != PLAIN) row.join_segments(cut);
      pick = row.draw(cut, a.u);
    }
  }
  if (threadIdx.x == 0) label[i] = pick;
}

// ---- rows that the lists do not hold ------------------------------------------------------------------------------

template <typename Z>
struct RowCut : RowSampler<Z, RT> {
  typedef RowSampler<Z, RT> Base;
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  static constexpr int N = Base::N;
  using Base::row;
  using Base::sh;
  using Base::weight;
  using Base::whole;
  __device__ __forceinline__ explicit RowCut(const Base& b) : Base(b) {}

  // place of the n-th (from 1) kept element that equals t
  __device__ __forceinline__ int nth_tie(const Cut<F>& cut, F t, int n) {
    __syncthreads();
    for (int i = threadIdx.x; i < SEGS; i += RT) sh.count[i] = 0;
    __syncthreads();
    int c = 0;
    walk<Z>(row,
            [&](F(&v)[N], int base) {
#pragma unroll
              for (int j = 0; j < N; ++j) c += v[j] == t && cut.keeps(t, base + j);
            },
            [&](int s) {
              c = wave_sum(c);
              if ((threadIdx.x & 63) == 0) sh.count[s] = c;
              c = 0;
            });
    __syncthreads();
    const int mine = sh.count[threadIdx.x];      // (as many segments as threads)
    unsigned long long total;
    const int upto = (int)block_scan<RT>((unsigned long long)mine, sh.wave_u, total);
    if (upto >= n && upto - mine < n) sh.which = threadIdx.x, sh.at = upto - mine;
    __syncthreads();
    const int s = sh.which;
    int before = sh.at;
    __syncthreads();
    if (threadIdx.x < 64)
#pragma unroll 1
      for (int r = 0; r < row.R && s * row.R + r < row.steps; ++r) {
        Chunk<Z> q;
        F v[N];
        load_chunk<Z>(q, row, s * row.R + r);
        chunk_values<Z>(v, q, row, s * row.R + r);
        const int base = chunk_base(row, s * row.R + r);
        int mine = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) mine += v[j] == t && cut.keeps(t, base + j);
        const int upto = wave_scan(mine);
        int k = before + upto - mine;
        if (k < n && k + mine >= n)
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (v[j] == t && cut.keeps(t, base + j) && ++k == n) sh.at = base + j;
        before += from_lane(upto, 63);
      }
    __syncthreads();
    return sh.at;
  }

  // The cut of top-k (`target` elements) or, MASS, of top-p (the share `target` of the weight) among the elements `cut` keeps.
  template <bool MASS>
  __device__ __forceinline__ Cut<F> select(Cut<F> cut, double target) {
    K a = MASS ? Key<Z>::of(this->sc.floor) : Key<Z>::of(-__builtin_inff()) + 1, b = Key<Z>::of(this->sc.m);
    const TwoWords two(row.V);
    bool share = MASS;
    if (threadIdx.x == 0) sh.above = sh.above_l = 0;
#pragma unroll 1
    for (;;) {
      __syncthreads();
      for (int i = threadIdx.x; i < BINS; i += RT) sh.hist[i] = sh.hist_l[i] = 0;
      if (threadIdx.x == 0) sh.n = 0;
      __syncthreads();
      int shift = 0;
      while (((b - a) >> shift) >= (K)BINS) ++shift;
      walk<Z>(row,
              [&](F(&v)[N], int base) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                  const K k = Key<Z>::of(v[j]);
                  if (k >= a && k <= b && cut.keeps(v[j], base + j)) {
                    const int bin = (int)((b - k) >> shift);
                    const Mass q = MASS ? two(weight(v[j], true)) : Mass{1, 0};
                    if (q.h) atomicAdd(&sh.hist[bin], q.h);
                    if (q.l) atomicAdd(&sh.hist_l[bin], q.l);
                  }
                }
              },
              NoEnd());
      __syncthreads();
      const int bin = MASS ? this->border_bin(two, target, share) : this->border_bin(sh.above, target, false);
      share = false;
      if (bin < 0) return cut;                        // fewer elements than asked for: all stay
      const K top = b - ((K)bin << shift), span = ((K)1 << shift) - 1, bottom = top - a > span ? top - span : a;
      __syncthreads();
      K lo = ~(K)0, hi = 0;
      walk<Z>(row,
              [&](F(&v)[N], int base) {
                uint32_t mask = 0;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                  const K k = Key<Z>::of(v[j]);
                  mask |= (uint32_t)(k >= bottom && k <= top && cut.keeps(v[j], base + j)) << j;
                }
                if (mask) {
                  int at = atomicAdd(&sh.n, __popc(mask));
#pragma unroll
                  for (int j = 0; j < N; ++j)
                    if (mask >> j & 1) {
                      const K k = Key<Z>::of(v[j]);
                      lo = k < lo ? k : lo;
                      hi = k > hi ? k : hi;
                      if (at < Base::CAP) list_put<Z, RT>(sh, at, {k, ~(uint32_t)(base + j)});
                      ++at;
                    }
                }
              },
              NoEnd());
      block_range<RT>(lo, hi, sh.wave_lo, sh.wave_hi);
      const int c = sh.n;
      if (c <= Base::CAP) {
        list_sort<Z, RT>(sh, c);
        if (MASS) return this->template sorted_cut<true>(c, (target - two.value({sh.above, sh.above_l})) * Whole::FIXED, 0);
        return this->template sorted_cut<false>(c, target, sh.above);
      }
      if (lo == hi) {                                 // one value: its first elements
        const F v = value_of<Z>(lo);
        const double need = ceil(MASS ? (target - two.value({sh.above, sh.above_l})) / weight(v, true) : target - (double)sh.above);
        return {v, nth_tie(cut, v, need < 1.0 ? 1 : need > (double)c ? c : (int)need)};
      }
      a = lo, b = hi;
    }
  }

  __device__ __forceinline__ void segment_sums(const Cut<F>& cut) {
    __syncthreads();
    for (int i = threadIdx.x; i < SEGS; i += RT) sh.seg[i] = 0;
    __syncthreads();
    const Limit<F> limit(cut, this->sc.least);
    double sum = 0;
    walk<Z>(row,
            [&](F(&v)[N], int base) {
              const F lim = limit.template of<N>(v, base);
#pragma unroll
              for (int j = 0; j < N; ++j) sum += weight(v[j], v[j] >= lim);
            },
            [&](int s) {
              sum = wave_sum(sum);
              if ((threadIdx.x & 63) == 0) sh.seg[s] = sum;
              sum = 0;
            });
  }
};

template <typename Z>
__global__ __launch_bounds__(RT) void row_slow_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args, Geometry g,
                                                      const RowWork<Z>* __restrict__ work, int64_t* __restrict__ label,
                                                      int64_t row0) {
  typedef typename Key<Z>::val_t F;
  __shared__ RowShared<Z, RT> sh;
  const int64_t i = row0 + blockIdx.x;
  if (label[i] != NOT_YET) return;
  const RowArgs a = row_args(args, i, g.V);
  fill_pow2(sh.pow2);
  const RowScale<Z> sc(largest<RT>(work[blockIdx.x].maxima, g.segs * g.per_seg, sh.wave_hi), a);
  const RowSampler<Z, RT> sampler = {sh, row_part(logits + (int64_t)blockIdx.x * ld, g, threadIdx.x >> 6, RW, sc.inf), sc,
                                     RowWeight<F>(sc.m, a.T, sh.pow2), Whole()};
  RowCut<Z> row(sampler);
  Cut<F> cut = {-__builtin_inff(), -1};
  if (a.k) cut = row.template select<false>(cut, (double)a.k);
  if (a.P < 1.0) cut = row.template select<true>(cut, a.P);
  row.segment_sums(cut);
  const int pick = row.draw(cut, a.u);
  if (threadIdx.x == 0) label[i] = pick;
}

constexpr int64_t ROW_BATCH = 512;      // rows that share the workspace
// (sizes on the host: std::min, the min of hip_runtime.h takes ints there)

template <typename Z>
int launch_rows(const Z* z, int64_t ld, const SampleArgs& a, int64_t* label, int64_t rows, int V, void* ws, int64_t ws_bytes,
                hipStream_t st) {
  if (!ws || ws_bytes < std::min(rows, ROW_BATCH) * (int64_t)sizeof(RowWork<Z>)) return TTK_EWORKSPACE;
  if ((uintptr_t)ws % 8) return TTK_EINVAL;
  RowWork<Z>* work = (RowWork<Z>*)ws;
  const Geometry g = geometry<Z>(V, std::min(rows, ROW_BATCH), a);
  // what the rows can need (parameters of their own: anything)
  const bool any_t = a.temperature || a.temperature_all > 0.0, all_k = !a.top_k && a.top_k_all > 0 && a.top_k_all < V;
  const bool any_p = a.top_p || a.top_p_all < 1.0, any_k = a.top_k || all_k || a.top_p || !(a.top_p_all > 0.0);      // (see row_args)
  const int most = !a.top_p && a.top_p_all < 1.0 ? g.most : g.alone;
  const bool no_list = all_k && a.top_k_all > most && !a.top_p && a.top_p_all > 0.0, sums = !all_k || a.top_k_all > most;
  for (int64_t r0 = 0; r0 < rows; r0 += ROW_BATCH) {
    const int64_t n = std::min(ROW_BATCH, rows - r0);
    const Z* p = z + r0 * ld;
    // workgroups a row: enough to fill the machine, each wave with a segment at least
    const int split = (int)std::max((int64_t)1, std::min((int64_t)(g.segs + TW - 1) / TW, (1024 + n - 1) / n));
    const int wide = (int)std::max((int64_t)1, std::min((int64_t)(g.segs + RW - 1) / RW, (256 + n - 1) / n));
    const dim3 grid((unsigned)split, (unsigned)n), big((unsigned)wide, (unsigned)n), one((unsigned)n);
    hipLaunchKernelGGL((row_maxima_kernel<Z>), grid, dim3(TB), 0, st, p, ld, g, work);
    if (any_t && any_k && !no_list) hipLaunchKernelGGL((row_collect_kernel<Z>), grid, dim3(TB), 0, st, p, ld, a, g, work, r0);
    if (any_t && sums) {
      if (any_p || any_k) {
        hipLaunchKernelGGL((row_counts_kernel<Z>), big, dim3(RT), 0, st, p, ld, a, g, work, r0);
        if (wide > 1) hipLaunchKernelGGL((row_window_kernel<Z>), one, dim3(RT), 0, st, a, g, work, r0);
      }
      hipLaunchKernelGGL((row_sums_kernel<Z>), grid, dim3(TB), 0, st, p, ld, a, g, work, r0);
    }
    hipLaunchKernelGGL((row_finish_kernel<Z>), one, dim3(TB), 0, st, p, ld, a, g, work, label, r0);
    if (any_t && (any_k || any_p)) hipLaunchKernelGGL((row_slow_kernel<Z>), one, dim3(RT), 0, st, p, ld, a, g, work, label, r0);
  }
  return hipGetLastError() == hipSuccess ? TTK_OK : TTK_ELAUNCH;
}

// Rows up to this long: a wave to eight waves a row, no workspace.  Sixteen waves are slower from here on where both top-k
// and top-p cut (1398 rows of 12000 float32, top-k 50 and top-p 0.9: 276 us against 119 us of the launches below).
constexpr int WAVE_ROW = 8192;

// The parameters from row `r` on.
SampleArgs from_row(SampleArgs a, int64_t r) {
  const auto at = [&](const void* p) { return p ? (const void*)((const char*)p + r * (a.f64 ? 8 : 4)) : p; };
  a.u = at(a.u), a.temperature = at(a.temperature), a.top_p = at(a.top_p), a.min_p = at(a.min_p);
  if (a.top_k) a.top_k += r;
  return a;
}

template <typename Z>
int launch(const void* logits, int64_t ld, const SampleArgs& args, int64_t* label, int64_t rows, int V, void* ws, int64_t ws_bytes,
           hipStream_t st) {
  const Z* z = (const Z*)logits;
  if (V > WAVE_ROW) return launch_rows<Z>(z, ld, args, label, rows, V, ws, ws_bytes, st);
  // a launch counts its threads in 32 bits (one of more runs a part of its workgroups without an error): 2^31 of them at a time
  const int threads = V <= FEW ? 1 : V <= 1024 ? 64 : V <= 2048 ? 128 : V <= 4096 ? 256 : 512;      // a row
  const int64_t most = (1ll << 31) / threads;
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int64_t n = std::min(most, rows - r0);
    const SampleArgs a = from_row(args, r0);
    const dim3 grid((unsigned)(V <= FEW ? (n + 63) / 64 : V <= 1024 ? (n + 3) / 4 : n));
#define L(THREADS, ...) hipLaunchKernelGGL((__VA_ARGS__), grid, dim3(THREADS), 0, st, z + r0 * ld, ld, a, label + r0, n, V)
#define K(E, W) L(W > 1 ? 64 * W : 256, sample_wave_kernel<Z, E, W>)
    if (V <= FEW)
      L(64, sample_few_kernel<Z>);
    else if (V <= 64)
      K(1, 1);
    else if (V <= 128)
      K(2, 1);
    else if (V <= 256)
      K(4, 1);
    else if (V <= 512)
      K(8, 1);
    else if (V <= 1024)
      K(16, 1);
    else if (V <= 2048)
      K(16, 2);
    else if (V <= 4096)
      K(16, 4);
    else
      K(16, 8);
#undef K
#undef L
  }
  return hipGetLastError() == hipSuccess ? TTK_OK : TTK_ELAUNCH;
}

}  // namespace

extern "C" {

int64_t ttk_sample_ws_bytes(int dtype, int64_t rows, int V) {
  if (dtype < 0 || dtype > 3 || rows < 1 || V < 1 || V > (1 << 30)) return TTK_EINVAL;
  if (V <= WAVE_ROW) return 0;
  return std::min(rows, ROW_BATCH) * (int64_t)(dtype == 0 ? sizeof(RowWork<double>) : sizeof(RowWork<float>));
}

int ttk_sample(int dtype, const void* logits, int64_t ld, const void* u, int f64, const void* temperature, double temperature_all,
               const int32_t* top_k, int top_k_all, const void* top_p, double top_p_all, const void* min_p, double min_p_all,
               int64_t* label, int64_t rows, int V, void* ws, int64_t ws_bytes, void* stream) {
  if (!logits || !u || !label || rows < 1 || V < 1 || V > (1 << 30) || ld < 0) return TTK_EINVAL;
  const SampleArgs a = {u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, f64};
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case 0: return launch<double>(logits, ld, a, label, rows, V, ws, ws_bytes, st);
    case 1: return launch<float>(logits, ld, a, label, rows, V, ws, ws_bytes, st);
    case 2: return launch<__bf16>(logits, ld, a, label, rows, V, ws, ws_bytes, st);
    case 3: return launch<_Float16>(logits, ld, a, label, rows, V, ws, ws_bytes, st);
  }
  return TTK_EINVAL;
}

}  // extern "C"
