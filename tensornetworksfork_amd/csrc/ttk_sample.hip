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
// Up to 64 E classes: a wave a row, E consecutive elements a lane.  Cuts are found bit by bit: the largest key t with
// enough elements (or weight) at or above it.
// ---------------------------------------------------------------------------------------
template <typename Z, int E>
__global__ __launch_bounds__(256) void sample_wave_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args,
                                                          int64_t* __restrict__ label, int64_t rows, int V) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const Z* p = logits + row * ld;
  const int e = (V + 63) / 64, c0 = lane * e;      // this lane's elements: c0 .. c0 + e - 1
  F z[E], m = -__builtin_inff();
  int first = 0x7FFFFFFF;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    z[i] = i < e && c0 + i < V ? Key<Z>::value(p[c0 + i]) : F(-__builtin_inff());
    if (z[i] > m) m = z[i], first = c0 + i;
  }
  const F mine = m;
  m = wave_max(m);
  const RowArgs a = row_args(args, row, V);
  if (!(m > -__builtin_inff()) || !(a.T > 0.0)) {
    const uint64_t who = __ballot(mine == m);
    const int f = __shfl(first, (int)__builtin_ctzll(who));
    if (lane == 0) label[row] = m > -__builtin_inff() ? f : -1;
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
    key[i] = Key<Z>::of(z[i]);
    w[i] = weight(z[i]);
  }
  constexpr int BITS = 8 * (int)sizeof(K), LOW = Key<Z>::LOW;
  // keeps, of the elements with w > 0, those in front of the cut: key above t, or the first `ties` of those with key t
  auto cut_at = [&](K t, int ties) {
    int before = 0;
    const K low = LOW ? (K)((1ull << LOW) - 1) : (K)0;
    t |= low;
#pragma unroll
    for (int i = 0; i < E; ++i) before += w[i] > 0 && (K)(key[i] | low) == t;
    before = wave_scan(before) - before;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const K k = key[i] | low;
      if (k < t || (k == t && w[i] > 0 && before++ >= ties)) w[i] = 0;
    }
  };
  if (a.k) {
    K t = 0;
    int above = 0, all = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) all += __popcll(__ballot(z[i] > -__builtin_inff()));
    if (all > a.k) {
      for (int bit = BITS - 1; bit >= LOW; --bit) {
        const K cand = t | ((K)1 << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) n += __popcll(__ballot(key[i] >= cand));
        if (n >= a.k)
          t = cand;
        else
          above = n;      // the last candidate with too few is the next key above the final t: what lies above t
      }
      // (elements of weight 0 lie below every other: they only matter as ties, where they are never drawn)
      cut_at(t, a.k - above);
    }
  }
  if (a.P < 1.0) {
    double total = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) total += w[i];
    total = wave_sum(total);
    const double target = a.P * total;
    K t = 0;
    double above = 0;
    for (int bit = BITS - 1; bit >= LOW; --bit) {
      const K cand = t | ((K)1 << bit);
      double s = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) s += key[i] >= cand ? w[i] : 0.0;
      s = wave_sum(s);
      if (s >= target)
        t = cand;
      else
        above = s;
    }
    double wt = 0;
    const K low = LOW ? (K)((1ull << LOW) - 1) : (K)0;
#pragma unroll
    for (int i = 0; i < E; ++i)
      if ((K)(key[i] | low) == (K)(t | low) && w[i] > 0) wt = w[i];
    wt = wave_max(wt);
    const double need = wt > 0 ? ceil((target - above) / wt) : 1.0;
    cut_at(t, need < 1.0 ? 1 : need > (double)V ? V : (int)need);
  }
  double s = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (!(w[i] >= a.M)) w[i] = 0;
    s += w[i];
  }
  const double upto = wave_scan(s), total = __shfl(upto, 63), target = a.u * total;
  uint64_t who = __ballot(s > 0 && upto > target);
  const bool last = who == 0;                       // u >= 1, or rounded up to it: the last kept element
  if (last) who = __ballot(s > 0);
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
// Many classes: a workgroup a row.
//
// The row is read from memory once and from the caches a few times more:
//   - the maximum (and its place, for temperature 0);
//   - top-k up to 512: the k-th largest of the 1024 threads' own maxima bounds the k-th largest element from below, so the
//     elements at or above that bound (a few more than k) are collected in LDS, sorted, cut and drawn from there;
//   - otherwise each cut is found by histograms: weights (counts for top-k) are added into 2048 bins, the bin with the
//     border is collected and sorted in LDS, or, where it holds too many, refined.  Weights enter as whole numbers
//     (2^-S of the largest, S = 62 - log2 V, at most 51), so that sums do not depend on the order of the atomics;
//   - the draw: float64 sums of the kept weights per segment of the row, their scan, and one wave over the segment that
//     holds u times the total.
// Elements of -inf do not exist for any of this.
// ---------------------------------------------------------------------------------------
constexpr int RT = 1024, RW = RT / 64, BINS = 2048, CAP = 2048, SEGS = 1024;

template <typename Z>
struct Chunk {
  static constexpr int N = 16 / (int)sizeof(Z);
  typedef uint32_t raw_t __attribute__((ext_vector_type(4), aligned(2)));
  union {
    uint32_t u[4];
    Z e[N];
  };
};

// A row as the waves of its workgroup see it: steps of 64 x 16 bytes, R steps a segment, wave w owns segments w, w + RW, ...
template <typename Z>
struct RowView {
  const Z* p;
  int V, steps, R;
  bool inf;        // the maximum is +inf
};

// The 16 bytes of this lane in step t.  Behind the row's end the last 16 bytes are read again (a row has more than that).
template <typename Z>
__device__ __forceinline__ int chunk_base(const RowView<Z>& row, int t) {
  return min((t * 64 + (int)(threadIdx.x & 63)) * Chunk<Z>::N, row.V - Chunk<Z>::N);
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
    const int again = (t * 64 + (int)(threadIdx.x & 63)) * N - chunk_base(row, t);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < again) v[j] = -__builtin_inff();
  }
  if (row.inf)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = finite(v[j], true);
}

// Calls f(values, first index) for every 16 bytes of the row and end(segment) after a wave's last step of a segment.  The
// next three steps are under way while one is worked on.
template <typename Z, typename Fn, typename End>
__device__ __forceinline__ void walk(const RowView<Z>& row, Fn f, End end) {
  constexpr int N = Chunk<Z>::N;
  int s = threadIdx.x >> 6, r = 0, ls = s, lr = 0;      // the step at work, the step to load next
  Chunk<Z> q[4];
  auto load = [&](Chunk<Z>& c) {
    load_chunk<Z>(c, row, ls * row.R + lr);
    if (++lr == row.R) lr = 0, ls += RW;
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
    if (full) r = 0, s += RW;
    t = s * row.R + r;
  }
}
struct NoEnd {
  __device__ __forceinline__ void operator()(int) const {}
};

template <typename Z>
struct RowShared {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  union {
    unsigned long long hist[BINS + 1];
    struct {
      uint64_t key[CAP];                                     // 32-bit keys: key << 32 | ~index
      uint32_t nidx[sizeof(K) == 8 ? CAP : 1];               // 64-bit keys: ~index
    } list;
    double seg[SEGS];
    int count[SEGS];
  };
  double pow2[32];
  double wave_d[RW];
  unsigned long long wave_u[RW];
  int wave_n[2][RW];
  F wave_f[RW];
  K wave_lo[RW], wave_hi[RW];
  int n, at, which, last;
  unsigned long long above;
  K cut_key;
  int cut_idx;
};

// The weight of Weight, with 2^(n / 32) from a table: 2^((z - m) log2(e) / T) = 2^(n div 32) pow2[n mod 32] 2^(f / 32),
// |f| <= 1/2, the last factor by its Taylor polynomial (relative error below 3e-15).  The 32 doubles lie in 64 different
// LDS banks.  m is finite.
template <typename F>
struct RowWeight {
  double m, c;
  const double* pow2;
  __device__ __forceinline__ RowWeight(F m_, double T, const double* table)
      : m((double)m_), c(fmin(32 * 1.4426950408889634074 / T, 1e300)), pow2(table) {}
  __device__ __forceinline__ double operator()(F z) const {
    double t = ((double)z - m) * c;
    t = t > -35200.0 ? t : -35200.0;
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

template <typename T>
__device__ __forceinline__ T block_scan(T v, T* buf, T& total) {      // inclusive; buf: RW values
  const int wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) buf[wave] = v;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    if (i < wave) before += buf[i];
    total += buf[i];
  }
  return v + before;
}

// an element of the list: what comes first sorts higher
template <typename Z>
__device__ __forceinline__ void list_put(RowShared<Z>& sh, int i, typename Key<Z>::type key, uint32_t nidx) {
  if constexpr (sizeof(key) == 4) {
    sh.list.key[i] = (uint64_t)key << 32 | nidx;
  } else {
    sh.list.key[i] = key;
    sh.list.nidx[i] = nidx;
  }
}
template <typename Z>
__device__ __forceinline__ void list_get(const RowShared<Z>& sh, int i, typename Key<Z>::type& key, uint32_t& nidx) {
  if constexpr (sizeof(key) == 4) {
    key = (uint32_t)(sh.list.key[i] >> 32);
    nidx = (uint32_t)sh.list.key[i];
  } else {
    key = sh.list.key[i];
    nidx = sh.list.nidx[i];
  }
}

// Bitonic sort of the first n2 (a power of two) elements, highest first: by (key, ~index), or by ~index alone.  A wave
// exchanges within its own 128 elements while the distance is at most 64: only longer ones need the workgroup's barrier.
template <typename Z>
__device__ __forceinline__ void list_sort(RowShared<Z>& sh, int n2, bool by_index) {
  typedef typename Key<Z>::type K;
  __syncthreads();
  for (int size = 2; size <= n2; size <<= 1)
    for (int d = size >> 1; d > 0; d >>= 1) {
      if (d > 64)
        __syncthreads();
      else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      const int t = threadIdx.x;
      if (t < n2 / 2) {
        const int i = 2 * t - (t & (d - 1)), j = i + d;
        K ki, kj;
        uint32_t ni, nj;
        list_get<Z>(sh, i, ki, ni);
        list_get<Z>(sh, j, kj, nj);
        const bool less = by_index ? ni < nj : ki < kj || (ki == kj && ni < nj);
        const bool more = by_index ? ni > nj : ki > kj || (ki == kj && ni > nj);
        if ((i & size) ? more : less) {
          list_put<Z>(sh, i, kj, nj);
          list_put<Z>(sh, j, ki, ni);
        }
      }
      if (d > 64) __syncthreads();
    }
  __syncthreads();
}

// Collects the elements `in` accepts into the list (the first CAP that come) and returns how many there are; lo / hi: the
// smallest and the largest of their keys.
template <typename Z, typename In>
__device__ int list_collect(RowShared<Z>& sh, const RowView<Z>& row, In in, typename Key<Z>::type& lo, typename Key<Z>::type& hi) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  K l = ~(K)0, h = 0;
  walk<Z>(row, [&](const F(&v)[N], int base) {
    uint32_t mask = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (in(v[j], base + j)) mask |= 1u << j;
    if (mask) {
      int at = atomicAdd(&sh.n, __popc(mask));
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (mask >> j & 1) {
          const K k = Key<Z>::of(v[j]);
          l = k < l ? k : l;
          h = k > h ? k : h;
          if (at < CAP) list_put<Z>(sh, at, k, ~(uint32_t)(base + j));
          ++at;
        }
    }
  }, NoEnd());
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const K a = __shfl_xor(l, s), b = __shfl_xor(h, s);
    l = a < l ? a : l;
    h = b > h ? b : h;
  }
  if ((threadIdx.x & 63) == 0) sh.wave_lo[threadIdx.x >> 6] = l, sh.wave_hi[threadIdx.x >> 6] = h;
  __syncthreads();
  lo = sh.wave_lo[0], hi = sh.wave_hi[0];
  for (int i = 1; i < RW; ++i) {
    lo = sh.wave_lo[i] < lo ? sh.wave_lo[i] : lo;
    hi = sh.wave_hi[i] > hi ? sh.wave_hi[i] : hi;
  }
  return sh.n;
}

// pads the list of c elements to a power of two with entries that sort last and returns it
template <typename Z>
__device__ int list_pad(RowShared<Z>& sh, int c) {
  int n2 = 2;
  while (n2 < c) n2 <<= 1;
  for (int i = c + threadIdx.x; i < n2; i += RT) list_put<Z>(sh, i, 0, 0);
  return n2;
}

// What is kept: the elements that do not come behind (v, idx) in the order.
template <typename F>
struct Cut {
  F v;
  int idx;
  __device__ __forceinline__ bool keeps(F z, int i) const { return z > v || (z == v && i <= idx); }
};

template <typename Z>
struct RowSampler {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  static constexpr int N = Chunk<Z>::N;
  RowShared<Z>& sh;
  RowView<Z> row;
  F m;
  RowWeight<F> weight;
  double fixed;      // 2^S

  __device__ __forceinline__ unsigned long long whole(double w) const {      // w 2^S, rounded; below 2^52
    return (unsigned long long)__double_as_longlong(w * fixed + 0x1p52) - 0x4330000000000000ull;
  }
  static __device__ __forceinline__ F value_of(K k) {
    if constexpr (sizeof(K) == 4)
      return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
    else
      return __longlong_as_double((int64_t)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
  }

  // place of the n-th (from 1) kept element that equals t
  __device__ __forceinline__ int nth_tie(const Cut<F>& cut, F t, int n) {
    __syncthreads();
    for (int i = threadIdx.x; i < SEGS; i += RT) sh.count[i] = 0;
    __syncthreads();
    int c = 0;
    walk<Z>(row, [&](const F(&v)[N], int base) {
#pragma unroll
      for (int j = 0; j < N; ++j) c += v[j] == t && cut.keeps(t, base + j);
    }, [&](int s) {
      c = wave_sum(c);
      if ((threadIdx.x & 63) == 0) sh.count[s] = c;
      c = 0;
    });
    __syncthreads();
    const int mine = sh.count[threadIdx.x];
    unsigned long long total;
    const int upto = (int)block_scan((unsigned long long)mine, sh.wave_u, total);
    if (upto >= n && upto - mine < n) sh.which = threadIdx.x, sh.at = upto - mine;
    __syncthreads();
    const int s = sh.which;
    int before = sh.at;
    __syncthreads();
    if (threadIdx.x < 64)
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

  // The cut of top-k (target elements) or, MASS, of top-p (share `target` of what `cut` keeps) among the elements `cut` keeps.
  template <bool MASS>
  __device__ __forceinline__ Cut<F> select(Cut<F> cut, double target, double range) {
    constexpr F none = -__builtin_inff();
    K a = Key<Z>::of(none) + 1, b = Key<Z>::of(m);
    bool linear = MASS;
    const F slope = (F)fmin((double)BINS / range, 1e38);      // bins a unit of z, over `range` below the maximum
    unsigned long long above = 0;
    for (;;) {
      __syncthreads();
      for (int i = threadIdx.x; i <= BINS; i += RT) sh.hist[i] = 0;
      __syncthreads();
      int shift = 0;
      if (!linear)
        while (((b - a) >> shift) >= (K)BINS) ++shift;
      unsigned long long beyond = 0;
      if (linear) {
        walk<Z>(row, [&](const F(&v)[N], int base) {
          int bin[N];
          unsigned long long q[N];
#pragma unroll
          for (int j = 0; j < N; ++j) {               // without branches: the eight chains overlap
            const F z = cut.keeps(v[j], base + j) ? v[j] : none;
            bin[j] = (int)fmin((m - z) * slope, F(BINS));
            q[j] = whole(weight(z));
            beyond += bin[j] < BINS ? 0ull : q[j];
          }
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (bin[j] < BINS) atomicAdd(&sh.hist[bin[j]], q[j]);
        }, NoEnd());
        beyond = wave_sum(beyond);
        if ((threadIdx.x & 63) == 0) atomicAdd(&sh.hist[BINS], beyond);
      } else {
        walk<Z>(row, [&](const F(&v)[N], int base) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const K k = Key<Z>::of(v[j]);
            if (k >= a && k <= b && cut.keeps(v[j], base + j))
              atomicAdd(&sh.hist[(int)((b - k) >> shift)], MASS ? whole(weight(v[j])) : 1ull);
          }
        }, NoEnd());
      }
      __syncthreads();
      const unsigned long long v0 = sh.hist[2 * threadIdx.x], v1 = sh.hist[2 * threadIdx.x + 1], over = sh.hist[BINS];
      unsigned long long total;
      const unsigned long long upto = above + block_scan(v0 + v1, sh.wave_u, total), from = upto - v0 - v1;
      if (linear) target *= (double)(total + over);
      if (threadIdx.x == 0 && (double)(above + total) < target) sh.which = linear ? BINS : -1, sh.above = above + total;
      if ((double)from < target && (double)(from + v0) >= target) sh.which = 2 * threadIdx.x, sh.above = from;
      if ((double)(from + v0) < target && (double)upto >= target) sh.which = 2 * threadIdx.x + 1, sh.above = from + v0;
      __syncthreads();
      const int bin = sh.which;
      above = sh.above;
      if (bin < 0) return cut;                        // fewer elements than asked for: all stay
      const K bb = b - (linear ? (K)0 : (K)bin << shift), width = linear ? (K)0 : ((K)1 << shift) - 1;
      K lo, hi;
      const int c = list_collect<Z>(sh, row, [&](F v, int i) {
        if (!(v > none) || !cut.keeps(v, i)) return false;
        if (linear) return (int)fmin((m - v) * slope, F(BINS)) == bin;
        const K k = Key<Z>::of(v);
        return k >= a && k <= bb && bb - k <= width;
      }, lo, hi);
      if (c <= CAP) {
        const int n2 = list_pad<Z>(sh, c);
        list_sort<Z>(sh, n2, false);
        K key[2];
        uint32_t nidx[2];
        unsigned long long q[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * threadIdx.x + e;
          if (i < c) {
            list_get<Z>(sh, i, key[e], nidx[e]);
            q[e] = MASS ? whole(weight(value_of(key[e]))) : 1ull;
          }
        }
        unsigned long long sum;
        unsigned long long before = above + block_scan(q[0] + q[1], sh.wave_u, sum) - q[0] - q[1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {                 // the last element with less than the target in front of it
          const int i = 2 * threadIdx.x + e;
          if (i < c && (double)before < target && (i == c - 1 || (double)(before + q[e]) >= target))
            sh.cut_key = key[e], sh.cut_idx = (int)~nidx[e];
          before += q[e];
        }
        __syncthreads();
        return {value_of(sh.cut_key), sh.cut_idx};
      }
      if (lo == hi) {                                 // one value: its first elements
        const F v = value_of(lo);
        const double each = MASS ? (double)whole(weight(v)) : 1.0;
        const double need = ceil((target - (double)above) / each);
        return {v, nth_tie(cut, v, need < 1.0 ? 1 : need > (double)c ? c : (int)need)};
      }
      a = lo, b = hi;
      linear = false;
    }
  }

  // the place, by index, where the running sum of the kept weights passes u times the total
  __device__ __forceinline__ int draw(const Cut<F>& cut, double u, double least) {
    __syncthreads();
    for (int i = threadIdx.x; i < SEGS; i += RT) sh.seg[i] = 0;
    if (threadIdx.x == 0) sh.which = SEGS, sh.last = -1;
    __syncthreads();
    double sum = 0;
    walk<Z>(row, [&](const F(&v)[N], int base) {
#pragma unroll
      for (int j = 0; j < N; ++j) {                   // without branches: the eight chains overlap
        const double w = weight(cut.keeps(v[j], base + j) ? v[j] : -__builtin_inff());
        sum += w >= least ? w : 0.0;
      }
    }, [&](int s) {
      sum = wave_sum(sum);
      if ((threadIdx.x & 63) == 0) sh.seg[s] = sum;
      sum = 0;
    });
    __syncthreads();
    const double mine = sh.seg[threadIdx.x];
    double total;
    const double upto = block_scan(mine, sh.wave_d, total), target = u * total;
    if (mine > 0) {
      if (upto > target) atomicMin(&sh.which, (int)threadIdx.x);
      atomicMax(&sh.last, (int)threadIdx.x);
    }
    __syncthreads();
    const bool last = sh.which == SEGS;                 // u >= 1, or rounded up to it: the last kept element
    const int s = last ? sh.last : sh.which;
    if ((int)threadIdx.x == s) sh.wave_d[0] = upto - mine;
    __syncthreads();
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x;
      double before = sh.wave_d[0];
      int pick = -1, end = -1;                          // end: the last kept element so far
      for (int r = 0; r < row.R && s * row.R + r < row.steps && pick < 0; ++r) {
        const int base = chunk_base(row, s * row.R + r);
        Chunk<Z> q;
        F v[N];
        load_chunk<Z>(q, row, s * row.R + r);
        chunk_values<Z>(v, q, row, s * row.R + r);
        double w[N], t = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          w[j] = weight(v[j]);
          if (!(cut.keeps(v[j], base + j) && w[j] >= least)) w[j] = 0;
          if (w[j] > 0) end = base + j;
          t += w[j];
        }
        const double upto = before + wave_scan(t);
        const uint64_t who = last ? 0 : __ballot(t > 0 && upto > target);
        if (who) {
          const int at = (int)__builtin_ctzll(who);
          double c = upto - t;
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (w[j] > 0 && !(pick >= 0 && c > target)) c += w[j], pick = base + j;
          pick = from_lane(pick, at);
        }
        before = from_lane(upto, 63);
      }
      end = wave_max(end);
      if (lane == 0) sh.at = pick >= 0 ? pick : end;
    }
    __syncthreads();
    return sh.at;
  }

  // top-k from the elements at or above `bound`, if the list holds them: true, and the label in `pick`
  __device__ __forceinline__ bool from_list(F bound, const RowArgs& a, int& pick) {
    const F none = -__builtin_inff();
    K lo, hi;
    const int c = list_collect<Z>(sh, row, [&](F v, int) { return v >= bound && v > none; }, lo, hi);
    if (c > CAP) return false;
    const int n2 = list_pad<Z>(sh, c);
    list_sort<Z>(sh, n2, false);
    const int kk = min(a.k, c);
    double w[2], total;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * threadIdx.x + e;
      K k;
      uint32_t n;
      w[e] = 0;
      if (i < kk) {
        list_get<Z>(sh, i, k, n);
        w[e] = weight(value_of(k));
      }
    }
    const double from = block_scan(w[0] + w[1], sh.wave_d, total) - w[0] - w[1], target = a.P * total;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * threadIdx.x + e;
      const bool front = a.P >= 1.0 || i == 0 || (e ? from + w[0] : from) < target;
      if (i < n2 && !(i < kk && front && w[e] >= a.M)) list_put<Z>(sh, i, 0, 0);
    }
    list_sort<Z>(sh, n2, true);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * threadIdx.x + e;
      K k;
      uint32_t n = 0;
      w[e] = 0;
      if (i < n2) list_get<Z>(sh, i, k, n);
      if (n) w[e] = weight(value_of(k));
    }
    if (threadIdx.x == 0) sh.which = CAP, sh.last = -1;
    const double upto = block_scan(w[0] + w[1], sh.wave_d, total), t = a.u * total;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (w[e] > 0) {
        const int i = 2 * threadIdx.x + e;
        if ((e ? upto : upto - w[1]) > t) atomicMin(&sh.which, i);
        atomicMax(&sh.last, i);
      }
    __syncthreads();
    K k;
    uint32_t n;
    list_get<Z>(sh, sh.which == CAP ? sh.last : sh.which, k, n);
    pick = (int)~n;
    return true;
  }
};

template <typename Z>
__global__ __launch_bounds__(RT) void sample_row_kernel(const Z* __restrict__ logits, int64_t ld, SampleArgs args,
                                                        int64_t* __restrict__ label, int64_t rows, int V) {
  typedef typename Key<Z>::type K;
  typedef typename Key<Z>::val_t F;
  constexpr int N = Chunk<Z>::N;
  __shared__ RowShared<Z> sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int steps = (V + 64 * N - 1) / (64 * N);
  // segments of up to 4 steps where every wave still gets several, more only where there are more than SEGS of them
  const int R = max((steps + SEGS - 1) / SEGS, max(1, min(4, steps / (4 * RW))));
  if (threadIdx.x < 32) sh.pow2[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    const RowArgs a = row_args(args, i, V);
    RowView<Z> row = {logits + i * ld, V, steps, R, false};
    F mine = -__builtin_inff();
    int at = V;                                        // the 16 bytes it was first seen in
    walk<Z>(row, [&](const F(&v)[N], int base) {
      F t = mine;
#pragma unroll
      for (int j = 0; j < N; ++j) t = v[j] > t ? v[j] : t;
      if (t > mine) mine = t, at = base;
    }, NoEnd());
    F m = wave_max(mine);
    __syncthreads();
    if (lane == 0) sh.wave_f[wave] = m;
    if (threadIdx.x == 0) sh.at = V;
    __syncthreads();
    for (int j = 0; j < RW; ++j) m = sh.wave_f[j] > m ? sh.wave_f[j] : m;
    if (!(m > -__builtin_inff()) || !(a.T > 0.0)) {
      if (mine == m && at < V) {
        int j = 0;
        while (Key<Z>::value(row.p[at + j]) != m) ++j;
        atomicMin(&sh.at, at + j);
      }
      __syncthreads();
      if (threadIdx.x == 0) label[i] = m > -__builtin_inff() ? sh.at : -1;
      continue;
    }
    row.inf = m == __builtin_inff();
    mine = finite(mine, row.inf);
    if (row.inf) m = 0;
    const int S = min(51, 30 + (int)__builtin_clz(V));      // 62 - log2 V, rounded down
    RowSampler<Z> r = {sh, row, m, RowWeight<F>(m, a.T, sh.pow2), ldexp(1.0, S)};
    int pick = -1;
    bool done = false;
    Cut<F> cut = {-__builtin_inff(), -1};
    if (a.k) {
      if (a.k <= RT / 2) {
        // the k-th largest of the threads' maxima, its upper 16 (64-bit keys: 24) bits
        const K key = Key<Z>::of(mine);
        K bound = 0;
        constexpr int BITS = 8 * (int)sizeof(K), END = BITS - (BITS == 64 ? 24 : 16);
        int turn = 0;
        for (int bit = BITS - 1; bit >= END; --bit, turn ^= 1) {
          const K cand = bound | ((K)1 << bit);
          const int c = __popcll(__ballot(key >= cand));
          if (lane == 0) sh.wave_n[turn][wave] = c;
          __syncthreads();
          int n = 0;
#pragma unroll
          for (int j = 0; j < RW; ++j) n += sh.wave_n[turn][j];
          if (n >= a.k) bound = cand;
        }
        const K none = Key<Z>::of(F(-__builtin_inff()));
        done = r.from_list(r.value_of(bound > none ? bound : none), a, pick);
      }
      if (!done) cut = r.template select<false>(cut, (double)a.k, 1.0);
    }
    if (!done) {
      // what lies further below the maximum than ln(V / (1 - P)) weighs less than 1 - P of the total: no bins for it
      if (a.P < 1.0) cut = r.template select<true>(cut, a.P, a.T * log((double)V / (1.0 - a.P)));
      pick = r.draw(cut, a.u, a.M);
    }
    if (threadIdx.x == 0) label[i] = pick;
  }
}

template <typename Z>
int launch(const void* logits, int64_t ld, const SampleArgs& a, int64_t* label, int64_t rows, int V, hipStream_t st) {
  const Z* z = (const Z*)logits;
  if (V <= FEW) {
    if ((rows + 63) / 64 > 0x7FFFFFFF) return TTK_EINVAL;
    hipLaunchKernelGGL((sample_few_kernel<Z>), dim3((unsigned)((rows + 63) / 64)), dim3(64), 0, st, z, ld, a, label, rows, V);
  } else if (V <= 1024) {
    const int64_t groups = (rows + 3) / 4;
    if (groups > 0x7FFFFFFF) return TTK_EINVAL;
    const dim3 grid((unsigned)groups);
    if (V <= 128)
      hipLaunchKernelGGL((sample_wave_kernel<Z, 2>), grid, dim3(256), 0, st, z, ld, a, label, rows, V);
    else if (V <= 512)
      hipLaunchKernelGGL((sample_wave_kernel<Z, 8>), grid, dim3(256), 0, st, z, ld, a, label, rows, V);
    else
      hipLaunchKernelGGL((sample_wave_kernel<Z, 16>), grid, dim3(256), 0, st, z, ld, a, label, rows, V);
  } else {
    hipLaunchKernelGGL((sample_row_kernel<Z>), dim3((unsigned)min(rows, (int64_t)65536)), dim3(RT), 0, st, z, ld, a, label, rows,
                       V);
  }
  return hipGetLastError() == hipSuccess ? TTK_OK : TTK_ELAUNCH;
}

}  // namespace

extern "C" {

int ttk_sample(int dtype, const void* logits, int64_t ld, const void* u, int f64, const void* temperature, double temperature_all,
               const int32_t* top_k, int top_k_all, const void* top_p, double top_p_all, const void* min_p, double min_p_all,
               int64_t* label, int64_t rows, int V, void* stream) {
  if (!logits || !u || !label || rows < 1 || V < 1 || V > (1 << 30) || ld < 0) return TTK_EINVAL;
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
