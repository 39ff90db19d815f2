// Sampling a token from each row of logits with temperature, top-k, top-p and min-p, from given
// uniform numbers, for gfx950.
//
//   e_j = exp((x_j - max x) / T);  order: value descending, index ascending
//   top-k: the first k of the order;  top-p: rank r stays iff the mass before r is below p times the
//   mass after top-k;  min-p: e_j >= min_p.  token: the first index whose running kept mass exceeds u
//   times the kept mass.
//
// Every filter keeps a prefix of the order, so what stays is described by one value and one index:
// x > cut.x, or x == cut.x and column <= cut.col. The weights and all sums are held in 64 bits: the
// result is an integer, and a border between two tokens that moves by 1e-8 of the mass (fp32 weights)
// gives another token once in some ten thousand rows of a broad distribution.
//
// One workgroup per row, which reads it once from memory and again from the caches:
//   1  maximum of the row (NaN propagates)
//   2  where top-k or top-p cut: a histogram over 2048 equal steps of the logit below the maximum --
//      counts for top-k, masses (64-bit fixed point: integer adds give the same sum in any order) for
//      top-p -- names the step that holds the cut; that step's few elements are sorted. Rows where the
//      step holds more than a list's worth (long runs of equal values, a cut far below the maximum)
//      take a radix search over the bits of the value
//   3  kept mass of each 64-vector segment in index order, the segment that holds u, the token in it
#include "../../include/fm_hip_tokens.h"
#include "fm_f64.hip.h"
#include "fm_topk.hip.h"

using namespace fm;

namespace {

constexpr int kBins = 2048;
constexpr int kList = 1024;          // candidates that are sorted
constexpr int kMaxSegs = 4096;       // segments of 64 vectors
constexpr int64_t kMaxCols = 1 << 20;

struct SampleArgs {
  const float* u;
  const float* temp;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temp0;
  int top_k0;
  float top_p0, min_p0;
  int64_t* token;
  float* logprob;
  int v;
};

__device__ __forceinline__ double wave_incl64(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(v, o, 64);
    if (lane >= o) v += t;
  }
  return v;
}

// A row as whole 16-byte vectors from the last 16-byte border at or before its first element; what
// the first and the last vector hold outside the row reads as -inf (weight zero, never kept) and is
// not loaded.
template <typename T>
struct RowView {
  static constexpr int EPV = Elem<T>::kVec;
  const T* base;    // 16-byte aligned; column c is base[c + lead]
  int lead;
  int v;
  int nvec;
  int w0, w1;       // vectors [w0, w1) lie inside the row
  __device__ __forceinline__ RowView(const T* row, int v_) : v(v_) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    base = row - lead;
    nvec = (v + lead + EPV - 1) / EPV;
    w0 = lead > 0 ? 1 : 0;
    w1 = (v + lead) / EPV;
  }
  __device__ __forceinline__ bool whole(int c) const { return c >= w0 && c < w1; }
  __device__ __forceinline__ int clamp(int c) const { return c < w0 ? w0 : (c < w1 ? c : w1 - 1); }
  __device__ __forceinline__ int col0(int c) const { return c * EPV - lead; }
  __device__ __forceinline__ u32x4 partial(int c) const {
    float f[EPV];
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      const int col = col0(c) + e;
      f[e] = (col >= 0 && col < v) ? Elem<T>::load1(base + (int64_t)c * EPV + e) : -INFINITY;
    }
    return Elem<T>::pack(f);
  }
  __device__ __forceinline__ u32x4 load(int c) const {
    return whole(c) ? load16(base + (int64_t)c * EPV) : partial(c);
  }
};

struct Cut {
  float x;      // kept: value > x, or value == x and column <= col
  int col;
};

template <int THREADS>
struct SampleShared {
  union {
    struct {
      unsigned long long bins[kBins];
      unsigned long long list[kList];
      unsigned long long sorted[kList];
    } h;
    double seg[kMaxSegs];
  };
  double red[THREADS / 64];
  float redf[2][THREADS / 64];
  unsigned long long redu[THREADS / 64];
  int redi[THREADS / 64];
  int count;
  int at;
  int col;
  float x;
  double mass;
};

// exp((x - m) / T) = 2^((x - m) c), to 1.1e-12. The maximum's weight is exactly 1, so that rows of few
// distinct values split evenly; that of -inf is zero.
struct Weight {
  double m, c;
  __device__ __forceinline__ double operator()(float x) const { return exp2_64(((double)x - m) * c); }
};

// First of `n` non-negative entries (in LDS, in order) whose running sum reaches `target`
// (strict: exceeds it); *before is the sum ahead of it. n when there is none. All threads call it.
template <int THREADS, bool STRICT, typename F>
__device__ __forceinline__ int find_running(F entry, int n, double target, SampleShared<THREADS>& sh, double* before) {
  constexpr int NW = THREADS / 64;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int per = (n + THREADS - 1) / THREADS;
  double mine = 0.0;
  for (int i = 0; i < per; ++i) {
    const int at = tid * per + i;
    if (at < n) mine += entry(at);
  }
  const double incl = wave_incl64(mine);
  if ((tid & 63) == 63) sh.red[wave] = incl;
  if (tid == 0) { sh.at = n; sh.mass = 0.0; }
  __syncthreads();
  double ahead = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) if (i < wave) ahead += sh.red[i];
  double run = ahead + (incl - mine);
  int hit = n;
  double hit_before = 0.0;
  for (int i = 0; i < per; ++i) {
    const int at = tid * per + i;
    if (at >= n) break;
    const double next = run + entry(at);
    if (STRICT ? next > target : next >= target) { hit = at; hit_before = run; break; }
    run = next;
  }
  if (hit < n) atomicMin(&sh.at, hit);
  __syncthreads();
  const int found = sh.at;
  if (hit < n && hit == found) sh.mass = hit_before;
  __syncthreads();
  *before = sh.mass;
  __syncthreads();
  return found;
}

// fn(vector, its index) for the vectors of the row, UN loads of a thread in flight.
template <typename T, int THREADS, int UN, typename F>
__device__ __forceinline__ void each_vector(const RowView<T>& rv, F fn) {
  const bool any = rv.w0 < rv.w1;
  for (int c0 = threadIdx.x; c0 < rv.nvec; c0 += THREADS * UN) {
    u32x4 raw[UN];
    if (any) {
#pragma unroll
      for (int i = 0; i < UN; ++i) raw[i] = load16(rv.base + (int64_t)rv.clamp(c0 + i * THREADS) * Elem<T>::kVec);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int c = c0 + i * THREADS;
      if (any) touch_whole(raw[i]);
      if (c < rv.nvec) {
        if (!rv.whole(c)) raw[i] = rv.partial(c);
        fn(raw[i], c);
      }
    }
  }
}
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void each_element(const RowView<T>& rv, F fn) {
  constexpr int EPV = Elem<T>::kVec;
  each_vector<T, THREADS, 1>(rv, [&](const u32x4& r, int c) {
    float x[EPV];
    Elem<T>::unpack(r, x);
#pragma unroll
    for (int e = 0; e < EPV; ++e) fn(x[e], rv.col0(c) + e);
  });
}

// The token among the segments whose weights are in sh.seg (nseg of them): the first column whose
// running weight exceeds `target`. weight_of(x, col) gives an element's weight. Rounding may leave the
// target at the very end: then the last column with a weight. Returns the column; *w its weight.
template <typename T, int THREADS, typename F>
__device__ __forceinline__ int pick(const RowView<T>& rv, int nseg, double target, F weight_of, SampleShared<THREADS>& sh,
                                    double* w) {
  constexpr int EPV = Elem<T>::kVec;
  double before;
  int s = find_running<THREADS, true>([&](int i) { return sh.seg[i]; }, nseg, target, sh, &before);
  const bool end = s == nseg;
  if (end) {          // the last segment with a weight
    if (threadIdx.x == 0) sh.at = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < nseg; i += THREADS) if (sh.seg[i] > 0.0) atomicMax(&sh.at, i);
    __syncthreads();
    s = sh.at;
  }
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const int c = s * 64 + lane;
    float x[EPV];
#pragma unroll
    for (int e = 0; e < EPV; ++e) x[e] = -INFINITY;
    if (c < rv.nvec) Elem<T>::unpack(rv.load(c), x);
    double wt[EPV];
    double mine = 0.0;
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      wt[e] = c < rv.nvec ? weight_of(x[e], rv.col0(c) + e) : 0.0;
      mine += wt[e];
    }
    const double incl = wave_incl64(mine);
    double run = before + (incl - mine);
    int hit = -1, last = -1;
    double hit_w = 0.0, last_w = 0.0;
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      run += wt[e];
      if (wt[e] > 0.0) { last = rv.col0(c) + e; last_w = wt[e]; }
      if (hit < 0 && wt[e] > 0.0 && run > target) { hit = rv.col0(c) + e; hit_w = wt[e]; }
    }
    const unsigned long long any = __ballot(!end && hit >= 0), some = __ballot(last >= 0);
    int from = 0;
    if (any != 0ull) from = __builtin_ctzll(any);
    else if (some != 0ull) from = 63 - __builtin_clzll(some);
    const int col = any != 0ull ? __shfl(hit, from, 64) : __shfl(last, from, 64);
    const double cw = any != 0ull ? __shfl(hit_w, from, 64) : __shfl(last_w, from, 64);
    if (lane == 0) { sh.col = col; sh.mass = cw; }
  }
  __syncthreads();
  const int col = sh.col;
  *w = sh.mass;
  __syncthreads();
  return col;
}

// Segment sums (64 vectors, a wave each) of weight_of over the row into sh.seg.
template <typename T, int THREADS, int UN, typename F>
__device__ __forceinline__ void segment_sums(const RowView<T>& rv, int nseg, F weight_of, SampleShared<THREADS>& sh) {
  constexpr int EPV = Elem<T>::kVec;
  __syncthreads();
  const bool any = rv.w0 < rv.w1;
  for (int c0 = threadIdx.x; (c0 >> 6) < nseg; c0 += THREADS * UN) {
    u32x4 raw[UN];
    if (any) {
#pragma unroll
      for (int i = 0; i < UN; ++i) raw[i] = load16(rv.base + (int64_t)rv.clamp(c0 + i * THREADS) * EPV);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int c = c0 + i * THREADS;
      if ((c >> 6) >= nseg) break;
      if (any) touch_whole(raw[i]);
      double mine = 0.0;
      if (c < rv.nvec) {
        if (!rv.whole(c)) raw[i] = rv.partial(c);
        float x[EPV];
        Elem<T>::unpack(raw[i], x);
#pragma unroll
        for (int e = 0; e < EPV; ++e) mine += weight_of(x[e], rv.col0(c) + e);
      }
      mine = wave_sum64(mine);
      if ((threadIdx.x & 63) == 0) sh.seg[c >> 6] = mine;
    }
  }
  __syncthreads();
}

// Radix search over the whole row, from memory: the value of the element at which the running amount
// (in descending order of value) reaches `target`, and the amount above that value. amount(x) is what
// an element of value x adds, as an integer. Equal neighbours of a thread are added up before they go
// to the histogram, so that a row of one value does not queue on one address.
template <typename T, int THREADS, typename F>
__device__ __forceinline__ uint32_t radix_cut(const RowView<T>& rv, double target, F amount, SampleShared<THREADS>& sh,
                                              unsigned long long* above) {
  uint32_t prefix = 0u;
  unsigned long long sum_above = 0ull;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += THREADS) sh.h.bins[i] = 0ull;
    __syncthreads();
    int open = -1;
    unsigned long long held = 0ull;
    each_element<T, THREADS>(rv, [&](float x, int col) {
      if (col < 0 || col >= rv.v) return;
      const uint32_t key = key_of(x);
      if (shift < 24 && ((key ^ prefix) >> (shift + 8)) != 0u) return;
      const int b = (int)((key >> shift) & 255u);
      if (b != open) {
        if (open >= 0) atomicAdd(&sh.h.bins[open], held);
        open = b;
        held = 0ull;
      }
      held += amount(x);
    });
    if (open >= 0) atomicAdd(&sh.h.bins[open], held);
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long run = sum_above;
      int b = 255, lowest = 0;
      for (; b >= 0; --b) {
        const unsigned long long w = sh.h.bins[b];
        if (w != 0ull) lowest = b;
        if (w != 0ull && (double)(run + w) >= target) break;
        run += w;
      }
      if (b < 0) {       // rounding: everything is kept, the lowest value is the cut
        b = lowest;
        run -= sh.h.bins[b];
      }
      sh.at = b;
      sh.redu[0] = run;
    }
    __syncthreads();
    prefix |= (uint32_t)sh.at << shift;
    sum_above = sh.redu[0];
  }
  __syncthreads();
  *above = sum_above;
  return prefix;
}

// Column of the c-th (1-based) element equal to x in index order; INT_MAX when there are no more than c.
template <typename T, int THREADS>
__device__ __forceinline__ int nth_equal(const RowView<T>& rv, int nseg, float x0, double c, SampleShared<THREADS>& sh) {
  auto equal = [&](float x, int col) { return x == x0 && col >= 0 && col < rv.v ? 1.0 : 0.0; };
  segment_sums<T, THREADS, 1>(rv, nseg, equal, sh);
  double mine = 0.0;
  for (int i = threadIdx.x; i < nseg; i += THREADS) mine += sh.seg[i];
  const double all = block_reduce64<THREADS / 64, Sum64>(mine, sh.red);
  if (c >= all) return 0x7fffffff;
  double w;
  return pick<T, THREADS>(rv, nseg, c - 0.5, equal, sh, &w);
}

template <typename T, int THREADS, int UN>
__global__ __launch_bounds__(THREADS) void sample_kernel(const T* __restrict__ logits, SampleArgs a) {
  constexpr int EPV = Elem<T>::kVec;
  constexpr int NW = THREADS / 64;
  __shared__ SampleShared<THREADS> sh;
  const int64_t row = blockIdx.x;
  const RowView<T> rv(logits + row * (int64_t)a.v, a.v);
  const int tid = threadIdx.x;

  const float T_ = a.temp != nullptr ? a.temp[row] : a.temp0;
  int k = a.top_k != nullptr ? a.top_k[row] : a.top_k0;
  float p = a.top_p != nullptr ? a.top_p[row] : a.top_p0;
  float min_p = a.min_p != nullptr ? a.min_p[row] : a.min_p0;
  const float u_in = a.u[row];
  // values of 1 and more count as the largest below 1, NaN and negative ones as 0
  const double u = u_in > 0.f ? (double)fminf(u_in, 1.f - 5.9604645e-8f) : 0.0;
  const bool use_k = k > 0 && k < a.v;
  const bool use_p = p < 1.f;
  if (!(p > 0.f)) p = 0.f;
  const bool use_m = min_p > 0.f;
  min_p = fminf(min_p, 1.f);
  auto each = [&](auto fn) { each_vector<T, THREADS, UN>(rv, fn); };

  // 1: the maximum; NaN propagates
  float mx = -INFINITY;
  each([&](const u32x4& r, int) {
    float x[EPV];
    Elem<T>::unpack(r, x);
#pragma unroll
    for (int e = 0; e < EPV; ++e) mx = __builtin_elementwise_maximum(mx, x[e]);
  });
  float wm = mx;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) wm = __builtin_elementwise_maximum(wm, __shfl_xor(wm, o, 64));
  // least of the threads' maxima, of those that have one: as many elements are not below it
  const bool some = mx > -INFINITY;
  const float wl = -group_reduce<64, OpMax>(some ? -mx : -INFINITY);
  const int wn = __builtin_popcountll(__ballot(some));
  if ((tid & 63) == 0) { sh.redf[0][tid >> 6] = wm; sh.redf[1][tid >> 6] = wl; sh.redi[tid >> 6] = wn; }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  float m = sh.redf[0][0], least = sh.redf[1][0];
  int vouched = sh.redi[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) {
    m = __builtin_elementwise_maximum(m, sh.redf[0][i]);
    least = fminf(least, sh.redf[1][i]);
    vouched += sh.redi[i];
  }
  // (NaN compares false everywhere)
  if (!(m < INFINITY && m > -INFINITY) || !(T_ >= 0.f && T_ < INFINITY)) {
    if (tid == 0) {
      a.token[row] = -1;
      if (a.logprob != nullptr) a.logprob[row] = __builtin_nanf("");
    }
    return;
  }
  const int nseg = (rv.nvec + 63) / 64;
  if (T_ == 0.f) {           // the first maximum
    __syncthreads();         // sh.redi
    int first = 0x7fffffff;
    each([&](const u32x4& r, int c) {
      float x[EPV];
      Elem<T>::unpack(r, x);
#pragma unroll
      for (int e = EPV - 1; e >= 0; --e) if (x[e] == m && rv.col0(c) + e < first) first = rv.col0(c) + e;
    });
    first = wave_min_i(first);
    if ((tid & 63) == 0) sh.redi[tid >> 6] = first;
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < NW; ++i) first = sh.redi[i] < first ? sh.redi[i] : first;
      a.token[row] = first;
      if (a.logprob != nullptr) a.logprob[row] = 0.f;
    }
    return;
  }
  const Weight weight{(double)m, 1.4426950408889634074 / (double)T_};

  // 2: the cut
  Cut cut{-INFINITY, 0x7fffffff};
  if (use_k || use_p) {
    // Steps of equal width below the maximum. For top-k over the range that the threads' maxima
    // vouch for (when there are k of them), else over 24 T: what lies below weighs less than 4e-11.
    float range = m - least;
    if (!(use_k && k <= vouched) || !(range < INFINITY)) range = 24.f * T_;
    float per = (float)(kBins - 2) / range;
    if (!(per <= 1e30f)) per = 1e30f;
    // 2^fx units of mass per 1: the sum of v weights of at most 1 stays below 2^62
    const int vbits = 62 - (32 - __builtin_clz((unsigned)a.v));
    const int fx = vbits < 50 ? vbits : 50;
    const double unit = __builtin_amdgcn_ldexp(1.0, fx);
    // w * unit to the nearest integer (w <= 1 and unit <= 2^50: below 2^52)
    auto fixed = [&](double w) {
      return __builtin_bit_cast(unsigned long long, __builtin_fma(w, unit, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    };
    for (int i = tid; i < kBins; i += THREADS) sh.h.bins[i] = 0ull;
    __syncthreads();
    const float last_bin = (float)(kBins - 1);
    double total = 0.0, target;
    if (use_k) {
      each([&](const u32x4& r, int c) {
        float x[EPV];
        Elem<T>::unpack(r, x);
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
          const float y = (m - x[e]) * per;
          if (y < last_bin) atomicAdd(&sh.h.bins[(int)y], 1ull);
        }
      });
      target = (double)k;
    } else {
      each([&](const u32x4& r, int c) {
        float x[EPV];
        Elem<T>::unpack(r, x);
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
          const double w = weight(x[e]);
          total += w;
          const float y = (m - x[e]) * per;
          if (y < last_bin) atomicAdd(&sh.h.bins[(int)y], fixed(w));
        }
      });
      total = block_reduce64<THREADS / 64, Sum64>(total, sh.red);
      target = (double)p * total * unit;
    }
    __syncthreads();
    double ahead;
    const int bin = find_running<THREADS, false>([&](int i) { return (double)sh.h.bins[i]; }, kBins, target, sh, &ahead);
    bool listed = bin < kBins;
    if (listed) {
      // candidates: the step of the cut, and for top-k (whose order the nucleus may need) all above it
      const float lo = use_k ? 0.f : (float)bin, hi = (float)(bin + 1);
      each([&](const u32x4& r, int c) {
        float x[EPV];
        Elem<T>::unpack(r, x);
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
          const float y = (m - x[e]) * per;
          if (y >= lo && y < hi) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kList) sh.h.list[at] = ((unsigned long long)key_of(x[e]) << 32) | (uint32_t)~(uint32_t)(rv.col0(c) + e);
          }
        }
      });
      __syncthreads();
      const int n = sh.count;
      listed = n <= kList;
      if (listed) {
        // order the candidates by counting those that come before each
        for (int i = tid; i < n; i += THREADS) {
          const unsigned long long me = sh.h.list[i];
          int rank = 0;
          for (int j = 0; j < n; ++j) rank += sh.h.list[j] > me ? 1 : 0;
          sh.h.sorted[rank] = me;
        }
        __syncthreads();
        auto value = [&](int i) { return float_of_key((uint32_t)(sh.h.sorted[i] >> 32)); };
        int kept = use_k ? k : n;
        if (use_p) {
          double goal, base = 0.0;
          if (use_k) {
            double mine = 0.0;
            for (int i = tid; i < k; i += THREADS) mine += weight(value(i));
            goal = (double)p * block_reduce64<THREADS / 64, Sum64>(mine, sh.red);
          } else {
            goal = (double)p * total;
            base = ahead / unit;
          }
          // the first rank at which the mass reaches the goal is the last one kept
          double unused;
          const int r = find_running<THREADS, false>([&](int i) { return weight(value(i)); }, kept, goal - base,
                                                     sh, &unused);
          kept = r < kept ? r + 1 : kept;
        }
        cut.x = value(kept - 1);
        cut.col = (int)~(uint32_t)sh.h.sorted[kept - 1];
        __syncthreads();
      }
    }
    if (!listed) {
      double ties = 0.0;
      unsigned long long above;
      if (use_k) {
        const uint32_t key = radix_cut<T, THREADS>(rv, (double)k, [](float) { return 1ull; }, sh, &above);
        cut.x = float_of_key(key);
        ties = (double)k - (double)above;
        if (use_p) {      // the mass of those k
          double mine = 0.0;
          each_element<T, THREADS>(rv, [&](float x, int) { if (x > cut.x) mine += weight(x); });
          total = block_reduce64<THREADS / 64, Sum64>(mine, sh.red) + ties * weight(cut.x);
        }
      }
      if (use_p) {
        const double goal = (double)p * total * unit;
        const uint32_t key = radix_cut<T, THREADS>(
            rv, goal, [&](float x) { return fixed(weight(x)); }, sh, &above);
        const float xp = float_of_key(key);
        const double each_w = (double)fixed(weight(xp));
        // equal values that the mass still needs: the r-th stays iff above + r * weight < goal
        double need = each_w > 0.0 ? ceil((goal - (double)above) / each_w) : 1.0;
        if (!(need >= 1.0)) need = 1.0;
        if (!use_k || xp > cut.x) {
          cut.x = xp;
          ties = need;
        } else if (xp == cut.x && need < ties) {
          ties = need;
        }
      }
      cut.col = nth_equal<T, THREADS>(rv, nseg, cut.x, ties, sh);
    }
  }
  if (use_m) {               // the least value with a weight of min_p; every equal one stays
    const double xm = (double)m + (double)T_ * log((double)min_p);
    float xf = (float)xm;                      // may be -inf: then everything stays
    if ((double)xf < xm) xf = float_of_key(key_of(xf) + 1u);      // the next float up
    if (xf > m) xf = m;
    if (xf > cut.x) {
      cut.x = xf;
      cut.col = 0x7fffffff;
    }
  }

  // 3: kept mass by segment, in index order
  auto kept_weight = [&](float x, int col) {
    return x > cut.x || (x == cut.x && col <= cut.col) ? weight(x) : 0.0;
  };
  segment_sums<T, THREADS, UN>(rv, nseg, kept_weight, sh);
  double mine = 0.0;
  for (int i = tid; i < nseg; i += THREADS) mine += sh.seg[i];
  const double kept = block_reduce64<THREADS / 64, Sum64>(mine, sh.red);
  double w;
  const int col = pick<T, THREADS>(rv, nseg, u * kept, kept_weight, sh, &w);
  if (tid == 0) {
    a.token[row] = col;
    if (a.logprob != nullptr) a.logprob[row] = (float)log(w / kept);
  }
}

template <typename T>
void launch(const void* logits, const SampleArgs& a, int64_t n, hipStream_t st) {
  const int64_t nvec = a.v / Elem<T>::kVec + 2;
#define GO(TH, UN) FM_LAUNCH((sample_kernel<T, TH, UN>), dim3((unsigned)n), dim3(TH), 0, st, static_cast<const T*>(logits), a)
  if (nvec <= 1024) GO(256, 4);
  else GO(1024, 4);
#undef GO
}

}  // namespace

extern "C" int fm_sample(const void* logits, const float* u, const float* temperature, const int32_t* top_k,
                         const float* top_p, const float* min_p, float temperature0, int top_k0, float top_p0,
                         float min_p0, int64_t* token, float* logprob, int64_t n, int64_t v, int dtype,
                         fm_stream_t stream) {
  FM_CHECK_ARG(n >= 0 && v > 0, "fm_sample: bad shape n=%lld v=%lld", (long long)n, (long long)v);
  FM_CHECK_ARG(dtype == FM_F32 || dtype == FM_F16 || dtype == FM_BF16, "fm_sample: bad dtype %d", dtype);
  if (n > 0x7fffffffLL || v > kMaxCols) {
    fm_host::set_error("fm_sample: n must be below 2^31 and v at most %lld", (long long)kMaxCols);
    return FM_ERR_UNSUPPORTED;
  }
  if (n == 0) return FM_OK;
  FM_CHECK_ARG(logits && u && token, "fm_sample: NULL pointer");
  FM_CHECK_ARG((reinterpret_cast<uintptr_t>(logits) & (dtype == FM_F32 ? 3u : 1u)) == 0,
               "fm_sample: logits are not aligned to their type");
  SampleArgs a;
  a.u = u; a.temp = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.temp0 = temperature0; a.top_k0 = top_k0; a.top_p0 = top_p0; a.min_p0 = min_p0;
  a.token = token; a.logprob = logprob; a.v = (int)v;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == FM_F32) launch<float>(logits, a, n, st);
  else if (dtype == FM_BF16) launch<bf16_t>(logits, a, n, st);
  else launch<f16_t>(logits, a, n, st);
  FM_CHECK_LAUNCH("fm_sample");
  return FM_OK;
}
