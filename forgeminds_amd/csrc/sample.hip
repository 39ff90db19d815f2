// Sampling a token from each row of logits with temperature, top-k, top-p and min-p, from given
// uniform numbers, for gfx950.
//
//   e_j = exp((x_j - max x) / T);  order: value descending, index ascending
//   top-k: the first k of the order;  top-p: rank r stays iff the mass before r is below p times the
//   mass after top-k;  min-p: e_j >= min_p.  token: the first index whose running kept mass exceeds u
//   times the kept mass.
//
// Every filter keeps a prefix of the order, so what stays is described by one value and one index:
// x > cut.x, or x == cut.x and column <= cut.col. The weights are computed in 64 bits: the result is an
// integer, and a border between two tokens that moves by 1e-8 of the mass (fp32 weights) gives another
// token once in some ten thousand rows of a broad distribution. From there on they are integers: a weight
// counts as the nearest multiple of 2^-fx (fx = 50 up to 8192 columns, 46 up to 2^17, 43 for 2^20), all sums
// are exact, and a decision is a comparison of integers. So a row's result is the same whichever of the
// ways below it takes, in whatever order its sums are formed: workgroup sizes go by the number of rows, and
// a row alone is the row among many. What rounding remains is half a unit an element: v 2^-(fx + 1) of a mass
// of at least 1 at worst, 9e-10 for 2^17 columns and 6e-8 for 2^20, the square root of that many units in
// earnest (1e-12).
//
// One workgroup per row, which reads it once from memory and again from the caches:
//   1  maximum of the row (NaN propagates)
//   2  candidates: the elements from the maximum down to a bound at or below the cut, into a list in LDS.
//      top-k: the waves' thread maxima vouch for k elements above the bound. min-p: its own bound. top-p
//      alone (and a top-k whose list overflows): a histogram of the row's masses (or counts) over 2048 equal
//      steps of the logit names the step that holds the cut
//   3  the exact cut: histograms of the list narrow it to one step, whose elements are put in order. A step
//      with more elements than that is searched by the bits of the value; among equal values the cut is a
//      count, which the last sweep turns into a column
//   4  token: masses of the segments in index order, the segment that holds u, the token in it -- from the
//      list, or over the row again where the list is too long (flat rows)
// Where nothing cuts, one sweep does: each segment's weights against its own maximum, summed in 64 bits in an
// order of the segment's own, brought to the row's maximum and rounded to the unit then.
// Weights are computed for the candidates only, unless the mass of the whole row is asked for.
//
// What bounds it: the arithmetic of those weights, some 27 instructions an element with the histogram, on
// the row's one compute unit; memory is far (256 rows of 128256 bf16 are 10 us of reading), but in the
// unfiltered sweep its 16 us ([512,50257] fp32) and the weights' 14 hardly overlap. Measured, bf16, us of the
// kernel, rows of power laws with exponents from 1 to 2 (the slowest row decides: at exponent 1 the list
// overflows and the kept weights are evaluated a second time):
//                 unfiltered  min-p 0.02  top-k 50  top-p 0.9  top-p 0.9, flat rows
//   [1,128256]            27          12        23         40                    99
//   [256,128256]          34          24        33        105                   113
//   [512,128256]          55          40        46        176                   188
//   [1024,32000]          33          26        45        101                   106
// Of the 40 us for one row the maximum takes 4, the histogram 23, the list 6. The first two would divide over
// several workgroups a row (their partial results are integers and a maximum); that has not been tried.
//
// What keeps it small counts too: the code that a call runs through fits the instruction cache (64 KB for
// two compute units). Putting the row's two partial vectors together in place, in every sweep, made each
// sweep 2 to 15 us longer; they stand in shared memory instead.
#include "../../include/fm_hip_tokens.h"
#include "fm_f64.hip.h"
#include "fm_topk.hip.h"
#include <type_traits>

using namespace fm;

namespace {

constexpr int kBins = 2048;
constexpr int kStep = 1024;          // candidates of one step (or one segment)
constexpr int kFew = 256;            // as many are ordered by comparing each with each
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

// A row as whole 16-byte vectors from the last 16-byte border at or before its first element; what
// the first and the last vector hold outside the row reads as -inf (weight zero, never kept) and is
// not loaded: those two are put together in shared memory once.
template <typename T>
struct RowView {
  static constexpr int EPV = Elem<T>::kVec;
  const T* base;    // 16-byte aligned; column c is base[c + lead]
  int lead;
  int v;
  int nvec;
  int w0, w1;       // vectors [w0, w1) lie inside the row
  u32x4* edges;     // shared memory, two vectors
  __device__ __forceinline__ RowView(const T* row, int v_, u32x4* edges_) : v(v_), edges(edges_) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    base = row - lead;
    nvec = (v + lead + EPV - 1) / EPV;
    w0 = lead > 0 ? 1 : 0;
    w1 = (v + lead) / EPV;
  }
  __device__ __forceinline__ bool whole(int c) const { return c >= w0 && c < w1; }
  __device__ __forceinline__ int clamp(int c) const { return c < w0 ? w0 : (c < w1 ? c : w1 - 1); }
  __device__ __forceinline__ int col0(int c) const { return c * EPV - lead; }
  // the first and the last vector, by the workgroup's first threads (a barrier is due)
  __device__ __forceinline__ void fill_edges() const {
    const int t = threadIdx.x;
    if (t >= 2 * EPV) return;
    const int col = col0(t < EPV ? 0 : nvec - 1) + t % EPV;
    const bool inside = col >= 0 && col < v;
    Elem<T>::store1(reinterpret_cast<T*>(edges) + t, inside ? Elem<T>::load1(base + lead + col) : -INFINITY);
  }
  __device__ __forceinline__ u32x4 partial(int c) const {
    return reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
        (const __attribute__((address_space(3))) void*)edges)[c < w0 ? 0 : 1];
  }
  // one whole vector: the address space is spelled out, since behind the views' pointers the compiler
  // takes the load for a flat one, whose wait is a wait for everything
  __device__ __forceinline__ u32x4 load_whole(int c) const {
    return *(const __attribute__((address_space(1))) u32x4*)(reinterpret_cast<const char*>(base) + (uint32_t)c * 16u);
  }
  // vectors c, c + STRIDE, ...; where one is not whole, some other that is (or nothing, in a row that has none)
  template <int STRIDE, int N>
  __device__ __forceinline__ void load_some(int c, u32x4 (&raw)[N]) const {
    if (w0 < w1) {
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = load_whole(clamp(c + i * STRIDE));
    }
  }
  __device__ __forceinline__ u32x4 load(int c) const { return whole(c) ? load_whole(c) : partial(c); }
};

// a value that all lanes hold alike, in scalar registers: branches on it stay scalar
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ double uniform(double v) { return readlane64(v, 0); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) { return readlane_u64(v, 0); }

// element e of a vector
template <typename T>
__device__ __forceinline__ float element(const u32x4& r, int e) {
  constexpr int per = 4 / sizeof(T);             // elements a register
  const int i = e / per;
  const uint32_t lo = i & 1 ? r.y : r.x, hi = i & 1 ? r.w : r.z;
  u32x4 one = {(i & 2 ? hi : lo) >> (e % per * 16), 0u, 0u, 0u};
  float x[Elem<T>::kVec];
  Elem<T>::unpack(one, x);
  return x[0];
}

struct OpMaximum {      // NaN stays
  __device__ static __forceinline__ float f(float a, float b) { return __builtin_elementwise_maximum(a, b); }
};

struct Cut {
  float x;      // kept: value > x, or value == x and column <= col
  int col;
};

template <int THREADS>
struct SampleShared {
  static constexpr int kList = 4 * THREADS;                  // candidates
  static constexpr int kSegs = 1040;   // segments (v <= 2^20)
  struct {
    unsigned long long bins[kBins];
    uint64_t list[kList];       // (key << 32) | ~column: larger comes first
    uint64_t step[kStep];       // the candidates of one step or segment ...
    uint64_t mass[kStep];       // ... and their weights
  } h;
  u32x4 edges[2];
  uint64_t seg[kSegs];
  union {
    float segm[kSegs];        // where nothing cuts: the segments' maxima
    int ties[kSegs];          // else: their elements equal to the cut
  };
  double red[THREADS / 64];
  float redf[1][THREADS / 64];
  uint64_t redu[THREADS / 64];
  int redi[THREADS / 64];
  int count;
  int at;
  uint32_t klo, khi;
  int hits[4], lasts[4];
  float hitx[4], lastx[4];
  uint64_t before;
};

// exp((x - m) / T) = 2^((x - m) c), c = log2(e) / T, by the polynomial of exp2_64, written out for several elements at once:
// seventeen operations each, the constants in scalar registers (the compiler otherwise copies each into
// two vector registers for every use, which doubles the work), and n from the low bits of t + 1.5 * 2^52.
// The maximum's weight is exactly 1, so that rows of few distinct values split evenly; that of -inf is 0.
struct Weight {
  double m, c;
  double k[9], magic, least;
  __device__ __forceinline__ Weight(double max_x, double c_) : m(max_x), c(c_) {
    k[8] = 1.3255224878668817e-06; k[7] = 1.5310079402249296e-05; k[6] = 0.00015403455852453838;
    k[5] = 0.0013333450568000645; k[4] = 0.009618129159402558; k[3] = 0.05550410941205933;
    k[2] = 0.2402265069581299; k[1] = 0.6931471805459335; k[0] = 1.0;
    magic = 6755399441055744.0;
    least = -1100.0;
#pragma unroll
    for (int i = 0; i < 9; ++i) asm volatile("" : "+s"(k[i]));
    asm volatile("" : "+s"(magic), "+s"(least));
  }
  // the same for one sweep: its constants take up scalar registers there only
  __device__ __forceinline__ Weight fresh() const { return Weight(m, c); }
  template <int N>
  __device__ __forceinline__ void eval(const float* x, double* w) const {
    double f[N], r[N];
    int n[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double t = ((double)x[i] - m) * c;
      asm("v_max_f64 %0, %1, %2" : "=v"(t) : "v"(t), "s"(least));
      const double s = t + magic;
      n[i] = (int)(uint32_t)__builtin_bit_cast(uint64_t, s);
      f[i] = t - (s - magic);
      r[i] = k[8];
    }
#pragma unroll
    for (int j = 7; j >= 0; --j) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = __builtin_fma(r[i], f[i], k[j]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = __builtin_amdgcn_ldexp(r[i], n[i]);
      if (N > 1) asm volatile("" : "+v"(w[i]));      // here, side by side, not where each is used
    }
  }
  __device__ __forceinline__ double operator()(float x) const {
    double w;
    eval<1>(&x, &w);
    return w;
  }
};

// The thread's number, formed anew at each use: otherwise every address made of it is kept in a register
// of its own over the loop of the two cuts.
__device__ __forceinline__ int thread_here() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// First of `n` entries (in LDS, in order) at which the running sum reaches `goal` (at least 1); *before is the
// sum ahead of it. n when there is none. All threads call it.
template <int THREADS, typename F>
__device__ __forceinline__ int find_running(F entry, int n, uint64_t goal, SampleShared<THREADS>& sh, uint64_t* before) {
  constexpr int NW = THREADS / 64;
  const int tid = thread_here(), lane = tid & 63, wave = tid >> 6;
  const int per = (n + THREADS - 1) / THREADS;
  uint64_t mine = 0ull;
  for (int i = 0; i < per; ++i) {
    const int at = tid * per + i;
    if (at < n) mine += entry(at);
  }
  uint64_t end = wave_incl_u64(mine);
  if (lane == 63) sh.redu[wave] = end;
  if (tid == 0) { sh.at = n; sh.before = 0ull; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) if (i < wave) end += sh.redu[i];
  uint64_t run = end - mine;
  if (run < goal && goal <= end) {        // one thread at most
    int at = tid * per;
    for (uint64_t w = entry(at); run + w < goal; w = entry(at)) { run += w; ++at; }
    sh.at = at;
    sh.before = run;
  }
  __syncthreads();
  const int found = uniform(sh.at);
  *before = uniform(sh.before);
  __syncthreads();
  return found;
}

// fn(vector, its index) for the vectors of the row, four loads of a thread in flight. (Loading the next four
// ahead of the work gained nothing here: [512,128256] top-p 0.9 93 us with it, 92 without.)
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void each_vector(const RowView<T>& rv, F fn) {
  constexpr int UN = 4;
  for (int c0 = thread_here(); c0 < rv.nvec; c0 += THREADS * UN) {
    u32x4 raw[UN];
    rv.template load_some<THREADS, UN>(c0, raw);
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int c = c0 + i * THREADS;
      touch_whole(raw[i]);
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
  each_vector<T, THREADS>(rv, [&](const u32x4& r, int c) {
    float x[EPV];
    Elem<T>::unpack(r, x);
#pragma unroll
    for (int e = 0; e < EPV; ++e) fn(x[e], rv.col0(c) + e);
  });
}

// A segment is G blocks of 64 vectors that one wave sweeps, a vector a lane: one reduction over the wave
// for G vectors a lane.
constexpr int seg_vecs(int G) { return 64 * G; }

// The first column at which the running weight reaches `goal`, from the weights of the nseg segments:
// weights_of(x, col0, w) gives those of a vector, as integers. (Where nothing cuts, a segment's rounded weight
// may be a few units more than its elements' together: then its last column with a weight.) Returns the
// column; *x is its logit, *seg its segment, *ahead the weight in front of that.
template <typename T, int THREADS, int G, typename E, typename F>
__device__ __forceinline__ int pick(const RowView<T>& rv, int nseg, E entry, uint64_t goal, F weights_of,
                                    SampleShared<THREADS>& sh, float* x_at, int* seg, uint64_t* ahead) {
  constexpr int EPV = Elem<T>::kVec;
  static_assert(G <= THREADS / 64, "a wave per block of the segment");
  uint64_t before;
  int s = find_running<THREADS>(entry, nseg, goal, sh, &before);
  s = s < nseg ? s : nseg - 1;
  *seg = s;
  *ahead = before;
  // its blocks, a wave each
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (s * G + wave) * 64 + lane;
  float x[EPV], kept[EPV];
  uint64_t w[EPV], mine = 0ull, incl = 0ull;
#pragma unroll
  for (int e = 0; e < EPV; ++e) { x[e] = -INFINITY; w[e] = 0ull; }
  if (wave < G) {
    if (c < rv.nvec) {
      Elem<T>::unpack(rv.load(c), x);
#pragma unroll
      for (int e = 0; e < EPV; ++e) kept[e] = x[e];
      weights_of(kept, rv.col0(c), w);
#pragma unroll
      for (int e = 0; e < EPV; ++e) mine += w[e];
    }
    incl = wave_incl_u64(mine);
    if (lane == 63) sh.redu[wave] = incl;
  }
  __syncthreads();
  for (int g = 0; g < G; ++g) if (g < wave) before += sh.redu[g];
  if (wave < G) {
    uint64_t run = before + (incl - mine);
    int hit = -1, last = -1;
    float hit_x = 0.f, last_x = 0.f;
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      run += w[e];
      if (w[e] != 0ull) {
        last = rv.col0(c) + e;
        last_x = x[e];
        if (hit < 0 && run >= goal) { hit = last; hit_x = x[e]; }
      }
    }
    // the first hit of the wave; of the waves' again the first
    const unsigned long long any = __ballot(hit >= 0), some = __ballot(last >= 0);
    if (any != 0ull ? lane == __builtin_ctzll(any) : lane == 0) { sh.hits[wave] = hit; sh.hitx[wave] = hit_x; }
    if (some != 0ull ? lane == 63 - __builtin_clzll(some) : lane == 0) { sh.lasts[wave] = last; sh.lastx[wave] = last_x; }
  }
  __syncthreads();
  int col = -1;
  float xc = 0.f;
  for (int g = G - 1; g >= 0; --g) if (sh.hits[g] >= 0) { col = sh.hits[g]; xc = sh.hitx[g]; }
  if (col < 0)
    for (int g = 0; g < G; ++g) if (sh.lasts[g] >= 0) { col = sh.lasts[g]; xc = sh.lastx[g]; }
  __syncthreads();
  *x_at = xc;
  return col;
}

// fn(vector, its index) for the vectors of each segment, a wave a segment, and done(segment) behind them;
// the next segment's loads are in flight meanwhile ([512,128256] min-p on flat rows: 94 us without, 92 with).
template <typename T, int THREADS, int G, typename F, typename D>
__device__ __forceinline__ void each_segment(const RowView<T>& rv, int nseg, F fn, D done) {
  const int tid = thread_here();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  u32x4 next[G];
  rv.template load_some<64, G>(wave * seg_vecs(G) + (tid & 63), next);
  for (int s = wave; s < nseg; s += THREADS / 64) {
    const int c0 = s * seg_vecs(G) + (tid & 63);
    u32x4 raw[G];
#pragma unroll
    for (int i = 0; i < G; ++i) raw[i] = next[i];
    rv.template load_some<64, G>(c0 + THREADS * G, next);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int c = c0 + i * 64;
      touch_whole(raw[i]);
      if (c < rv.nvec) {
        if (!rv.whole(c)) raw[i] = rv.partial(c);
        fn(raw[i], c);
      }
    }
    done(s);
  }
}

// Search by the bits of the value, over the row: the key among [lo, hi] at which the running amount, in
// descending order of value and `ahead` at the start, reaches `goal`; *above gets the amount above that
// key. amount(x) is what an element adds, an integer. 2048 equal ranges of keys a round. Equal
// neighbours of a thread are added up before they go to the histogram, so that a row of few values does
// not queue on few addresses.
template <typename T, int THREADS, typename F>
__device__ __forceinline__ uint32_t key_search(const RowView<T>& rv, uint32_t lo, uint32_t hi, uint64_t ahead,
                                               uint64_t goal, F amount, SampleShared<THREADS>& sh, uint64_t* above) {
  while (lo < hi) {
    const int bits = 32 - __builtin_clz(hi - lo);
    const int shift = bits > 11 ? bits - 11 : 0;
    __syncthreads();
    for (int i = thread_here(); i < kBins; i += THREADS) sh.h.bins[i] = 0ull;
    __syncthreads();
    int open = -1;
    uint64_t held = 0ull;
    each_element<T, THREADS>(rv, [&](float x, int col) {
      const uint32_t key = key_of(x);
      if (key < lo || key > hi || col < 0 || col >= rv.v) return;
      const int b = (int)((hi - key) >> shift);
      if (b != open) {
        if (open >= 0) atomicAdd(&sh.h.bins[open], (unsigned long long)held);
        open = b;
        held = 0ull;
      }
      held += amount(x);
    });
    if (open >= 0) atomicAdd(&sh.h.bins[open], (unsigned long long)held);
    __syncthreads();
    uint64_t before;
    int b = find_running<THREADS>([&](int i) { return (uint64_t)sh.h.bins[i]; }, kBins, goal - ahead, sh, &before);
    b = b < kBins ? b : kBins - 1;       // (some range reaches it)
    ahead += before;
    const uint32_t top = hi - ((uint32_t)b << shift);
    const uint32_t span = (1u << shift) - 1u;
    lo = top - lo > span ? top - span : lo;
    hi = top;
  }
  __syncthreads();
  *above = ahead;
  return lo;
}

// Column of the c-th (1-based) element equal to x0 > -inf in index order; INT_MAX when there are no more
// than c.
template <typename T, int THREADS, int G>
__device__ __forceinline__ int nth_equal(const RowView<T>& rv, int nseg, float x0, int c, SampleShared<THREADS>& sh) {
  constexpr int EPV = Elem<T>::kVec;
  auto equal = [&](float* x, int, uint64_t* w) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < EPV; ++e) w[e] = x[e] == x0 ? 1ull : 0ull;
  };
  int count = 0;
  __syncthreads();
  each_segment<T, THREADS, G>(rv, nseg,
      [&](const u32x4& r, int) {
        float x[EPV];
        Elem<T>::unpack(r, x);
#pragma unroll
        for (int e = 0; e < EPV; ++e) count += x[e] == x0 ? 1 : 0;
      },
      [&](int s) {
        const int all = wave_sum_i(count);
        if ((threadIdx.x & 63) == 0) sh.ties[s] = all;
        count = 0;
      });
  __syncthreads();
  uint64_t mine = 0ull;
  for (int i = thread_here(); i < nseg; i += THREADS) mine += (uint64_t)sh.ties[i];
  const uint64_t all = uniform(block_sum_int64<THREADS / 64>(mine, sh.redu));
  if ((uint64_t)c >= all) return 0x7fffffff;
  float x;
  uint64_t before;
  int s;
  return pick<T, THREADS, G>(rv, nseg, [&](int i) { return (uint64_t)sh.ties[i]; }, (uint64_t)c, equal, sh, &x, &s, &before);
}

// Few entries, their amounts in sh.h.mass: fn(i, amount ahead of entry i, its own, all) for each of them, on
// every lane of the eight that share it, where `ahead` counts the entries that are larger than it as
// `key` puts them. Each is compared with each, which for a few hundred is quicker than a histogram with a
// search in it, or a sort ([1,128256] bf16 min-p: 12 us, 15 without; top-p 0.9: 39, 43 without). The amounts
// are integers, the sums exact.
template <int THREADS, typename K, typename F>
__device__ __forceinline__ void each_of_few(const uint64_t* from, int n, SampleShared<THREADS>& sh, K key, F fn) {
  const int tid = thread_here(), part = tid & 7;
  for (int i0 = 0; i0 < n; i0 += THREADS / 8) {
    const int i = i0 + (tid >> 3);
    const auto mine = key(from[i < n ? i : n - 1]);
    uint64_t ahead = 0ull, all = 0ull;
    for (int o = part; o < n; o += 8) {
      const uint64_t w = sh.h.mass[o];
      all += w;
      ahead += key(from[o]) > mine ? w : 0ull;
    }
#pragma unroll
    for (int d = 1; d < 8; d *= 2) {
      ahead += __shfl_xor(ahead, d, 64);
      all += __shfl_xor(all, d, 64);
    }
    if (i < n) fn(i, ahead, sh.h.mass[i], all);
  }
}

// sh.h.step[0 .. n) in descending order (n <= kStep), by the workgroup
template <int THREADS>
__device__ __forceinline__ void sort_step(SampleShared<THREADS>& sh, int n) {
  int N = 2;
  while (N < n) N *= 2;
  for (int i = n + thread_here(); i < N; i += THREADS) sh.h.step[i] = 0ull;
  __syncthreads();
  for (int k = 2; k <= N; k *= 2) {
    for (int j = k / 2; j > 0; j /= 2) {
      for (int p = thread_here(); p < N / 2; p += THREADS) {
        const int i = 2 * p - (p & (j - 1)), o = i + j;
        const uint64_t a = sh.h.step[i], b = sh.h.step[o];
        const bool up = (i & k) != 0;            // ascending half
        if ((a < b) != up) { sh.h.step[i] = b; sh.h.step[o] = a; }
      }
      __syncthreads();
    }
  }
}

template <typename T, int THREADS, int G>
__global__ __launch_bounds__(THREADS) void sample_kernel(const T* __restrict__ logits, SampleArgs a) {
  constexpr int EPV = Elem<T>::kVec;
  constexpr int NW = THREADS / 64;
  constexpr int kList = SampleShared<THREADS>::kList;
  __shared__ SampleShared<THREADS> sh;
  const int64_t row = blockIdx.x;
  const RowView<T> rv(logits + row * (int64_t)a.v, a.v, sh.edges);
  rv.fill_edges();
  __syncthreads();
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
  auto each = [&](auto fn) { each_vector<T, THREADS>(rv, fn); };
  const int nseg = (rv.nvec + seg_vecs(G) - 1) / seg_vecs(G);
  auto no_row = [&]() {            // no distribution
    if (tid == 0) {
      a.token[row] = -1;
      if (a.logprob != nullptr) a.logprob[row] = __builtin_nanf("");
    }
  };
  auto total_of = [](const double* w) {
    double t = w[0];
#pragma unroll
    for (int e = 1; e < EPV; ++e) t += w[e];
    return t;
  };
  const bool t_ok = T_ >= 0.f && T_ < INFINITY;
  float m;
  uint32_t vouch = 0u;
  const bool whole = t_ok && T_ > 0.f && !use_k && !use_p && !use_m;
  // 2^fx units of mass per 1: the sum of v weights of at most 1 stays at or below 2^63
  const int vbits = a.v > 1 ? 32 - __builtin_clz((unsigned)a.v - 1u) : 0;
  const int fx = 63 - vbits < 50 ? 63 - vbits : 50;
  const double unit = __builtin_amdgcn_ldexp(1.0, fx);
  // w * unit to the nearest integer (w <= 1 and unit <= 2^50: below 2^52), above the bits of 2^52
  constexpr uint64_t kAbove = 0x4330000000000000ull;
  auto fixed_above = [&](double w) { return __builtin_bit_cast(uint64_t, __builtin_fma(w, unit, 4503599627370496.0)); };
  auto fixed = [&](double w) { return fixed_above(w) - kAbove; };
  if (whole) {
    // Nothing cuts: one sweep, each segment's weights against its own maximum, brought together below.
    const double c = kLog2ed / (double)T_;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int s = wave; s < nseg; s += NW) {
      const int c0 = s * seg_vecs(G) + (tid & 63);
      u32x4 raw[G];
      rv.template load_some<64, G>(c0, raw);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        touch_whole(raw[i]);
        if (c0 + i * 64 < rv.nvec) {
          if (!rv.whole(c0 + i * 64)) raw[i] = rv.partial(c0 + i * 64);
          float x[EPV];
          Elem<T>::unpack(raw[i], x);
#pragma unroll
          for (int e = 0; e < EPV; ++e) top = __builtin_elementwise_maximum(top, x[e]);
        }
      }
      top = group_reduce<64, OpMaximum>(top);
      double mine = 0.0;
      if (top > -INFINITY && top < INFINITY) {
        const Weight seg_weight((double)top, c);
#pragma unroll
        for (int i = 0; i < G; ++i) {
          if (c0 + i * 64 < rv.nvec) {
            float x[EPV];
            double w[EPV];
            Elem<T>::unpack(raw[i], x);
            seg_weight.template eval<EPV>(x, w);
            mine += total_of(w);
          }
        }
      }
      mine = wave_sum64(mine);
      if ((tid & 63) == 0) { sh.seg[s] = __builtin_bit_cast(uint64_t, mine); sh.segm[s] = top; }
    }
    __syncthreads();
    m = -INFINITY;
    for (int i = tid & 63; i < nseg; i += 64) m = __builtin_elementwise_maximum(m, sh.segm[i]);
    m = uniform(group_reduce<64, OpMaximum>(m));
    if (!(m < INFINITY && m > -INFINITY)) { no_row(); return; }
    for (int i = tid; i < nseg; i += THREADS)
      sh.seg[i] = (uint64_t)__builtin_rint(__builtin_bit_cast(double, sh.seg[i]) *
                                           (exp2_64(((double)sh.segm[i] - (double)m) * c) * unit));
    __syncthreads();
  } else {
    // 1: the maximum; NaN propagates
    float mx = -INFINITY;
    each_vector<T, THREADS>(rv, [&](const u32x4& r, int) {
      float x[EPV];
      Elem<T>::unpack(r, x);
#pragma unroll
      for (int e = 0; e < EPV; ++e) mx = __builtin_elementwise_maximum(mx, x[e]);
    });
    const float wm = group_reduce<64, OpMaximum>(mx);
    // A value that at least k elements are not below: in each wave the ceil(k / waves)-th largest of the
    // threads' maxima, found bit by bit with ballots, and the least of those over the waves.
    if (use_k && k <= 64 * NW) {
      const uint32_t key = key_of(mx);
      const int q = (k + NW - 1) / NW;
      for (uint32_t bit = 0x80000000u; bit != 0u; bit >>= 1)
        if (__builtin_popcountll(__ballot(key >= (vouch | bit))) >= q) vouch |= bit;
    }
    if ((tid & 63) == 0) { sh.redf[0][tid >> 6] = wm; sh.redi[tid >> 6] = (int)vouch; }
    __syncthreads();
    m = sh.redf[0][0];
    vouch = (uint32_t)sh.redi[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) {
      m = __builtin_elementwise_maximum(m, sh.redf[0][i]);
      vouch = (uint32_t)sh.redi[i] < vouch ? (uint32_t)sh.redi[i] : vouch;
    }
    m = uniform(m);
    vouch = (uint32_t)uniform((int)vouch);
    // (NaN compares false everywhere)
    if (!(m < INFINITY && m > -INFINITY) || !t_ok) { no_row(); return; }
  }
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
  const Weight base((double)m, uniform(kLog2ed / (double)T_));
  Cut cut{-INFINITY, -1};           // -inf itself is never kept
  auto kept = [&](float x, int col) { return x > cut.x || (x == cut.x && col <= cut.col); };
  // a vector's elements that are cut become -inf: one comparison each but in the vector of cut.col itself
  auto mask = [&](float* x, int col0) __attribute__((always_inline)) {
    const float from = col0 + EPV - 1 <= cut.col ? cut.x : float_of_key(key_of(cut.x) + 1u);
    if (col0 <= cut.col && cut.col < col0 + EPV - 1) {
#pragma unroll
      for (int e = 0; e < EPV; ++e) x[e] = kept(x[e], col0 + e) ? x[e] : -INFINITY;
    } else {
#pragma unroll
      for (int e = 0; e < EPV; ++e) x[e] = x[e] >= from ? x[e] : -INFINITY;
    }
  };
  int ties = 0;                     // > 0: so many of the elements equal to cut.x stay, and cut.col is not known
  if (!whole) {
    float x_min = -INFINITY;          // min-p: the least value with a weight of min_p
    if (use_m) {
      const double xm = (double)m + (double)T_ * (log2_64((double)min_p) * kLn2d);
      x_min = (float)xm;                      // may be -inf: then everything stays
      if ((double)x_min < xm) x_min = float_of_key(key_of(x_min) + 1u);      // the next float up
      if (x_min > m) x_min = m;
    }
    auto value = [](uint64_t e) { return float_of_key((uint32_t)(e >> 32)); };
    auto column = [](uint64_t e) { return (int)~(uint32_t)e; };

    // steps of equal width from the maximum down
    float per = 0.f;
    const float last_bin = (float)(kBins - 1);
    auto steps_over = [&](float range) {
      per = (float)(kBins - 2) / range;
      if (!(per <= 1e30f)) per = 1e30f;
    };
    // What lies further below the maximum than T log(n / (1 - p)) has less than 1 - p of the mass of n
    // elements: top-p cuts above that.
    auto reach = [&](int n) { return T_ * (0.6931472f * fast_log2((float)n / fmaxf(1.f - p, 5.9604645e-8f)) + 0.01f); };
    auto step_of = [&](float x) { return (m - x) * per; };       // grows as x falls; never NaN

    // 2: the list of candidates
    float bound = x_min;
    bool listed = false;
    int n = 0, nb = 0;
    auto entry_of = [&](const u32x4& r, int c, int e) __attribute__((always_inline)) {
      return ((uint64_t)key_of(element<T>(r, e)) << 32) | (uint32_t)~(uint32_t)(rv.col0(c) + e);
    };
    // `entry` of the lanes `who` behind what the waves before this one put there; false past the end
    auto put = [&](int& count, uint64_t* to, int room, unsigned long long who, bool mine, uint64_t entry) __attribute__((always_inline)) {
      int base = 0;
      const int first = __builtin_ctzll(who);
      if ((threadIdx.x & 63) == first) base = atomicAdd(&count, (int)__builtin_popcountll(who));
      base = __builtin_amdgcn_readlane(base, first);
      const int at = base + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
      if (mine && at < room) to[at] = entry;
      return base + (int)__builtin_popcountll(who) <= room;
    };
    // The list: what the cut so far keeps and is not below `bound`, or (by_step) lies in the steps before `hi`.
    auto list_up = [&](bool by_step, float hi) __attribute__((always_inline)) {
      const bool restricted = cut.x > -INFINITY;
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
      bool full = false;
      each([&](const u32x4& r, int c) {
        if (full) return;
        float x[EPV];
        Elem<T>::unpack(r, x);
        if (restricted) mask(x, rv.col0(c));
        float top = x[0];
#pragma unroll
        for (int e = 1; e < EPV; ++e) top = __builtin_elementwise_maximum(top, x[e]);
        if (__ballot(by_step ? step_of(top) < hi : top >= bound) == 0ull) return;
        uint32_t todo = 0u;       // a bit per element
#pragma unroll
        for (int e = 0; e < EPV; ++e)
          todo |= (by_step ? step_of(x[e]) < hi : x[e] >= bound && x[e] > -INFINITY) ? 1u << e : 0u;
        while (!full) {
          const unsigned long long who = __ballot(todo != 0u);
          if (who == 0ull) break;
          const int e = todo != 0u ? __builtin_ctz(todo) : 0;
          full = !put(sh.count, sh.h.list, kList, who, todo != 0u, entry_of(r, c, e));
          todo &= todo - 1u;
        }
      });
      __syncthreads();
      n = uniform(sh.count);
      listed = n <= kList;
      __syncthreads();
    };
    // One step from the row: its elements, unless they are known to be too many (over), and their ends.
    auto step_up = [&](float lo, float hi, bool over) __attribute__((always_inline)) {
      const bool restricted = cut.x > -INFINITY;
      __syncthreads();
      if (tid == 0) { sh.at = over ? kStep + 1 : 0; sh.klo = 0xFFFFFFFFu; sh.khi = 0u; }
      __syncthreads();
      float step_min = INFINITY, step_max = -INFINITY;
      each([&](const u32x4& r, int c) {
        float x[EPV];
        Elem<T>::unpack(r, x);
        if (restricted) mask(x, rv.col0(c));
        uint32_t todo = 0u;
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
          const float y = step_of(x[e]);
          const bool in = y >= lo && y < hi;
          step_min = __builtin_elementwise_minimum(step_min, in ? x[e] : INFINITY);
          step_max = __builtin_elementwise_maximum(step_max, in ? x[e] : -INFINITY);
          if (!over) todo |= in ? 1u << e : 0u;
        }
        while (!over) {
          const unsigned long long who = __ballot(todo != 0u);
          if (who == 0ull) break;
          const int e = todo != 0u ? __builtin_ctz(todo) : 0;
          over = !put(sh.at, sh.h.step, kStep, who, todo != 0u, entry_of(r, c, e));
          todo &= todo - 1u;
        }
      });
      if (step_min <= step_max) {
        atomicMin(&sh.klo, key_of(step_min));
        atomicMax(&sh.khi, key_of(step_max));
      }
      __syncthreads();
      nb = uniform(sh.at);
      __syncthreads();
    };

    // the amounts of entries, 0 for what the cut so far does not keep, into sh.h.mass
    auto amounts = [&](const uint64_t* from, int many, auto by_count) __attribute__((always_inline)) {
      const Weight weight = base.fresh();
#pragma unroll 1
      for (int i = tid; i < many; i += THREADS) {
        const uint64_t e = from[i];
        sh.h.mass[i] = !kept(value(e), column(e)) ? 0ull : decltype(by_count)::value ? 1ull : fixed(weight(value(e)));
      }
      __syncthreads();
    };

    // 3: the exact cuts, first by count, then by the mass of what that leaves. The cut is the first element,
    // in descending order, at which the running amount reaches the goal (the mass before it is below p times
    // the whole: the first multiple of the unit that is not).
    auto goal_of = [&](uint64_t mass) {
      const uint64_t g = (uint64_t)__builtin_ceil((double)p * (double)mass);
      return uniform(g > 1ull ? g : (uint64_t)1);
    };
    if (use_k) {
      bound = vouch <= 0x007FFFFFu ? -INFINITY : float_of_key(vouch);      // that is key_of(-inf)
      const float range = m - bound;
      steps_over(range < INFINITY ? range : 24.f * T_);
    } else {
      steps_over(reach(a.v));
    }
    // (with top-p alone there is no bound to list by)
    if (use_k ? bound > -INFINITY || a.v <= kList : !use_p) list_up(false, 0.f);
    auto settle = [&](auto by_count) __attribute__((always_inline)) {
      constexpr bool count = decltype(by_count)::value;
      if (count && listed && n < k) return;         // all of them stay
      const bool by_list = listed;
      const bool restricted = cut.x > -INFINITY;
      if (!by_list && use_k && !count) steps_over(reach(k));
      __syncthreads();
      for (int i = tid; i < kBins; i += THREADS) sh.h.bins[i] = 0ull;
      __syncthreads();
      // the amount by step
      const Weight weight = base.fresh();
      uint64_t goal = (uint64_t)(count ? k : 0);
      if (by_list) {
        uint64_t mine = 0ull;
#pragma unroll 1
        for (int i = tid; i < n; i += THREADS) {
          const uint64_t e = sh.h.list[i];
          if (!kept(value(e), column(e))) continue;
          const uint64_t w = count ? 1ull : fixed(weight(value(e)));
          const float y = step_of(value(e));
          atomicAdd(&sh.h.bins[y < last_bin ? (int)y : kBins - 1], (unsigned long long)w);
          mine += w;
        }
        if (!count) goal = goal_of(block_sum_int64<NW>(mine, sh.redu));
      } else {
        uint64_t total = 0ull;
        each([&](const u32x4& r, int c) {
          float x[EPV];
          Elem<T>::unpack(r, x);
          if (restricted) mask(x, rv.col0(c));
          if (count) {
#pragma unroll
            for (int e = 0; e < EPV; ++e) {
              const float y = step_of(x[e]);
              if (y < last_bin) atomicAdd(&sh.h.bins[(int)y], 1ull);
            }
          } else {
            double w[EPV];
            weight.template eval<EPV>(x, w);
            total -= EPV * kAbove;
#pragma unroll
            for (int e = 0; e < EPV; ++e) {
              const uint64_t f = fixed_above(w[e]);
              total += f;
              const float y = step_of(x[e]);
              if (y < last_bin) atomicAdd(&sh.h.bins[(int)y], (unsigned long long)(f - kAbove));
            }
          }
        });
        if (!count) goal = goal_of(block_sum_int64<NW>(total, sh.redu));
      }
      __syncthreads();
      // the step that holds the cut, its elements in sh.h.step
      uint64_t ahead;
      const int b = find_running<THREADS>([&](int i) { return (uint64_t)sh.h.bins[i]; }, kBins, goal, sh, &ahead);
      if (by_list && b == kBins) return;         // everything stays
      if (!by_list && b < kBins) {
        // How many there are at least, from the mass and the largest weight of each step: rows whose list or
        // step is sure to overflow spare the way there.
        float most = 0.f, in_b = 0.f;
        for (int i = tid; i <= b; i += THREADS) {
          const float least = count ? (float)sh.h.bins[i]
                                    : (float)sh.h.bins[i] * fast_exp2((float)i / per * (float)base.c - (float)fx);
          most += least;
          if (i == b) in_b = least;
        }
        most = (float)block_reduce64<NW, Sum64>((double)most, sh.red);
        in_b = (float)block_reduce64<NW, Sum64>((double)in_b, sh.red);
        if (uniform(most) <= 1.01f * kList) list_up(true, (float)(b + 1));
        if (!listed) step_up((float)b, (float)(b + 1), uniform(in_b) > 1.01f * kStep);
      }
      if (listed) {
        if (tid == 0) { sh.at = 0; sh.klo = 0xFFFFFFFFu; sh.khi = 0u; }
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < n; i += THREADS) {
          const uint64_t e = sh.h.list[i];
          const float y = step_of(value(e));
          if ((y < last_bin ? (int)y : kBins - 1) == b && kept(value(e), column(e))) {
            const int at = atomicAdd(&sh.at, 1);
            if (at < kStep) sh.h.step[at] = e;
            atomicMin(&sh.klo, (uint32_t)(e >> 32));
            atomicMax(&sh.khi, (uint32_t)(e >> 32));
          }
        }
        __syncthreads();
        nb = uniform(sh.at);
      }
      if (b < kBins && nb <= kFew) {
        amounts(sh.h.step, nb, by_count);
        if (tid == 0) sh.at = 0;
        __syncthreads();
        const uint64_t left = goal - ahead;
        each_of_few<THREADS>(sh.h.step, nb, sh, [](uint64_t e) { return e; },
            [&](int i, uint64_t before, uint64_t w, uint64_t) {
              if (before < left && left <= before + w) sh.at = i;      // one entry
            });
        __syncthreads();
        cut.x = uniform(value(sh.h.step[sh.at]));
        cut.col = uniform(column(sh.h.step[sh.at]));
        __syncthreads();
        return;
      }
      if (b < kBins && nb <= kStep) {
        sort_step<THREADS>(sh, nb);
        uint64_t unused;
        int r = find_running<THREADS>(
            [&](int i) { return count ? (uint64_t)1 : fixed(weight(value(sh.h.step[i]))); }, nb, goal - ahead, sh, &unused);
        r = r < nb ? r : nb - 1;
        cut.x = uniform(value(sh.h.step[r]));
        cut.col = uniform(column(sh.h.step[r]));
        return;
      }
      // More elements than that: by the bits of the value, then by column among equal ones.
      uint32_t lo = 0u, hi = 0xFFFFFFFEu;
      uint64_t above = 0ull;
      if (b < kBins) {
        lo = (uint32_t)uniform((int)sh.klo);
        hi = (uint32_t)uniform((int)sh.khi);
        above = ahead;
      }
      const uint32_t key = key_search<T, THREADS>(
          rv, lo, hi, above, goal, [&](float x) { return count ? (uint64_t)1 : fixed(weight(x)); }, sh, &above);
      const float x = float_of_key(key);
      const uint64_t each_w = count ? (uint64_t)1 : fixed(weight(x));
      // the r-th of the equal ones stays iff above + (r - 1) * weight < goal
      const uint64_t left = goal - above;
      uint64_t r = each_w > 0ull ? (uint64_t)((double)left / (double)each_w) : 1ull;       // the quotient, or one off
      if (r * each_w < left) ++r;
      if (r > 1ull && (r - 1ull) * each_w >= left) --r;
      const int need = uniform((int)(r > 1ull ? r : 1ull));
      if (!count || !use_p) {       // the last cut: the sweep below counts the equal ones by the way
        listed = false;
        if (x > cut.x) {
          cut = Cut{x, -1};
          ties = need;
          return;
        }
      }
      const int col = x >= cut.x && x > -INFINITY ? nth_equal<T, THREADS, G>(rv, nseg, x, need, sh) : -1;
      if (x > cut.x || (x == cut.x && col < cut.col)) cut = Cut{x, col};
      listed = listed && b < kBins;
    };
    if (use_k) settle(std::true_type{});
    if (use_p) settle(std::false_type{});
    if (x_min > cut.x) {       // every value equal to the bound stays
      ties = 0;
      cut.x = x_min;
      cut.col = 0x7fffffff;
    }

    // 4 on the list
    if (listed && n <= kFew) {
      amounts(sh.h.list, n, std::false_type{});
      // larger: of a lower index
      each_of_few<THREADS>(sh.h.list, n, sh, [](uint64_t e) { return (uint32_t)e; },
          [&](int i, uint64_t ahead, uint64_t w, uint64_t all) {
            const uint64_t target = (uint64_t)(u * (double)all);
            if ((tid & 7) == 0 && ahead <= target && target < ahead + w) {
              const uint64_t e = sh.h.list[i];
              a.token[row] = column(e);
              if (a.logprob != nullptr)
                a.logprob[row] = (float)(log2_64(base(value(e)) * unit / (double)all) * kLn2d);
            }
          });
      return;
    }
    if (listed) {
      constexpr int PER = (kList + THREADS - 1) / THREADS;
      int shift = 6;
      while ((rv.nvec >> shift) >= kBins) ++shift;
      const uint32_t seg_bits = (EPV == 8 ? 3 : 2) + shift;             // a segment has at most kStep elements
      __syncthreads();
      for (int i = tid; i < kBins; i += THREADS) sh.h.bins[i] = 0ull;
      __syncthreads();
      const Weight weight = base.fresh();
      uint64_t me[PER], w[PER], mine = 0ull;
      int seg[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = j * THREADS + tid;
        seg[j] = -1;
        if (j * THREADS >= n) continue;
        if (i >= n) continue;
        me[j] = sh.h.list[i];
        if (!kept(value(me[j]), column(me[j]))) continue;
        w[j] = fixed(weight(value(me[j])));
        seg[j] = (int)(((uint32_t)column(me[j]) + (uint32_t)rv.lead) >> seg_bits);
        atomicAdd(&sh.h.bins[seg[j]], (unsigned long long)w[j]);
        mine += w[j];
      }
      const double mass = uniform((double)block_sum_int64<NW>(mine, sh.redu));
      const uint64_t target = uniform((uint64_t)(u * mass));
      uint64_t ahead;
      const int s = find_running<THREADS>([&](int i) { return (uint64_t)sh.h.bins[i]; }, kBins, target + 1ull, sh, &ahead);
      if (tid == 0) sh.at = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (seg[j] == s) {
          const int at = atomicAdd(&sh.at, 1);
          sh.h.step[at] = me[j];
          sh.h.mass[at] = w[j];
        }
      }
      __syncthreads();
      const int ns = uniform(sh.at);
      for (int i = tid; i < ns; i += THREADS) {
        const int col = column(sh.h.step[i]);
        uint64_t before = ahead;
        for (int o = 0; o < ns; ++o) before += column(sh.h.step[o]) < col ? sh.h.mass[o] : 0ull;
        if (before <= target && target < before + sh.h.mass[i]) {
          a.token[row] = col;
          if (a.logprob != nullptr)
            a.logprob[row] = (float)(log2_64(weight(value(sh.h.step[i])) * unit / mass) * kLn2d);
        }
      }
      return;
    }
  }

  // 4 over the row: kept mass by segment, in index order (the weight of -inf is 0). Vectors without a kept
  // element cost their comparison only.
  const Weight weight = base.fresh();
  auto kept_doubles = [&](float* x, int col0, double* w) __attribute__((always_inline)) {
    float top = x[0];
#pragma unroll
    for (int e = 1; e < EPV; ++e) top = __builtin_elementwise_maximum(top, x[e]);
    if (__ballot(top >= cut.x) == 0ull) return false;
    mask(x, col0);
    weight.template eval<EPV>(x, w);
    return true;
  };
  auto kept_weights = [&](float* x, int col0, uint64_t* w) __attribute__((always_inline)) {
    double wd[EPV];
    if (!kept_doubles(x, col0, wd)) return;
#pragma unroll
    for (int e = 0; e < EPV; ++e) w[e] = fixed(wd[e]);
  };
  auto equal = [&](float* x, int, uint64_t* w) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < EPV; ++e) w[e] = x[e] == cut.x ? 1ull : 0ull;
  };
  int at_seg;
  float x_at;
  uint64_t ahead;
  if (!whole) {
    __syncthreads();
    uint64_t mine = 0ull;
    int equals = 0;
    each_segment<T, THREADS, G>(rv, nseg,
        [&](const u32x4& r, int c) {
          float x[EPV];
          Elem<T>::unpack(r, x);
          if (ties > 0) {
#pragma unroll
            for (int e = 0; e < EPV; ++e) equals += x[e] == cut.x ? 1 : 0;
          }
          double w[EPV];
          if (kept_doubles(x, rv.col0(c), w)) {
            mine -= EPV * kAbove;
#pragma unroll
            for (int e = 0; e < EPV; ++e) mine += fixed_above(w[e]);
          }
        },
        [&](int s) {
          mine = wave_sum_u64(mine);
          const int all_equals = ties > 0 ? wave_sum_i(equals) : 0;
          if ((tid & 63) == 0) { sh.seg[s] = mine; sh.ties[s] = all_equals; }
          mine = 0ull;
          equals = 0;
        });
    __syncthreads();
    if (ties > 0) {
      uint64_t mine = 0ull;
      for (int i = tid; i < nseg; i += THREADS) mine += (uint64_t)sh.ties[i];
      int s_cut = nseg;
      uint64_t before = 0ull;
      cut.col = 0x7fffffff;
      if ((uint64_t)ties < uniform(block_sum_int64<NW>(mine, sh.redu)))
        cut.col = pick<T, THREADS, G>(rv, nseg, [&](int i) { return (uint64_t)sh.ties[i]; }, (uint64_t)ties, equal, sh, &x_at, &s_cut, &before);
      const uint64_t each_w = fixed(weight(cut.x));
      __syncthreads();
      for (int i = tid; i < nseg; i += THREADS)
        sh.seg[i] += each_w * (i < s_cut ? (uint64_t)sh.ties[i] : i == s_cut ? (uint64_t)ties - before : (uint64_t)0);
      __syncthreads();
    }
  }
  uint64_t mine = 0ull;
  for (int i = tid; i < nseg; i += THREADS) mine += sh.seg[i];
  const double mass = uniform((double)block_sum_int64<NW>(mine, sh.redu));
  const uint64_t goal = uniform((uint64_t)(u * mass)) + 1ull;
  const int col = pick<T, THREADS, G>(rv, nseg, [&](int i) { return sh.seg[i]; }, goal, kept_weights, sh, &x_at, &at_seg, &ahead);
  if (tid == 0) {
    a.token[row] = col;
    if (a.logprob != nullptr) a.logprob[row] = (float)(log2_64(weight(x_at) * unit / mass) * kLn2d);
  }
}

template <typename T>
void launch(const void* logits, const SampleArgs& a, int64_t n, hipStream_t st) {
  const int64_t nvec = a.v / Elem<T>::kVec + 2;
#define GO(TH, G) FM_LAUNCH((sample_kernel<T, TH, G>), dim3((unsigned)n), dim3(TH), 0, st, static_cast<const T*>(logits), a)
  // Short rows: four waves, a block of 64 vectors a segment, so that each wave has segments to sweep
  // ([2048,8000] bf16 top-p 0.9: 84 us with 512 threads, 68 with these). Rows for which there is a compute
  // unit each: all of its waves ([1,128256] top-p 0.95: 46 us with 512 threads, 40 with these; [256,128256]
  // top-k 50 is slower by it, 30 and 33). More rows: half-size workgroups, two rows a unit in different phases
  // ([1024,32000] top-p 0.9: 130 us with the large ones, 103 with these; where a quarter of 512 rows of min-p
  // is flat it is the other way round, 79 and 88). The choice does not show in the results.
  if (nvec <= 1024) GO(256, 1);
  else if (n <= fm_host::num_cus()) GO(1024, 4);
  else GO(512, 4);
#undef GO
}

}  // namespace

extern "C" int fm_sample(const void* logits, const float* u, const float* temperature, const int32_t* top_k,
                         const float* top_p, const float* min_p, float temperature0, int top_k0, float top_p0,
                         float min_p0, int64_t* token, float* logprob, int64_t n, int64_t v, int dtype,
                         fm_stream_t stream) {
  FM_CHECK_ARG(n >= 0 && v > 0, "fm_sample: bad shape n=%lld v=%lld", (long long)n, (long long)v);
  FM_CHECK_ARG(dtype == FM_F32 || dtype == FM_F16 || dtype == FM_BF16, "fm_sample: bad dtype %d", dtype);
  // (a launch has less than 2^32 threads, and a row up to 1024)
  if (n >= (1LL << 22) || v > kMaxCols) {
    fm_host::set_error("fm_sample: n must be below 2^22 and v at most %lld", (long long)kMaxCols);
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
