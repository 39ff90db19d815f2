// KL(teacher || student) from a teacher that is known at k listed columns of each row, forward and
// backward, for gfx950.
//
//   q_j           the teacher's probability of listed column j (softmax over the list, or exp(t - lse))
//   row_loss      sum_j q_j (log q_j - log p_j)  [+ q_r (log q_r - log p_r), the unlisted columns as one]
//   dstudent_j    (p_j sum(q) - q_j) scale;  unlisted, with the bucket: (p_j - q_r p_j / p_r) scale
//
// Bound by the student's row: 2 (+ 2) bytes per 16-bit logit against 12 bytes per listed column. One
// workgroup per row: the list is turned into a small LDS table while the row is on its way into
// registers, the row is folded into a running (maximum, sum) of its columns (of its UNLISTED columns
// where the bucket is wanted: log p_r then never is the log of 1 - sum p, which loses every digit when
// the student agrees with the list), and the gradient is written from the registers.
//
// Every unlisted column's gradient is one coefficient times exp2(z - m): the coefficient, the listed
// columns and the loss are computed in 64 bits by the threads that hold the list (the loss is a small
// difference of terms ten to a hundred times its size), the sweep over the row in fp32.
//
// Measured, lists of 64, loss and gradient from one launch: [8192,32000] bf16 204 us (5.1 TB/s, the rate of a
// copy), [4096,128256] bf16 418 us (5.0), [1024,128256] fp32 with lists of 256 204 us (5.1); losses alone,
// [4096,128256] bf16, 157 to 185 us (5.7 to 6.7 TB/s); loss and gradient in two launches, [1021,50257] fp16,
// 24 and 43 us, one loss a row at [8192,32000] bf16 102 and 183; [16,32000] bf16 14 us, where the steps of
// one row count.
#include "../../include/fm_hip_tokens.h"
#include "fm_f64.hip.h"

using namespace fm;

namespace {

constexpr int kMaxList = 1024;
constexpr int kSmallList = 128;
constexpr uint16_t kEnd = 0xFFFFu;
// up to this many rows every workgroup counts the listed rows itself; beyond, one launch counts
constexpr int kCountInKernel = 256;

struct ListArgs {
  const void* idx;
  const void* teacher;
  const float* teacher_lse;
  int k;
  bool idx64;
  int teacher_dtype;
  int probs;         // FM_TEACHER_PROBS
  int tail;          // FM_TAIL_*
  double inv_t;
  float c;           // log2(e) / temperature, what the logits are multiplied by
};

__device__ __forceinline__ int64_t list_idx(const ListArgs& a, int64_t at) {
  return a.idx64 ? static_cast<const int64_t*>(a.idx)[at] : (int64_t)static_cast<const int32_t*>(a.idx)[at];
}
// A slot's column and teacher value as loaded. The loads name no branch, whatever the two types, and
// nothing is converted yet: the wait for them comes where they are used, behind the row's own loads.
struct SlotBits {
  uint32_t lo, hi;
  uint16_t t0, t1;
};
__device__ __forceinline__ SlotBits slot_load(const ListArgs& a, int64_t at) {
  SlotBits b;
  const char* i = static_cast<const char*>(a.idx) + at * (a.idx64 ? 8 : 4);
  b.lo = *reinterpret_cast<const uint32_t*>(i);
  b.hi = *reinterpret_cast<const uint32_t*>(i + (a.idx64 ? 4 : 0));
  const char* t = static_cast<const char*>(a.teacher) + at * (a.teacher_dtype == FM_F32 ? 4 : 2);
  b.t0 = *reinterpret_cast<const uint16_t*>(t);
  b.t1 = *reinterpret_cast<const uint16_t*>(t + (a.teacher_dtype == FM_F32 ? 2 : 0));
  return b;
}
__device__ __forceinline__ int slot_sign(const ListArgs& a, int64_t at) {
  return static_cast<const int32_t*>(a.idx)[a.idx64 ? at * 2 + 1 : at];
}
__device__ __forceinline__ int64_t slot_col(const ListArgs& a, const SlotBits& b) {
  const uint32_t hi = a.idx64 ? b.hi : (uint32_t)((int32_t)b.lo >> 31);
  return (int64_t)(((uint64_t)hi << 32) | b.lo);
}
__device__ __forceinline__ float slot_value(const ListArgs& a, const SlotBits& b) {
  const uint32_t word = ((uint32_t)b.t1 << 16) | (a.teacher_dtype == FM_F32 ? b.t0 : 0);
  const float half = (float)__builtin_bit_cast(_Float16, b.t0);
  return a.teacher_dtype == FM_F16 ? half : u2f(word);
}

// element d of a packed vector: its value, and the vector with the element's bits replaced
template <typename T>
__device__ __forceinline__ uint32_t word_at(const u32x4& r, int w) {
  const uint32_t a = w & 1 ? r.y : r.x, b = w & 1 ? r.w : r.z;
  return w & 2 ? b : a;
}
template <typename T>
__device__ __forceinline__ float get_elem(const u32x4& r, int d) {
  if constexpr (sizeof(T) == 4) {
    return u2f(word_at<T>(r, d));
  } else {
    const uint32_t w = word_at<T>(r, d >> 1);
    T t;
    t.bits = (uint16_t)(d & 1 ? w >> 16 : w);
    return Elem<T>::load1(&t);
  }
}
template <typename T>
__device__ __forceinline__ void set_elem(u32x4& r, int d, uint32_t bits) {
  uint32_t w = bits;
  int at = d;
  if constexpr (sizeof(T) == 2) {
    at = d >> 1;
    const uint32_t old = word_at<T>(r, at);
    w = d & 1 ? (old & 0xffffu) | (bits << 16) : (old & 0xffff0000u) | bits;
  }
  r.x = at == 0 ? w : r.x;
  r.y = at == 1 ? w : r.y;
  r.z = at == 2 ? w : r.z;
  r.w = at == 3 ? w : r.w;
}
// the bits of a value as stored in T (for the half types in the low 16)
template <typename T>
__device__ __forceinline__ uint32_t bits_of(float f) {
  if constexpr (std::is_same<T, float>::value) return f2u(f);
  else if constexpr (std::is_same<T, bf16_t>::value) return pack_bf16(f, 0.f) & 0xffffu;
  else return pack_f16(f, 0.f) & 0xffffu;
}

// A running (maximum, sum) whose sum is held in 64 bits. Where x * c is so large that fp32 cannot tell the
// maximum from its neighbours (|x c| > 2^31, a row or all of its unlisted columns masked with the type's
// lowest value), the sum is negative and the maximum is the logit itself (exact_pairs).
struct Pair64 {
  float m;
  double s;
  __device__ __forceinline__ double top(float c) const { return s < 0.0 ? (double)m * (double)c : (double)m; }
  __device__ __forceinline__ double sum() const { return __builtin_fabs(s); }
  // the largest weight of a row is 1, off by 2^-25 |x c| in the exponent
  __device__ __forceinline__ bool sound() const { return s >= 0.25 && s <= 1e12; }
};
// An unlisted column's weight is exp2(x * c - m).
struct Sweep {
  float c, m;
};
__device__ __forceinline__ Sweep sweep_of(const Pair64& rest, float c) {
  if (!(rest.s < 0.0)) return Sweep{c, rest.m};
  // 2^7 or more between neighbouring logits: the weight is 1 for the maximum and 0 for everything else,
  // which a power of two in place of c shows without rounding
  int e = 120 - __builtin_amdgcn_frexp_expf(rest.m);
  e = e < 127 ? e : 127;
  const float p = __builtin_amdgcn_ldexpf(1.f, e);
  return Sweep{p, rest.m * p};
}
template <int NW>
struct MergeShared {
  double s[2][NW];
  float m[2][NW];
};
// Workgroup merge of a running pair per thread: one barrier, the sums in 64 bits, fixed order. The factors
// that bring the sums to a common maximum are formed in 64 bits too: the fp32 one is off by up to 6e-8, and
// with the bucket the quotient of two such sums goes into the loss as it is (2e-5 of a loss of 2e-4).
template <int NW>
__device__ __forceinline__ Pair64 merge_pairs(const MaxSum& run, MergeShared<NW>& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float wm = wave_max(run.m);
  const double ws = wave_sum64((double)run.s * exp2_64((double)(run.m - wm)));
  if (lane == 0) { sh.m[0][wave] = wm; sh.s[0][wave] = ws; }
  __syncthreads();
  const float mine = sh.m[0][lane & (NW - 1)];
  const float m = group_reduce<NW, OpMax>(mine);
  return Pair64{m, group_reduce64<NW, Sum64>(sh.s[0][lane & (NW - 1)] * exp2_64((double)(mine - m)))};
}
// The pair of the unlisted columns with `more`, of the thread's listed ones against rest.m, added: another
// barrier. A sum past fp32 (more than a few hundred between the two) is not sound.
template <int NW>
__device__ __forceinline__ Pair64 with_listed(const Pair64& rest, double more, MergeShared<NW>& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  more = wave_sum64(more);
  if (lane == 0) sh.s[1][wave] = more;
  __syncthreads();
  const double s = rest.s + group_reduce64<NW, Sum64>(sh.s[1][lane & (NW - 1)]);
  const double top = (double)rest.m + (double)__builtin_amdgcn_frexp_exp(s);
  const float m = (float)top;
  return Pair64{m, __builtin_amdgcn_frexp_mant(s) * exp2_64(top - (double)m)};
}
// one element into a running pair
__device__ __forceinline__ void fold1(MaxSum& run, float x, float c) {
  const float cm = __builtin_elementwise_maximum(run.m, x * c);
  run.s = run.s * fast_exp2(run.m - cm) + fast_exp2(__builtin_fmaf(x, c, -cm));
  run.m = cm;
}

// The list of one row in LDS: per-thread chains. Chain t holds the listed columns among the vectors that
// thread t sweeps, and bit i % 31 of mask[t] says that there may be one in its i-th vector (bit 31: in
// the row's unaligned ends). A column that occurs twice is found where its chain is walked first; its
// first slot then leads and takes over what the others have, added in slot order.
template <int THREADS, int KCAP>
struct ListShared {
  union {
    double q[KCAP];      // while slots are merged
    struct {
      float x[KCAP];     // the student's logit there
      uint32_t g[KCAP];  // the gradient there, as stored bits
    };
  };
  double red[THREADS / 64];
  MergeShared<THREADS / 64> merge;
  int col[KCAP];         // -1: empty, or merged into another slot
  uint32_t mask[THREADS];
  uint16_t nxt[KCAP];
  uint16_t head[THREADS];
  int redi[THREADS / 64];
  int count[THREADS / 64];
  float top[THREADS / 64];
  int twice;
};

// What a thread keeps of its slots (slot j * THREADS + tid) across the sweep.
template <int SL>
struct Mine {
  int col[SL];       // -1: not the leader of a column
  double q[SL];
};

template <int THREADS, int SL>
__device__ __forceinline__ void list_load(const ListArgs& a, int64_t row, SlotBits (&bits)[SL]) {
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    const int s = j * THREADS + (int)threadIdx.x;
    bits[j] = slot_load(a, row * a.k + (s < a.k ? s : 0));
  }
}

// The first two listed columns of a thread's chain among its vectors 0 .. RI-1, in registers (vector,
// element, slot), and the mask of the vectors that hold more of them. A wave meets a listed column in a
// quarter to most of its vectors; from registers it costs a dozen operations there instead of a walk of
// dependent LDS reads ([8192,32000] bf16, lists of 64: 235 us with the walk, 228 without).
constexpr uint32_t kNone = 0xFFFFFFFFu;
struct Near {
  uint32_t e0, e1;     // vector | element << 8 | slot << 16
  uint32_t more;       // as mask, of what is not e0 or e1
};
// `twice`: set when two entries of the chain name one column (the walk then ends)
template <typename T, int THREADS, int KCAP, int RI>
__device__ __forceinline__ Near near_of(const ListShared<THREADS, KCAP>& sh, const RowSplit& sp, uint16_t head, bool* twice) {
  constexpr int EPV = Elem<T>::kVec;
  Near n{kNone, kNone, 0u};
#pragma unroll 1
  for (uint32_t s = head; s != kEnd; s = sh.nxt[s]) {
    const int col = sh.col[s];
    if (col < 0) continue;
    bool same = false;
#pragma unroll 1
    for (uint32_t o = sh.nxt[s]; o != kEnd && !same; o = sh.nxt[o]) same = sh.col[o] == col;
    if (same) { *twice = true; break; }
    if (col < sp.head || col >= sp.tail0) { n.more |= 1u << 31; continue; }
    const uint32_t vec = (uint32_t)(col - sp.head) / EPV, d = (uint32_t)(col - sp.head) % EPV, i = vec / THREADS;
    const uint32_t e = i | d << 8 | s << 16;
    if (i < (uint32_t)RI && n.e0 == kNone) n.e0 = e;
    else if (i < (uint32_t)RI && n.e1 == kNone) n.e1 = e;
    else n.more |= 1u << (i % 31);
  }
  return n;
}

// Fills the chains and returns the sum of q (NaN when a column is out of range); *unique gets the number
// of distinct columns. Three barriers; columns that occur twice cost three more. Only columns among the
// vectors [c_begin, c_end) and, with `ends`, the row's unaligned ends are hung into chains. All threads
// of the workgroup call it.
template <typename T, int THREADS, int KCAP, int SL, int RI>
__device__ __forceinline__ double list_build(const ListArgs& a, const RowSplit& sp, int v, const SlotBits (&bits)[SL],
                                             float lse_t, int c_begin, int c_end, bool ends,
                                             ListShared<THREADS, KCAP>& sh, Mine<SL>& mine, Near* near, int* unique) {
  constexpr int NW = THREADS / 64;
  constexpr int EPV = Elem<T>::kVec;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool renorm = a.tail == FM_TAIL_RENORM, logits = a.probs == FM_TEACHER_LOGITS;
  sh.mask[tid] = 0u;
  sh.head[tid] = kEnd;
  if (tid == 0) sh.twice = 0;
  bool bad = false;
  float t[SL];
  bool used[SL];
  float mx = -INFINITY;
  int places = 0;
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    const int s = j * THREADS + tid;
    const int64_t c = s < a.k ? slot_col(a, bits[j]) : -1;
    t[j] = slot_value(a, bits[j]);
    used[j] = c >= 0;
    bad |= c >= v;
    mine.col[j] = c >= 0 && c < v ? (int)c : -1;
    if (s < KCAP) sh.col[s] = mine.col[j];
    if (used[j]) mx = fmaxf(mx, t[j]);
    places += mine.col[j] >= 0 ? 1 : 0;
  }
  if (renorm && logits) {
    mx = wave_max(mx);
    if (lane == 0) sh.top[wave] = mx;
  }
  __syncthreads();
  // teacher probabilities, and the slots into the chains of the threads that sweep their columns
  const double shift = !logits ? 0.0
                       : renorm ? (double)group_reduce<NW, OpMax>(sh.top[lane & (NW - 1)]) * a.inv_t : (double)lse_t;
  double sum = bad ? __builtin_nan("") : 0.0;
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    const int s = j * THREADS + tid, col = mine.col[j];
    mine.q[j] = 0.0;
    if (used[j]) mine.q[j] = logits ? exp2_64(((double)t[j] * a.inv_t - shift) * kLog2ed) : (double)t[j];
    sum += mine.q[j];
    if (col < 0) continue;
    int owner;
    uint32_t bit;
    if (col >= sp.head && col < sp.tail0) {
      const int vec = (col - sp.head) / EPV;
      if (vec < c_begin || vec >= c_end) continue;
      owner = vec % THREADS;
      bit = 1u << ((vec / THREADS) % 31);
    } else {
      if (!ends) continue;
      owner = (col < sp.head ? col : sp.head + (col - sp.tail0)) % THREADS;
      bit = 1u << 31;
    }
    atomicOr(&sh.mask[owner], bit);
    // 16-bit exchange on the 32-bit word that holds the head
    uint32_t* word = reinterpret_cast<uint32_t*>(&sh.head[owner & ~1]);
    const int shift16 = (owner & 1) * 16;
    uint32_t old = *word, seen;
    do {
      seen = old;
      const uint32_t now = (seen & ~(0xFFFFu << shift16)) | ((uint32_t)s << shift16);
      old = atomicCAS(word, seen, now);
    } while (old != seen);
    sh.nxt[s] = (uint16_t)(seen >> shift16);
  }
  sum = wave_sum64(sum);
  places = wave_sum_i(places);
  if (lane == 0) { sh.red[wave] = sum; sh.redi[wave] = places; }
  __syncthreads();
  bool twice = false;
  *near = near_of<T, THREADS, KCAP, RI>(sh, sp, sh.head[tid], &twice);
  if (twice) sh.twice = 1;
  sum = group_reduce64<NW, Sum64>(sh.red[lane & (NW - 1)]);
  int u = 0;
  for (int i = 0; i < NW; ++i) u += sh.redi[i];
  if (renorm) {
    const double r = 1.0 / sum;
#pragma unroll
    for (int j = 0; j < SL; ++j) mine.q[j] *= r;
    sum = sum * r;                                    // 1, or NaN
  }
  __syncthreads();
  if (sh.twice) {
    int lost = 0;
#pragma unroll
    for (int j = 0; j < SL; ++j) if (j * THREADS + tid < KCAP) sh.q[j * THREADS + tid] = mine.q[j];
    __syncthreads();
    bool follows[SL];
#pragma unroll
    for (int j = 0; j < SL; ++j) {
      const int s = j * THREADS + tid;
      follows[j] = false;
      if (mine.col[j] < 0) continue;
      double q = 0.0;
      for (int o = 0; o < a.k; ++o) {      // in slot order, whichever slot leads
        const double more = sh.q[o];
        const bool same = sh.col[o] == mine.col[j];
        if (same) q += more;
        follows[j] |= same && o < s;
      }
      mine.q[j] = q;
      if (follows[j]) ++lost;
    }
    lost = wave_sum_i(lost);
    if (lane == 0) sh.count[wave] = lost;
    __syncthreads();
    for (int i = 0; i < NW; ++i) u -= sh.count[i];
#pragma unroll
    for (int j = 0; j < SL; ++j) if (follows[j]) { sh.col[j * THREADS + tid] = -1; mine.col[j] = -1; mine.q[j] = 0.0; }
    __syncthreads();
    *near = near_of<T, THREADS, KCAP, RI>(sh, sp, sh.head[tid], &twice);
  }
  *unique = u;
  return sum;
}

// the chain's entries in the EPV columns from col0: fn(element, slot)
template <int EPV, int THREADS, int KCAP, typename F>
__device__ __forceinline__ void walk(const ListShared<THREADS, KCAP>& sh, uint16_t head, int col0, F fn) {
#pragma unroll 1
  for (uint32_t s = head; s != kEnd; s = sh.nxt[s]) {
    const int d = sh.col[s] - col0;
    if ((unsigned)d < (unsigned)EPV) fn(d, (int)s);
  }
}

// What the merged pairs and the list make of a row.
struct RowTerms {
  double x0, lse2;   // log2 p = (x - x0) c - lse2: the base-2 log-sum-exp of the whole row, of its
                     // differences to x0 where the maximum is a logit
  double q_r;        // probability of the bucket
  double total;      // sum of q and the bucket
};
__device__ __forceinline__ RowTerms row_terms(const ListArgs& a, const Pair64& all, double sum_q, int unique, int v) {
  RowTerms t;
  t.x0 = all.s < 0.0 ? (double)all.m : 0.0;
  t.lse2 = (all.s < 0.0 ? 0.0 : (double)all.m) + log2_64(all.sum());
  t.q_r = 0.0;
  if (a.tail == FM_TAIL_BUCKET && unique < v) {
    t.q_r = 1.0 - sum_q;
    if (t.q_r < 0.0) t.q_r = 0.0;          // (a NaN stays)
  }
  t.total = sum_q + t.q_r;
  return t;
}
// The listed columns' gradients into sh.g, as stored bits (a barrier ends it); returns the coefficient
// of an unlisted column, which its weight (sweep_of) is multiplied by.
template <typename T, int THREADS, int KCAP, int SL>
__device__ __forceinline__ float row_gradient(const ListArgs& a, ListShared<THREADS, KCAP>& sh, const Mine<SL>& mine,
                                              const Pair64& all, const Pair64& rest, const RowTerms& t, double scale) {
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    if (mine.col[j] < 0) continue;
    const int s = j * THREADS + (int)threadIdx.x;
    const double lp2 = ((double)sh.x[s] - t.x0) * (double)a.c - t.lse2;
    sh.g[s] = bits_of<T>((float)((exp2_64(lp2) * t.total - mine.q[j]) * scale));
  }
  __syncthreads();
  double coef = t.total * exp2_64(rest.top(a.c) - all.top(a.c)) / all.sum();
  if (!(t.q_r == 0.0)) coef -= t.q_r / rest.sum();
  // no unlisted column with any probability: their logits are -inf and their gradient 0 (a row of nothing
  // but -inf is no distribution: NaN, as its loss)
  if (rest.s == 0.0 && t.q_r == 0.0) coef = all.s == 0.0 ? __builtin_nan("") : 0.0;
  return (float)(coef * scale);
}
template <int THREADS, int KCAP, int SL>
__device__ __forceinline__ void row_loss_of(const ListArgs& a, ListShared<THREADS, KCAP>& sh, const Mine<SL>& mine,
                                            const Pair64& all, const Pair64& rest, const RowTerms& t, double sum_q,
                                            float* loss_at) {
  double term = 0.0;
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    if (mine.col[j] < 0 || mine.q[j] == 0.0) continue;
    const double lp2 = ((double)sh.x[j * THREADS + (int)threadIdx.x] - t.x0) * (double)a.c - t.lse2;
    term += mine.q[j] * (log2_64(mine.q[j]) - lp2);
  }
  term = block_reduce64<THREADS / 64, Sum64>(term, sh.red);
  if (threadIdx.x == 0) {
    if (!(t.q_r == 0.0))
      term += t.q_r * (log2_64(t.q_r) - ((rest.top(a.c) - all.top(a.c)) + (log2_64(rest.sum()) - log2_64(all.sum()))));
    *loss_at = (float)(sum_q != sum_q ? sum_q : term * kLn2d);
  }
}

// one vector into the running (maximum, sum); a NaN reaches both
template <typename T>
__device__ __forceinline__ void fold(MaxSum& run, const u32x4& r, float c) {
  constexpr int EPV = Elem<T>::kVec;
  float x[EPV];
  Elem<T>::unpack(r, x);
  float mx = x[0];
#pragma unroll
  for (int e = 1; e < EPV; ++e) mx = __builtin_elementwise_maximum(mx, x[e]);
  const float cm = __builtin_elementwise_maximum(run.m, mx * c);
  float acc = run.s * fast_exp2(run.m - cm);
#pragma unroll
  for (int e = 0; e < EPV; ++e) acc += fast_exp2(__builtin_fmaf(x[e], c, -cm));
  run.m = cm;
  run.s = acc;
}

template <typename T>
__device__ __forceinline__ void store_bits(T* p, uint32_t bits) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = bits;
  else *reinterpret_cast<uint16_t*>(p) = (uint16_t)bits;
}

// The two pairs of a row from its logits' differences to their maxima, in 64 bits: two more readings of the
// row, for rows whose pairs in fp32 are not sound -- x * c beyond fp32 or so large that the rounding of its
// maximum weighs more than the weights. NaN and +inf make the sum NaN. All threads of the workgroup call it.
template <typename T, int THREADS, int KCAP>
__device__ __forceinline__ void exact_pairs(const T* rp, const RowSplit& sp, int ne, float c, bool bucket, uint32_t mask,
                                            uint16_t head, ListShared<THREADS, KCAP>& sh, Pair64* rest, Pair64* all) {
  constexpr int EPV = Elem<T>::kVec;
  constexpr int NW = THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // fn(logit, whether it is one of the listed columns that count apart)
  auto own = [&](auto fn) {
#pragma unroll 1
    for (int i = tid; i < sp.nvec; i += THREADS) {
      uint32_t hit = 0u;
      const int col0 = sp.head + i * EPV;
      if (bucket && ((mask >> ((i / THREADS) % 31)) & 1u))
        walk<EPV, THREADS, KCAP>(sh, head, col0, [&](int d, int) { hit |= 1u << d; });
      float x[EPV];
      Elem<T>::unpack(load16(rp + col0), x);
#pragma unroll
      for (int e = 0; e < EPV; ++e) fn(x[e], (hit >> e) & 1u);
    }
#pragma unroll 1
    for (int e = tid; e < ne; e += THREADS) {
      uint32_t hit = 0u;
      const int col = edge_col(sp, e);
      if (bucket && (mask >> 31)) walk<1, THREADS, KCAP>(sh, head, col, [&](int, int) { hit = 1u; });
      fn(Elem<T>::load1(rp + col), hit);
    }
  };
  float top = -INFINITY, top_l = -INFINITY;
  own([&](float x, uint32_t hit) {
    const float y = x == x ? x : INFINITY;
    top = fmaxf(top, hit ? -INFINITY : y);
    top_l = fmaxf(top_l, hit ? y : -INFINITY);
  });
  top = wave_max(top);
  top_l = wave_max(top_l);
  __syncthreads();
  if (lane == 0) { sh.merge.m[0][wave] = top; sh.merge.m[1][wave] = top_l; }
  __syncthreads();
  top = group_reduce<NW, OpMax>(sh.merge.m[0][lane & (NW - 1)]);
  top_l = group_reduce<NW, OpMax>(sh.merge.m[1][lane & (NW - 1)]);
  double sum = 0.0, sum_l = 0.0;
  own([&](float x, uint32_t hit) {
    if (x == -INFINITY) return;            // (top may be -inf itself)
    const double w = exp2_64(((double)x - (double)(hit ? top_l : top)) * (double)c);
    sum += hit ? 0.0 : w;
    sum_l += hit ? w : 0.0;
  });
  sum = wave_sum64(sum);
  sum_l = wave_sum64(sum_l);
  if (lane == 0) { sh.merge.s[0][wave] = sum; sh.merge.s[1][wave] = sum_l; }
  __syncthreads();
  sum = group_reduce64<NW, Sum64>(sh.merge.s[0][lane & (NW - 1)]);
  sum_l = group_reduce64<NW, Sum64>(sh.merge.s[1][lane & (NW - 1)]);
  if (top == INFINITY) sum = __builtin_nan("");
  if (top_l == INFINITY) sum_l = __builtin_nan("");
  auto pair = [&](float m, double s) {
    if (s == 0.0) return Pair64{kNegBig, 0.0};
    const double t = (double)m * (double)c;
    if (!(__builtin_fabs(t) <= 2147483648.0) && s == s) return Pair64{m, -s};
    const float f = (float)t;
    return Pair64{f, s * exp2_64(t - (double)f)};
  };
  *rest = pair(top, sum);
  *all = *rest;
  if (sum_l != 0.0) {
    const float m = fmaxf(top, top_l);
    double s = sum_l * exp2_64(((double)top_l - (double)m) * (double)c);
    if (sum != 0.0) s += sum * exp2_64(((double)top - (double)m) * (double)c);
    *all = pair(m, s);
  }
}

// the gradient of vector c (its first column col0), packed
template <typename T, int THREADS, int KCAP>
__device__ __forceinline__ u32x4 grad_of(const u32x4& r, const Sweep& w, float coef,
                                         const ListShared<THREADS, KCAP>& sh, uint32_t mask, uint16_t head, int c,
                                         int col0) {
  constexpr int EPV = Elem<T>::kVec;
  float x[EPV];
  Elem<T>::unpack(r, x);
#pragma unroll
  for (int e = 0; e < EPV; ++e) x[e] = coef * fast_exp2(__builtin_fmaf(x[e], w.c, -w.m));
  u32x4 o = Elem<T>::pack(x);
  if ((mask >> ((c / THREADS) % 31)) & 1u)
    walk<EPV, THREADS, KCAP>(sh, head, col0, [&](int d, int s) { set_elem<T>(o, d, sh.g[s]); });
  return o;
}

// GRAD: loss and gradient, RI vectors a thread held in registers between the fold and the store,
// what a row has beyond them read twice. !GRAD: loss and stats from one streaming read (RI vectors
// a thread in flight). VEC: the buffers are 16-byte aligned and every row holds a whole vector, so the
// row's loads stand behind no branch -- behind one, the first wait of the list's loads would be a wait
// for all of them ([4096,128256] bf16, loss and gradient, one workgroup a row and compute unit: 552 us
// behind one, 479 without). !VEC: one element at a time.
template <typename T, int THREADS, int KCAP, int RI, bool GRAD, bool VEC>
__global__ __launch_bounds__(THREADS) void kl_topk_kernel(const T* student, ListArgs a, float* __restrict__ row_loss,
                                                          float* __restrict__ stats, const float* __restrict__ n_valid,
                                                          int count_n, T* dstudent, int v) {
  constexpr int EPV = Elem<T>::kVec;
  constexpr int NW = THREADS / 64;
  constexpr int SL = (KCAP + THREADS - 1) / THREADS;
  __shared__ ListShared<THREADS, KCAP> sh;
  const int64_t row = blockIdx.x;
  const T* rp = student + row * (int64_t)v;
  T* gp = GRAD ? dstudent + row * (int64_t)v : nullptr;
  const RowSplit sp = split_row<EPV>(row, v, VEC);
  const int tid = threadIdx.x;
  const int ne = edge_count(sp, v);
  const bool bucket = a.tail == FM_TAIL_BUCKET;

  if (list_idx(a, row * a.k) < 0) {     // no list: nothing is read, the gradient is zero
    if (GRAD) {
      const u32x4 zero = {0u, 0u, 0u, 0u};
      for (int c = tid; c < sp.nvec; c += THREADS) store16_stream(gp + sp.head + (int64_t)c * EPV, zero);
      for (int e = tid; e < ne; e += THREADS) Elem<T>::store1(gp + edge_col(sp, e), 0.f);
    }
    if (tid == 0) row_loss[row] = 0.f;
    if (tid < 4 && stats != nullptr) stats[row * 4 + tid] = 0.f;
    return;
  }
  // the list's loads go first: waiting for them then waits for nothing of the row
  SlotBits bits[SL];
  list_load<THREADS, SL>(a, row, bits);
  // where the rows are few (count_n <= kCountInKernel), every workgroup counts those with a list itself,
  // kCount of them a thread
  constexpr int kCount = GRAD ? (kCountInKernel + THREADS - 1) / THREADS : 1;
  int first[kCount];
#pragma unroll
  for (int j = 0; j < kCount; ++j) {
    const int r = j * THREADS + tid;
    first[j] = GRAD ? slot_sign(a, (int64_t)(r < count_n ? r : 0) * a.k) : 0;
  }
  const float nv = *(GRAD && n_valid != nullptr ? n_valid : static_cast<const float*>(a.idx));
  const float lse_t = *(a.teacher_lse != nullptr ? a.teacher_lse + row : static_cast<const float*>(a.idx));
  const T* vp = rp + sp.head;              // 16-byte aligned where there are vectors
  auto at = [&](int c) { return reinterpret_cast<const T*>(reinterpret_cast<const char*>(vp) + (uint32_t)c * 16u); };
  u32x4 raw[RI];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < RI; ++i) raw[i] = load16_stream(at(clamp_col(i * THREADS + tid, sp.nvec)));
  }
  Mine<SL> mine;
  int unique;
  Near near;
  const double sum_q = list_build<T, THREADS, KCAP, SL, VEC ? RI : 0>(a, sp, v, bits, lse_t, 0, sp.nvec, true, sh, mine,
                                                                      &near, &unique);
  uint32_t mask = sh.mask[tid];
  const uint16_t head = sh.head[tid];

  if (GRAD && count_n > 0) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < kCount; ++j) c += __builtin_popcountll(__ballot(j * THREADS + tid < count_n && first[j] >= 0));
    if ((tid & 63) == 0) sh.count[tid >> 6] = c;
  }

  // The sweep leaves the listed logits in sh.x and, for the bucket, folds the others only. (The listed ones are
  // added from there, by slot: a chain's order is that in which the waves got to its head.)
  MaxSum run{kNegBig, 0.f};
  auto meet = [&](u32x4& r, int d, int s) {
    const float x = get_elem<T>(r, d);
    sh.x[s] = x;
    if (bucket) set_elem<T>(r, d, bits_of<T>(-INFINITY));
  };
  auto take = [&](u32x4 r, int c) {       // what the registers of near_of do not cover
    if (c >= sp.nvec) return;
    if ((near.more >> ((c / THREADS) % 31)) & 1u) {
      walk<EPV, THREADS, KCAP>(sh, head, sp.head + c * EPV, [&](int d, int s) {
        if (s != (int)(near.e0 >> 16) && s != (int)(near.e1 >> 16)) meet(r, d, s);
      });
    }
    fold<T>(run, r, a.c);
  };
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      u32x4 r = raw[i];
      if ((mask >> (i % 31)) & 1u) {
        if ((near.e0 & 255u) == (uint32_t)i) meet(r, (near.e0 >> 8) & 15u, (int)(near.e0 >> 16));
        if ((near.e1 & 255u) == (uint32_t)i) meet(r, (near.e1 >> 8) & 15u, (int)(near.e1 >> 16));
      }
      take(r, i * THREADS + tid);
    }
    constexpr int UN = GRAD ? 2 : RI;
    for (int c0 = RI * THREADS; c0 < sp.nvec; c0 += UN * THREADS) {
      u32x4 more[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const T* from = at(clamp_col(c0 + u * THREADS + tid, sp.nvec));
        more[u] = GRAD ? load16(from) : load16_stream(from);
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        touch_whole(more[u]);
        take(more[u], c0 + u * THREADS + tid);
      }
    }
  }
  for (int e = tid; e < ne; e += THREADS) {
    const int col = edge_col(sp, e);
    float x = Elem<T>::load1(rp + col);
    if (mask >> 31) {
      walk<1, THREADS, KCAP>(sh, head, col, [&](int, int s) {
        sh.x[s] = x;
        if (bucket) x = -INFINITY;
      });
    }
    fold1(run, x, a.c);
  }
  Pair64 rest = merge_pairs<NW>(run, sh.merge);      // its barrier also publishes sh.x
  Pair64 all = rest;
  if (bucket) {
    double more = 0.0;
#pragma unroll
    for (int j = 0; j < SL; ++j)
      if (mine.col[j] >= 0) more += exp2_64((double)sh.x[j * THREADS + tid] * (double)a.c - (double)rest.m);
    all = with_listed<NW>(rest, more, sh.merge);
  }
  // (alike in all lanes, and the compiler has to know: behind a lane's branch the row's registers stay taken)
  if (__builtin_expect(__builtin_amdgcn_readfirstlane(rest.sound() && all.sound()) == 0, 0)) {
    exact_pairs<T, THREADS, KCAP>(rp, sp, ne, a.c, bucket, mask, head, sh, &rest, &all);
    if constexpr (GRAD && VEC) {       // the row's registers were free meanwhile, and so were its addresses'
      int me = tid;
      asm volatile("" : "+v"(me));
#pragma unroll
      for (int i = 0; i < RI; ++i) raw[i] = load16(at(clamp_col(i * THREADS + me, sp.nvec)));
    }
  }
  const RowTerms terms = row_terms(a, all, sum_q, unique, v);
  if (tid == 0 && stats != nullptr) {
    stats[row * 4] = all.m;
    stats[row * 4 + 1] = (float)all.s;
    stats[row * 4 + 2] = rest.m;
    stats[row * 4 + 3] = (float)rest.s;
  }
  if constexpr (GRAD) {
    double scale = a.inv_t;
    if (count_n > 0) {
      int rows = 0;
      for (int i = 0; i < NW; ++i) rows += sh.count[i];
      scale /= (double)(rows > 0 ? rows : 1);
    } else if (n_valid != nullptr) {
      scale /= (double)nv;
    }
    const float coef = row_gradient<T, THREADS, KCAP, SL>(a, sh, mine, all, rest, terms, scale);
    const uint32_t g0 = near.e0 != kNone ? sh.g[near.e0 >> 16] : 0u, g1 = near.e1 != kNone ? sh.g[near.e1 >> 16] : 0u;
    // taken afresh: the comparisons of the sweep are not worth keeping in scalar registers until here
    int me = tid;
    asm volatile("" : "+v"(near.e0), "+v"(near.e1), "+v"(near.more), "+v"(mask), "+v"(me));
    T* vg = gp + sp.head;
    const Sweep w = sweep_of(rest, a.c);
    auto put = [&](const u32x4& r, int c) {
      if (c >= sp.nvec) return;
      store16_stream(reinterpret_cast<T*>(reinterpret_cast<char*>(vg) + (uint32_t)c * 16u),
                     grad_of<T, THREADS, KCAP>(r, w, coef, sh, mask, head, c, sp.head + c * EPV));
    };
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        touch_whole(raw[i]);
        const int c = i * THREADS + me;
        if (c >= sp.nvec) continue;
        u32x4 o = grad_of<T, THREADS, KCAP>(raw[i], w, coef, sh, near.more, head, c, sp.head + c * EPV);
        if ((mask >> (i % 31)) & 1u) {
          if ((near.e0 & 255u) == (uint32_t)i) set_elem<T>(o, (near.e0 >> 8) & 15u, g0);
          if ((near.e1 & 255u) == (uint32_t)i) set_elem<T>(o, (near.e1 >> 8) & 15u, g1);
        }
        store16_stream(reinterpret_cast<T*>(reinterpret_cast<char*>(vg) + (uint32_t)c * 16u), o);
      }
      for (int c0 = RI * THREADS; c0 < sp.nvec; c0 += 2 * THREADS) {
        u32x4 more[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) more[u] = load16_stream(at(clamp_col(c0 + u * THREADS + tid, sp.nvec)));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          touch_whole(more[u]);
          put(more[u], c0 + u * THREADS + tid);
        }
      }
    }
    for (int e = tid; e < ne; e += THREADS) {
      const int col = edge_col(sp, e);
      float o = coef * fast_exp2(__builtin_fmaf(Elem<T>::load1(rp + col), w.c, -w.m));
      uint32_t one = bits_of<T>(o);
      if (mask >> 31) walk<1, THREADS, KCAP>(sh, head, col, [&](int, int s) { one = sh.g[s]; });
      store_bits(gp + col, one);
    }
  }
  // last: the reduction runs while the stores drain
  row_loss_of<THREADS, KCAP, SL>(a, sh, mine, all, rest, terms, sum_q, row_loss + row);
}

// The gradient from saved stats. chunks > 1: a workgroup takes one tile of THREADS * UN vectors of a
// row (the row's unaligned ends go with its first tile); each tile builds the row's list again.
template <typename T, int THREADS, int KCAP, int UN>
__global__ __launch_bounds__(THREADS) void kl_topk_bwd_kernel(const T* student, ListArgs a,
                                                              const float* __restrict__ stats,
                                                              const float* __restrict__ n_valid,
                                                              const float* __restrict__ grad_out, int grad_per_row,
                                                              T* dstudent, int v, bool vec_ok, int chunks) {
  constexpr int EPV = Elem<T>::kVec;
  constexpr int SL = (KCAP + THREADS - 1) / THREADS;
  __shared__ ListShared<THREADS, KCAP> sh;
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)chunks);
  const T* rp = student + row * (int64_t)v;
  T* gp = dstudent + row * (int64_t)v;
  const RowSplit sp = split_row<EPV>(row, v, vec_ok);
  const int tid = threadIdx.x;
  const int ne = chunk == 0 ? edge_count(sp, v) : 0;
  const int c_begin = chunk * THREADS * UN;
  int c_end = chunks > 1 ? c_begin + THREADS * UN : sp.nvec;
  if (c_end > sp.nvec) c_end = sp.nvec;

  if (list_idx(a, row * a.k) < 0) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int c = c_begin + tid; c < c_end; c += THREADS) store16_stream(gp + sp.head + (int64_t)c * EPV, zero);
    for (int e = tid; e < ne; e += THREADS) Elem<T>::store1(gp + edge_col(sp, e), 0.f);
    return;
  }
  SlotBits bits[SL];
  list_load<THREADS, SL>(a, row, bits);
  const float lse_t = *(a.teacher_lse != nullptr ? a.teacher_lse + row : static_cast<const float*>(a.idx));
  const Pair64 all{stats[row * 4], (double)stats[row * 4 + 1]}, rest{stats[row * 4 + 2], (double)stats[row * 4 + 3]};
  double scale = a.inv_t;
  if (grad_out != nullptr) scale *= (double)grad_out[grad_per_row ? row : 0];
  if (n_valid != nullptr) scale /= (double)*n_valid;
  Mine<SL> mine;
  int unique;
  Near near;
  const double sum_q = list_build<T, THREADS, KCAP, SL, 0>(a, sp, v, bits, lse_t, c_begin, c_end, chunk == 0, sh, mine,
                                                           &near, &unique);
#pragma unroll
  for (int j = 0; j < SL; ++j)
    if (mine.col[j] >= 0) sh.x[j * THREADS + tid] = Elem<T>::load1(rp + mine.col[j]);
  const uint32_t mask = sh.mask[tid];
  const uint16_t head = sh.head[tid];
  const float coef = row_gradient<T, THREADS, KCAP, SL>(a, sh, mine, all, rest, row_terms(a, all, sum_q, unique, v), scale);
  const Sweep w = sweep_of(rest, a.c);
  for (int c0 = c_begin; c0 < c_end; c0 += THREADS * UN) {
    u32x4 raw[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      raw[u] = load16_stream(rp + sp.head + (int64_t)clamp_col(c0 + u * THREADS + tid, sp.nvec) * EPV);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int c = c0 + u * THREADS + tid;
      touch_whole(raw[u]);
      if (c < c_end)
        store16_stream(gp + sp.head + (int64_t)c * EPV,
                       grad_of<T, THREADS, KCAP>(raw[u], w, coef, sh, mask, head, c, sp.head + c * EPV));
    }
  }
  for (int e = tid; e < ne; e += THREADS) {
    const int col = edge_col(sp, e);
    float o = coef * fast_exp2(__builtin_fmaf(Elem<T>::load1(rp + col), w.c, -w.m));
    uint32_t one = bits_of<T>(o);
    if (mask >> 31) walk<1, THREADS, KCAP>(sh, head, col, [&](int, int s) { one = sh.g[s]; });
    store_bits(gp + col, one);
  }
}

// *n_valid = rows with a list (COUNT); *loss = sum of row_loss [/ n_valid] (LOSS). One workgroup, eight
// rows' loads of a thread in flight, 64-bit sum in a fixed order.
template <bool COUNT, bool LOSS>
__global__ __launch_bounds__(1024) void kl_topk_reduce_kernel(const float* __restrict__ row_loss, ListArgs a, int64_t n,
                                                              int mean, float* __restrict__ loss,
                                                              float* __restrict__ n_valid) {
  __shared__ double sd[16];
  __shared__ int si[16];
  double s = 0.0;
  int cnt = 0;
  for (int64_t i = threadIdx.x; i < n; i += 8 * 1024) {
    float r[8];
    int used[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t at = i + u * 1024 < n ? i + u * 1024 : i;
      if (LOSS) r[u] = row_loss[at];
      // the sign of slot 0
      if (COUNT) used[u] = slot_sign(a, at * a.k);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (i + u * 1024 < n) {
        if (LOSS) s += (double)r[u];
        if (COUNT) cnt += used[u] >= 0 ? 1 : 0;
      }
    }
  }
  if (LOSS) s = block_reduce64<16, Sum64>(s, sd);
  if (COUNT) {
    cnt = wave_sum_i(cnt);
    if ((threadIdx.x & 63) == 0) si[threadIdx.x >> 6] = cnt;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    float nv = 1.f;
    if (COUNT) {
      int c = 0;
      for (int i = 0; i < 16; ++i) c += si[i];
      nv = c > 0 ? (float)c : 1.f;
      *n_valid = nv;
    } else if (mean) {
      nv = *n_valid;
    }
    if (LOSS) *loss = (float)(mean ? s / (double)nv : s);
  }
}

int check(const char* what, int64_t n, int64_t v, int k, int dtype, int index_bits, int teacher_dtype, int kind,
          int tail, double temperature) {
  FM_CHECK_ARG(n >= 0 && v > 0, "%s: bad shape n=%lld v=%lld", what, (long long)n, (long long)v);
  FM_CHECK_ARG(k >= 1, "%s: k must be positive (got %d)", what, k);
  FM_CHECK_ARG(dtype == FM_F32 || dtype == FM_F16 || dtype == FM_BF16, "%s: bad dtype %d", what, dtype);
  FM_CHECK_ARG(teacher_dtype == FM_F32 || teacher_dtype == FM_F16 || teacher_dtype == FM_BF16,
               "%s: bad teacher_dtype %d", what, teacher_dtype);
  FM_CHECK_ARG(index_bits == 32 || index_bits == 64, "%s: index_bits must be 32 or 64 (got %d)", what, index_bits);
  FM_CHECK_ARG(kind == FM_TEACHER_LOGITS || kind == FM_TEACHER_PROBS, "%s: bad teacher_kind %d", what, kind);
  FM_CHECK_ARG(tail == FM_TAIL_RENORM || tail == FM_TAIL_DROP || tail == FM_TAIL_BUCKET, "%s: bad tail %d", what, tail);
  FM_CHECK_ARG(temperature > 0.0 && temperature < (double)INFINITY, "%s: temperature must be positive and finite", what);
  // (a launch has less than 2^32 threads, and a row up to 1024; offsets inside a row are 32 bits of bytes)
  if (n >= (1LL << 22) || v >= (1LL << 30) || k > kMaxList) {
    fm_host::set_error("%s: n must be below 2^22, v below 2^30 and k at most %d", what, kMaxList);
    return FM_ERR_UNSUPPORTED;
  }
  return FM_OK;
}

ListArgs list_args(const void* idx, const void* teacher, const float* lse, int k, int index_bits, int teacher_dtype,
                   int kind, int tail, double temperature) {
  ListArgs a;
  a.idx = idx; a.teacher = teacher; a.teacher_lse = lse; a.k = k; a.idx64 = index_bits == 64;
  a.teacher_dtype = teacher_dtype; a.probs = kind; a.tail = tail; a.inv_t = 1.0 / temperature;
  a.c = (float)(1.4426950408889634074 / temperature);
  if (a.c == 0.f) a.c = 1.40129846e-45f;       // past 1e45: every finite logit counts the same, and -inf * c is -inf
  return a;
}

template <typename T, int KCAP>
void launch_loss_grad(const void* student, const ListArgs& a, float* row_loss, float* stats, const float* n_valid,
                      int count_n, void* dstudent, int64_t n, int v, bool vec_ok, hipStream_t st) {
  const int64_t nvec = v / Elem<T>::kVec;
#define GO(TH, RI, VEC)                                                                                      \
  FM_LAUNCH((kl_topk_kernel<T, TH, KCAP, RI, true, VEC>), dim3((unsigned)n), dim3(TH), 0, st,                \
            static_cast<const T*>(student), a, row_loss, stats, n_valid, count_n, static_cast<T*>(dstudent), v)
  // Smallest workgroups that hold a row in 16 vectors a thread: several rows a compute unit, in different
  // phases. Wide rows do better with half of the row held by each of two workgroups a unit and the rest
  // read again from the caches than with one workgroup that holds all of it ([4185,128256] bf16: 433
  // against 520 us; [2684,200000]: 455 against 458; fp32 [2092,128256]: 508 against 430, so not beyond
  // 20480 vectors), unless there is no second row for the unit ([16,128256]: 27 us against 29).
  // A long list (KCAP 1024) wants more threads than a short row does.
  const bool few = n <= fm_host::num_cus();
  if (!vec_ok || v < 2 * Elem<T>::kVec) GO(256, 2, false);
  else if (nvec > (few ? 8192 : 20480)) GO(1024, 16, true);
  else if (nvec > 4096 || (few && nvec > 2048)) GO(512, 16, true);
  else if (nvec > 2048) GO(256, 16, true);
  else if constexpr (KCAP > kSmallList) GO(256, 8, true);
  else if (nvec > 1024) GO(128, 16, true);
  else if (nvec > 512) GO(128, 8, true);
  else GO(64, 8, true);
#undef GO
}

template <typename T, int KCAP>
void launch_fwd(const void* student, const ListArgs& a, float* row_loss, float* stats, int64_t n, int v, bool vec_ok,
                hipStream_t st) {
  const int64_t nvec = v / Elem<T>::kVec;
#define GO(TH, RI, VEC)                                                                                      \
  FM_LAUNCH((kl_topk_kernel<T, TH, KCAP, RI, false, VEC>), dim3((unsigned)n), dim3(TH), 0, st,               \
            static_cast<const T*>(student), a, row_loss, stats, nullptr, 0, static_cast<T*>(nullptr), v)
  // one streaming read: rows in small workgroups, more threads where few rows have to fill the device
  const bool few = n <= fm_host::num_cus();
  if (!vec_ok || v < 2 * Elem<T>::kVec) GO(256, 4, false);
  else if (few && nvec > 8192) GO(1024, 4, true);
  else if (nvec > 8192) GO(512, 4, true);
  else if (few && nvec > 2048) GO(512, 8, true);
  else if (nvec > 2048) GO(256, 8, true);
  else if constexpr (KCAP > kSmallList) GO(256, 4, true);
  else if (nvec > 256) GO(128, 8, true);
  else GO(64, 4, true);
#undef GO
}

template <typename T, int KCAP>
void launch_bwd(const void* student, const ListArgs& a, const float* stats, const float* n_valid, const float* grad_out,
                int per_row, void* dstudent, int64_t n, int v, bool vec_ok, hipStream_t st) {
  const int64_t nvec = v / Elem<T>::kVec;
#define GO(TH, UN)                                                                                            \
  do {                                                                                                        \
    int64_t chunks = (nvec + TH * UN - 1) / (TH * UN);                                                        \
    if (chunks < 1 || n * chunks >= (1LL << 32) / TH) chunks = 1;                                                \
    FM_LAUNCH((kl_topk_bwd_kernel<T, TH, KCAP, UN>), dim3((unsigned)(n * chunks)), dim3(TH), 0, st,           \
              static_cast<const T*>(student), a, stats, n_valid, grad_out, per_row, static_cast<T*>(dstudent), \
              v, vec_ok, (int)chunks);                                                                        \
  } while (0)
  if (nvec > 2048 && KCAP > kSmallList) GO(512, 8);
  else if (nvec > 1024) GO(256, 8);
  else if constexpr (KCAP > kSmallList) GO(256, 4);
  else if (nvec > 256) GO(128, 4);
  else GO(64, 4);
#undef GO
}

#define FM_KLT_DISPATCH(dtype, k, FN, ...)                                          \
  do {                                                                              \
    const bool small__ = (k) <= kSmallList;                                         \
    if ((dtype) == FM_F32) { if (small__) FN<float, kSmallList>(__VA_ARGS__); else FN<float, kMaxList>(__VA_ARGS__); }        \
    else if ((dtype) == FM_BF16) { if (small__) FN<bf16_t, kSmallList>(__VA_ARGS__); else FN<bf16_t, kMaxList>(__VA_ARGS__); } \
    else { if (small__) FN<f16_t, kSmallList>(__VA_ARGS__); else FN<f16_t, kMaxList>(__VA_ARGS__); }                          \
  } while (0)

}  // namespace

extern "C" {

int fm_kl_topk_fwd(const void* student, const void* idx, const void* teacher, const float* teacher_lse,
                   float* row_loss, float* stats, float* loss, float* n_valid, int64_t n, int64_t v, int k, int dtype,
                   int index_bits, int teacher_dtype, int teacher_kind, int tail, double temperature, int reduction,
                   fm_stream_t stream) {
  const int rc = check("fm_kl_topk_fwd", n, v, k, dtype, index_bits, teacher_dtype, teacher_kind, tail, temperature);
  if (rc != FM_OK) return rc;
  FM_CHECK_ARG(reduction == FM_REDUCE_NONE || reduction == FM_REDUCE_SUM || reduction == FM_REDUCE_MEAN,
               "fm_kl_topk_fwd: bad reduction %d", reduction);
  FM_CHECK_ARG(reduction == FM_REDUCE_NONE || (loss && n_valid), "fm_kl_topk_fwd: NULL scalar output");
  FM_CHECK_ARG(n == 0 || (student && idx && teacher && row_loss), "fm_kl_topk_fwd: NULL pointer");
  FM_CHECK_ARG(n == 0 || teacher_lse || teacher_kind == FM_TEACHER_PROBS || tail == FM_TAIL_RENORM,
               "fm_kl_topk_fwd: teacher logits need teacher_lse unless the list is renormalised");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const ListArgs a = list_args(idx, teacher, teacher_lse, k, index_bits, teacher_dtype, teacher_kind, tail, temperature);
  if (n > 0) {
    const bool vec_ok = fm_host::aligned16(student);
    FM_KLT_DISPATCH(dtype, k, launch_fwd, student, a, row_loss, stats, n, (int)v, vec_ok, st);
    FM_CHECK_LAUNCH("fm_kl_topk_fwd");
  }
  if (reduction != FM_REDUCE_NONE) {
    hipLaunchKernelGGL((kl_topk_reduce_kernel<true, true>), dim3(1), dim3(1024), 0, st, row_loss, a, n,
                       reduction == FM_REDUCE_MEAN ? 1 : 0, loss, n_valid);
    FM_CHECK_LAUNCH("fm_kl_topk_fwd(finalize)");
  }
  return FM_OK;
}

int fm_kl_topk_loss_grad(const void* student, const void* idx, const void* teacher, const float* teacher_lse,
                         float* row_loss, float* stats, float* loss, float* n_valid, void* dstudent, int64_t n,
                         int64_t v, int k, int dtype, int index_bits, int teacher_dtype, int teacher_kind, int tail,
                         double temperature, int reduction, fm_stream_t stream) {
  const int rc = check("fm_kl_topk_loss_grad", n, v, k, dtype, index_bits, teacher_dtype, teacher_kind, tail, temperature);
  if (rc != FM_OK) return rc;
  FM_CHECK_ARG(reduction == FM_REDUCE_SUM || reduction == FM_REDUCE_MEAN,
               "fm_kl_topk_loss_grad: reduction must be sum or mean (got %d)", reduction);
  FM_CHECK_ARG(loss && n_valid, "fm_kl_topk_loss_grad: NULL scalar output");
  FM_CHECK_ARG(n == 0 || (student && idx && teacher && row_loss && dstudent), "fm_kl_topk_loss_grad: NULL pointer");
  FM_CHECK_ARG(n == 0 || teacher_lse || teacher_kind == FM_TEACHER_PROBS || tail == FM_TAIL_RENORM,
               "fm_kl_topk_loss_grad: teacher logits need teacher_lse unless the list is renormalised");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const ListArgs a = list_args(idx, teacher, teacher_lse, k, index_bits, teacher_dtype, teacher_kind, tail, temperature);
  const bool mean = reduction == FM_REDUCE_MEAN;
  if (n > 0) {
    const bool count_here = mean && n <= kCountInKernel;
    if (mean && !count_here) {
      hipLaunchKernelGGL((kl_topk_reduce_kernel<true, false>), dim3(1), dim3(1024), 0, st, nullptr, a, n, 0, loss,
                         n_valid);
      FM_CHECK_LAUNCH("fm_kl_topk_loss_grad(count)");
    }
    const bool vec_ok = fm_host::aligned16(student) && fm_host::aligned16(dstudent);
    FM_KLT_DISPATCH(dtype, k, launch_loss_grad, student, a, row_loss, stats, mean ? n_valid : nullptr,
                    count_here ? (int)n : 0, dstudent, n, (int)v, vec_ok, st);
    FM_CHECK_LAUNCH("fm_kl_topk_loss_grad");
  }
  if (mean && n > kCountInKernel)      // n_valid is there
    hipLaunchKernelGGL((kl_topk_reduce_kernel<false, true>), dim3(1), dim3(1024), 0, st, row_loss, a, n, 1, loss, n_valid);
  else
    hipLaunchKernelGGL((kl_topk_reduce_kernel<true, true>), dim3(1), dim3(1024), 0, st, row_loss, a, n, mean ? 1 : 0, loss,
                       n_valid);
  FM_CHECK_LAUNCH("fm_kl_topk_loss_grad(finalize)");
  return FM_OK;
}

int fm_kl_topk_bwd(const void* student, const void* idx, const void* teacher, const float* teacher_lse,
                   const float* stats, const float* n_valid, const float* grad_out, int grad_per_row, void* dstudent,
                   int64_t n, int64_t v, int k, int dtype, int index_bits, int teacher_dtype, int teacher_kind,
                   int tail, double temperature, fm_stream_t stream) {
  const int rc = check("fm_kl_topk_bwd", n, v, k, dtype, index_bits, teacher_dtype, teacher_kind, tail, temperature);
  if (rc != FM_OK) return rc;
  if (n == 0) return FM_OK;
  FM_CHECK_ARG(student && idx && teacher && stats && dstudent, "fm_kl_topk_bwd: NULL pointer");
  FM_CHECK_ARG(student != dstudent, "fm_kl_topk_bwd: dstudent must not be the student buffer");
  FM_CHECK_ARG(!grad_per_row || grad_out, "fm_kl_topk_bwd: a gradient per row needs grad_out");
  FM_CHECK_ARG(teacher_lse || teacher_kind == FM_TEACHER_PROBS || tail == FM_TAIL_RENORM,
               "fm_kl_topk_bwd: teacher logits need teacher_lse unless the list is renormalised");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const ListArgs a = list_args(idx, teacher, teacher_lse, k, index_bits, teacher_dtype, teacher_kind, tail, temperature);
  const bool vec_ok = fm_host::aligned16(student) && fm_host::aligned16(dstudent);
  FM_KLT_DISPATCH(dtype, k, launch_bwd, student, a, stats, n_valid, grad_out, grad_per_row, dstudent, n, (int)v, vec_ok, st);
  FM_CHECK_LAUNCH("fm_kl_topk_bwd");
  return FM_OK;
}

}  // extern "C"
