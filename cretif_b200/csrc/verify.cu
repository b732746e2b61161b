// Verification of drafted tokens against the model's probabilities, from given uniform numbers.
//
// Sequence b brings n drafts x_0 .. x_{n-1} and n + 1 rows of logits (row j: what follows the tokens
// before x_j).  p_j = softmax(logits / T) over the kept ids of row j (all, or the top_k largest, of
// equals the lowest ids), q_j the same of the logits that x_j was drawn from, or 1 at x_j where there
// are none.  Draft j stands while u_j q_j(x_j) < p_j(x_j); behind the first that does not, the token
// is drawn from max(p_j - q_j, 0), behind a sequence whose drafts all stand from p_n: the first id
// whose cumulative sum, in id order, exceeds u' times the total.  So the tokens are distributed as if
// each had been drawn from its p.  T <= 0: a draft stands where it is the arg max.
//
// A row's terms are 2^((x - max) log2 e / T); an entry equal to the row's maximum counts 1 whatever
// it is, so that a row of equal infinities is uniform; NaN counts as -infinity.
//
// Two launches.  The first looks at all rows: what decides whether a draft stands are its row's
// maximum and sum (32-bit terms, off by about 1e-7 of the sum), with top_k the kept entries
// themselves (in 64 bits).  The second decides and draws.  Where u q and p lie so close that the 32-bit
// sums cannot tell which is larger, the draft's rows are summed in 64 bits first.  An id is drawn at one
// of V borders, so sums that are off by 1e-7 would draw another id once in V 1e-7 draws (1 in 200
// at 49,152 ids): the one or two rows that a sequence draws from are summed again in 64 bits.
//
// The reference has no counterpart (its sampling: src/embedding.cu:343-406).
#include <cooperative_groups.h>

#include <type_traits>

#include "api.h"
#include "common.cuh"

namespace cretif {

namespace cg = cooperative_groups;

constexpr int kVfMaxTopK = 1024;

struct VfArgs {
  const float* logits;
  long long ld;                 // (rows may lie more than 2^31 numbers apart)
  int n_rows;
  const int* cu;
  const int* drafts;
  long long ld_drafts;
  int K, B, V;
  const float* draft_logits;
  long long ld_seq, ld_place;
  const float* accept_u;
  long long ld_u;
  const float* next_u;
  double log2_t;                // log2 e / T, within what float32 holds
  float reach;                  // how far below the largest entry an entry counts: 1000 / log2_t
  int top_k;
  int* accepted;
  int* tokens;
  long long ld_tokens;
  unsigned int* fault;
  // what the first launch leaves: rows 0 .. n_rows - 1 are the logits', n_rows + b K + j draft j's
  void* stats;                  // [rows][slices] VfPart, with top_k [rows] VfKept, greedy [rows][slices] u64
  int slices, slice_vectors;    // vectors of four a slice
  float* list_v;                // top_k: [rows][top_k] kept values and ids
  int* list_i;
};
struct VfPart {                 // of a slice of a row
  float m, z;
};
struct VfKept {
  double z;
  unsigned long long thr;       // (key, ~id) of the last entry kept
  float top;
  int pad;
};

__device__ __forceinline__ unsigned int vf_key(float v) {
  if (v == 0.f) v = 0.f;                                   // the two zeros are equal
  if (v != v) v = -INFINITY;
  const unsigned int b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);       // larger float -> larger key
}
__device__ __forceinline__ float vf_value(unsigned int key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// Larger value first, of equals the lower id.
__device__ __forceinline__ unsigned long long vf_rank(float v, int id) {
  return ((unsigned long long)vf_key(v) << 32) | (0xffffffffu - (unsigned)id);
}
__device__ __forceinline__ float vf_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float vf_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ VfPart vf_merge(VfPart a, VfPart b, float c) {
  VfPart r;
  r.m = fmaxf(a.m, b.m);
  r.z = (a.m == r.m ? a.z : a.z * vf_ex2((a.m - r.m) * c)) + (b.m == r.m ? b.z : b.z * vf_ex2((b.m - r.m) * c));
  return r;
}

// The drafts of sequence b and its first row; false where it has no such rows.
__device__ __forceinline__ bool vf_sequence(const VfArgs& a, int b, int& row0, int& n) {
  row0 = a.cu[b];
  n = a.cu[b + 1] - row0 - 1;
  return n >= 0 && n <= a.K && row0 >= 0 && row0 <= a.n_rows - 1 - n;
}
// Row i of the first launch, null where there is none to look at.
__device__ __forceinline__ const float* vf_row(const VfArgs& a, int i) {
  if (i < a.n_rows) return a.logits + (size_t)i * a.ld;
  const int at = i - a.n_rows, b = at / a.K, j = at - b * a.K;
  int row0, n;
  if (!vf_sequence(a, b, row0, n) || j >= n) return nullptr;
  return a.draft_logits + b * a.ld_seq + j * a.ld_place;
}

// ---- first launch: maximum and sum, or arg max, of a slice of a row.  A thread asks for all of its
// NV vectors at once.  Rows may begin anywhere: the vectors begin at the first 16-byte boundary, the
// up to three entries before it and behind the last vector are the first slice's.
constexpr int kVsThreads = 256, kVsWarps = kVsThreads / 32;

// A thread's entries of a slice, -infinity behind its end.
template <int NV>
struct VsSlice {
  float v[4 * NV];
  float extra;                  // an entry before or behind the vectors
  int at, end, head, extra_id;  // the first vector, the slice's end, entries before the row's first vector

  __device__ __forceinline__ void load(const VfArgs& a, const float* x, int slice) {
    const int tid = threadIdx.x;
    const float none = -INFINITY;
    head = min(a.V, (int)((0u - (unsigned)((uintptr_t)x >> 2)) & 3u));
    const int n4 = (a.V - head) >> 2;
    const float4* x4 = reinterpret_cast<const float4*>(x + head);
    at = slice * a.slice_vectors + tid;
    end = min(n4, (slice + 1) * a.slice_vectors);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float4 f = make_float4(none, none, none, none);
      if (at + i * kVsThreads < end) f = __ldcs(x4 + at + i * kVsThreads);
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
    extra_id = -1;
    if (slice == 0 && tid < a.V - 4 * n4) {
      extra_id = tid < head ? tid : 4 * n4 + tid;
      extra = __ldg(x + extra_id);
    }
  }
  __device__ __forceinline__ bool there(int i) const { return at + (i >> 2) * kVsThreads < end; }
  __device__ __forceinline__ float largest() const {
    float m[2] = {-INFINITY, -INFINITY};                  // (NaN is passed over)
#pragma unroll
    for (int i = 0; i < 4 * NV; i += 2) m[(i >> 1) & 1] = vf_max3(m[(i >> 1) & 1], v[i], v[i + 1]);
    return fmaxf(m[0], m[1]);
  }
  __device__ __forceinline__ unsigned long long best() const {
    const float m = largest();
    int first = -1;
#pragma unroll
    for (int i = 4 * NV - 1; i >= 0; --i)
      if (v[i] == m) first = i;
    if (m == -INFINITY) {                                 // (all are, or are not there, or NaN)
      first = -1;
#pragma unroll
      for (int i = 4 * NV - 1; i >= 0; --i)
        if (there(i)) first = i;
    }
    unsigned long long b = first < 0 ? 0ull : vf_rank(m, head + 4 * (at + (first >> 2) * kVsThreads) + (first & 3));
    if (extra_id >= 0) {
      const unsigned long long k = vf_rank(extra, extra_id);
      b = k > b ? k : b;
    }
    return b;
  }
  __device__ __forceinline__ VfPart sum(float c) const {
    const float ninf = -INFINITY, m = largest();
    VfPart mine{m, 0.f};
    if (fabsf(m) != INFINITY) {
      // two entries an instruction (x - max is rounded before it is scaled: the largest counts exactly 1)
      float2 z[2] = {{0.f, 0.f}, {0.f, 0.f}};
      const float2 neg = make_float2(-m, -m), cc = make_float2(c, c);
#pragma unroll
      for (int i = 0; i < 4 * NV; i += 2) {
        const float2 d = __fmul2_rn(__fadd2_rn(make_float2(v[i], v[i + 1]), neg), cc);
        z[(i >> 1) & 1] = __fadd2_rn(z[(i >> 1) & 1], make_float2(vf_ex2(d.x), vf_ex2(d.y)));
      }
      const float2 s = __fadd2_rn(z[0], z[1]);
      mine.z = s.x + s.y;
      if (mine.z != mine.z) {                             // a NaN's term is nothing
        mine.z = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) mine.z += vf_ex2((fmaxf(v[i], ninf) - m) * c);
      }
    } else {
      // equal infinities count 1 each (a NaN that is the row's as -infinity)
      int equal = 0;
#pragma unroll
      for (int i = 0; i < 4 * NV; ++i) equal += there(i) && fmaxf(v[i], ninf) == m;
      mine.z = (float)equal;
    }
    if (extra_id >= 0) mine = vf_merge(mine, VfPart{fmaxf(extra, ninf), 1.f}, c);
    return mine;
  }
};

// The slice's numbers out of its threads', into place `to`.
template <int NV, bool GREEDY>
__device__ __forceinline__ void vs_finish(const VfArgs& a, const VsSlice<NV>& s, float c, size_t to) {
  __shared__ VfPart part[kVsWarps];
  __shared__ unsigned long long best_s[kVsWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (GREEDY) {
    unsigned long long best = s.best();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) best_s[warp] = best;
  } else {
    VfPart mine = s.sum(c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      VfPart p;
      p.m = __shfl_xor_sync(0xffffffffu, mine.m, o);
      p.z = __shfl_xor_sync(0xffffffffu, mine.z, o);
      mine = vf_merge(mine, p, c);
    }
    if (lane == 0) part[warp] = mine;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (GREEDY) {
      unsigned long long best = best_s[0];
      for (int w = 1; w < kVsWarps; ++w) best = best_s[w] > best ? best_s[w] : best;
      static_cast<unsigned long long*>(a.stats)[to] = best;
    } else {
      VfPart mine = part[0];
      for (int w = 1; w < kVsWarps; ++w) mine = vf_merge(mine, part[w], c);
      static_cast<VfPart*>(a.stats)[to] = mine;
    }
  }
}

template <int NV, bool GREEDY>
__global__ void __launch_bounds__(kVsThreads)
verify_rows_kernel(const __grid_constant__ VfArgs a) {
  dependent_begin();
  const float* x = vf_row(a, blockIdx.x);
  if (!x) return;
  VsSlice<NV> s;
  s.load(a, x, blockIdx.y);
  vs_finish<NV, GREEDY>(a, s, (float)a.log2_t, (size_t)blockIdx.x * a.slices + blockIdx.y);
}

// ---- second launch, greedy: a warp a sequence
__global__ void __launch_bounds__(128) verify_greedy_kernel(const __grid_constant__ VfArgs a) {
  dependent_begin();
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b >= a.B) return;
  int row0, n;
  int* out = a.tokens + (size_t)b * a.ld_tokens;
  if (!vf_sequence(a, b, row0, n)) {
    for (int j = lane; j <= a.K; j += 32) out[j] = -1;
    if (lane == 0) { a.accepted[b] = 0; atomicOr(a.fault, (unsigned)kFaultTokenRange); }
    return;
  }
  // a lane a place: its row's arg max, and whether its draft is that
  int accepted = n, next = 0;
  bool found = false;
  for (int j0 = 0; j0 <= n && !found; j0 += 32) {
    const int j = j0 + lane;
    int best = -1, d = -1;
    if (j <= n) {
      const unsigned long long* s = static_cast<const unsigned long long*>(a.stats) + (size_t)(row0 + j) * a.slices;
      unsigned long long k = 0ull;
      for (int i = 0; i < a.slices; ++i) k = s[i] > k ? s[i] : k;
      best = (int)(0xffffffffu - (unsigned)k);
      if (j < n) {
        d = a.drafts[(size_t)b * a.ld_drafts + j];
        if (d < 0 || d >= a.V) d = -2;
      }
    }
    const unsigned stop = __ballot_sync(0xffffffffu, j <= n && (j == n || d != best));
    if (stop) {
      const int at = __ffs(stop) - 1;
      accepted = j0 + at;
      next = __shfl_sync(0xffffffffu, best, at);
      if (lane == at && d == -2) atomicOr(a.fault, (unsigned)kFaultTokenRange);
      found = true;
    }
  }
  for (int j = lane; j <= a.K; j += 32)
    out[j] = j < accepted ? a.drafts[(size_t)b * a.ld_drafts + j] : j == accepted ? next : -1;
  if (lane == 0) a.accepted[b] = accepted;
}

// ---- second launch, whole vocabulary: a cluster a sequence, its CTAs share the vocabulary
constexpr int kVdSeg = 128;                               // entries a warp takes at once

// 2^(i / 16) and 2^(i / 256): their products are the table of 256 that a CTA makes for itself.
__device__ const double kVfCoarse[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474,
};
__device__ const double kVfFine[16] = {
    1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175,
    1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738,
    1.0218971486541166, 1.0246677928971357, 1.0274459491187637, 1.030231637686041,
    1.0330248790212284, 1.0358256936019572, 1.0386341019613787, 1.041450124688316,
};

// A row's terms 2^((v - top) c) in 64 bits.  256 (v - top) c = n + f with |f| <= 1/2; 2^(n / 256) from the
// table and a power of two, 2^(f / 256) by its series to the third power (the fourth term is below
// 1.4e-13) (table-driven exponential, P. T. P. Tang, 1989).  What bounds the drawing is how many
// instructions its warps issue: some 16 a term, eight of them 64-bit.
struct VfTerm {
  double c256, top;             // 256 log2 e / T, the row's maximum
  float lo;                     // entries below it (2^-1000 of the largest) and NaN count 0
  bool infinite;                // the maximum is: entries equal to it count 1, all others 0
  __device__ __forceinline__ void set(float top_, double c, float reach) {       // reach: 1000 / c
    infinite = fabsf(top_) == INFINITY;
    top = top_;
    c256 = 256.0 * c;
    lo = top_;
    if (!infinite) {
      lo = top_ - reach;
      // (rounded down too far, an entry's n would not fit an exponent)
      while (lo < top_ && ((double)lo - (double)top_) * c < -1020.0) lo = nextafterf(lo, INFINITY);
    }
  }
  __device__ __forceinline__ double plain(float v, const double* table) const {  // of an entry that is not below lo
    const double magic = 6755399441055744.0;              // 1.5 * 2^52: rounds to an integer
    const double d = (double)v - top;
    const double big = fma(d, c256, magic);
    const int n = __double2loint(big);
    const double f = fma(d, c256, magic - big);
    // (ln2 / 256)^k / k!
    double p = fma(f, 3.308302680541371e-09, 3.665565596910106e-06);
    p = fma(f, p, 0.0027076061740622863);
    p = fma(f, p, 1.0);
    p *= table[n & 255];
    return __hiloint2double(__double2hiint(p) + ((n >> 8) << 20), __double2loint(p));
  }
  __device__ __forceinline__ double operator()(float v, const double* table) const {
    if (infinite) return fmaxf(v, -INFINITY) == (float)top ? 1.0 : 0.0;
    return v >= lo ? plain(v, table) : 0.0;
  }
  // Four at once, by a whole warp.
  __device__ __forceinline__ void four(const float (&v)[4], double (&to)[4], const double* table) const {
    const bool all = v[0] >= lo && v[1] >= lo && v[2] >= lo && v[3] >= lo;
    if (!infinite && __all_sync(0xffffffffu, all)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = plain(v[e], table);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = (*this)(v[e], table);
    }
  }
};

__device__ __forceinline__ double vf_warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The entries 4 i .. 4 i + 3 of a row (NaN behind its end).
__device__ __forceinline__ void vf_four(const float* x, int V, int i, bool aligned, float (&v)[4]) {
  if (aligned && 4 * i + 3 < V) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(x) + i);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = 4 * i + e < V ? __ldg(x + 4 * i + e) : __uint_as_float(0x7fffffffu);
  }
}

// max(p - w q, 0) is summed in the one pass over the rows that sums p and q, before w = sum p / sum q is known in
// 64 bits: with w0 from the first launch's sums, off by some 1e-7 of it, and beside it the q of the entries where
// p > w0 q, so that a sum of max(p - w q, 0) is that of max(p - w0 q, 0) less (w - w0) times that of the q.  That
// is wrong, by at most |w - w0| q, in the entries where p lies between w q and w0 q: they are counted with the
// wrong sign, or not at all.  Together that is |w - w0| sum q at most; where it could be more than kVdSlack of what
// is left to draw from, the pass is made again with w in w0's place (rows that are nearly alike).  The
// segment that is drawn from is computed again with w.  (Two passes, the terms between them in 100 KB of shared
// memory that leave an SM two CTAs: 55.5 us against 48.1 for 64 sequences of seven drafts, 11.6 against 11.2 for one.)
constexpr double kVdSlack = 1.0 / (1 << 17);
// How far u q and p have to lie apart, as a share of p, for the first launch's sums to tell them.  A term's exponent x
// is off by 3 |x| 2^-24 (its subtraction, its product, log2 e / T as a float), and the mean of |x| over a row's terms is
// log2 V, 24, at most; each of up to 20 rescalings on a term's way (threads, warps, slices; 55 with 13 million
// ids) adds an exponential's 2^-22 and two roundings: 2^-15 a row at most, and there are two.
constexpr double kVdDoubt = 1.0 / (1 << 14);
// What rounding leaves of numbers that are alike, as a share of them: 64-bit sums of some hundred additions in a row.
constexpr double kVdNothing = 1e-13;
template <int kVdThreads, int kCtas, int kAhead>
__global__ void __launch_bounds__(kVdThreads, kCtas)
verify_draw_kernel(const __grid_constant__ VfArgs a) {
  extern __shared__ __align__(16) double2 vd_smem[];      // the segments' two sums; before them the rows' numbers
  constexpr int kWarps = kVdThreads / 32;
  static_assert(4 * kWarps % 32 == 0, "whole warps go through the sums");
  __shared__ double table[256];
  __shared__ double sums[4 * kWarps];
  __shared__ double shared_tot[4];                        // this CTA's sums: p, q, max(p - w0 q, 0), q where p > w0 q
  enum { kDraw, kNothingLeft, kAgain };
  __shared__ int step_s;
  __shared__ double weight_s;
  __shared__ int first_bad;                               // 2 j: draft j does not stand; 2 j + 1: it may
  cg::cluster_group cluster = cg::this_cluster();
  const int C = gridDim.x, rank = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < 256; i += kVdThreads) table[i] = kVfCoarse[i >> 4] * kVfFine[i & 15];
  if (tid == 0) first_bad = 0x7fffffff;
  dependent_begin();
  int row0, n;
  int* out = a.tokens + (size_t)b * a.ld_tokens;
  if (!vf_sequence(a, b, row0, n)) {                      // (all CTAs of the cluster alike)
    if (rank == 0) {
      for (int j = tid; j <= a.K; j += kVdThreads) out[j] = -1;
      if (tid == 0) { a.accepted[b] = 0; atomicOr(a.fault, (unsigned)kFaultTokenRange); }
    }
    return;
  }
  // ---- the rows' maxima and sums, a warp a row: the logits' n + 1 rows, then the drafts' n; meanwhile
  // a thread a draft has its numbers on their way
  const float cf = (float)a.log2_t;
  const VfPart* stats = static_cast<const VfPart*>(a.stats);
  VfPart* rows = reinterpret_cast<VfPart*>(vd_smem);      // [2 K + 1]
  const bool proposed = a.draft_logits != nullptr;
  int d = -1;
  float u = 0.f, xd = 0.f, yd = 0.f;
  auto draft = [&](int j) {
    d = a.drafts[(size_t)b * a.ld_drafts + j];
    u = a.accept_u[(size_t)b * a.ld_u + j];
    if (d >= 0 && d < a.V) {
      xd = a.logits[(size_t)(row0 + j) * a.ld + d];
      if (proposed) yd = a.draft_logits[b * a.ld_seq + j * a.ld_place + d];
    }
  };
  int have = tid < n ? tid : -1;                          // whose numbers they are
  if (tid < n) draft(tid);
  for (int i = warp; i < (proposed ? 2 * n + 1 : n + 1); i += kWarps) {
    const size_t row = i <= n ? row0 + i : a.n_rows + (size_t)b * a.K + (i - n - 1);
    VfPart p{-INFINITY, 0.f};
    for (int s = lane; s < a.slices; s += 32) p = vf_merge(p, stats[row * a.slices + s], cf);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      VfPart q;
      q.m = __shfl_xor_sync(0xffffffffu, p.m, o);
      q.z = __shfl_xor_sync(0xffffffffu, p.z, o);
      p = vf_merge(p, q, cf);
    }
    if (lane == 0) rows[i] = p;
  }
  __syncthreads();
  // ---- which drafts stand
  VfTerm tp, tq;
  // draft j's p and q as they compare with u, given its rows' sums
  auto judge = [&](int j, double zp, double zq, double& px, double& uq) {
    if (j != have) { draft(j); have = j; }
    px = 0.0;
    uq = 0.0;
    if (d < 0 || d >= a.V) return;
    tp.set(rows[j].m, a.log2_t, a.reach);
    px = tp(xd, table) / zp;
    double qx = 1.0;
    if (proposed) {
      tq.set(rows[n + 1 + j].m, a.log2_t, a.reach);
      qx = tq(yd, table) / zq;
    }
    uq = (double)u * qx;
  };
  // the 64-bit sum of a row, by the whole CTA (all CTAs of the cluster do the same)
  auto row_sum = [&](const VfTerm& row, const float* x) {
    const bool aligned = ((uintptr_t)x & 15) == 0;
    double mine = 0.0;
    for (int s = warp; s * kVdSeg < a.V; s += kWarps) {
      float f[4];
      double v[4];
      vf_four(x, a.V, s * 32 + lane, aligned, f);
      row.four(f, v, table);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s * kVdSeg + 4 * lane + e < a.V) mine += v[e];
    }
    mine = vf_warp_sum(mine);
    __syncthreads();
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    double all = 0.0;
    for (int w = 0; w < kWarps; ++w) all += sums[w];
    return all;
  };
  int j;
  for (int from = 0;; from = j + 1) {
    for (int i = from + tid; i < n; i += kVdThreads) {
      double px, uq;
      judge(i, (double)rows[i].z, proposed ? (double)rows[n + 1 + i].z : 1.0, px, uq);
      const bool doubt = px > 0.0 && fabs(uq - px) <= kVdDoubt * px;
      if (doubt || !(uq < px)) atomicMin(&first_bad, 2 * i + (doubt ? 1 : 0));
    }
    __syncthreads();
    const int code = first_bad;
    j = min(code >> 1, n);
    if (j == n || !(code & 1)) break;
    double px, uq;
    judge(j, 1.0, 1.0, px, uq);                           // (sets the terms)
    const double zp = row_sum(tp, a.logits + (size_t)(row0 + j) * a.ld);
    const double zq = proposed ? row_sum(tq, a.draft_logits + b * a.ld_seq + j * a.ld_place) : 1.0;
    if (!(uq / zq < px / zp)) break;
    __syncthreads();
    if (tid == 0) first_bad = 0x7fffffff;
    __syncthreads();
  }
  const bool rest = j < n;
  d = rest ? a.drafts[(size_t)b * a.ld_drafts + j] : -1;
  if (rest && (d < 0 || d >= a.V) && rank == 0 && tid == 0) atomicOr(a.fault, (unsigned)kFaultTokenRange);
  // ---- the row (two rows) to draw from
  const bool minus_q = rest && proposed;
  const float* xp = a.logits + (size_t)(row0 + j) * a.ld;
  const float* xq = minus_q ? a.draft_logits + b * a.ld_seq + j * a.ld_place : xp;
  const bool ap = ((uintptr_t)xp & 15) == 0, aq = ((uintptr_t)xq & 15) == 0;
  tp.set(rows[j].m, a.log2_t, a.reach);
  tq = tp;
  double w0 = 0.0;
  if (minus_q) {
    tq.set(rows[n + 1 + j].m, a.log2_t, a.reach);
    w0 = (double)rows[j].z / (double)rows[n + 1 + j].z;
  }
  __syncthreads();                                        // (the rows' numbers give way to the segments')
  const int segs = (a.V + kVdSeg - 1) / kVdSeg;
  const int s0 = (int)((long long)segs * rank / C), s1 = (int)((long long)segs * (rank + 1) / C);
  // the four terms of a lane in a segment of a row (0 behind the vocabulary)
  auto look = [&](const VfTerm& row, const float* x, bool aligned, int s, double (&v)[4]) {
    float f[4];
    vf_four(x, a.V, s * 32 + lane, aligned, f);
    row.four(f, v, table);
    if ((s + 1) * kVdSeg > a.V) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (s * kVdSeg + 4 * lane + e >= a.V) v[e] = 0.0;
    }
  };
  for (int turn = rest ? 0 : 1; turn < 2; ++turn) {       // (the second where p and q leave nothing)
    const bool minus = turn == 0;
    double mine[4] = {0.0, 0.0, 0.0, 0.0};
    // the loads of kAhead segments go out together
    auto pass = [&](auto constant) {
      constexpr bool kQ = decltype(constant)::value;
      for (int first = s0 + warp; first < s1; first += kAhead * kWarps) {
        float fp[kAhead][4], fq[kAhead][4];
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
          const int s = first + x * kWarps;
          if (s >= s1) continue;
          vf_four(xp, a.V, s * 32 + lane, ap, fp[x]);
          if (kQ) vf_four(xq, a.V, s * 32 + lane, aq, fq[x]);
        }
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
          const int s = first + x * kWarps;
          if (s >= s1) continue;
          double vp[4], vq[4], r = 0.0, qa = 0.0;
          tp.four(fp[x], vp, table);
          if (kQ) tq.four(fq[x], vq, table);
          const int id = s * kVdSeg + 4 * lane;
          if ((s + 1) * kVdSeg > a.V) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (id + e >= a.V) { vp[e] = 0.0; if (kQ) vq[e] = 0.0; }
          }
          if (kQ) {
            mine[0] += (vp[0] + vp[1]) + (vp[2] + vp[3]);
            mine[1] += (vq[0] + vq[1]) + (vq[2] + vq[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const double over = fma(-w0, vq[e], vp[e]);
              if (over > 0.0) { r += over; qa += vq[e]; }
            }
            qa = vf_warp_sum(qa);
          } else {
            if (minus && (unsigned)(d - id) < 4u) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (id + e == d) vp[e] = 0.0;
            }
            r = (vp[0] + vp[1]) + (vp[2] + vp[3]);
          }
          r = vf_warp_sum(r);
          if (lane == 0) {
            vd_smem[s - s0] = make_double2(r, qa);
            mine[2] += r;
            mine[3] += qa;
          }
        }
      }
      if (kQ) {
        mine[0] = vf_warp_sum(mine[0]);
        mine[1] = vf_warp_sum(mine[1]);
      }
    };
    if (minus && minus_q) pass(std::true_type{});
    else pass(std::false_type{});
    // ---- the cluster's sums: lane r < C of warp 0 has CTA r's
    if (lane == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) sums[q * kWarps + warp] = mine[q];
    }
    __syncthreads();
    if (warp == 0) {                                      // lanes of kWarps a sum
#pragma unroll
      for (int at = lane; at < 4 * kWarps; at += 32) {
        double v = sums[at];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (at % kWarps == 0) shared_tot[at / kWarps] = v;
      }
    }
    cluster.sync();
    double total = 0.0, base = 0.0, own = 0.0, weight = 0.0;
    int last_rank = -1;
    if (warp == 0) {
      double t4[4] = {0.0, 0.0, 0.0, 0.0};
      if (lane < C) {
        const double* there = cluster.map_shared_rank(shared_tot, lane);
#pragma unroll
        for (int q = 0; q < 4; ++q) t4[q] = there[q];
      }
      double least = 0.0, slack = 0.0;
      if (minus && minus_q) {
        const double all_p = vf_warp_sum(t4[0]), all_q = vf_warp_sum(t4[1]);
        weight = all_p / all_q;
        // (a CTA with nothing to draw has exactly zero: below it, two CTAs would find the goal in their ranges)
        t4[2] = fma(w0 - weight, t4[3], t4[2]);
        if (!(t4[2] > kVdNothing * t4[0])) t4[2] = 0.0;
        least = kVdNothing * all_p;
        slack = fabs(w0 - weight) * all_q;
      }
      for (int r = 0; r < C; ++r) {                       // (in the same order everywhere)
        const double t = __shfl_sync(0xffffffffu, t4[2], r);
        if (r == rank) { base = total; own = t; }
        if (t > 0.0) last_rank = r;
        total += t;
      }
      // (all CTAs of the cluster have the same numbers and decide alike)
      if (lane == 0) {
        step_s = slack > kVdSlack * total ? kAgain : !minus || total > least ? kDraw : kNothingLeft;
        weight_s = weight;
      }
    }
    cluster.barrier_arrive();                             // its reads of the others' memory are done
    __syncthreads();
    if (step_s != kDraw) {
      if (step_s == kAgain) {                             // (once: the same sums give the same w, and no slack)
        w0 = weight_s;
        --turn;
      }
      cluster.barrier_wait();
      continue;
    }
    // (a number that is not in [0, 1) counts as the nearest that is)
    double goal = (double)a.next_u[b] * total;
    if (!(goal >= 0.0)) goal = 0.0;
    const bool past = goal >= total;                      // the last id with any
    const bool here = past ? rank == last_rank : base <= goal && goal < base + own;
    if (here && warp == 0) {
      // the segment, 32 at a time, and the place in it
      double run = base;
      int seg = -1, last_seg = 0;
      double seg_base = 0.0;
      for (int i0 = 0; i0 < s1 - s0 && seg < 0; i0 += 32) {
        double v = 0.0;
        if (i0 + lane < s1 - s0) {
          const double2 both = vd_smem[i0 + lane];
          v = minus && minus_q ? fma(w0 - weight, both.y, both.x) : both.x;
        }
        double inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double w = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += w;
        }
        const unsigned any = __ballot_sync(0xffffffffu, v > 0.0);
        const unsigned hit = past ? 0u : __ballot_sync(0xffffffffu, v > 0.0 && run + inc > goal);
        if (hit) {
          seg = i0 + __ffs(hit) - 1;
          double before = __shfl_up_sync(0xffffffffu, inc, 1);
          if (lane == 0) before = 0.0;
          seg_base = run + __shfl_sync(0xffffffffu, before, __ffs(hit) - 1);
        }
        if (any) last_seg = i0 + 31 - __clz(any);
        run += __shfl_sync(0xffffffffu, inc, 31);
      }
      const bool take_last = seg < 0;                     // (rounding passed the last border)
      if (take_last) seg = last_seg;
      // what is drawn from in the segment, four entries a lane
      double v[4];
      look(tp, xp, ap, s0 + seg, v);
      if (minus && minus_q) {
        double vq[4];
        look(tq, xq, aq, s0 + seg, vq);
#pragma unroll
        for (int e = 0; e < 4; ++e) vq[e] = fmax(fma(-weight, vq[e], v[e]), 0.0);
        // (where nothing is left but what rounding made of a sum, any id with a probability)
        if (__any_sync(0xffffffffu, vq[0] > 0.0 || vq[1] > 0.0 || vq[2] > 0.0 || vq[3] > 0.0)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = vq[e];
        }
      } else if (minus) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((s0 + seg) * kVdSeg + 4 * lane + e == d) v[e] = 0.0;
      }
      const double four = (v[0] + v[1]) + (v[2] + v[3]);
      double inc = four;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double w = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += w;
      }
      double run4 = seg_base + inc - four;
      int first = 0x7fffffff, last = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int id = (s0 + seg) * kVdSeg + 4 * lane + e;
        run4 += v[e];
        if (v[e] > 0.0) {
          last = id;
          if (!take_last && run4 > goal && first == 0x7fffffff) first = id;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
        last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
      }
      const int next = first != 0x7fffffff ? first : last;
      for (int i = lane; i <= a.K; i += 32)
        out[i] = i < j ? a.drafts[(size_t)b * a.ld_drafts + i] : i == j ? next : -1;
      if (lane == 0) a.accepted[b] = j;
    }
    cluster.barrier_wait();                               // nobody leaves before all have read
    break;
  }
}

// ---- top_k: a CTA a row finds the kept entries.
// The k-th largest of the threads' own maxima is at most the row's k-th largest; the entries at or
// above it are few more than k.  They are listed in a second look at the row (from L2) and sorted by
// (value, id).  Where they are too many for the list (equal logits in masses) the k-th largest is
// found digit by digit over the whole row.
// (512 threads: three CTAs of them fit an SM, and one's sort runs under another's loads.  250 rows of 49,152:
// 21.4 us, with 1,024 threads, one CTA an SM, 35.)
constexpr int kVkThreads = 512, kVkWarps = kVkThreads / 32, kVkList = 4096;
constexpr int kVkMaxima = kVfMaxTopK / kVkThreads;        // maxima a thread keeps: together at least top_k

struct VkShared {
  unsigned long long list[kVkList];
  double sums[kVkWarps];
  unsigned int hist[256];
  unsigned int digit, need, count;
  unsigned int best[kVkWarps];
};

// The key of the need-th largest of what `each` hands to its argument, 8 bits at a time; `need` is
// left as how many equals of it are among them.
template <typename Each>
__device__ __forceinline__ unsigned int vk_select(VkShared& s, unsigned int need, unsigned int& equal_need, Each each) {
  const int tid = threadIdx.x;
  unsigned int prefix = 0u;
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    const unsigned int mask = pass == 0 ? 0u : 0xffffffffu << (shift + 8);
    if (tid < 256) s.hist[tid] = 0u;
    __syncthreads();
    each([&](unsigned int k) {
      if ((k & mask) == prefix) atomicAdd(&s.hist[(k >> shift) & 255u], 1u);
    });
    __syncthreads();
    if (tid < 32) {                        // lane l: digits 255 - 8 l down to 248 - 8 l
      unsigned int c[8], sum = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) { c[i] = s.hist[255 - 8 * tid - i]; sum += c[i]; }
      unsigned int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (tid >= o) inc += v;
      }
      unsigned int before = inc - sum;
      if (before < need && inc >= need) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < need && before + c[i] >= need) {
            s.digit = 255 - 8 * tid - i;
            s.need = need - before;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    prefix |= s.digit << shift;
    need = s.need;
    __syncthreads();
  }
  equal_need = need;
  return prefix;
}

__global__ void __launch_bounds__(kVkThreads, 3)
verify_kept_kernel(const __grid_constant__ VfArgs a) {
  __shared__ VkShared s;
  dependent_begin();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V, k = a.top_k;
  const float* x = vf_row(a, blockIdx.x);
  if (!x) return;
  const int head = min(V, (int)((0u - (unsigned)((uintptr_t)x >> 2)) & 3u));
  const int n4 = (V - head) >> 2, tail = V - head - 4 * n4;
  const float4* x4 = reinterpret_cast<const float4*>(x + head);
  // f(value, id, turn) for every entry of the row
  auto each = [&](auto f) {
    constexpr int U = 4;
    for (int i0 = tid; i0 < n4; i0 += U * kVkThreads) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kVkThreads < n4) v[u] = __ldg(x4 + i0 + u * kVkThreads);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kVkThreads;
        if (i < n4) {
          f(v[u].x, head + 4 * i, u);
          f(v[u].y, head + 4 * i + 1, u);
          f(v[u].z, head + 4 * i + 2, u);
          f(v[u].w, head + 4 * i + 3, u);
        }
      }
    }
    if (tid < head + tail) {
      const int id = tid < head ? tid : 4 * n4 + tid;
      f(x[id], id, 0);
    }
  };
  float mine[kVkMaxima];
#pragma unroll
  for (int i = 0; i < kVkMaxima; ++i) mine[i] = -INFINITY;
  each([&](float v, int, int u) { mine[u % kVkMaxima] = fmaxf(mine[u % kVkMaxima], v); });
  unsigned int best = 0u;
#pragma unroll
  for (int i = 0; i < kVkMaxima; ++i) best = max(best, vf_key(mine[i]));
  best = __reduce_max_sync(0xffffffffu, best);
  if (lane == 0) s.best[warp] = best;
  if (tid == 0) s.count = 0u;
  __syncthreads();
  best = __reduce_max_sync(0xffffffffu, s.best[lane % kVkWarps]);
  const float top = vf_value(best);
  // (a maximum of no entries is -infinity; where that is among the k largest everything is listed)
  unsigned int equal;
  const unsigned int floor_key = vk_select(s, (unsigned)k, equal, [&](auto f) {
#pragma unroll
    for (int i = 0; i < kVkMaxima; ++i) f(vf_key(mine[i]));
  });
  const float floor_value = vf_value(floor_key);
  each([&](float v, int id, int) {
    if (fmaxf(v, -INFINITY) >= floor_value) {              // (NaN counts as -infinity)
      const unsigned int at = atomicAdd(&s.count, 1u);
      if (at < kVkList) s.list[at] = vf_rank(v, id);
    }
  });
  __syncthreads();
  unsigned int n = s.count;
  if (n > kVkList) {
    // list the larger ones and the equals with the lowest ids: the equals' ids are taken in the row's order
    const unsigned int kth = vk_select(s, (unsigned)k, equal, [&](auto f) { each([&](float v, int, int) { f(vf_key(v)); }); });
    if (tid == 0) s.count = 0u;
    __syncthreads();
    each([&](float v, int id, int) {
      if (vf_key(v) > kth) s.list[atomicAdd(&s.count, 1u)] = vf_rank(v, id);
    });
    __syncthreads();
    unsigned int left = equal;
    const unsigned int at0 = (unsigned)k - equal;
    for (int i0 = 0; i0 < V && left > 0u; i0 += kVkThreads) {
      const bool eq = i0 + tid < V && vf_key(x[i0 + tid]) == kth;
      const unsigned int votes = __ballot_sync(0xffffffffu, eq);
      if (lane == 0) s.best[warp] = __popc(votes);
      __syncthreads();
      unsigned int before = __popc(votes & ((1u << lane) - 1u)), all = 0u;
      for (int w = 0; w < kVkWarps; ++w) {
        if (w < warp) before += s.best[w];
        all += s.best[w];
      }
      if (eq && before < left) s.list[at0 + (equal - left) + before] = vf_rank(x[i0 + tid], i0 + tid);
      left -= min(left, all);
      __syncthreads();
    }
    n = (unsigned)k;
    __syncthreads();
  }
  // sort: the largest first
  int np2 = 1;
  while (np2 < (int)n) np2 <<= 1;
  for (int i = (int)n + tid; i < np2; i += kVkThreads) s.list[i] = 0ull;
  __syncthreads();
  for (int size = 2; size <= np2; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = tid; i < np2; i += kVkThreads) {
        const int p = i ^ stride;
        if (p > i) {
          const unsigned long long u = s.list[i], v = s.list[p];
          if ((u > v) != ((i & size) == 0)) { s.list[i] = v; s.list[p] = u; }
        }
      }
      __syncthreads();
    }
  // the kept ones, their sum in 64 bits
  const double c = a.log2_t;
  double z = 0.0;
  for (int i = tid; i < k; i += kVkThreads) {
    const unsigned long long r = s.list[i];
    const float v = vf_value((unsigned int)(r >> 32));
    const size_t at = (size_t)blockIdx.x * k + i;
    a.list_v[at] = v;
    a.list_i[at] = (int)(0xffffffffu - (unsigned)r);
    z += v == top ? 1.0 : fabsf(top) == INFINITY ? 0.0 : exp2(((double)v - (double)top) * c);
  }
  z = vf_warp_sum(z);
  if (lane == 0) s.sums[warp] = z;
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < kVkWarps; ++w) t += s.sums[w];
    static_cast<VfKept*>(a.stats)[blockIdx.x] = VfKept{t, s.list[k - 1], top, 0};
  }
}

// ---- second launch, top_k: a CTA a sequence
constexpr int kVlThreads = 256;

__global__ void __launch_bounds__(kVlThreads)
verify_kept_draw_kernel(const __grid_constant__ VfArgs a) {
  __shared__ unsigned long long order[kVfMaxTopK];         // (id, place in the list), by id
  __shared__ double term[kVfMaxTopK];
  int* term_ids = reinterpret_cast<int*>(term);            // (before the terms are)
  __shared__ double sums[kVlThreads / 32];
  __shared__ int first_bad, chosen;
  dependent_begin();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.top_k;
  constexpr int kWarps = kVlThreads / 32;
  int row0, n;
  int* out = a.tokens + (size_t)b * a.ld_tokens;
  if (!vf_sequence(a, b, row0, n)) {
    for (int j = tid; j <= a.K; j += kVlThreads) out[j] = -1;
    if (tid == 0) { a.accepted[b] = 0; atomicOr(a.fault, (unsigned)kFaultTokenRange); }
    return;
  }
  if (tid == 0) { first_bad = 0x7fffffff; chosen = -1; }
  __syncthreads();
  const VfKept* kept = static_cast<const VfKept*>(a.stats);
  const double c = a.log2_t;
  auto value = [&](const VfKept& r, float v, int id) {     // the term of a row's entry, 0 where it is not kept
    if (vf_rank(v, id) < r.thr) return 0.0;
    v = fmaxf(v, -INFINITY);
    return v == r.top ? 1.0 : fabsf(r.top) == INFINITY ? 0.0 : exp2(((double)v - (double)r.top) * c);
  };
  for (int j = tid; j < n; j += kVlThreads) {              // a thread a draft
    const int d = a.drafts[(size_t)b * a.ld_drafts + j];
    bool stands = false;
    if (d >= 0 && d < a.V) {
      const VfKept p = kept[row0 + j];
      const double px = value(p, a.logits[(size_t)(row0 + j) * a.ld + d], d) / p.z;
      double qx = 1.0;
      if (a.draft_logits) {
        const VfKept q = kept[a.n_rows + b * a.K + j];
        qx = value(q, a.draft_logits[b * a.ld_seq + j * a.ld_place + d], d) / q.z;
      }
      stands = (double)a.accept_u[(size_t)b * a.ld_u + j] * qx < px;
    }
    if (!stands) atomicMin(&first_bad, j);
  }
  __syncthreads();
  const int j = min(first_bad, n);
  const bool rest = j < n, minus_q = rest && a.draft_logits != nullptr;
  const int d = rest ? a.drafts[(size_t)b * a.ld_drafts + j] : -1;
  if (rest && (d < 0 || d >= a.V) && tid == 0) atomicOr(a.fault, (unsigned)kFaultTokenRange);
  const VfKept p = kept[row0 + j];
  const VfKept q = minus_q ? kept[a.n_rows + b * a.K + j] : p;
  const float* xq = minus_q ? a.draft_logits + b * a.ld_seq + j * a.ld_place : nullptr;
  const double weight = p.z / q.z;
  const size_t list = (size_t)(row0 + j) * k;
  // the kept ids in ascending order: an id's place is how many are smaller where a thread has one id,
  // else they are sorted
  if (k <= kVlThreads) {
    unsigned long long mine = 0ull;
    if (tid < k) term_ids[tid] = a.list_i[list + tid];
    __syncthreads();
    if (tid < k) {
      const int id = term_ids[tid];
      mine = ((unsigned long long)(unsigned)id << 32) | (unsigned)tid;
      int at = 0;
      for (int i = 0; i < k; ++i) at += term_ids[i] < id;
      order[at] = mine;
    }
    __syncthreads();
  } else {
    int np2 = 1;
    while (np2 < k) np2 <<= 1;
    for (int i = tid; i < np2; i += kVlThreads)
      order[i] = i < k ? ((unsigned long long)(unsigned)a.list_i[list + i] << 32) | (unsigned)i : ~0ull;
    __syncthreads();
    for (int size = 2; size <= np2; size <<= 1)
      for (int stride = size >> 1; stride > 0; stride >>= 1) {
        for (int i = tid; i < np2; i += kVlThreads) {
          const int o = i ^ stride;
          if (o > i) {
            const unsigned long long u = order[i], v = order[o];
            if ((u < v) != ((i & size) == 0)) { order[i] = v; order[o] = u; }
          }
        }
        __syncthreads();
      }
  }
  int next = 0;
  for (int turn = rest ? 0 : 1; turn < 2; ++turn) {
    // a thread's entries lie together: `per` of them
    const int per = (k + kVlThreads - 1) / kVlThreads, lo = min(k, tid * per), hi = min(k, lo + per);
    double mine = 0.0;
    for (int i = lo; i < hi; ++i) {
      const int id = (int)(order[i] >> 32);
      double t = value(p, a.list_v[list + (unsigned)order[i]], id);
      if (turn == 0) {
        if (minus_q) t = fmax(t - weight * value(q, xq[id], id), 0.0);
        else if (id == d) t = 0.0;
      }
      term[i] = t;
      mine += t;
    }
    double inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    double prev = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) prev = 0.0;
    __syncthreads();
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    double base = 0.0, total = 0.0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) base = total;
      total += sums[w];
    }
    if (!(total > 0.0)) continue;
    double goal = (double)a.next_u[b] * total;
    if (!(goal >= 0.0)) goal = 0.0;
    if (base + prev <= goal && goal < base + inc) {
      double run = base + prev;
      int at = -1;
      for (int i = lo; i < hi; ++i) {
        if (term[i] > 0.0) at = (int)(order[i] >> 32);     // (the last one where rounding passes the end)
        run += term[i];
        if (run > goal) break;
      }
      chosen = at;
    }
    __syncthreads();
    const bool past = chosen < 0;
    __syncthreads();
    if (past) {                                            // the number was not below 1: the last id with any
      for (int i = lo; i < hi; ++i)
        if (term[i] > 0.0) atomicMax(&chosen, (int)(order[i] >> 32));
      __syncthreads();
    }
    next = chosen;
    break;
  }
  for (int i = tid; i <= a.K; i += kVlThreads)
    out[i] = i < j ? a.drafts[(size_t)b * a.ld_drafts + i] : i == j ? next : -1;
  if (tid == 0) a.accepted[b] = j;
}

// How the first launch cuts rows: vectors of four a slice, and slices.  A CTA takes 12 vectors a
// thread where there are rows enough to fill the chip with such CTAs, else 4.  Whether it does.
constexpr int kVsMany = 12, kVsFew = 4;
static bool vf_cut(const VfArgs& a, int rows, int& vectors, int& slices) {
  const long long n4 = a.V / 4 + 1;
  const bool many = (n4 + kVsMany * kVsThreads - 1) / (kVsMany * kVsThreads) * rows >= 2 * kSmCount;
  const long long per = (many ? kVsMany : kVsFew) * kVsThreads;
  vectors = (int)per;
  slices = (int)((n4 + per - 1) / per);
  return many;
}

constexpr size_t kVdMost = 200 * 1024;

template <int kThreads, int kCtas, int kAhead>
static int vd_launch(const VfArgs& a, int C, size_t smem, cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  // (the limit is asked for once a device, and always for the most: two threads that ask for what they each need
  // could leave the smaller one)
  constexpr int kDevices = 64;
  static bool asked[kDevices];
  if (dev >= kDevices || !asked[dev]) {
    e = cudaFuncSetAttribute(verify_draw_kernel<kThreads, kCtas, kAhead>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kVdMost);
    if (e != cudaSuccess) return (int)e;
    if (dev < kDevices) asked[dev] = true;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = C * a.B <= kSmCount ? dependent_launch_enabled() : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C, a.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, verify_draw_kernel<kThreads, kCtas, kAhead>, a);
  return e == cudaSuccess ? launch_status() : (int)e;
}

}  // namespace cretif

using namespace cretif;

extern "C" int cretif_max_top_k();

extern "C" long long cretif_verify_scratch(int n_rows, int B, int K, int V, int top_k, int draft_rows) {
  if (n_rows <= 0 || B < 0 || K < 0 || V <= 0) return 0;
  const long long rows = (long long)n_rows + (draft_rows ? (long long)B * K : 0);
  if (top_k > 0 && top_k < V) return rows * (long long)(sizeof(VfKept) + 8LL * top_k);
  return rows * 8LL * (V / 4 / (kVsFew * kVsThreads) + 1);
}

extern "C" int cretif_verify_drafts(const float* logits, long long ld, int n_rows, const int* cu,
                                    const int* drafts, long long ld_drafts, int K, const float* draft_logits,
                                    long long ld_seq, long long ld_place, const float* accept_u,
                                    long long ld_u, const float* next_u, int B, int V, double temperature,
                                    int top_k, int* accepted, int* tokens, long long ld_tokens,
                                    void* scratch, unsigned int* fault, void* stream) {
  if (B <= 0) return kOk;
  if (V <= 0 || ld < 0 || K < 0 || n_rows <= 0 || (B > 1 && ld_tokens < K + 1) || top_k < 0 ||
      temperature != temperature || (temperature > 0 && top_k > kVfMaxTopK && top_k < V) || ld_drafts < 0 || ld_u < 0 ||
      ld_seq < 0 || ld_place < 0 || B > 65535 || !scratch)
    return kBadArgument;
  const bool greedy = temperature <= 0.0;
  if (greedy) draft_logits = nullptr;
  const long long rows = (long long)n_rows + (draft_logits ? (long long)B * K : 0);
  const bool kept = !greedy && top_k > 0 && top_k < V;
  if (rows > 0x7fffffffLL) return kBadArgument;
  cudaStream_t st = (cudaStream_t)stream;
  VfArgs a{logits, ld, n_rows, cu, drafts, ld_drafts, K, B, V, draft_logits, ld_seq, ld_place, accept_u, ld_u, next_u,
           greedy ? 1.0 : fmin(fmax(1.4426950408889634 / temperature, 1e-30), 3e38), 0.f, top_k, accepted, tokens, ld_tokens, fault, scratch, 0, 0,
           nullptr, nullptr};
  a.reach = (float)fmin(1000.0 / a.log2_t, 3e38);
  if (kept) {
    a.list_v = reinterpret_cast<float*>(static_cast<char*>(scratch) + rows * sizeof(VfKept));
    a.list_i = reinterpret_cast<int*>(a.list_v + rows * top_k);
    launch_dependent(verify_kept_kernel, dim3((unsigned)rows), dim3(kVkThreads), 0, st, a);
    launch_dependent(verify_kept_draw_kernel, dim3(B), dim3(kVlThreads), 0, st, a);
    return launch_status();
  }
  const bool many = vf_cut(a, (int)rows, a.slice_vectors, a.slices);
  auto kernel = greedy ? (many ? verify_rows_kernel<kVsMany, true> : verify_rows_kernel<kVsFew, true>)
                       : (many ? verify_rows_kernel<kVsMany, false> : verify_rows_kernel<kVsFew, false>);
  launch_dependent(kernel, dim3((unsigned)rows, a.slices), dim3(kVsThreads), 0, st, a);
  if (greedy) {
    launch_dependent(verify_greedy_kernel, dim3((B + 3) / 4), dim3(128), 0, st, a);
    return launch_status();
  }
  // CTAs a sequence: as many as a cluster holds, 1,024 entries each at least
  int C = 8;
  while (C > 1 && V < 1024 * C) C >>= 1;
  const int segs = ((V + kVdSeg - 1) / kVdSeg + C - 1) / C + 1;
  // segments' sums, and before them the rows' numbers (half of 16 bytes each)
  const long long room = segs > K + 1LL ? segs : K + 1LL;
  if (K > 8191 || room * 16 > (long long)kVdMost) return kBadArgument;
  const size_t smem = (size_t)room * 16;
  // A CTA an SM of 512 threads, or four of 256, which are all there at once.  (One sequence 13.8 us with 256 threads,
  // 64 sequences 54.3 with two CTAs of 512.)
  return C * B <= kSmCount ? vd_launch<512, 1, 2>(a, C, smem, st) : vd_launch<256, 4, 1>(a, C, smem, st);
}
