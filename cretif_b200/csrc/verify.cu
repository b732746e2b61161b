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
// A row's terms are 2^((x - max) / T log2 e); an entry equal to the row's maximum counts 1 whatever
// it is, so that a row of equal infinities is uniform; NaN counts as -infinity.  Sums are 64-bit: the
// drawn id is decided at one of V borders, and sums that are off by 1e-8 of the total would draw
// another id once in V * 1e-8 draws (1 in 2,000 at 49,152 ids).
//
// The reference has no counterpart (its sampling: src/embedding.cu:343-406).
#include "api.h"
#include "common.cuh"

namespace cretif {

constexpr int kVfThreads = 1024;

__device__ __forceinline__ unsigned int vf_key(float v) {
  if (v == 0.f) v = 0.f;                                   // the two zeros are equal
  if (v != v) v = -INFINITY;
  const unsigned int b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);       // larger float -> larger key
}

template <typename V, typename Op>
__device__ __forceinline__ V vf_reduce(V v, V* scratch, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[threadIdx.x & 31];                           // 32 warps
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

struct VfRow {                // a row's distribution: kept are (key, id) at or before the threshold
  const float* x;
  unsigned int top;           // key of the largest
  float top_value;
  unsigned int thr;           // key of the last one kept, and its largest kept id
  int thr_id;
  double total;
};

// A kept entry's term (0 where it is not kept).
__device__ __forceinline__ double vf_term(const VfRow& r, int i, double inv_t) {
  const float v = r.x[i];
  const unsigned int k = vf_key(v);
  if (k < r.thr || (k == r.thr && i > r.thr_id)) return 0.0;
  return k == r.top ? 1.0 : v != v ? 0.0 : exp(((double)v - (double)r.top_value) * inv_t);
}

struct VfShared {
  unsigned int u[32];
  double d[32];
  int i[32];
  int hist[256];
  unsigned int prefix;
  int need;
};

__device__ void vf_row(VfRow& r, const float* x, int V, int top_k, double inv_t, VfShared& s) {
  const int tid = threadIdx.x;
  r.x = x;
  unsigned int best = 0u;
  for (int i = tid; i < V; i += kVfThreads) best = max(best, vf_key(x[i]));
  best = vf_reduce(best, s.u, [](unsigned a, unsigned b) { return a > b ? a : b; });
  r.top = best;
  r.top_value = __uint_as_float((best & 0x80000000u) ? (best & 0x7fffffffu) : ~best);
  r.thr = 0u;
  r.thr_id = V - 1;
  if (top_k > 0 && top_k < V) {
    // the key of the k-th largest, 8 bits at a time, then the id of the last of its equals kept
    if (tid == 0) { s.prefix = 0u; s.need = top_k; }
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      if (tid < 256) s.hist[tid] = 0;
      __syncthreads();
      const unsigned int mask = pass == 0 ? 0u : 0xffffffffu << (shift + 8), prefix = s.prefix;
      for (int i = tid; i < V; i += kVfThreads) {
        const unsigned int k = vf_key(x[i]);
        if ((k & mask) == prefix) atomicAdd(&s.hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int need = s.need, b = 255;
        for (; b > 0 && s.hist[b] < need; --b) need -= s.hist[b];
        s.prefix = prefix | ((unsigned int)b << shift);
        s.need = need;
      }
      __syncthreads();
    }
    r.thr = s.prefix;
    // equals of the threshold in id order: the need-th one's id
    int left = s.need, id = V - 1;
    for (int i0 = 0; i0 < V && left > 0; i0 += kVfThreads) {
      const bool eq = i0 + tid < V && vf_key(x[i0 + tid]) == r.thr;
      const int n = __syncthreads_count(eq);
      if (n >= left) {
        const unsigned int mine = __ballot_sync(0xffffffffu, eq);
        __syncthreads();
        if ((tid & 31) == 0) s.i[tid >> 5] = __popc(mine);
        __syncthreads();
        int before = 0;
        for (int w = 0; w < (tid >> 5); ++w) before += s.i[w];
        before += __popc(mine & ((1u << (tid & 31)) - 1u));
        if (eq && before == left - 1) s.need = i0 + tid;
        __syncthreads();
        id = s.need;
      }
      left -= n;
    }
    r.thr_id = id;
  }
  double sum = 0.0;
  for (int i = tid; i < V; i += kVfThreads) sum += vf_term(r, i, inv_t);
  r.total = vf_reduce(sum, s.d, [](double a, double b) { return a + b; });
}

__global__ void __launch_bounds__(kVfThreads)
verify_kernel(const float* __restrict__ logits, int ld, const int* __restrict__ cu, int n_rows,
              const int* __restrict__ drafts, int ld_drafts, int K, const float* __restrict__ draft_logits,
              long long ld_seq, long long ld_place, const float* __restrict__ accept_u, int ld_u,
              const float* __restrict__ next_u, int V, double temperature, int top_k,
              int* __restrict__ accepted, int* __restrict__ tokens, int ld_tokens,
              unsigned int* __restrict__ fault) {
  __shared__ VfShared s;
  const int b = blockIdx.x, tid = threadIdx.x;
  dependent_begin();
  const int row0 = cu[b];
  int n = cu[b + 1] - row0 - 1;
  if (n < 0 || n > K || row0 < 0 || row0 + n >= n_rows) {      // no row of the logits, or more drafts than there are
    if (tid == 0) {
      atomicOr(fault, (unsigned)kFaultTokenRange);
      accepted[b] = 0;
    }
    for (int j = tid; j <= K; j += kVfThreads) tokens[(size_t)b * ld_tokens + j] = -1;
    return;
  }
  const bool greedy = temperature <= 0.0;
  const double inv_t = greedy ? 1.0 : 1.0 / temperature;
  int j = 0, next = 0;
  VfRow p, q;
  for (;; ++j) {
    const float* x = logits + (size_t)(row0 + j) * ld;
    if (greedy) {
      unsigned long long best = 0ull;
      for (int i = tid; i < V; i += kVfThreads) {
        const unsigned long long k = ((unsigned long long)vf_key(x[i]) << 32) | (0xffffffffu - (unsigned)i);
        if (k > best) best = k;
      }
      best = vf_reduce(best, reinterpret_cast<unsigned long long*>(s.d),
                       [](unsigned long long a, unsigned long long c) { return a > c ? a : c; });
      next = (int)(0xffffffffu - (unsigned)best);
    } else {
      vf_row(p, x, V, top_k, inv_t, s);
    }
    if (j == n) break;
    const int d = drafts[(size_t)b * ld_drafts + j];
    const bool in = d >= 0 && d < V;
    if (!in && tid == 0) atomicOr(fault, (unsigned)kFaultTokenRange);
    bool stands;
    if (greedy) {
      stands = in && d == next;
    } else {
      if (draft_logits) vf_row(q, draft_logits + b * ld_seq + j * ld_place, V, top_k, inv_t, s);
      const double u = accept_u[(size_t)b * ld_u + j];
      const double px = in ? vf_term(p, d, inv_t) / p.total : 0.0;
      const double qx = !in ? 0.0 : draft_logits ? vf_term(q, d, inv_t) / q.total : 1.0;
      stands = in && u * qx < px;
    }
    if (!stands) break;
  }
  if (!greedy) {
    // the token: from max(p - q, 0) behind a draft that did not stand, else (and where nothing is
    // left of p) from p
    const bool rest = j < n;
    const int d = rest ? drafts[(size_t)b * ld_drafts + j] : -1;
    const double wq = rest && draft_logits ? p.total / q.total : 0.0;
    auto term = [&](int i, bool minus) {
      double v = vf_term(p, i, inv_t);
      if (!minus) return v;
      if (draft_logits) return fmax(v - wq * vf_term(q, i, inv_t), 0.0);
      return i == d ? 0.0 : v;
    };
    const int chunk = (V + kVfThreads - 1) / kVfThreads, lo = min(V, tid * chunk), hi = min(V, lo + chunk);
    for (int turn = rest ? 0 : 1; turn < 2; ++turn) {
      double mine = 0.0;
      for (int i = lo; i < hi; ++i) mine += term(i, turn == 0);
      double inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, inc, o);
        if ((tid & 31) >= o) inc += v;
      }
      // a thread's interval [before, after): each begins exactly where the one before it ends
      double prev = __shfl_up_sync(0xffffffffu, inc, 1);
      if ((tid & 31) == 0) prev = 0.0;
      __syncthreads();
      if ((tid & 31) == 31) s.d[tid >> 5] = inc;
      if (tid == 0) s.need = -1;
      __syncthreads();
      double base = 0.0, total = 0.0;
      for (int w = 0; w < 32; ++w) {
        if (w == (tid >> 5)) base = total;
        total += s.d[w];
      }
      if (!(total > 0.0)) continue;
      const double goal = (double)next_u[b] * total;
      if (base + prev <= goal && goal < base + inc) {
        double run = base + prev;
        int at = -1;
        for (int i = lo; i < hi; ++i) {
          const double v = term(i, turn == 0);
          if (v > 0.0) at = i;                 // (the chunk's last one where rounding passes its end)
          run += v;
          if (run > goal) break;
        }
        s.need = at;
      }
      __syncthreads();
      next = s.need;
      if (next < 0) {                          // the number was not in [0, 1): the last id with any
        __syncthreads();
        int last = -1;
        for (int i = lo; i < hi; ++i)
          if (term(i, turn == 0) > 0.0) last = i;
        next = vf_reduce(last, s.i, [](int a, int c) { return a > c ? a : c; });
      }
      break;
    }
  }
  for (int i = tid; i <= K; i += kVfThreads)
    tokens[(size_t)b * ld_tokens + i] = i < j ? drafts[(size_t)b * ld_drafts + i] : i == j ? next : -1;
  if (tid == 0) accepted[b] = j;
}

}  // namespace cretif

using namespace cretif;

extern "C" int cretif_max_top_k();

extern "C" int cretif_verify_drafts(const float* logits, int ld, int n_rows, const int* cu,
                                    const int* drafts, int ld_drafts, int K, const float* draft_logits,
                                    long long ld_seq, long long ld_place, const float* accept_u,
                                    int ld_u, const float* next_u, int B, int V, double temperature,
                                    int top_k, int* accepted, int* tokens, int ld_tokens,
                                    unsigned int* fault, void* stream) {
  if (B <= 0) return kOk;
  if (V <= 0 || ld < V || K < 0 || n_rows <= 0 || ld_tokens < K + 1 || top_k < 0 || temperature != temperature ||
      (temperature > 0 && top_k > cretif_max_top_k() && top_k < V) || (K > 0 && ld_drafts < K) ||
      (draft_logits && ld_place < V))
    return kBadArgument;
  launch_dependent(verify_kernel, dim3(B), dim3(kVfThreads), 0, (cudaStream_t)stream, logits, ld, cu, n_rows,
                   drafts, ld_drafts, K, draft_logits, ld_seq, ld_place, accept_u, ld_u, next_u, V,
                   temperature, top_k, accepted, tokens, ld_tokens, fault);
  return launch_status();
}
