// Attention of few new tokens a sequence for a batch whose sequences share prefixes: the keys of a
// group's prefix are read once for all its members, each sequence's own keys once for its tokens
// (attn_shared.h has the formula).  The reference decodes one sequence at a time and has nothing of
// the kind (its attention walks one cache, src/attention.cu:410-494).
//
// shared_pieces: a block of 256 threads per (item, key/value head), 32 rows and 64 keys a step in
// 32-bit FMA; every element type.  shared_join: a warp per row joins its pieces.
#include "api.h"
#include "attn_shared.h"

namespace cretif {

constexpr int kShRows = 32, kShThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kShThreads)
shared_pieces_kernel(const SharedArgs a) {
  extern __shared__ __align__(16) float sh_smem[];
  const int hd = a.hd, ldk = hd + 4;
  float* qs = sh_smem;                        // [32][hd + 4]
  float* ks = qs + kShRows * ldk;             // [64][hd + 4]
  float* vs = ks + kShBlk * ldk;              // [64][hd]
  float* ps = vs + kShBlk * hd;               // [32][65]
  const int kvh = blockIdx.y, g = a.nh / a.nkv, tid = threadIdx.x;
  const int tx = tid & 15, ty = tid >> 4;
  dependent_begin();

  // ---- this block's rows and keys
  int seq, row0, n_rows, row_base = -1, tok0 = 0, key0, key_end, piece;
  if ((int)blockIdx.x < a.n_pre) {
    const SharedPrefixItem it = a.pre[blockIdx.x];
    seq = it.seq; row0 = it.row0; n_rows = it.n_rows; row_base = it.row_base;
    key0 = it.blk0 * kShBlk; key_end = it.blk1 * kShBlk; piece = it.piece;
  } else {
    const int x = blockIdx.x - a.n_pre, split = x % a.own_splits;
    const SharedOwnItem it = a.own[x / a.own_splits];
    seq = it.seq; row0 = it.row0; n_rows = it.n_rows; tok0 = it.tok0;
    const int prefix = it.prefix;
    const int end = shared_own_end(a, prefix, a.tok_pos[tok0 + (row0 + n_rows - 1) / g]);
    const int blocks = (end - prefix + kShBlk - 1) / kShBlk;
    key0 = prefix + (int)((long long)blocks * split / a.own_splits) * kShBlk;
    key_end = min(end, prefix + (int)((long long)blocks * (split + 1) / a.own_splits) * kShBlk);
    piece = a.max_pieces - a.own_splits + split;
  }
  auto token = [&](int r) {
    return row_base >= 0 ? a.rows[row_base + r / g] : tok0 + r / g;
  };
  for (int i = tid; i < kShRows * hd; i += kShThreads) {
    const int r = i / hd, d = i - r * hd;
    qs[r * ldk + d] = r < n_rows
        ? to_float(static_cast<const T*>(a.q)[(size_t)token(row0 + r) * a.ldq +
                                              (size_t)(kvh * g + (row0 + r) % g) * hd + d])
        : 0.f;
  }
  int pos[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = ty + 16 * i;
    pos[i] = r < n_rows ? (row_base >= 0 ? key_end - 1 : a.tok_pos[token(row0 + r)]) : -1;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[2][2][4] = {};
  for (int k0 = key0; k0 < key_end; k0 += kShBlk) {
    __syncthreads();                          // the last step's readers are done (and Q is there)
    const size_t at = ((size_t)shared_block(a, seq, k0 / kShBlk) * a.nkv + kvh) * kShBlk * hd;
    const int n = min(kShBlk, key_end - k0);
    for (int i = tid; i < kShBlk * hd; i += kShThreads) {
      const int r = i / hd, d = i - r * hd;   // (nothing past the last key is looked at)
      ks[r * ldk + d] = r < n ? to_float(static_cast<const T*>(a.kc)[at + i]) : 0.f;
      vs[i] = r < n ? to_float(static_cast<const T*>(a.vc)[at + i]) : 0.f;
    }
    __syncthreads();
    float s[2][4] = {};
    for (int d = 0; d < hd; d += 4) {
      float4 kk[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) kk[c] = *reinterpret_cast<const float4*>(ks + (tx + 16 * c) * ldk + d);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 qq = *reinterpret_cast<const float4*>(qs + (ty + 16 * i) * ldk + d);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          s[i][c] = fmaf(qq.x, kk[c].x, fmaf(qq.y, kk[c].y, fmaf(qq.z, kk[c].z, fmaf(qq.w, kk[c].w, s[i][c]))));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int key = k0 + tx + 16 * c;
        s[i][c] = key < key_end && key <= pos[i] ? s[i][c] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[i][c]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float m_new = fmaxf(m[i], mx);
      const float alpha = m[i] == -INFINITY ? 0.f : exp2f(m[i] - m_new);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = s[i][c] == -INFINITY ? 0.f : exp2f(s[i][c] - m_new);
        sum += p;
        ps[(ty + 16 * i) * 65 + tx + 16 * c] = p;
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[i] = l[i] * alpha + sum;
      m[i] = m_new;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][c][e] *= alpha;
    }
    __syncwarp();                             // a row's probabilities are its own half warp's
    for (int k = 0; k < n; ++k) {
      const float p0 = ps[ty * 65 + k], p1 = ps[(ty + 16) * 65 + k];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = tx * 4 + 64 * c;
        if (d < hd) {
          const float4 v = *reinterpret_cast<const float4*>(vs + k * hd + d);
          o[0][c][0] = fmaf(p0, v.x, o[0][c][0]); o[0][c][1] = fmaf(p0, v.y, o[0][c][1]);
          o[0][c][2] = fmaf(p0, v.z, o[0][c][2]); o[0][c][3] = fmaf(p0, v.w, o[0][c][3]);
          o[1][c][0] = fmaf(p1, v.x, o[1][c][0]); o[1][c][1] = fmaf(p1, v.y, o[1][c][1]);
          o[1][c][2] = fmaf(p1, v.z, o[1][c][2]); o[1][c][3] = fmaf(p1, v.w, o[1][c][3]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = ty + 16 * i;
    if (r >= n_rows) continue;
    const size_t row = (size_t)piece * a.T * a.nh + (size_t)token(row0 + r) * a.nh + kvh * g + (row0 + r) % g;
    if (tx == 0) a.part_ml[row] = make_float2(m[i], l[i]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int d = tx * 4 + 64 * c;
      if (d < hd)
        *reinterpret_cast<float4*>(a.part_o + row * hd + d) =
            make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kShThreads) shared_join_kernel(const SharedArgs a) {
  dependent_begin();
  const int row = blockIdx.x * (kShThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.T * a.nh) return;
  const int t = row / a.nh, h = row - t * a.nh, pre = a.tok_pieces[t];
  const size_t stride = (size_t)a.T * a.nh;
  const int own0 = a.max_pieces - a.own_splits, n = pre + a.own_splits;
  auto at = [&](int i) { return (i < pre ? i : own0 + i - pre) * stride + row; };
  float mx = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
  for (int i = lane; i < n; i += 32) mx = fmaxf(mx, a.part_ml[at(i)].x);
  mx = warp_max(mx);
  if (mx == -INFINITY) mx = 0.f;              // (a row that sees nothing gives zeros)
  float den = 0.f;
  float acc[4] = {};
  for (int i = 0; i < n; ++i) {
    const float2 ml = a.part_ml[at(i)];
    if (ml.x == -INFINITY) continue;          // a piece without keys
    const float w = exp2f(ml.x - mx);
    den = fmaf(w, ml.y, den);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < a.hd) acc[c] = fmaf(w, a.part_o[at(i) * a.hd + lane + 32 * c], acc[c]);
  }
  if (a.sink) den += exp2f(a.sink[h] * 1.4426950408889634f - mx);
  const float inv = den > 0.f ? 1.0f / den : 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < a.hd)
      static_cast<T*>(a.out)[(size_t)t * a.ldo + (size_t)h * a.hd + lane + 32 * c] = from_float<T>(acc[c] * inv);
}

int launch_shared_bf16(const SharedArgs& a, cudaStream_t st);        // attn_shared_tc.cu

template <typename T>
static int launch_join(const SharedArgs& a, cudaStream_t st) {
  launch_dependent(shared_join_kernel<T>, dim3((a.T * a.nh + 7) / 8), dim3(kShThreads), 0, st, a);
  return launch_status();
}

static int launch_shared_f32(const SharedArgs& a, cudaStream_t st) {
  const size_t smem = ((size_t)(kShRows + kShBlk) * (a.hd + 4) + (size_t)kShBlk * a.hd + kShRows * 65) * 4;
  cudaError_t e = cudaFuncSetAttribute(shared_pieces_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem);
  if (e != cudaSuccess) return (int)e;
  launch_dependent(shared_pieces_kernel<float>, dim3(a.n_pre + a.n_own * a.own_splits, a.nkv), dim3(kShThreads),
                   smem, st, a);
  return launch_join<float>(a, st);
}

}  // namespace cretif

using namespace cretif;

extern "C" int cretif_attn_shared(const void* q, int ldq, int dt, void* out, int ldo, const void* kc,
                                  const void* vc, long long n_blocks, const int* table,
                                  int table_stride, int n_slots, const int* tok_pos,
                                  const int* seq_slot, const int* plan, int n_pre, int n_own,
                                  int own_rows, int own_splits, int max_pieces, int n_rows, int T, int nh,
                                  int nkv, int hd, int bt, float scale, const float* sink,
                                  float* part_o, float* part_ml, unsigned int* fault, void* stream) {
  if (T <= 0) return kOk;
  if (nh <= 0 || nkv <= 0 || nh % nkv || hd % 16 || hd < 16 || hd > 128 || bt != kShBlk || own_rows <= 0 ||
      n_pre < 0 || n_own <= 0 || own_splits <= 0 || max_pieces < own_splits || n_rows < 0 ||
      nkv > 65535 || (long long)T * nh > (1LL << 30) || n_blocks <= 0 || !(scale > 0.f) ||
      (long long)n_pre + (long long)n_own * own_splits > 0x7fffffffLL)
    return kBadArgument;
  if (dt != kF32 && dt != kBF16) return kBadDType;
  if ((((uintptr_t)kc | (uintptr_t)vc | (uintptr_t)plan | (uintptr_t)part_o) & 15) || ((uintptr_t)part_ml & 7))
    return kMisaligned;
  SharedArgs a{};
  a.q = q; a.kc = kc; a.vc = vc; a.out = out; a.ldq = ldq; a.ldo = ldo; a.n_blocks = n_blocks;
  a.table = table; a.table_stride = table_stride; a.n_slots = n_slots;
  a.tok_pos = tok_pos; a.seq_slot = seq_slot;
  a.pre = reinterpret_cast<const SharedPrefixItem*>(plan);
  a.own = reinterpret_cast<const SharedOwnItem*>(plan + 8 * (size_t)n_pre);
  a.rows = plan + 8 * ((size_t)n_pre + n_own);
  a.tok_pieces = a.rows + n_rows;
  a.n_pre = n_pre; a.n_own = n_own; a.own_rows = own_rows; a.own_splits = own_splits; a.max_pieces = max_pieces; a.T = T;
  a.nh = nh; a.nkv = nkv; a.hd = hd; a.scale_log2 = scale * 1.4426950408889634f; a.sink = sink;
  a.part_o = part_o; a.part_ml = reinterpret_cast<float2*>(part_ml); a.fault = fault;
  if (dt == kF32) return launch_shared_f32(a, (cudaStream_t)stream);
  const int e = launch_shared_bf16(a, (cudaStream_t)stream);
  return e || own_splits == 1 ? e : launch_join<__nv_bfloat16>(a, (cudaStream_t)stream);
}
