// Attention of few new tokens a sequence for a batch whose sequences share prefixes: the keys of a
// group's prefix are read once for all its members, each sequence's own keys once for its tokens
// (attn_shared.h has the formula).  The reference decodes one sequence at a time and has nothing of
// the kind (its attention walks one cache, src/attention.cu:410-494).
//
// Here the 32-bit kernel and the joining of pieces; the bfloat16 kernels are in attn_shared_tc.cu.
#include "api.h"
#include "attn_shared.h"

namespace cretif {

constexpr int kShRows = 32, kShThreads = 256;

// 32-bit pieces: a block of 256 threads per (item, key/value head), up to 32 rows and 64 keys a step.
// A warp has rows w, w + 8, w + 16, w + 24, those that there are: a lane two keys of their scores and VD
// channels of their outputs, so a softmax is the warp's own.  The next step's keys and values are on
// their way in registers.  (Eight answers at 1,984 tokens: 13.5 us; 16 x 16 threads on 32 rows whatever
// there were took 25, most of it on the own keys' three rows.  One CTA an SM is all that fits: said so, the
// compiler takes 235 registers instead of 171, and 0.4 us less.)
template <int VD>
__global__ void __launch_bounds__(kShThreads, 1)
shared_pieces_kernel(const SharedArgs a) {
  extern __shared__ __align__(16) float sh_smem[];
  const int hd = a.hd, ldk = hd + 4, quads = hd >> 2;
  float* qs = sh_smem;                        // [32][hd + 4]
  float* ks = qs + kShRows * ldk;             // [64][hd + 4]
  float* vs = ks + kShBlk * ldk;              // [64][hd]
  float* ps = vs + kShBlk * hd;               // [32][64]
  __shared__ int toks[kShRows], pieces[kShRows];   // a row's token, and this piece of it among all
  const int kvh = blockIdx.y, g = a.nh / a.nkv, tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31;
  constexpr int kRows = kShRows / 8;          // of a warp
  dependent_begin();

  // ---- this block's rows and keys
  int seq, row0, n_rows, row_base = -1, tok0 = 0, at0 = 0, a_token = 0, key0, key_end;
  if ((int)blockIdx.x < a.n_pre) {
    const SharedPrefixItem it = a.pre[blockIdx.x];
    seq = it.seq; row0 = it.row0; n_rows = it.n_rows; row_base = it.row_base;
    key0 = it.blk0 * kShBlk; key_end = it.blk1 * kShBlk; at0 = it.piece;
  } else {
    const int x = blockIdx.x - a.n_pre, split = x % a.own_splits;
    const SharedOwnItem it = a.own[x / a.own_splits];
    seq = it.seq; row0 = it.row0; n_rows = it.n_rows; tok0 = it.tok0;
    at0 = it.first + it.pieces + split; a_token = it.pieces + a.own_splits;
    const int prefix = it.prefix;
    const int end = shared_own_end(a, it, a.tok_pos[tok0 + (row0 + n_rows - 1) / g]);
    const int blocks = (end - prefix + kShBlk - 1) / kShBlk;
    key0 = prefix + (int)((long long)blocks * split / a.own_splits) * kShBlk;
    key_end = min(end, prefix + (int)((long long)blocks * (split + 1) / a.own_splits) * kShBlk);
  }
  // a thread's share of a step's tile: keys tid / quads, + step, ...; at most 8 of four channels
  const int slot = a.seq_slot[seq];
  const int k_of = tid / quads, ch = (tid - k_of * quads) * 4, k_step = kShThreads / quads;
  const bool loads = k_of < k_step;           // (quads need not divide the threads)
  float4 kr[8], vr[8];
  auto fetch = [&](int k0) {
    const size_t at = ((size_t)shared_block_of(a, slot, k0 / kShBlk) * a.nkv + kvh) * kShBlk * hd;
    const int n = min(kShBlk, key_end - k0);  // (nothing past the last key is looked at)
    const float *kp = static_cast<const float*>(a.kc) + at + ch, *vp = static_cast<const float*>(a.vc) + at + ch;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k_of + i * k_step;
      kr[i] = vr[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (loads && k < n) {
        kr[i] = *reinterpret_cast<const float4*>(kp + (size_t)k * hd);
        vr[i] = *reinterpret_cast<const float4*>(vp + (size_t)k * hd);
      }
    }
  };
  if (key0 < key_end) fetch(key0);
  if (tid < kShRows) {
    const int r = row0 + tid;
    toks[tid] = tid >= n_rows ? -1 : row_base >= 0 ? a.rows[row_base + r / g] : tok0 + r / g;
    pieces[tid] = at0 + (tid >= n_rows ? 0 : row_base >= 0 ? a.rows_first[row_base + r / g] : r / g * a_token);
  }
  __syncthreads();
  for (int i = tid; i < kShRows * quads; i += kShThreads) {
    const int r = i / quads, d = (i - r * quads) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < n_rows) {
      const float* src = static_cast<const float*>(a.q) + (size_t)toks[r] * a.ldq + (size_t)(kvh * g + (row0 + r) % g) * hd + d;
      v = make_float4(src[0], src[1], src[2], src[3]);     // (queries may begin anywhere)
    }
    *reinterpret_cast<float4*>(qs + r * ldk + d) = v;
  }
  const int mine = warp < n_rows ? (n_rows - warp + 7) >> 3 : 0;      // rows of this warp
  int pos[kRows];
  float m[kRows], l[kRows], o[kRows][VD];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    pos[i] = i < mine ? (row_base >= 0 ? key_end - 1 : a.tok_pos[toks[warp + 8 * i]]) : -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < VD; ++e) o[i][e] = 0.f;
  }
  const int d0 = lane * VD;                   // this lane's channels
  const bool has_d = d0 < hd;
  for (int k0 = key0; k0 < key_end; k0 += kShBlk) {
    __syncthreads();                          // the last step's readers are done (and Q is there)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k_of + i * k_step;
      if (loads && k < kShBlk) {
        *reinterpret_cast<float4*>(ks + k * ldk + ch) = kr[i];
        *reinterpret_cast<float4*>(vs + k * hd + ch) = vr[i];
      }
    }
    __syncthreads();
    if (k0 + kShBlk < key_end) fetch(k0 + kShBlk);
    // (the number of rows is a constant inside: a branch a row kept the loads from overlapping)
    auto step = [&](auto constant) {
      constexpr int R = decltype(constant)::value;
      float s[R][2][2] = {};
#pragma unroll 4
      for (int d = 0; d < hd; d += 4) {
        const float4 ka = *reinterpret_cast<const float4*>(ks + lane * ldk + d);
        const float4 kb = *reinterpret_cast<const float4*>(ks + (lane + 32) * ldk + d);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float4 qq = *reinterpret_cast<const float4*>(qs + (warp + 8 * i) * ldk + d);
          s[i][0][0] = fmaf(qq.x, ka.x, fmaf(qq.y, ka.y, s[i][0][0]));
          s[i][0][1] = fmaf(qq.z, ka.z, fmaf(qq.w, ka.w, s[i][0][1]));
          s[i][1][0] = fmaf(qq.x, kb.x, fmaf(qq.y, kb.y, s[i][1][0]));
          s[i][1][1] = fmaf(qq.z, kb.z, fmaf(qq.w, kb.w, s[i][1][1]));
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float t2[2], mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int key = k0 + lane + 32 * c;
          t2[c] = key < key_end && key <= pos[i] ? (s[i][c][0] + s[i][c][1]) * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, t2[c]);
        }
        mx = warp_max(mx);
        const float m_new = fmaxf(m[i], mx);
        const float alpha = m[i] == -INFINITY ? 0.f : exp2f(m[i] - m_new);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float p = t2[c] == -INFINITY ? 0.f : exp2f(t2[c] - m_new);
          sum += p;
          ps[(warp + 8 * i) * kShBlk + lane + 32 * c] = p;
        }
        l[i] = l[i] * alpha + warp_sum(sum);
        m[i] = m_new;
#pragma unroll
        for (int e = 0; e < VD; ++e) o[i][e] *= alpha;
      }
      __syncwarp();
      if (has_d) {
        float part[R][VD] = {};               // of the even pairs of keys
#pragma unroll 4
        for (int k = 0; k < kShBlk; k += 4) { // (keys past the last have probability and value zero)
          float v[4][VD];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if constexpr (VD == 2) {
              const float2 f = *reinterpret_cast<const float2*>(vs + (k + x) * hd + d0);
              v[x][0] = f.x; v[x][1] = f.y;
            } else {
              const float4 f = *reinterpret_cast<const float4*>(vs + (k + x) * hd + d0);
              v[x][0] = f.x; v[x][1] = f.y; v[x][2] = f.z; v[x][3] = f.w;
            }
          }
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float4 p = *reinterpret_cast<const float4*>(ps + (warp + 8 * i) * kShBlk + k);
#pragma unroll
            for (int e = 0; e < VD; ++e) {
              part[i][e] = fmaf(p.x, v[0][e], fmaf(p.y, v[1][e], part[i][e]));
              o[i][e] = fmaf(p.z, v[2][e], fmaf(p.w, v[3][e], o[i][e]));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < VD; ++e) o[i][e] += part[i][e];
      }
    };
    if (mine == 1) step(std::integral_constant<int, 1>{});
    else if (mine == 2) step(std::integral_constant<int, 2>{});
    else if (mine == 3) step(std::integral_constant<int, 3>{});
    else if (mine == 4) step(std::integral_constant<int, 4>{});
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (i < mine) {
      const int r = warp + 8 * i;
      const size_t row = (size_t)pieces[r] * a.nh + kvh * g + (row0 + r) % g;
      if (lane == 0) a.part_ml[row] = make_float2(m[i], l[i]);
      if (has_d) {
        float* to = a.part_o + row * hd + d0;
        if constexpr (VD == 2) *reinterpret_cast<float2*>(to) = make_float2(o[i][0], o[i][1]);
        else *reinterpret_cast<float4*>(to) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
      }
    }
}

// A warp joins the pieces of a row: four lanes' channels of a piece at once, so that 32 / (hd / 4) pieces
// are read side by side, and eight of those at a time; the parts meet by shuffles.
template <typename T>
__global__ void __launch_bounds__(kShThreads) shared_join_kernel(const SharedArgs a) {
  dependent_begin();
  const int row = blockIdx.x * (kShThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.T * a.nh) return;
  const int t = row / a.nh, h = row - t * a.nh, first = a.first[t], n = a.first[t + 1] - first;
  auto at = [&](int i) { return ((size_t)first + i) * a.nh + h; };
  // `side` groups of `wide` lanes (a power of two, at least hd / 4) take the pieces in turns
  int wide = 4;
  while (wide < a.hd >> 2) wide <<= 1;
  const int side = 32 / wide, mine = lane / wide, ch = (lane & (wide - 1)) * 4;
  const bool live = ch < a.hd;
  const float sink = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
  float ref = -INFINITY, den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kAtOnce = 8;
  for (int i0 = mine; i0 < n; i0 += side * kAtOnce) {
    float2 ml[kAtOnce];
    float4 x[kAtOnce];
    float top = ref;
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      const int i = i0 + e * side;
      ml[e] = i < n ? a.part_ml[at(i)] : make_float2(-INFINITY, 0.f);
      x[e] = i < n && live ? *reinterpret_cast<const float4*>(a.part_o + at(i) * a.hd + ch) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) top = fmaxf(top, ml[e].x);
    if (top == -INFINITY) continue;           // pieces without keys
    const float keep = ref == -INFINITY ? 0.f : exp2f(ref - top);
    den *= keep; acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      const float w = ml[e].x == -INFINITY ? 0.f : exp2f(ml[e].x - top);
      den = fmaf(w, ml[e].y, den);
      acc.x = fmaf(w, x[e].x, acc.x); acc.y = fmaf(w, x[e].y, acc.y);
      acc.z = fmaf(w, x[e].z, acc.z); acc.w = fmaf(w, x[e].w, acc.w);
    }
    ref = top;
  }
  float top = fmaxf(ref, sink);
  for (int o = wide; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float w = ref == -INFINITY ? 0.f : exp2f(ref - top);
  den *= w; acc.x *= w; acc.y *= w; acc.z *= w; acc.w *= w;
  for (int o = wide; o < 32; o <<= 1) {
    den += __shfl_xor_sync(0xffffffffu, den, o);
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
  }
  if (a.sink) den += sink == top ? 1.0f : exp2f(sink - top);
  if (mine == 0 && live) {
    const float inv = den > 0.f ? 1.0f / den : 0.f;       // (a row that sees nothing gives zeros)
    T* dst = static_cast<T*>(a.out) + (size_t)t * a.ldo + (size_t)h * a.hd + ch;
    dst[0] = from_float<T>(acc.x * inv); dst[1] = from_float<T>(acc.y * inv);
    dst[2] = from_float<T>(acc.z * inv); dst[3] = from_float<T>(acc.w * inv);
  }
}

int launch_shared_bf16(const SharedArgs& a, cudaStream_t st);        // attn_shared_tc.cu

template <typename T>
static int launch_join(const SharedArgs& a, cudaStream_t st) {
  launch_dependent(shared_join_kernel<T>, dim3((a.T * a.nh + 7) / 8), dim3(kShThreads), 0, st, a);
  return launch_status();
}

template <int VD>
static int launch_shared_f32(const SharedArgs& a, cudaStream_t st) {
  auto bytes = [](int hd) { return ((size_t)(kShRows + kShBlk) * (hd + 4) + (size_t)kShBlk * hd + kShRows * kShBlk) * 4; };
  const size_t smem = bytes(a.hd);
  // (the limit of the largest heads for all: another thread's call may be asking for its own)
  const cudaError_t e = cudaFuncSetAttribute(shared_pieces_kernel<VD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)bytes(32 * VD));
  if (e != cudaSuccess) return (int)e;
  launch_dependent(shared_pieces_kernel<VD>, dim3(a.n_pre + a.n_own * a.own_splits, a.nkv), dim3(kShThreads), smem, st,
                   a);
  return launch_join<float>(a, st);
}

}  // namespace cretif

using namespace cretif;

extern "C" int cretif_attn_shared(const void* q, long long ldq, int dt, void* out, long long ldo, const void* kc,
                                  const void* vc, long long n_blocks, const int* table,
                                  long long table_stride, int table_width, int n_slots, const int* tok_pos,
                                  const int* seq_slot, const int* plan, int n_pre, int n_own,
                                  int own_rows, int own_splits, int n_rows, int T, int nh,
                                  int nkv, int hd, int bt, float scale, const float* sink,
                                  float* part_o, float* part_ml, unsigned int* fault, void* stream) {
  if (T <= 0) return kOk;
  if (nh <= 0 || nkv <= 0 || nh % nkv || hd % 16 || hd < 16 || hd > 128 || bt != kShBlk || own_rows <= 0 ||
      n_pre < 0 || n_own <= 0 || own_splits <= 0 || n_rows < 0 ||
      nkv > 65535 || (long long)T * nh > (1LL << 30) || n_blocks <= 0 || !(scale > 0.f) ||
      (long long)n_pre + (long long)n_own * own_splits > 0x7fffffffLL)
    return kBadArgument;
  if (dt != kF32 && dt != kBF16) return kBadDType;
  if ((((uintptr_t)kc | (uintptr_t)vc | (uintptr_t)plan | (uintptr_t)part_o) & 15) || ((uintptr_t)part_ml & 7))
    return kMisaligned;
  if (!part_o && (dt == kF32 || n_pre > 0 || own_splits > 1)) return kBadArgument;
  SharedArgs a{};
  a.q = q; a.kc = kc; a.vc = vc; a.out = out; a.ldq = ldq; a.ldo = ldo; a.n_blocks = n_blocks;
  a.table = table; a.table_stride = table_stride; a.table_width = table_width; a.n_slots = n_slots;
  a.tok_pos = tok_pos; a.seq_slot = seq_slot;
  a.pre = reinterpret_cast<const SharedPrefixItem*>(plan);
  a.own = reinterpret_cast<const SharedOwnItem*>(plan + 8 * (size_t)n_pre);
  a.rows = plan + 8 * ((size_t)n_pre + n_own);
  a.rows_first = a.rows + n_rows;
  a.first = a.rows_first + n_rows;
  a.n_pre = n_pre; a.n_own = n_own; a.own_rows = own_rows; a.own_splits = own_splits; a.T = T;
  a.nh = nh; a.nkv = nkv; a.hd = hd; a.scale_log2 = scale * 1.4426950408889634f; a.sink = sink;
  a.part_o = part_o; a.part_ml = reinterpret_cast<float2*>(part_ml); a.fault = fault;
  if (dt == kF32)
    return hd <= 64 ? launch_shared_f32<2>(a, (cudaStream_t)stream) : launch_shared_f32<4>(a, (cudaStream_t)stream);
  const int e = launch_shared_bf16(a, (cudaStream_t)stream);
  return e || own_splits == 1 ? e : launch_join<__nv_bfloat16>(a, (cudaStream_t)stream);
}
