// The bfloat16 kernels of the attention over shared prefixes (attn_shared.h has the formula).
//
// shared_prefix_tc: the prefix's keys against all rows of a group on the tcgen05 tensor cores.
// shared_own_mma: a sequence's own keys against its few rows, and the joining of a row's pieces.
//
// What is held in fewer than 32 bits: a probability is rounded to bfloat16 where it becomes an operand of P V, as in the
// framework's other attention kernels, because the tensor cores take a 32-bit operand at an eighth of the rate and in
// twice the shared memory.  It is off by half a step, 2^-9 at most of each term p |v| of an output; the sums l of
// the same probabilities are 32-bit and not rounded.  (Error against 64 bits, as a share of the largest output: 2.0 to
// 2.35e-3 with the output's own rounding, which alone is 1.7e-3.)  Exponentials are ex2.approx.ftz, off by 2^-22.
#include <cuda.h>

#include "api.h"
#include "attn_decode_mma.cuh"
#include "attn_shared.h"
#include "tc_common.cuh"

namespace cretif {

// ---------------------------------------------------------------------------------------
// Prefix: a CTA takes up to 128 rows (tokens x heads of a key/value head) and a range of the
// prefix's blocks, 64 keys a step; two CTAs fit an SM and fill each other's gaps.
//   warps 0-3  softmax: a thread owns a row (a lane of tensor memory);
//   warp 4     TMA producer: K and V tiles straight out of the block cache;
//   warp 5     one thread issues S = Q K^T and O += P V.
// Tensor memory: two score tiles of 64 columns, O, and for head sizes up to 64 the queries (as A
// operand in shared memory, read again for every 64 keys, they took the memory's bandwidth: a product
// of 16 channels reads 6 KB instead of 2).  A row's thread writes its probabilities as
// bfloat16 over the scores it has read, from where the product P V takes them as its A operand; it
// adds into O itself, since a row's reference for the exponentials moves only when a score exceeds
// it by 2^8 (then the row's thread waits for the product before and scales O).
// The tiles come in pairs: {K_0, K_1}, then {V_j, K_{j+2}}: one barrier to wait for a step, and one
// commit a step, behind P V of step j and the scores of step j + 2, which tells the softmax threads
// that the scores are there and the producer that the pair may be replaced.
// (An issuing thread pays 200 to 250 cycles for a wait, even one that is over, so the step's two are
// polled together.  One thread for the scores and one for P V, which then wait for each other, was
// slower: 135 us against 115 with 64 answers with drafts at 30,016.)
//
// Few rows (FOLD = 2 or 4: up to 64 or 32): the rows lie in tensor memory FOLD times, and each copy
// takes its share of every step's keys (zeros stand for the others), so that all four warps work;
// the copies are joined at the end.
constexpr int kSpThreads = 192, kSpRows = 128, kSpTile = kShBlk * 128;   // a 64 x 64 tile's bytes
constexpr int kSpDone = 8;                // commit c arrives on barrier c % 8 (see the producer)

struct SpSmem {
  int q, ring, pairs, bars, xch, total;
  __host__ __device__ explicit SpSmem(int n_sub) {
    pairs = n_sub == 1 ? 6 : 2;
    q = 0;
    ring = n_sub == 1 ? 0 : n_sub * kSpRows * 128;
    bars = ring + pairs * 2 * n_sub * kSpTile;
    xch = bars + (kSpDone + 6 + 4) * 8 + 16;
    total = xch + kSpRows * 16 + 1024;
  }
};

__device__ __forceinline__ float sp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sp_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// MN-major operand (V): a key is a row of 128 bytes, 64-wide column groups are a tile apart.
__device__ __forceinline__ uint64_t sp_desc_v(const void* tile) {
  uint64_t d = 0;
  d |= (uint64_t)((tc::smem_u32(tile) & 0x3FFFFu) >> 4);
  d |= (uint64_t)(kSpTile >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Wait for two barriers at once: the polls of both are in flight together.
__device__ __forceinline__ bool sp_wait_both(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, volatile int* abort) {
  const uint32_t aa = tc::smem_u32(a), ab = tc::smem_u32(b);
  for (unsigned spin = 0; spin < tc::kSpinLimit; ++spin) {
    uint32_t oa, ob;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%2], %3;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%4], %5;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "selp.u32 %1, 1, 0, q;\n\t}"
        : "=r"(oa), "=r"(ob)
        : "r"(aa), "r"(pa), "r"(ab), "r"(pb)
        : "memory");
    if (oa & ob) return true;
    if (!oa) { if (!tc::mbar_wait(a, pa, abort)) return false; }
    else if (!tc::mbar_wait(b, pb, abort)) return false;
  }
  *abort = 1;
  return false;
}

template <int FOLD>
__device__ __forceinline__ void sp_softmax(uint32_t lane_addr, int hd, int n_steps, int copy, float scale_log2,
                                           uint64_t* done, uint64_t* p_full, volatile int* abort, float& m_out,
                                           float& l_out) {
  constexpr int NK = kShBlk / FOLD;       // this thread's keys of a step
  constexpr uint32_t kColO = 128;
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < n_steps; ++j) {
    tc::mbar_wait(&done[j % kSpDone], (uint32_t)((j / kSpDone) & 1), abort);
    tc::tc_fence_after();
    const uint32_t s_addr = lane_addr + (uint32_t)(j & 1) * 64;
    uint32_t r[NK];
    if constexpr (FOLD == 1) {
      uint32_t (&lo)[32] = *reinterpret_cast<uint32_t (*)[32]>(&r[0]);
      uint32_t (&hi)[32] = *reinterpret_cast<uint32_t (*)[32]>(&r[32]);
      tc::tmem_load_32(s_addr, lo);
      tc::tmem_load_32(s_addr + 32, hi);
    } else if constexpr (FOLD == 2) {
      tc::tmem_load_32(s_addr + copy * 32, r);
    } else {
      tc::tmem_load_16(s_addr + copy * 16, r);
    }
    tc::tmem_load_wait();
    float mx[4] = {__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2]), __uint_as_float(r[3])};
#pragma unroll
    for (int c = 4; c + 3 < NK; c += 4) {
      const int i = (c >> 2) & 1;
      mx[2 * i] = sp_max3(mx[2 * i], __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
      mx[2 * i + 1] = sp_max3(mx[2 * i + 1], __uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
    }
    // (the scale is positive: the largest raw score is the largest scaled one)
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2;
    if (j == 0) {
      m = top;
    } else if (__any_sync(0xffffffffu, top > m + 8.0f)) {
      const float m_new = fmaxf(m, top);
      const float alpha = m == -INFINITY ? 0.f : sp_exp2(m - m_new);
      // O is scaled in place, once the product of the step before has gone into it
      tc::mbar_wait(&done[(j + 1) % kSpDone], (uint32_t)(((j + 1) / kSpDone) & 1), abort);
      tc::tc_fence_after();
      for (int c0 = 0; c0 < hd; c0 += 32) {
        uint32_t o[32];
        tc::tmem_load_32(lane_addr + kColO + (uint32_t)c0, o);
        tc::tmem_load_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
        tc::tmem_store_32(lane_addr + kColO + (uint32_t)c0, o);
      }
      l *= alpha;
      m = m_new;
    }
    const float neg_m = m == -INFINITY ? 0.f : -m;
    const float2 scale2 = make_float2(scale_log2, scale_log2), neg2 = make_float2(neg_m, neg_m);
    float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
    uint32_t packed[NK / 2];
#pragma unroll
    for (int c = 0; c < NK; c += 2) {
      const float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, neg2);
      const float2 p = make_float2(sp_exp2(x.x), sp_exp2(x.y));
      sum[(c >> 1) & 1] = __fadd2_rn(sum[(c >> 1) & 1], p);
      packed[c >> 1] = pack_bf16(p.x, p.y);
    }
    if constexpr (FOLD == 1) {
      tc::tmem_store_32(s_addr, packed);
    } else {
      uint32_t all[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) all[e] = e / (NK / 2) == copy ? packed[e % (NK / 2)] : 0u;
      tc::tmem_store_32(s_addr, all);
    }
    const float2 s2 = __fadd2_rn(sum[0], sum[1]);
    l += s2.x + s2.y;
    tc::tmem_store_wait();                 // P (and O) are in tensor memory, S has been read
    tc::tc_fence_before();
    tc::mbar_arrive(&p_full[j & 1]);
  }
  m_out = m;
  l_out = l;
}

__global__ void __launch_bounds__(kSpThreads, 2)
shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ SharedArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int hd = a.hd, n_sub = (hd + 63) >> 6;
  const SpSmem L(n_sub);
  uint64_t* done = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* full = done + kSpDone;
  uint64_t* p_full = full + 6;
  uint64_t* q_full = p_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* xch = reinterpret_cast<float2*>(smem + L.xch);  // [128] references and sums, then the rows' places
  long long* place = reinterpret_cast<long long*>(xch + kSpRows);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const SharedPrefixItem it = a.pre[blockIdx.x];
  const int kvh = blockIdx.y, g = a.nh / a.nkv;
  const int n = it.blk1 - it.blk0;
  const int fold = it.n_rows <= 32 ? 4 : it.n_rows <= 64 ? 2 : 1;
  const int span = kSpRows / fold;                       // lanes of a copy
  // warps whose lanes hold rows: the others neither wait nor arrive
  const int warps_a_copy = (it.n_rows + 31) >> 5;
  constexpr uint32_t kColO = 128, kColQ = 192;            // (kColQ: up to 64 channels)

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSpDone; ++i) tc::mbar_init(&done[i], 1);
    for (int i = 0; i < L.pairs; ++i) tc::mbar_init(&full[i], 1);
    tc::mbar_init(&p_full[0], 32 * warps_a_copy * fold);
    tc::mbar_init(&p_full[1], 32 * warps_a_copy * fold);
    tc::mbar_init(q_full, kSpRows);
    *abort = 0;
    tc::fence_barrier_init();
    tc::tma_prefetch_descriptor(&map_k);
    tc::tma_prefetch_descriptor(&map_v);
  }
  if (warp == 5) {
    tc::tmem_alloc(tmem_slot, 256);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Everything before this call's first kernel is done and visible behind the wait; the kernel
  // behind this one may start only then, so that it may read the queries without a wait of its own.
  dependent_wait();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 4) {
    // Block ids come 32 at a time, a lane each, and a window ahead of their use: read one by one they
    // cost two dependent loads a step (64 answers with drafts at 30,016: 123 us with, 114.5 without).
    auto window = [&](int w) { return 32 * w + lane < n ? shared_block(a, it.seq, it.blk0 + 32 * w + lane) : 0; };
    int here = window(0), next = window(1), s = 0;        // windows of V's block, and the one behind it
    for (int p = 0; p <= n; ++p) {
      const int jv = p - 1, jk = p + 1;                   // pair 0: K_0 and K_1; pair p: V_{p-1}, K_{p+1}
      if (jv > 0 && (jv & 31) == 0) {
        here = next;
        next = window((jv >> 5) + 1);
      }
      const int from = (jk >> 5) > ((jv > 0 ? jv : 0) >> 5) ? next : here;
      const int blk_k = __shfl_sync(0xffffffffu, from, jk & 31);
      const int blk_first = __shfl_sync(0xffffffffu, here, p == 0 ? 0 : jv & 31);
      bool go = true;
      if (lane == 0 && p >= L.pairs) {
        // pair p - L.pairs has been read when commit p - L.pairs + 1 arrives (the one 8 commits later
        // cannot arrive before this pair is loaded)
        const int c = p - L.pairs + 1;
        go = tc::mbar_wait(&done[c % kSpDone], (uint32_t)((c / kSpDone) & 1), abort);
      }
      if (!__shfl_sync(0xffffffffu, go, 0)) break;
      if (lane == 0) {
        const bool second = jk < n;
        tc::mbar_expect_tx(&full[s], (uint32_t)((second ? 2 : 1) * n_sub * kSpTile));
        unsigned char* slot = smem + L.ring + s * 2 * n_sub * kSpTile;
        for (int sub = 0; sub < n_sub; ++sub) {
          tc::tma_load_2d(slot + sub * kSpTile, p == 0 ? &map_k : &map_v, 64 * sub,
                          (blk_first * a.nkv + kvh) * kShBlk, &full[s]);
          if (second)
            tc::tma_load_2d(slot + (n_sub + sub) * kSpTile, &map_k, 64 * sub, (blk_k * a.nkv + kvh) * kShBlk, &full[s]);
        }
      }
      if (++s == L.pairs) s = 0;
    }
  } else if (warp == 5) {
    if (lane == 0) {
      const uint32_t idesc_qk = tc::instr_desc_bf16(kSpRows, kShBlk);
      const uint32_t idesc_pv = tc::instr_desc_bf16(kSpRows, hd) | (1u << 16);   // B is MN-major
      const int k_steps = hd >> 4;
      const uint64_t qd = tc::smem_desc_k_sw128(smem + L.q);
      const uint64_t kd0 = tc::smem_desc_k_sw128(smem + L.ring), vd0 = sp_desc_v(smem + L.ring);
      const uint64_t tile = (uint64_t)((n_sub * kSpTile) >> 4);   // a tile, in descriptor units
      auto scores = [&](int j, int slot) {                // K_j is tile `slot` of the ring
        const uint64_t kd = kd0 + slot * tile;
        const uint32_t d = tmem + (uint32_t)(j & 1) * 64;
        if (n_sub == 1) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk < k_steps) tc::umma_bf16_a_tmem(d, tmem + kColQ + 8 * kk, kd + 2 * kk, idesc_qk, kk != 0);
        } else {
          for (int kk = 0; kk < k_steps; ++kk)
            tc::umma_bf16(d, qd + (uint64_t)((kk >> 2) * ((kSpRows * 128) >> 4) + 2 * (kk & 3)),
                          kd + (uint64_t)((kk >> 2) * (kSpTile >> 4) + 2 * (kk & 3)), idesc_qk, kk != 0);
        }
      };
      bool ok = tc::mbar_wait(q_full, 0u, abort) && tc::mbar_wait(&full[0], 0u, abort);
      if (ok) {
        tc::tc_fence_after();
        scores(0, 0);
        tc::umma_commit(&done[0]);
        if (n > 1) scores(1, 1);
        tc::umma_commit(&done[1]);
      }
      for (int j = 0, s = 1, turn = 0; j < n && ok; ++j) {   // pair j + 1 in slot s
        ok = sp_wait_both(&full[s], (uint32_t)(turn & 1), &p_full[j & 1], (uint32_t)((j >> 1) & 1), abort);
        if (!ok) break;
        tc::tc_fence_after();
        const uint64_t vd = vd0 + 2 * s * tile;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)                    // 16 keys: two 1,024-byte atoms of V
          tc::umma_bf16_a_tmem(tmem + kColO, tmem + (uint32_t)((j & 1) * 64 + kk * 8), vd + (uint64_t)(kk * 128),
                               idesc_pv, (j | kk) != 0);
        if (j + 2 < n) scores(j + 2, 2 * s + 1);
        tc::umma_commit(&done[(j + 2) % kSpDone]);
        if (++s == L.pairs) { s = 0; ++turn; }
      }
    }
  } else {
    // ---- the queries into tensor memory, or into shared memory
    const int row = threadIdx.x, copy = row / span, r = row - copy * span;
    size_t at = 0;                                        // the row's place among the pieces
    {
      const bool there = r < it.n_rows;
      const int rr = it.row0 + r, of = rr / g, head = kvh * g + rr - of * g;
      const __nv_bfloat16* src = nullptr;
      if (there) {
        const int token = a.rows[it.row_base + of];
        src = static_cast<const __nv_bfloat16*>(a.q) + (size_t)token * a.ldq + (size_t)head * hd;
        at = ((size_t)a.rows_first[it.row_base + of] + it.piece) * a.nh + head;
      }
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      if (n_sub == 1) {                                   // two channels a column
        uint32_t all[32];
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          const uint4 v = there && 8 * ch < hd ? *reinterpret_cast<const uint4*>(src + 8 * ch) : zero;
          all[4 * ch] = v.x; all[4 * ch + 1] = v.y; all[4 * ch + 2] = v.z; all[4 * ch + 3] = v.w;
        }
        tc::tmem_store_32(tmem + ((uint32_t)(warp * 32) << 16) + kColQ, all);
        tc::tmem_store_wait();
        tc::tc_fence_before();
      } else {                                            // the operand's swizzled layout
        for (int ch = 0; ch < hd >> 3; ++ch) {
          const uint4 v = there ? *reinterpret_cast<const uint4*>(src + 8 * ch) : zero;
          *reinterpret_cast<uint4*>(smem + L.q + (ch >> 3) * kSpRows * 128 + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) = v;
        }
        tc::fence_proxy_async();
      }
      tc::mbar_arrive(q_full);
    }
    const uint32_t lane_addr = tmem + ((uint32_t)(warp * 32) << 16);
    const bool active = (warp * 32) % span < it.n_rows;
    float m = -INFINITY, l = 0.f;
    if (active) {
      if (fold == 1) sp_softmax<1>(lane_addr, hd, n, 0, a.scale_log2, done, p_full, abort, m, l);
      else if (fold == 2) sp_softmax<2>(lane_addr, hd, n, copy, a.scale_log2, done, p_full, abort, m, l);
      else sp_softmax<4>(lane_addr, hd, n, copy, a.scale_log2, done, p_full, abort, m, l);
      tc::mbar_wait(&done[(n + 1) % kSpDone], (uint32_t)(((n + 1) / kSpDone) & 1), abort);
      tc::tc_fence_after();
    }
    if (fold == 1) {
      const bool there = r < it.n_rows;
      if (there) a.part_ml[at] = make_float2(m, l);
      if (active)
        for (int c0 = 0; c0 < hd; c0 += 32) {
          uint32_t o[32];
          tc::tmem_load_32(lane_addr + kColO + (uint32_t)c0, o);
          tc::tmem_load_wait();
          if (there) {
            float4* dst = reinterpret_cast<float4*>(a.part_o + at * hd + c0);
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (c0 + e < hd)
                dst[e >> 2] = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                          __uint_as_float(o[e + 3]));
          }
        }
    } else {
      // the copies meet in shared memory (queries, keys and values have been read)
      float* buf = reinterpret_cast<float*>(smem);
      const int ld = hd + 4;
      asm volatile("bar.sync 1, 128;" ::: "memory");      // all rows' products are done
      if (copy == 0) place[r] = (long long)at;
      if (active) {
        xch[row] = make_float2(m, l);
        for (int c0 = 0; c0 < hd; c0 += 32) {
          uint32_t o[32];
          tc::tmem_load_32(lane_addr + kColO + (uint32_t)c0, o);
          tc::tmem_load_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (c0 + e < hd)
              *reinterpret_cast<float4*>(buf + row * ld + c0 + e) =
                  make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                              __uint_as_float(o[e + 3]));
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      // four channels a thread, `step` rows at once
      const int quads = hd >> 2, step = kSpRows / quads, mine = threadIdx.x / quads;
      const int ch = (threadIdx.x - mine * quads) * 4;
      for (int rr = mine; mine < step && rr < it.n_rows; rr += step) {
        float mm = -INFINITY, den = 0.f;
        for (int f = 0; f < fold; ++f) mm = fmaxf(mm, xch[f * span + rr].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int f = 0; f < fold; ++f) {
          const float2 ml = xch[f * span + rr];
          const float w = ml.x == -INFINITY ? 0.f : sp_exp2(ml.x - mm);
          const float4 o = *reinterpret_cast<const float4*>(buf + (f * span + rr) * ld + ch);
          den = fmaf(w, ml.y, den);
          acc.x = fmaf(w, o.x, acc.x); acc.y = fmaf(w, o.y, acc.y);
          acc.z = fmaf(w, o.z, acc.z); acc.w = fmaf(w, o.w, acc.w);
        }
        const size_t to = (size_t)place[rr];
        if (ch == 0) a.part_ml[to] = make_float2(mm, den);
        *reinterpret_cast<float4*>(a.part_o + to * hd + ch) = acc;
      }
    }
  }
  if (*abort && threadIdx.x == 0) atomicOr(a.fault, (unsigned)kFaultWaitExpired);
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    __syncwarp();
    tc::tmem_dealloc(tmem, 256);
  }
}

// ---------------------------------------------------------------------------------------
// Own keys: up to 16 rows of one sequence and key/value head are an item; its warps take 16 keys each
// in turn.  A warp fetches its own keys and values (boxes of 16 keys, TMA, 128-byte swizzle) into a ring
// of its own and needs no other warp until the end: scores and P V are m16n8k16 products with the
// rows as their rows (NR = 1: up to 8 rows, and the products' other 8 are empty).
// (Keys and values straight into the operands' registers, with no shared memory, took 120 registers and
// kept 4 KB a warp in flight: 22 us against 20.5 for 64 sequences on 32 heads with 95 own keys.)
// WPI warps share an item, a CTA has four.  Four an item where there are few; one where there are items
// enough to fill the chip with warps.
// With JOIN the item's warps hold all of the rows' own keys and join the rows' prefix pieces (the kernel is
// launched while the prefix kernel runs and waits for it only then); else they leave pieces.
constexpr int kSoWarps = 4, kSoThreads = kSoWarps * 32, kSoStages = 3;
template <int HDG, int KEYS>
constexpr int kSoStage = 2 * HDG * KEYS * 128;            // bytes: keys, then values

template <int HDG, int NR, int KEYS, int WPI, bool JOIN>
__global__ void __launch_bounds__(kSoThreads)
shared_own_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ SharedArgs a, int after_prefix) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int hd = a.hd, g = a.nh / a.nkv, kvh = blockIdx.y;
  const int cta_warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int of_cta = cta_warp / WPI, warp = cta_warp % WPI;   // item, warp of the item
  const int index = blockIdx.x * (kSoWarps / WPI) + of_cta;
  const int split = JOIN ? 0 : index % a.own_splits, splits = JOIN ? 1 : a.own_splits;
  const int which = JOIN ? index : index / a.own_splits;
  const bool none = which >= a.n_own;                     // (a warp of its own: WPI is 1)
  // (the plan is never written by a kernel)
  SharedOwnItem it;
  {
    const int4* from = reinterpret_cast<const int4*>(a.own + (none ? 0 : which));
    *reinterpret_cast<int4*>(&it.seq) = __ldcg(from);
    *reinterpret_cast<int4*>(&it.prefix) = __ldcg(from + 1);
  }
  constexpr int kRing = kSoStages * kSoStage<HDG, KEYS>;
  unsigned char* ring = smem + cta_warp * kRing;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kSoWarps * kRing) + cta_warp * kSoStages;
  int* abort_word = reinterpret_cast<int*>(smem + kSoWarps * kRing + kSoWarps * kSoStages * 8) + cta_warp;
  volatile int* abort = abort_word;                       // (of the warp)
  if (lane == 0) {
    for (int i = 0; i < kSoStages; ++i) tc::mbar_init(&full[i], 1);
    *abort = 0;
    tc::fence_barrier_init();
    tc::tma_prefetch_descriptor(&map_k);
    tc::tma_prefetch_descriptor(&map_v);
  }
  __syncwarp();
  if (!after_prefix) dependent_wait();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (none) {
    if (after_prefix) dependent_wait();
    return;
  }
  const int prefix = it.prefix, blk0 = prefix / kShBlk;
  const int slot = __ldcg(a.seq_slot + it.seq);
  const int last = __ldcg(a.tok_pos + it.tok0 + (it.row0 + it.n_rows - 1) / g);
  const int end = shared_own_end(a, it, last);
  // KEYS keys a warp and step: keys KEYS i .. of the own ones, i = first, first + stride, ...
  const int first = split * WPI + warp, stride = splits * WPI;
  const int chunks = (end - prefix + KEYS - 1) / KEYS;
  const int steps = chunks > first ? (chunks - first + stride - 1) / stride : 0;
  // the physical blocks of 32 steps, a lane each
  auto window = [&](int k0) {
    return k0 + lane < steps ? shared_block_of(a, slot, blk0 + (first + (k0 + lane) * stride) / (kShBlk / KEYS)) : 0;
  };
  int blocks = window(0);
  auto fetch = [&](int k) {                               // step k into the ring
    if (k > 0 && (k & 31) == 0) blocks = window(k);
    const int blk = __shfl_sync(0xffffffffu, blocks, k & 31);
    if (lane == 0) {
      const int s = k % kSoStages, i = first + k * stride;
      const int row = (blk * a.nkv + kvh) * kShBlk + i % (kShBlk / KEYS) * KEYS;
      unsigned char* at = ring + s * kSoStage<HDG, KEYS>;
      tc::mbar_expect_tx(&full[s], (uint32_t)kSoStage<HDG, KEYS>);
#pragma unroll
      for (int sub = 0; sub < HDG; ++sub) {
        tc::tma_load_2d(at + sub * KEYS * 128, &map_k, 64 * sub, row, &full[s]);
        tc::tma_load_2d(at + (HDG + sub) * KEYS * 128, &map_v, 64 * sub, row, &full[s]);
      }
    }
  };
  for (int k = 0; k < kSoStages && k < steps; ++k) fetch(k);
  // ---- queries: row r (and r + 8)
  uint32_t qa[HDG * 4][NR][2];                            // [16 channels][row][half]
  int pos[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int row = r + 8 * i, rr = it.row0 + row;
    const bool there = row < it.n_rows;
    const int t = it.tok0 + (there ? rr / g : 0);
    pos[i] = there ? __ldcg(a.tok_pos + t) : -1;
    const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) + (size_t)t * a.ldq +
                               (size_t)(kvh * g + (there ? rr % g : 0)) * hd;
#pragma unroll
    for (int d = 0; d < HDG * 4; ++d) {
      const bool in = there && 16 * d < hd;
      qa[d][i][0] = in ? __ldcg(reinterpret_cast<const uint32_t*>(src + 16 * d + 2 * c)) : 0u;
      qa[d][i][1] = in ? __ldcg(reinterpret_cast<const uint32_t*>(src + 16 * d + 8 + 2 * c)) : 0u;
    }
  }
  float o[HDG * 8][2 * NR];                               // [8 channels][row: 2c, 2c + 1]
#pragma unroll
  for (int t = 0; t < HDG * 8; ++t)
#pragma unroll
    for (int e = 0; e < 2 * NR; ++e) o[t][e] = 0.f;
  float m[NR], l[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
  const int mat = lane >> 3, rin = lane & 7;
  bool ok = true;
  for (int k = 0, s = 0, turn = 0; k < steps; ++k) {
    if (!tc::mbar_wait(&full[s], (uint32_t)(turn & 1), abort)) { ok = false; break; }
    const int key0 = prefix + (first + k * stride) * KEYS, n = end - key0;
    const uint32_t kbase = tc::smem_u32(ring + s * kSoStage<HDG, KEYS>), vbase = kbase + HDG * KEYS * 128;
    constexpr int X = KEYS / 16;
    float sc[2 * X][4];
#pragma unroll
    for (int x = 0; x < 2 * X; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[x][e] = 0.f;
#pragma unroll
    for (int d = 0; d < HDG * 4; ++d) {
      if (16 * d < hd) {
#pragma unroll
        for (int x = 0; x < X; ++x) {
          const int key = 16 * x + (mat >> 1) * 8 + rin, chunk = 2 * d + (mat & 1);
          uint32_t kb[4];
          ldmatrix_x4(kb, kbase + (chunk >> 3) * (KEYS * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
#pragma unroll
          for (int y = 0; y < 2; ++y)
            mma_16816_f32(sc[2 * x + y], qa[d][0][0], NR == 2 ? qa[d][NR - 1][0] : 0u, qa[d][0][1],
                          NR == 2 ? qa[d][NR - 1][1] : 0u, kb[2 * y], kb[2 * y + 1]);
        }
      }
    }
    uint32_t pa[X][4];
#pragma unroll
    for (int w = 0; w < NR; ++w) {                        // rows r, r + 8
      float t4[4 * X], mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4 * X; ++e) {
        const int key = key0 + 8 * (e >> 1) + 2 * c + (e & 1);
        t4[e] = key <= pos[w] ? sc[e >> 1][2 * w + (e & 1)] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, t4[e]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m[w], mx);
      const float alpha = m[w] == -INFINITY ? 0.f : sp_exp2(m[w] - m_new);
      float p[4 * X], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4 * X; ++e) {
        p[e] = t4[e] == -INFINITY ? 0.f : sp_exp2(t4[e] - m_new);
        sum += p[e];
      }
      l[w] = l[w] * alpha + sum;
      m[w] = m_new;
#pragma unroll
      for (int x = 0; x < X; ++x) {
        pa[x][w] = pack_bf16(p[4 * x], p[4 * x + 1]);
        pa[x][2 + w] = pack_bf16(p[4 * x + 2], p[4 * x + 3]);
        if (NR == 1) pa[x][1] = pa[x][3] = 0u;
      }
#pragma unroll
      for (int t = 0; t < HDG * 8; ++t) { o[t][2 * w] *= alpha; o[t][2 * w + 1] *= alpha; }
    }
    // values past the last key count for nothing, whatever they are
    const bool whole = n >= KEYS;
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const int at = 16 * x + 2 * c;
      const uint32_t keep0 = (at < n ? 0xffffu : 0u) | (at + 1 < n ? 0xffff0000u : 0u);
      const uint32_t keep1 = (at + 8 < n ? 0xffffu : 0u) | (at + 9 < n ? 0xffff0000u : 0u);
#pragma unroll
      for (int d = 0; d < HDG * 4; ++d) {
        if (16 * d < hd) {
          const int key = 16 * x + (mat & 1) * 8 + rin, chunk = 2 * d + (mat >> 1);
          uint32_t vb[4];
          ldmatrix_x4_trans(vb, vbase + (chunk >> 3) * (KEYS * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
          if (!whole) { vb[0] &= keep0; vb[1] &= keep1; vb[2] &= keep0; vb[3] &= keep1; }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float* to = o[2 * d + y];
            float acc[4] = {to[0], to[1], NR == 2 ? to[2 * NR - 2] : 0.f, NR == 2 ? to[2 * NR - 1] : 0.f};
            mma_16816_f32(acc, pa[x][0], pa[x][1], pa[x][2], pa[x][3], vb[2 * y], vb[2 * y + 1]);
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) to[e] = acc[e];
          }
        }
      }
    }
    if (k + kSoStages < steps) {                          // the stage has been read: its next turn
      tc::fence_proxy_async();
      __syncwarp();
      fetch(k + kSoStages);
    }
    if (++s == kSoStages) { s = 0; ++turn; }
  }
  if (!ok && lane == 0) atomicOr(a.fault, (unsigned)kFaultWaitExpired);
  __syncwarp();
  // ---- the warps' parts meet in shared memory, in the rings' place
  const int ld = hd + 4;
  float2* sml = reinterpret_cast<float2*>(smem + (size_t)(cta_warp - warp) * kRing);      // of the item's warp 0
  constexpr int kPart = kRing / 4;                        // a warp's part: [8 NR] (m, l), then [8 NR][hd + 4]
  auto part_ml_of = [&](int w) { return sml + w * (kPart / 2); };
  auto part_o_of = [&](int w) { return reinterpret_cast<float*>(sml) + w * kPart + 16 * NR; };
#pragma unroll
  for (int w = 0; w < NR; ++w) {
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
    l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
    if (c == 0) part_ml_of(warp)[r + 8 * w] = make_float2(m[w], l[w]);
    if (r + 8 * w < it.n_rows) {
      float* dst = part_o_of(warp) + (r + 8 * w) * ld + 2 * c;
#pragma unroll
      for (int t = 0; t < HDG * 8; ++t)
        if (8 * t < hd) *reinterpret_cast<float2*>(dst + 8 * t) = make_float2(o[t][2 * w], o[t][2 * w + 1]);
    }
  }
  // The prefix pieces are there; and this kernel ends behind the prefix kernel, so that what waits
  // for this one need not wait for that one.
  if (after_prefix) dependent_wait();
  if (WPI == 1) __syncwarp();
  else __syncthreads();
  const int quads = hd >> 2, n_pieces = JOIN ? it.pieces : 0;
  const int pieces_a_token = it.pieces + (JOIN ? 0 : a.own_splits);
  for (int i = warp * 32 + lane; i < it.n_rows * quads; i += WPI * 32) {
    const int row = i / quads, ch = (i - row * quads) * 4, rr = it.row0 + row;
    const int t = it.tok0 + rr / g, h = kvh * g + rr % g;
    const size_t at = ((size_t)it.first + (size_t)(t - it.tok0) * pieces_a_token) * a.nh + h;
    float ref = -INFINITY, den = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // N parts at a time: one wait for their loads, one move of the reference
    auto add = [&](auto& ml, auto& x) {
      constexpr int N = sizeof(ml) / sizeof(ml[0]);
      float top = ref;
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, ml[e].x);
      if (top == -INFINITY) return;
      const float keep = ref == -INFINITY ? 0.f : sp_exp2(ref - top);
      den *= keep;
      acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float w = ml[e].x == -INFINITY ? 0.f : sp_exp2(ml[e].x - top);
        den = fmaf(w, ml[e].y, den);
        acc.x = fmaf(w, x[e].x, acc.x); acc.y = fmaf(w, x[e].y, acc.y);
        acc.z = fmaf(w, x[e].z, acc.z); acc.w = fmaf(w, x[e].w, acc.w);
      }
      ref = top;
    };
    constexpr int kAtOnce = 8;
    for (int p0 = 0; p0 < n_pieces; p0 += kAtOnce) {
      float2 ml[kAtOnce];
      float4 x[kAtOnce];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const bool in = p0 + e < n_pieces;
        const size_t from = (size_t)(in ? p0 + e : p0) * a.nh + at;
        ml[e] = __ldcg(&a.part_ml[from]);
        x[e] = __ldcg(reinterpret_cast<const float4*>(a.part_o + from * hd + ch));
        if (!in) ml[e] = make_float2(-INFINITY, 0.f);
      }
      add(ml, x);
    }
    float2 ml[WPI];
    float4 x[WPI];
#pragma unroll
    for (int w = 0; w < WPI; ++w) {
      ml[w] = part_ml_of(w)[row];
      x[w] = *reinterpret_cast<const float4*>(part_o_of(w) + row * ld + ch);
    }
    add(ml, x);
    if (JOIN) {
      if (a.sink) {
        const float sink = a.sink[h] * 1.4426950408889634f, top = fmaxf(ref, sink);
        const float keep = ref == -INFINITY ? 0.f : sp_exp2(ref - top);
        den = den * keep + (sink == top ? 1.0f : exp2f(sink - top));
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
      }
      const float inv = den > 0.f ? 1.0f / den : 0.f;
      const uint2 packed = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (size_t)t * a.ldo + (size_t)h * hd + ch) = packed;
    } else {
      const size_t to = (size_t)(it.pieces + split) * a.nh + at;
      if (ch == 0) a.part_ml[to] = make_float2(ref, den);
      *reinterpret_cast<float4*>(a.part_o + to * hd + ch) = acc;
    }
  }
}

constexpr int kShDevices = 64;

template <typename... Params, typename... Args>
static int sp_launch(bool* asked, void (*kernel)(Params...), dim3 grid, int threads, size_t smem, size_t most, cudaStream_t st, Args&&... args) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  // (asked for once a device, and always for the `most` that any launch takes: two threads that ask for what they
  // each need could leave the smaller one)
  if (dev >= kShDevices || !asked[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) return (int)e;
    if (dev < kShDevices) asked[dev] = true;
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = dependent_launch_enabled();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
  return e == cudaSuccess ? launch_status() : (int)e;
}

// How an item's keys are cut, by how many warps the launch keeps busy.
enum SoCut { kSoWide, kSoNarrow, kSoWarp };               // 32 keys, 16 keys, a warp an item

template <int HDG, int NR, int KEYS, int WPI, bool JOIN>
static int launch_own_as(const SharedArgs& a, cudaStream_t st) {
  constexpr size_t smem = (size_t)kSoWarps * kSoStages * (kSoStage<HDG, KEYS> + 8) + kSoWarps * 4 + 1024;
  static bool asked[kShDevices];
  CUtensorMap mk, mv;
  const int rows = (int)(a.n_blocks * a.nkv * kShBlk);
  if (make_tile_map_bf16(&mk, a.kc, rows, a.hd, a.hd, KEYS) || make_tile_map_bf16(&mv, a.vc, rows, a.hd, a.hd, KEYS))
    return kBadArgument;
  const int ctas = JOIN ? (a.n_own * WPI + kSoWarps - 1) / kSoWarps : a.n_own * a.own_splits;
  return sp_launch(asked, shared_own_mma_kernel<HDG, NR, KEYS, WPI, JOIN>, dim3(ctas, a.nkv), kSoThreads, smem, smem, st,
                   mk, mv, a, (int)(a.n_pre > 0));
}

template <int HDG, int NR>
static int launch_own(const SharedArgs& a, cudaStream_t st) {
  const long long items = (long long)a.n_own * a.nkv;
  // (own keys are cut where there are few items, and few items have up to 8 rows)
  if (a.own_splits > 1) {
    if constexpr (NR == 1) return launch_own_as<HDG, NR, 32, 4, false>(a, st);
    else return kBadArgument;
  }
  const SoCut cut = items > 8 * kSmCount ? kSoWarp : items > (HDG == 1 ? 2 : 1) * kSmCount ? kSoNarrow : kSoWide;
  if (cut == kSoWarp) return launch_own_as<HDG, NR, 16, 1, true>(a, st);
  if constexpr (HDG == 1 || NR == 1)
    if (cut == kSoWide) return launch_own_as<HDG, NR, 32, 4, true>(a, st);
  return launch_own_as<HDG, NR, 16, 4, true>(a, st);
}

// The prefix pieces and the own keys; joins the rows where the own keys are in one piece.
int launch_shared_bf16(const SharedArgs& a, cudaStream_t st) {
  if (((uintptr_t)a.q & 15) || a.ldq % 8 || ((uintptr_t)a.out & 7) || a.ldo % 4) return kMisaligned;
  const long long cache_rows = a.n_blocks * a.nkv * kShBlk;
  if (cache_rows > 0x7fffffffLL) return kBadArgument;
  if (a.n_pre > 0) {
    CUtensorMap mk, mv;
    if (make_tile_map_bf16(&mk, a.kc, (int)cache_rows, a.hd, a.hd, kShBlk) ||
        make_tile_map_bf16(&mv, a.vc, (int)cache_rows, a.hd, a.hd, kShBlk))
      return kBadArgument;
    const SpSmem L((a.hd + 63) / 64);
    static const int kSpMost = SpSmem(1).total > SpSmem(2).total ? SpSmem(1).total : SpSmem(2).total;
    static bool asked[kShDevices];
    const int e = sp_launch(asked, shared_prefix_tc_kernel, dim3(a.n_pre, a.nkv), kSpThreads, L.total,
                            kSpMost, st, mk, mv, a);
    if (e) return e;
  }
  if (a.own_rows <= 8) return a.hd <= 64 ? launch_own<1, 1>(a, st) : launch_own<2, 1>(a, st);
  return a.hd <= 64 ? launch_own<1, 2>(a, st) : launch_own<2, 2>(a, st);
}

}  // namespace cretif
