// What the kernels of the attention over a shared prefix have in common (attn_shared.cu).
//
// The keys of a batch's queries are cut into pieces: a prefix that a group of sequences shares in
// ranges of whole blocks, each walked once for all the group's rows, and every sequence's own keys
// behind it.  A piece leaves, for each of its rows (a token and a query head), the largest scaled
// score m (times log2 e), l = sum 2^(s - m) and o = sum 2^(s - m) v; a row's output is
//   sum_i 2^(m_i - m) o_i / (sum_i 2^(m_i - m) l_i + 2^(sink - m)),   m = max_i m_i.
#pragma once

#include <cuda_runtime.h>

#include "common.cuh"

namespace cretif {

constexpr int kShBlk = 64;                 // tokens of a cache block

// A range of blocks of a group's prefix for some of the group's rows.  Row r of a key/value head is
// query head kvh * g + r % g of token rows[row_base + r / g].
struct alignas(16) SharedPrefixItem {
  int row_base, row0, n_rows;
  int seq;                                 // a member: its table is read
  int blk0, blk1;                          // blocks [blk0, blk1)
  int piece;                               // the piece's index among the rows' pieces
  int pad;
};
// Some rows of one sequence over its own keys: row r is head kvh * g + r % g of token tok0 + r / g.
struct alignas(16) SharedOwnItem {
  int seq, tok0, row0, n_rows;
  int prefix, pieces;                      // tokens that are other items' work, and pieces they are in
  int least;                               // the least position of the sequence: the tokens it shares
  int first;                               // token tok0's first piece
};

// What every kernel of a call reads.
struct SharedArgs {
  const void *q, *kc, *vc;
  void* out;
  long long ldq, ldo;                      // (rows may lie more than 2^31 numbers apart)
  long long n_blocks;
  const int* table;
  long long table_stride;
  int table_width, n_slots;                // (a row's places lie a stride apart; a view's may be fewer)
  const int *tok_pos, *seq_slot;
  // The plan: prefix items, own items (of up to own_rows rows), the tokens of the groups, and where the pieces
  // lie: a token has as many as it needs, one behind the other, so that a long prefix of few sequences costs
  // the others no room.  [n_rows] first piece of the groups' tokens, [T + 1] of all.
  const SharedPrefixItem* pre;
  const SharedOwnItem* own;
  const int *rows, *rows_first, *first;
  int n_pre, n_own, own_rows, own_splits, T;
  int nh, nkv, hd;
  float scale_log2;
  const float* sink;
  float* part_o;                           // [pieces of all tokens][nh][hd]
  float2* part_ml;                         // [pieces of all tokens][nh]
  unsigned int* fault;
};

// The physical block at place `at` of a slot's table; 0 and a fault bit where there is none.
// (What the step's earlier kernels and copies wrote is read from L2 here: the own keys' kernel starts under the
// prefix kernel and has no wait of its own in front.)
__device__ __forceinline__ int shared_block_of(const SharedArgs& a, int slot, int at) {
  int blk = -1;
  if (slot >= 0 && slot < a.n_slots && at >= 0 && at < a.table_width)
    blk = __ldcg(a.table + (size_t)slot * a.table_stride + at);
  if (blk < 0 || blk >= a.n_blocks) {
    atomicOr(a.fault, (unsigned)kFaultBlockTable);
    blk = 0;
  }
  return blk;
}
__device__ __forceinline__ int shared_block(const SharedArgs& a, int seq, int at) {
  return shared_block_of(a, __ldcg(a.seq_slot + seq), at);
}

// One past the last own key that an item's row at position `last` sees.  A position inside the shared
// tokens or behind the table is a caller's mistake: the fault bit is set and there are none (walked
// all the same, a position of 2^31 would keep a warp for seconds).
__device__ __forceinline__ int shared_own_end(const SharedArgs& a, const SharedOwnItem& it, int last) {
  if (last >= it.least && last < (long long)a.table_width * kShBlk && last < 0x7fffff00) return last + 1;
  atomicOr(a.fault, (unsigned)kFaultBlockTable);
  return it.prefix;
}

}  // namespace cretif
