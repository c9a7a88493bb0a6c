// qr_kv_pool.h -- the layout of a shared 8-bit KV pool (qr_kv_pool of
// qr_hip.h) as its kernels see it, and how a ragged batch's rows are found.
//
// A block is 16 tokens of one kv head of one layer: int8 K [16][hd], then int8
// V [hd][16], and two fp32 scales.  V lies column by column, so that 16 bytes
// of it are one column's 16 tokens: what a lane widens to its operands of two
// 16x16x32 fp16 MFMA of the value product.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qr_internal.h"

namespace qr {

constexpr int kKvBlock = 16;  // tokens of a scale

// One layer of a pool.
struct PoolView {
  int8_t* data;
  float* scale;
  const int32_t* table;
  const int32_t* len;
  int n_pages, n_kv_heads, hd, n_seqs, max_pages;
  int page_shift;
};

// The rows of a ragged batch: sequence i owns rows start[i] .. start[i + 1] - 1,
// which stand for its last positions.  T rows exist; values outside 0 .. T are
// cut to it, so a bad array reads and writes no row that is not there.
struct Ragged {
  const int32_t* seqs;   // [n] rows of the table, or null: 0 .. n - 1
  const int32_t* start;  // [n + 1]
  int n, T;
};

__device__ inline int ragged_start(const Ragged& r, int i) {
  const int s = r.start[i];
  return s < 0 ? 0 : s > r.T ? r.T : s;
}

// A sequence of the batch: its row of the table (0 and not `there` where it does not
// exist), its rows and its length.
struct SeqRows {
  int seq, row0, m, len;
  bool there;
};
__device__ inline int seq_len(const PoolView& p, const SeqRows& s) {
  const long cap = (long)p.max_pages << p.page_shift;
  const int n = __builtin_amdgcn_readfirstlane(p.len[s.seq]);
  return !s.there || n < 0 ? 0 : n > cap ? (int)cap : n;
}

// Which sequence a slot serves, where each sequence's rows are cut into pieces
// of q rows: sequence i has the slots from start[i] / q + extra * i on.  There
// are never fewer than its pieces (floor(b / q) - floor(a / q) + 1 >=
// ceil((b - a) / q)), so the host sizes the grid by T / q + extra * n without
// knowing the lengths, and a slot without a piece ends.  *piece: which of the
// sequence's slots this is, < 0 for none.  The length is not looked up here: other loads go
// out beside it (seq_len).
//
// All lanes of the wave search at once, 64 places a step, and what is needed of
// the place is loaded beside it: up to 64 sequences take two dependent
// loads (a binary search took one for each of its steps, 5 us of a launch over 32).
__device__ inline SeqRows slot_rows(const PoolView& p, const Ragged& r, int slot, int q, int extra,
                                    int* piece) {
  const int lane = (int)(threadIdx.x & 63);
  int lo = 0, count = r.n, at, first, next, seq;
  unsigned long long below;
  for (;;) {
    const int step = (count + 63) >> 6;
    at = lo + lane * step;
    const bool in = lane * step < count;
    if (!in) at = lo;
    first = ragged_start(r, at);
    next = 0;
    seq = at;
    if (step == 1) {
      next = ragged_start(r, at + 1);
      if (r.seqs) seq = r.seqs[at];
    }
    below = __ballot(in && first / q + extra * at <= slot);
    const int k = below ? 63 - __builtin_clzll(below) : 0;
    if (step == 1) {
      SeqRows s;
      s.row0 = __builtin_amdgcn_readlane(first, k);
      s.m = __builtin_amdgcn_readlane(next, k) - s.row0;
      if (s.m < 0) s.m = 0;
      s.seq = __builtin_amdgcn_readlane(seq, k);
      *piece = slot - (s.row0 / q + extra * (lo + k));
      s.there = (unsigned)s.seq < (unsigned)p.n_seqs;
      if (!s.there) s.seq = 0;
      s.len = 0;
      return s;
    }
    lo += k * step;
    count = count - k * step < step ? count - k * step : step;
  }
}

// The physical page of a sequence's logical page, -1 where there is none.
__device__ inline int page_at(const PoolView& p, int seq, int lp) {
  if ((unsigned)lp >= (unsigned)p.max_pages) return -1;
  const int g = p.table[(size_t)seq * p.max_pages + lp];
  return (unsigned)g < (unsigned)p.n_pages ? g : -1;
}

// Index of a block of the layer: (page, kv head, block of the page).
__device__ inline size_t block_at(const PoolView& p, int page, int kvh, int b) {
  return (((size_t)page * p.n_kv_heads + kvh) << (p.page_shift - 4)) + (size_t)b;
}

// qr_kv_attn.hip
hipError_t kv_attention_launch(const PoolView& p, const Ragged& r, int n_heads, const float* q,
                               long q_stride, float* out, long out_stride, int max_len, int window,
                               float scale, void* work, hipStream_t st);
size_t kv_attention_scratch(const PoolView& p, const Ragged& r, int n_heads, int max_len,
                            int window);

}  // namespace qr
