// What the kernels of attention in parts share: which rows see which keys, and the layout of the partial results.
//
// The softmax of a row over its keys 0..p is taken in parts, each over a range of the keys: (m, l, o) with m the largest
// scaled score in log2 units, l = sum 2^(s - m) and o = sum 2^(s - m) v; parts join as
//   M = max m_i, out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.
// A part without a key has m = -infinity and l = 0, and its o is not written nor read.
//
// Sequences of a pass may fall into groups whose members hold the same first `len` positions in the same pages. The prefix
// part takes those for all rows of a group at once (through the first member's page table), the own parts a sequence's
// other keys. Without groups the own parts take every key.
#pragma once

#include "common.cuh"

struct Segments {
  const int *cu_q, *seq_slot, *seq_start, *seq_qlen;  // per sequence; see BatchMeta
  const int *group_cu, *group_len, *seq_group;        // first sequence of each group (and their number), its shared positions, group of each sequence
  int n_seqs, n_groups;
  const int* table;
  int width;
};

// The rows and keys of one unit of work: rows row0 .. row0 + n_tok - 1 of the step (times the G heads of a kv head), keys
// key_lo .. key_hi - 1 of slot `slot`; token t sees keys up to start + t (of a prefix all: its start lies behind every key).
struct Unit {
  int row0, n_tok, key_lo, key_hi, slot, start;
};

__device__ __forceinline__ Unit prefix_unit(const Segments& s, int group) {
  Unit u;
  const int first = s.group_cu[group], last = s.group_cu[group + 1];
  u.row0 = s.cu_q[first];
  u.n_tok = s.cu_q[last] - u.row0;
  u.key_lo = 0;
  u.key_hi = min(s.group_len[group], s.width * KRK_PAGE);  // no page beyond a slot's
  u.slot = s.seq_slot[first];
  u.start = 0x3fffffff;  // every key of the prefix lies before every row
  return u;
}

__device__ __forceinline__ Unit own_unit(const Segments& s, int seq) {
  Unit u;
  u.row0 = s.cu_q[seq];
  u.n_tok = s.seq_qlen[seq];
  u.start = s.seq_start[seq];
  u.key_lo = s.n_groups > 0 ? s.group_len[s.seq_group[seq]] : 0;
  u.key_hi = min(u.start + u.n_tok, s.width * KRK_PAGE);  // no page beyond a slot's
  u.slot = s.seq_slot[seq];
  return u;
}

// Split `split` of n of the pages of keys lo .. hi - 1 (lo on a page's first position): pages j_lo .. j_hi - 1.
__device__ __forceinline__ void split_pages(int lo, int hi, int split, int n, int& j_lo, int& j_hi) {
  const int first = lo / KRK_PAGE, last = (hi + KRK_PAGE - 1) / KRK_PAGE;
  const int per = (max(last - first, 0) + n - 1) / n;
  j_lo = min(first + split * per, last);
  j_hi = min(j_lo + per, last);
}

// Partial results: o[part][row][head][D] and (m, l)[part][row][head].
struct Parts {
  float* o;
  float2* ml;
  int rows, HQ;
  __device__ __forceinline__ size_t at(int part, int row, int head) const { return ((size_t)part * rows + row) * HQ + head; }
};
