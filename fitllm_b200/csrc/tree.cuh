// Trees of drafted tokens behind a 16-bit key/value cache whose sequences have lengths of
// their own: addressing shared by the append, attention and keep kernels (tree.cu,
// tree_attn.cu).
//
// A tree is parents[T], T <= 64: the index of token i's parent (below i), -1 for a token
// right behind the cached positions, -2 where there is no token.  Token i of sequence b
// stands in slot prefix[b] + i; it sees the cached positions, its ancestors and itself, a
// 64-bit word with bit j for token j.  As parents lie below their children the walk to the
// root ends for every content of the array.
#pragma once
#include "common.cuh"
#include "kv4.cuh"

namespace fitq {

constexpr int kTreeTokens = 64;

struct TreeView {
  const int32_t* parents;
  int64_t parents_stride;  // entries from sequence to sequence, 0: one tree for all
  const int32_t* prefix;   // [batch] cached positions
  int batch, tokens, kv_heads;
  int64_t capacity;        // slots of a sequence
  int64_t stride_b, stride_h, stride_p;  // elements between sequences, KV heads and slots
};

// Parent of token i of sequence b; -2 for anything that is no parent, *bad set where it
// is not the -2 that says so.
__device__ __forceinline__ int tree_parent(const TreeView& t, int64_t b, int i, bool* bad) {
  const int p = t.parents[b * t.parents_stride + i];
  if (p >= -1 && p < i) return p;
  if (p != -2) *bad = true;
  return -2;
}

// Walks from token i to its root through `up` (parents as tree_parent gives them): the
// token's word and depth; false where the token or an ancestor is absent.
__device__ __forceinline__ bool tree_walk(const int* up, int i, uint64_t* seen, int* depth) {
  uint64_t word = 0;
  int d = -1, cur = i;
  while (cur >= 0) {
    word |= 1ull << cur;
    ++d;
    cur = up[cur];
  }
  *seen = word;
  *depth = d;
  return cur == -1;
}

}  // namespace fitq
