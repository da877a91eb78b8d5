// The walk of a verify step down the drafted tree, shared by the greedy and the sampled acceptance.
#pragma once
#include "cfh_common.h"

namespace {

// One wave walks one request's n nodes: from the root row (cur = -1), emit the row's token; move to the first child
// whose drafted token equals it (64 nodes tested at a time, a ballot picks the lowest); stop where none does, or
// where the row has no token (negative).  tok(row), par(node), drafted(node) read the request's rows 0 .. n and nodes;
// emit(pos, row, token) stores an output and took(pos, node) an accepted node (every lane calls them).  -> nodes taken.
template <typename Tok, typename Par, typename Draft, typename Emit, typename Took>
__device__ __forceinline__ int walk_tree(int n, int max_spec, Tok tok, Par par, Draft drafted, Emit emit, Took took) {
  const int lane = threadIdx.x & 63;
  int cur = -1, pos = 0;
  for (int step = 0; step <= max_spec; ++step) {
    const int t = tok(cur + 1);
    if (t < 0) break;
    emit(pos, cur + 1, t);
    int nxt = -1;
    if (pos < max_spec) {
      for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        const unsigned long long m = __ballot(i < n && par(i) == cur && drafted(i) == t);
        if (m) {
          nxt = i0 + __ffsll((long long)m) - 1;
          break;
        }
      }
    }
    if (nxt < 0) break;
    took(pos, nxt);
    cur = nxt;
    ++pos;
  }
  return pos;
}

}  // namespace
