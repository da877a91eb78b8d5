// Sequences of rows given by bounds cu[0 .. S] on the device: sequence s has the rows cu[s] .. cu[s + 1].
#pragma once
#include <algorithm>

#include "cfh_common.h"

namespace {

// The last i in [0, n) with pred(i), for a pred that holds up to some i and not behind it; 0 where it holds nowhere.
// 64 a step, the same over the wave.
template <typename F>
__device__ __forceinline__ int last_where(int n, F pred) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const unsigned long long m = __ballot(i < lo + n && pred(i));
    const int k = m ? 63 - __builtin_clzll(m) : 0;
    n = min(step, lo + n - (lo + k * step));
    lo += k * step;
  }
  return lo;
}

// The number of sequences before the first bound that falls below the one before it (S: none does).  Sequences from
// there on are skipped: a search over bounds that do not ascend would miss some of those before it, too.
//   Each wave looks for itself up to ASC_OWN sequences, all loads in flight together (the delta rule over 64 single rows
// 33.8 us without, 33.9 with); of more, one workgroup looks for all before them (k_ascending; 500 sequences of one or two
// rows: 266 us without, 275, and 290 with every wave looking).
constexpr int ASC_OWN = 256;
__device__ __forceinline__ int first_fall(const int* cu, int S, int lo, int hi) {
  const int lane = threadIdx.x & 63;
  int first = S;
  for (int b = lo; b < hi; b += ASC_OWN) {
    int x[ASC_OWN / 64], y[ASC_OWN / 64];
#pragma unroll
    for (int u = 0; u < ASC_OWN / 64; ++u) {
      const int i = min(b + 64 * u + lane, hi - 1);
      x[u] = cu[i];
      y[u] = cu[i + 1];
    }
#pragma unroll
    for (int u = ASC_OWN / 64 - 1; u >= 0; --u) {
      const unsigned long long m = __ballot(x[u] > y[u]);
      if (m) first = min(first, b + 64 * u + __builtin_ctzll(m));
    }
  }
  return first;                                    // (behind hi - 1 the last place's again, which is found before)
}
__device__ __forceinline__ int ascending(const int* cu, int S) { return first_fall(cu, S, 0, S); }

__global__ void __launch_bounds__(1024) k_ascending(const int* cu, int S, int* whole) {
  __shared__ int found[16];
  const int wave = threadIdx.x >> 6, per = (S + 15) / 16;
  const int first = first_fall(cu, S, min(S, wave * per), min(S, (wave + 1) * per));
  if ((threadIdx.x & 63) == 0) found[wave] = first;
  __syncthreads();
  if (threadIdx.x == 0) {
    int w = S;
    for (int i = 15; i >= 0; --i) w = min(w, found[i]);
    *whole = w;
  }
}

// The last sequence i with pred(i, cu[i]) of those before the first bound that falls, and its bounds; s = -1 where there
// is none.  pred holds up to some i and not behind it.  `whole`: k_ascending's count, or null: the bounds are looked over
// on the way, 64 U of them at a time, which needs no load behind the first where one place holds them all.
struct Seq { int s, c0, c1; };
template <int U, typename F>
__device__ __forceinline__ Seq find_looking(const int* cu, int S, F pred) {
  const int lane = threadIdx.x & 63;
  Seq f = {-1, 0, 0};
  for (int b = 0; b < S; b += 64 * U) {
    int x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(b + 64 * u + lane, S - 1);
      x[u] = cu[i];
      y[u] = cu[i + 1];
    }
    bool on = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = b + 64 * u + lane;
      const unsigned long long in = __ballot(i < S && pred(i, x[u])), fall = __ballot(x[u] > y[u]);
      const unsigned long long m = on ? in & (fall ? (fall & -fall) - 1 : ~0ull) : 0;
      if (m) {
        const int k = 63 - __builtin_clzll(m);
        f = {b + 64 * u + k, __builtin_amdgcn_readlane(x[u], k), __builtin_amdgcn_readlane(y[u], k)};
      }
      on = m == ~0ull;
    }
    if (!on) break;
  }
  return f;
}
template <typename F>
__device__ __forceinline__ Seq find_seq(const int* cu, int S, const int* whole, F pred) {
  if (!whole) return S <= 64 ? find_looking<1>(cu, S, pred) : find_looking<4>(cu, S, pred);
  const int n = *whole, s = last_where(n, [&](int i) { return pred(i, cu[i]); });
  return {s < n ? s : -1, cu[s], cu[s + 1]};
}

// The rows of [0, T) that some sequence has, of the first n, whose bounds ascend: one range, as those that begin below 0
// come first and those that end behind T last.
struct Rows { int lo, hi; };
__device__ __forceinline__ Rows covered(const int* cu, int n, int T) {
  const int i0 = cu[0] < 0 ? last_where(n + 1, [&](int i) { return cu[i] < 0; }) + 1 : 0;
  if (i0 > n || cu[i0] > T) return {0, 0};
  return {cu[i0], cu[last_where(n + 1, [&](int i) { return cu[i] <= T; })]};
}

// f(row) for the rows of [0, T) outside a range, dealt out over `parts` workgroups.
template <typename F>
__device__ __forceinline__ void each_outside(const Rows& r, int T, int part, int parts, F f) {
  for (int i = part; i < r.lo + T - r.hi; i += parts) f(i < r.lo ? i : i - r.lo + r.hi);
}

// Workgroups that clear such rows, of `bytes` in all: 32 KB each, as far as that goes.
inline unsigned clearing(long long bytes) { return (unsigned)std::min(256ll, (bytes + 32767) / 32768); }

}  // namespace
