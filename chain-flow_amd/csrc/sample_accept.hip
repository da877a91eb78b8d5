// The sampled verify on MI355X: each row's target token drawn from its filtered softmax by a given uniform number,
// and the walk down the drafted tree that accepts what was drawn.
//
// The drafts come from a beam search, so a drafted token stands for itself with probability one, and rejection
// sampling against the target's p reduces to: draw t from the row's p, step to the child that holds t.  (At a node
// with children x_1 .. x_c that is the recursive rule: x_i is accepted with p(x_i) / (1 - p(x_1) - .. - p(x_{i-1})),
// and where none is, the token comes from p without them.)
//
// A row's tokens are ordered by (logit descending, index ascending); NaN and -inf are no tokens.  With m the largest:
//     w_j = exp((x_j - m) / T),  the first k of the order,  of those the shortest prefix with sum >= P * (their sum),
//     token = the first whose running sum exceeds u * (sum of what is kept),  log p = log(w / that sum).
// T = 0 takes the first of the order.
//
// 16-bit logits have at most 65,536 values, so a row is its count of each value: counts are whole numbers (their order of
// addition does not matter), a value's weight is computed once for all tokens that have it, in 64 bits, and the cuts of k and
// P and the draw are searches over the counts.  In 32 bits a running sum over 248,320 tokens would be off by more than
// many a token's share.
#include <math.h>

#include <type_traits>

#include "cfh_host.h"
#include "cfh_kv.h"
#include "cfh_seq.h"
#include "cfh_walk.h"

namespace {

constexpr int SA_T = 1024, SA_W = SA_T / 64;   // threads and waves of a row
constexpr int SA_GROUPS = 65536 / (4 * SA_T);  // groups of 4 values a thread: 16
constexpr int SA_CELLS = SA_GROUPS * SA_W;     // (group, wave): 256 values each, in the order's order

struct SampleArgs {
  const u16* logits;
  long long ld;
  int V, R, B;
  const int* cu_rows;        // [B] inclusive cumulative rows
  const float* u;            // [R]
  const float* temp;         // [B]
  const int* top_k;          // [B] or null
  const float* top_p;        // [B] or null
  int* tok;                  // [R]
  float* lp;                 // [R]
};

// Order-preserving 16-bit key of a logit (-0 as 0); -1: no token (NaN, -inf).
template <bool BF>
__device__ __forceinline__ int key_of(unsigned x) {
  constexpr unsigned INF = BF ? 0x7f80u : 0x7c00u;
  const unsigned mag = x & 0x7fffu;
  if (mag > INF || x == (0x8000u | INF)) return -1;
  if (mag == 0) return 0x8000;
  return (int)(x & 0x8000u ? 0xffffu - x : x | 0x8000u);
}
template <bool BF>
__device__ __forceinline__ double value_of(int key) {
  const unsigned x = key & 0x8000 ? key & 0x7fffu : 0xffffu - (unsigned)key;
  if constexpr (BF) return (double)__uint_as_float(x << 16);
  else return (double)__builtin_bit_cast(_Float16, (u16)x);
}

__device__ __forceinline__ double shfl_up_d(double v, int d) { return __shfl_up(v, d); }

// What a row's searches share.
struct Row {
  double m, T;
  int key_max;
  bool wide;                 // 32-bit counts of one half of the values at a time (see k_sample_rows)
};

// The weight of a value: 1 at the largest, nothing else beside an infinite one.
template <bool BF>
__device__ __forceinline__ double weight_of(const Row& r, int key) {
  if (key == r.key_max) return 1.0;
  if (isinf(r.m)) return 0.0;
  return exp((value_of<BF>(key) - r.m) / r.T);
}

// Counts of the four values at order positions 4096 g + 4 t .. + 3 (position o = value 65535 - o).  hist[w] holds
// value w + 32768's count in its high half and value w's in its low one, or, `wide`, the whole count of one of the two.
__device__ __forceinline__ void counts_of(const unsigned* hist, bool wide, int g, int t, unsigned (&c)[4]) {
  const int o = (g & 7) * 4 * SA_T + 4 * t;
  const uint4 w = *(const uint4*)(hist + 32768 - 4 - o);
  const unsigned v[4] = {w.w, w.z, w.y, w.x};
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] = wide ? v[e] : g < 8 ? v[e] >> 16 : v[e] & 0xffffu;
}

// The place where a running count or sum passes a goal: the value, and what stands before it.
struct Place { int key; unsigned count; double w, before_m; long long before_n; };

template <bool BF, bool VEC>
__global__ void __launch_bounds__(SA_T) k_sample_rows(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned hist[32768];
  __shared__ double cell_m[SA_CELLS];
  __shared__ int cell_n[SA_CELLS];
  __shared__ int s_int[SA_W], s_key[SA_W];
  __shared__ Place s_place;
  const int row = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  // request b > 0 has the rows cu_rows[b - 1] .. cu_rows[b], the first those below cu_rows[0]
  int b = 0;
  if (row >= a.cu_rows[0]) {
    const Seq f = find_looking<1>(a.cu_rows, a.B - 1, [&](int, int c) { return c <= row; });
    b = f.s >= 0 && row < f.c1 ? f.s + 1 : -1;
  }
  if (b < 0) {                                       // a row of no request
    if (t == 0) { a.tok[row] = -1; a.lp[row] = 0.f; }
    return;
  }
  const float Tf = a.temp[b];
  const bool greedy = !(Tf > 0.f);
  Row r;
  r.T = Tf;
  r.wide = false;
  const u16* x = a.logits + (size_t)row * a.ld;
  const int V = a.V, nvec = (V + 7) / 8;

  // eight logits from 8 j on, -inf behind the row's end
  auto load8 = [&](int j, unsigned (&e)[8]) {
    constexpr unsigned NONE = BF ? 0xff80u : 0xfc00u;
    if (VEC && 8 * j + 8 <= V) {
      const uint4 w = *(const uint4*)(x + (size_t)8 * j);
      const unsigned q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { e[2 * i] = q[i] & 0xffffu; e[2 * i + 1] = q[i] >> 16; }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = 8 * j + i < V ? x[(size_t)8 * j + i] : NONE;
    }
  };
  // counts of the row's values (half < 0: all, packed; else of the values whose top bit is `half`); the largest key and
  // the number of tokens counted
  auto count = [&](int half, int& key_max, int& n) {
    for (int i = t; i < 32768 / 4; i += SA_T) ((uint4*)hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    int mine = -1, num = 0;
    for (int j = t; j < nvec; j += SA_T) {
      unsigned e[8];
      load8(j, e);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = key_of<BF>(e[i]);
        mine = max(mine, k);
        if (k < 0 || (half >= 0 && k >> 15 != half)) continue;
        ++num;
        if (!greedy) atomicAdd(&hist[k & 0x7fff], half < 0 && k >> 15 ? 0x10000u : 1u);
      }
    }
    for (int off = 32; off >= 1; off >>= 1) {
      mine = max(mine, __shfl_xor(mine, off));
      num += __shfl_xor(num, off);
    }
    if (lane == 0) { s_key[wave] = mine; s_int[wave] = num; }
    __syncthreads();
    key_max = -1;
    n = 0;
    for (int w = 0; w < SA_W; ++w) { key_max = max(key_max, s_key[w]); n += s_int[w]; }
    __syncthreads();
  };
  // count and weight of every cell of the groups g0 .. g1 - 1; -> tokens in them
  auto cells = [&](int g0, int g1) {
    for (int g = g0; g < g1; ++g) {
      unsigned c[4];
      counts_of(hist, r.wide, g, t, c);
      int n = (int)(c[0] + c[1] + c[2] + c[3]);
      double m = 0.0;
      if (n)
        for (int e = 0; e < 4; ++e)
          if (c[e]) m += c[e] * weight_of<BF>(r, 65535 - (g * 4 * SA_T + 4 * t + e));
      for (int off = 32; off >= 1; off >>= 1) {
        n += __shfl_xor(n, off);
        m += __shfl_xor(m, off);
      }
      if (lane == 0) { cell_n[g * SA_W + wave] = n; cell_m[g * SA_W + wave] = m; }
    }
  };
  int held = -1;                                     // (wide) the half whose counts hist holds
  auto hold = [&](int half) {
    if (!r.wide || held == half) return;
    int km, n;
    count(half, km, n);
    held = half;
  };

  int total;
  count(-1, r.key_max, total);
  if (r.key_max < 0) {                               // nothing to draw from
    if (t == 0) { a.tok[row] = -1; a.lp[row] = 0.f; }
    return;
  }
  r.m = value_of<BF>(r.key_max);
  int key = r.key_max;
  unsigned rank = 0;
  double lp = 0.0;
  if (!greedy) {
    cells(0, SA_GROUPS);
    __syncthreads();
    int sum = 0;
    for (int i = lane; i < SA_CELLS; i += 64) sum += cell_n[i];
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
    // A value that 65,536 tokens have leaves its 16 bits: a low half's carry makes the sum 65,535 too small, a high
    // half's 65,536, so that the sum is right only where no count left its half.  Then each half of the values is counted in 32 bits.
    if (sum != total) {
      r.wide = true;
      for (int half = 1; half >= 0; --half) {
        __syncthreads();
        hold(half);
        cells(half ? 0 : 8, half ? 8 : 16);
      }
      __syncthreads();
    }
    // The first value at which the running sum (by_n: count) reaches goal_m (goal_n), strictly passing it if `past`; the
    // last one of any weight where rounding leaves none.  Only the first `end_n` tokens of the order count.
    auto find = [&](bool by_n, long long goal_n, double goal_m, bool past, long long end_n) {
      __shared__ int s_cell;
      __shared__ double s_m;
      __shared__ long long s_n;
      if (wave == 0) {
        constexpr int PER = SA_CELLS / 64;
        long long n[PER], nl = 0;
        double m[PER], ml = 0.0;
        for (int i = 0; i < PER; ++i) {
          nl += cell_n[lane * PER + i]; ml += cell_m[lane * PER + i];
          n[i] = nl; m[i] = ml;
        }
        long long ns = nl;
        double ms = ml;
        for (int off = 1; off < 64; off <<= 1) {
          const long long on = __shfl_up(ns, off);
          const double om = shfl_up_d(ms, off);
          if (lane >= off) { ns += on; ms += om; }
        }
        // sums before this lane's cells: the lane before's inclusive ones
        long long nb = __shfl_up(ns, 1);
        double mb = shfl_up_d(ms, 1);
        if (lane == 0) { nb = 0; mb = 0.0; }
        int hit = -1, last = -1;
        for (int i = PER - 1; i >= 0; --i) {
          const long long n0 = nb + (i ? n[i - 1] : 0);
          const int here = (int)(nb + n[i] - n0);
          if (!here || n0 >= end_n || (!by_n && !(m[i] > (i ? m[i - 1] : 0.0)))) continue;
          if (last < 0) last = lane * PER + i;
          if (by_n ? nb + n[i] >= goal_n : past ? mb + m[i] > goal_m : mb + m[i] >= goal_m) hit = lane * PER + i;
        }
        const unsigned long long any = __ballot(hit >= 0), some = __ballot(last >= 0);
        const int from = any ? __ffsll((long long)any) - 1 : 63 - __builtin_clzll(some);
        const int cell = __shfl(any ? hit : last, from);
        if (lane == cell / PER) {
          const int i = cell % PER;
          s_cell = cell;
          s_m = mb + (i ? m[i - 1] : 0.0);
          s_n = nb + (i ? n[i - 1] : 0);
        }
      }
      __syncthreads();
      const int cell = s_cell, g = cell / SA_W;
      hold(g < 8);
      if (wave == 0) {
        const int tt = (cell % SA_W) * 64 + lane;
        unsigned c[4];
        counts_of(hist, r.wide, g, tt, c);
        double w[4], ml = 0.0;
        long long nl = 0;
        for (int e = 0; e < 4; ++e) {
          w[e] = c[e] ? weight_of<BF>(r, 65535 - (g * 4 * SA_T + 4 * tt + e)) : 0.0;
          ml += c[e] * w[e];
          nl += c[e];
        }
        long long ns = nl;
        double ms = ml;
        for (int off = 1; off < 64; off <<= 1) {
          const long long on = __shfl_up(ns, off);
          const double om = shfl_up_d(ms, off);
          if (lane >= off) { ns += on; ms += om; }
        }
        long long nb = __shfl_up(ns, 1);
        double mb = shfl_up_d(ms, 1);
        if (lane == 0) { nb = 0; mb = 0.0; }
        nb += s_n;
        mb += s_m;
        int hit = -1, last = -1;
        Place ph = {}, pl = {};
        for (int e = 0; e < 4; ++e) {
          if (c[e] && nb < end_n && (by_n || w[e] > 0.0)) {
            const Place p = {65535 - (g * 4 * SA_T + 4 * tt + e), c[e], w[e], mb, nb};
            pl = p;
            last = e;
            const double m1 = mb + c[e] * w[e];
            if (hit < 0 && (by_n ? nb + c[e] >= goal_n : past ? m1 > goal_m : m1 >= goal_m)) { hit = e; ph = p; }
          }
          nb += c[e];
          mb += c[e] * w[e];
        }
        const unsigned long long any = __ballot(hit >= 0), some = __ballot(last >= 0);
        const int from = any ? __ffsll((long long)any) - 1 : 63 - __builtin_clzll(some);
        if (lane == from) s_place = any ? ph : pl;
      }
      __syncthreads();
      const Place p = s_place;
      __syncthreads();
      return p;
    };
    long long kept_n = total;
    double kept_m;
    const int k = a.top_k ? a.top_k[b] : 0;
    if (k > 0 && k < kept_n) kept_n = k;
    {
      const Place p = find(true, kept_n, 0.0, false, kept_n);
      kept_m = p.before_m + (double)(kept_n - p.before_n) * p.w;
    }
    const float P = a.top_p ? a.top_p[b] : 1.f;
    if (P < 1.f) {
      const double goal = (double)P * kept_m;
      const Place p = find(false, 0, goal, false, kept_n);
      const double more = ceil((goal - p.before_m) / p.w);
      const long long most = min((long long)p.count, kept_n - p.before_n);
      const long long i = more >= (double)most ? most : more >= 1.0 ? (long long)more : 1;
      kept_n = p.before_n + i;
      kept_m = p.before_m + (double)i * p.w;
    }
    const float u = a.u[row];
    const double goal = (u > 0.f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0) * kept_m;
    const Place p = find(false, 0, goal, true, kept_n);
    const double past = floor((goal - p.before_m) / p.w);
    const long long most = min((long long)p.count, kept_n - p.before_n) - 1;
    key = p.key;
    rank = (unsigned)(past >= (double)most ? most : past > 0.0 ? (long long)past : 0);
    lp = log(p.w / kept_m);
  }
  // the index of the rank-th token that has the value: each wave counts its part of the row, the one that holds it looks again
  const int per = (nvec + SA_W - 1) / SA_W, j0 = wave * per, j1 = min(nvec, j0 + per);
  int num = 0;
  for (int j = j0 + lane; j < j1; j += 64) {
    unsigned e[8];
    load8(j, e);
#pragma unroll
    for (int i = 0; i < 8; ++i) num += key_of<BF>(e[i]) == key;
  }
  for (int off = 32; off >= 1; off >>= 1) num += __shfl_xor(num, off);
  if (lane == 0) s_int[wave] = num;
  __syncthreads();
  unsigned before = 0;
  for (int w = 0; w < wave; ++w) before += s_int[w];
  if (rank < before || rank >= before + (unsigned)num) return;
  for (int j = j0; j < j1; j += 64) {
    unsigned e[8];
    int hits = 0;
    if (j + lane < j1) {
      load8(j + lane, e);
#pragma unroll
      for (int i = 0; i < 8; ++i) hits += key_of<BF>(e[i]) == key;
    }
    int run = hits;
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(run, off);
      if (lane >= off) run += o;
    }
    const unsigned first = before + run - hits;
    if (hits && rank >= first && rank < first + hits) {
      unsigned left = rank - first;
      for (int i = 0; i < 8; ++i)
        if (key_of<BF>(e[i]) == key && left-- == 0) { a.tok[row] = 8 * (j + lane) + i; a.lp[row] = (float)lp; }
    }
    before += __shfl(run, 63);
    if (before > rank) break;
  }
}

struct WalkArgs {
  const int* cu_draft;
  const int* cu_rows;
  const int* draft;
  const int* parents;
  const int* tok;            // [R]
  const float* lp;           // [R]
  int* out_tokens;           // [B][max_spec + 1]
  int* path;                 // [B][max_spec]
  int* len;                  // [B]
  float* out_lp;             // [B][max_spec + 1]
  int* status;
  int B, R, D, max_spec;
};

// One wave a request; counts that do not lie in the rows and drafts refuse the request (one of no rows: padding).
__global__ void __launch_bounds__(64) k_sample_walk(WalkArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const long long d0 = b ? a.cu_draft[b - 1] : 0, d1 = a.cu_draft[b], s0 = b ? a.cu_rows[b - 1] : 0, s1 = a.cu_rows[b];
  int* ot = a.out_tokens + (size_t)b * (a.max_spec + 1);
  int* pt = a.path + (size_t)b * a.max_spec;
  float* ol = a.out_lp + (size_t)b * (a.max_spec + 1);
  for (int i = lane; i <= a.max_spec; i += 64) { ot[i] = -1; ol[i] = 0.f; }
  for (int i = lane; i < a.max_spec; i += 64) pt[i] = -1;
  const long long n = d1 - d0;
  const int whole = ascending(a.cu_rows, a.B - 1);   // (bounds that fall refuse the requests from there on)
  const bool ok = b <= whole && d0 >= 0 && n >= 0 && d1 <= a.D && s0 >= 0 && s1 <= a.R && s1 - s0 == n + 1;
  if (!ok) {
    if (lane == 0) {
      a.len[b] = 0;
      if (a.status && !(b <= whole && n == 0 && s1 == s0)) a.status[0] = 1;
    }
    return;
  }
  __syncthreads();                                   // (one wave: the stores above are out before those below)
  const int pos = walk_tree(
      (int)n, a.max_spec, [&](int row) { return a.tok[s0 + row]; }, [&](int i) { return a.parents[d0 + i]; },
      [&](int i) { return a.draft[d0 + i]; },
      [&](int p, int row, int tok) { if (lane == 0) { ot[p] = tok; ol[p] = a.lp[s0 + row]; } },
      [&](int p, int node) { if (lane == 0) pt[p] = node; });
  if (lane == 0) a.len[b] = pos;
}

}  // namespace

extern "C" {

int64_t cfh_tree_sample_ws_bytes(int n_rows) { return n_rows < 0 ? -1 : (int64_t)n_rows * 8; }

int cfh_tree_sample_accept(const void* logits, long long ld, int V, int n_rows, int is_bf16, const int32_t* cu_draft,
                           const int32_t* cu_sampled, const int32_t* draft_ids, const int32_t* parents, int n_drafts, int B,
                           int max_spec, const float* uniforms, const float* temperature, const int32_t* top_k,
                           const float* top_p, int32_t* out_tokens, int32_t* accepted_path, int32_t* accepted_len,
                           float* out_logprobs, void* ws, int32_t* status, void* stream) {
  if (B == 0) return CFH_OK;
  if (!logits || !cu_draft || !cu_sampled || !uniforms || !temperature || !out_tokens || !accepted_len || !out_logprobs ||
      !ws || (max_spec > 0 && !accepted_path) || (n_drafts > 0 && (!draft_ids || !parents)) || V <= 0 || n_rows <= 0 || B < 0 ||
      max_spec < 0 || n_drafts < 0 || ld < V)
    return CFH_E_INVALID;
  if (V > (1 << 24)) return CFH_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  int* tok = (int*)ws;
  float* lp = (float*)(tok + n_rows);
  SampleArgs s = {(const u16*)logits, ld, V, n_rows, B, cu_sampled, uniforms, temperature, top_k, top_p, tok, lp};
  const bool vec = ld % 8 == 0 && ((uintptr_t)logits & 15) == 0;
  auto launch = [&](auto bf, auto v) {
    hipLaunchKernelGGL((k_sample_rows<bf.value, v.value>), dim3(n_rows), dim3(SA_T), 0, st, s);
  };
  if (is_bf16) vec ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
  else vec ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
  CFH_LAUNCH_CHECK();
  WalkArgs w = {cu_draft, cu_sampled, draft_ids, parents, tok, lp, out_tokens, accepted_path, accepted_len, out_logprobs,
                status, B, n_rows, n_drafts, max_spec};
  hipLaunchKernelGGL(k_sample_walk, dim3(B), dim3(64), 0, st, w);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

}  // extern "C"
