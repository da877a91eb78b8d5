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
#include "cfh_scan.h"
#include "cfh_seq.h"
#include "cfh_walk.h"

namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));

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
  int parts;                 // of a row, counted on their own before (1: none)
  unsigned* part_counts;     // [R][parts][PART_WORDS]
  int* part_high;            // [R][parts]
  int* part_masked;          // [R][parts]
};
struct Range { int from, to; };
__device__ __forceinline__ Range part_range(int vectors, int part, int parts) {
  const int per = (vectors + parts - 1) / parts;
  return {min(part * per, vectors), min((part + 1) * per, vectors)};
}
constexpr int PART_WORDS = 32768;   // a part's counts: those of k_sample_rows with 16 bits a value

// Order position o of a 16-bit value: 0 the largest NaN pattern of a positive sign, then descending, +0 at 32,767, -0 behind it.
__device__ __forceinline__ int raw_of(int o) { return o < 0x8000 ? 0x7fff - o : o; }
template <bool BF>
__device__ __forceinline__ double value_of(int o) {
  const unsigned x = (unsigned)raw_of(o);
  if constexpr (BF) return (double)__uint_as_float(x << 16);
  else return (double)__builtin_bit_cast(_Float16, (u16)x);
}
// Positions of numbers above -inf: the first and the last.
template <bool BF> constexpr int O_FIRST = 0x7fff - (BF ? 0x7f80 : 0x7c00);
template <bool BF> constexpr int O_LAST = 0x8000 + (BF ? 0x7f80 : 0x7c00) - 1;

// 2^t in 64 bits, t <= 0: t = q / 32 + g, 2^(q / 32) by exponent and a table of 32, 2^g by the exponential series to the 6th power
// (its next term is below 4e-18 for |g| <= 1 / 64).  0 from 2^-1100 on.
__device__ __forceinline__ double pow2(const double* table, double t) {
  t = fmax(t, -1100.0);
  const double q = rint(t * 32.0), z = fma(q, -1.0 / 32.0, t) * 0.693147180559945309417;
  double p = 1.0 / 720.0;
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, 1.0 / 24.0);
  p = fma(p, z, 1.0 / 6.0);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  const int i = (int)q;
  return ldexp(table[i & 31] * p, i >> 5);
}
// The table: 2^(i / 32), the series to the 20th power.
__device__ __forceinline__ double pow2_of_32(int i) {
  const double z = (double)i * (0.693147180559945309417 / 32.0);
  double p = 1.0;
  for (int n = 20; n >= 1; --n) p = fma(p * z, 1.0 / (double)n, 1.0);
  return p;
}

// The place where a running count or sum passes a goal: the value, and what stands before it.
struct Place { int o; unsigned count; double w, before_m; int before_n; };

// Eight logits from 8 j on.
template <bool VEC>
__device__ __forceinline__ v4u load8(const u16* x, int j) {
  if constexpr (VEC) return *(const v4u*)(x + (size_t)8 * j);
  v4u w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = x[(size_t)8 * j + 2 * i] | (unsigned)x[(size_t)8 * j + 2 * i + 1] << 16;
  return w;
}
// f(j, eight logits) for this thread's vectors j of from .. to - 1, AHEAD of them in flight; meanwhile() while the first arrive.
template <bool VEC, int T, typename F, typename G>
__device__ __forceinline__ void each_of(const u16* x, int from, int to, F f, G meanwhile) {
  constexpr int AHEAD = VEC ? 8 : 2;
  if (from >= to) return meanwhile();
  v4u ring[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) ring[i] = load8<VEC>(x, min(from + (int)threadIdx.x + i * T, to - 1));
  meanwhile();
#pragma unroll 1
  for (int j = from + threadIdx.x; j < to; j += AHEAD * T) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const v4u w = ring[i];
      ring[i] = load8<VEC>(x, min(j + (i + AHEAD) * T, to - 1));
      if (j + i * T < to) f(j + i * T, w);
    }
  }
}
template <bool VEC, int T, typename F>
__device__ __forceinline__ void each_of(const u16* x, int from, int to, F f) {
  each_of<VEC, T>(x, from, to, f, []() {});
}
// Whether a wave has one and the same value everywhere (a mask): counted one by one, each would wait for the others.
__device__ __forceinline__ bool one_value(v4u w, unsigned& v) {
  const unsigned first = __builtin_amdgcn_readfirstlane(w[0]);
  v = first & 0xffffu;
  return __ballot(w[0] != first) == 0 && first >> 16 == v && __ballot(w[1] != first || w[2] != first || w[3] != first) == 0;
}
// The likely mask of a row: the lowest of 64 logits spread over it, where two have it and it is below 0 (NONE: there is none).
// Tokens of that value are counted apart, in 32 bits: lanes that added to one count would wait for each other, and its count
// would leave the narrow fields (248,320 logits, every second -inf: 41 rows in 45 us, 378 without).  Any value is as right.
constexpr unsigned NONE = 0x10000;
__device__ __forceinline__ unsigned sample_of(const u16* x, int V) { return x[(long long)(threadIdx.x & 63) * (V - 1) / 63]; }
template <bool BF>
__device__ __forceinline__ unsigned mask_of_sample(unsigned v) {
  const unsigned lowest = wave_largest(v <= (BF ? 0xff80u : 0xfc00u) ? v : 0);   // (negative patterns ascend as values fall; no NaN)
  return lowest > 0x8000u && __builtin_popcountll(__ballot(v == lowest)) > 1 ? lowest : NONE;
}
// The narrow counts of the vectors from .. to - 1 and of the n_tail logits behind them (few operations a logit: they are what
// counting costs), but for those of value h, the likely mask: to the thread's n_h.  -> the thread's largest pattern as a signed number: the
// largest number, where there is a positive one
template <bool BF, bool VEC, int T, int BITS>
__device__ __forceinline__ int count_narrow(const u16* x, int from, int to, int n_tail, unsigned* hist, unsigned sample, unsigned& h,
                                            int& n_h) {
  constexpr int WORDS = BITS == 8 ? 1 << 14 : 1 << 15;
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 most = {-32768, -32768};
  auto add = [&](unsigned v, unsigned n) __attribute__((always_inline)) {
    atomicAdd(&hist[v & (WORDS - 1)], BITS == 16 ? n * ((v >> 15) * 0xffffu + 1) : n << ((v >> 11) & 24));
  };
  n_h = 0;
  each_of<VEC, T>(x, from, to, [&](int, v4u w) __attribute__((always_inline)) {
    bool masked = false;
    if (h != NONE) {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 low = {0, 0};                            // the lowest, as there is one below 0
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned u = w[i];
        low = __builtin_elementwise_max(low, __builtin_bit_cast(u16x2, u));
      }
      masked = low[0] >= h || low[1] >= h;
    }
    unsigned v;
    if (one_value(w, v)) {
      const unsigned long long on = __ballot(true);
      if (v == h) n_h += 8;
      else if ((threadIdx.x & 63) == __builtin_ctzll(on)) add(v, 8u * __builtin_popcountll(on));
    } else if (__ballot(masked)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned v = w[i >> 1] >> (16 * (i & 1)) & 0xffffu;
        if (v == h) ++n_h;
        else add(v, 1u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        add(w[i] & 0xffffu, 1u);
        add(w[i] >> 16, 1u);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = w[i];
      most = __builtin_elementwise_max(most, __builtin_bit_cast(s16x2, u));
    }
  }, [&]() __attribute__((always_inline)) { h = mask_of_sample<BF>(sample); });
  int high = max((int)most[0], (int)most[1]);
  if ((int)threadIdx.x < n_tail) {
    const unsigned v = x[(size_t)8 * to + threadIdx.x];
    if (v == h) ++n_h;
    else add(v, 1u);
    high = max(high, (int)(short)v);
  }
  return high;
}
// The largest of v over W waves.
template <int W>
__device__ __forceinline__ int over_all(int v, int* s_int) {
  for (int off = 32; off >= 1; off >>= 1) v = max(v, __shfl_xor(v, off));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_int[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < W; ++w) v = max(v, s_int[w]);
  return v;
}
// The sum of v over W waves.
template <int W>
__device__ __forceinline__ int sum_over_all(int v, int* s_int) {
  v = scan64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s_int[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < W; ++w) v += s_int[w];
  return v;
}

// Few long rows leave most CUs idle, and a CU counts 64 logits in 10 cycles: then each row is counted in parts, a workgroup a
// part, and k_sample_rows adds the parts' counts up (6 rows of 248,320 in 4 parts: 10 us here and 15.7 there, 31 in one).
template <bool BF, bool VEC>
__global__ void __launch_bounds__(1024, 4) k_sample_parts(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned hist[PART_WORDS];
  __shared__ int s_int[16];
  const int row = blockIdx.x, part = blockIdx.y, t = threadIdx.x, whole = a.V / 8;
  const u16* x = a.logits + (size_t)row * a.ld;
  for (int i = t; i < PART_WORDS / 4; i += 1024) ((uint4*)hist)[i] = make_uint4(0, 0, 0, 0);
  const unsigned sample = sample_of(x, a.V);
  __syncthreads();
  const Range r = part_range(whole, part, a.parts);
  unsigned h;
  int masked;
  int high = count_narrow<BF, VEC, 1024, 16>(x, r.from, r.to, part == a.parts - 1 ? a.V % 8 : 0, hist, sample, h, masked);
  high = over_all<16>(high, s_int);                  // (and the counts are whole)
  masked = sum_over_all<16>(masked, s_int);
  const size_t at = (size_t)row * a.parts + part;
  uint4* out = (uint4*)(a.part_counts + at * PART_WORDS);
  for (int i = t; i < PART_WORDS / 4; i += 1024) out[i] = ((uint4*)hist)[i];
  if (t == 0) { a.part_high[at] = high; a.part_masked[at] = masked; }
}

// One workgroup of T threads a row.  BITS: a value's count in LDS, 32 / BITS values a word (the low bits of the value name the
// word, the high ones the field).  The counts are right where they add up to V: one that leaves its BITS takes 2^BITS from its own
// for each 1 that it adds to the next, so that the sum only falls.  Then (a constant row, values that crowd) half of them
// are counted at a time, in twice the bits, which V cannot leave.  8 bits (64 KB) are for many rows of V < 65,536, 16 bits (128 KB)
// for all others (the rule and what both cost stand at the launch).  The row is read again, from the caches, for the drawn token's index.
// What bounds a row of 248,320 bf16 logits on its CU: 17 us of counting (an LDS atomic a logit, a wave's 64 in 10 cycles), 2.2 the
// cells (fp16: 4.2, more values are in use), 1.5 a search (one wave's latency), 4 the index.  1,968 rows of 32,000: 11 us a row and
// CU in fp16, 1.5 TB/s; the stages of two rows overlap there, and the searches' latency and the weights of many values
// are what remains.
template <bool BF, bool VEC, int T, int BITS>
__global__ void __launch_bounds__(T, 4) k_sample_rows(SampleArgs a) {
  constexpr int W = T / 64, LOG = BITS == 8 ? 14 : 15, WORDS = 1 << LOG;
  constexpr int N = 8, GROUPS = 65536 / (N * T), CELLS = GROUPS * W;   // a cell: a wave's 64 x N values of a group, in the order
  static_assert(CELLS == 128, "a lane searches two cells");
  __shared__ __attribute__((aligned(16))) unsigned hist[WORDS];
  __shared__ double cell_m[CELLS];                   // sums of the cells, then up to and with each
  __shared__ int cell_n[CELLS];
  constexpr int MANT = BF ? 7 : 10;                  // bits of a binade's values
  __shared__ double table[32], ratio[0x8000 >> MANT];
  __shared__ int s_int[W], s_masked[W];
  __shared__ Place s_place;
  __shared__ int s_half[3], s_cell, s_rank;
  __shared__ double s_kept;
  const int row = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const bool in_parts = T == 1024 && a.parts > 1;
  if (!in_parts)
    for (int i = t; i < WORDS / 4; i += T) ((uint4*)hist)[i] = make_uint4(0, 0, 0, 0);   // (while the bounds arrive)
  const u16* x = a.logits + (size_t)row * a.ld;
  const int V = a.V;
  const unsigned sample = sample_of(x, V);
  // request b > 0 has the rows cu_rows[b - 1] .. cu_rows[b], the first those below cu_rows[0]
  int b = 0;
  if (row >= a.cu_rows[0]) {
    const Seq f = find_seq(a.cu_rows, a.B - 1, nullptr, [&](int, int c) { return c <= row; });
    b = f.s >= 0 && row < f.c1 ? f.s + 1 : -1;
  }
  auto give = [&](int tok, float lp) __attribute__((always_inline)) { a.tok[row] = tok; a.lp[row] = lp; };
  if (b < 0) {                                       // a row of no request
    if (t == 0) give(-1, 0.f);
    return;
  }
  const float Tf = a.temp[b], u = a.u[row], P = a.top_p ? a.top_p[b] : 1.f;   // (here, so that they arrive during the count)
  const int K = a.top_k ? a.top_k[b] : 0;
  const int whole = V / 8;                           // vectors of eight; the row's last logits are one more, from `tail`
  v4u tail = {};                                     // (the last logit again behind the row's end)
  if (V % 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) tail[i] = x[min(8 * whole + 2 * i, V - 1)] | (unsigned)x[min(8 * whole + 2 * i + 1, V - 1)] << 16;
  }
  bool wide = false;
  unsigned h = NONE;                                 // the value that hist does not hold, and its tokens (a thread's, then the row's)
  int n_h = 0;
  int half = 0;                                      // (wide) the top bit of the values whose counts hist holds
  auto count_half = [&](int top_bit) __attribute__((always_inline)) {
    half = top_bit;
    for (int i = t; i < WORDS / 4; i += T) ((uint4*)hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto add_wide = [&](unsigned v, unsigned n) __attribute__((always_inline)) {
      if (v == 0x8000u) v = 0;                       // -0 counts as +0
      if ((int)(v >> 15) == top_bit) atomicAdd(&hist[v & (WORDS - 1)], n << (((v & 0x7fffu) >> LOG) * (2 * BITS & 31)));
    };
#pragma unroll 1
    for (int j = t; j < whole; j += T) {
      const v4u w = load8<VEC>(x, j);
      unsigned v;
      if (one_value(w, v)) {
        const unsigned long long on = __ballot(true);
        if (lane == __builtin_ctzll(on)) add_wide(v, 8u * __builtin_popcountll(on));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) add_wide(w[i >> 1] >> (16 * (i & 1)) & 0xffffu, 1u);
      }
    }
    if (t < V % 8) add_wide(x[8 * whole + t], 1u);
    __syncthreads();
  };
  // counts of this lane's N values of a cell (the same one in the whole wave), 0 for those that are no numbers above -inf
  auto counts_of = [&](int cell, unsigned (&c)[N]) __attribute__((always_inline)) {
    const bool pos = cell < CELLS / 2;
    const int o0 = cell * 64 * N, raw0 = pos ? 0x7fff - o0 - (64 * N - 1) : o0;      // its first position, its lowest pattern
    const uint4* w = (const uint4*)(hist + (raw0 & (WORDS - 1)) + (pos ? 63 - lane : lane) * N);
    const uint4 w0 = w[0], w1 = w[1];
    const unsigned v[N] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
    const int bits = wide ? 2 * BITS : BITS, field = (wide ? raw0 & 0x7fff : raw0) >> LOG;
    const int shift = bits == 32 ? 0 : field * bits;
    const unsigned mask = bits == 32 ? ~0u : (1u << bits) - 1;
    if (pos) {
#pragma unroll
      for (int e = 0; e < N; ++e) c[e] = v[N - 1 - e] >> shift & mask;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) c[e] = v[e] >> shift & mask;
    }
    if (h - o0 < 64u * N) {                          // (a value below 0 is its own position)
#pragma unroll
      for (int e = 0; e < N; ++e) c[e] += (int)h == o0 + N * lane + e ? n_h : 0;
    }
    if (o0 < O_FIRST<BF> || o0 + 64 * N - 1 > O_LAST<BF>) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int o = o0 + N * lane + e;
        c[e] = o >= O_FIRST<BF> && o <= O_LAST<BF> ? c[e] : 0;
      }
    }
  };
  int top = -1;
  double m = 0.0, rate = 0.0;
  // f(e, weight) for the values at order positions o .. o + N - 1, o a multiple of N: they lie in one binade, a step apart, so that
  // each is the one before times 2^(-step / T).  1 at the largest (none lies above it), 0 beside an infinite one.
  auto weights = [&](int o, auto f) __attribute__((always_inline)) {
    const int base = max(o, top);
    double x = pow2(table, base == top ? 0.0 : isinf(m) ? -INFINITY : (value_of<BF>(base) - m) * rate);
    const double r = ratio[(raw_of(base) & 0x7fff) >> MANT];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      f(e, x);
      x = o + e >= top ? x * r : x;
    }
  };
  // the weight of the tokens counted there: where the whole wave lies below the largest, a polynomial in the step's ratio
  auto weight_of = [&](int o, const unsigned (&c)[N]) __attribute__((always_inline)) {
    double s = 0.0;
    if (__ballot(o < top)) {
      weights(o, [&](int e, double w) __attribute__((always_inline)) { s = fma((double)c[e], w, s); });
    } else {
      const double r = ratio[(raw_of(o) & 0x7fff) >> MANT];
#pragma unroll
      for (int e = N - 1; e >= 0; --e) s = fma(s, r, (double)c[e]);
      s *= pow2(table, isinf(m) ? o == top ? 0.0 : -INFINITY : (value_of<BF>(o) - m) * rate);
    }
    return s;
  };
  // All cells from the narrow counts: each word is read once, and most are 0 in a whole wave.  (The positive values' order runs
  // against their words'.)  -> this thread's tokens, numbers or not
  auto cells_narrow = [&]() __attribute__((always_inline)) {
    constexpr int F = 32 / BITS, BLOCKS = WORDS / (N * T);
    int all = 0;
#pragma unroll 2
    for (int k = 0; k < BLOCKS; ++k) {
      const uint4 q0 = ((const uint4*)hist)[2 * (k * T + t)], q1 = ((const uint4*)hist)[2 * (k * T + t) + 1];
      const unsigned q[N] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
      if (!__ballot((q[0] | q[1] | q[2] | q[3] | q[4] | q[5] | q[6] | q[7]) != 0)) continue;
      int cn[F] = {};
      double cs[F] = {};
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const bool pos = f < F / 2;
        unsigned c[N];
        int n = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          c[e] = q[pos ? N - 1 - e : e] >> (f * BITS) & ((1u << BITS) - 1);
          n += (int)c[e];
        }
        if (!__ballot(n != 0)) continue;
        all += n;
        const int at = f * BLOCKS + k, raw = N * (at * T + t), o = pos ? 0x7fff - (N - 1) - raw : raw;
        if (o < O_FIRST<BF> || o + N - 1 > O_LAST<BF>) {
          n = 0;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            c[e] = o + e >= O_FIRST<BF> && o + e <= O_LAST<BF> ? c[e] : 0;
            n += (int)c[e];
          }
        }
        cn[f] = n;
        if (n) cs[f] = weight_of(o, c);
      }
      // the F cells' sums at once: halves and rows of lanes exchanged, so that a cell's are in lanes 64 / F f .. + 15
      if constexpr (F == 4) {
        swap_add<32>(cn[0], cn[2]); swap_add<32>(cn[1], cn[3]); swap_add<16>(cn[0], cn[1]);
        swap_add<32>(cs[0], cs[2]); swap_add<32>(cs[1], cs[3]); swap_add<16>(cs[0], cs[1]);
      } else {
        swap_add<32>(cn[0], cn[1]); swap_add<16>(cn[0], 0);
        swap_add<32>(cs[0], cs[1]); swap_add<16>(cs[0], 0.0);
      }
      cn[0] = row_scan(cn[0]);
      cs[0] = row_scan(cs[0]);
      const int f = lane / (64 / F), at = f * BLOCKS + k;
      const int cell = f < F / 2 ? (GROUPS / 2 - 1 - at) * W + W - 1 - wave : at * W + wave;
      if (lane % (64 / F) == 15) { cell_n[cell] = cn[0]; cell_m[cell] = cs[0]; }
    }
    return all;
  };
  // the cells of groups g0 .. g1 - 1
  auto cells = [&](int g0, int g1) __attribute__((always_inline)) {
#pragma unroll 1
    for (int g = g0; g < g1; ++g) {
      const int cell = __builtin_amdgcn_readfirstlane(g * W + wave);
      unsigned c[N];
      counts_of(cell, c);
      int n = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) n += (int)c[e];
      double s = n ? weight_of(64 * N * cell + N * lane, c) : 0.0;
      n = scan64(n);
      s = scan64(s);
      if (lane == 63) { cell_n[cell] = n; cell_m[cell] = s; }
    }
  };

  if (t < 32) table[t] = pow2_of_32(t);
  if (t < CELLS) { cell_n[t] = 0; cell_m[t] = 0.0; }
  __syncthreads();
  int high = -32768;
  if (in_parts) {
    constexpr int PER = WORDS / (4 * T);
    const v4u* part = (const v4u*)(a.part_counts + (size_t)row * a.parts * PART_WORDS) + t;
    v4u sum[PER] = {};
#pragma unroll 2
    for (int p = 0; p < a.parts; ++p) {
#pragma unroll
      for (int k = 0; k < PER; ++k) sum[k] += part[(size_t)p * (PART_WORDS / 4) + k * T];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) ((v4u*)hist)[k * T + t] = sum[k];
    if (t < a.parts) {
      high = a.part_high[(size_t)row * a.parts + t];
      n_h = a.part_masked[(size_t)row * a.parts + t];
    }
    h = mask_of_sample<BF>(sample);
  } else {
    high = count_narrow<BF, VEC, T, BITS>(x, 0, whole, V % 8, hist, sample, h, n_h);
  }
  const unsigned masked = h;
  constexpr int INF = BF ? 0x7f80 : 0x7c00;
  high = over_all<W>(high, s_int);
  if (t == 0) {                                      // -0 counts as +0
    const unsigned w = hist[0], at = (0x8000 >> LOG) * BITS, c = w >> at & ((1u << BITS) - 1);
    hist[0] = w - (c << at) + c;
  }
  if (high < 0 || high > INF) {                      // no positive pattern, or a positive NaN: the numbers alone, in their order
    int best = -65536;
    auto look = [&](int v) __attribute__((always_inline)) {
      const int o = v < 0x8000 ? 0x7fff - v : v == 0x8000 ? 0x7fff : v;
      if (o >= O_FIRST<BF> && o <= O_LAST<BF>) best = max(best, -o);
    };
    each_of<VEC, T>(x, 0, whole, [&](int, v4u w) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) look(w[i >> 1] >> (16 * (i & 1)) & 0xffff);
    });
    if (t < V % 8) look(x[8 * whole + t]);
    best = over_all<W>(best, s_int);
    top = best > -65536 ? -best : -1;
  } else {
    top = 0x7fff - high;
  }
  __syncthreads();
  if (top < 0) {                                     // nothing to draw from
    if (t == 0) give(-1, 0.f);
    return;
  }
  const bool greedy = !(Tf > 0.f);
  m = value_of<BF>(top);
  rate = greedy ? 0.0 : 1.4426950408889634074 / (double)Tf;
  if (t < (0x8000 >> MANT)) {                        // 2^(-step / T) of every binade
    const int o = 0x7fff - (t << MANT);
    ratio[t] = isinf(m) ? 0.0 : pow2(table, (value_of<BF>(o) - value_of<BF>(o - 1)) * rate);
  }
  __syncthreads();
  Place p = {top, 0, 1.0, 0.0, 0};                   // (as a greedy request's: the first of the largest)
  int rank = 0;
  double kept_m = 1.0;
  if (!greedy) {
    int all = scan64(cells_narrow() + n_h);
    n_h = scan64(n_h);
    if (lane == 63) { s_int[wave] = all; s_masked[wave] = n_h; }
    __syncthreads();
    all = n_h = 0;
    for (int w = 0; w < W; ++w) { all += s_int[w]; n_h += s_masked[w]; }
    if (all != V) {
      wide = true;
      h = NONE;                                      // (counted with the others)
      for (int top_bit = 1; top_bit >= 0; --top_bit) {
        __syncthreads();
        count_half(top_bit);
        cells(top_bit ? GROUPS / 2 : 0, top_bit ? GROUPS : GROUPS / 2);
      }
      __syncthreads();
    }
    // One wave finds the places (where counts are wide, the others help it to the half that it looks at): up to three searches,
    // each for the first value at which the running sum (of counts: by_n) reaches a goal, or passes it (the draw), or the last
    // one of any weight where rounding leaves none, among the first kept_n tokens: the cut of k, the cut of P, the draw.
    if (wave == 0 || wide) {
      int n0 = cell_n[2 * lane], n1 = cell_n[2 * lane + 1];
      double s0 = cell_m[2 * lane], s1 = cell_m[2 * lane + 1];
      const int o_h = (int)h;
      if (o_h >= 0x8000 && o_h <= O_LAST<BF> && o_h / (128 * N) == lane) {   // (-inf is no token)
        const double sum = (double)n_h * pow2(table, o_h == top ? 0.0 : isinf(m) ? -INFINITY : (value_of<BF>(o_h) - m) * rate);
        const bool second = o_h / (64 * N) % 2;
        n0 += second ? 0 : n_h;
        n1 += second ? n_h : 0;
        s0 += second ? 0.0 : sum;
        s1 += second ? sum : 0.0;
      }
      n1 += n0;
      s1 += s0;
      const int up_n = scan64(n1), from_n = up_n - n1;
      const double up_m = scan64(s1);
      double from_m = __shfl_up(up_m, 1);            // (as the lanes before add up, to the bit)
      if (lane == 0) from_m = 0.0;
      const int upto_n[3] = {from_n, from_n + n0, up_n};          // up to the lane's two cells, between them and behind them
      const double upto_m[3] = {from_m, from_m + s0, up_m};
      int kept_n = __builtin_amdgcn_readlane(up_n, 63);
      kept_m = from_lane(up_m, 63);
#pragma unroll 1
      for (int stage = 0; stage < 3; ++stage) {
        const bool by_n = stage == 0, past = stage == 2;
        double goal = 0.0, below = 0.0;              // reached by a sum above `below`
        if (by_n) {
          if (K < 1 || K >= kept_n) continue;
          kept_n = K;
        } else if (!past) {
          if (!(P < 1.f)) continue;
          goal = fmax((double)P * kept_m, 0x1p-60);  // (the first token at least: it weighs 1)
          below = __longlong_as_double(__double_as_longlong(goal) - 1);
        } else {
          below = goal = (u > 0.f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0) * kept_m;
        }
        // the first of the places that count and reach it, else the last that counts (a bit a lane)
        auto choose = [](unsigned long long counts, unsigned long long reaches) __attribute__((always_inline)) {
          reaches &= counts;
          return reaches ? __builtin_ctzll(reaches) : counts ? 63 - __builtin_clzll(counts) : 0;
        };
        unsigned long long in[2], reach[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          in[i] = __ballot(upto_n[i + 1] > upto_n[i] && upto_n[i] < kept_n && (by_n || upto_m[i + 1] > upto_m[i]));
          reach[i] = in[i] & __ballot(by_n ? upto_n[i + 1] >= kept_n : upto_m[i + 1] > below);
        }
        const int at = choose(in[0] | in[1], reach[0] | reach[1]);
        const int i = (reach[0] | reach[1]) ? !(reach[0] >> at & 1) : (int)(in[1] >> at & 1);
        if (wide) {                                  // (wave 0's: kept_n and the rest are its own)
          if (t == 0) s_half[stage] = at >= 32;
          __syncthreads();
          if (half != s_half[stage]) count_half(!half);
          if (wave) continue;
        }
        const int cell = 2 * at + i, o = 64 * N * cell + N * lane;
        unsigned c[N];
        counts_of(cell, c);
        int ns = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) ns += (int)c[e];
        double w[N], ss = 0.0;
        if (64 * N * cell < top) {
          weights(o, [&](int e, double x) __attribute__((always_inline)) { w[e] = x; });
        } else {
          const double r = ratio[(raw_of(o) & 0x7fff) >> MANT];
          w[0] = pow2(table, isinf(m) ? o == top ? 0.0 : -INFINITY : (value_of<BF>(o) - m) * rate);
#pragma unroll
          for (int e = 1; e < N; ++e) w[e] = w[e - 1] * r;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          w[e] = c[e] ? w[e] : 0.0;
          ss = fma((double)c[e], w[e], ss);
        }
        const int nb = scan64(ns) - ns + __builtin_amdgcn_readlane(i ? upto_n[1] : upto_n[0], at);
        double mb = __shfl_up(scan64(ss), 1);
        if (lane == 0) mb = 0.0;
        mb += from_lane(i ? upto_m[1] : upto_m[0], at);
        // the lane, then its N values a lane each
        const bool counts = ns > 0 && nb < kept_n && (by_n || ss > 0.0);
        const int from = choose(__ballot(counts), __ballot(by_n ? nb + ns >= kept_n : mb + ss > below));
        unsigned ce = 0;
        double we = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const unsigned x = __builtin_amdgcn_readlane(c[e], from);
          const double y = from_lane(w[e], from);
          ce = lane == e ? x : ce;
          we = lane == e ? y : we;
        }
        const int n1 = __builtin_amdgcn_readlane(nb, from) + row_scan((int)ce), n0 = n1 - (int)ce;
        const double sum = row_scan((double)ce * we), m0 = from_lane(mb, from), m1 = m0 + sum;
        const double before = m0 + moved<DPP_SHR1, 0xf>(sum);
        const int pick = choose(__ballot(ce && n0 < kept_n && (by_n || we > 0.0)), __ballot(by_n ? n1 >= kept_n : m1 > below));
        p.o = 64 * N * cell + N * from + pick;
        p.count = __builtin_amdgcn_readlane(ce, pick);
        p.w = from_lane(we, pick);
        p.before_m = from_lane(before, pick);
        p.before_n = __builtin_amdgcn_readlane(n0, pick);
        const int most = min((int)p.count, kept_n - p.before_n);
        if (by_n) {
          kept_m = p.before_m + (double)most * p.w;
        } else if (!past) {
          const double more = ceil((goal - p.before_m) / p.w);
          const int i = more >= (double)most ? most : more >= 1.0 ? (int)more : 1;
          kept_n = p.before_n + i;
          kept_m = p.before_m + (double)i * p.w;
        } else {
          const double over = floor((goal - p.before_m) / p.w);
          rank = over >= (double)(most - 1) ? most - 1 : over > 0.0 ? (int)over : 0;
        }
      }
      if (t == 0) { s_place = p; s_rank = rank; s_kept = kept_m; }
    }
    __syncthreads();
    p = s_place;
    rank = s_rank;
    kept_m = s_kept;
    __syncthreads();
  }

  // The index of the rank-th token of that value: where it is alone, the one; else how many each 64 vectors hold, in
  // order, in the counts' place (2^24 tokens: 32,768 words and one for the tail), and those 64 again.
  const unsigned raw = (unsigned)raw_of(p.o), both = raw | raw << 16, care = p.o == 0x7fff ? 0x7fff7fffu : ~0u;   // (0 and -0)
  auto mask_of = [&](v4u w) __attribute__((always_inline)) {   // bit i: the i-th of eight has it
    unsigned hits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) hits |= (unsigned)(((w[i >> 1] ^ both) & care) >> (16 * (i & 1)) << 16 == 0) << i;
    return hits;
  };
  auto any_of = [&](v4u w) __attribute__((always_inline)) {    // whether one of eight has it: a half of the least is 0
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 least = {0xffff, 0xffff};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = (w[i] ^ both) & care;
      least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, u));
    }
    return least[0] == 0 || least[1] == 0;
  };
  Range in = {0, whole};
  bool with_tail = V % 8 != 0, alone = p.count == 1;
  if (in_parts) {                                    // the part that has it (a part holds fewer than 2^16 logits)
    int n = 0;
    if (lane < a.parts) {
      const unsigned w = a.part_counts[((size_t)row * a.parts + lane) * PART_WORDS + (raw & (PART_WORDS - 1))];
      n = raw == masked ? a.part_masked[(size_t)row * a.parts + lane]
                   : p.o == 0x7fff ? (w & 0xffffu) + (w >> 16) : w >> (raw >> 15) * 16 & 0xffffu;
    }
    const int upto = scan64(n), part = __builtin_ctzll(__ballot(upto > rank));
    rank -= __builtin_amdgcn_readlane(upto - n, part);
    alone = __builtin_amdgcn_readlane(n, part) == 1;
    in = part_range(whole, part, a.parts);
    with_tail = with_tail && part == a.parts - 1;
  }
  const int steps = (in.to - in.from + 63) / 64;     // (the tail: step `steps`)
  auto found = [&](int tok) __attribute__((always_inline)) { give(tok, (float)log(p.w / kept_m)); };
  const unsigned tail_hits = with_tail ? mask_of(tail) & ((1u << V % 8) - 1) : 0;
  if (alone) {
    each_of<VEC, T>(x, in.from, in.to, [&](int j, v4u w) __attribute__((always_inline)) {
      if (any_of(w)) found(8 * j + __builtin_ctz(mask_of(w)));
    });
    if (t == 0 && tail_hits) found(8 * whole + __builtin_ctz(tail_hits));
    return;
  }
  each_of<VEC, T>(x, in.from, in.to, [&](int j, v4u w) __attribute__((always_inline)) {
    int n = 0;
    if (__ballot(any_of(w))) {
      const unsigned hits = mask_of(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) n += __builtin_popcountll(__ballot(hits >> i & 1));
    }
    if (lane == 0) hist[(j - in.from) >> 6] = n;
  });
  __syncthreads();
  const int per = (steps + T - 1) / T;
  int mine = 0;
  for (int i = t * per; i < min(steps, (t + 1) * per); ++i) mine += hist[i];
  int upto = scan64(mine);
  if (lane == 63) s_int[wave] = upto;
  if (t == 0) { s_cell = steps; s_rank = -1; }
  __syncthreads();
  int all_steps = 0;
  for (int w = 0; w < W; ++w) {
    if (w < wave) upto += s_int[w];
    all_steps += s_int[w];
  }
  if (rank < upto && rank >= upto - mine) {
    int left = rank - (upto - mine), i = t * per;
    while (left >= (int)hist[i]) left -= hist[i++];
    s_cell = i;
    s_rank = left;
  }
  __syncthreads();
  if (wave) return;
  const bool last = s_cell == steps;                 // none of the whole vectors: in the tail
  const int j = in.from + s_cell * 64 + lane;
  const unsigned hits = last ? lane == 0 ? tail_hits : 0 : j < in.to ? mask_of(load8<VEC>(x, j)) : 0;
  const int own = __builtin_popcount(hits);
  int left = (last ? rank - all_steps : s_rank) - (scan64(own) - own);
  if (left < 0 || left >= own) return;
  unsigned rest = hits;
  for (; left > 0; --left) rest &= rest - 1;
  found(8 * (last ? whole : j) + __builtin_ctz(rest));
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

constexpr int WALK_LDS = 1024;   // drafts of a request staged in LDS

// One wave a request: round trips, the walk itself in LDS (one request 3.8 us, 48 5.6).  Counts that do not lie in the rows and
// drafts refuse the request (one of no rows: padding).
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
  __shared__ int s_par[WALK_LDS], s_draft[WALK_LDS], s_tok[WALK_LDS + 1];
  const bool lds = n <= WALK_LDS;
  if (lds)
    for (int i = lane; i <= n; i += 64) {
      s_tok[i] = a.tok[s0 + i];
      if (i < n) { s_par[i] = a.parents[d0 + i]; s_draft[i] = a.draft[d0 + i]; }
    }
  __syncthreads();                                   // (one wave: the stores above are out before those below)
  const int pos = walk_tree(
      (int)n, a.max_spec, [&](int row) { return lds ? s_tok[row] : a.tok[s0 + row]; },
      [&](int i) { return lds ? s_par[i] : a.parents[d0 + i]; }, [&](int i) { return lds ? s_draft[i] : a.draft[d0 + i]; },
      [&](int p, int row, int tok) { if (lane == 0) { ot[p] = tok; ol[p] = a.lp[s0 + row]; } },
      [&](int p, int node) { if (lane == 0) pt[p] = node; });
  if (lane == 0) a.len[b] = pos;
}

// How many parts a row is counted in.  The whole call over 248,320 logits: 6 rows 34.8 us in one part, 31.4 in 2, 29.3 in 4, 34.6
// in 8 (a part's counts are 128 KB to read for the row's CU, 1.4 us).  One part and 4 by rows, bf16 with k and P (deviation 2.5
// around 0; 0.7 around -6): 6 rows 37.8 and 32.4 us; 61.0 and 52.2.  24 rows 38.6 and 33.4; 62.5 and 54.5.  36 rows 39.9 and 37.9; 63.5
// and 57.5.  64 rows 39.7 and 39.9; 63.9 and 59.4.  82 rows 42.0 and 49.1; 65.3 and 69.4.  (So parts lose above 64 rows, and 25 to
// 64 would gain 0 to 6 us by them.)  A part's counts stay below 2^16.
int parts_of(int n_rows, int V) {
  const int parts = max(4, V / 65528 + 1);
  return n_rows <= 24 && V >= 65536 && parts <= 8 ? parts : 1;
}

}  // namespace

extern "C" {

int64_t cfh_tree_sample_ws_bytes(int n_rows, int V) {
  if (n_rows < 0 || V <= 0) return -1;
  const int parts = parts_of(n_rows, V);
  return ((int64_t)n_rows * 8 + 15) / 16 * 16 + (parts > 1 ? (int64_t)n_rows * parts * (PART_WORDS * 4 + 8) : 0);
}

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
  const int parts = parts_of(n_rows, V);
  unsigned* part_counts = (unsigned*)((char*)ws + ((size_t)n_rows * 8 + 15) / 16 * 16);
  SampleArgs s = {(const u16*)logits, ld, V, n_rows, B, cu_sampled, uniforms, temperature, top_k, top_p, tok, lp, parts,
                  part_counts, (int*)(part_counts + (size_t)n_rows * parts * PART_WORDS),
                  (int*)(part_counts + (size_t)n_rows * parts * (PART_WORDS + 1))};
  const bool vec = (n_rows == 1 || ld % 8 == 0) && ((uintptr_t)logits & 15) == 0;
  if (parts > 1) {
    auto* fn = is_bf16 ? (vec ? k_sample_parts<true, true> : k_sample_parts<true, false>)
                       : (vec ? k_sample_parts<false, true> : k_sample_parts<false, false>);
    hipLaunchKernelGGL(fn, dim3(n_rows, parts), dim3(1024), 0, st, s);
    CFH_LAUNCH_CHECK();
  }
  // 8 bits let two workgroups share a CU, but a value that more than 255 have sends its row to the wide counts.  8 and 16 bits over
  // 1,968 rows of 32,000 logits with k and P: fp16 102 and 161 us around 0, 100 and 164 around -6, 105 and 172 of deviation 0.7 there.
  // bf16, whose values are eight times as far apart: 91 and 150 around 0, where they lie densest, but 207 and 165 of deviation 1.5 around -6,
  // 170 and 150 of 3 around 8.  300 rows, fp16 30 and 40; bf16 25 and 37 around 0, 56 and 40 around -6.  (The host cannot tell where the
  // logits lie: bf16 takes the side that gains the more.)  246 rows (a CU each) take the same either way.
  const bool narrow = V < 65536 && n_rows > 256 && (!is_bf16 || V <= 32768);
  auto launch = [&](auto bf, auto v) {
    constexpr bool BF = bf.value, VEC = v.value;
    if (narrow) hipLaunchKernelGGL((k_sample_rows<BF, VEC, 512, 8>), dim3(n_rows), dim3(512), 0, st, s);
    else hipLaunchKernelGGL((k_sample_rows<BF, VEC, 1024, 16>), dim3(n_rows), dim3(1024), 0, st, s);
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
