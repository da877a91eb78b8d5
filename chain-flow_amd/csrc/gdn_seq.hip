// The gated delta rule over committed tokens on MI355X: the recurrent step of a decode batch and the rule
// over whole prefill chunks, in the layout, with the gates and the state slots of the serving tree form
// (gdn.hip): value head hv of a row of mixed_qkv [T][2 H K + HV V] uses q/k head hv / (HV / H),
//     g = -exp(A_log) softplus(a + dt_bias),  beta = bf16(sigmoid(b)),
//     S = e^g S;  d = beta (v - S k^);  S += d k^T;  o = S q^
// with k^ = k / sqrt(|k|^2 + 1e-6), q^ = scale q / sqrt(|q|^2 + 1e-6) and S a slot [V][K] of the state.
// The state is carried in fp32 and rounded to the slot's type once, at the end of the call.
//
// Whole chunks (k_gdn_prep, k_gdn_chunks).  Over a chunk of C = 64 rows, with G_i the sum of g up to row i and
// D_ij = e^(G_i - G_j), the rows' updates d_i solve one triangular system and everything else is products:
//     (I + L) d = R,   L_ij = beta_i D_ij k^_i.k^_j (j < i),   R_i = beta_i (v_i - e^G_i S k^_i)
//     o_i = e^G_i S q^_i + sum_(j <= i) D_ij (q^_i.k^_j) d_j,   S = e^G_C S + sum_j D_Cj d_j k^_j^T
// L and its inverse, and the matrix of the second term, do not depend on S: k_gdn_prep makes them for all
// chunks at once.  k_gdn_chunks then carries S through the chunks of each (sequence, value head), 16 value
// columns a workgroup (they do not mix).
//   Precision: q and k enter MFMA as the bf16 numbers they are, their norms and decays are fp32 factors of the
// rows; fp32 operands are split into bf16 parts: R and d, on the way to an fp32 state, into three, the others into two
// (2^-18; the state's error is 1.3e-7 over 8,000 rows, 5 to 7 times that with two parts of R or d, the same with
// three of S).
// Differences of G are taken in 64 bits: a strong decay earlier in the chunk must not cost a weak one later its
// digits (decays below e^-200 are taken as that: both are 0 in fp32).
//   A row that is not finite must not reach the rows before it, whose triangular products multiply it by zeros.  Entries
// of R and d past the largest finite bf16 enter the products as that number, and from the first of them on the outputs
// of their column, and its state, are NaN.
#include <algorithm>
#include <type_traits>

#include "cfh_gdn.h"
#include "cfh_host.h"
#include "cfh_kernels.h"
#include "cfh_seq.h"
#include "cfh_tr.h"

namespace {

struct GdnSeqArgs {
  const uint16_t* qkv;   // [T][ld] bf16
  const uint16_t* ga;    // [T][HV] bf16
  const uint16_t* gb;    // [T][HV] bf16
  const float* A_log;    // [HV]
  const float* dt_bias;  // [HV]
  void* state;           // [nslots][HV][V][K]
  const int* slots;      // [S]
  const int* cu;         // [S + 1], or null: sequence s is row s
  const uint8_t* initial;  // [S] or null: 0 = start from zero instead of the slot
  uint16_t* out;         // [T][HV][V] bf16
  int* status;
  int T, S, H, HV, V, ld, nslots, l2norm;
  int few;               // k_gdn_rows takes the sequences of up to so many rows, the chunk kernels the others (0: all)
  int step, plus;        // the chunks' places (chunk_start)
  int nlong;             // sequences that k_gdn_chunks has workgroups for: all S, or as many as can have over `few` rows
  float scale;
  int fresh;             // out holds nothing yet: rows of no sequence, skipped and padding ones become 0
  int work;              // workgroups with a part of the work; those behind them clear rows of no sequence
  int* whole;            // the sequences before the first bound that falls (cfh_seq.h); null: one sequence
  int known;             // by k_ascending; else k_gdn_rows sets it for the chunk kernels
};

// softplus by log1p: with log(1 + exp(x)) a decay near 1 (x below -5, the usual ones) keeps few digits of its
// logarithm, which thousands of tokens add up.
__device__ __forceinline__ void seq_gates(float x, float Aexp, float b, float& g, float& beta) {
  g = -Aexp * (x <= 20.0f ? log1pf(expf(x)) : x);
  const float t = expf(-fabsf(b));             // (e^-b overflows below -88, where the sigmoid is still a number)
  beta = round_bf16((b < 0.f ? t : 1.0f) / (1.0f + t));
}

// Whether sequence s may use its slot: 1 yes, 0 a padding entry (slot -1), -1 refused (outside the state, or
// shared with another sequence, whose updates would race).  Uniform over the wave.
__device__ __forceinline__ int slot_verdict(const int* slots, int S, int s, int nslots) {
  const int mine = slots[s], lane = threadIdx.x & 63;
  if (mine == -1) return 0;
  int same = 0;
  for (int i = lane; i < S; i += 64) same += i != s && slots[i] == mine;
  return (__ballot(same > 0) || mine < 0 || mine >= nslots) ? -1 : 1;
}

// A workgroup behind those of the work: its share of the rows of no sequence, as zeros (of a padding one where it is the
// only one; beside others k_gdn_rows clears those).
__device__ __forceinline__ void clear_outside(const GdnSeqArgs& a) {
  const int n = a.HV * a.V / 8;
  const bool none = a.S == 1 && a.slots[0] == -1;
  const Rows r = none ? Rows{0, 0} : covered(a.cu, a.known ? *a.whole : ascending(a.cu, a.S), a.T);
  each_outside(r, a.T, blockIdx.x - a.work, gridDim.x - a.work, [&](int t) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) ((uint4*)a.out)[(size_t)t * n + i] = make_uint4(0, 0, 0, 0);
  });
}

// The simplest form, and the decode step: a wave takes 16 value rows of one (sequence, value head) and its
// tokens one after another.  Lane 16 g + p holds an 8-element share of K of rows 4 g + (0..3) (cfh_gdn.h);
// a dot product is 8 products and a 16-lane DPP sum.  No LDS and no barrier.
//   A decode step reads and writes each state once and is bound by that: 61 sequences of 32 value heads with fp32
// states (257 MB) 51.4 us, 5.0 TB/s, as a large copy; one sequence in bf16 4.4 us, a launch.
// CLEAR: with workgroups behind the work's that clear rows of no sequence (beside the chunk kernels k_gdn_prep has them:
// the branch in front of 128,000 short waves costs them 20 of 220 us).
template <typename T, bool CLEAR>
__global__ void __launch_bounds__(64) k_gdn_rows(GdnSeqArgs a) {
  constexpr int NR = sizeof(T) / 2;
  const int nvs = a.V / 16;
  int u = blockIdx.x;
  if constexpr (CLEAR) {
    if (u >= a.work) {
      clear_outside(a);
      return;
    }
  }
  const int vs = u % nvs;
  u /= nvs;
  const int hv = u % a.HV, s = u / a.HV;
  const int lane = threadIdx.x, p = lane & 15, r0 = vs * 16 + (lane >> 4) * 4;
  const int t0 = a.cu ? a.cu[s] : s, t1 = a.cu ? a.cu[s + 1] : s + 1;
  const int whole = !a.cu ? a.S : a.known ? *a.whole : ascending(a.cu, a.S);
  if (a.whole && !a.known && blockIdx.x == 0 && lane == 0) *a.whole = whole;
  const int ok = slot_verdict(a.slots, a.S, s, a.nslots);
  const bool rows = s < whole && t0 >= 0 && t1 <= a.T && t0 <= t1;
  if (ok ? a.few && rows && t1 - t0 > a.few : !a.fresh || !rows) return;
  if (ok <= 0 || !rows) {          // (padding sequences of any length)
    if (ok && a.status && lane == 0) a.status[0] = 1;
    if (rows)
      for (int t = t0; t < t1; ++t)
        if (p < 4) a.out[((size_t)t * a.HV + hv) * a.V + r0 + p] = ok ? 0x7fc0 : 0;
    return;
  }
  if (t0 == t1) return;
  T* const st = (T*)a.state + (((size_t)a.slots[s] * a.HV + hv) * a.V + r0) * GDN_DK;
  float S[4][8];
  uint4 raw[4][NR];
  if (!a.initial || a.initial[s]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) row_load(st + i * GDN_DK, p, raw[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) row_widen(raw[i], S[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < 8; ++x) S[i][x] = 0.f;
  }
  const float Aexp = expf(a.A_log[hv]), dtb = a.dt_bias[hv];
  const int h = hv / (a.HV / a.H);
  const size_t qo = (size_t)h * GDN_DK, ko = ((size_t)a.H + h) * GDN_DK;
  const size_t vo = 2 * (size_t)a.H * GDN_DK + (size_t)hv * a.V + r0;
  for (int t = t0; t < t1; ++t) {
    const uint16_t* row = a.qkv + (size_t)t * a.ld;
    // the lane's share of k and q, in the order of its share of the state's rows
    float k[8], q[8], v[4], g, beta;
    uint2 kw[2], qw[2];
    const int x0 = sizeof(T) == 2 ? 8 * p : 4 * p, x1 = sizeof(T) == 2 ? 8 * p + 4 : 64 + 4 * p;
    kw[0] = *(const uint2*)(row + ko + x0); kw[1] = *(const uint2*)(row + ko + x1);
    qw[0] = *(const uint2*)(row + qo + x0); qw[1] = *(const uint2*)(row + qo + x1);
    const uint2 vw = *(const uint2*)(row + vo);
    const size_t m = (size_t)t * a.HV + hv;
    seq_gates(bf16f(a.ga[m]) + dtb, Aexp, bf16f(a.gb[m]), g, beta);
    const float e = expf(g);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      k[4 * i] = __uint_as_float(kw[i].x << 16); k[4 * i + 1] = __uint_as_float(kw[i].x & 0xffff0000u);
      k[4 * i + 2] = __uint_as_float(kw[i].y << 16); k[4 * i + 3] = __uint_as_float(kw[i].y & 0xffff0000u);
      q[4 * i] = __uint_as_float(qw[i].x << 16); q[4 * i + 1] = __uint_as_float(qw[i].x & 0xffff0000u);
      q[4 * i + 2] = __uint_as_float(qw[i].y << 16); q[4 * i + 3] = __uint_as_float(qw[i].y & 0xffff0000u);
    }
    v[0] = __uint_as_float(vw.x << 16); v[1] = __uint_as_float(vw.x & 0xffff0000u);
    v[2] = __uint_as_float(vw.y << 16); v[3] = __uint_as_float(vw.y & 0xffff0000u);
    float rk = 1.f, rq = a.scale;
    if (a.l2norm) {
      float kk = 0.f, qq = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) { kk += k[x] * k[x]; qq += q[x] * q[x]; }
      rk = 1.0f / sqrtf(row_sum(kk) + 1e-6f);
      rq = a.scale / sqrtf(row_sum(qq) + 1e-6f);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) { k[x] *= rk; q[x] *= rq; }
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float d0 = 0.f, d1 = 0.f;
#pragma unroll
      for (int x = 0; x < 8; x += 2) {
        S[i][x] *= e; S[i][x + 1] *= e;
        d0 += S[i][x] * k[x]; d1 += S[i][x + 1] * k[x + 1];
      }
      const float d = (v[i] - row_sum(d0 + d1)) * beta;
      d0 = d1 = 0.f;
#pragma unroll
      for (int x = 0; x < 8; x += 2) {
        S[i][x] += k[x] * d; S[i][x + 1] += k[x + 1] * d;
        d0 += S[i][x] * q[x]; d1 += S[i][x + 1] * q[x + 1];
      }
      o[i] = row_sum(d0 + d1);
    }
    const float mine = p & 2 ? (p & 1 ? o[3] : o[2]) : (p & 1 ? o[1] : o[0]);
    if (p < 4) a.out[m * a.V + r0 + p] = to_bf16(mine);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    row_pack(S[i], raw[i]);
    row_store(st + i * GDN_DK, p, raw[i]);
  }
}

// ---------------------------------------------------------------- whole chunks
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

constexpr int GC = 64;                             // rows a chunk
// a chunk and value head's place in the workspace: the inverse and the attention matrix in two parts each,
// [row tile][k-step][part][lane] 16 B; then the rows' factors, fp32 [4][64], and e^G_C
constexpr int GW_ATT = 4 * 2 * 2 * 64 * 16, GW_VEC = 2 * GW_ATT;
constexpr int GW_BYTES = GW_VEC + 4 * GC * 4 + 256;
constexpr int GW_WHOLE = GW_VEC + (4 * GC + 1) * 4;   // GdnSeqArgs::whole, in the first place's spare bytes

constexpr float GDN_RANGE = 0x1.fep127f;           // the largest finite bf16

__device__ __forceinline__ f32x4 mfma_b(const uint4& x, const uint4& y, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, x), __builtin_bit_cast(b16x8, y), acc, 0, 0, 0);
}

// x = the sum of N bf16 parts, to 2^-(8 N + 1).
template <int N>
__device__ __forceinline__ void split4(const f32x4& x, uint2 (&p)[N]) {
  f32x4 r = x;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = make_uint2(pack_bf16(r[0], r[1]), pack_bf16(r[2], r[3]));
    if (i + 1 < N) {
      r[0] -= __uint_as_float(p[i].x << 16); r[1] -= __uint_as_float(p[i].x & 0xffff0000u);
      r[2] -= __uint_as_float(p[i].y << 16); r[3] -= __uint_as_float(p[i].y & 0xffff0000u);
    }
  }
}

// Chunk slots: a sequence in chunks, of n rows, uses the ceil(n / 64) from chunk_start on.  No two share one: with
// floor(cu[s] / 64) + s sequences lie at least that many apart; with floor(cu[s] / (few + 1)), for few < 32, one of
// more than `few` rows lies at least floor(n / (few + 1)) >= ceil(n / 64) before the next.
__device__ __forceinline__ int chunk_start(const GdnSeqArgs& a, int s) { return a.cu[s] / a.step + a.plus * s; }

// The order of a contraction over 32 k-slots, element e of lane group g: 16-row MFMA results (row 4 g + r of two
// tiles, r = e % 4, tile e / 4) are operands as they stand.  The other operand follows it.
//   slot (g, e) = row 16 (e / 4) + 4 g + e % 4

// L, (I + L)^-1, the attention matrix and the rows' factors of one chunk and value head.  Four waves, a
// 16-row tile each.  Bound by the substitution and the block products behind each other: 8,000 rows of 32 value heads
// 65 us (4,032 workgroups, three a CU at once); sharing K K^T among the value heads of a q/k head leaves fewer waves
// a SIMD and takes 66.
__global__ void __launch_bounds__(256) k_gdn_prep(GdnSeqArgs a, char* ws) {
  __shared__ __align__(16) float Ls[GC][GC + 4], Ts[GC][GC + 4];
  __shared__ __align__(16) float rks[GC], rqs[GC], bts[GC];
  __shared__ double Gs[GC];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, tl = lane & 15;
  const int slot = blockIdx.x / a.HV, hv = blockIdx.x % a.HV;
  if ((int)blockIdx.x >= a.work) {
    clear_outside(a);
    return;
  }
  const int whole = a.whole ? *a.whole : a.S;
  const int s = last_where(whole, [&](int i) { return chunk_start(a, i) <= slot; });
  const int c0 = a.cu[s], c1 = a.cu[s + 1];
  if (s >= whole || c0 < 0 || c0 > c1 || c1 > a.T || c1 - c0 <= a.few) return;
  const int chunk = slot - chunk_start(a, s);
  if (chunk < 0 || chunk >= (c1 - c0 + GC - 1) / GC) return;
  const int t0 = c0 + chunk * GC, n = min(GC, c1 - t0);
  const int h = hv / (a.HV / a.H);
  char* const w = ws + ((size_t)slot * a.HV + hv) * GW_BYTES;

  // this lane's share of row tl of each tile: columns 32 ks + 8 g .. + 7, the operand of either side
  uint4 kf[4][4], qf[4];
#pragma unroll
  for (int tile = 0; tile < 4; ++tile) {
    const int row = 16 * tile + tl;
    const uint16_t* p = a.qkv + (size_t)(t0 + min(row, n - 1)) * a.ld + ((size_t)a.H + h) * GDN_DK + 8 * g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      kf[tile][ks] = make_uint4(0, 0, 0, 0);
      if (tile <= wave) {
        kf[tile][ks] = *(const uint4*)(p + 32 * ks);
        if (row >= n) kf[tile][ks] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  {
    const int row = 16 * wave + tl;
    const uint16_t* p = a.qkv + (size_t)(t0 + min(row, n - 1)) * a.ld + (size_t)h * GDN_DK + 8 * g;
    float kk = 0.f, qq = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      qf[ks] = *(const uint4*)(p + 32 * ks);
      if (row >= n) qf[ks] = make_uint4(0, 0, 0, 0);
      // (the wave's own tile of kf: selected without an index that varies)
      uint4 own = kf[0][ks];
#pragma unroll
      for (int tile = 1; tile < 4; ++tile)
        if (tile == wave) own = kf[tile][ks];
      auto sq = [](const uint4& r) {
        float x = 0.f;
        const unsigned v[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float lo = __uint_as_float(v[e] << 16), hi = __uint_as_float(v[e] & 0xffff0000u);
          x += lo * lo;
          x += hi * hi;
        }
        return x;
      };
      kk += sq(own);
      qq += sq(qf[ks]);
    }
    kk += __shfl_xor(kk, 16); kk += __shfl_xor(kk, 32);
    qq += __shfl_xor(qq, 16); qq += __shfl_xor(qq, 32);
    if (lane < 16) {
      rks[row] = a.l2norm ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f;
      rqs[row] = a.l2norm ? a.scale / sqrtf(qq + 1e-6f) : a.scale;
    }
  }
  if (wave == 0) {
    float gl = 0.f, bt = 0.f;
    if (lane < n) {
      const size_t m = (size_t)(t0 + lane) * a.HV + hv;
      seq_gates(bf16f(a.ga[m]) + a.dt_bias[hv], expf(a.A_log[hv]), bf16f(a.gb[m]), gl, bt);
      gl = gl < -200.f ? -200.f : gl;
    }
    double G = gl;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double x = __shfl_up(G, o);
      if (lane >= o) G += x;
    }
    Gs[lane] = G;
    bts[lane] = bt;
  }
  __syncthreads();

  // L into LDS, the attention matrix A kept for later: element (row 16 wave + 4 g + r, column 16 tile + tl)
  const float4 rk4 = *(const float4*)&rks[16 * wave + 4 * g], rq4 = *(const float4*)&rqs[16 * wave + 4 * g];
  const float4 bt4 = *(const float4*)&bts[16 * wave + 4 * g];
  const float rkr[4] = {rk4.x, rk4.y, rk4.z, rk4.w}, rqr[4] = {rq4.x, rq4.y, rq4.z, rq4.w};
  const float btr[4] = {bt4.x, bt4.y, bt4.z, bt4.w};
  f32x4 att[4];
#pragma unroll
  for (int tile = 0; tile < 4; ++tile) {
    att[tile] = f32x4{};
    f32x4 kk = {}, qk = {};
    if (tile <= wave) {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint4 own = kf[0][ks];
#pragma unroll
        for (int x = 1; x < 4; ++x)
          if (x == wave) own = kf[x][ks];
        kk = mfma_b(own, kf[tile][ks], kk);
        qk = mfma_b(qf[ks], kf[tile][ks], qk);
      }
      const int j = 16 * tile + tl;
      const double Gj = Gs[j];
      const float rkj = rks[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * g + r;
        const float d = expf((float)(Gs[i] - Gj));
        kk[r] = j < i ? btr[r] * d * (rkr[r] * rkj) * kk[r] : 0.f;
        att[tile][r] = j <= i ? d * (rqr[r] * rkj) * qk[r] : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) Ls[16 * wave + 4 * g + r][16 * tile + tl] = kk[r];
  }
  if (wave == 0) {
    // the rows' factors: beta, beta e^G |k|^-1, e^G |q|^-1 scale, e^(G_C - G) |k|^-1
    float* v = (float*)(w + GW_VEC);
    const float e = expf((float)Gs[lane]);
    v[lane] = bts[lane];
    v[GC + lane] = bts[lane] * e * rks[lane];
    v[2 * GC + lane] = e * rqs[lane];
    v[3 * GC + lane] = expf((float)(Gs[GC - 1] - Gs[lane])) * rks[lane];
    if (lane == 0) v[4 * GC] = expf((float)Gs[GC - 1]);
  }
  // the inverse, by 16 x 16 blocks.  Diagonal: column tl by substitution down the rows, in registers (the four
  // lane groups do the same work)
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float d = i == tl ? 1.f : 0.f;
#pragma unroll
    for (int l = 0; l < i; ++l) d -= Ls[16 * wave + i][16 * wave + l] * x[l];
    x[i] = d;
  }
  if (g == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) Ts[16 * wave + i][16 * wave + tl] = x[i];
  }
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (b > wave)
#pragma unroll
      for (int r = 0; r < 4; ++r) Ts[16 * wave + 4 * g + r][16 * b + tl] = 0.f;
  // below it: T_ab = -T_aa sum_(b <= c < a) L_ac T_cb, in fp32 MFMA (16 x 16 x 4: operand lanes tl = row or
  // column, g = k), block diagonal by block diagonal; the sum's result is the second product's operand as it is
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    __syncthreads();
    if (wave >= d) {
      const int b = wave - d;
      f32x4 m = {}, t = {};
      for (int c = b; c < wave; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          m = __builtin_amdgcn_mfma_f32_16x16x4f32(Ls[16 * wave + tl][16 * c + 4 * k + g], Ts[16 * c + 4 * k + g][16 * b + tl], m, 0, 0, 0);
      // (a row of L that is not finite: its R is not either, which k_gdn_chunks answers for)
#pragma unroll
      for (int r = 0; r < 4; ++r) m[r] = fabsf(m[r]) < INFINITY ? m[r] : 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        t = __builtin_amdgcn_mfma_f32_16x16x4f32(Ts[16 * wave + tl][16 * wave + 4 * g + r], m[r], t, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) Ts[16 * wave + 4 * g + r][16 * b + tl] = -t[r];
    }
  }
  __syncthreads();
  // both matrices as operands, split (A by way of L's place); columns past the tile's rows are zero, never read
#pragma unroll
  for (int tile = 0; tile < 4; ++tile)
#pragma unroll
    for (int r = 0; r < 4; ++r) Ls[16 * wave + 4 * g + r][16 * tile + tl] = att[tile][r];
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float(*M)[GC + 4] = m ? Ls : Ts;
    uint4* out = (uint4*)(w + m * GW_ATT) + (size_t)wave * 4 * 64 + lane;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks > wave / 2) break;
      uint2 p0[2], p1[2];
      split4(*(const f32x4*)&M[16 * wave + tl][32 * ks + 4 * g], p0);
      split4(*(const f32x4*)&M[16 * wave + tl][32 * ks + 16 + 4 * g], p1);
#pragma unroll
      for (int p = 0; p < 2; ++p) out[(ks * 2 + p) * 64] = make_uint4(p0[p].x, p0[p].y, p1[p].x, p1[p].y);
    }
  }
}

// S through the chunks of one (sequence, value head), 16 value columns, in a chain that no other workgroup can
// shorten: what counts is the time from one chunk's S to the next one's, 1.6 us (8,000 rows of 32 value heads: 125
// chunks in 200 us on all CUs; five prompts of up to 300 rows 39: 1,280 workgroups, one a CU, so five rounds of up to
// five chunks and their ramps).  Waves 0 - 3 carry the chain, waves
// 4 - 7 compute the outputs beside it, waves 8 - 11 bring K, v and the rows' factors into LDS.  Three barriers a
// chunk.
//   B1  every chain wave multiplies all of K with its own 32 k rows of S (from registers), the partial products
//       meet in LDS
//   B2  each chain wave makes R of its 16 rows of them
//   B3  and d of its rows of the inverse and R; then its 32 k rows of S from all d
// What a phase reads of LDS but does not wait for is read before the barrier in front of it.
// Rows of S in a wave's MFMA tiles: tile u, row 4 g + r is k row 32 wave + 8 g + 4 u + r, so that the two tiles
// of a lane make eight neighbouring k rows, the natural operand order of K and Q.
// Global accesses go through buffer descriptors of the chunk (base and size in scalar registers, one lane offset
// for all chunks): rows behind the sequence read as zero and are not written, with no branch and no select.  A
// branch around a load or store has the compiler count it as perhaps not issued, and a wait for an older load
// becomes a wait for everything behind it.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2b __attribute__((ext_vector_type(2)));
__device__ __forceinline__ __amdgpu_buffer_rsrc_t span(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x27000);
}
__device__ __forceinline__ uint4 span_load16(__amdgpu_buffer_rsrc_t b, int at) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0));
}

struct KeyIn {                     // a lane of a staging wave, one chunk
  uint4 k[4];
  uint2 v;
  float f;
};
struct OutIn {                     // a lane of an output wave, one chunk
  uint4 q[4], at[2][2];            // row 16 wave + tl of Q; its rows of the attention matrix: [k-step][part]
  float4 cq;                       // factors of rows 16 wave + 4 g + r
};

template <typename T>
__global__ void __launch_bounds__(768) k_gdn_chunks(GdnSeqArgs a, const char* ws) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 2;                // parts of R and d
  __shared__ __align__(16) uint16_t kl[2][GC * GDN_DK];     // K, chunks of 16 bytes in swz order
  __shared__ __align__(16) f32x4 sX[4][4][64];              // partial K S: [chain wave][row tile][lane]
  __shared__ __align__(16) uint4 sS[4][2][64];              // S for the outputs: [k-step = wave][part][lane]
  __shared__ __align__(16) uint2 sR[NP][2][64][2], sE[NP][2][64][2], sD[2][2][64][2];   // [part][k-step][lane][tile of it]
  __shared__ __align__(16) uint2 sV[2][4][64];              // v: [row tile][row, 4 columns]
  __shared__ int sBad[2][16];                               // the first row of each column that is not finite
  __shared__ __align__(16) float sF[2][4][GC];              // beta, beta e^G |k|^-1, e^(G_C - G) |k|^-1, e^G_C
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, tl = lane & 15;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wv & 3;
  const int nsl = a.V / 16;
  // the column slices of a (sequence, value head) read the same chunks: on one XCD, whose L2 holds them
  const int pair = (blockIdx.x / 8 / nsl) * 8 + blockIdx.x % 8, sl = blockIdx.x / 8 % nsl;
  if (pair >= a.nlong * a.HV) return;
  int s = pair / a.HV;
  const int hv = pair % a.HV, whole = a.whole ? *a.whole : a.S;
  if (a.nlong < a.S) {             // the s-th sequence in chunks, 64 a step
    int skip = s, i = 0;
    unsigned long long m = 0;
    for (; i < whole; i += 64) {
      const int j = min(i + lane, whole - 1), b0 = a.cu[j], b1 = a.cu[j + 1];
      m = __ballot(i + lane < whole && b0 >= 0 && b1 <= a.T && b1 - b0 > a.few);
      const int n = __popcll(m);
      if (skip < n) break;
      skip -= n;
    }
    if (i >= whole) return;
    for (; skip; --skip) m &= m - 1;
    s = i + __builtin_ctzll(m);
  }
  const int c0 = a.cu[s], c1 = a.cu[s + 1];
  const bool rows = s < whole && c0 >= 0 && c0 <= c1 && c1 <= a.T;
  if (rows && a.few && c1 - c0 <= a.few) return;
  const int ok = slot_verdict(a.slots, a.S, s, a.nslots);
  if (ok == 0) return;
  if (ok < 0 || !rows) {
    if (a.status && tid == 0) a.status[0] = 1;
    if (rows)
      for (int t = c0 + tid / 16; t < c1; t += 48) a.out[((size_t)t * a.HV + hv) * a.V + sl * 16 + tid % 16] = 0x7fc0;
    return;
  }
  if (c0 == c1) return;
  const int h = hv / (a.HV / a.H), nc = (c1 - c0 + GC - 1) / GC;
  const char* const wb = ws + ((size_t)chunk_start(a, s) * a.HV + hv) * GW_BYTES;
  auto place = [&](int c) { return wb + (size_t)c * a.HV * GW_BYTES; };
  // (chunks past the last one: the last one again)
  auto rows_of = [&](int c) {      // the chunk's rows of mixed_qkv
    const int t0 = c0 + c * GC, n = min(GC, c1 - t0);
    return span(a.qkv + (size_t)t0 * a.ld, n * a.ld * 2);
  };

  if (wv >= 8) {
    const int koff = ((tid - 512) / 16 * a.ld + (a.H + h) * GDN_DK + (tid % 16) * 8) * 2, krow = 16 * a.ld * 2;
    const int voff = ((16 * wave + lane / 4) * a.ld + 2 * a.H * GDN_DK + hv * a.V + sl * 16 + 4 * (lane & 3)) * 2;
    const int foff = GW_VEC + (wave == 3 ? 4 * GC : (wave == 2 ? 3 : wave) * GC + lane) * 4;
    auto load = [&](int c, KeyIn& in) {
      const auto b = rows_of(c);
#pragma unroll
      for (int x = 0; x < 4; ++x) in.k[x] = span_load16(b, koff + x * krow);
      in.v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(b, voff, 0, 0));
      in.f = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(span(place(c), GW_BYTES), foff, 0, 0));
    };
    auto stage = [&](int c, const KeyIn& in) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = 16 * x + (tid - 512) / 16;
        *(uint4*)&kl[c & 1][row * GDN_DK + (((tid % 16) ^ swz<GDN_DK>(row)) * 8)] = in.k[x];
      }
      sV[c & 1][wave][lane] = in.v;
      sF[c & 1][wave][lane] = in.f;
      if (tid < 512 + 16) sBad[c & 1][tid - 512] = GC;
    };
    auto work = [&](int c, KeyIn& in, const KeyIn& next) {
      lds_barrier();                                         // B1
      load(min(c + 2, nc - 1), in);
      lds_barrier();                                         // B2: the other buffer's readers are done
      stage(c + 1, next);
      lds_barrier();                                         // B3: and it holds the next chunk
    };
    KeyIn A, B;
    load(0, A);
    load(min(1, nc - 1), B);
    stage(0, A);
    lds_barrier();                                           // the first chunk's K, v and factors are there
    for (int c = 0;;) {
      work(c, A, B);
      if (++c >= nc) return;
      work(c, B, A);
      if (++c >= nc) return;
    }
  }

  if (wv >= 4) {
    const int qoff = ((16 * wave + tl) * a.ld + h * GDN_DK + 8 * g) * 2;
    // (nk: the k-steps of the wave's rows of a triangular matrix, one for the first two row tiles)
    auto load_q = [&](int c, OutIn& in) {
      const auto b = rows_of(c);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) in.q[ks] = span_load16(b, qoff + 64 * ks);
    };
    auto load_a = [&](int c, OutIn& in, auto nk) {
      const auto b = span(place(c), GW_BYTES);
#pragma unroll
      for (int x = 0; x < 2 * nk.value; ++x) in.at[x / 2][x % 2] = span_load16(b, GW_ATT + ((wave * 4 + x) * 64 + lane) * 16);
      in.cq = __builtin_bit_cast(float4, span_load16(b, GW_VEC + (2 * GC + 16 * wave + 4 * g) * 4));
    };
    const size_t rs = (size_t)a.HV * a.V;
    const int ooff = ((16 * wave + 4 * g) * (int)rs + hv * a.V + sl * 16 + tl) * 2;
    auto work = [&](int c, const OutIn& in, OutIn& next, auto nk) {
      lds_barrier();                                         // B1
      f32x4 Y[2] = {};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        Y[0] = mfma_b(in.q[ks], sS[ks][0][lane], Y[0]);
        Y[1] = mfma_b(in.q[ks], sS[ks][1][lane], Y[1]);
      }
      const float cq[4] = {in.cq.x, in.cq.y, in.cq.z, in.cq.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) Y[0][r] = cq[r] * (Y[0][r] + Y[1][r]);
      lds_barrier();                                         // B2
      load_q(min(c + 1, nc - 1), next);
      lds_barrier();                                         // B3
      f32x4 o[3] = {};
#pragma unroll
      for (int ks = 0; ks < nk.value; ++ks) {
        const uint4 hi = *(const uint4*)sD[0][ks][lane], lo = *(const uint4*)sD[1][ks][lane];
        o[0] = mfma_b(in.at[ks][0], hi, o[0]);
        o[1] = mfma_b(in.at[ks][0], lo, o[1]);
        o[2] = mfma_b(in.at[ks][1], hi, o[2]);
      }
      load_a(min(c + 1, nc - 1), next, nk);
      f32x4 O = Y[0] + (o[0] + (o[1] + o[2]));
      const int bad = sBad[c & 1][tl] - (16 * wave + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r) O[r] = r < bad ? O[r] : __builtin_nanf("");
      const int t0 = c0 + c * GC;
      const auto b = span(a.out + (size_t)t0 * rs, min(GC, c1 - t0) * (int)rs * 2);
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b16(to_bf16(O[r]), b, ooff + r * (int)rs * 2, 0, 0);
    };
    OutIn A, B;
    auto chunks = [&](auto nk) {
      load_q(0, A);
      load_a(0, A, nk);
      lds_barrier();
      for (int c = 0;;) {
        work(c, A, B, nk);
        if (++c >= nc) break;
        work(c, B, A, nk);
        if (++c >= nc) break;
      }
    };
    if (wave < 2) chunks(std::integral_constant<int, 1>{});
    else chunks(std::integral_constant<int, 2>{});
    return;
  }

  T* const st = (T*)a.state + (((size_t)a.slots[s] * a.HV + hv) * a.V + sl * 16 + tl) * GDN_DK + 32 * wave + 8 * g;
  f32x4 S[2] = {};
  if (!a.initial || a.initial[s]) {
    if constexpr (sizeof(T) == 4) {
      S[0] = *(const f32x4*)st;
      S[1] = *(const f32x4*)(st + 4);
    } else {
      const uint4 x = *(const uint4*)st;
      S[0] = f32x4{__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16),
                   __uint_as_float(x.y & 0xffff0000u)};
      S[1] = f32x4{__uint_as_float(x.z << 16), __uint_as_float(x.z & 0xffff0000u), __uint_as_float(x.w << 16),
                   __uint_as_float(x.w & 0xffff0000u)};
    }
  }
  auto load_t = [&](int c, uint4 (&t)[2][2], auto nk) {      // its rows of the inverse: [k-step][part]
    const auto b = span(place(c), GW_BYTES);
#pragma unroll
    for (int x = 0; x < 2 * nk.value; ++x) t[x / 2][x % 2] = span_load16(b, ((wave * 4 + x) * 64 + lane) * 16);
  };
  // a chunk's K at the wave's k columns, rows 16 i + tl; v of rows 16 wave + 4 g + r, column tl; the factors
  uint4 kx[4];
  uint2 vv;
  f32x4 fb, fx, fe;
  float eg;
  auto read_in = [&](int c) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      kx[i] = *(const uint4*)&kl[c & 1][(16 * i + tl) * GDN_DK + (((4 * wave + g) ^ swz<GDN_DK>(tl)) * 8)];
    vv = read_tr((const uint16_t*)&sV[c & 1][wave][16 * g] + 4 * tl);
    fb = *(const f32x4*)&sF[c & 1][0][16 * wave + 4 * g];
    fx = *(const f32x4*)&sF[c & 1][1][16 * wave + 4 * g];
    fe = *(const f32x4*)&sF[c & 1][2][16 * wave + 4 * g];
    eg = sF[c & 1][3][0];
  };
  // entries out of range come back inside it; the first of the lane's four rows that has one (or `first`).  No branch:
  // it would cost the loads in flight more than the selects.
  auto into_range = [&](f32x4& x, int first) {
#pragma unroll
    for (int r = 3; r >= 0; --r) {
      const float y = __builtin_amdgcn_fmed3f(x[r], -GDN_RANGE, GDN_RANGE);
      first = x[r] == y ? first : min(first, 16 * wave + 4 * g + r);
      x[r] = y;
    }
    return first;
  };
  // (inlined whatever its size: a call would have everything it refers to in scratch memory)
  auto work = [&](int c, const uint4 (&t)[2][2], uint4 (&tnext)[2][2], auto nk) __attribute__((always_inline)) {
    const uint16_t* kt = kl[c & 1];
    uint2 p0[2], p1[2], pn[NP];
    uint4 sp[2];
    split4(S[0], p0);
    split4(S[1], p1);
#pragma unroll
    for (int p = 0; p < 2; ++p) sp[p] = make_uint4(p0[p].x, p0[p].y, p1[p].x, p1[p].y);
    f32x4 X[4] = {};
#pragma unroll
    for (int p = 1; p >= 0; --p)
#pragma unroll
      for (int i = 0; i < 4; ++i) X[i] = mfma_b(kx[i], sp[p], X[i]);
    sS[wave][0][lane] = sp[0];
    sS[wave][1][lane] = sp[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) sX[wave][i][lane] = X[i];
    lds_barrier();                                           // B1
    const f32x4 x = (sX[0][wave][lane] + sX[1][wave][lane]) + (sX[2][wave][lane] + sX[3][wave][lane]);
    const f32x4 v = {__uint_as_float(vv.x << 16), __uint_as_float(vv.x & 0xffff0000u), __uint_as_float(vv.y << 16),
                     __uint_as_float(vv.y & 0xffff0000u)};
    f32x4 R;
#pragma unroll
    for (int r = 0; r < 4; ++r) R[r] = fb[r] * v[r] - fx[r] * x[r];
    int bad = into_range(R, GC);
    split4(R, pn);
#pragma unroll
    for (int p = 0; p < NP; ++p) sR[p][wave >> 1][lane][wave & 1] = pn[p];
    lds_barrier();                                           // B2
    f32x4 d[3] = {};
#pragma unroll
    for (int ks = 0; ks < nk.value; ++ks) {
      uint4 y[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) y[p] = *(const uint4*)sR[p][ks][lane];
      d[0] = mfma_b(t[ks][0], y[0], d[0]);
      d[1] = mfma_b(t[ks][0], y[1], d[1]);
      d[2] = mfma_b(t[ks][1], y[0], d[2]);
      if constexpr (NP == 3) {
        d[1] = mfma_b(t[ks][0], y[2], d[1]);
        d[2] = mfma_b(t[ks][1], y[1], d[2]);
      }
    }
    load_t(min(c + 1, nc - 1), tnext, nk);
    // K's columns as rows, by transposed reads: row of S 16 u + tl, tokens in slot order
    uint4 kf[2][2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int r0 = 32 * ks + 4 * g + tl / 4, r1 = r0 + 16, ch = 4 * wave + (tl & 3);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint2 y = read_tr(&kt[r0 * GDN_DK + ((ch ^ swz<GDN_DK>(r0)) * 8) + 4 * u]);
        const uint2 z = read_tr(&kt[r1 * GDN_DK + ((ch ^ swz<GDN_DK>(r1)) * 8) + 4 * u]);
        kf[ks][u] = make_uint4(y.x, y.y, z.x, z.y);
      }
    }
    f32x4 D = d[0] + (d[1] + d[2]);
    bad = into_range(D, bad);
    __hip_atomic_fetch_min(&sBad[c & 1][tl], bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    split4(D * fe, pn);
#pragma unroll
    for (int p = 0; p < NP; ++p) sE[p][wave >> 1][lane][wave & 1] = pn[p];
    split4(D, p1);
#pragma unroll
    for (int p = 0; p < 2; ++p) sD[p][wave >> 1][lane][wave & 1] = p1[p];
    const float eg0 = eg;
    lds_barrier();                                           // B3
    f32x4 up[2][2] = {};
    uint4 y[2][NP];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int p = 0; p < NP; ++p) y[ks][p] = *(const uint4*)sE[p][ks][lane];
    const float keep = sBad[c & 1][tl] < GC ? __builtin_nanf("") : eg0;
    read_in(min(c + 1, nc - 1));
#pragma unroll
    for (int p = NP - 1; p >= 0; --p)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) up[u][ks] = mfma_b(kf[ks][u], y[ks][p], up[u][ks]);
#pragma unroll
    for (int u = 0; u < 2; ++u) S[u] = S[u] * keep + (up[u][0] + up[u][1]);
  };
  __builtin_amdgcn_s_setprio(3);     // (the outputs fill what the chain leaves)
  uint4 A[2][2], B[2][2];
  auto chunks = [&](auto nk) {
    load_t(0, A, nk);
    lds_barrier();
    read_in(0);
    for (int c = 0;;) {
      work(c, A, B, nk);
      if (++c >= nc) break;
      work(c, B, A, nk);
      if (++c >= nc) break;
    }
  };
  if (wave < 2) chunks(std::integral_constant<int, 1>{});
  else chunks(std::integral_constant<int, 2>{});
  if constexpr (sizeof(T) == 4) {
    *(f32x4*)st = S[0];
    *(f32x4*)(st + 4) = S[1];
  } else {
    *(uint4*)st = make_uint4(pack_bf16(S[0][0], S[0][1]), pack_bf16(S[0][2], S[0][3]), pack_bf16(S[1][0], S[1][1]),
                             pack_bf16(S[1][2], S[1][3]));
  }
}

// The rows up to which a sequence goes one after another (k_gdn_rows): 8, and 1 more for each round of workgroups that
// k_gdn_chunks takes, one a CU (32 value heads of 128, calls one after another / in chunks: one sequence of 8 rows 12.3 /
// 13.9 us, of 12 16.7 / 14.0; eight of 12 42 / 45, of 16 53 / 49, of 24 74 / 50; 32 of 14 108 / 145, of 20 148 / 148).
// Lengths are known on the device only, so with more than one sequence and rows enough for a long one both forms are
// launched, each for its sequences: 63 single rows beside 500 76 us, 603 when one form served all of a call.  Launches
// without a sequence of theirs cost 3 to 16 us (two of 12, eight of 16).
constexpr int GDN_ROWS_MIN = 9, GDN_ROWS_MAX = 16, GDN_CUS = 256;
static_assert(GDN_ROWS_MAX < 32, "chunk slots");

// Places of chunks by either rule of chunk_start.
inline long long slots_by_chunks(int T, int S) { return (long long)T / GC + S; }
inline long long slots_by_rows(int T, int few) { return T / (few + 1) + 1; }
inline long long places(int T, int S, int few) { return std::min(slots_by_chunks(T, S), slots_by_rows(T, few)); }

// How a prefill is split, from what the host knows.
struct PrefillPlan {
  int few;               // rows up to which a sequence goes one after another
  int step, plus;        // chunk_start
  int nlong;             // sequences of more rows, at most
  long long places;      // chunks they use, at most
};
PrefillPlan prefill_plan(int T, int S, int HV, int V) {
  PrefillPlan p;
  const long long rounds = ((long long)S * HV * (V / 16) + GDN_CUS - 1) / GDN_CUS;
  p.few = (int)std::min<long long>(GDN_ROWS_MIN - 1 + std::max(1ll, rounds), GDN_ROWS_MAX);
  const bool by_rows = slots_by_rows(T, p.few) < slots_by_chunks(T, S);
  p.step = by_rows ? p.few + 1 : GC;
  p.plus = by_rows ? 0 : 1;
  p.nlong = S > 1 ? std::min(S, T / (p.few + 1)) : 1;
  p.places = places(T, S, p.few);
  return p;
}

constexpr int GDN_SEQS = 4096;   // sequences a call (every wave looks for its slot among theirs)

int seq_args(GdnSeqArgs& g, const void* mixed_qkv, const void* a, const void* b, const float* A_log,
             const float* dt_bias, void* ssm_state, int nslots, const int32_t* slots, int S, int T, int H, int HV, int K,
             int V, int use_l2norm, float scale, void* out, int32_t* status, int fresh) {
  if (T < 0 || S < 0 || H < 1 || HV < H || HV % H || V < 16 || V % 16 || nslots < 1) return CFH_E_INVALID;
  if (K != GDN_DK || S > GDN_SEQS || 2ll * H * K + (long long)HV * V > 1 << 20) return CFH_E_UNSUPPORTED;
  if (T == 0 || S == 0) return CFH_OK;
  if (!mixed_qkv || !a || !b || !A_log || !dt_bias || !ssm_state || !slots || !out) return CFH_E_INVALID;
  if (((uintptr_t)mixed_qkv | (uintptr_t)ssm_state) % 16 || (uintptr_t)out % (fresh ? 16 : 2)) return CFH_E_INVALID;
  g.qkv = (const uint16_t*)mixed_qkv; g.ga = (const uint16_t*)a; g.gb = (const uint16_t*)b; g.A_log = A_log;
  g.dt_bias = dt_bias; g.state = ssm_state; g.slots = slots; g.out = (uint16_t*)out; g.status = status; g.T = T;
  g.S = S; g.H = H; g.HV = HV; g.V = V; g.ld = 2 * H * K + HV * V; g.nslots = nslots; g.l2norm = use_l2norm ? 1 : 0;
  g.scale = scale; g.fresh = fresh;
  return CFH_OK;
}

// Workgroups behind the work's that clear rows of no sequence.
unsigned clearing_of(const GdnSeqArgs& g) { return g.fresh && g.cu ? clearing(2ll * g.T * g.HV * g.V) : 0; }

int launch_rows(GdnSeqArgs& g, int state_bf16, bool clear, hipStream_t st) {
  const long long blocks = (long long)g.S * g.HV * (g.V / 16);
  if (blocks > 0x7fff0000ll) return CFH_E_UNSUPPORTED;
  const unsigned more = clear ? clearing_of(g) : 0;
  g.work = (int)blocks;
  auto go = [&](auto k) { hipLaunchKernelGGL(k, dim3((unsigned)blocks + more), dim3(64), 0, st, g); };
  if (more) state_bf16 ? go(k_gdn_rows<uint16_t, true>) : go(k_gdn_rows<float, true>);
  else state_bf16 ? go(k_gdn_rows<uint16_t, false>) : go(k_gdn_rows<float, false>);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

int decode(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias, void* ssm_state,
           int state_bf16, int nslots, const int32_t* slots, int S, int H, int HV, int K, int V, int use_l2norm, float scale,
           void* out, int32_t* status, void* stream, int fresh) {
  GdnSeqArgs g = {};
  if (int rc = seq_args(g, mixed_qkv, a, b, A_log, dt_bias, ssm_state, nslots, slots, S, S, H, HV, K, V, use_l2norm,
                        scale, out, status, fresh))
    return rc;
  if (S == 0) return CFH_OK;
  return launch_rows(g, state_bf16, false, (hipStream_t)stream);
}

int prefill(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias, void* ssm_state,
            int state_bf16, int nslots, const int32_t* slots, const int32_t* cu_seqlens, const uint8_t* initial, int S,
            int T, int H, int HV, int K, int V, int use_l2norm, float scale, void* out, void* ws, int32_t* status,
            void* stream, int fresh) {
  GdnSeqArgs g = {};
  if (int rc = seq_args(g, mixed_qkv, a, b, A_log, dt_bias, ssm_state, nslots, slots, S, T, H, HV, K, V, use_l2norm,
                        scale, out, status, fresh))
    return rc;
  if (S == 0 || T == 0) return CFH_OK;
  if (!cu_seqlens) return CFH_E_INVALID;
  g.cu = cu_seqlens;
  g.initial = initial;
  hipStream_t st = (hipStream_t)stream;
  const PrefillPlan p = prefill_plan(T, S, HV, V);
  if (T <= p.few) return launch_rows(g, state_bf16, true, st);
  if (!ws || (uintptr_t)ws % 256) return CFH_E_INVALID;
  if (S > 1) {
    g.few = p.few;
    g.whole = (int*)((char*)ws + GW_WHOLE);
    if (S > ASC_OWN) {
      g.known = 1;
      hipLaunchKernelGGL(k_ascending, dim3(1), dim3(1024), 0, st, cu_seqlens, S, g.whole);
      CFH_LAUNCH_CHECK();
    }
    if (int rc = launch_rows(g, state_bf16, false, st)) return rc;
  }
  g.step = p.step;
  g.plus = p.plus;
  g.nlong = p.nlong;
  const long long prep = p.places * HV;
  const long long blocks = ((long long)g.nlong * HV + 7) / 8 * 8 * (V / 16);
  if (prep > 0x7fff0000ll || blocks > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  g.work = (int)prep;
  hipLaunchKernelGGL(k_gdn_prep, dim3((unsigned)prep + clearing_of(g)), dim3(256), 0, st, g, (char*)ws);
  CFH_LAUNCH_CHECK();
  if (state_bf16) hipLaunchKernelGGL(k_gdn_chunks<uint16_t>, dim3((unsigned)blocks), dim3(768), 0, st, g, (const char*)ws);
  else hipLaunchKernelGGL(k_gdn_chunks<float>, dim3((unsigned)blocks), dim3(768), 0, st, g, (const char*)ws);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

}  // namespace

extern "C" {

int cfh_gdn_decode(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias,
                   void* ssm_state, int state_bf16, int nslots, const int32_t* slots, int S, int H, int HV, int K, int V,
                   int use_l2norm, float scale, void* out, int32_t* status, void* stream) {
  return decode(mixed_qkv, a, b, A_log, dt_bias, ssm_state, state_bf16, nslots, slots, S, H, HV, K, V, use_l2norm, scale, out,
                status, stream, 0);
}

int cfh_gdn_decode_fresh(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias,
                         void* ssm_state, int state_bf16, int nslots, const int32_t* slots, int S, int H, int HV, int K, int V,
                         int use_l2norm, float scale, void* out, int32_t* status, void* stream) {
  return decode(mixed_qkv, a, b, A_log, dt_bias, ssm_state, state_bf16, nslots, slots, S, H, HV, K, V, use_l2norm, scale, out,
                status, stream, 1);
}

int64_t cfh_gdn_prefill_ws_bytes(int T, int S, int HV) {
  if (T < 0 || S < 0 || HV < 1) return -1;
  if (T <= GDN_ROWS_MIN || S == 0) return 0;
  return places(T, S, GDN_ROWS_MIN) * HV * GW_BYTES;   // (a larger `few` needs no more)
}

int cfh_gdn_prefill_plan(int T, int S, int HV, int V, int32_t* plan) {
  if (T < 0 || S < 1 || HV < 1 || V < 16 || !plan) return CFH_E_INVALID;
  if (S > GDN_SEQS || (long long)HV * V > 1 << 20) return CFH_E_UNSUPPORTED;
  const PrefillPlan p = prefill_plan(T, S, HV, V);
  plan[0] = p.few; plan[1] = p.step; plan[2] = p.plus; plan[3] = p.nlong; plan[4] = (int)p.places;
  return CFH_OK;
}

int cfh_gdn_prefill(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias,
                    void* ssm_state, int state_bf16, int nslots, const int32_t* slots, const int32_t* cu_seqlens,
                    const uint8_t* initial, int S, int T, int H, int HV, int K, int V, int use_l2norm, float scale,
                    void* out, void* ws, int32_t* status, void* stream) {
  return prefill(mixed_qkv, a, b, A_log, dt_bias, ssm_state, state_bf16, nslots, slots, cu_seqlens, initial, S, T, H, HV, K, V,
                 use_l2norm, scale, out, ws, status, stream, 0);
}

int cfh_gdn_prefill_fresh(const void* mixed_qkv, const void* a, const void* b, const float* A_log, const float* dt_bias,
                          void* ssm_state, int state_bf16, int nslots, const int32_t* slots, const int32_t* cu_seqlens,
                          const uint8_t* initial, int S, int T, int H, int HV, int K, int V, int use_l2norm, float scale,
                          void* out, void* ws, int32_t* status, void* stream) {
  return prefill(mixed_qkv, a, b, A_log, dt_bias, ssm_state, state_bf16, nslots, slots, cu_seqlens, initial, S, T, H, HV, K, V,
                 use_l2norm, scale, out, ws, status, stream, 1);
}

}  // extern "C"
