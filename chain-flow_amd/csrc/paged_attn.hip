// Attention of new rows over a paged cache on MI355X: a prefill chunk, a decode step's single rows, or the
// nodes of draft trees over the committed prefix.
//
// Sequence s has the query rows cu_q[s] .. cu_q[s + 1] and seq_lens[s] tokens in its pages table[s][..].
// Its row i of n sees token j where j < len and, if causal, j <= len - n + i (the chunk's own rows are the
// cache's last ones).  Head h reads kv head h / G, G = H / Hkv.
//     o = sum_j softmax_j(scale q.k_j) v_j,   lse = log sum_j exp(scale q.k_j)
// A row that sees nothing gives o = 0 and lse = -inf.
//
// The G heads of a kv head are packed beside each other as rows (row r = token r / G, head r % G), so each
// cache row is read once for all of them.  Both kernels compute the transposed scores S^T = K Q^T with MFMA:
// a lane then holds one query row's scores, the running maximum and sum of its softmax are lane-local but
// for one exchange, and the probabilities are already where the next MFMA wants its second operand
// (O^T += V^T P^T), only in another order of the tokens, which the first operand's loads follow.
// Probabilities are rounded to the 2-byte type once for that product, whose matrix instructions take no wider operand at
// this rate: half a step (2^-8, 2^-11) of each, so at most that much of sum p |v|, beside the same half step of the
// rounded output (errors of 2.3e-3 for 1.7e-3 with bf16).  Scores, statistics and sums are fp32.
//   k_attn_tiles  many rows: workgroups of NW waves x 32 rows over tiles of tokens staged in LDS
//   k_attn_rows   few rows (decode): one tile of 16 rows, each wave its own tokens, no barrier but the join's
// The long axis is cut into pieces of `piece` tokens where the rows alone do not fill the chip; k_attn_join
// then merges the pieces' (max, sum, O).
#include "cfh_host.h"
#include "cfh_kernels.h"
#include "cfh_kv.h"
#include "cfh_seq.h"
#include "cfh_tr.h"

namespace {

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

struct PagedArgs {
  const u16* q;                // [T][H][D], row stride q_ld
  u16* out;                    // [T][H][D], row stride o_ld
  float* lse;                  // [H][T]
  const void* kc; const void* vc;
  const uint8_t* ke; const uint8_t* ve;
  const int* table;            // [S][table_ld]
  const int* lens;             // [S]
  const int* cu;               // [S + 1]
  const int* whole;            // the sequences before the first bound that falls, by k_ascending (null: look)
  int* status;
  float* po;                   // pieces' O [npiece][T][H][D] (npiece > 1)
  float2* pml;                 // pieces' (max in log2 units, sum) [npiece][T][H]
  long long q_ld, o_ld, bs_k, bs_v;
  unsigned pmagic;             // j / page = (2 j * pmagic >> 32) >> pshift, j < 2^30
  int pshift;
  int T, H, Hkv, G, S, blocks, page, table_ld, max_blocks, causal;
  int piece, npiece, tiles;    // tokens a piece, pieces, row-tile slots
  int spread;                  // on average at most one tile of k_attn_tiles a sequence
  int few;                     // rows (tokens * G) up to which a sequence is k_attn_rows' (0: none)
  int qsign;                   // of the scale: the sign goes into q, so that the scores' maximum scales
  float c;                     // |scale| log2(e)
  int fresh;                   // lse (1), and out too (2), hold nothing yet: rows of no sequence become -inf and 0
  int work;                    // workgroups with a part of the work; those behind them clear such rows
};

// Whether a sequence's rows lie in the query.
__device__ __forceinline__ bool bounds_ok(const PagedArgs& a, int c0, int c1) { return c0 >= 0 && c0 <= c1 && c1 <= a.T; }

__device__ __forceinline__ int page_of(const PagedArgs& a, int j) { return (int)(__umulhi((unsigned)j << 1, a.pmagic) >> a.pshift); }

// What one workgroup works on: rows [r0, r0 + R) of the n * G packed rows of sequence s and kv head hk, and
// the tokens [j0, j1) of one piece.
struct Work {
  int s, c0, n, len, hk, piece, r0, j0, j1, jend;   // jend: tokens any of the tile's rows sees
  bool bad;                                         // a length the table cannot hold
};

// The number of tokens row token i of n sees.
__device__ __forceinline__ int seen(const PagedArgs& a, int len, int n, int i) {
  return a.causal ? max(0, min(len, len - n + i + 1)) : len;
}

template <int R, bool ROWS>
__device__ __forceinline__ bool find_work(const PagedArgs& a, Work& w) {
  // (kv head, piece) groups and row tiles: consecutive workgroups go to the eight XCDs in turn, and each XCD
  // has its own L2, so a group's row tiles, which read the same tokens, are kept on one XCD (or an even share
  // of the XCDs) where the group count allows.  Where sequences have a tile each there is nothing to share, and
  // with lengths that differ the late pieces are few: an odd stride spreads every group and every sequence over all
  // XCDs (48 rows over 2,400 to 9,000 tokens, 2 kv heads, in 8 pieces: 61 us, 69 with a piece's rows on two XCDs)
  const int groups = a.Hkv * a.npiece;
  int g, t;
  const int b = blockIdx.x;
  if (ROWS || a.spread) {
    g = b % (groups | 1);
    t = b / (groups | 1);
  } else if (8 % groups == 0) {
    const int per = 8 / groups, x = b % 8;
    g = x / per;
    t = b / 8 * per + x % per;
  } else if (groups % 8 == 0) {
    g = b % 8 + 8 * (b / 8 / a.tiles);
    t = b / 8 % a.tiles;
  } else {
    g = b % groups;
    t = b / groups;
  }
  if (g >= groups || t >= a.tiles) return false;
  w.hk = g % a.Hkv;
  w.piece = g / a.Hkv;
  // Row-tile slot -> (sequence, tile): sequence s has the slots from floor(cu[s] G / R) + s on, at most
  // ceil(n G / R) of them used, so no two sequences share one.  (Bounds outside the query as its ends: times G they would
  // pass 32 bits, and start would no longer ascend.)  Beside k_attn_tiles: one tile of a.few rows a sequence
  const bool own = ROWS && a.few;
  const int slot = own ? t : a.tiles - 1 - t;      // (late rows see the most: first)
  auto start = [&](int i, int c) { return own ? i : min(max(c, 0), a.T) * a.G / R + i; };
  const Seq f = find_seq(a.cu, a.S, a.whole, [&](int i, int c) { return start(i, c) <= slot; });
  const int tile = slot - start(f.s, f.c0), c1 = f.c1;
  if (f.s < 0 || tile < 0 || (own && tile)) return false;
  w.s = f.s;
  w.c0 = f.c0;
  if (!bounds_ok(a, w.c0, c1)) return false;
  w.n = c1 - w.c0;
  if (ROWS ? (a.few && (long long)w.n * a.G > a.few) : (long long)w.n * a.G <= a.few) return false;
  w.r0 = tile * R;
  if (w.r0 >= w.n * a.G) return false;
  w.len = a.lens[w.s];
  w.bad = w.len < 0 || w.len > (long long)a.max_blocks * a.page;
  if (w.bad) w.len = 0;
  w.jend = seen(a, w.len, w.n, min(w.n * a.G - 1, w.r0 + R - 1) / a.G);
  w.j0 = min(w.piece * a.piece, w.jend);
  w.j1 = w.piece + 1 == a.npiece ? w.jend : min(w.j0 + a.piece, w.jend);
  // a piece past the tile's tokens has nothing to do; the first one also answers for rows that see nothing
  return w.piece == 0 || w.j0 < w.j1;
}

// A workgroup behind those of the work: its share of the rows of no sequence.
__device__ __forceinline__ void clear_outside(const PagedArgs& a, int D) {
  const int n = a.H * D / 8;
  const int whole = a.whole ? *a.whole : ascending(a.cu, a.S);
  each_outside(covered(a.cu, whole, a.T), a.T, blockIdx.x - a.work, gridDim.x - a.work, [&](int t) {
    for (int h = threadIdx.x; h < a.H; h += blockDim.x) a.lse[(size_t)h * a.T + t] = -INFINITY;
    if (a.fresh & 2)
      for (int i = threadIdx.x; i < n; i += blockDim.x) *(uint4*)(a.out + (size_t)t * a.o_ld + 8 * i) = make_uint4(0, 0, 0, 0);
  });
}

// Sequences whose rows do not lie in the query are skipped: the status word says so.
__device__ __forceinline__ void check_bounds(const PagedArgs& a) {
  if (a.status && blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.S; i += blockDim.x)
      if (!bounds_ok(a, a.cu[i], a.cu[i + 1])) a.status[0] = 1;
}

// Where token j lies: the table's entry for its page, as loaded, and its row in the block.  Looked at only when
// the token's own loads are issued (a check at once would wait for the table).  Past the work's tokens: the last
// one's.
struct Place { int blk, row; };
__device__ __forceinline__ Place look_up(const PagedArgs& a, const Work& w, int j) {
  j = min(j, w.j1 - 1);
  const int p = page_of(a, j);
  return {a.table[(size_t)w.s * a.table_ld + p], j - p * a.page};
}
// Whether token j is one of the work's and its block one of the cache's (one that is not is noted); if not, the
// place becomes one that can be read.
__device__ __forceinline__ bool resolve(const PagedArgs& a, const Work& w, int j, Place& at, int* first_bad) {
  const bool in = (unsigned)at.blk < (unsigned)a.blocks;
  if (!in) {
    if (j < w.j1) atomicMin(first_bad, j);
    at.blk = 0;
  }
  return in && j < w.j1;
}

// 16 bytes (8 elements of a 2-byte cache, 16 of an 8-bit one) of a token's row, or 8 of an 8-bit one.
template <int ES>
__device__ __forceinline__ const char* row_at(const PagedArgs& a, const void* c, long long bs, const Place& at, int hk, int D, int col) {
  return (const char*)c + ((size_t)(unsigned)at.blk * (size_t)bs + (unsigned)((at.row * a.Hkv + hk) * D + col)) * ES;
}
template <bool F8>
__device__ __forceinline__ uint4 load_row(const PagedArgs& a, const void* c, long long bs, const Place& at, int hk, int D, int col) {
  if constexpr (F8) {
    const uint2 x = *(const uint2*)row_at<1>(a, c, bs, at, hk, D, col);
    return make_uint4(x.x, x.y, 0, 0);
  } else {
    return *(const uint4*)row_at<2>(a, c, bs, at, hk, D, col);
  }
}
template <bool F8>
__device__ __forceinline__ int load_exp(const PagedArgs& a, const uint8_t* ex, const Place& at, int hk) {
  if constexpr (F8) return ex[((size_t)at.blk * a.page + at.row) * a.Hkv + hk];
  return 127;
}
template <bool BF, bool F8>
__device__ __forceinline__ uint4 to_rows(const uint4& r, int code) {
  if constexpr (F8) return dequant8<BF>(make_uint2(r.x, r.y), code);
  else return r;
}

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(const uint4& x, const uint4& y, f32x16 acc) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, x), __builtin_bit_cast(b16x8, y), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, x), __builtin_bit_cast(h16x8, y), acc, 0, 0, 0);
}

__device__ __forceinline__ float swap_max(float x) {
  const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float swap_sum(float x) {
  const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Whether any of the eight 2-byte elements is infinite or NaN.
template <bool BF>
__device__ __forceinline__ bool any_nonfinite(const uint4& r) {
  constexpr unsigned E = BF ? 0x7f80u : 0x7c00u;
  bool f = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned w = i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w;
    f |= (w & E) == E || (w & (E << 16)) == (E << 16);
  }
  return f;
}
// The same elements with zeros for those.
template <bool BF>
__device__ __forceinline__ uint4 only_finite(const uint4& r) {
  constexpr unsigned E = BF ? 0x7f80u : 0x7c00u;
  auto two = [](unsigned w) { return ((w & E) == E ? 0u : w & 0xffffu) | ((w & (E << 16)) == (E << 16) ? 0u : w & 0xffff0000u); };
  return make_uint4(two(r.x), two(r.y), two(r.z), two(r.w));
}

// Values that are not finite and that some rows of the tile do not see: 0 * NaN must not reach those.  In token
// tiles that not every row sees whole they enter LDS as zeros and their tokens are noted (bit j - base of
// `odd`); at the end each row adds those it sees to its results, where they decide by themselves.
template <bool BF, bool F8>
__device__ __forceinline__ void add_odd(const PagedArgs& a, const Work& w, unsigned* odd, int words, int base, int vis, int col,
                                        int D, float (&o)[4]) {
  for (int i = 0; i < words; ++i)
    for (unsigned m = odd[i]; m; m &= m - 1) {
      const int j = base + 32 * i + __builtin_ctz(m);
      if (j >= vis) break;
      const int p = page_of(a, j);                                       // (noted tokens lie in blocks of the cache)
      const Place at = {a.table[(size_t)w.s * a.table_ld + p], j - p * a.page};
      const uint4 r = to_rows<BF, F8>(load_row<F8>(a, a.vc, a.bs_v, at, w.hk, D, col & ~7), load_exp<F8>(a, a.ve, at, w.hk));
      float x[8];
      widen8<BF>(r, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = col & 4 ? x[4 + e] : x[e];
        if (!(fabsf(v) < INFINITY)) o[e] += v;
      }
    }
}

constexpr float LAZY = 8.f;   // log2 units the running maximum may lag behind (probabilities up to 2^8)
// fp16 probabilities are taken 2^7 as large (up to 2^15, the statistics with them): it ends at 2^-24, and beside one
// token with nearly all the weight, tens of thousands of others of 2^-25 each would vanish from the product with V.
template <bool BF>
constexpr float LIFT = BF ? 0.f : 7.f;

// Many rows.  Wave v of a workgroup takes rows 32 v .. 32 v + 31 of its tile; lane l of a wave holds query
// row l % 32, and of every group of eight tokens the four with (t / 4) % 2 == l / 32.  Token tiles of TK go
// global -> registers -> LDS one tile ahead (the 8-bit cache is widened on that way), double-buffered, one
// barrier a tile.
//   3,841 rows (16 / 4 heads of 256) over up to 9,001 tokens take 540 us: 760 TFLOP/s, 54% of a large matrix product's rate
// (D = 128: 720).  244 workgroups of 3,551 to 9,001 tokens, one a CU: over the longest one's time the CUs work 69.5% of
// it, at 78% of the product's rate while they do.  That rest is the waves' own chain scores -> softmax -> products (matrix
// instructions busy 28% of the time, LDS 31%): at D = 256 the accumulators leave room for two waves a SIMD, whose turns do
// not cover each other's exponentials.  The kernel for D = 256 spills 8 vector registers (8-bit cache: 6).
template <bool BF, bool F8, int D, int NW, int TK>
__global__ void __launch_bounds__(NW * 64, 2) k_attn_tiles(PagedArgs a) {
  constexpr int R = NW * 32, NT = NW * 64;
  constexpr int CH = D / 8;                       // 16-byte chunks a token's row
  constexpr int CPT = TK * CH / NT;               // chunks a thread stages (of K, and of V)
  constexpr int RS = NT / CH;                     // tokens between a thread's chunks
  static_assert(CPT >= 1 && TK % 32 == 0 && RS % 16 == 0, "a tile is at least a chunk a thread; one chunk order a thread");
  __shared__ __align__(16) u16 lds[2][2][TK * D];
  // the tokens that some but not all rows see lie within R of each other, and a tile on either side
  constexpr int OW = (R + 2 * TK + 31) / 32;
  __shared__ int first_bad;
  __shared__ unsigned odd[OW];
  if (__builtin_expect((int)blockIdx.x >= a.work, 0)) {
    clear_outside(a, D);
    return;
  }
  check_bounds(a);
  Work w;
  if (!find_work<R, false>(a, w)) return;         // (the whole workgroup)
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
  if (tid == 0) first_bad = 0x7fffffff;
  if (tid < OW) odd[tid] = 0;
  __syncthreads();

  const int r = w.r0 + wave * 32 + (lane & 31), rows = w.n * a.G;
  const bool live = r < rows;
  const int i = min(r, rows - 1) / a.G, hh = min(r, rows - 1) % a.G;
  const int t = w.c0 + i, h = w.hk * a.G + hh;
  const int vis = min(seen(a, w.len, w.n, i), w.j1);
  // the fewest tokens a row of the wave, and of the workgroup, sees: tiles below need no mask
  const int vis_wave = min(seen(a, w.len, w.n, min(w.r0 + wave * 32, rows - 1) / a.G), w.j1);
  const int vis_wg = min(seen(a, w.len, w.n, w.r0 / a.G), w.j1);
  uint4 qf[D / 16];
  {
    const u16* q = a.q + (size_t)t * a.q_ld + (size_t)h * D + 8 * half;
    const unsigned flip = a.qsign < 0 ? 0x80008000u : 0u, keep = a.qsign ? 0xffffffffu : 0u;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      uint4 x = *(const uint4*)(q + 16 * s);
      qf[s] = make_uint4((x.x ^ flip) & keep, (x.y ^ flip) & keep, (x.z ^ flip) & keep, (x.w ^ flip) & keep);
    }
  }

  const int srow = tid / CH, scol = tid % CH;     // this thread's chunks: tokens srow + RS x, chunk scol
  // Operand addresses: chunk c of token t lies at c ^ z(t), z below 2 KA, so only the low bits of c take part and the
  // rest, like the rows of a tile, is an offset in the instruction.  At D = 256 the accumulators leave no registers
  // for the 16 addresses of swz (they spill: 764 us where the 6 of swz8, whose reads take twice the LDS cycles, take
  // 541; 3,841 rows over 9,001 tokens, 16 / 4 heads)
  constexpr bool S8 = D == 256;
  constexpr int KA = S8 || D == 64 ? 4 : 8, VA = KA / 2;
  auto order = [](int t) { return S8 ? swz8(t) : swz<D>(t); };
  const int sat = srow * D + ((scol ^ order(srow)) * 8);
  int ka[KA], va[2][VA];
  {
    const int kt = lane & 31, vt = 4 * half + (lane & 15) / 4, vc = 2 * ((lane >> 4) & 1) + (lane & 3) / 2;
#pragma unroll
    for (int i = 0; i < KA; ++i) ka[i] = kt * D + (((2 * i + half) ^ order(kt)) * 8);
#pragma unroll
    for (int i = 0; i < VA; ++i) {
      va[0][i] = vt * D + (((4 * i + vc) ^ order(vt)) * 8) + 4 * (lane & 1);
      va[1][i] = S8 ? va[0][i] : (vt + 8) * D + (((4 * i + vc) ^ order(vt + 8)) * 8) + 4 * (lane & 1);
    }
  }
  uint4 kr[CPT], vr[CPT];
  int kx[CPT], vx[CPT];
  bool ok[CPT];
  Place pl[CPT];
  auto places = [&](int jt) {
#pragma unroll
    for (int x = 0; x < CPT; ++x) pl[x] = look_up(a, w, jt + srow + RS * x);
  };
  auto fetch = [&](int jt) {
#pragma unroll
    for (int x = 0; x < CPT; ++x) {
      ok[x] = resolve(a, w, jt + srow + RS * x, pl[x], &first_bad);
      kr[x] = load_row<F8>(a, a.kc, a.bs_k, pl[x], w.hk, D, scol * 8);
      vr[x] = load_row<F8>(a, a.vc, a.bs_v, pl[x], w.hk, D, scol * 8);
      kx[x] = load_exp<F8>(a, a.ke, pl[x], w.hk);
      vx[x] = load_exp<F8>(a, a.ve, pl[x], w.hk);
    }
  };
  const int odd_base = w.j0 + max(0, vis_wg - w.j0) / TK * TK;   // the first tile that not every row sees whole
  auto stage = [&](int jt, int buf) {
#pragma unroll
    for (int x = 0; x < CPT; ++x) {
      const int tok = srow + RS * x, at = sat + RS * x * D;
      // (V's rows of no token enter as zeros: 0 * NaN would reach the sums.  K's scores are masked)
      uint4 v = to_rows<BF, F8>(vr[x], vx[x]);
      v = ok[x] ? v : make_uint4(0, 0, 0, 0);
      *(uint4*)&lds[buf][0][at] = to_rows<BF, F8>(kr[x], kx[x]);
      if (jt + TK > vis_wg && any_nonfinite<BF>(v)) {
        v = only_finite<BF>(v);
        atomicOr(&odd[(jt + tok - odd_base) / 32], 1u << ((jt + tok - odd_base) & 31));
      }
      *(uint4*)&lds[buf][1][at] = v;
    }
  };

  f32x16 o[D / 32] = {};
  float m = -INFINITY, l = 0.f;                   // (m in log2 units; l: this half's tokens)
  if (w.j0 < w.j1) {
    places(w.j0);
    fetch(w.j0);
    places(w.j0 + TK);
    stage(w.j0, 0);
  }
  int buf = 0;
  for (int jt = w.j0; jt < w.j1; jt += TK, buf ^= 1) {
    lds_barrier();
    const bool more = jt + TK < w.j1;
    if (more) {
      fetch(jt + TK);
      places(jt + 2 * TK);
    }
    if (jt < w.j1 && w.r0 + wave * 32 < rows) {
      const u16* kt = lds[buf][0];
      const u16* vt = lds[buf][1];
      f32x16 sc[TK / 32];
#pragma unroll
      for (int b = 0; b < TK / 32; ++b) sc[b] = f32x16{};
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
#pragma unroll
        for (int b = 0; b < TK / 32; ++b)
          sc[b] = mfma32<BF>(*(const uint4*)&kt[ka[s % KA] + 32 * b * D + s / KA * 16 * KA], qf[s], sc[b]);
      }
      if (jt + TK > vis_wave) {
#pragma unroll
        for (int b = 0; b < TK / 32; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (jt + 32 * b + 8 * (e / 4) + 4 * half + e % 4 >= vis) sc[b][e] = -INFINITY;
      }
      float mx = sc[0][0];
#pragma unroll
      for (int b = 0; b < TK / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[b][e]);
      mx = swap_max(mx) * a.c - LIFT<BF>;
      if (__any(mx > m + LAZY || (m == -INFINITY && mx > m))) {
        const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] *= f;
        m = mn;
      }
      const float base = m == -INFINITY ? 0.f : m;
      uint4 pf[TK / 16];
#pragma unroll
      for (int b = 0; b < TK / 32; ++b) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          sc[b][e] = __builtin_amdgcn_exp2f(fmaf(sc[b][e], a.c, -base));
          l += sc[b][e];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
          pf[2 * b + s] = make_uint4(pack2<BF>(sc[b][8 * s], sc[b][8 * s + 1]), pack2<BF>(sc[b][8 * s + 2], sc[b][8 * s + 3]),
                                     pack2<BF>(sc[b][8 * s + 4], sc[b][8 * s + 5]), pack2<BF>(sc[b][8 * s + 6], sc[b][8 * s + 7]));
      }
      // the transposed reads: lane block (lane / 16) % 2 takes 16 of the 32 columns, half the tokens 4 half ..
      auto vfrag = [&](int d, int s) {
        const int at = 16 * s * D + d / VA * 32 * VA;
        const uint2 x = read_tr(&vt[va[0][d % VA] + at]), y = read_tr(&vt[va[1][d % VA] + at + (S8 ? 8 * D : 0)]);
        return make_uint4(x.x, x.y, y.x, y.y);
      };
#pragma unroll
      for (int s = 0; s < TK / 16; ++s)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[d] = mfma32<BF>(vfrag(d, s), pf[s], o[d]);
    }
    if (more) stage(jt + TK, buf ^ 1);
  }
  __syncthreads();
  l = swap_sum(l);
  if (w.bad || first_bad < vis) {
    l = __builtin_nanf("");
    if (a.status && live) a.status[0] = 1;
  }
  if (!live) return;
  if (a.npiece == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    u16* out = a.out + (size_t)t * a.o_ld + (size_t)h * D + 4 * half;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(uint2*)(out + 32 * d + 8 * g) = make_uint2(pack2<BF>(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                                                     pack2<BF>(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
    if (half == 0) a.lse[(size_t)h * a.T + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
  } else {
    const size_t at = ((size_t)w.piece * a.T + t) * a.H + h;
    float* po = a.po + at * D + 4 * half;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(float4*)(po + 32 * d + 8 * g) = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    if (half == 0) a.pml[at] = make_float2(m, l);
  }
  unsigned any = 0;
#pragma unroll
  for (int x = 0; x < OW; ++x) any |= odd[x];
  if (any) {                                      // (to what was just stored: the sums stay in registers)
#pragma unroll 1
    for (int c = 4 * half; c < D; c += 8) {
      float y[4] = {0.f, 0.f, 0.f, 0.f};
      add_odd<BF, F8>(a, w, odd, OW, odd_base, vis, c, D, y);
      if (a.npiece == 1) {
        u16* out = a.out + (size_t)t * a.o_ld + (size_t)h * D + c;
        for (int e = 0; e < 4; ++e) {
          float was[8];
          widen8<BF>(make_uint4(out[e], 0, 0, 0), was);
          out[e] = (u16)pack2<BF>(was[0] + y[e], 0.f);
        }
      } else {
        float* po = a.po + (((size_t)w.piece * a.T + t) * a.H + h) * D + c;
        for (int e = 0; e < 4; ++e) po[e] += y[e];
      }
    }
  }
}

// Few rows: a tile of 16, one workgroup of four waves a (row tile, kv head, piece), each wave the tokens of
// every fourth group of TG.  K goes from memory straight into the first operand's registers (16 tokens x
// 64-byte segments a load), V through the wave's own rows of LDS for the transposed reads; both one group
// ahead, 16 KB a wave (an 8-bit cache: 8 at D = 64, else 16), with no branch around a load: behind one the compiler
// waits for everything.  Waves do not wait for each other before the join of their (max, sum, O) at the end.
//   Bound by memory latency: one row over 30,011 tokens (16 / 4 heads of 256, 123 MB) is 236 workgroups, one a CU, with 64 KB
// in flight: 38.5 us, 3.2 TB/s, and the join 5 beside it; 48 rows over up to 9,000 (16 / 2 heads of 256), two workgroups a
// CU with 128 KB, 131 us together, 4.3 TB/s, and in 8 bits 97, where widening the elements shares the waves' time and
// 17 vector and 9 scalar registers spill (D = 128 in 8 bits: 8 scalar ones).  At D = 64 (and 128 in 2 bytes) 48 bytes a
// lane of scratch memory are no spill but add_odd's arrays, touched only where a value is not finite.
template <bool BF>
__device__ __forceinline__ f32x4 mfma16(const uint4& x, const uint4& y, f32x4 acc) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, x), __builtin_bit_cast(b16x8, y), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, x), __builtin_bit_cast(h16x8, y), acc, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f32x4 mfma16h(const uint2& x, const uint2& y, f32x4 acc) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, x), __builtin_bit_cast(s16x4, y), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h16x4, x), __builtin_bit_cast(h16x4, y), acc, 0, 0, 0);
}

template <bool BF, bool F8, int D>
__global__ void __launch_bounds__(256, 2) k_attn_rows(PagedArgs a) {
  constexpr int R = 16, NW = 4, KS = D / 32;      // MFMA steps of 32 along the head
  constexpr int U = F8 ? (D == 256 ? 2 : 4) : 256 / D, TG = 16 * U;   // 16-token tiles a group, its tokens
  constexpr int CE = F8 ? 16 : 8, CH = D / CE;    // elements of a 16-byte load, loads a token's row
  constexpr int KL = D / (4 * CE), VL = TG * CH / 64;   // a lane's 16-byte loads: of K a tile, of V a group
  __shared__ __align__(16) union { u16 v[NW][TG * D]; float o[NW][16 * D]; } sh;
  __shared__ float2 ml[NW][16];
  __shared__ int first_bad;
  __shared__ unsigned odd[4];                     // (the tokens not all rows see: 16, and a group on either side)
  if (__builtin_expect((int)blockIdx.x >= a.work, 0)) {
    clear_outside(a, D);
    return;
  }
  check_bounds(a);
  Work w;
  if (!find_work<R, true>(a, w)) return;          // (the whole workgroup)
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, tl = lane & 15;
  if (tid == 0) first_bad = 0x7fffffff;
  if (tid < 4) odd[tid] = 0;
  __syncthreads();
  const int rows = w.n * a.G, r = w.r0 + tl;
  const int i = min(r, rows - 1) / a.G, hh = min(r, rows - 1) % a.G;
  const int t = w.c0 + i, h = w.hk * a.G + hh;
  const int vis = min(seen(a, w.len, w.n, i), w.j1);
  const int vis_all = min(seen(a, w.len, w.n, w.r0 / a.G), w.j1);
  // contraction order: step s, lane group g, element e is column 32 s + 8 g + e, or with an 8-bit cache, whose
  // 16-byte loads hold two steps' elements, column 64 (s / 2) + 16 g + 8 (s % 2) + e
  uint4 qf[KS];
  {
    const u16* q = a.q + (size_t)t * a.q_ld + (size_t)h * D;
    const unsigned flip = a.qsign < 0 ? 0x80008000u : 0u, keep = a.qsign ? 0xffffffffu : 0u;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 x = *(const uint4*)(q + (F8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g));
      qf[s] = make_uint4((x.x ^ flip) & keep, (x.y ^ flip) & keep, (x.z ^ flip) & keep, (x.w ^ flip) & keep);
    }
  }
  u16* const vt = sh.v[wave];
  constexpr int VA = D == 64 ? 4 : 8;             // (as in k_attn_tiles)
  int va[VA];
#pragma unroll
  for (int x = 0; x < VA; ++x) {
    const int tr = 4 * g + tl / 4;
    va[x] = tr * D + (((2 * x + (tl & 3) / 2) ^ swz<D>(tr)) * 8) + 4 * (tl & 1);
  }
  // this lane's token of K's tile u is 16 u + tl; its chunks of V are of tokens (lane + 64 x) / CH
  uint4 kr[U][KL], vr[VL];
  int kx[U], vx[VL];
  bool vok[VL];
  Place kp[U], vp[VL];
  auto k_places = [&](int jt) {
#pragma unroll
    for (int u = 0; u < U; ++u) kp[u] = look_up(a, w, jt + 16 * u + tl);
  };
  auto v_places = [&](int jt) {
#pragma unroll
    for (int x = 0; x < VL; ++x) vp[x] = look_up(a, w, jt + (lane + 64 * x) / CH);
  };
  auto k_fetch = [&](int jt) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      resolve(a, w, jt + 16 * u + tl, kp[u], &first_bad);
#pragma unroll
      for (int s = 0; s < KL; ++s)
        kr[u][s] = *(const uint4*)row_at<F8 ? 1 : 2>(a, a.kc, a.bs_k, kp[u], w.hk, D, 4 * CE * s + CE * g);
      kx[u] = load_exp<F8>(a, a.ke, kp[u], w.hk);
    }
  };
  auto v_fetch = [&](int jt) {
#pragma unroll
    for (int x = 0; x < VL; ++x) {
      vok[x] = resolve(a, w, jt + (lane + 64 * x) / CH, vp[x], &first_bad);
      vr[x] = *(const uint4*)row_at<F8 ? 1 : 2>(a, a.vc, a.bs_v, vp[x], w.hk, D, (lane + 64 * x) % CH * CE);
      vx[x] = load_exp<F8>(a, a.ve, vp[x], w.hk);
    }
  };
  f32x4 o[D / 16] = {};
  float m = -INFINITY, l = 0.f;
  const int step = TG * NW;
  const int odd_base = w.j0 + max(0, vis_all - w.j0) / TG * TG;   // the first group that not every row sees whole
  int jt = w.j0 + TG * wave;
  if (jt < w.j1) {
    k_places(jt);
    v_places(jt);
    k_fetch(jt);
    v_fetch(jt);
    k_places(jt + step);
    v_places(jt + step);
  }
  for (; jt < w.j1; jt += step) {
    const bool edge = jt + TG > vis_all;          // (uniform)
#pragma unroll
    for (int x = 0; x < VL; ++x) {
      const int c = lane + 64 * x, tok = c / CH, ch = c % CH * (CE / 8);
#pragma unroll
      for (int y = 0; y < CE / 8; ++y) {
        uint4 v = F8 ? dequant8<BF>(y ? make_uint2(vr[x].z, vr[x].w) : make_uint2(vr[x].x, vr[x].y), vx[x]) : vr[x];
        v = vok[x] ? v : make_uint4(0, 0, 0, 0);
        if (edge && any_nonfinite<BF>(v)) {
          v = only_finite<BF>(v);
          atomicOr(&odd[(jt + tok - odd_base) / 32], 1u << ((jt + tok - odd_base) & 31));
        }
        *(uint4*)&vt[tok * D + (((ch + y) ^ swz<D>(tok)) * 8)] = v;
      }
    }
    v_fetch(jt + step);                           // (past the work's tokens: its last ones again, never used)
    v_places(jt + 2 * step);
    f32x4 sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sc[u] = f32x4{};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 kf;
        if constexpr (F8) kf = dequant8<BF>(s % 2 ? make_uint2(kr[u][s / 2].z, kr[u][s / 2].w) : make_uint2(kr[u][s / 2].x, kr[u][s / 2].y), kx[u]);
        else kf = kr[u][s];
        sc[u] = mfma16<BF>(kf, qf[s], sc[u]);
      }
    }
    k_fetch(jt + step);
    k_places(jt + 2 * step);
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (jt + 16 * u + 4 * g + e >= vis) sc[u][e] = -INFINITY;
        mx = fmaxf(mx, sc[u][e]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = swap_max(mx) * a.c - LIFT<BF>;
    if (__any(mx > m + LAZY || (m == -INFINITY && mx > m))) {
      const float mn = fmaxf(m, mx), fac = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= fac;
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] *= fac;
      m = mn;
    }
    const float base = m == -INFINITY ? 0.f : m;
    uint2 pf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[u][e] = __builtin_amdgcn_exp2f(fmaf(sc[u][e], a.c, -base));
        l += sc[u][e];
      }
      pf[u] = make_uint2(pack2<BF>(sc[u][0], sc[u][1]), pack2<BF>(sc[u][2], sc[u][3]));
    }
    // (a wave's LDS accesses complete in order: its reads see its own writes above)
    auto vfrag = [&](int d, int u) { return read_tr(&vt[va[d % VA] + 16 * u * D + d / VA * 16 * VA]); };
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      if constexpr (U == 1) {
        o[d] = mfma16h<BF>(vfrag(d, 0), pf[0], o[d]);
      } else {
#pragma unroll
        for (int u = 0; u < U; u += 2) {          // two tiles a step: elements 0 - 3 of the first, 4 - 7 of the second
          const uint2 x = vfrag(d, u), y = vfrag(d, u + 1);
          o[d] = mfma16<BF>(make_uint4(x.x, x.y, y.x, y.y), make_uint4(pf[u].x, pf[u].y, pf[u + 1].x, pf[u + 1].y), o[d]);
        }
      }
    }
  }
  // the four waves' join: each row's maximum, then the sums of what the waves hold under it
  l += __shfl_xor(l, 16);
  l = swap_sum(l);
  if (lane < 16) ml[wave][lane] = make_float2(m, l);
  __syncthreads();                                // (and the waves are done with sh.v)
  float mj = -INFINITY;
#pragma unroll
  for (int v = 0; v < NW; ++v) mj = fmaxf(mj, ml[v][tl].x);
  const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mj);
#pragma unroll
  for (int d = 0; d < D / 16; ++d)
    *(f32x4*)&sh.o[wave][tl * D + 16 * (d ^ (tl & (D / 16 - 1))) + 4 * g] = o[d] * mine;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 16 * D / 4 / 256; ++x) {
    const int c = tid + 256 * x, row = c / (D / 4), col = c % (D / 4) * 4;
    const int rr = w.r0 + row;
    if (rr >= rows) break;
    const int ti = rr / a.G, tt = w.c0 + ti, th = w.hk * a.G + rr % a.G;
    f32x4 sum = {};
    float ls = 0.f, mr = -INFINITY;
#pragma unroll
    for (int v = 0; v < NW; ++v) mr = fmaxf(mr, ml[v][row].x);
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      sum += *(const f32x4*)&sh.o[v][row * D + 16 * ((col / 16) ^ (row & (D / 16 - 1))) + col % 16];
      ls += ml[v][row].x == -INFINITY ? ml[v][row].y : ml[v][row].y * __builtin_amdgcn_exp2f(ml[v][row].x - mr);
    }
    if (odd[0] | odd[1] | odd[2] | odd[3]) {
      float y[4] = {sum[0], sum[1], sum[2], sum[3]};
      add_odd<BF, F8>(a, w, odd, 4, odd_base, min(seen(a, w.len, w.n, ti), w.j1), col, D, y);
      sum = f32x4{y[0], y[1], y[2], y[3]};
    }
    if (w.bad || first_bad < min(seen(a, w.len, w.n, ti), w.j1)) {
      ls = __builtin_nanf("");
      if (a.status) a.status[0] = 1;
    }
    if (a.npiece == 1) {
      const float inv = ls == 0.f ? 0.f : 1.f / ls;
      *(uint2*)(a.out + (size_t)tt * a.o_ld + (size_t)th * D + col) =
          make_uint2(pack2<BF>(sum[0] * inv, sum[1] * inv), pack2<BF>(sum[2] * inv, sum[3] * inv));
      if (col == 0) a.lse[(size_t)th * a.T + tt] = ls == 0.f ? -INFINITY : (mr + log2f(ls)) * 0.69314718055994530942f;
    } else {
      const size_t at = ((size_t)w.piece * a.T + tt) * a.H + th;
      *(f32x4*)(a.po + at * D + col) = sum;
      if (col == 0) a.pml[at] = make_float2(mr, ls);
    }
  }
}

// The pieces of each (row, head): the largest maximum, then the sums under it, in piece order.  W waves a (row,
// head), each a share of the pieces, four of them in flight, D / 64 columns a lane.
template <bool BF, int D, int W>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 64) k_attn_join(PagedArgs a) {
  constexpr int E = D / 64, B = 4;
  typedef float vec __attribute__((ext_vector_type(E)));
  __shared__ float so[W > 1 ? W : 1][D], sl[W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int at = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x, part = W == 1 ? 0 : wave;
  const int t = at / a.H, h = at % a.H;
  if (t >= a.T) return;
  const Seq f = find_seq(a.cu, a.S, a.whole, [&](int, int c) { return c <= t; });
  const int s = f.s, c0 = f.c0, c1 = f.c1;
  if (s < 0 || t < c0 || t >= c1 || !bounds_ok(a, c0, c1)) return;   // a row of no sequence
  int len = a.lens[s];
  if (len < 0 || len > (long long)a.max_blocks * a.page) len = 0;
  // the row's pieces: those that start below what it sees, and the first always
  const int np = max(1, min(a.npiece, (seen(a, len, c1 - c0, t - c0) + a.piece - 1) / a.piece));
  const size_t row = (size_t)t * a.H + h, rows = (size_t)a.T * a.H;
  float m = -INFINITY;
  for (int p = lane; p < np; p += 64) m = fmaxf(m, a.pml[p * rows + row].x);
  m = wave_max(m);
  float l = 0.f;
  vec o = {};
  const int per = (np + W - 1) / W, p1 = min(np, (part + 1) * per);
  for (int p = part * per; p < p1; p += B) {
    float2 x[B];
    vec y[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const size_t q = min(p + i, p1 - 1) * rows + row;
      x[i] = a.pml[q];
      y[i] = *(const vec*)(a.po + q * D + lane * E);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (p + i >= p1) break;
      // (a piece that saw nothing: maximum -inf, sum 0, or NaN for a bad table)
      const float f = x[i].x == -INFINITY ? x[i].y : __builtin_amdgcn_exp2f(x[i].x - m);
      l += x[i].x == -INFINITY ? x[i].y : x[i].y * f;
      o += y[i] * f;
    }
  }
  if constexpr (W > 1) {
    *(vec*)&so[part][lane * E] = o;
    if (lane == 0) sl[part] = l;
    __syncthreads();
    if (part) return;
    o = vec{};
    l = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      o += *(const vec*)&so[i][lane * E];
      l += sl[i];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  u16* out = a.out + (size_t)t * a.o_ld + (size_t)h * D + lane * E;
  if constexpr (E == 1) {
    *out = (u16)pack2<BF>(o[0] * inv, 0.f);
  } else {
    unsigned y[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2) y[e / 2] = pack2<BF>(o[e] * inv, o[e + 1] * inv);
    if constexpr (E == 2) *(unsigned*)out = y[0];
    else *(uint2*)out = make_uint2(y[0], y[1]);
  }
  if (lane == 0) a.lse[(size_t)h * a.T + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
}

// How a call is split, from what the host knows (sizes and an upper bound of the lengths).
struct Plan {
  bool rows, tiles;      // which kernels run
  int few;               // (both: the rows up to which a sequence is k_attn_rows')
  int nrow, ntile;       // row-tile slots of each
  int piece, npiece;
};

constexpr int FEW_ROWS = 16;

constexpr int tile_rows(int D) { return D == 256 ? 256 : 128; }

Plan plan(int T, int H, int Hkv, int D, int S, int max_len) {
  const int G = H / Hkv;
  Plan p = {};
  const long long packed = (long long)T * G;
  // on average at most one tile of 16 rows a sequence: all sequences are few-row ones
  p.rows = packed <= (long long)FEW_ROWS * S || packed <= FEW_ROWS;
  p.tiles = !p.rows;
  p.few = 0;
  if (p.tiles && S > 1) {         // some sequences may be few-row ones
    p.rows = true;
    p.few = FEW_ROWS;
  }
  p.nrow = p.few ? S : (int)(packed / FEW_ROWS) + S;
  p.ntile = (int)(packed / tile_rows(D)) + S;
  // Pieces so that (row tiles) x (kv heads) x pieces fill the chip with the workgroups it holds at once, one a CU at
  // D = 256 with many rows, else two.  Many rows are left whole from three quarters of a workgroup a CU on
  // (9,001 tokens, 16 / 4 heads of 256, whole / cut by the rule below / best cut: 128 workgroups 529 / 313 / 313, 160 531 /
  // 578 / 412, 192 531 / 585 / 501, 208 530 / 588 / 525, 256 553 / 607 / 607; at D = 128, where two workgroups share a CU,
  // cutting wins up to 256 of them and loses at 320: 192 in two 183 for 227, 256 198 for 228, 320 290 for 276); few rows are not (100 x 2 kv heads: whole 100
  // us, in three 65; 64 x 4: 72, in two 55; 125 x 4: 129, in two 128).  More and shorter pieces of few rows lose
  // again (48 x 2 kv heads, D = 128 in 8 bits: 3 pieces 65 us, 6 51, 8 61, 18 65).  Pieces of 512 tokens at least where
  // rows are few (one row over 30,011: 256 tokens 25 / 29 us at D = 64 / 128, 512 tokens 20 / 24), 256 where they are
  // many.
  const int fill = p.tiles && D == 256 ? 256 : 512, least = p.tiles ? 256 : 512;
  const long long items = (long long)Hkv * std::max<long long>(p.tiles ? (packed + tile_rows(D) - 1) / tile_rows(D) : S, std::min(S, T));
  const long long want = p.tiles && items >= 192 ? 1 : (fill + items - 1) / items;
  long long piece = ((long long)max_len + want - 1) / want;
  piece = std::max<long long>(least, (piece + 63) / 64 * 64);
  p.npiece = (int)std::max(1ll, ((long long)max_len + piece - 1) / piece);
  p.piece = (int)std::min<long long>(piece, 0x40000000);
  return p;
}

// Sequences up to which every workgroup looks over the bounds on its way to its sequence; k_ascending before the others
// for more (300 of 500 tokens 51.9 us so and 55.4 with k_ascending, 1,000 of 300 tokens 119 and 115, 110 unchecked).
constexpr int ASC_FIND = 512;

// The workspace: the pieces' O, their (max, sum), and the count of sequences where k_ascending makes it.
struct Space { int64_t pml, whole, all; };
Space space(const Plan& p, int T, int H, int D, int S) {
  Space w = {};
  if (p.npiece > 1) {
    w.pml = cfh::align256((size_t)p.npiece * T * H * D * sizeof(float));
    w.whole = w.pml + cfh::align256((size_t)p.npiece * T * H * sizeof(float2));
  }
  w.all = w.whole + (S > ASC_FIND ? 256 : 0);
  return w;
}

int attend(const void* q, long long q_ld, int T, int H, int Hkv, int D, int is_bf16, const void* k_cache,
           long long bs_k, const void* v_cache, long long bs_v, const uint8_t* k_exp, const uint8_t* v_exp,
           int blocks, int page, const int32_t* table, int table_ld, int max_blocks, const int32_t* seq_lens,
           const int32_t* cu_q, int S, float scale, int causal, int max_len, void* out, long long o_ld,
           float* lse, void* ws, int32_t* status, void* stream, int fresh) {
  if (T < 0 || S < 0 || H < 1 || Hkv < 1 || H % Hkv || blocks < 1 || page < 1 || max_blocks < 0 ||
      table_ld < max_blocks || max_len < 0)
    return CFH_E_INVALID;
  if (D != 64 && D != 128 && D != 256) return CFH_E_UNSUPPORTED;
  if ((long long)blocks * page > 0x7fffffffll || (long long)max_blocks * page > 0x3fffffffll ||
      (long long)T * H > 0x3fffffffll || S > 1 << 20)
    return CFH_E_UNSUPPORTED;
  const bool f8 = k_exp || v_exp;
  if (!k_cache || !v_cache || (f8 && (!k_exp || !v_exp))) return CFH_E_INVALID;
  const long long inner = (long long)page * Hkv * D;
  if (inner > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  if (bs_k < inner || bs_v < inner || bs_k % 16 || bs_v % 16 || ((uintptr_t)k_cache | (uintptr_t)v_cache) % 16)
    return CFH_E_INVALID;
  if (T == 0 || S == 0) return CFH_OK;
  if (!q || !out || !lse || !seq_lens || !cu_q || (max_blocks && !table) || q_ld < (long long)H * D ||
      o_ld < (long long)H * D || q_ld % 8 || o_ld % 8 || ((uintptr_t)q | (uintptr_t)out) % 16)
    return CFH_E_INVALID;
  const Plan p = plan(T, H, Hkv, D, S, max_len);
  const Space w = space(p, T, H, D, S);
  if (w.all && (!ws || (uintptr_t)ws % 256)) return CFH_E_INVALID;
  PagedArgs a = {};
  a.q = (const u16*)q; a.out = (u16*)out; a.lse = lse; a.kc = k_cache; a.vc = v_cache; a.ke = k_exp; a.ve = v_exp;
  a.table = table; a.lens = seq_lens; a.cu = cu_q; a.status = status; a.q_ld = q_ld; a.o_ld = o_ld; a.bs_k = bs_k;
  a.bs_v = bs_v; a.T = T; a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.S = S; a.blocks = blocks; a.page = page;
  a.table_ld = table_ld; a.max_blocks = max_blocks; a.causal = causal ? 1 : 0;
  a.fresh = fresh;
  a.qsign = scale > 0.f ? 1 : scale < 0.f ? -1 : 0;
  a.c = scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f;
  a.po = (float*)ws;
  a.pml = (float2*)((char*)ws + w.pml);
  a.piece = p.piece; a.npiece = p.npiece; a.few = p.few;
  // j / page for j < 2^30 as j M >> (31 + l), 2^l >= page > 2^(l - 1), M = floor(2^(31 + l) / page) + 1 < 2^32: M is
  // above 2^(31 + l) / page by at most 1, which adds less than 2^30 / 2^(31 + l) < 1 / page to the quotient
  int l = 0;
  while ((1ll << l) < page) ++l;
  a.pshift = l;
  a.pmagic = (unsigned)((1ull << (31 + l)) / (unsigned)page + 1);
  hipStream_t st = (hipStream_t)stream;
  const long long groups = (long long)Hkv * p.npiece;
  a.spread = (long long)T * a.G <= (long long)tile_rows(D) * S;
  auto grid_of = [&](int tiles, bool spread) {    // (whole rounds of the XCD mapping)
    if (spread) return (groups | 1) * tiles;
    const long long per = 8 % groups == 0 ? 8 / groups : 1;
    return 8 % groups == 0 ? (tiles + per - 1) / per * 8 : groups * tiles;
  };
  if (std::max(grid_of(p.nrow, true), grid_of(p.ntile, a.spread)) > 0x7fff0000ll) return CFH_E_UNSUPPORTED;
  const unsigned more = fresh ? clearing((long long)T * H * (fresh & 2 ? 2 * D + 4 : 4)) : 0;
  if (S > ASC_FIND) {
    a.whole = (int*)((char*)ws + w.whole);
    hipLaunchKernelGGL(k_ascending, dim3(1), dim3(1024), 0, st, cu_q, S, (int*)((char*)ws + w.whole));
    CFH_LAUNCH_CHECK();
  }
  if (p.tiles) {
    a.tiles = p.ntile;
    a.work = (int)grid_of(p.ntile, a.spread);
    const dim3 grid(a.work + (p.rows ? 0 : more));
    kv_dispatch(is_bf16, f8, D, [&](auto bf, auto e8, auto d) {
      constexpr int NW = tile_rows(d.value) / 32, TK = d.value == 256 ? 32 : 64;
      hipLaunchKernelGGL((k_attn_tiles<bf.value, e8.value, d.value, NW, TK>), grid, dim3(NW * 64), 0, st, a);
    });
    CFH_LAUNCH_CHECK();
  }
  if (p.rows) {
    a.tiles = p.nrow;
    a.work = (int)grid_of(p.nrow, true);
    const dim3 grid(a.work + more);
    kv_dispatch(is_bf16, f8, D, [&](auto bf, auto e8, auto d) {
      hipLaunchKernelGGL((k_attn_rows<bf.value, e8.value, d.value>), grid, dim3(256), 0, st, a);
    });
    CFH_LAUNCH_CHECK();
  }
  if (p.npiece > 1) {
    // Up to 8 pieces a wave takes a (row, head) by itself; above that a workgroup does, of 16 waves while there are few
    // of them, else of 4 (the whole call, 16 / 4 waves a workgroup: 16 (row, head)s of 59 pieces 44.4 / 47.5 us, 192 of
    // 18 27.4 / 29.1, 960 33.5 / 31.9, 1,712 of 16 48.5 / 42.9, 3,200 45.9 / 36.7; one wave: 63, 37, 37, 45, 37)
    const long long rows = (long long)T * H;
    kv_dispatch(is_bf16, false, D, [&](auto bf, auto, auto d) {
      auto join = [&](auto w) {
        constexpr int W = w.value;
        const dim3 grid((unsigned)(W == 1 ? (rows + 3) / 4 : rows)), block(W == 1 ? 256 : W * 64);
        hipLaunchKernelGGL((k_attn_join<bf.value, d.value, W>), grid, block, 0, st, a);
      };
      if (p.npiece <= 8) join(std::integral_constant<int, 1>{});
      else if (rows <= 512) join(std::integral_constant<int, 16>{});
      else join(std::integral_constant<int, 4>{});
    });
    CFH_LAUNCH_CHECK();
  }
  return CFH_OK;
}

}  // namespace

extern "C" {

int64_t cfh_paged_attn_ws_bytes(int T, int H, int Hkv, int D, int S, int max_len) {
  if (T < 0 || H < 1 || Hkv < 1 || H % Hkv || S < 0 || max_len < 0 || D < 1) return -1;
  if (T == 0 || S == 0) return 0;
  return space(plan(T, H, Hkv, D, S, max_len), T, H, D, S).all;
}

int cfh_paged_attn(const void* q, long long q_ld, int T, int H, int Hkv, int D, int is_bf16, const void* k_cache,
                   long long bs_k, const void* v_cache, long long bs_v, const uint8_t* k_exp, const uint8_t* v_exp,
                   int blocks, int page, const int32_t* table, int table_ld, int max_blocks, const int32_t* seq_lens,
                   const int32_t* cu_q, int S, float scale, int causal, int max_len, void* out, long long o_ld,
                   float* lse, void* ws, int32_t* status, void* stream) {
  return attend(q, q_ld, T, H, Hkv, D, is_bf16, k_cache, bs_k, v_cache, bs_v, k_exp, v_exp, blocks, page, table,
                table_ld, max_blocks, seq_lens, cu_q, S, scale, causal, max_len, out, o_ld, lse, ws, status, stream, 0);
}

int cfh_paged_attn_fresh(const void* q, long long q_ld, int T, int H, int Hkv, int D, int is_bf16,
                         const void* k_cache, long long bs_k, const void* v_cache, long long bs_v,
                         const uint8_t* k_exp, const uint8_t* v_exp, int blocks, int page, const int32_t* table,
                         int table_ld, int max_blocks, const int32_t* seq_lens, const int32_t* cu_q, int S,
                         float scale, int causal, int max_len, void* out, long long o_ld, float* lse, void* ws,
                         int32_t* status, int out_too, void* stream) {
  return attend(q, q_ld, T, H, Hkv, D, is_bf16, k_cache, bs_k, v_cache, bs_v, k_exp, v_exp, blocks, page, table,
                table_ld, max_blocks, seq_lens, cu_q, S, scale, causal, max_len, out, o_ld, lse, ws, status, stream,
                out_too ? 3 : 1);
}

}  // extern "C"
