// Rows times a matrix of 4-bit weights with a scale for each group of columns, on MI355X: the drafter's head at a quarter of
// its fp16 bytes.
//
//   y[m][n] = sum_g s[n][g] sum_{k in group g} (u[n][k] - 8) x[m][k],   u in 0 .. 15
//
// Weight rows are u[n][K / 2] bytes, column 2 i in the low half of byte i; scales s[n][K / group] fp16; x and y fp16.  Four bits
// as the last of 0x6400 are the fp16 number 1024 + u, and at bits 4 .. 7 of 0x5400 64 + u: one shift a word, and two operations
// (and-or, a packed addition of -1032 or -72, which is exact) for two weights.  Products are exact in fp32 and sums are fp32 (MFMA),
// of the terms (u - 8) x themselves: G adds of at most 2^-23 of the sum of their magnitudes a group.  (16 + u, with 24 sum x
// taken off behind the products, takes no fewer operations, and a column whose weight is 8 would cost 24 |x| 2^-24 of the
// sum: with an x of 60,000 beside ones of 1, many times the rounding to fp16.)
//
// A wave takes 16 weight rows and 256 columns at a time, in two loads of 8 rows and 128 bytes each: whole lines (a bare read
// of such a matrix reached 5.9 TB/s so, 5.2 with 16 rows and 64 bytes a load).  Lanes 8 apart exchange halves, so that lane
// (n, kg) has 32 bytes of row n.  With groups below 128 columns they are 64 kg .. of the 256, and the 4 x 4 words of the four lanes of a
// row are exchanged too, so that an MFMA's 32 columns lie side by side and mix no groups; with 128 they are columns 32 kg .. of both
// halves, and the MFMAs take them as they are.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "cfh_host.h"
#include "cfh_common.h"

namespace {

typedef unsigned short u16;
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));

constexpr int MV_ROWS = 16;      // rows of x a launch at most
constexpr long long MV_LDS = 158 * 1024, MV_HALF = 79 * 1024;   // one workgroup a compute unit, two

struct MvArgs {
  const h16* x;                  // [M][ld_x]
  const h16* a;                  // rows behind x's columns, gathered: a[ids[m]][r], or null
  const int* ids;
  const uint8_t* w;              // [n][ld_w] bytes
  const h16* s;                  // [n][ld_s]
  h16* y;                        // [M][ld_y]
  long long ld_x, ld_y;
  int ids_stride, a_rows, r;
  int M, d, K, n, ld_w, ld_s;    // K = d + r columns
  int ks, chunk;                 // waves a tile of 16 weight rows; steps of 128 columns whose x lies in LDS at a time
};

// The eight weights of a word as fp16 numbers u - 8, in the order 0 4 1 5 2 6 3 7.  (`e` is 0x64006400 and 0x54005400 in vector
// registers and the masks in scalar ones: and-or is then one operation, which takes no literals.)
struct Exponents { unsigned at0, at4; };
__device__ __forceinline__ h16x8 less8(unsigned w, const Exponents& e) {
  auto low = [&](unsigned v) __attribute__((always_inline)) {    // bits 0 .. 3 of both halves
    const unsigned u = (v & 0x000f000fu) | e.at0;
    return __builtin_bit_cast(h16x2, u) + h16x2{(h16)-1032.f, (h16)-1032.f};
  };
  auto high = [&](unsigned v) __attribute__((always_inline)) {   // bits 4 .. 7
    const unsigned u = (v & 0x00f000f0u) | e.at4;
    return __builtin_bit_cast(h16x2, u) + h16x2{(h16)-72.f, (h16)-72.f};
  };
  const unsigned w8 = w >> 8;
  const h16x2 a = low(w), b = high(w), c = low(w8), d = high(w8);
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// Words of four lanes (kg = lane / 16) transposed: word j of lane kg becomes word kg of lane j.
__device__ __forceinline__ void swap4(unsigned (&w)[4]) {
  auto s32 = [](unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0]; b = r[1];
  };
  auto s16 = [](unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0]; b = r[1];
  };
  s32(w[0], w[2]);
  s32(w[1], w[3]);
  s16(w[0], w[1]);
  s16(w[2], w[3]);
}

// G: columns a scale; NW waves.  Bound by the weights' bytes where they are many: 62,642 rows of 2,560 columns, one row of x, 18-20
// us with the weights in memory (4.0-4.5 TB/s), 15 where the caches hold them from the call before (5.5); of 5,376, four rows, 42
// (4.3) and 31 (5.8).  By the launch, x's way into LDS and the joined parts where they are few: 8,191 rows of 4,096, 16 rows of x, 10
// us for 19 MB, 8.5 from the caches.  A step of 128 columns costs a wave 52 to 70 vector operations (61 with groups of 64) beside its
// loads, so that two steps' loads in flight are enough (four cost one row of x 2 us, as registers leave fewer waves).
template <int G, int NW>
__global__ void __launch_bounds__(NW * 64, 4) k_matvec4(MvArgs a) {
  // x [M][chunk columns + 8], eights of them in the order 0 4 1 5 2 6 3 7
  extern __shared__ __attribute__((aligned(16))) h16 xs[];
  constexpr int S = 128 / G;     // scales a step
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, kg = lane >> 4;
  const int tile = blockIdx.x * (NW / a.ks) + wave / a.ks, part_k = wave % a.ks;
  const int steps = a.K / 128, s0 = steps * part_k / a.ks, s1 = steps * (part_k + 1) / a.ks;
  const int col = tile * 16 + (lane & 15);
  const size_t row = min(col, a.n - 1);              // (lanes behind the last row read it again)
  struct __attribute__((packed, aligned(256 / G))) Sc { h16 v[S]; };
  struct __attribute__((packed, aligned(256 / G))) Sc2 { unsigned v[S]; };   // of two steps (as words: halves would be taken apart,
                                                                             // and so waited for, where they are loaded)
  const h16* sc = a.s + row * a.ld_s + s0 * S;
  // an odd step first, by 64 bytes of each of the 16 rows; then pairs of steps, the next one in flight
  const bool odd = (s1 - s0) % 2;
  const int pairs = (s1 - s0) / 2;
  struct Pair { v4u lo, hi; Sc2 s; };                // rows lane % 8 and 8 more
  const int unit = G < 128 ? lane / 8 : kg + 4 * (lane / 8 % 2), r8 = tile * 16 + lane % 8;
  const v4u* lo = (const v4u*)(a.w + (size_t)min(r8, a.n - 1) * a.ld_w) + (s0 + odd) * 4 + unit;
  const v4u* hi = (const v4u*)(a.w + (size_t)min(r8 + 8, a.n - 1) * a.ld_w) + (s0 + odd) * 4 + unit;
  v4u first = {};
  Sc first_s = {};
  if (odd) {
    first = ((const v4u*)(a.w + row * a.ld_w))[s0 * 4 + kg];
    first_s = *(const Sc*)sc;
    sc += S;
  }
  Pair next = {};
  if (pairs) next = {lo[0], hi[0], *(const Sc2*)sc};

  // x's columns 128 c0 .. 128 c1 into LDS
  const int ldx = a.chunk * 128 + 8;
  auto stage = [&](int c0, int c1) __attribute__((always_inline)) {
    constexpr int XB = 4;                            // eights of columns a thread has in flight (16 rows of 4,096: 9.7 us; 2: 10.2; 8: 9.7)
    const int eights = (c1 - c0) * 16, all = a.M * eights;
    for (int i0 = threadIdx.x; i0 < all; i0 += XB * NW * 64) {
      h16x8 v[XB];
      int to[XB];
#pragma unroll
      for (int u = 0; u < XB; ++u) {
        const int i = min(i0 + u * NW * 64, all - 1), m = i / eights, here = (i - m * eights) * 8, k = c0 * 128 + here;
        to[u] = m * ldx + here;
        v[u] = k < a.d ? *(const h16x8*)(a.x + m * a.ld_x + k)
                       : *(const h16x8*)(a.a + (size_t)min(max(a.ids[m * a.ids_stride], 0), a.a_rows - 1) * a.r + (k - a.d));
      }
#pragma unroll
      for (int u = 0; u < XB; ++u) *(h16x8*)(xs + to[u]) = __builtin_shufflevector(v[u], v[u], 0, 4, 1, 5, 2, 6, 3, 7);
    }
    __syncthreads();
  };
  const int m = lane & 15;
  const h16* const x0 = xs + (m < a.M ? m : 0) * ldx + kg * (G < 128 ? 8 : 32);
  const h16* xr = x0;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  Exponents ex = {0x64006400u, 0x54005400u};
  asm("" : "+v"(ex.at0), "+v"(ex.at4));
  auto scaled = [&](float f, const f32x4& sum) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, sum[e], acc[e]);
  };
  auto one_step = [&]() __attribute__((always_inline)) {
    unsigned q[4] = {first[0], first[1], first[2], first[3]};
    if (G < 128) swap4(q);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j % (G / 32) == 0) sum = {0.f, 0.f, 0.f, 0.f};
      sum = mfma_f16(*(const h16x8*)(xr + j * (G < 128 ? 32 : 8)), less8(q[j], ex), sum);
      if ((j + 1) % (G / 32) == 0) scaled((float)first_s.v[j / (G / 32)], sum);
    }
    xr += 128;
  };
  auto two_steps = [&](const Pair& b) __attribute__((always_inline)) {
    constexpr int ROR8 = 0x128;                      // lanes 8 apart
    unsigned q[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q[0][j] = __builtin_amdgcn_update_dpp((int)b.lo[j], (int)b.hi[j], ROR8, 0xf, 0xc, false);
      q[1][j] = __builtin_amdgcn_update_dpp((int)b.hi[j], (int)b.lo[j], ROR8, 0xf, 0x3, false);
    }
    if (G < 128) {
      swap4(q[0]);
      swap4(q[1]);
    }
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {                    // 32 columns each
      if (i % (G / 32) == 0) sum = {0.f, 0.f, 0.f, 0.f};
      const unsigned word = G < 128 ? q[i & 1][i >> 1] : q[i >> 2][i & 3];
      sum = mfma_f16(*(const h16x8*)(xr + (G < 128 ? i * 32 : i / 4 * 128 + i % 4 * 8)), less8(word, ex), sum);
      if ((i + 1) % (G / 32) == 0) {
        const int at = i / (G / 32);
        scaled((float)__builtin_bit_cast(h16, (u16)(b.s.v[at / 2] >> (16 * (at % 2)))), sum);
      }
    }
    xr += 256;
  };
  // the first chunk has the odd step; split waves have one chunk, of all columns
  for (int c0 = 0, c1; c0 < steps; c0 = c1) {
    const int extra = c0 == 0 && odd && a.ks == 1;
    c1 = a.ks > 1 ? steps : min(steps, c0 + extra + (a.chunk - extra) / 2 * 2);
    if (c0) __syncthreads();                         // (the chunk before is done with)
    stage(c0, c1);
    xr = x0 + (a.ks > 1 ? s0 : 0) * 128;
    if (c0 == 0 && odd) one_step();
    // (the last pair of all: behind the loop, which has no branch around its loads)
    const int here = (a.ks > 1 ? pairs : (c1 - c0 - extra) / 2) - (c1 == steps ? 1 : 0);
    for (int i = 0; i < here; ++i) {
      const Pair now = next;
      lo += 8;
      hi += 8;
      sc += 2 * S;
      next = {*lo, *hi, *(const Sc2*)sc};
      asm volatile("" ::: "memory");                 // (the loads together, not each where its words are used)
      two_steps(now);
    }
  }
  if (pairs) two_steps(next);
  if (a.ks > 1) {                // the waves of a tile joined in their order
    f32x4* part = (f32x4*)xs;    // (x's place: NW KB)
    __syncthreads();
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (part_k) return;
    for (int i = 1; i < a.ks; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += part[(wave + i) * 64 + lane][e];
  }
  if (col >= a.n) return;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (4 * kg + e < a.M) a.y[(4 * kg + e) * a.ld_y + col] = (h16)acc[e];
}

// A group of weights to whole numbers -7 .. 7 (stored + 8) times the least fp16 scale whose seven reach its largest
// magnitude, so that no weight is off by more than half a scale.  A group with a NaN or an infinity has a NaN scale.
struct QuantArgs {
  const h16* w;                  // [rows][d]
  const h16* w2;                 // [rows][r], the columns behind, or null
  const int* sl;                 // rows taken, or null: all
  uint8_t* q;
  h16* s;
  int n, d, r, group;
};

// Eight columns a thread, group / 8 threads a group: run once, when a head is laid out.
__global__ void __launch_bounds__(256) k_quantize4(QuantArgs a) {
  const int K = a.d + a.r, per = K / 8;
  const size_t all = (size_t)a.n * per;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (all + 63) / 64 * 64; i += (size_t)gridDim.x * 256) {
    const size_t c = min(i, all - 1);
    const int row = (int)(c / per), k = (int)(c - (size_t)row * per) * 8;
    const size_t src = a.sl ? (size_t)a.sl[row] : (size_t)row;
    const h16x8 v = k < a.d ? *(const h16x8*)(a.w + src * a.d + k) : *(const h16x8*)(a.w2 + src * a.r + (k - a.d));
    float most = 0.f;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most = fmaxf(most, fabsf((float)v[e]));
      odd |= !(fabsf((float)v[e]) < INFINITY);
    }
    int any = odd;
    for (int off = 1; off < a.group / 8; off <<= 1) {
      most = fmaxf(most, __shfl_xor(most, off));
      any |= __shfl_xor(any, off);
    }
    h16 s = any ? (h16)__builtin_nanf("") : (h16)(most / 7.f);
    if (!any && (float)s * 7.f < most) s = __builtin_bit_cast(h16, (u16)(__builtin_bit_cast(u16, s) + 1));
    const float f = (float)s;
    unsigned word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = any || f == 0.f ? 0.f : fminf(fmaxf(rintf((float)v[e] / f), -7.f), 7.f);
      word |= (unsigned)((int)q + 8) << (4 * e);
    }
    if (i >= all) continue;
    *(unsigned*)(a.q + (size_t)row * (K / 2) + k / 2) = word;
    if (k % a.group == 0) a.s[(size_t)row * (K / a.group) + k / a.group] = s;
  }
}

}  // namespace

extern "C" {

int cfh_quantize4(const void* w, const void* w2, const int32_t* rows, int n, int d, int r, int group, uint8_t* q, void* scale,
                  void* stream) {
  if (n < 0 || d < 1 || r < 0 || (group != 32 && group != 64 && group != 128)) return CFH_E_INVALID;
  if (d % group || r % group || (d + r) % 128) return CFH_E_UNSUPPORTED;
  if (n == 0) return CFH_OK;
  if (!w || !q || !scale || (r > 0 && !w2) || ((uintptr_t)w | (uintptr_t)w2) % 16 || (uintptr_t)q % 4) return CFH_E_INVALID;
  QuantArgs a = {(const h16*)w, (const h16*)w2, rows, q, (h16*)scale, n, d, r, group};
  const long long work = (long long)n * ((d + r) / 8);
  const unsigned grid = (unsigned)std::min<long long>((work + 255) / 256, 8192);
  hipLaunchKernelGGL(k_quantize4, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

int cfh_matvec4(const void* x, long long ld_x, int M, int d, const uint8_t* w, int ld_w, const void* scale, int ld_s, int group,
                int n, const void* a, int a_rows, const int32_t* a_ids, int a_ids_stride, int r, void* y, long long ld_y,
                void* stream) {
  const long long K = (long long)d + r;
  if (M < 0 || n < 0 || d < 1 || r < 0 || (group != 32 && group != 64 && group != 128)) return CFH_E_INVALID;
  if (K > 65536 || K % 128 || d % 8) return CFH_E_UNSUPPORTED;
  if (M == 0 || n == 0) return CFH_OK;
  if (!x || !w || !scale || !y || ld_x < d || ld_x % 8 || ld_y < n || ld_w < K / 2 || ld_w % 16 || ld_s < K / group ||
      ld_s % (128 / group) || (uintptr_t)x % 16 || (uintptr_t)w % 16 || (uintptr_t)scale % (256 / group))
    return CFH_E_INVALID;
  if (r > 0 && (!a || !a_ids || a_rows < 1 || (uintptr_t)a % 16 || r % 8)) return CFH_E_INVALID;
  const long long tiles = ((long long)n + 15) / 16, steps = K / 128;
  auto lds_of = [](int rows, long long c) { return rows * (c * 128 + 8) * 2; };
  for (int m0 = 0, rows; m0 < M; m0 += rows) {
    rows = std::min(MV_ROWS, M - m0);
    MvArgs v = {};
    v.x = (const h16*)x + m0 * ld_x; v.ld_x = ld_x; v.d = d; v.K = (int)K; v.n = n;
    v.w = w; v.ld_w = ld_w; v.s = (const h16*)scale; v.ld_s = ld_s;
    v.a = (const h16*)a; v.a_rows = a_rows; v.r = r; v.ids = a_ids + (long long)m0 * a_ids_stride; v.ids_stride = a_ids_stride;
    v.y = (h16*)y + m0 * ld_y; v.ld_y = ld_y;
    auto launch = [&](auto g, auto nw) -> int {
      constexpr int NW = nw.value;
      // K split over a workgroup's waves until there are 200 workgroups: 16 rows times 8,191 x 4,096, 9.7 us in 8 parts, 11.7 in
      // 4, 14.7 in 16, 29 in one; one row times 62,642 x 2,560, 18.1 in one, 20.6 in 2.  Unsplit, x that two workgroups of a compute
      // unit cannot both hold comes in chunks (16 rows of 5,376: 48 us; in two launches of 8 rows 82).
      int ks = 1;
      while (ks < NW && tiles * ks < 200 * NW) ks *= 2;
      long long c = steps;
      if (ks > 1) {
        while (rows > 1 && lds_of(rows, c) > MV_LDS) rows = (rows + 1) / 2;
        if (lds_of(rows, c) > MV_LDS) ks = 1;
      }
      if (ks == 1)
        while (lds_of(rows, c) > MV_HALF) c = (c + 1) / 2;
      v.M = rows; v.ks = ks; v.chunk = (int)c;
      const size_t lds = std::max<size_t>(lds_of(rows, c), ks > 1 ? (size_t)NW * 1024 : (size_t)0);
      auto* fn = k_matvec4<g.value, NW>;
      if (lds > 49152) CFH_HIP(hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
      hipLaunchKernelGGL(fn, dim3((unsigned)((tiles * ks + NW - 1) / NW)), dim3(NW * 64), lds, (hipStream_t)stream, v);
      CFH_LAUNCH_CHECK();
      return CFH_OK;
    };
    auto of_group = [&](auto nw) {
      return group == 32 ? launch(std::integral_constant<int, 32>{}, nw) : group == 64 ? launch(std::integral_constant<int, 64>{}, nw)
                                                                              : launch(std::integral_constant<int, 128>{}, nw);
    };
    // 16 waves share x where two workgroups of 8 do not fit: 62,642 x 5,376, 16 rows 47.9 us (of 8 waves 48.5), with the weights in
    // the caches 36.2 (40.3); 8 rows 46.1 (45.3), 33.5 (35.4)
    const bool big = lds_of(rows, steps) > MV_HALF;
    if (int rc = big ? of_group(std::integral_constant<int, 16>{}) : of_group(std::integral_constant<int, 8>{})) return rc;
  }
  return CFH_OK;
}

}  // extern "C"
