// Rows times a matrix of 4-bit weights with a scale for each group of columns, on MI355X: the drafter's head at a quarter of
// its fp16 bytes.
//
//   y[m][n] = sum_g s[n][g] sum_{k in group g} (u[n][k] - 8) x[m][k],   u in 0 .. 15
//
// Weight rows are u[n][K / 2] bytes, column 2 i in the low half of byte i; scales s[n][K / group] fp16; x and y fp16.  The
// whole numbers u - 8 are exact in fp16, products and sums are fp32 (MFMA), each group's sum is scaled in fp32, and the
// result is rounded once.
//
// A wave takes 16 weight rows and 128 columns a step: 16 bytes a lane (row lane % 16, columns 32 (lane / 16) ..), 4 x 4
// words of the four lanes of a row exchanged so that word j of lane (n, kg) holds columns 32 j + 8 kg .. + 7 of the step:
// one 16 x 16 x 32 MFMA a word, and no MFMA mixes groups of 32 columns or more.
#include <math.h>

#include <algorithm>

#include "cfh_host.h"
#include "cfh_common.h"

namespace {

typedef unsigned short u16;
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));

constexpr int MV_W = 8;          // waves a workgroup
constexpr int MV_PF = 4;         // steps a wave has in flight
constexpr int MV_ROWS = 16;      // rows of x a launch at most
constexpr int MV_LDS = 150 * 1024;

struct MvArgs {
  const h16* x;                  // [M][ld_x]
  const h16* a;                  // rows behind x's columns, gathered: a[ids[m]][r], or null
  const int* ids;
  const uint8_t* w;              // [n][ld_w] bytes
  const h16* s;                  // [n][ld_s]
  h16* y;                        // [M][ld_y]
  long long ld_x, ld_y;
  int ids_stride, a_rows, r;
  int M, d, K, n, ld_w, ld_s, ks; // K = d + r columns; waves a tile of 16 weight rows
};

// The eight weights of a word as whole numbers in fp16, in the order 0 4 1 5 2 6 3 7: 0x6400 + u is 1024 + u.
__device__ __forceinline__ h16x8 whole8(unsigned w) {
  h16x8 out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const h16x2 v = __builtin_bit_cast(h16x2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u) - (h16x2){(h16)1032.f, (h16)1032.f};
    out[2 * i] = v[0];
    out[2 * i + 1] = v[1];
  }
  return out;
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

// G: columns a scale.
template <int G>
__global__ void __launch_bounds__(MV_W * 64) k_matvec4(MvArgs a) {
  extern __shared__ __attribute__((aligned(16))) h16 xs[];     // [M][K + 8], eights of columns in the order 0 4 1 5 2 6 3 7
  __shared__ f32x4 part[MV_W][64];
  constexpr int S = 128 / G;     // scales a step
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, kg = lane >> 4;
  const int tile = blockIdx.x * (MV_W / a.ks) + wave / a.ks, part_k = wave % a.ks;
  const int steps = a.K / 128, s0 = steps * part_k / a.ks, s1 = steps * (part_k + 1) / a.ks;
  const int col = tile * 16 + (lane & 15);
  const size_t row = min(col, a.n - 1);              // (lanes behind the last row read it again)
  const v4u* w = (const v4u*)(a.w + row * a.ld_w) + kg;
  const h16* sc = a.s + row * a.ld_s;
  v4u buf[MV_PF];
  struct Sc { h16 v[S]; } sbuf[MV_PF];
  auto fetch = [&](int p, int st) {
    const int c = min(st, s1 - 1);
    buf[p] = w[c * 4];
    sbuf[p] = *(const Sc*)(sc + c * S);
  };
  if (s1 > s0) {
#pragma unroll
    for (int p = 0; p < MV_PF; ++p) fetch(p, s0 + p);
  }
  const int ldx = a.K + 8, eights = a.K / 8;
  for (int i = threadIdx.x; i < a.M * eights; i += MV_W * 64) {
    const int m = i / eights, k = (i - m * eights) * 8;
    h16x8 v;
    if (k < a.d) v = *(const h16x8*)(a.x + m * a.ld_x + k);
    else v = *(const h16x8*)(a.a + (size_t)min(max(a.ids[m * a.ids_stride], 0), a.a_rows - 1) * a.r + (k - a.d));
    *(h16x8*)(xs + m * ldx + k) = __builtin_shufflevector(v, v, 0, 4, 1, 5, 2, 6, 3, 7);
  }
  __syncthreads();
  const int m = lane & 15;
  const h16* xr = xs + (m < a.M ? m : 0) * ldx + kg * 8;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int st = s0; st < s1; st += MV_PF) {
#pragma unroll
    for (int p = 0; p < MV_PF; ++p) {
      unsigned q[4] = {buf[p][0], buf[p][1], buf[p][2], buf[p][3]};
      const Sc s = sbuf[p];
      const int here = st + p;
      fetch(p, here + MV_PF);
      swap4(q);
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum = mfma_f16(*(const h16x8*)(xr + min(here, s1 - 1) * 128 + j * 32), whole8(q[j]), sum);
        if ((j + 1) % (G / 32) == 0) {
          const float f = here < s1 ? (float)s.v[j / (G / 32)] : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = here < s1 ? fmaf(f, sum[e], acc[e]) : acc[e];
          sum = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
  }
  if (a.ks > 1) {                // the waves of a tile joined in their order
    part[wave][lane] = acc;
    __syncthreads();
    if (part_k) return;
    for (int i = 1; i < a.ks; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += part[wave + i][lane][e];
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

// eight columns a thread, group / 8 threads a group
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
  const int most = (int)std::min<long long>(MV_ROWS, MV_LDS / ((K + 8) * 2));
  if (most < 1) return CFH_E_UNSUPPORTED;
  const long long tiles = ((long long)n + 15) / 16;
  int ks = 1;
  while (ks < MV_W && tiles * ks < 2048) ks *= 2;
  for (int m0 = 0; m0 < M; m0 += most) {
    MvArgs v = {};
    v.M = std::min(most, M - m0);
    v.x = (const h16*)x + m0 * ld_x; v.ld_x = ld_x; v.d = d; v.K = (int)K; v.n = n;
    v.w = w; v.ld_w = ld_w; v.s = (const h16*)scale; v.ld_s = ld_s;
    v.a = (const h16*)a; v.a_rows = a_rows; v.r = r; v.ids = a_ids + (long long)m0 * a_ids_stride; v.ids_stride = a_ids_stride;
    v.y = (h16*)y + m0 * ld_y; v.ld_y = ld_y; v.ks = ks;
    const dim3 grid((unsigned)((tiles * ks + MV_W - 1) / MV_W)), block(MV_W * 64);
    const size_t lds = (size_t)v.M * (K + 8) * 2;
    const hipStream_t st = (hipStream_t)stream;
    auto* fn = group == 32 ? k_matvec4<32> : group == 64 ? k_matvec4<64> : k_matvec4<128>;
    if (lds > 49152) CFH_HIP(hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(fn, grid, block, lds, st, v);
    CFH_LAUNCH_CHECK();
  }
  return CFH_OK;
}

}  // extern "C"
