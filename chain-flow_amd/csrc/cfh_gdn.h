// Device helpers shared by the gated delta net's kernels (tree, recurrent and chunked forms).
#pragma once
#include "cfh_common.h"

namespace {

constexpr int GDN_DK = 128;    // the q / k head width

__device__ __forceinline__ float bf16f(uint16_t b) { return __uint_as_float((unsigned)b << 16); }

// round to nearest even, as torch's cast does: gfx950 converts in hardware (v_cvt_pk_bf16_f32, two
// values an instruction), inf unchanged, NaN stays NaN
__device__ __forceinline__ float round_bf16(float x) { return (float)(__bf16)x; }
__device__ __forceinline__ uint16_t to_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
// two values rounded by one instruction (rounded one by one, each takes one and two more to join them)
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  const f32x2 v = {lo, hi};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, b16x2));
}

// Element order of k and q in LDS: the lanes' first float4s, then their second ones.
template <typename T>
__device__ __forceinline__ int kq_pos(int x) {
  return sizeof(T) == 2 ? ((x >> 2) & 1) * 64 + (x >> 3) * 4 + (x & 3) : x;
}

// One lane's share of a state row: 8 elements from global memory and back.
__device__ __forceinline__ void row_load(const uint16_t* row, int p, uint4 (&r)[1]) { r[0] = *(const uint4*)(row + 8 * p); }
__device__ __forceinline__ void row_load(const float* row, int p, uint4 (&r)[2]) {
  r[0] = *(const uint4*)(row + 4 * p);
  r[1] = *(const uint4*)(row + 64 + 4 * p);
}
__device__ __forceinline__ void row_store(uint16_t* row, int p, const uint4 (&r)[1]) { *(uint4*)(row + 8 * p) = r[0]; }
__device__ __forceinline__ void row_store(float* row, int p, const uint4 (&r)[2]) {
  *(uint4*)(row + 4 * p) = r[0];
  *(uint4*)(row + 64 + 4 * p) = r[1];
}
__device__ __forceinline__ void row_widen(const uint4 (&r)[1], float (&S)[8]) {
  const unsigned w[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    S[2 * e] = __uint_as_float(w[e] << 16);
    S[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void row_widen(const uint4 (&r)[2], float (&S)[8]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    S[4 * q] = __uint_as_float(r[q].x); S[4 * q + 1] = __uint_as_float(r[q].y);
    S[4 * q + 2] = __uint_as_float(r[q].z); S[4 * q + 3] = __uint_as_float(r[q].w);
  }
}
__device__ __forceinline__ void row_pack(const float (&S)[8], uint4 (&r)[1]) {
  r[0] = make_uint4(pack_bf16(S[0], S[1]), pack_bf16(S[2], S[3]), pack_bf16(S[4], S[5]), pack_bf16(S[6], S[7]));
}
__device__ __forceinline__ void row_pack(const float (&S)[8], uint4 (&r)[2]) {
#pragma unroll
  for (int q = 0; q < 2; ++q)
    r[q] = make_uint4(__float_as_uint(S[4 * q]), __float_as_uint(S[4 * q + 1]), __float_as_uint(S[4 * q + 2]),
                      __float_as_uint(S[4 * q + 3]));
}

}  // namespace
