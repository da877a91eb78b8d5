// Device and host helpers shared by the paged cache's kernels (rows in and out, attention).
#pragma once
#include <math.h>

#include <type_traits>

#include "cfh_common.h"

namespace {

typedef unsigned short u16;
typedef float f32x2k __attribute__((ext_vector_type(2)));
typedef __bf16 b16x2k __attribute__((ext_vector_type(2)));
typedef _Float16 h16x2k __attribute__((ext_vector_type(2)));

// Two floats rounded to the 2-byte type (nearest even; NaN and infinities kept) in one word.
template <bool BF>
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
  const f32x2k v = {lo, hi};
  if constexpr (BF) return __builtin_bit_cast(unsigned, __builtin_convertvector(v, b16x2k));
  else return __builtin_bit_cast(unsigned, __builtin_convertvector(v, h16x2k));
}

// Eight 2-byte elements as floats.
template <bool BF>
__device__ __forceinline__ void widen8(const uint4& r, float (&x)[8]) {
  const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const h16x2k v = __builtin_bit_cast(h16x2k, w[i]);
      x[2 * i] = (float)v[0];
      x[2 * i + 1] = (float)v[1];
    }
  }
}

// Four floats of magnitude up to 448 (or NaN) as e4m3, nearest even.
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Eight e4m3 elements times 2^(code - 127), rounded to the 2-byte type (nearest even): one conversion for two.
template <bool BF>
__device__ __forceinline__ uint4 dequant8(const uint2& w, int code) {
  const float s = __uint_as_float((unsigned)code << 23);
  auto two = [&](unsigned word, auto hi) {
    if constexpr (BF) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, s, hi.value));
    else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, s, hi.value));
  };
  return make_uint4(two(w.x, std::false_type{}), two(w.x, std::true_type{}), two(w.y, std::false_type{}),
                    two(w.y, std::true_type{}));
}

// f(bf16?, 8-bit cache?, head width) with the three as types.
template <typename F>
inline void kv_dispatch(bool bf, bool f8, int D, F f) {
  auto d = [&](auto b, auto q) {
    if (D == 64) f(b, q, std::integral_constant<int, 64>{});
    else if (D == 128) f(b, q, std::integral_constant<int, 128>{});
    else f(b, q, std::integral_constant<int, 256>{});
  };
  auto q = [&](auto b) { f8 ? d(b, std::true_type{}) : d(b, std::false_type{}); };
  bf ? q(std::true_type{}) : q(std::false_type{});
}

}  // namespace
