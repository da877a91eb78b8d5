// Running sums over a wave.
#pragma once
#include "cfh_common.h"

namespace {

// Running sums over the wave's lanes, each with its own, by DPP: steps of 1, 2, 4 and 8 within a row of 16 lanes, then the
// rows' last lanes (a step costs a few cycles; by ds_bpermute, some hundred).
enum { DPP_SHR1 = 0x111, DPP_SHR2 = 0x112, DPP_SHR4 = 0x114, DPP_SHR8 = 0x118, DPP_BCAST15 = 0x142, DPP_BCAST31 = 0x143 };
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long moved(unsigned long long u) {
  const unsigned lo = moved<CTRL, ROWS>((int)u), hi = moved<CTRL, ROWS>((int)(u >> 32));
  return (unsigned long long)hi << 32 | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  return __builtin_bit_cast(double, moved<CTRL, ROWS>(__builtin_bit_cast(unsigned long long, v)));
}
template <typename N>
__device__ __forceinline__ N row_scan(N v) {
  v += moved<DPP_SHR1, 0xf>(v);
  v += moved<DPP_SHR2, 0xf>(v);
  v += moved<DPP_SHR4, 0xf>(v);
  v += moved<DPP_SHR8, 0xf>(v);
  return v;
}
template <typename N>
__device__ __forceinline__ N scan64(N v) {
  v = row_scan(v);
  v += moved<DPP_BCAST15, 0xa>(v);
  v += moved<DPP_BCAST31, 0xc>(v);
  return v;
}

// a lane's value, for all
__device__ __forceinline__ double from_lane(double v, int lane) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_readlane((int)u, lane), hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// the largest of the wave's unsigned numbers, for all lanes
__device__ __forceinline__ unsigned wave_largest(unsigned v) {
  v = max(v, (unsigned)moved<DPP_SHR1, 0xf>((int)v));
  v = max(v, (unsigned)moved<DPP_SHR2, 0xf>((int)v));
  v = max(v, (unsigned)moved<DPP_SHR4, 0xf>((int)v));
  v = max(v, (unsigned)moved<DPP_SHR8, 0xf>((int)v));
  v = max(v, (unsigned)moved<DPP_BCAST15, 0xa>((int)v));
  v = max(v, (unsigned)moved<DPP_BCAST31, 0xc>((int)v));
  return __builtin_amdgcn_readlane(v, 63);
}

// Two sums over lanes in the operations of one: with a's odd groups of L lanes exchanged for b's even ones, a + b is a's two
// halves' sum in the even groups and b's in the odd ones.
template <int L>
__device__ __forceinline__ void swap_lanes(int& a, int& b) {
  static_assert(L == 16 || L == 32, "");
  const auto r = L == 32 ? __builtin_amdgcn_permlane32_swap(a, b, false, false) : __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
template <int L>
__device__ __forceinline__ void swap_add(int& a, int b) {
  swap_lanes<L>(a, b);
  a += b;
}
template <int L>
__device__ __forceinline__ void swap_add(double& a, double b) {
  const unsigned long long x = __builtin_bit_cast(unsigned long long, a), y = __builtin_bit_cast(unsigned long long, b);
  int al = (int)x, ah = (int)(x >> 32), bl = (int)y, bh = (int)(y >> 32);
  swap_lanes<L>(al, bl);
  swap_lanes<L>(ah, bh);
  a = __builtin_bit_cast(double, (unsigned long long)(unsigned)ah << 32 | (unsigned)al) +
      __builtin_bit_cast(double, (unsigned long long)(unsigned)bh << 32 | (unsigned)bl);
}

}  // namespace
