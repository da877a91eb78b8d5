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
__device__ __forceinline__ double moved(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = moved<CTRL, ROWS>((int)u), hi = moved<CTRL, ROWS>((int)(u >> 32));
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <typename N>
__device__ __forceinline__ N scan64(N v) {
  v += moved<DPP_SHR1, 0xf>(v);
  v += moved<DPP_SHR2, 0xf>(v);
  v += moved<DPP_SHR4, 0xf>(v);
  v += moved<DPP_SHR8, 0xf>(v);
  v += moved<DPP_BCAST15, 0xa>(v);
  v += moved<DPP_BCAST31, 0xc>(v);
  return v;
}

}  // namespace
