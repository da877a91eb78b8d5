// LDS tiles of 2-byte rows that MFMA operands are read from both along the rows and across them.
#pragma once
#include "cfh_common.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Four elements of one column from four rows of 16-lane blocks in LDS (lane l of a block points at row l / 4,
// columns 4 (l % 4) .. + 3 and receives column l of rows 0 .. 3).
__device__ __forceinline__ uint2 read_tr(const unsigned short* p) {
  typedef __attribute__((address_space(3))) s16x4* lptr;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)p));
}

// 16-byte chunk order within rows of D 2-byte elements: chunk c of row t lies at c ^ swz<D>(t).  LDS has 64 banks of
// 4 bytes, 16 chunks.  A 16-byte read serves 16 lanes a cycle: 16 rows with one chunk fall on different chunks.  A
// transposed read serves 32: 4 rows with 4 neighbouring chunks, and 8 rows with 2, do too (D = 64, where two rows share
// the 16 chunks: 4 rows with 4 chunks take two cycles).
template <int D>
__device__ __forceinline__ int swz(int t) {
  if (D == 64) t >>= 1;
  const int z = ((t & 3) << 2) | ((t >> 1) & 2) | ((t >> 3) & 1);
  return D == 64 ? z >> 1 : z;
}
// The order that repeats after 8 rows: reads take two cycles for one, but half as many operand addresses are kept.
__device__ __forceinline__ int swz8(int t) { return ((t & 3) << 1) | ((t >> 2) & 1); }

}  // namespace
