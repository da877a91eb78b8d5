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

// 16-byte chunk order within a row of a multiple of 128 bytes: chunk c of row t lies at c ^ swz(t).  Eight rows
// with one chunk (operands read along the rows), and four rows with two neighbouring chunks (transposed reads,
// or 8-byte pieces), each cover all 128 bytes of the banks.
__device__ __forceinline__ int swz(int t) { return ((t & 3) << 1) | ((t >> 2) & 1); }

}  // namespace
