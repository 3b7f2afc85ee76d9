// Shared definitions of the 4-bit weights: the packed layout and the widening
// of E2M1 codes.
//
// Layout: 16-row x 128-column blocks of 1 KiB, [ceil(n/16)][ceil(k/128)].  Lane l
// of a wave owns 16 bytes: dword j holds the eight codes of row l%16, columns
// 32 j + 8 (l/16) .. +7, i.e. its B operand of the j-th v_mfma_f32_16x16x32_bf16
// of the block; a wave's 128-bit loads fetch one contiguous KiB.  Each MFMA spans
// 32 neighbouring columns, so it lies inside one group for every group size, and
// the group's scale multiplies its fp32 result instead of the widened codes.
//
// Scales: per block [16 rows][S groups] bf16 (S = 128 / group): the accumulator lane
// l holds sums of row l%16, whose scales are one load of 2 S bytes.
#pragma once

#include "pgs_linear.h"

namespace pgs {

__host__ __device__ inline int64_t fp4_kblocks(int64_t k) { return (k + 127) / 128; }
__host__ __device__ inline int64_t fp4_blocks(int64_t n, int64_t k) { return ((n + 15) / 16) * fp4_kblocks(k); }

// eight codes -> eight bf16 (exact), the low nibble first: four
// v_cvt_scalef32_pk_bf16_fp4, where integer codes would need about four times as
// many instructions (extract, convert, pack)
__device__ __forceinline__ bf16x8 fp4x8_to_bf16x8(uint32_t d) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, 1.0f, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, 1.0f, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, 1.0f, 2);
  const bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, 1.0f, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

__device__ __forceinline__ void fp4x8_to_f32(uint32_t d, float* f) {
  const bf16x8 v = fp4x8_to_bf16x8(d);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(v[i]);
}

}  // namespace pgs
