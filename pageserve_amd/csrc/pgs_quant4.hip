// 4-bit weights with group scales: quantizer and dequantizer (gfx950).
//
// Per group of G columns of a row: scale s = bf16(max(absmax, 1e-8) / 6) and
// per weight the E2M1 value nearest to w / s, ties to the even code.  The
// midpoints between neighbouring values (1/4, 3/4, 5/4, 7/4, 5/2, 7/2, 5) have at
// most three significant bits and s has eight, so their products are exact in
// fp32 and comparing |w| with them decides the code without a division or a
// rounding: code = [a > s/4] + [a >= 3s/4] + [a > 5s/4] + ... (> where the lower
// neighbour is even, >= where the upper one is).
//
// One wave per 16-row x 128-column block of the packed layout (pgs_fp4.h): lane l
// owns row l%16 and of each 32 columns j the eight from 32 j + 8 (l/16), which are
// dword j of its 16 bytes, so the block leaves as one contiguous KiB and nothing
// crosses waves.  A group's maximum is the lane's own over its dwords, then two
// lane exchanges over the four lanes of the row.  Bound by memory: each weight is
// read once into registers (all of a lane's loads in flight together).  Measured at 11008 x
// 2048 in fp32, groups of 128: 22.9 us, 4.5 TB/s; back to fp32 17.9 us, 5.7 TB/s.
#include "pgs_fp4.h"

namespace pgs {
namespace {

constexpr int kQ4Threads = 256;  // four blocks, neighbours along K

__device__ __forceinline__ float xor_max_bits(uint32_t v) {
  v = max(v, __shfl_xor(v, 16));
  v = max(v, __shfl_xor(v, 32));
  return __uint_as_float(v);
}

// |w| as ordered bits (an infinity above every finite value, a NaN above that)
// -> the group's scale: a NaN stays one
__device__ __forceinline__ uint16_t group_scale(uint32_t bits) {
  const float amax = __uint_as_float(bits);
  return f32_to_bf16_bits((bits > 0x7f800000u ? amax : fmaxf(amax, 1e-8f)) / 6.0f);
}

__device__ __forceinline__ uint32_t code4(float w, float s) {
  const float a = fabsf(w);
  const uint32_t c = (a > 0.25f * s) + (a >= 0.75f * s) + (a > 1.25f * s) + (a >= 1.75f * s) + (a > 2.5f * s) +
                     (a >= 3.5f * s) + (a > 5.0f * s);
  return c | (c && w < 0.f ? 8u : 0u);
}

template <bool BF16, int S>  // S: groups of a block's row, 128 / group
__global__ __launch_bounds__(kQ4Threads) void quantize4_kernel(const void* __restrict__ w, int64_t n, int k,
                                                               int64_t blocks, uint4* __restrict__ qp,
                                                               uint16_t* __restrict__ sp) {
  const int lane = threadIdx.x & 63;
  const int64_t blk = static_cast<int64_t>(blockIdx.x) * (kQ4Threads / 64) + uniform(static_cast<int>(threadIdx.x >> 6));
  if (blk >= blocks) return;
  const int kb = static_cast<int>(fp4_kblocks(k));
  const int64_t trow = blk / kb;
  const int c0 = static_cast<int>(blk - trow * kb) * 128;
  const int64_t row = trow * 16 + (lane & 15);
  const int col = c0 + 8 * (lane >> 4);  // of dword 0; dword j: + 32 j
  float f[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // (k is a multiple of 8: the eight columns are all inside or all padding)
    const bool in = row < n && col + 32 * j < k;
    const int64_t e = in ? row * k + col + 32 * j : 0;
    if constexpr (BF16) {
      u32x4 v = in ? ld16_stream(static_cast<const uint16_t*>(w) + e) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[j][2 * i] = __uint_as_float(v[i] << 16);
        f[j][2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
      }
    } else {
      const float* p = static_cast<const float*>(w) + e;
      const u32x4 a = in ? ld16_stream(p) : u32x4{0, 0, 0, 0}, b = in ? ld16_stream(p + 4) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[j][i] = __uint_as_float(a[i]);
        f[j][4 + i] = __uint_as_float(b[i]);
      }
    }
  }
  uint16_t sbits[S];
  uint32_t out[4];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    uint32_t mx = 0;
#pragma unroll
    for (int j = s * (4 / S); j < (s + 1) * (4 / S); ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(f[j][i]) & 0x7fffffffu);
    sbits[s] = group_scale(__float_as_uint(xor_max_bits(mx)));
    const float sc = bf16_bits_to_f32(sbits[s]);
#pragma unroll
    for (int j = s * (4 / S); j < (s + 1) * (4 / S); ++j) {
      uint32_t d = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) d |= code4(f[j][i], sc) << (4 * i);
      out[j] = d;
    }
  }
  qp[blk * 64 + lane] = make_uint4(out[0], out[1], out[2], out[3]);
  if (lane < 16) {
    uint16_t* d = sp + (blk * 16 + lane) * S;
#pragma unroll
    for (int s = 0; s < S; ++s) d[s] = row < n && c0 + s * (128 / S) < k ? sbits[s] : 0;
  }
}

template <int OUT, int S>
__global__ __launch_bounds__(kQ4Threads) void dequantize4_kernel(const uint4* __restrict__ qp,
                                                                 const uint16_t* __restrict__ sp, int64_t n, int k,
                                                                 int64_t blocks, void* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t blk = static_cast<int64_t>(blockIdx.x) * (kQ4Threads / 64) + uniform(static_cast<int>(threadIdx.x >> 6));
  if (blk >= blocks) return;
  const int kb = static_cast<int>(fp4_kblocks(k));
  const int64_t trow = blk / kb;
  const int r = lane & 15;
  const int64_t row = trow * 16 + r;
  const int col = static_cast<int>(blk - trow * kb) * 128 + 8 * (lane >> 4);
  const uint4 v = qp[blk * 64 + lane];
  const uint32_t d[4] = {v.x, v.y, v.z, v.w};
  float sc[S];
#pragma unroll
  for (int s = 0; s < S; ++s) sc[s] = bf16_bits_to_f32(sp[(blk * 16 + r) * S + s]);
  if (row >= n) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (col + 32 * j >= k) break;
    float f[8];
    fp4x8_to_f32(d[j], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= sc[j * S / 4];
    const int64_t e = row * k + col + 32 * j;
    store_dequant16<OUT>(out, e, f);
    if constexpr (OUT == PGS_DTYPE_F32) store_dequant16<OUT>(out, e + 4, f + 4);
  }
}

int check_sizes(const char* fn, int64_t n, int64_t k, int64_t group) {
  if (n < 0 || k < 0) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (group != 32 && group != 64 && group != 128)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: group=%lld must be 32, 64 or 128", fn, (long long)group);
  if (k % 16 != 0 || k > kMaxK)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: k=%lld must be a multiple of 16 and at most %d", fn, (long long)k, kMaxK);
  if (fp4_blocks(n, k) > (int64_t{1} << 33))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: too large", fn);
  return PGS_OK;
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" int64_t pgs_packed4_bytes(int64_t n, int64_t k) { return n < 0 || k < 0 ? -1 : fp4_blocks(n, k) * 1024; }

extern "C" int64_t pgs_packed4_scales(int64_t n, int64_t k, int64_t group) {
  if (n < 0 || k < 0 || (group != 32 && group != 64 && group != 128)) return -1;
  return fp4_blocks(n, k) * 16 * (128 / group);
}

extern "C" int pgs_quantize4_packed(const void* w, int w_dtype, int64_t n, int64_t k, int64_t group, void* qp, void* sp,
                                    void* stream) {
  const char* fn = "pgs_quantize4_packed";
  if (int rc = check_sizes(fn, n, k, group)) return rc;
  if (w_dtype != PGS_DTYPE_F32 && w_dtype != PGS_DTYPE_BF16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: weight dtype %d must be fp32 or bf16", fn, w_dtype);
  if (n == 0 || k == 0) return PGS_OK;
  if (!w || !qp || !sp) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(w, 16) || !aligned(qp, 16) || !aligned(sp, 2))
    return fail(PGS_ERR_MISALIGNED, "%s: weight and codes must be 16-byte aligned", fn);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const int64_t blocks = fp4_blocks(n, k);
  const dim3 grid(static_cast<unsigned>((blocks + 3) / 4)), block(kQ4Threads);
  auto* q = static_cast<uint4*>(qp);
  auto* s = static_cast<uint16_t*>(sp);
  const int ki = static_cast<int>(k);
  auto go = [&](auto bf16, auto groups) {
    hipLaunchKernelGGL((quantize4_kernel<decltype(bf16)::value, decltype(groups)::value>), grid, block, 0, st, w, n, ki,
                       blocks, q, s);
  };
  auto by_group = [&](auto bf16) {
    if (group == 128) go(bf16, Int<1>{});
    else if (group == 64) go(bf16, Int<2>{});
    else go(bf16, Int<4>{});
  };
  if (w_dtype == PGS_DTYPE_BF16) by_group(Int<1>{});
  else by_group(Int<0>{});
  return check_launch("quantize4 kernel");
}

extern "C" int pgs_dequantize4_packed(const void* qp, const void* sp, int64_t n, int64_t k, int64_t group, void* out,
                                      int out_dtype, void* stream) {
  const char* fn = "pgs_dequantize4_packed";
  if (int rc = check_sizes(fn, n, k, group)) return rc;
  if (out_dtype != PGS_DTYPE_F32 && out_dtype != PGS_DTYPE_BF16 && out_dtype != PGS_DTYPE_F16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: bad output dtype %d", fn, out_dtype);
  if (n == 0 || k == 0) return PGS_OK;
  if (!qp || !sp || !out) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(qp, 16) || !aligned(sp, 2) || !aligned(out, 16))
    return fail(PGS_ERR_MISALIGNED, "%s: codes and output must be 16-byte aligned", fn);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const int64_t blocks = fp4_blocks(n, k);
  const dim3 grid(static_cast<unsigned>((blocks + 3) / 4)), block(kQ4Threads);
  const auto* q = static_cast<const uint4*>(qp);
  const auto* s = static_cast<const uint16_t*>(sp);
  const int ki = static_cast<int>(k);
  auto go = [&](auto dt, auto groups) {
    hipLaunchKernelGGL((dequantize4_kernel<decltype(dt)::value, decltype(groups)::value>), grid, block, 0, st, q, s, n,
                       ki, blocks, out);
  };
  auto by_group = [&](auto dt) {
    if (group == 128) go(dt, Int<1>{});
    else if (group == 64) go(dt, Int<2>{});
    else go(dt, Int<4>{});
  };
  if (out_dtype == PGS_DTYPE_F32) by_group(Int<PGS_DTYPE_F32>{});
  else if (out_dtype == PGS_DTYPE_BF16) by_group(Int<PGS_DTYPE_BF16>{});
  else by_group(Int<PGS_DTYPE_F16>{});
  return check_launch("dequantize4 kernel");
}
