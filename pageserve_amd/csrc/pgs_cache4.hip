// Rows of keys and values into the 4-bit cache and back (gfx950; the layout is in
// pgs_window.h).  Per 32 dims of a token and head:
//   scale = max(absmax, 1e-8) / 6 cut to its first 6 significant bits
//   code  = the value nearest to x / scale, a tie to the even code
// Cut, not rounded: 6 scale is then at most absmax, so no value that the cache stands for
// leaves the range of the rows' type; the largest of a group is off by up to a thirty-second.
#include "pgs_window.h"

namespace pgs {
namespace {

constexpr int kRowThreads = 256;

struct Cache4 {
  uint8_t *k, *v;
  uint16_t *ks, *vs;
  int64_t nslots;
  int bs, heads;
};
inline Cache4 cache4_of(const pgs_kv_cache4& c) {
  return Cache4{static_cast<uint8_t*>(c.k),        static_cast<uint8_t*>(c.v),
                static_cast<uint16_t*>(c.k_scale), static_cast<uint16_t*>(c.v_scale),
                c.blocks * c.block_size,           static_cast<int>(c.block_size),
                static_cast<int>(c.kv_heads)};
}
// Row of [blocks * kv_heads * block_size] that holds slot s of head h, and its token of 16.
__device__ __forceinline__ int64_t cache_row(const Cache4& c, int64_t slot, int h, int& token) {
  const int64_t b = slot / c.bs;
  const int at = static_cast<int>(slot - b * c.bs);
  token = at & 15;
  return (b * c.heads + h) * c.bs + at;
}

struct Write4 {
  const uint16_t *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  Cache4 c;
  const int64_t* slots;
  int64_t units;  // rows * heads * 8, of k and as many of v
};

template <bool F16>
__device__ __forceinline__ float widen(uint32_t bits) {
  return F16 ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits))) : low_bf16(bits);
}

// the code of x at scale s, by exact products (of 6 and of at most 3 bits)
__device__ __forceinline__ uint32_t code_of(float x, float s) {
  const float a = fabsf(x);
  const uint32_t c = static_cast<uint32_t>(a > 0.25f * s) + (a >= 0.75f * s) + (a > 1.25f * s) + (a >= 1.75f * s) +
                     (a > 2.5f * s) + (a >= 3.5f * s) + (a > 5.0f * s);
  return x < 0 && c ? c + 8 : c;
}
// the scale of a group whose largest magnitude has these bits (a NaN lies above all)
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float a = __uint_as_float(top);
  const float s = (a < 1e-8f ? 1e-8f : a) / 6.0f;
  return __uint_as_float(__float_as_uint(s) & 0xfffc0000u);
}

// Eight lanes per row and head of k, and eight of v.  Of k a lane has D/8 neighbouring dims
// (its codes are whole dwords), of v dims 2 i and 2 i + 1 of every sixteen (whole bytes of
// two neighbouring dims' codes).  Bound by the launch: 64 rows of 2 x 64 dims 3.5 us; 8192 rows of
// 2 x 128 dims 6.5, two of them for what memory needs, the rest for the words of values that go out
// by four bytes.
template <int D, bool F16>
__global__ __launch_bounds__(kRowThreads) void write_kv4_kernel(Write4 a) {
  constexpr int C = D / 32;
  int64_t u = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  const bool values = u >= a.units;
  if (values) u -= a.units;
  if (u >= a.units) return;  // (units are multiples of 8: a row's lanes stay together)
  const int i = static_cast<int>(u & 7);
  const int64_t row = (u >> 3) / a.c.heads;
  const int h = static_cast<int>((u >> 3) - row * a.c.heads);
  const int64_t slot = a.slots[row];
  if (slot < 0 || slot >= a.c.nslots) return;
  int token;
  const int64_t at = cache_row(a.c, slot, h, token);
  if (!values) {
    const uint16_t* p = a.k + row * a.k_row + h * a.k_head + i * (D / 8);
    uint32_t w[D / 16], top = 0;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const u32x4 x = ld16(p + 8 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * j + e] = x[e];
    }
    float f[D / 8];
#pragma unroll
    for (int e = 0; e < D / 8; ++e) {
      f[e] = widen<F16>(w[e >> 1] >> (16 * (e & 1)) & 0xffff);
      top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
    }
    // (a group is 256 / D lanes)
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
    if constexpr (D == 64) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
    const float s = scale_of(top);
    const int c = i * (D / 8) / 32, first = i * (D / 8) % 32 / 8;
    if (first == 0) a.c.ks[at * C + c] = static_cast<uint16_t>(__float_as_uint(s) >> 16);
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      uint32_t codes = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) codes |= code_of(f[8 * j + e], s) << (4 * e);
      reinterpret_cast<uint32_t*>(a.c.k + at * (D / 2))[C * (first + j) + c] = codes;
    }
  } else {
    const uint16_t* p = a.v + row * a.v_row + h * a.v_head + 2 * i;
    uint32_t w[2 * C];
#pragma unroll
    for (int d = 0; d < 2 * C; ++d) w[d] = *reinterpret_cast<const uint32_t*>(p + 16 * d);
    uint32_t codes[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint32_t top = 0;
      float f[2][2];  // [half of the group][dim]
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          f[e][m] = widen<F16>(w[2 * c + e] >> (16 * m) & 0xffff);
          top = max(top, __float_as_uint(f[e][m]) & 0x7fffffffu);
        }
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), x)));
      const float s = scale_of(top);
      if (i == c) a.c.vs[at * C + c] = static_cast<uint16_t>(__float_as_uint(s) >> 16);
#pragma unroll
      for (int m = 0; m < 2; ++m) codes[m] |= (code_of(f[0][m], s) | code_of(f[1][m], s) << 4) << (8 * c);
    }
    uint8_t* to = a.c.v + (at - token) * (D / 2) + (16 * (token >> 2) * 4 + (token & 3)) * C;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint8_t* d = to + (2 * i + m) * (4 * C);
      if constexpr (C == 4) *reinterpret_cast<uint32_t*>(d) = codes[m];
      else *reinterpret_cast<uint16_t*>(d) = static_cast<uint16_t>(codes[m]);
    }
  }
}

struct Read4 {
  Cache4 c;
  const int64_t* slots;
  void *k, *v;
  int64_t units;  // rows * heads * D / 8, of k and as many of v
};

// One thread per eight dims of a row.  Bound by the launch and one load behind another (slots, then
// codes and scales): the same sizes 3.4 and 5.2 us.
template <int D, int OUT>
__global__ __launch_bounds__(kRowThreads) void read_kv4_kernel(Read4 a) {
  constexpr int C = D / 32, P = D / 8;
  int64_t u = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  const bool values = u >= a.units;
  if (values) u -= a.units;
  if (u >= a.units) return;
  const int i = static_cast<int>(u % P), c = i / 4;
  const int64_t row = u / P / a.c.heads;
  const int h = static_cast<int>(u / P - row * a.c.heads);
  const int64_t slot = a.slots[row];
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 0.f;
  if (slot >= 0 && slot < a.c.nslots) {
    int token;
    const int64_t at = cache_row(a.c, slot, h, token);
    uint32_t codes = 0;
    if (!values) {
      codes = reinterpret_cast<const uint32_t*>(a.c.k + at * (D / 2))[C * (i % 4) + c];
    } else {
      const uint8_t* p = a.c.v + (at - token) * (D / 2) + ((16 * (token >> 2) + 8 * (i & 1)) * 4 + (token & 3)) * C + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) codes |= (p[e * 4 * C] >> (i & 2 ? 4 : 0) & 15u) << (4 * e);
    }
    const float s = low_bf16((values ? a.c.vs : a.c.ks)[at * C + c]);
    fp4x8_to_f32(codes, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= s;
  }
  void* out = values ? a.v : a.k;
#pragma unroll
  for (int j = 0; j < (OUT == PGS_DTYPE_F32 ? 2 : 1); ++j) store_dequant16<OUT>(out, u * 8 + 4 * j, f + 4 * j);
}

int check_cache4(const char* fn, const pgs_kv_cache4* cache, int64_t rows) {
  if (!cache) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
  const pgs_kv_cache4& c = *cache;
  if (c.head_dim != 64 && c.head_dim != 128)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: head_dim=%lld must be 64 or 128", fn, (long long)c.head_dim);
  if (c.blocks < 0 || c.blocks > 0x7fffffff || c.block_size < 16 || c.block_size > 0x10000 || c.block_size % 16 != 0 ||
      c.kv_heads < 1 || c.kv_heads > 4096)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: the cache needs blocks of a multiple of 16 tokens (block_size=%lld)", fn,
                (long long)c.block_size);
  // (a launch has fewer than 2^32 threads, each of four numbers at least, in whole workgroups)
  if (rows < 0 || rows > ((int64_t{1} << 34) - 4 * kRowThreads) / (c.kv_heads * c.head_dim))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: rows=%lld: rows x kv_heads x head_dim must be at most 2^34 - 1024", fn, (long long)rows);
  if (rows > 0 && c.blocks > 0 && (!c.k || !c.k_scale || !c.v || !c.v_scale))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(c.k, 16) || !aligned(c.k_scale, 16) || !aligned(c.v, 16) || !aligned(c.v_scale, 16))
    return fail(PGS_ERR_MISALIGNED, "%s: the cache must be 16-byte aligned", fn);
  return PGS_OK;
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" int pgs_write_kv4(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                             int dtype, const pgs_kv_cache4* cache, const int64_t* slots, int64_t rows, void* stream) {
  const char* fn = "pgs_write_kv4";
  if (int rc = check_cache4(fn, cache, rows)) return rc;
  if (dtype != PGS_DTYPE_BF16 && dtype != PGS_DTYPE_F16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: dtype %d must be bf16 or fp16", fn, dtype);
  for (int64_t s : {k_row, k_head, v_row, v_head})
    if (s < 0 || s % 8 != 0) return fail(PGS_ERR_MISALIGNED, "%s: strides must be multiples of 8 elements", fn);
  const pgs_kv_cache4& c = *cache;
  if (rows == 0 || c.blocks == 0) return PGS_OK;
  if (!k || !v || !slots) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8)) return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const Write4 a{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), k_row, k_head, v_row, v_head,
                 cache4_of(c), slots, rows * c.kv_heads * 8};
  const dim3 grid(static_cast<unsigned>((2 * a.units + kRowThreads - 1) / kRowThreads)), block(kRowThreads);
  const bool f16 = dtype == PGS_DTYPE_F16;
  if (c.head_dim == 64) {
    if (f16) hipLaunchKernelGGL((write_kv4_kernel<64, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((write_kv4_kernel<64, false>), grid, block, 0, st, a);
  } else {
    if (f16) hipLaunchKernelGGL((write_kv4_kernel<128, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((write_kv4_kernel<128, false>), grid, block, 0, st, a);
  }
  return check_launch("write_kv4 kernel");
}

extern "C" int pgs_read_kv4(const pgs_kv_cache4* cache, const int64_t* slots, int64_t rows, void* k, void* v, int dtype,
                            void* stream) {
  const char* fn = "pgs_read_kv4";
  if (int rc = check_cache4(fn, cache, rows)) return rc;
  if (dtype != PGS_DTYPE_BF16 && dtype != PGS_DTYPE_F16 && dtype != PGS_DTYPE_F32)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: dtype %d", fn, dtype);
  if (rows == 0) return PGS_OK;
  if (!k || !v || !slots) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8)) return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const pgs_kv_cache4& c = *cache;
  const Read4 a{cache4_of(c), slots, k, v, rows * c.kv_heads * (c.head_dim / 8)};
  const dim3 grid(static_cast<unsigned>((2 * a.units + kRowThreads - 1) / kRowThreads)), block(kRowThreads);
  auto go = [&](auto out) {
    constexpr int OUT = decltype(out)::value;
    if (c.head_dim == 64) hipLaunchKernelGGL((read_kv4_kernel<64, OUT>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((read_kv4_kernel<128, OUT>), grid, block, 0, st, a);
  };
  if (dtype == PGS_DTYPE_F32) go(Int<PGS_DTYPE_F32>{});
  else if (dtype == PGS_DTYPE_BF16) go(Int<PGS_DTYPE_BF16>{});
  else go(Int<PGS_DTYPE_F16>{});
  return check_launch("read_kv4 kernel");
}
