// Shared by the kernels of attention over a paged cache: LDS and loads past the
// registers, the element types with their matrix products, and the exponents of a
// softmax in one pass.
#pragma once

#include <math.h>

#include "pgs_linear.h"

namespace pgs {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// The lane number where it is used: lane-dependent offsets computed from it are not kept
// in registers across a loop.
__device__ __forceinline__ int here(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// LDS by its byte address
template <typename T>
__device__ __forceinline__ __attribute__((address_space(3))) T* lds(uint32_t address) {
  return reinterpret_cast<__attribute__((address_space(3))) T*>(address);
}
template <typename T>
__device__ __forceinline__ uint32_t lds_address(T& v) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)&v));
}
// Four keys x 16 dims per 16 lanes from LDS, transposed: lane i of them gives the address
// of dims 4 (i % 4) .. +3 of key i / 4 and gets dim i of the four keys.
__device__ __forceinline__ u32x2 read_transposed(uint32_t address) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<s16x4>(address)));
}

// 16 bytes per lane from memory to LDS (lane l's to `address` + 16 l, wave-uniform) past
// the registers.  The compiler does not count this load: whoever uses what it brings waits
// with arrived(n), n: how many such loads issued later may still be on their way.
__device__ __forceinline__ void load_lds(const uint16_t* p, uint32_t address) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(address), "v"(p) : "m0", "memory");
}
// The same from `base` (wave-uniform) + the lane's `offset` bytes.
__device__ __forceinline__ void load_lds(const void* base, uint32_t offset, uint32_t address) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(address), "v"(offset), "s"(base)
               : "m0", "memory");
}
template <int N>
__device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <bool F16>
struct Elem;
template <>
struct Elem<false> {
  typedef bf16x8 x8;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return mfma16x16x32(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
  static constexpr uint32_t kOnes = 0x3f803f80u, kExp = 0x7f80u;  // 1.0 twice; the exponent's bits
  // A reference is this much (in powers of two) below the maximum that it is taken from.
  static constexpr float kHead = 0.f;
};
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <>
struct Elem<true> {
  typedef f16x8 x8;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
  }
  static __device__ __forceinline__ float low(uint32_t v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v)));
  }
  static constexpr uint32_t kOnes = 0x3c003c00u, kExp = 0x7c00u;
  // fp16 has no steps finer than 2^-24: beside a weight of 1, n others of up to 2^-25 would be
  // lost, n 2^-25 of the sum.  With the largest at 2^7 to 2^15 (kSlack; the type ends at 2^16)
  // that is n 2^-32.
  static constexpr float kHead = 7.f;
};

// the maximum over lanes l, l ^ 16, l ^ 32, l ^ 48 (each swap leaves the two halves
// of its exchange in two registers)
__device__ __forceinline__ float quad_max(float v) {
  const uint32_t x = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A maximum nothing has raised yet: the lowest value that is finite.
constexpr float kLow = -3.402823466e38f;
// The reference of the exponents follows the maximum only when a score exceeds it
// by this (in powers of two) and Elem::kHead: p stays below 2^8 times 2^kHead, as exact as
// below 1, and the sums are rescaled a few times per row instead of at every step.
constexpr float kSlack = 8.0f;
// A reference is a rounded product c s, and fma(s, c, -reference) sees that rounding: up to
// half a step of the reference, which the largest weight is off by (as a power of two; all
// weights of the row are alike).  Beyond kFar that is more than 1/2 and in the end out of any
// range, so there the product is rounded before the reference is taken off, as it was for
// the reference: the largest weight is 2^0.
constexpr float kFar = 8388608.0f;
__device__ __forceinline__ float exponent(float s, float c, float reference, bool far) {
#pragma clang fp contract(off)
  const float t = s * c;
  return far ? t - reference : fmaf(s, c, -reference);
}

// token / bs without a division: the product's high half is the quotient or one more
// (bs_inv is too large by less than 1, token below 2^31), which the remainder's sign
// shows
template <typename Args>
__device__ __forceinline__ int block_of(const Args& a, int token, int& slot) {
  int q = static_cast<int>(__umulhi(static_cast<uint32_t>(token), a.bs_inv));
  int r = token - q * a.bs;
  if (r < 0) --q, r += a.bs;
  slot = r;
  return q;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// ln sum_j e^(score_j) of weights 2^(c s_j - ref) that add up to sum; -inf where there are none.
__device__ __forceinline__ float log_sum(float ref, float sum) {
  return sum == 0.f ? -INFINITY : (ref + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
}

// The kernel's argument again, read from its segment at this point: for the parts of a
// kernel outside its inner loop, whose fields would otherwise all sit in scalar
// registers throughout (and push vector registers out to memory).
template <typename Args>
__device__ __forceinline__ Args again() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  Args a;
  __builtin_memcpy(&a, (const void*)p, sizeof(a));
  return a;
}

// Four rows' outputs from n parts' sums each: brought to one reference, added in order and
// divided by the joined sum.  Sixteen lanes per row, each with DIMS/16 neighbouring dims of the
// DIMS that `parts` points to; slot(i): where part i of the lane's row is; p: the lane's dims of
// the output, or null.
// STATS: numbers of a part, 2 (reference, sum) or 4 (and the sum of the weights before they
// were rounded, whose logarithm goes to lse; the fourth is unused).  WAVES: of the workgroup,
// each taking that share of the parts (all must call it), joined in LDS; or 1.  Bound by
// memory and, few rows of many parts, by its latency: BATCH parts' loads are on their way
// together.
template <int D, bool F16, int WAVES, int STATS, int DIMS = D, int BATCH = STATS == 2 ? 8 : 4, typename Slot>
__device__ __forceinline__ void join_rows(const float* parts, const float* stats, int n, int lane, int wave, uint16_t* p,
                                          float* lse, Slot slot) {
  constexpr int W = DIMS / 16;
  const int li = lane & 15;
  typedef float Stat __attribute__((ext_vector_type(STATS)));
  float ref = kLow, sum = 0.f, exact = 0.f, o[W];
#pragma unroll
  for (int d = 0; d < W; ++d) o[d] = 0.f;
  const int end = WAVES == 1 ? n : n * (wave + 1) / WAVES;
  auto batch = [&](int i0, auto count) {
    constexpr int U = decltype(count)::value;
    Stat st[U];
    f32x4 x[U][W / 4];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int64_t at = slot(min(i0 + e, end - 1));
      st[e] = *reinterpret_cast<const Stat*>(stats + STATS * at);
#pragma unroll
      for (int d = 0; d < W / 4; ++d) x[e][d] = *reinterpret_cast<const f32x4*>(parts + at * D + W * li + 4 * d);
    }
    float top = ref;
#pragma unroll
    for (int e = 0; e < U; ++e) top = fmaxf(top, st[e][0]);
    const float f = __builtin_amdgcn_exp2f(ref - top);
    ref = top;
    sum *= f;
    if constexpr (STATS == 4) exact *= f;
#pragma unroll
    for (int d = 0; d < W; ++d) o[d] *= f;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      if (i0 + e >= end) break;  // (a part read again)
      const float g = __builtin_amdgcn_exp2f(st[e][0] - ref);
      sum = fmaf(g, st[e][1], sum);
      if constexpr (STATS == 4) exact = fmaf(g, st[e][2], exact);
#pragma unroll
      for (int d = 0; d < W; ++d) o[d] = fmaf(g, x[e][d / 4][d % 4], o[d]);
    }
  };
  int i = WAVES == 1 ? 0 : n * wave / WAVES;
  if constexpr (BATCH == 8) {
    for (; end - i > 4; i += 8) batch(i, Int<8>{});
    if (end - i > 2) batch(i, Int<4>{});
    else if (end > i) batch(i, Int<2>{});
  } else {
    for (; end - i > 2; i += 4) batch(i, Int<4>{});
    if (end > i) batch(i, Int<2>{});
  }
  if constexpr (WAVES > 1) {
    __shared__ float lref[WAVES][64], lsum[WAVES][64], lexact[STATS == 4 ? WAVES : 1][64], lo[WAVES][W][64];
    lref[wave][lane] = ref;
    lsum[wave][lane] = sum;
    if constexpr (STATS == 4) lexact[wave][lane] = exact;
#pragma unroll
    for (int d = 0; d < W; ++d) lo[wave][d][lane] = o[d];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) ref = fmaxf(ref, lref[w][lane]);
    sum = exact = 0.f;
#pragma unroll
    for (int d = 0; d < W; ++d) o[d] = 0.f;
    constexpr int kUnroll = BATCH == 4 ? 4 : WAVES;  // (registers)
#pragma unroll kUnroll
    for (int w = 0; w < WAVES; ++w) {
      const float g = __builtin_amdgcn_exp2f(lref[w][lane] - ref);
      sum = fmaf(g, lsum[w][lane], sum);
      if constexpr (STATS == 4) exact = fmaf(g, lexact[w][lane], exact);
#pragma unroll
      for (int d = 0; d < W; ++d) o[d] = fmaf(g, lo[w][d][lane], o[d]);
    }
  }
  if (!p) return;
  if constexpr (STATS == 4)
    if (lse && li == 0) *lse = log_sum(ref, exact);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t w[W / 2];
#pragma unroll
  for (int d = 0; d < W / 2; ++d) w[d] = Elem<F16>::pack(o[2 * d] * inv, o[2 * d + 1] * inv);
  if constexpr (W == 8) *reinterpret_cast<u32x4*>(p) = u32x4{w[0], w[1], w[2], w[3]};
  else *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
}

}  // namespace
}  // namespace pgs
