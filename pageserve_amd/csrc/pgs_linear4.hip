// Linear with 4-bit weights and group scales (W4A16) for the few tokens of a
// drafting step (gfx950):
//
//   y[t, n] = sum over groups g of scale[n, g] * ( sum over k in g of value[n, k] * x[t, k] )  (+ bias, + residual)
//
// The inner sums are v_mfma_f32_16x16x32_bf16 over the exactly widened E2M1 values
// (pgs_fp4.h), accumulated in fp32; a group's sum is scaled in fp32 and added up, so
// neither the weights nor the scales are rounded anywhere.
//
// Memory bound: every packed KiB is read once, as one 128-bit load per lane that is
// already the A operand of four MFMAs.  A workgroup owns R 16-row tiles over all of K;
// its NW waves take 128-column chunks round robin, U per batch, a batch's loads issued
// together, and the waves' partial tiles meet in LDS in a fixed order.
#include "pgs_fp4.h"

namespace pgs {
namespace {

struct Lin4 {
  const uint16_t* x;
  const char* qp;
  const uint16_t* sp;
  const uint16_t* bias;  // or null
  const uint16_t* res;   // or null
  void* y;
  int m, n, k;
};

constexpr int kNowhere = 0x40000000;  // a lane offset past every activation block (at most 64 rows of kMaxK)

template <int NW, int U, int TM, int R, int S, bool OUT_F32>
__global__ __launch_bounds__(64 * NW) void linear4_kernel(Lin4 a) {
  constexpr int MT = 16 * TM;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int kb = (a.k + 127) >> 7;
  const int tiles = (a.n + 15) >> 4;
  const int tile0 = blockIdx.x * R;
  const int m0 = blockIdx.y * MT;
  const int rows = min(a.m - m0, MT);
  const int kq = lane >> 4;  // this lane's eight columns of each 32

  // (one resource per tile: a chunk past K, or a tile past N, reads zeros)
  __amdgpu_buffer_rsrc_t wres[R], sres[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t t = tile0 + r;
    const bool live = t < tiles;
    wres[r] = make_rsrc(a.qp + (live ? t : 0) * kb * 1024, live ? static_cast<int64_t>(kb) * 1024 : 0);
    sres[r] = make_rsrc(a.sp + (live ? t : 0) * kb * (16 * S), live ? static_cast<int64_t>(kb) * (32 * S) : 0);
  }
  const __amdgpu_buffer_rsrc_t xres =
      make_rsrc(a.x + static_cast<int64_t>(m0) * a.k, static_cast<int64_t>(rows) * a.k * 2);
  int xoff[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) xoff[t] = min(16 * t + (lane & 15), rows - 1) * a.k * 2 + kq * 16;

  f32x4 acc[R][TM];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < TM; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Chunk {
    u32x4 w[R];
    uint32_t s[R][2 * S];
    u32x4 x[4][TM];
  };
  auto load = [&](Chunk& b, int c) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      b.w[r] = __builtin_amdgcn_raw_buffer_load_b128(wres[r], lane * 16, c * 1024, kLoadNT);
      if constexpr (S == 1) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(sres[r], kq * 8, c * 32, kLoadNT);
        b.s[r][0] = v[0], b.s[r][1] = v[1];
      } else {
#pragma unroll
        for (int h = 0; h < S / 2; ++h) {
          const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(sres[r], kq * (8 * S) + 16 * h, c * (32 * S), kLoadNT);
#pragma unroll
          for (int i = 0; i < 4; ++i) b.s[r][4 * h + i] = v[i];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (columns from K on: zeros, not the next row's values, which may be
      // infinite and would not vanish against the zero codes there)
      const bool in = c * 128 + 32 * j + 8 * kq < a.k;
#pragma unroll
      for (int t = 0; t < TM; ++t)
        b.x[j][t] = __builtin_amdgcn_raw_buffer_load_b128(xres, in ? xoff[t] : kNowhere, c * 256 + 64 * j, 0);
    }
  };
  auto mac = [&](const Chunk& b) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      bf16x8 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = fp4x8_to_bf16x8(b.w[r][j]);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        f32x4 sc;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sc[2 * i] = __uint_as_float(b.s[r][2 * s + i] << 16);
          sc[2 * i + 1] = __uint_as_float(b.s[r][2 * s + i] & 0xffff0000u);
        }
#pragma unroll
        for (int t = 0; t < TM; ++t) {
          f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = s * (4 / S); j < (s + 1) * (4 / S); ++j)
            p = mfma16x16x32(w[j], __builtin_bit_cast(bf16x8, b.x[j][t]), p);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][t][i] = fmaf(p[i], sc[i], acc[r][t][i]);
        }
      }
    }
  };

  for (int c = wave * U; c < kb; c += NW * U) {
    Chunk b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(b[u], c + u);
#pragma unroll
    for (int u = 0; u < U; ++u) mac(b[u]);
  }

  __shared__ f32x4 part[NW][R][TM][64];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < TM; ++t) part[wave][r][t][lane] = acc[r][t];
  __syncthreads();
  const float* pf = reinterpret_cast<const float*>(part);
  for (int o = threadIdx.x; o < rows * 16 * R; o += 64 * NW) {
    const int mm = o / (16 * R), i = o % (16 * R);
    const int n = tile0 * 16 + i;
    if (n >= a.n) continue;
    const int r = i >> 4, at = ((((i & 15) >> 2) * 16 + (mm & 15)) << 2) + (i & 3);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += pf[((w * R + r) * TM + (mm >> 4)) * 256 + at];
    if (a.bias) v += bf16_bits_to_f32(a.bias[n]);
    const int64_t e = static_cast<int64_t>(m0 + mm) * a.n + n;
    store_out<OUT_F32>(a.y, e, add_residual<OUT_F32>(v, a.res, e));
  }
}

template <int NW, int U, int TM, int R, int S, bool OUT_F32>
int launch(const Lin4& a, hipStream_t st) {
  const int tiles = (a.n + 15) / 16;
  const dim3 grid((tiles + R - 1) / R, (a.m + 16 * TM - 1) / (16 * TM));
  hipLaunchKernelGGL((linear4_kernel<NW, U, TM, R, S, OUT_F32>), grid, dim3(64 * NW), 0, st, a);
  note_launch(__PRETTY_FUNCTION__, static_cast<long long>(grid.x) * grid.y, 1);
  return check_launch("linear4 kernel");
}

template <int S, bool OUT_F32>
int pick(const Lin4& a, hipStream_t st) {
  if (a.m <= 16) return launch<8, 2, 1, 1, S, OUT_F32>(a, st);
  if (a.m <= 32) return launch<8, 1, 2, 2, S, OUT_F32>(a, st);
  return launch<8, 1, 4, 2, S, OUT_F32>(a, st);
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" int pgs_w4a16_linear(const void* x, const void* qp, const void* sp, const void* bias, const void* residual,
                                void* y, int y_dtype, int64_t m, int64_t n, int64_t k, int64_t group, void* stream) {
  const char* fn = "pgs_w4a16_linear";
  if (m < 0 || n < 0 || k < 0) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (y_dtype != PGS_DTYPE_BF16 && y_dtype != PGS_DTYPE_F32)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: output dtype %d must be bf16 or fp32", fn, y_dtype);
  if (group != 32 && group != 64 && group != 128)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: group=%lld must be 32, 64 or 128", fn, (long long)group);
  if (k % 16 != 0 || k > kMaxK)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: k=%lld must be a multiple of 16 and at most %d", fn, (long long)k, kMaxK);
  if (n > 0x7ffffff0 || m > 65535 * 16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: m=%lld n=%lld too large", fn, (long long)m, (long long)n);
  if (m == 0 || n == 0) return PGS_OK;
  if (!y || (k > 0 && (!x || !qp || !sp))) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(x, 16) || !aligned(qp, 16) || !aligned(sp, 16) || !aligned(bias, 2) || !aligned(residual, 2) ||
      !aligned(y, y_dtype == PGS_DTYPE_F32 ? 4 : 2))
    return fail(PGS_ERR_MISALIGNED, "%s: activations, codes and scales must be 16-byte aligned", fn);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const Lin4 a{static_cast<const uint16_t*>(x),    static_cast<const char*>(qp),         static_cast<const uint16_t*>(sp),
               static_cast<const uint16_t*>(bias), static_cast<const uint16_t*>(residual), y,
               static_cast<int>(m),                static_cast<int>(n),                  static_cast<int>(k)};
  const bool f32 = y_dtype == PGS_DTYPE_F32;
  if (group == 128) return f32 ? pick<1, true>(a, st) : pick<1, false>(a, st);
  if (group == 64) return f32 ? pick<2, true>(a, st) : pick<2, false>(a, st);
  return f32 ? pick<4, true>(a, st) : pick<4, false>(a, st);
}
