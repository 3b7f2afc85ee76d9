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
  float* part;  // [splits][m][n], or null: one split, the epilogue here
  int m, n, k;
  int splits;   // workgroups along K (gridDim.z)
};

constexpr int64_t kMaxRows4 = 0x7ffffff0, kMaxTokens4 = 65535 * 16;
constexpr int kNowhere = 0x40000000;  // a lane offset past every activation block (at most 64 rows of kMaxK)

// FOLD (m <= 8): a workgroup owns eight rows of a tile (half blockIdx.x % 2) and each MFMA
// takes two chunks: A rows 0-7 are its rows in chunk 2 c, A rows 8-15 the same rows in
// chunk 2 c + 1, B columns 0-7 the tokens in chunk 2 c and 8-15 in 2 c + 1, so that output
// (token t, row i) is D[i][t] + D[i + 8][t + 8] (the other two quarters mix chunks and are
// ignored).  Twice the workgroups for the same bytes and products.
template <int NW, int U, int TM, int R, int S, bool FOLD, bool OUT_F32>
__global__ __launch_bounds__(64 * NW) void linear4_kernel(Lin4 a) {
  static_assert(!FOLD || (TM == 1 && R == 1), "folding serves up to eight tokens");
  constexpr int MT = FOLD ? 8 : 16 * TM;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int li = lane & 15, kq = lane >> 4;  // kq: this lane's eight columns of each 32
  const int kb = (a.k + 127) >> 7;
  const int slots = FOLD ? (kb + 1) >> 1 : kb;
  const int tiles = (a.n + 15) >> 4;
  const int unit = FOLD ? xcd_remap(blockIdx.x, gridDim.x) : blockIdx.x;  // (a tile's halves on one XCD)
  const int tile0 = FOLD ? unit >> 1 : unit * R;
  const int half = FOLD ? unit & 1 : 0;
  const int m0 = blockIdx.y * MT;
  const int rows = min(a.m - m0, MT);

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
  const int sub = FOLD ? li >> 3 : 0;  // this lane's chunk of the slot, as A row and B column
  const int woff = FOLD ? sub * 1024 + (8 * half + (li & 7) + 16 * kq) * 16 : lane * 16;
  const int soff = FOLD ? (kq >> 1) * (32 * S) + (2 * half + (kq & 1)) * (8 * S) : kq * (8 * S);
  int xoff[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t)
    xoff[t] = min(FOLD ? li & 7 : 16 * t + li, rows - 1) * a.k * 2 + sub * 256 + kq * 16;

  f32x4 acc[R][TM];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < TM; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Slot {
    u32x4 w[R];
    uint32_t s[R][2 * S];
    u32x4 x[4][TM];
  };
  auto load = [&](Slot& b, int slot) {
    const int c = FOLD ? 2 * slot : slot;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      b.w[r] = __builtin_amdgcn_raw_buffer_load_b128(wres[r], woff, c * 1024, kLoadNT);
      if constexpr (S == 1) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(sres[r], soff, c * 32, 0);
        b.s[r][0] = v[0], b.s[r][1] = v[1];
      } else {
#pragma unroll
        for (int h = 0; h < S / 2; ++h) {
          const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(sres[r], soff + 16 * h, c * (32 * S), 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) b.s[r][4 * h + i] = v[i];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (columns from K on: zeros, not the next row's values, which may be
      // infinite and would not vanish against the zero codes there)
      const bool in = (c + sub) * 128 + 32 * j + 8 * kq < a.k;
#pragma unroll
      for (int t = 0; t < TM; ++t)
        b.x[j][t] = __builtin_amdgcn_raw_buffer_load_b128(xres, in ? xoff[t] : kNowhere, c * 256 + 64 * j, 0);
    }
  };
  auto mac = [&](const Slot& b) {
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

  const int cb = static_cast<int>(static_cast<int64_t>(slots) * blockIdx.z / a.splits);
  const int ce = static_cast<int>(static_cast<int64_t>(slots) * (blockIdx.z + 1) / a.splits);
  for (int c = cb + wave * U; c < ce; c += NW * U) {
    Slot b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(b[u], c + u < ce ? c + u : slots);  // (slots: all zeros)
    __builtin_amdgcn_sched_barrier(0);  // (all loads of the batch before its first product)
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
  constexpr int PER = FOLD ? 8 : 16 * R;  // weight rows
  for (int o = threadIdx.x; o < rows * PER; o += 64 * NW) {
    const int mm = o / PER, i = o % PER;
    const int n = tile0 * 16 + 8 * half + i;
    if (n >= a.n) continue;
    // the accumulator lane of D row i % 16, column mm % 16: 16 (i % 16 / 4) + mm % 16, element i % 4
    const int r = i >> 4, at = ((((i & 15) >> 2) * 16 + (mm & 15)) << 2) + (i & 3);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* p = pf + ((w * R + r) * TM + (mm >> 4)) * 256 + at;
      v += FOLD ? p[0] + p[(32 + 8) * 4] : p[0];
    }
    const int64_t e = static_cast<int64_t>(m0 + mm) * a.n + n;
    if (a.part) {
      a.part[blockIdx.z * static_cast<int64_t>(a.m) * a.n + e] = v;
      continue;
    }
    if (a.bias) v += bf16_bits_to_f32(a.bias[n]);
    store_out<OUT_F32>(a.y, e, add_residual<OUT_F32>(v, a.res, e));
  }
}

// The splits' sums in order, then the epilogue.  A thread per output.
template <bool OUT_F32>
__global__ __launch_bounds__(256) void linear4_sum_kernel(Lin4 a) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, mn = static_cast<int64_t>(a.m) * a.n;
  if (e >= mn) return;
  float v = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) v += a.part[s * mn + e];
  if (a.bias) v += bf16_bits_to_f32(a.bias[e % a.n]);
  store_out<OUT_F32>(a.y, e, add_residual<OUT_F32>(v, a.res, e));
}

// How a call is laid out.  The chip is filled before anything else: a workgroup is one
// long chain of loads and products, so twice the workgroups is close to half the time
// until there are one to two per CU.  Measured, microseconds (own/other choice), m x n x k:
// - up to 8 tokens and fewer than 512 tiles: folded halves of tiles.  5x2048x11008 6.7/8.5
//   (whole tiles), 1x2048x2048 2.9/3.1.
// - from 128 workgroups of four tiles on: four tiles (the activations are read once per 64
//   rows).  16x11008x2048 8.0/8.6 (two tiles), 10x151936x2048 35.6/44.8, 30x8192x2048
//   9.5/10.0 (one tile), 60x8192x2048 16.2/18.4.
// - else, for a long K, four tiles with K split over workgroups: 16x2048x11008 9.3/13.7,
//   30x2048x11008 12.5/22.3, 60x2048x11008 17.9/42.4, 60x4096x4096 15.7/18.1 (one tile).
//   More than 8 splits: 13.0 for 12.5, 19.8 for 17.9.
// - else one tile: the second launch costs more than it gains.  16x4096x4096 6.7/8.9,
//   30x4096x4096 10.0/10.7, 60x4096x2048 10.9/12.7, 16x2048x2048 4.5/6.5.
struct Plan {
  int tm;      // 16-token tiles of a workgroup
  int wide;    // 16-row tiles of a workgroup: 4, or 1; 0: folded halves
  int splits;  // of K
};
Plan plan(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = (n + 15) / 16, kb = (k + 127) / 128;
  if (m <= 8 && tiles < 512) return {1, 0, 1};
  const int tm = m <= 16 ? 1 : m <= 32 ? 2 : 4;
  const int64_t units = (tiles + 3) / 4 * ((m + 16 * tm - 1) / (16 * tm));
  if (units >= 128) return {tm, 4, 1};
  if (kb * (tm + 1) < 128) return {tm, 1, 1};
  const int64_t s = 256 / units;
  return {tm, 4, static_cast<int>(s < 8 ? s : 8)};
}
size_t part_bytes(const Plan& p, int64_t m, int64_t n) {
  return p.splits > 1 ? static_cast<size_t>(p.splits) * m * n * 4 : 0;
}

template <int NW, int U, int TM, int R, int S, bool FOLD, bool OUT_F32>
int launch(const Lin4& a, hipStream_t st) {
  const int tiles = (a.n + 15) / 16;
  const int mt = FOLD ? 8 : 16 * TM;
  const dim3 grid(FOLD ? 2 * tiles : (tiles + R - 1) / R, (a.m + mt - 1) / mt, a.splits);
  hipLaunchKernelGGL((linear4_kernel<NW, U, TM, R, S, FOLD, OUT_F32>), grid, dim3(64 * NW), 0, st, a);
  note_launch(__PRETTY_FUNCTION__, static_cast<long long>(grid.x) * grid.y * grid.z, a.splits,
              a.part ? "linear4_sum_kernel" : nullptr);
  if (int rc = check_launch("linear4 kernel")) return rc;
  if (!a.part) return PGS_OK;
  const int64_t blocks = (static_cast<int64_t>(a.m) * a.n + 255) / 256;
  hipLaunchKernelGGL(linear4_sum_kernel<OUT_F32>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, a);
  return check_launch("linear4 sum kernel");
}

// (waves, chunks per batch: the batch's loads are all in flight while its registers still
// leave two waves per SIMD; the next larger ones measured equal or slower)
template <int S, bool OUT_F32>
int pick(const Plan& p, const Lin4& a, hipStream_t st) {
  if (p.wide == 0) return launch<8, 2, 1, 1, S, true, OUT_F32>(a, st);
  if (p.wide == 1) {
    if (p.tm == 1) return launch<8, 2, 1, 1, S, false, OUT_F32>(a, st);
    if (p.tm == 2) return launch<8, 2, 2, 1, S, false, OUT_F32>(a, st);
    return launch<8, 1, 4, 1, S, false, OUT_F32>(a, st);
  }
  if (p.tm == 1) return launch<8, 1, 1, 4, S, false, OUT_F32>(a, st);
  if (p.tm == 2) return launch<4, 2, 2, 4, S, false, OUT_F32>(a, st);
  return launch<4, 1, 4, 4, S, false, OUT_F32>(a, st);
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" size_t pgs_w4a16_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k < 0 || k > kMaxK || n > kMaxRows4 || m > kMaxTokens4) return 0;
  return part_bytes(plan(m, n, k), m, n);
}

extern "C" int pgs_w4a16_linear(const void* x, const void* qp, const void* sp, const void* bias, const void* residual,
                                void* y, int y_dtype, int64_t m, int64_t n, int64_t k, int64_t group,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "pgs_w4a16_linear";
  if (m < 0 || n < 0 || k < 0) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (y_dtype != PGS_DTYPE_BF16 && y_dtype != PGS_DTYPE_F32)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: output dtype %d must be bf16 or fp32", fn, y_dtype);
  if (group != 32 && group != 64 && group != 128)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: group=%lld must be 32, 64 or 128", fn, (long long)group);
  if (k % 16 != 0 || k > kMaxK)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: k=%lld must be a multiple of 16 and at most %d", fn, (long long)k, kMaxK);
  if (n > kMaxRows4 || m > kMaxTokens4)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: m=%lld n=%lld too large", fn, (long long)m, (long long)n);
  if (m == 0 || n == 0) return PGS_OK;
  if (!y || (k > 0 && (!x || !qp || !sp))) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(x, 16) || !aligned(qp, 16) || !aligned(sp, 16) || !aligned(bias, 2) || !aligned(residual, 2) ||
      !aligned(y, y_dtype == PGS_DTYPE_F32 ? 4 : 2))
    return fail(PGS_ERR_MISALIGNED, "%s: activations, codes and scales must be 16-byte aligned", fn);
  const Plan p = plan(m, n, k);
  const size_t need = part_bytes(p, m, n);
  if (need && !workspace) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null workspace", fn);
  if (!aligned(workspace, 16)) return fail(PGS_ERR_MISALIGNED, "%s: the workspace must be 16-byte aligned", fn);
  if (workspace_bytes < need)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, %zu needed", fn, workspace_bytes, need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const Lin4 a{static_cast<const uint16_t*>(x),
               static_cast<const char*>(qp),
               static_cast<const uint16_t*>(sp),
               static_cast<const uint16_t*>(bias),
               static_cast<const uint16_t*>(residual),
               y,
               need ? static_cast<float*>(workspace) : nullptr,
               static_cast<int>(m),
               static_cast<int>(n),
               static_cast<int>(k),
               p.splits};
  const bool f32 = y_dtype == PGS_DTYPE_F32;
  if (group == 128) return f32 ? pick<1, true>(p, a, st) : pick<1, false>(p, a, st);
  if (group == 64) return f32 ? pick<2, true>(p, a, st) : pick<2, false>(p, a, st);
  return f32 ? pick<4, true>(p, a, st) : pick<4, false>(p, a, st);
}
