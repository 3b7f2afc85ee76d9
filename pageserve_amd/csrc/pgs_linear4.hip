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
// already the B operand of four MFMAs.  A workgroup owns R 16-row tiles over its share of K;
// its NW waves take 128-column chunks round robin, U per batch, a batch's loads issued
// together, and the waves' partial tiles meet in LDS in a fixed order.
//
// Measured in a replayed graph, weights in no cache: 1 x 151936 x 2048, groups of 128, 29 us,
// 5.5 TB/s of codes and scales; 30 tokens, groups of 32, 59 us: each wave loads the tokens'
// values for its four tiles, twice the bytes of their codes, from L2, and scales eight products
// a tile; 60 tokens 110 us, groups of 128 98: four times the bytes of the codes.  Nothing is on
// its way while a batch is multiplied: 1 x 11008 x 2048 5.1 us, a launch and two rounds of loads
// (16 chunks on eight waves); 5 x 2048 x 11008 6.6 us, three rounds (43 pairs of chunks,
// sixteen a round).
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
constexpr int kNowhere = 0x40000000;  // a lane offset past every resource (the largest: 64 rows of kMaxK activations)

// The tokens are the A operand and the weights the B operand: lane l's four sums are of
// weight row l%16, so it needs the scales of that row only.  (With the weights as A its
// sums are of four rows: four times the scales to load and widen, 68 us for 62 at
// 30 x 151936 x 2048 with groups of 32, when this was changed.)
//
// FOLD (m <= 8): a workgroup owns eight rows of a tile (half blockIdx.x % 2) and each MFMA
// takes two chunks: A rows 0-7 are the tokens in chunk 2 c, A rows 8-15 the same tokens in
// chunk 2 c + 1, B columns 0-7 the weight rows in chunk 2 c and 8-15 in 2 c + 1, so that
// output (token t, row i) is D[t][i] + D[t + 8][i + 8] (the other two quarters mix chunks
// and are ignored).  Twice the workgroups for the same bytes and products.
//
// (At least two waves per SIMD are asked for: with fewer the products land in accumulation
// registers, and each has to be copied out to be scaled: 150 us for 106 at 60 x 151936 x 2048.)
template <int NW, int U, int TM, int R, int S, bool FOLD, bool OUT_F32>
__global__ __launch_bounds__(64 * NW, 2) void linear4_kernel(Lin4 a) {
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

  // One resource per tile (a tile past N: the last one again, its sums are not stored).  What
  // lies past K reads zeros by a lane offset past every resource; the scalar offset added
  // to it never passes the resource's end, so the check holds however it counts that.
  __amdgpu_buffer_rsrc_t wres[R], sres[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t t = min(tile0 + r, tiles - 1);
    wres[r] = make_rsrc(a.qp + t * kb * 1024, static_cast<int64_t>(kb) * 1024);
    sres[r] = make_rsrc(a.sp + t * kb * (16 * S), static_cast<int64_t>(kb) * (32 * S));
  }
  // (up to the last chunk's end of the last row)
  const __amdgpu_buffer_rsrc_t xres =
      make_rsrc(a.x + static_cast<int64_t>(m0) * a.k, (static_cast<int64_t>(rows - 1) * a.k + 128 * kb) * 2);
  const int sub = FOLD ? li >> 3 : 0;  // this lane's chunk of the slot, as token and as weight row
  const int woff = FOLD ? sub * 1024 + (8 * half + (li & 7) + 16 * kq) * 16 : lane * 16;
  const int soff = FOLD ? sub * (32 * S) + (8 * half + (li & 7)) * (2 * S) : li * (2 * S);
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
    uint32_t s[R][(S + 1) / 2];
    u32x4 x[4][TM];
  };
  auto load = [&](Slot& b, int slot) {
    const int c0 = FOLD ? 2 * slot : slot, c = min(c0, kb - 1);
    const bool live = c0 + sub < kb;
    const int wo = live ? woff : kNowhere, so = live ? soff : kNowhere;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      b.w[r] = __builtin_amdgcn_raw_buffer_load_b128(wres[r], wo, c * 1024, kLoadNT);
      if constexpr (S == 1) {
        b.s[r][0] = __builtin_amdgcn_raw_buffer_load_b16(sres[r], so, c * 32, 0);
      } else if constexpr (S == 2) {
        b.s[r][0] = __builtin_amdgcn_raw_buffer_load_b32(sres[r], so, c * 64, 0);
      } else {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(sres[r], so, c * 128, 0);
        b.s[r][0] = v[0], b.s[r][1] = v[1];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (columns from K on: zeros, not the next row's values, which may be
      // infinite and would not vanish against the zero codes there)
      const bool in = (c0 + sub) * 128 + 32 * j + 8 * kq < a.k;
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
        const uint32_t v = b.s[r][s / 2];
        const float sc = __uint_as_float(s & 1 ? v & 0xffff0000u : v << 16);
#pragma unroll
        for (int t = 0; t < TM; ++t) {
          f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = s * (4 / S); j < (s + 1) * (4 / S); ++j)
            p = mfma16x16x32(__builtin_bit_cast(bf16x8, b.x[j][t]), w[j], p);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][t][i] = fmaf(p[i], sc, acc[r][t][i]);
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

  __shared__ float part[NW][R][TM][4][64];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[wave][r][t][i][lane] = acc[r][t][i];
  __syncthreads();
  const float* pf = &part[0][0][0][0][0];
  constexpr int PER = FOLD ? 8 : 16 * R;  // weight rows
  for (int o = threadIdx.x; o < rows * PER; o += 64 * NW) {
    const int mm = o / PER, i = o % PER;
    const int n = tile0 * 16 + 8 * half + i;
    if (n >= a.n) continue;
    // D row mm % 16, column i % 16: element mm % 4 of lane 16 (mm % 16 / 4) + i % 16
    const int r = i >> 4, at = (mm & 3) * 64 + ((mm & 15) >> 2) * 16 + (i & 15);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* p = pf + ((w * R + r) * TM + (mm >> 4)) * 256 + at;
      v += FOLD ? p[0] + p[32 + 8] : p[0];
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
// - up to 8 tokens while the halves of the tiles are at most one per CU: folded halves.
//   5x2048x11008 6.8/8.1 (whole tiles), 1x2048x2048 3.0/3.2; above: 8x4096x4096 5.3 whole,
//   6.8 folded.
// - from 128 workgroups of four tiles on: four tiles (the activations are read once per 64
//   rows).  1x11008x2048 5.1/5.3 (one tile), 16x11008x2048 6.3/8.6, 10x151936x2048
//   33.8/62.9, 30x8192x2048 8.5/9.6, 60x8192x2048 15.5/18.1.
// - else, for a long K, four tiles with K split over workgroups: 16x2048x11008 8.6/13.2 (one
//   tile), 30x2048x11008 11.1/21.9, 60x2048x11008 17.1/41.9, 60x4096x4096 14.9/17.7.  Half
//   the splits: 10.5 for 8.6, 22.1 for 17.1; twice: 9.6 and 18.9.
// - else one tile: the second launch costs more than it gains.  16x4096x4096 6.5/8.3,
//   30x4096x4096 9.8/10.0, 60x4096x2048 10.6/11.9, 16x2048x2048 4.4/6.7.
struct Plan {
  int tm;      // 16-token tiles of a workgroup
  int wide;    // 16-row tiles of a workgroup: 4, or 1; 0: folded halves
  int splits;  // of K
};
Plan plan(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = (n + 15) / 16, kb = (k + 127) / 128;
  if (m <= 8 && tiles <= 128) return {1, 0, 1};
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

// (waves, chunks per batch: with fewer of either, too few loads are in flight at 11008 rows
// and fewer: 30x11008x2048 8.7 for 9.7 with four waves.  Registers, of 256: 66 with 16 tokens
// and four tiles, where a second chunk would fit, up to 237 with 64.  Four waves there: eight
// spill over two waves per SIMD, 101 us for 155 at 60x151936x2048.)
template <int S, bool OUT_F32>
int pick(const Plan& p, const Lin4& a, hipStream_t st) {
  if (p.wide == 0) return launch<8, 2, 1, 1, S, true, OUT_F32>(a, st);
  if (p.wide == 1) {
    if (p.tm == 1) return launch<8, 2, 1, 1, S, false, OUT_F32>(a, st);
    if (p.tm == 2) return launch<8, 2, 2, 1, S, false, OUT_F32>(a, st);
    return launch<8, 1, 4, 1, S, false, OUT_F32>(a, st);
  }
  if (p.tm == 1) return launch<8, 1, 1, 4, S, false, OUT_F32>(a, st);
  if (p.tm == 2) return launch<8, 1, 2, 4, S, false, OUT_F32>(a, st);
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
