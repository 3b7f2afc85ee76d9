// Attention of a request's newest rows over the cached tokens of a sliding window and the
// first few (sinks), the paged cache in 16 or in 4 bits (gfx950; pgs_window.h).  For row
// (t, h) over the tokens j that it sees:
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c s_j - m),  s_j = q . k_j,  c = scale log2(e)
//   lse = ln sum_j e^(scale s_j) = (m + log2 sum_j p_j) ln 2
//
// in one pass with a running maximum m and sums.  Rows and keys lie as in the attention of
// drafted tokens (pgs_attend.hip): S^T = K Q^T and O^T = V^T P^T by v_mfma_f32_16x16x32, the
// tokens x query heads of one key head as columns, so that a row's scores, maximum, sums and
// output stay in the lanes l%16 = row.
#include <algorithm>
#include <cmath>

#include "pgs_window.h"

namespace pgs {
namespace {

// The order of a block that has M matrix products, T exponentials and V more vector
// instructions: the others spread between the products.
template <int M, int T, int V>
__device__ __forceinline__ void interleave() {
  auto part = [](int i, int n) { return (i + 1) * n / M - i * n / M; };
#pragma unroll
  for (int i = 0; i < M; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (n < part(i, V)) __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
      if (n < part(i, T)) __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
    }
  }
}

// 16 R rows of a wave and their running sums.  The output MFMA d covers the dims
// (4 lg + i) D/16 + d of its lanes (SPREAD: values straight from 16-bit rows), or 16 d + 4 lg + i.
// PAIR (4-bit): columns l%16 and l%16 + 8 are one of eight rows, the first with its q and output
// of the even chunks of 32 dims, the second of the odd ones, so that a lane multiplies by half
// the scales.
template <int D, int R, bool F16, bool SPREAD, bool PAIR>
struct Rows {
  static_assert(!PAIR || (R == 1 && !SPREAD));
  static constexpr int kRows = PAIR ? 8 : 16;  // of a tile
  using E = Elem<F16>;
  static constexpr int DC = D / 32, DV = D / 16;
  u32x4 q[R][DC];
  f32x4 o[R][DV], l[R];  // (l: every element the same)
  float exact[R], mx[R];  // the lane's own part of the weights' sum before they are rounded; the reference
  int pos[R];  // where the row stands
  bool far;               // some row's reference is beyond kFar (the same in all lanes)

  __device__ __forceinline__ void load(const Window& a, const Ragged& rq, int kh, int row0, int nrows, int li, int lg) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = min(row0 + 16 * r + li % kRows, nrows - 1), t = row / a.group;  // (rows past the last repeat it)
      const uint16_t* p = a.q + (rq.row0 + t) * a.q_row + (kh * a.group + row - t * a.group) * a.q_head + 8 * lg;
#pragma unroll
      for (int d = 0; d < DC; ++d) {
        q[r][d] = (ld16(p + 32 * d) ^ a.flip) & a.keep;
        if (PAIR && (li >> 3) != (d & 1)) q[r][d] = u32x4{};
      }
      pos[r] = rq.first + t;
    }
    // (they have arrived here: a wait for them inside the loop over the keys would be
    // a wait for the keys on their way too)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int d = 0; d < DC; ++d) asm volatile("" : "+v"(q[r][d]));
    far = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mx[r] = kLow;
      exact[r] = 0.f;
      l[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DV; ++i) o[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // New references, the largest score of each row so far, if a score x[r][e] (of those in
  // ok[r]) passes its row's by too much.
  __device__ __forceinline__ void raise(const Window& a, const float (&x)[R][8], const uint32_t (&ok)[R]) {
    float top[R];
    bool over = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      top[r] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) top[r] = fmaxf(top[r], ok[r] >> e & 1 ? x[r][e] * a.c : -INFINITY);
      over = over || top[r] - mx[r] > kSlack + E::kHead;
    }
    if (!__ballot(over)) return;
    bool beyond = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float t = quad_max(top[r]);
      const float ref = fmaxf(fabsf(t) > kFar ? t : t - E::kHead, mx[r]), f = __builtin_amdgcn_exp2f(mx[r] - ref);
      mx[r] = ref;
      beyond = beyond || fabsf(ref) > kFar;
      exact[r] *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) l[r][i] *= f;
#pragma unroll
      for (int d = 0; d < DV; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[r][d][i] *= f;
      }
    }
    far = __ballot(beyond);
  }
  // which of the step's eight keys of this lane its row r sees
  __device__ __forceinline__ uint32_t seen(const Window& a, int r, int key0, bool bad0, bool bad1, int lg) const {
    const uint32_t m = visible32(key0, pos[r], low_of(pos[r], a.window), a.sinks) & ((bad0 ? 0 : 0xffffu) | (bad1 ? 0 : 0xffff0000u));
    const uint32_t t = m >> (4 * lg);
    return (t & 0xf) | (t >> 12 & 0xf0);
  }
  // Weights of a step: s[r][h] the scores of keys key0 + 16 h + 4 lg + i, x[r][4 h + i] the
  // weights against the rows' references, which are raised first where a score needs it.
  // masked: some row may not see some key, or a half's block is absent (bad).
  __device__ __forceinline__ void weights(const Window& a, const f32x4 (&s)[R][2], float (&x)[R][8], int key0, bool masked,
                                          bool bad0, bool bad1, int lg) {
    bool over = masked || far;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[r][e] = s[r][e >> 2][e & 3];
        top = fmaxf(top, x[r][e]);
      }
      over = over || fmaf(top, a.c, -mx[r]) > kSlack + E::kHead;
    }
    uint32_t ok[R];
    if (__ballot(over)) {
#pragma unroll
      for (int r = 0; r < R; ++r) ok[r] = masked ? seen(a, r, key0, bad0, bad1, lg) : 0xff;
      raise(a, x, ok);
    }
    if (masked || far) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[r][e] = ok[r] >> e & 1 ? __builtin_amdgcn_exp2f(exponent(x[r][e], a.c, mx[r], far)) : 0.f;
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[r][e] = __builtin_amdgcn_exp2f(fmaf(x[r][e], a.c, -mx[r]));
    }
  }

  // The step's part of the sums and outputs, the weights rounded to the rows' type; the row
  // sum that divides adds the rounded ones, the logarithm's (want) those before.  values(d):
  // A operand of output MFMA d.  odd: keys whose values are not finite (values() holds
  // zeros for them); value(j) is the row of key key0 + j.
  template <typename Values, typename Value>
  __device__ __forceinline__ void add(const Window& a, const float (&x)[R][8], Values values, int key0, uint32_t odd,
                                      bool want, int li, int lg, Value value) {
    u32x4 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[r][i] = E::pack(x[r][2 * i], x[r][2 * i + 1]);
    if (want)
#pragma unroll
      for (int r = 0; r < R; ++r)
        exact[r] += ((x[r][0] + x[r][1]) + (x[r][2] + x[r][3])) + ((x[r][4] + x[r][5]) + (x[r][6] + x[r][7]));
    const u32x4 ones = {E::kOnes, E::kOnes, E::kOnes, E::kOnes};
#pragma unroll
    for (int r = 0; r < R; ++r) l[r] = E::mfma(ones, p[r], l[r]);
#pragma unroll
    for (int d = 0; d < DV; ++d) {
      const u32x4 v = values(d);
#pragma unroll
      for (int r = 0; r < R; ++r) o[r][d] = E::mfma(v, p[r], o[r][d]);
    }
    if (odd) add_odd(a, p, key0, odd, li, lg, value);
  }
  template <typename Value>
  __device__ __forceinline__ void add_odd(const Window& a, const u32x4 (&p)[R], int key0, uint32_t odd, int li, int lg, Value value) {
    for (uint32_t w = odd; w; w &= w - 1) {
      const int j = __builtin_ctz(w);
      const auto row = value(j);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t lo = j & 2 ? p[r][1] : p[r][0], hi = j & 2 ? p[r][3] : p[r][2];
        const float pj = E::low(__shfl(j & 16 ? hi : lo, 16 * (j >> 2 & 3) + li) >> (16 * (j & 1)));
        const bool in = visible(key0 + j, pos[r], low_of(pos[r], a.window), a.sinks);
#pragma unroll
        for (int d = 0; d < DV; ++d) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = o[r][d][i] + pj * row(SPREAD ? (4 * lg + i) * DV + d : 16 * d + 4 * lg + i);
            o[r][d][i] = in ? y : o[r][d][i];
          }
        }
      }
    }
  }

  // The same from 4-bit values, whose scales multiply the weights in front of the rounding:
  // one operand per 32 dims (PAIR: per 64, the lanes of even columns with the first's scales).  It
  // is bf16 whatever the rows are (a weight times a scale may leave fp16's range; the codes are
  // exact in both), in two terms where they are fp16, whose finer rounding the output shall have.
  // A token that is not seen has weight 0 whatever its scale holds.
  __device__ __forceinline__ void add4(const Window& a, const float (&x)[R][8], Values4<D>& n, int key0, bool masked,
                                       bool bad0, bool bad1, int li, int lg) {
    static_assert(!SPREAD && R == 1, "the codes' order, one row's mask");
    if (masked) {
      const uint32_t ok = seen(a, 0, key0, bad0, bad1, lg);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int c = 0; c < DC / 2; ++c) {
          uint32_t& w = n.s[e >> 2][(e & 3) * (DC / 2) + c];
          w = ok >> e & 1 ? w : 0;
        }
    }
    exact[0] += ((x[0][0] + x[0][1]) + (x[0][2] + x[0][3])) + ((x[0][4] + x[0][5]) + (x[0][6] + x[0][7]));
    // codes of two keys side by side: dims 32 c + l%16 (byte c of `low`) and 16 further
    uint32_t low[4], high[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t* v = n.v[i >> 1];
      if constexpr (DC == 4) {
        const uint32_t v0 = v[2 * (i & 1)], v1 = v[2 * (i & 1) + 1];
        low[i] = (v0 & 0x0f0f0f0fu) | (v1 << 4 & 0xf0f0f0f0u);
        high[i] = (v0 >> 4 & 0x0f0f0f0fu) | (v1 & 0xf0f0f0f0u);
      } else {
        const uint32_t w = v[i & 1];
        low[i] = (w & 0x0f0fu) | (w >> 12 & 0xf0f0u);
        high[i] = (w >> 4 & 0x0f0fu) | (w >> 16 & 0xf0f0u);
      }
    }
    const uint32_t sel = pair_half(li);
    auto group = [&](auto first) {
      constexpr int G = decltype(first)::value;
      u32x4 p, rest;
      __builtin_amdgcn_sched_barrier(0);  // (one after the other: registers)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int e = 2 * i + j;
          y[j] = x[0][e] * (PAIR ? half_of(n.s[e >> 2][(e & 3) * (DC / 2) + G / 2], sel) : n.scale(e >> 2, e & 3, G));
        }
        p[i] = pack_bf16x2(y[0], y[1]);
        if constexpr (F16) rest[i] = pack_bf16x2(y[0] - low_bf16(p[i]), y[1] - high_bf16(p[i]));
      }
      auto product = [&](auto chunk) {
        constexpr int C = decltype(chunk)::value;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          u32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = widen2<C>(d ? high[i] : low[i]);
          o[0][2 * C + d] = Elem<false>::mfma(v, p, o[0][2 * C + d]);
          if constexpr (F16) o[0][2 * C + d] = Elem<false>::mfma(v, rest, o[0][2 * C + d]);
        }
      };
      product(first);
      if constexpr (PAIR) product(Int<G + 1>{});
    };
    group(Int<0>{});
    if constexpr (PAIR) {
      if constexpr (DC == 4) group(Int<2>{});
    } else {
      group(Int<1>{});
      if constexpr (DC == 4) group(Int<2>{}), group(Int<3>{});
    }
  }

  // The rows' outputs, or (whole false: other keys of theirs are elsewhere) their
  // sums.  slot(row, token, head): where to.
  template <typename Slot>
  __device__ __forceinline__ void store(const Window& a, const Ragged& rq, int kh, int row0, int nrows, int li, int lg,
                                        bool whole, Slot slot) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = row0 + 16 * r + li % kRows;
      if (row >= nrows) continue;
      const int t = row / a.group, head = kh * a.group + row - t * a.group;
      const int64_t token = rq.row0 + t;
      if constexpr (PAIR) {  // (the lane's chunks into the places of the even ones)
#pragma unroll
        for (int e = 0; e < DV; ++e)
          if (!(e & 2)) o[r][e] = li < 8 ? o[r][e] : o[r][e + 2];
      }
      const bool first = lg == 0 && li < kRows;
      const int shift = PAIR && li >= 8 ? 32 : 0;
      if (whole) {
        const float inv = l[r][0] == 0.f ? 0.f : 1.f / l[r][0];
        uint16_t* d = a.out + token * a.out_row + head * a.out_head + 4 * lg * (SPREAD ? DV : 1);
        if constexpr (SPREAD) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[DC];
#pragma unroll
            for (int e = 0; e < DC; ++e) w[e] = E::pack(o[r][2 * e][i] * inv, o[r][2 * e + 1][i] * inv);
            if constexpr (DC == 4) *reinterpret_cast<u32x4*>(d + i * DV) = u32x4{w[0], w[1], w[2], w[3]};
            else *reinterpret_cast<u32x2*>(d + i * DV) = u32x2{w[0], w[1]};
          }
        } else {
#pragma unroll
          for (int e = 0; e < DV; ++e)
            if (!PAIR || !(e & 2))
              *reinterpret_cast<u32x2*>(d + shift + 16 * e) = u32x2{E::pack(o[r][e][0] * inv, o[r][e][1] * inv),
                                                                    E::pack(o[r][e][2] * inv, o[r][e][3] * inv)};
        }
        if (a.lse && first) a.lse[token * a.q_heads + head] = log_sum(mx[r], exact[r]);
      } else {
        const int64_t at = slot(row, token, head);
        float* d = a.part + at * D + 4 * lg * (SPREAD ? DV : 1);
        if constexpr (SPREAD) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < DV; e += 4)
              *reinterpret_cast<f32x4*>(d + i * DV + e) =
                  f32x4{o[r][e][i], o[r][e + 1][i], o[r][e + 2][i], o[r][e + 3][i]};
        } else {
#pragma unroll
          for (int e = 0; e < DV; ++e)
            if (!PAIR || !(e & 2)) *reinterpret_cast<f32x4*>(d + shift + 16 * e) = o[r][e];
        }
        if (first) *reinterpret_cast<f32x4*>(a.stat + 4 * at) = f32x4{mx[r], l[r][0], exact[r], 0.f};
      }
    }
  }
};

// Parts that the keys of a row group are cut into, of the `splits` that the grid has, by its
// steps of 32 keys (twice those where two waves share a step): none below kWholeSteps, else
// of min_steps at least.
constexpr int kWholeSteps = 32, kCoarseSteps = 16, kFineSteps = 8;
__device__ __forceinline__ int parts_of(const Window& a, int tiles, int wr) {
  const int steps = tiles * wr;
  return steps < kWholeSteps ? 1 : max(min(a.splits, steps / a.min_steps), 1);
}
// what the rows [first, first + RG) of a request's `nrows` see
template <int RG>
__device__ __forceinline__ Span group_span(const Window& a, const Ragged& rq, int first, int nrows) {
  return span_of<5>(a, rq.first + first / a.group, rq.first + (min(first + RG, nrows) - 1) / a.group);
}

// Rows straight from memory: a workgroup's NW waves are WR row tiles of 16 R x NW/WR key
// slices; each wave loads the keys and values of its steps into registers.  16 bits: bound by
// memory, 48 requests of one row and 4100 tokens each 35 us, 5.7 TB/s (a part from caches).  4
// bits: by what a step's vector instructions take next to its loads (of 32 keys and eight rows
// some 260; 500 without pairs of columns), 32 requests of 8000 to 16000 tokens (111 MB) 25.4 us, 4.4 TB/s.
template <int D, int R, int WR, int NW, bool F16, bool FP4, bool PAIR>
__global__ __launch_bounds__(64 * NW, 2) void window_kernel(Window a) {
  static_assert(!PAIR || WR == 1);
  using W = Rows<D, R, F16, !FP4, PAIR>;
  using E = Elem<F16>;
  constexpr int DC = W::DC, DV = W::DV;
  constexpr int WK = NW / WR;      // key slices
  constexpr int RG = 16 * R * WR;  // rows of a workgroup
  const int lane = threadIdx.x & 63;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int li = lane & 15, lg = lane >> 4;
  const int wr = wave % WR, wk = wave / WR;
  // unit: (request, row group, key head), part
  const int part = blockIdx.x % a.splits;
  int unit = blockIdx.x / a.splits;
  const int kh = unit % a.kv_heads;
  unit /= a.kv_heads;
  const int rg = unit % a.groups, b = unit / a.groups;
  const Ragged rq = ragged(a, b);
  const int nrows = rq.tokens * a.group;
  if (rg * RG >= nrows) return;
  const Span span = group_span<RG>(a, rq, rg * RG, nrows);
  const int parts = parts_of(a, span.tiles, FP4 ? (WR + 1) / 2 : WR);
  if (part >= parts) return;
  const int pmin = rq.first + rg * RG / a.group, pmax = rq.first + (min(rg * RG + RG, nrows) - 1) / a.group;
  const int row0 = rg * RG + wr * (16 * R);  // of this wave
  const int t0 = static_cast<int>(static_cast<int64_t>(span.tiles) * part / parts);
  const int t1 = static_cast<int>(static_cast<int64_t>(span.tiles) * (part + 1) / parts);
  const int32_t* table = a.tables + b * a.tstride;

  // the block ids of a step's two halves, loaded a step ahead of its keys (a half behind the
  // last key reads the other one's block instead, and is masked)
  auto first_of = [&](int key0, int h) { return key0 + (key0 + 16 * h <= pmax ? 16 * h : 0); };
  auto ids = [&](int t, int (&id)[2]) {
    if (t >= t1) return;
    const int key0 = span.tile(t) * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int slot;
      // (not provably uniform: the value stays in a vector register, unwaited for, until
      // it is used)
      id[h] = table[block_of(a, first_of(key0, h), slot) + (here(lane) >> 6)];
    }
  };
  int id[2] = {0, 0};
  ids(t0 + wk, id);
  W w;
  w.load(a, rq, kh, min(row0, nrows - 1), nrows, li, lg);
  const bool want = a.lse != nullptr;
  for (int t = t0 + wk; t < t1; t += WK) {
    const int key0 = span.tile(t) * 32;
    bool bad[2];
    int64_t blk[2];
    int slot[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = uniform(id[h]);
      bad[h] = i < 0 || i >= a.blocks;
      blk[h] = bad[h] ? 0 : i;
      block_of(a, first_of(key0, h), slot[h]);
    }
    const bool masked = bad[0] || bad[1] || !all_visible(a, key0, key0 + 31, pmin, pmax);
    f32x4 s[R][2];
    float x[R][8];
    if constexpr (FP4) {
      Keys4<D> k;
      Values4<D> v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t row = row_of(a, blk[h], slot[h], kh);
        load_keys4<D>(a, row, li, lg, k.k[h], k.s[h]);
        load_values4<D>(a, row, li, lg, v.v[h], v.s[h]);
      }
      ids(t + WK, id);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if constexpr (PAIR) s[r][h] = pair_scores<D, F16>(k, h, w.q[r], pair_half(li));
          else s[r][h] = scores<D, F16>(k, h, w.q[r]);
        }
      w.weights(a, s, x, key0, masked, bad[0], bad[1], lg);
      w.add4(a, x, v, key0, masked, bad[0], bad[1], li, lg);
    } else {
      Keys16<D> k;
      Values16<D> v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_keys<D>(a, blk[h], slot[h], kh, li, lg, k.k[h]);
        load_values<D>(a, blk[h], slot[h], kh, li, lg, v.v + 4 * h);
      }
      ids(t + WK, id);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][h] = scores<D, F16>(k, h, w.q[r]);
      // No value that a row does not see may meet its weight 0 as an infinity or NaN: those
      // of a masked step that are not finite are left out of the products (bit of `odd`) and
      // added for the rows that see them.
      uint32_t odd = 0;
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool gone = key0 + 16 * (e >> 2) + 4 * lg + (e & 3) > pmax || bad[e >> 2];
          bool wild = false;
#pragma unroll
          for (int i = 0; i < DC; ++i) {
            if (gone) v.v[e][i] = 0;
            wild = wild || (v.v[e][i] & E::kExp) == E::kExp || (v.v[e][i] & E::kExp << 16) == E::kExp << 16;
          }
          const unsigned long long m = __ballot(wild);
          if (m) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
              if (m >> (16 * g) & 0xffff) odd |= 1u << (16 * (e >> 2) + 4 * g + (e & 3));
            if (m >> (16 * lg) & 0xffff)
#pragma unroll
              for (int i = 0; i < DC; ++i) v.v[e][i] = 0;
          }
        }
      }
      w.weights(a, s, x, key0, masked, bad[0], bad[1], lg);
      auto values = [&](int d) {
        u32x4 vt;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          vt[e] = __builtin_amdgcn_perm(v.v[2 * e + 1][d >> 1], v.v[2 * e][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
        return vt;
      };
      w.add(a, x, values, key0, odd, want, li, lg, [&](int j) {
        const int h = j >> 4;
        const uint16_t* p = static_cast<const uint16_t*>(a.vc) + blk[h] * a.vc_block +
                            static_cast<int64_t>(slot[h] + (j & 15)) * a.vc_slot + kh * a.vc_head;
        return [p](int i) { return E::low(p[i]); };
      });
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    w.exact[r] = quad_sum(w.exact[r]);
    if constexpr (FP4) w.l[r][0] = w.exact[r];  // (4-bit: the weights are rounded once per scale group)
  }

  // join the key slices: slice 0 adds the others' sums, brought to one reference
  if constexpr (WK > 1) {
    __shared__ float lo_[(WK - 1) * WR][R][DV * 4][64];
    __shared__ float ls_[(WK - 1) * WR][R][3][64];
    if (wk > 0) {
      const int n = (wk - 1) * WR + wr;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ls_[n][r][0][lane] = w.mx[r];
        ls_[n][r][1][lane] = w.l[r][0];
        ls_[n][r][2][lane] = w.exact[r];
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) lo_[n][r][4 * d + i][lane] = w.o[r][d][i];
      }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float ref = w.mx[r];
#pragma unroll
      for (int s = 0; s < WK - 1; ++s) ref = fmaxf(ref, ls_[s * WR + wr][r][0][lane]);
      const float f = __builtin_amdgcn_exp2f(w.mx[r] - ref);
      w.mx[r] = ref;
      w.l[r][0] *= f;
      w.exact[r] *= f;
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[r][d][i] *= f;
#pragma unroll
      for (int s = 0; s < WK - 1; ++s) {
        const int n = s * WR + wr;
        const float g = __builtin_amdgcn_exp2f(ls_[n][r][0][lane] - ref);
        w.l[r][0] += g * ls_[n][r][1][lane];
        w.exact[r] += g * ls_[n][r][2][lane];
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) w.o[r][d][i] += g * lo_[n][r][4 * d + i][lane];
      }
    }
  }
  w.store(a, rq, kh, row0, nrows, li, lg, parts == 1,
          [&](int, int64_t token, int head) { return (token * a.q_heads + head) * a.splits + part; });
}

// Waves that join four rows: sixteen if those have eight parts and there are few of them, so
// that the parts' latency counts, else one (and four times four rows a workgroup).
constexpr int kJoinWaves = 16;
inline bool join_by_many(int64_t parts, int64_t fours) { return parts >= 8 && fours <= 512; }
constexpr int join_threads(int waves) { return waves == 1 ? 256 : 64 * waves; }

// Behind window_kernel: four rows of a key head, of one row group.  SLICED (sixteen waves): a
// workgroup for each 64 of their dims, with twice the parts' loads on their way, where no CU
// gets two of them: 234 parts of one request's 16 rows take 7.5 us, 10.5 without; 48 requests'
// eleven parts each would take 6.7, 4.9 without.
constexpr bool join_sliced(int64_t fours, int dim) { return fours * (dim / 64) <= 256; }
template <int D, bool F16, int WAVES, int RG, bool SLICED>
__global__ __launch_bounds__(join_threads(WAVES)) void window_join_kernel(Window a, int wr) {
  const int lane = threadIdx.x & 63, li = lane & 15, wave = uniform(static_cast<int>(threadIdx.x >> 6));
  constexpr int S = SLICED ? D / 64 : 1, DIMS = D / S;
  int64_t u = WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
  const int dim0 = static_cast<int>(u % S) * DIMS;
  u /= S;
  const int quads = (a.max_tokens * a.group + 3) >> 2;
  const int first = static_cast<int>(u % quads) * 4;
  u /= quads;
  const int kh = static_cast<int>(u % a.kv_heads), b = static_cast<int>(u / a.kv_heads);
  if (b >= a.requests) return;
  const Ragged rq = ragged(a, b);
  const int rows = rq.tokens * a.group;
  if (first >= rows) return;
  const int parts = parts_of(a, group_span<RG>(a, rq, first / RG * RG, rows).tiles, wr);
  if (parts == 1) return;
  const int row = min(first + (lane >> 4), rows - 1), t = row / a.group, head = kh * a.group + row - t * a.group;
  const int64_t of = static_cast<int64_t>(rq.row0 + t) * a.q_heads + head, at = of * a.splits;
  uint16_t* p = a.out + (rq.row0 + t) * a.out_row + head * a.out_head + dim0 + DIMS / 16 * li;
  join_rows<D, F16, WAVES, 4, DIMS, SLICED ? 8 : 4>(a.part + dim0, a.stat, parts, lane, wave, first + (lane >> 4) < rows ? p : nullptr,
                                    a.lse && dim0 == 0 ? a.lse + of : nullptr, [&](int i) { return at + i; });
}

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------

// The wide kernel's work: the tiles of all units, (request, key head, group of RG rows), in
// that order, cut into equal shares for the workgroups, whatever the requests' rows and lengths
// are.  What a group costs is counted in keys times `group`, so that it grows by RG from one
// to the next until the window holds it, and sums over groups need no loop: group g of a
// request costs min(base + RG (g + 1), cap) + unit (unit alone while that is below 0).  A share takes of
// each unit the part of its tiles that its part of the counts covers; of a unit that is not whole it
// leaves sums in slot 2 share (the unit began in an earlier share) or 2 share + 1.
constexpr int kTileBits = 6, kTile = 1 << kTileBits;  // keys of a tile
constexpr int kShares = 256;  // workgroups: one per CU
constexpr int kUnit = 256;    // what a unit costs besides its tiles, in keys

struct Groups {
  int n;            // of a request
  int none, rising;  // those before `none` see nothing; those before `rising` cost less than cap
  int64_t base, cap, unit;
  // counts of group m
  template <int RG>
  __device__ __forceinline__ int64_t cost(int m) const {
    return unit + (m < none ? 0 : m < rising ? base + RG * static_cast<int64_t>(m + 1) : cap);
  }
  // counts of the first m groups
  template <int RG>
  __device__ __forceinline__ int64_t upto(int m) const {
    const int64_t lo = min(m, none), hi = min(m, rising);
    return m * unit + (hi - lo) * base + RG * ((hi * (hi + 1) - lo * (lo + 1)) / 2) + (m - hi) * cap;
  }
};
template <int RG>
__device__ __forceinline__ Groups groups_of(const Window& a, const Ragged& rq) {
  Groups g;
  g.n = (rq.tokens * a.group + RG - 1) / RG;
  g.base = static_cast<int64_t>(rq.first) * a.group;
  // (the most that a group sees: its windows and the sinks)
  g.cap = least(static_cast<int64_t>(a.window) + min(a.sinks, rq.len), rq.len) * a.group + RG;
  g.none = static_cast<int>(least(largest(-g.base, 0) / RG, g.n));
  g.rising = static_cast<int>(least(largest((g.cap - g.base) / RG, g.none), g.n));
  g.unit = static_cast<int64_t>(kUnit) * a.group;
  return g;
}
// A unit of T tiles costs at most (kUnit + T kTile) group + RG counts: from two tiles on less than a
// share for each of them, so that a share inside of the unit has one of its tiles at least.  A unit of one
// tile may be longer than a share: the share that holds its end takes it whole, the others leave nothing.
__device__ __forceinline__ int shares_of(const Window& a, int64_t total) {
  return static_cast<int>(least(kShares, largest(1, total / (4 * (kTile * a.group + 128)))));
}
__device__ __forceinline__ int64_t share_begin(int64_t total, int g, int n) {
  // (total * g may pass 64 bits only where total passes 2^54)
  return total / n * g + total % n * g / n;
}

template <int RG, int NT>
struct Work {
  Window a;
  int64_t* pre;   // LDS [NT]: counts up to and with request base + i
  int64_t* wsum;  // LDS [NT / 64]
  int base;
  int64_t carry, total;
  struct Unit {
    Ragged rq;
    int b, kh, rg;
    int64_t begin, cost;  // where its counts begin, how many they are
  };
  // the unit behind u; whether it is one of its request and head
  __device__ __forceinline__ bool step(Unit& u) const {
    const Groups g = groups_of<RG>(a, u.rq);
    if (u.rg + 1 >= g.n) return false;
    ++u.rg;
    u.begin += u.cost;
    u.cost = uniform64(g.template cost<RG>(u.rg));
    return true;
  }
  // pre for the requests from `first` on; every thread must call it
  __device__ __forceinline__ void fill(int first, int64_t before) {
    const int thread = here(threadIdx.x), lane = thread & 63, wave = thread >> 6;
    base = first;
    carry = before;
    int64_t v = 0;
    if (first + thread < a.requests) {
      const Groups g = groups_of<RG>(a, ragged(a, first + thread));
      v = g.template upto<RG>(g.n) * a.kv_heads;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = __shfl_up(v, d);
      if (lane >= d) v += o;
    }
    __syncthreads();  // (the last fill's readers are done)
    if (lane == 63) wsum[wave] = v;
    __syncthreads();
    v += carry;
    for (int i = 0; i < wave; ++i) v += wsum[i];
    pre[thread] = v;
    __syncthreads();
  }
  // the total
  __device__ __forceinline__ void start() {
    total = 0;
    for (int f = 0; f < a.requests; f += NT) {
      fill(f, total);
      total = uniform64(pre[NT - 1]);
    }
    if (base) fill(0, 0);
  }
  // the unit at pos < total, pos not before the last call's
  __device__ __forceinline__ Unit find(int64_t pos) {
    while (pos >= uniform64(pre[NT - 1])) fill(base + NT, uniform64(pre[NT - 1]));
    int lo = 0, hi = NT - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= pos) lo = mid + 1;
      else hi = mid;
    }
    Unit u;
    u.b = base + uniform(lo);
    const Ragged rq = ragged(a, u.b);
    u.rq = Ragged{uniform(rq.row0), uniform(rq.tokens), uniform(rq.len), uniform(rq.first)};
    const Groups g = groups_of<RG>(a, u.rq);
    const int64_t first = uniform64(lo ? pre[lo - 1] : carry), per = g.template upto<RG>(g.n);
    int kh = 0;  // (few: no division)
    while (kh + 1 < a.kv_heads && first + (kh + 1) * per <= pos) ++kh;
    u.kh = uniform(kh);
    const int64_t head = first + u.kh * per;
    // the last group that begins by pos
    int at = 0, end = g.n - 1;
    while (at < end) {
      const int mid = (at + end + 1) >> 1;
      if (head + g.template upto<RG>(mid) <= pos) at = mid;
      else end = mid - 1;
    }
    u.rg = uniform(at);
    u.begin = uniform64(head + g.template upto<RG>(u.rg));
    u.cost = uniform64(g.template cost<RG>(u.rg));
    return u;
  }
};
// a < b, both wave-uniform: 64-bit numbers are compared in vector registers, where none shall
// be kept for it
__device__ __forceinline__ bool below(int64_t a, int64_t b) {
  asm volatile("" : "+s"(b));
  return a < b;
}
// The first of a unit's `tiles` that lies behind `counts` of its cost.  (In floats: any rule does
// that never falls as counts grow and that both shares of a border follow; a 64-bit division takes
// a hundred instructions.)
__device__ __forceinline__ int tile_at(int64_t counts, int64_t cost, int tiles) {
  if (counts <= 0) return 0;
  if (counts >= cost) return tiles;
  const float per = static_cast<float>(tiles) * __builtin_amdgcn_rcpf(static_cast<float>(cost));
  return min(static_cast<int>(static_cast<float>(counts) * per), tiles);
}

// 32 rows of a wave and their running sums, for v_mfma_f32_32x32x16: lane l holds row l%32 and
// of a step's 32 keys or of 32 dims those 8 b + 4 (l/32) + i (b, i < 4).  S^T = K Q^T: A = K
// (lane: key l%32, 8 dims from 8 (l/32) of each sixteen), B = Q^T.  O^T = V^T P^T: B = P^T as
// it lies there, two products of sixteen keys, A = V^T in the same order.
template <int D, bool F16>
struct Rows32 {
  using E = Elem<F16>;
  static constexpr int DC = D / 16, DV = D / 32;
  u32x4 q[DC];
  f32x16 o[DV];
  float mx, sum;  // the reference; the lane's own part of the weights' sum
  int pos;        // where the row stands
  bool far;       // some row's reference is beyond kFar (the same in all lanes)

  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    typedef typename E::x8 x8;
    if constexpr (F16)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float both(float v, bool max) {
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max ? fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])) : __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }

  __device__ __forceinline__ void load(const Window& a, const Ragged& rq, int kh, int row0, int nrows, int lane) {
    const int row = min(row0 + (lane & 31), nrows - 1), t = row / a.group;  // (rows past the last repeat it)
    const uint16_t* p = a.q + (rq.row0 + t) * a.q_row + (kh * a.group + row - t * a.group) * a.q_head + 8 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < DC; ++d) q[d] = (ld16(p + 16 * d) ^ a.flip) & a.keep;
    pos = rq.first + t;
    // (they have arrived here: a wait for them inside the loop over the keys would be
    // a wait for the keys on their way too)
#pragma unroll
    for (int d = 0; d < DC; ++d) asm volatile("" : "+v"(q[d]));
    far = false;
    mx = kLow;
    sum = 0.f;
#pragma unroll
    for (int d = 0; d < DV; ++d) o[d] = f32x16{};
  }

  static __device__ __forceinline__ int key_of(int e, int lane) { return 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }
  // the scores of a step at key0, -infinity where the lane's row does not see the key; bad: its absent sixteens
  __device__ __forceinline__ void hide(const Window& a, f32x16& x, int key0, uint32_t bad, int lane) const {
    const uint32_t m = visible32(key0, pos, low_of(pos, a.window), a.sinks) & ((bad & 1 ? 0 : 0xffffu) | (bad & 2 ? 0 : 0xffff0000u));
    const uint32_t t = m >> (4 * (lane >> 5));
    const uint32_t ok = (t & 0xf) | (t >> 4 & 0xf0) | (t >> 8 & 0xf00) | (t >> 12 & 0xf000);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = ok >> e & 1 ? x[e] : -INFINITY;
  }
  // The reference for two more steps' scores: another one, the largest so far, if one of them passes
  // the row's by too much; what was summed so far is brought to it later (settle).
  __device__ __forceinline__ bool lift(const Window& a, const f32x16 (&x)[2], float& next) {
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(fmaxf(top, x[0][e]), x[1][e]);
    top *= a.c;
    if (!__ballot(top - mx > kSlack + E::kHead)) return false;
    const float t = both(top, true);
    next = fmaxf(fabsf(t) > kFar ? t : t - E::kHead, mx);
    far = __ballot(fabsf(next) > kFar);
    return true;
  }
  __device__ __forceinline__ void settle(float next) {
    const float f = __builtin_amdgcn_exp2f(mx - next);
    mx = next;
    sum *= f;
#pragma unroll
    for (int d = 0; d < DV; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] *= f;
  }
  // Weights of a quarter n of a step against reference ref, rounded in p; their sum.
  static __device__ __forceinline__ float weights(const Window& a, const f32x16& x, int n, float ref, u32x4 (&p)[2]) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_amdgcn_exp2f(fmaf(x[4 * n + e], a.c, -ref));
    return take(y, n, p);
  }
  static __device__ __forceinline__ float take(const float (&y)[4], int n, u32x4 (&p)[2]) {
    p[n >> 1][2 * (n & 1)] = E::pack(y[0], y[1]);
    p[n >> 1][2 * (n & 1) + 1] = E::pack(y[2], y[3]);
    return (y[0] + y[1]) + (y[2] + y[3]);
  }
  // The same of a whole step, for references that the exponent's rounding matters for.
  static __device__ __forceinline__ float weights_far(const Window& a, const f32x16& x, float ref, u32x4 (&p)[2]) {
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __builtin_amdgcn_exp2f(exponent(x[4 * n + e], a.c, ref, true));
      sum += take(y, n, p);
    }
    return sum;
  }
  // values that are not finite (bit of odd; the products had zeros for them), for the rows that see them
  template <typename Value>
  __device__ __forceinline__ void add_odd(const Window& a, const u32x4& p0, const u32x4& p1, int key0, uint32_t odd, int lane,
                                          Value value) {
    for (uint32_t w = odd; w; w &= w - 1) {
      const int j = __builtin_ctz(w), e = 4 * (j >> 3) + (j & 3);
      const auto row = value(j);
      uint32_t y = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) y = e >> 1 == i ? (i >> 2 ? p1 : p0)[i & 3] : y;
      const float pj = E::low(__shfl(y, (lane & 31) + 32 * (j >> 2 & 1)) >> (16 * (e & 1)));
      if (!visible(key0 + j, pos, low_of(pos, a.window), a.sinks)) continue;
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] += pj * row(32 * d + key_of(i, lane));
    }
  }
  // The row's output, or (whole false: other keys of its are elsewhere) its sums at `slot0` + row.
  __device__ __forceinline__ void store(const Window& a, const Ragged& rq, int kh, int row0, int nrows, int lane, bool whole,
                                        int64_t slot0) {
    const int row = row0 + (lane & 31), at = 4 * (lane >> 5);
    const float total = both(sum, false);
    if (row >= nrows) return;
    const int t = row / a.group, head = kh * a.group + row - t * a.group;
    const int64_t token = rq.row0 + t;
    if (whole) {
      const float inv = total == 0.f ? 0.f : 1.f / total;
      uint16_t* p = a.out + token * a.out_row + head * a.out_head + at;
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *reinterpret_cast<u32x2*>(p + 32 * d + 8 * b) = u32x2{E::pack(o[d][4 * b] * inv, o[d][4 * b + 1] * inv),
                                                                E::pack(o[d][4 * b + 2] * inv, o[d][4 * b + 3] * inv)};
      if (a.lse && lane < 32) a.lse[token * a.q_heads + head] = log_sum(mx, total);
    } else {
      float* p = a.part + (slot0 + row) * D + at;
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *reinterpret_cast<f32x4*>(p + 32 * d + 8 * b) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
      if (lane < 32) *reinterpret_cast<f32x4*>(a.stat + 4 * (slot0 + row)) = f32x4{mx, total, total, 0.f};
    }
  }
};

// Eight waves of 32 rows share tiles of 64 keys through LDS.  A tile goes from memory to LDS past
// the registers, three ahead of the one that is computed: one barrier per tile, behind which
// the next one is whole and the last one's buffer is free.
//
// LDS rows are D/8 pieces of 16 bytes.  A wave reads keys as A operands, piece 2 c + l/32 of
// key l%32: piece p of key r lies at p ^ (r D / 128), so that the sixteen lanes of an access
// meet all banks.  Values are read transposed, 4 keys x 16 dims per 16 lanes (ds_read_b64_tr_b16:
// lane n gets dim n of the four keys), a pair of pieces of four keys per access: pairs are
// exchanged by twos, so that four keys x two pairs meet all banks.
//
// Bound by issue: the products of a step of 32 keys and 256 rows take 1024 cycles of a SIMD, its
// softmax nearly as many of the vector unit (an exponential takes four times an addition).  Between
// products of 32 x 32 there is room for six other instructions each, between those of 16 x 16,
// half as long, for one or two.  So a wave's products and softmax overlap: the products of the next
// tile's scores run beside the weights of this one's second step, those of this one's output
// beside the weights of the next one's first step, once its references are known.  Four requests of
// 1024 to 2048 rows over 4160 of their 4000 to 8000 tokens (201 GFLOP) in fp16: 251 us under a trace, 800
// TFLOP/s, the join 15, and as much without a trace for both; matrix units busy 46 %, LDS 20 % (all of a
// tile's weights beside the scores, its maxima beside the output: 258; two row tiles per wave of
// 16 x 16: 317 to 400; halves of the workgroup half a tile apart: 333).
template <int D, bool F16>
__global__ __launch_bounds__(64 * 8, 2) void window_wide_kernel(Window a0) {
  using W = Rows32<D, F16>;
  using E = Elem<F16>;
  constexpr int DC = W::DC, DV = W::DV, NW = 8, TK = kTile, RG = 32 * NW;
  constexpr int P = D / 8;       // pieces per row
  constexpr int KI = 64 / P;     // keys of one wave-wide load
  constexpr int KW = TK / NW;    // keys of a wave's loads: of one block
  constexpr int J = KW / KI;     // loads per wave, tile and matrix
  constexpr int kBuffers = 4;
  static_assert(16 % KW == 0 && TK == 64);
  __shared__ __attribute__((aligned(256))) uint16_t lkv[kBuffers][2][TK * D];  // (whole rows aligned: k_at)
  __shared__ uint32_t lflags[kBuffers][NW];  // of a wave's keys: those whose values are not finite; absent (bit 16)
  __shared__ __attribute__((aligned(16))) uint32_t lfrom[64 * NW][2 * J];
  __shared__ uint32_t lany;  // some block of the unit's has been absent
  __shared__ int64_t lpre[64 * NW], lsum[NW];
  const int lane = threadIdx.x & 63;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  // the exchanges of row r
  auto turn_k = [](int r) { return r * P / 16 & (P - 1); };
  auto turn_v = [](int r) { return P == 16 ? 4 * (r & 3) : 4 * (r >> 1 & 1); };
  // LDS byte addresses of this lane's pieces of the first step: key l%32, piece l/32; and of
  // dims 16 (l/16 % 2) + 4 (l%4) .. +3 of key 4 (l/32) + l/4 % 4
  const int vkey = 4 * (lane >> 5) + (lane >> 2 & 3);
  const uint32_t k_at = lds_address(lkv) + (lane & 31) * (2 * D) + 16 * ((lane >> 5) ^ turn_k(lane & 31));
  const uint32_t v_at = lds_address(lkv) + TK * D * 2 + vkey * (2 * D) +
                        16 * ((2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ turn_v(vkey)) + 8 * (lane & 1);
  Work<RG, 64 * NW> work{again<Window>(), lpre, lsum, 0, 0, 0};
  work.start();
  const int shares = shares_of(work.a, work.total), share = xcd_remap(blockIdx.x, gridDim.x);
  if (threadIdx.x == 0) a0.begun[share].b = -1;
  if (share >= shares) return;
  const int64_t begin = uniform64(share_begin(work.total, share, shares));
  const int64_t end = uniform64(share_begin(work.total, share + 1, shares));

  typename Work<RG, 64 * NW>::Unit un;
  bool known = false;
  for (int64_t pos = begin; below(pos, end);) {
    work.a = again<Window>();
    if (known) known = work.step(un);
    if (!known) un = work.find(pos);
    known = true;
    const Window& a = a0;
    const Ragged& rq = un.rq;
    const int kh = un.kh, nrows = rq.tokens * a.group, first_row = un.rg * RG;
    const int pmin = rq.first + first_row / a.group, pmax = rq.first + (min(first_row + RG, nrows) - 1) / a.group;
    const Span span = span_of<kTileBits>(a, pmin, pmax);
    // this share's tiles of the unit
    const int t0 = uniform(tile_at(pos - un.begin, un.cost, span.tiles));
    const int t1 = uniform(tile_at(end - un.begin, un.cost, span.tiles));
    pos = un.begin + un.cost;  // the next unit's
    const bool whole = t0 == 0 && t1 == span.tiles;
    if (t0 == 0 && t1 > 0 && !whole && threadIdx.x == 0) {
      int64_t total = work.total;
      asm volatile("" : "+s"(total));
      a0.begun[share] = Begun{un.b, kh, un.rg, !below(un.begin, begin), un.begin, un.cost, total};
    }
    if (t0 >= t1 && !(span.tiles == 0 && !below(un.begin, begin))) continue;
    const int row0 = first_row + wave * 32;  // of this wave (that has none: it computes the last row)
    // where this wave's rows stand
    const int wmin = rq.first + min(row0, nrows - 1) / a.group, wmax = rq.first + (min(row0 + 32, nrows) - 1) / a.group;

    const int32_t* table = a.tables + un.b * a.tstride;
    const uint16_t *kc = static_cast<const uint16_t*>(a.kc) + kh * a.kc_head;
    const uint16_t *vc = static_cast<const uint16_t*>(a.vc) + kh * a.vc_head;
    // the share's tiles of whose keys every row sees all (of the windows' part): plain0 .. plain0 + plains - 1
    const int plain0 = max(max(low_of(pmax, a.window) + TK, 0) / TK - span.from, 0) + span.sinks;
    const int plains = max((pmin + 1) / TK - span.from + span.sinks - plain0, 0);
    auto plain = [&](int i) { return static_cast<uint32_t>(i - plain0) < static_cast<uint32_t>(plains); };
    // Lane i: the block of this wave's keys of tile number id0 + i.  (Waited for where it is
    // loaded: a wait for it further on would be one for the keys on their way too.)
    int id_lane = 0, id0 = -(1 << 30);
    uint32_t absent = 0;  // bit i % 4: this wave's keys of the share's i-th tile are of an absent block
    uint32_t flagged = ~0u;  // bit i % 4: the wave's flags of that buffer may not be 0
    // The lane's pieces of its wave's rows (it fills piece l % P of its key's row in LDS: the
    // exchange picks what it reads), kept in LDS.
    {
      uint32_t from[2 * J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int ln = here(lane), piece = ln % P, at = j * KI + ln / P, r = wave * KW + at;
        from[2 * j] = 2 * (at * a.kc_slot + 8 * (piece ^ turn_k(r)));
        from[2 * j + 1] = 2 * (at * a.vc_slot + 8 * (piece ^ turn_v(r)));
      }
#pragma unroll
      for (int j = 0; j < 2 * J; ++j) lfrom[here(threadIdx.x)][j] = from[j];
    }
    // This share's i-th tile into its buffer, in three pieces that stand between the products of
    // another one (behind the last tile: that one again, where nothing reads it).
    int load_slot = 0, load_block = 0;
    auto fetch_ids = [&](int t) {
      const int last = (pmax & ~15) + wave * KW % 16;
      id0 = t;
      int slot;
      const int64_t key = least(static_cast<int64_t>(t + here(lane)) * TK + wave * KW, last);
      id_lane = table[block_of(a, static_cast<int>(key), slot)];
    };
    auto load_id = [&](int i) {
      const int t = span.tile(min(i, t1 - 1));
      // (keys of a sixteen past the last one are those of the sixteen with the last one instead, and masked)
      const int last = (pmax & ~15) + wave * KW % 16;
      if (__builtin_expect(static_cast<uint32_t>(t - id0) >= 64u, 0)) {
        fetch_ids(t);
        asm volatile("" : "+v"(id_lane));
      }
      const int id = __builtin_amdgcn_readlane(id_lane, t - id0);
      block_of(a, min(t * TK + wave * KW, last), load_slot);
      const bool bad = static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.blocks);
      absent = (absent & ~(1u << i % kBuffers)) | static_cast<uint32_t>(bad) << i % kBuffers;
      load_block = bad ? 0 : id;
    };
    auto load_part = [&](int i, int m) {  // m: keys, values
      const uint32_t to = lds_address(lkv) + (i % kBuffers) * (4 * TK * D) + m * (2 * TK * D) + wave * (KW * 2 * D);
      const uint16_t* base = m ? vc + (static_cast<int64_t>(load_block) * a.vc_block + static_cast<int64_t>(load_slot) * a.vc_slot)
                               : kc + (static_cast<int64_t>(load_block) * a.kc_block + static_cast<int64_t>(load_slot) * a.kc_slot);
      uint32_t from[J];
#pragma unroll
      for (int j = 0; j < J; ++j) from[j] = lfrom[here(threadIdx.x)][2 * j + m];
#pragma unroll
      for (int j = 0; j < J; ++j) load_lds(base, from[j], to + 1024 * j);
    };
    auto load = [&](int i) {
      load_id(i);
      load_part(i, 0);
      load_part(i, 1);
    };
    // This wave's part of the i-th tile has arrived: as in window_kernel, no infinity or NaN
    // may meet a weight of 0.
    auto to_settle = [&](int i) { return i < t1 && !(plain(i) && !((absent | flagged) >> i % kBuffers & 1)); };
    auto settle = [&](int i) {
      const int in = i % kBuffers;
      const int key0 = span.tile(i) * TK + wave * KW;
      const bool bad = absent >> in & 1, seen = !bad && all_visible(a, key0, key0 + KW - 1, pmin, pmax);
      uint32_t flags = bad ? 1u << 16 : 0;
      flagged = (flagged & ~(1u << in)) | static_cast<uint32_t>(!seen) << in;
      if (!seen) {
        const int ln = here(lane), kin = ln / P;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          u32x4* const at = reinterpret_cast<u32x4*>(&lkv[in][1][(wave * J + j) * 512 + 8 * ln]);
          const bool gone = bad || key0 + j * KI + kin > pmax;
          const u32x4 v = *at;
          bool wild = false;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            wild = wild || (v[x] & E::kExp) == E::kExp || (v[x] & E::kExp << 16) == E::kExp << 16;
          const unsigned long long m = __ballot(wild && !gone), one = P == 16 ? 0xffffull : 0xffull;
#pragma unroll
          for (int k = 0; k < KI; ++k)
            if (m >> (P * k) & one) flags |= 1u << (j * KI + k);
          const uint32_t zero = here(0);  // (no register keeps it meanwhile)
          if (gone || (m >> (P * kin) & one)) *at = u32x4{zero, zero, zero, zero};
        }
      }
      if (here(lane) == 0) {
        lflags[in][wave] = flags;
        if (bad) lany = 1;
      }
    };
    // bit h: sixteen h of the share's i-th tile is absent, from its flags
    auto absent_of = [&](uint32_t flags) {
      const uint32_t m = static_cast<uint32_t>(__ballot(here(lane) < NW && flags >> 16));
      uint32_t b = 0;
#pragma unroll
      for (int h = 0; h < 4; ++h) b |= (m >> (h * (16 / KW)) & 1) << h;
      return b;
    };

    W w;
    typedef f32x16 Scores[2];  // of a tile's two steps
    // keys of a quarter n of tile i's (step n / 2, half of the dims n % 2) as A operands: a piece's
    // exchange is an exclusive or of its row's address with 16 bytes times the piece, steps are
    // whole sixteens apart
    auto read_keys = [&](int i, int n, u32x4 (&k)[DC / 2]) {
      const uint32_t at = k_at + (i % kBuffers) * (4 * TK * D) + 32 * (n >> 1) * (2 * D);
#pragma unroll
      for (int d = 0; d < DC / 2; ++d) k[d] = *lds<const u32x4>(at ^ (32 * (d + (n & 1) * (DC / 2))));
    };
    auto multiply_keys = [&](int n, const u32x4 (&k)[DC / 2], Scores& s) {
      if ((n & 1) == 0) s[n >> 1] = f32x16{};
#pragma unroll
      for (int d = 0; d < DC / 2; ++d) s[n >> 1] = W::mfma(k[d], w.q[d + (n & 1) * (DC / 2)], s[n >> 1]);
    };
    // values of a quarter's sixteen keys, transposed
    auto read_values = [&](int i, int n, u32x4 (&v)[DV]) {
      const uint32_t at0 = v_at + (i % kBuffers) * (4 * TK * D) + 16 * n * (2 * D);
#pragma unroll
      for (int d = 0; d < DV; ++d) {
        const uint32_t at = at0 ^ (64 * d);
        const u32x2 lo = read_transposed(at), hi = read_transposed(at + 8 * (2 * D));
        v[d] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    // Tile i's scores in s, whether one of them may need a higher reference: what its rows do not
    // see is hidden; the reference that they go by.
    auto take = [&](int i, Scores& s, bool over, uint32_t any, float& ref, bool& lifted) {
      bool masked = !plain(i);
      uint32_t bm = 0;
      if (__builtin_expect(masked || any, 0)) {
        bm = absent_of(lflags[i % kBuffers][here(lane) & (NW - 1)]);
        const int key0 = span.tile(i) * TK;
        masked = bm || !all_visible(a, key0, key0 + TK - 1, wmin, wmax);
        if (masked) {
          w.hide(a, s[0], key0, bm, here(lane));
          w.hide(a, s[1], key0 + 32, bm >> 2, here(lane));
        }
      }
      if (__builtin_expect(masked || over || w.far, 0)) lifted = w.lift(a, s, ref);
    };

    constexpr int L = 2 * J;  // loads of a wave per tile
    if (threadIdx.x == 0) lany = 0;
    if (t0 < t1) fetch_ids(span.tile(t0));
    w.load(again<Window>(), rq, kh, min(row0, nrows - 1), nrows, here(lane));
    __syncthreads();
    if (t0 < t1) {
#pragma unroll 1
      for (int i = t0; i < t0 + 3; ++i) load(i);
      Scores s0, s1;
      arrived<2 * L>();
      settle(t0);
      __syncthreads();
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        u32x4 k[DC / 2];
        read_keys(t0, n, k);
        multiply_keys(n, k, s0);
      }
      float ref = w.mx;
      bool lifted = false, settles = to_settle(t0 + 1);
      take(t0, s0, true, lany, ref, lifted);
      if (lifted) w.settle(ref);
      u32x4 first[2];  // the weights of a tile's first step
#pragma unroll
      for (int n = 0; n < 4; ++n) w.sum += W::weights(a, s0[0], n, w.mx, first);
      if (w.far) w.sum = W::weights_far(a, s0[0], w.mx, first);

      // Tile i, its scores in x, its first step's weights in `first`; the next one's go to s and
      // `first`.
      auto tile = [&](int i, const Scores& x, Scores& s) {
        // One barrier per tile: behind it the next one is whole, and the buffer of the one
        // before free.
        arrived<L>();  // (all but the tile after the next)
        if (__builtin_expect(settles, 0)) settle(i + 1);
        __syncthreads();
        const uint32_t any_v = lany;
        u32x4 k[2][DC / 2], v[2][DV], second[2];
        float sum = 0.f, top = -INFINITY;
        read_keys(i + 1, 0, k[0]);
        // the next one's scores beside the second step's weights (behind the last: of what lies there)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          __builtin_amdgcn_sched_barrier(0);
          if (n < 3) read_keys(i + 1, n + 1, k[~n & 1]);
          else read_values(i, 0, v[0]);
          __builtin_amdgcn_sched_barrier(0);
          multiply_keys(n, k[n & 1], s);
          sum += W::weights(a, x[1], n, w.mx, second);
          if (n >= 2)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, s[0][8 * (n & 1) + e]);
          asm volatile("" : "+v"(second[n >> 1]), "+v"(sum));  // (here, not where they are used)
          interleave<DC / 2, 4, 10>();
          __builtin_amdgcn_sched_barrier(0);
          if (n == 0) load_id(i + 3);
          if (n == 1 || n == 2) load_part(i + 3, n - 1);
          if (n == 3) settles = to_settle(i + 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__builtin_expect(w.far, 0)) sum = W::weights_far(a, x[1], w.mx, second);
        w.sum += sum;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[1][e]);
        float ref = w.mx;
        bool lifted = false;
        if (i + 1 < t1)
          take(i + 1, s, __ballot(fmaf(top, a.c, -w.mx) > kSlack + E::kHead), uniform(static_cast<int>(any_v)), ref, lifted);
        // this one's output beside the next one's weights of its first step
        u32x4 next[2];
        sum = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          __builtin_amdgcn_sched_barrier(0);
          if (n < 3) read_values(i, n + 1, v[~n & 1]);
          __builtin_amdgcn_sched_barrier(0);
          const u32x4 p = n < 2 ? first[n] : second[n - 2];
#pragma unroll
          for (int d = 0; d < DV; ++d) w.o[d] = W::mfma(v[n & 1][d], p, w.o[d]);
          sum += W::weights(a, s[0], n, ref, next);
          asm volatile("" : "+v"(next[n >> 1]), "+v"(sum));
          interleave<DV, 4, 10>();
        }
        __builtin_amdgcn_sched_barrier(0);
        // (settle took values out of a tile for all rows where one of the workgroup's does not see it
        // whole, so this wave's may see it whole and still be owed them)
        if (__builtin_expect(!plain(i), 0)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t odd = 0;
#pragma unroll
            for (int n = 0; n < 32 / KW; ++n) odd |= (lflags[i % kBuffers][j * (32 / KW) + n] & 0xffff) << (n * KW);
            odd = uniform(static_cast<int>(odd));
            const int key0 = span.tile(i) * TK + 32 * j;
            if (odd) w.add_odd(a, j ? second[0] : first[0], j ? second[1] : first[1], key0, odd, here(lane), [&](int n) {
              int slot;
              const int id = table[block_of(a, key0 + n, slot)];
              const uint16_t* at = vc + static_cast<int64_t>(id) * a.vc_block + static_cast<int64_t>(slot) * a.vc_slot;
              return [at](int e) { return E::low(at[e]); };
            });
          }
        }
        if (__builtin_expect(w.far, 0)) sum = W::weights_far(a, s[0], ref, next);
        if (__builtin_expect(lifted, 0)) w.settle(ref);
        if (i + 1 < t1) w.sum += sum;
        first[0] = next[0], first[1] = next[1];
      };
      for (int i = t0; i < t1; i += 2) {
        tile(i, s0, s1);
        if (i + 1 < t1) tile(i + 1, s1, s0);
      }
      __syncthreads();  // (the next unit's tiles go where these were)
    }
    w.store(again<Window>(), rq, kh, row0, nrows, here(lane), whole,
            static_cast<int64_t>(2 * share + (!below(un.begin, begin))) * RG - first_row);
  }
  arrived<0>();  // (no load into LDS outlives the workgroup)
}

// Behind window_wide_kernel: the units that a share began and left to others, four rows a wave.
// Bound by memory: two parts a share at most, 69 MB in 14.5 us.
template <int D, bool F16, int RG>
__global__ __launch_bounds__(join_threads(1)) void window_wide_join_kernel(Window a) {
  const int lane = threadIdx.x & 63, li = lane & 15, wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int s0 = blockIdx.x / (RG / 16), first = (blockIdx.x % (RG / 16)) * 16 + 4 * wave;
  const Begun u = a.begun[s0];
  if (u.b < 0) return;
  const Ragged rq = ragged(a, u.b);
  const int rows = rq.tokens * a.group, first_row = u.rg * RG;
  if (first_row + first >= rows) return;
  const Span span = span_of<kTileBits>(a, rq.first + first_row / a.group,
                                       rq.first + (min(first_row + RG, rows) - 1) / a.group);
  // the last share that has some of its tiles
  const int64_t total = u.total;
  const int n = shares_of(a, total);
  int s1 = static_cast<int>(least((u.begin + u.cost) / largest(total / n, 1), n - 1));
  while (s1 > s0 && tile_at(share_begin(total, s1, n) - u.begin, u.cost, span.tiles) >= span.tiles) --s1;
  const int row = min(first_row + first + (lane >> 4), rows - 1), t = row / a.group, head = u.kh * a.group + row - t * a.group;
  uint16_t* p = a.out + (rq.row0 + t) * a.out_row + head * a.out_head + D / 16 * li;
  join_rows<D, F16, 1, 4>(a.part, a.stat, s1 - s0 + 1, lane, wave, first_row + first + (lane >> 4) < rows ? p : nullptr,
                          a.lse ? a.lse + static_cast<int64_t>(rq.row0 + t) * a.q_heads + head : nullptr, [&](int i) {
                            return static_cast<int64_t>(2 * (s0 + i) + (i == 0 ? u.slot : 0)) * RG + row - first_row;
                          });
}

// Many rows over a 4-bit cache: every request's tokens are widened once into 16-bit blocks of
// sixteen, [request][columns][head][16][D], exactly (fp16: below 2^-16 to a multiple of
// 2^-24, which moves a score by 2^-25 sum |q| at most and a value by half a step of the output),
// with a table of their own, and the wide kernel reads those.  Each value is read by hundreds of
// rows, which this costs one write and one read of 16 bits; widened in the wide kernel it would
// be a third more instructions beside its products.  One workgroup per block: a thread has eight dims
// of a token.  8000 and 16000 tokens of 2 x 128 dims (6.9 MB to 24.6 MB) 9.5 us, 3.3 TB/s of the 5.1 of a
// copy: a workgroup's loads wait for its block's number, and it has one turn of them.
struct Widen {
  Window w;
  uint16_t *k, *v;
  int32_t* tables;  // [requests][columns]
  int32_t columns, grid;  // grid: workgroups of a request
};
template <int D, bool F16>
__device__ __forceinline__ void widen_block(const Widen& g, int b, int col) {
  const Window& a = g.w;
  constexpr int C = D / 32, P = D / 8;
  int slot;
  const int id = a.tables[b * a.tstride + block_of(a, col * 16, slot)];
  const bool bad = id < 0 || id >= a.blocks;
  const int at0 = b * g.columns + col;
  if (threadIdx.x == 0) g.tables[at0] = bad ? -1 : at0;
  if (bad) return;
  for (int u = threadIdx.x; u < a.kv_heads * 16 * P; u += 256) {
    const int i = u % P, token = u / P % 16, h = u / (16 * P), c = i / 4;
    const int64_t row = row_of(a, id, slot, h), at = row + token;
    const uint32_t key = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.kc) + at * (D / 2))[C * (i % 4) + c];
    const uint8_t* p = static_cast<const uint8_t*>(a.vc) + row * (D / 2) + ((16 * (token >> 2) + 8 * (i & 1)) * 4 + (token & 3)) * C + c;
    uint32_t value = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) value |= (p[e * 4 * C] >> (i & 2 ? 4 : 0) & 15u) << (4 * e);
    const float ks = low_bf16(a.ks[at * C + c]), vs = low_bf16(a.vs[at * C + c]);
    const int64_t to = (static_cast<int64_t>(at0) * a.kv_heads * 16 + (h * 16 + token)) * D + 8 * i;
    float f[8];
    fp4x8_to_f32(key, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= ks;
    store_dequant16<F16 ? PGS_DTYPE_F16 : PGS_DTYPE_BF16>(g.k, to, f);
    fp4x8_to_f32(value, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= vs;
    store_dequant16<F16 ? PGS_DTYPE_F16 : PGS_DTYPE_BF16>(g.v, to, f);
  }
}

template <int D, bool F16>
__global__ __launch_bounds__(256) void widen_kernel(Widen g) {
  const Window& a = g.w;
  const int b = blockIdx.x / g.grid;
  const Ragged rq = ragged(a, b);
  if (rq.tokens == 0) return;
  for (int64_t col = blockIdx.x % g.grid; col * 16 < rq.len; col += g.grid) {
    // (what no row of the request sees is left out)
    if (col * 16 + 15 <= low_of(rq.first, a.window) && col * 16 >= a.sinks) continue;
    widen_block<D, F16>(g, b, static_cast<int>(col));
  }
}

// The launch shape, a function of sizes the host knows (never of what the device
// arrays hold, so that a captured call replays with other lengths).
struct Plan {
  int wide;   // rows of a group that share tiles through LDS, or 0
  int r, wr;  // else row tiles per wave, waves per key slice (4-bit: one tile per wave, r times the waves)
  bool pair;  // (4-bit) eight rows at most, in pairs of columns
  int groups, splits, min_steps;
  int64_t columns, chunk, widen;  // (wide, 4-bit) blocks of sixteen a request, requests widened at a time, workgroups each
};
constexpr int64_t kWidened = int64_t{1} << 29;  // bytes of 16-bit keys and values at a time, if one request's are no more
Plan plan(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens, int64_t max_context,
          int64_t window, int64_t sinks, bool fp4, int64_t columns, int64_t block_size) {
  const int64_t rows = max_tokens * (q_heads / kv_heads);
  Plan p{};
  p.splits = 1;
  const int64_t tokens = std::min<int64_t>(max_tokens, 64);  // of a row group
  // (the most tokens that a row group sees)
  const int64_t seen = window + std::min(sinks, max_context) + tokens >= max_context ? max_context : window + sinks + tokens;
  p.groups = static_cast<int>((rows + 63) / 64);
  const int64_t units = requests * kv_heads * p.groups;
  // Rows that share tiles through LDS run at three times the rate, but their equal shares cost 30
  // us before that.  By units x steps of 32 keys, us straight from memory and shared (128 dims,
  // 16 bits): 256 (64 rows over 500 tokens) 21 / 38, 2048 (four of 64 over 1000) 22 / 44, 4032
  // (256 over 2000) 31 / 48, 8192 (1024 over 1024) 45 / 47, 16000 (512 over 4000) 67 / 57.  Of
  // 64 dims, and of 4 bits, which are not widened first then, they meet at twice as many: 14000
  // (512 over 4000, 64 dims) 42 / 44, 16000 (512 over 4000, 4 bits) 63 / 62, 28000 (2048 over 2048, 64
  // dims) 48 / 46.  (For the batch as a whole, by its longest request: one prompt among single tokens
  // takes them into shared tiles too, where each of them is a row group of its own.)
  const int64_t few = fp4 || head_dim == 64 ? 16384 : 8192;
  p.wide = rows <= 64 || units * std::max<int64_t>(1, (seen + 31) / 32) <= few ? 0 : 256;
  if (p.wide) {
    if (fp4) {
      p.columns = (columns * block_size + 15) / 16;
      // (a launch has fewer than 2^32 threads: of several requests' chunk it always has)
      p.widen = std::max<int64_t>(1, std::min({p.columns, (max_context + 15) / 16, int64_t{0xffffffff / 256}}));
      p.chunk = std::max<int64_t>(1, std::min<int64_t>(requests, kWidened / std::max<int64_t>(1, p.columns * kv_heads * 64 * head_dim)));
    }
    return p;
  }
  p.r = rows <= 16 ? 1 : 2;
  p.pair = fp4 && rows <= 8;
  p.wr = rows <= 32 ? 1 : 2;
  const int64_t steps = (seen + 31) / 32 * p.wr;
  p.min_steps = units * (steps / kCoarseSteps) <= 128 ? kFineSteps : kCoarseSteps;
  // (as many workgroups as run at a time: 4-bit rows leave registers for three per CU, where a
  // fourth would wait: 32 requests of 8000 to 16000 tokens in 25.6 instead of 29.0 us)
  if (steps >= kWholeSteps)
    p.splits = static_cast<int>(
        std::max<int64_t>(1, std::min<int64_t>({((fp4 ? 768 : 1024) + units - 1) / units, steps / p.min_steps, 256})));
  return p;
}
int64_t slots_of(const Plan& p, int64_t rows, int64_t q_heads) {
  return p.wide ? int64_t{2} * kShares * p.wide : p.splits == 1 ? 0 : rows * q_heads * p.splits;
}
// the sums of parts, then (wide) the units begun, then (4-bit) keys, values and tables
size_t parts_bytes(const Plan& p, int64_t rows, int64_t q_heads, int64_t head_dim) {
  return (static_cast<size_t>(slots_of(p, rows, q_heads)) * (head_dim + 4) * 4 + (p.wide ? kShares * sizeof(Begun) : 0) + 255) /
         256 * 256;
}
size_t workspace_bytes(const Plan& p, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  return parts_bytes(p, rows, q_heads, head_dim) + static_cast<size_t>(p.chunk * p.columns) * (kv_heads * 64 * head_dim + 4);
}

bool sizes_ok(int64_t rows, int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens,
              int64_t max_context, int64_t window, int64_t sinks) {
  if (!(rows >= 0 && rows <= 0x7fffffff / 64 && requests >= 0 && requests <= 0x100000 && kv_heads >= 1 &&
        q_heads >= kv_heads && q_heads % kv_heads == 0 && q_heads <= 4096 && (head_dim == 64 || head_dim == 128) &&
        max_tokens >= 1 && max_tokens <= 0x7fffffff / 64 && max_context >= 0 && max_context <= 0x7fffffff && window >= 1 &&
        window <= 0x7fffffff && sinks >= 0 && sinks <= 0x7fffffff))
    return false;
  const int64_t most = std::min(max_tokens, std::max<int64_t>(rows, 1)) * q_heads;  // rows x heads of a request
  // (Rows straight from memory: workgroups of 256 threads for requests x key heads, or few, and fewer
  // than 2^32 threads.  Shared tiles have one grid whatever there is.)
  return most <= 0x3fffffff && requests * kv_heads <= 0xffffff && requests * most <= int64_t{1} << 40;
}

template <int D, bool F16>
int launch_wide(const Window& a, hipStream_t st) {
  hipLaunchKernelGGL((window_wide_kernel<D, F16>), dim3(kShares), dim3(512), 0, st, a);
  if (int rc = check_launch("window attention kernel")) return rc;
  hipLaunchKernelGGL((window_wide_join_kernel<D, F16, 256>), dim3(kShares * 16), dim3(256), 0, st, a);
  return check_launch("window attention join kernel");
}

template <int D, bool F16>
int launch_wide4(const Window& a, const Plan& p, char* widened, hipStream_t st) {
  const int64_t block = static_cast<int64_t>(a.kv_heads) * 16 * D;
  for (int64_t b = 0; b < a.requests; b += p.chunk) {
    Widen g{a, reinterpret_cast<uint16_t*>(widened), nullptr, nullptr, static_cast<int32_t>(p.columns), static_cast<int32_t>(p.widen)};
    g.v = g.k + p.chunk * p.columns * block;
    g.tables = reinterpret_cast<int32_t*>(g.v + p.chunk * p.columns * block);
    Window& w = g.w;
    w.requests = static_cast<int32_t>(std::min<int64_t>(p.chunk, a.requests - b));
    w.lens += b, w.offsets += b, w.tables += b * a.tstride;
    hipLaunchKernelGGL((widen_kernel<D, F16>), dim3(static_cast<unsigned>(w.requests * p.widen)), dim3(256), 0, st, g);
    if (int rc = check_launch("widen kernel")) return rc;
    w.kc = g.k, w.vc = g.v;
    w.kc_block = w.vc_block = block, w.kc_head = w.vc_head = 16 * D, w.kc_slot = w.vc_slot = D;
    w.blocks = static_cast<int32_t>(w.requests * p.columns), w.bs = 16, w.bs_inv = 1u << 28;
    // (lengths are cut to what the caller's tables hold, a multiple of sixteen too)
    w.tables = g.tables, w.tstride = p.columns, w.cols = static_cast<int32_t>(p.columns);
    if (int rc = launch_wide<D, F16>(w, st)) return rc;
  }
  return PGS_OK;
}

template <int D, bool F16, bool FP4>
int launch(const Window& a, const Plan& p, char* widened, hipStream_t st) {
  if (p.wide) {
    if constexpr (FP4) return p.columns == 0 ? launch_wide<D, F16>(a, st) : launch_wide4<D, F16>(a, p, widened, st);
    else return launch_wide<D, F16>(a, st);
  }
  const dim3 g(static_cast<unsigned>(static_cast<int64_t>(a.requests) * a.kv_heads * p.groups * p.splits));
  constexpr int R = FP4 ? 1 : 2;
  if (FP4 && p.pair) hipLaunchKernelGGL((window_kernel<D, 1, 1, 4, F16, FP4, FP4>), g, dim3(256), 0, st, a);
  else if (p.r == 1) hipLaunchKernelGGL((window_kernel<D, 1, 1, 4, F16, FP4, false>), g, dim3(256), 0, st, a);
  else if (p.wr == 1) hipLaunchKernelGGL((window_kernel<D, R, 2 / R, 4, F16, FP4, false>), g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((window_kernel<D, R, 4 / R, 4, F16, FP4, false>), g, dim3(256), 0, st, a);
  if (int rc = check_launch("window attention kernel")) return rc;
  if (p.splits == 1) return PGS_OK;
  const int64_t quads = static_cast<int64_t>(a.requests) * a.kv_heads * ((a.max_tokens * a.group + 3) / 4);
  auto join = [&](auto waves, auto rg, auto sliced) {
    constexpr int W = decltype(waves)::value;
    constexpr bool S = decltype(sliced)::value;
    hipLaunchKernelGGL((window_join_kernel<D, F16, W, decltype(rg)::value, S>),
                       dim3(static_cast<unsigned>(W == 1 ? (quads + 3) / 4 : quads * (S ? D / 64 : 1))), dim3(join_threads(W)), 0,
                       st, a, p.wr);
  };
  auto by = [&](auto waves, auto sliced) {
    if (p.r == 1) join(waves, Int<16>{}, sliced);
    else if (p.wr == 1) join(waves, Int<32>{}, sliced);
    else join(waves, Int<64>{}, sliced);
  };
  if (!join_by_many(p.splits, quads)) by(Int<1>{}, Int<0>{});
  else if (join_sliced(quads, D)) by(Int<kJoinWaves>{}, Int<1>{});
  else by(Int<kJoinWaves>{}, Int<0>{});
  return check_launch("window attention join kernel");
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" size_t pgs_window_attention_workspace_bytes(const pgs_window_attention_args* args) {
  if (!args || !args->cache == !args->cache4) return 0;
  const pgs_window_attention_args& g = *args;
  const int64_t kv = g.cache ? g.cache->kv_heads : g.cache4->kv_heads, dim = g.cache ? g.cache->head_dim : g.cache4->head_dim;
  const int64_t size = g.cache ? g.cache->block_size : g.cache4->block_size;
  if (!sizes_ok(g.rows, g.requests, g.q_heads, kv, dim, g.max_tokens, g.max_context, g.window, g.sinks) || g.rows == 0 ||
      g.requests == 0 || size < 16 || size > 0x10000 || g.columns < 0 || g.columns > 0x7fff0000 / size)
    return 0;
  const Plan p = plan(g.requests, g.q_heads, kv, dim, std::min(g.max_tokens, g.rows), g.max_context, g.window, g.sinks,
                      !g.cache, g.columns, size);
  return workspace_bytes(p, g.rows, g.q_heads, kv, dim);
}

extern "C" int pgs_window_attention(const pgs_window_attention_args* args, void* workspace, size_t workspace_bytes_given,
                                    void* stream) {
  const char* fn = "pgs_window_attention";
  if (!args) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null arguments", fn);
  const pgs_window_attention_args& g = *args;
  if (g.dtype != PGS_DTYPE_BF16 && g.dtype != PGS_DTYPE_F16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: dtype %d must be bf16 or fp16", fn, g.dtype);
  Window a{};
  if (int rc = take_cache(fn, a, g.cache, g.cache4, true, g.block_tables, g.table_stride, g.columns, g.requests))
    return rc;
  const int64_t dim = g.cache ? g.cache->head_dim : g.cache4->head_dim;
  if (!sizes_ok(g.rows, g.requests, g.q_heads, a.kv_heads, dim, g.max_tokens, g.max_context, g.window, g.sinks))
    return fail(PGS_ERR_INVALID_ARGUMENT,
                "%s: rows=%lld requests=%lld q_heads=%lld kv_heads=%d max_tokens=%lld window=%lld sinks=%lld: q_heads is a "
                "multiple of kv_heads, max_tokens and window 1 at least, sinks 0 at least",
                fn, (long long)g.rows, (long long)g.requests, (long long)g.q_heads, a.kv_heads, (long long)g.max_tokens,
                (long long)g.window, (long long)g.sinks);
  for (int64_t s : {g.q_row, g.q_head, g.out_row, g.out_head})
    if (s < 0 || s % 8 != 0) return fail(PGS_ERR_MISALIGNED, "%s: strides must be multiples of 8 elements", fn);
  if (!(g.scale == g.scale)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: scale is NaN", fn);
  if (g.rows == 0 || g.requests == 0) return PGS_OK;
  if (!g.q || !g.out || !g.lens || !g.offsets) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(g.q, 16) || !aligned(g.out, 16) || !aligned(g.lse, 4) || !aligned(g.lens, 4) || !aligned(g.offsets, 4))
    return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  const int64_t most = std::min(g.max_tokens, g.rows);  // (no request has more rows than the batch)
  const Plan p = plan(g.requests, g.q_heads, a.kv_heads, dim, most, g.max_context, g.window, g.sinks, !g.cache, g.columns, a.bs);
  const size_t need = workspace_bytes(p, g.rows, g.q_heads, a.kv_heads, dim);
  // (what all units cost has to fit 64 bits)
  const double group = static_cast<double>(g.q_heads / a.kv_heads);
  const double counts = (static_cast<double>(g.rows) * group / 256 + static_cast<double>(g.requests)) * a.kv_heads *
                        (static_cast<double>(g.columns) * a.bs + 2 * kUnit) * group;
  if (p.chunk * p.columns > 0x7fffffff || (p.wide && counts > 4e18))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: too large", fn);
  if (need > 0 && (!workspace || workspace_bytes_given < need || !aligned(workspace, 256)))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: needs a 256-byte aligned workspace of %zu bytes", fn, need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  a.q = static_cast<const uint16_t*>(g.q);
  a.out = static_cast<uint16_t*>(g.out);
  a.lse = g.lse;
  a.q_row = g.q_row, a.q_head = g.q_head, a.out_row = g.out_row, a.out_head = g.out_head;
  a.lens = g.lens, a.offsets = g.offsets;
  a.rows = static_cast<int32_t>(g.rows), a.requests = static_cast<int32_t>(g.requests);
  a.q_heads = static_cast<int32_t>(g.q_heads), a.group = a.q_heads / a.kv_heads;
  a.max_tokens = static_cast<int32_t>(most);
  a.window = static_cast<int32_t>(g.window), a.sinks = static_cast<int32_t>(g.sinks);
  a.groups = p.groups, a.splits = p.splits, a.min_steps = p.min_steps;
  // (a negative scale changes the rows' signs: the largest score is then always the largest weight's)
  a.c = std::fabs(g.scale) * 1.44269504088896340736f;
  // (and a scale of 0 the rows to zeros: -infinity times it would be no score)
  a.flip = std::signbit(g.scale) ? 0x80008000u : 0, a.keep = g.scale == 0.f ? 0 : ~0u;
  if (g.scale == 0.f) a.c = 1.f;
  a.part = static_cast<float*>(workspace);
  a.stat = a.part + slots_of(p, g.rows, g.q_heads) * dim;
  a.begun = reinterpret_cast<Begun*>(a.stat + slots_of(p, g.rows, g.q_heads) * 4);
  char* widened = static_cast<char*>(workspace) + parts_bytes(p, g.rows, g.q_heads, dim);
  auto go = [&](auto d, auto f16) {
    constexpr int D = decltype(d)::value;
    constexpr bool F = decltype(f16)::value;
    return g.cache ? launch<D, F, false>(a, p, widened, st) : launch<D, F, true>(a, p, widened, st);
  };
  if (dim == 64) return g.dtype == PGS_DTYPE_F16 ? go(Int<64>{}, Int<1>{}) : go(Int<64>{}, Int<0>{});
  return g.dtype == PGS_DTYPE_F16 ? go(Int<128>{}, Int<1>{}) : go(Int<128>{}, Int<0>{});
}
