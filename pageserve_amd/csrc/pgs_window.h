// Shared by the kernels over a sliding window with sinks: the call's arguments, which
// tokens a row sees, and a step's keys and values of the 16-bit or the 4-bit cache.
//
// Row t of a request of n rows and len cached tokens (the rows' own among them) stands at
// p = len - n + t and sees token j if j <= p and (j > p - window or j < sinks).
//
// The 4-bit cache, heads in front of slots, all contiguous (D: head_dim, C = D / 32):
//   k, v      uint8 [blocks][kv_heads][block_size][D / 2]: E2M1 codes
//   k_scale, v_scale  bf16 [blocks][kv_heads][block_size][C], one per 32 dims of a token,
//             of 6 significant bits: value * scale has 8, so it is a bf16 number
// A key's byte 4 (C a + c) + i holds dims 32 c + 8 a + 2 i (low half) and the next one:
// lane (a = l/16) reads its dims of all C chunks at once, each the A operand of a
// v_mfma_f32_16x16x32 after four conversions.
// Values, of 16 tokens: token 4 a + b has its dims m, 16 + m, 32 + m, ... (m < 16) in the
// C bytes from ((16 a + m) 4 + b) C on, low halves first: lane (a, m) reads those of its
// four tokens at once, and the dims 16 d + m of a product lie in the scale group d / 2.
// A token's bytes are its own in both, so rows are written independently.
#pragma once

#include <initializer_list>

#include "pgs_attend.h"
#include "pgs_fp4.h"

namespace pgs {
namespace {

// (the device's own min and max of two 64-bit integers go by way of doubles)
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t largest(int64_t a, int64_t b) { return a > b ? a : b; }

// A unit of work whose first part a share computed and the rest others; b < 0: none.
struct Begun {
  int32_t b, kh, rg, slot;  // slot: which of the share's two holds its sums
  int64_t begin, cost, total;
};

struct Window {
  const uint16_t* q;
  uint16_t* out;
  float* lse;  // [rows][q_heads], or null
  int64_t q_row, q_head, out_row, out_head;
  // the cache: 16-bit, or codes with their scales
  const void *kc, *vc;
  const uint16_t *ks, *vs;
  int64_t kc_block, kc_head, vc_block, vc_head;
  uint32_t kc_slot, vc_slot;
  int32_t blocks, bs;
  uint32_t bs_inv;  // ceil(2^32 / bs)
  const int32_t* tables;
  int64_t tstride;
  int32_t cols;
  const int32_t *lens, *offsets;
  int32_t rows, requests, q_heads, kv_heads, group;  // group: q_heads / kv_heads
  int32_t max_tokens, window, sinks;
  int32_t groups, splits, min_steps;  // row groups of a request; parts of the keys
  float c;      // |scale| * log2(e) (accumulate_weights: signed)
  uint32_t flip, keep;  // for the rows: the sign bits of a negative scale; no bits where it is 0
  float* part;  // sums of the parts of rows: [slots][D]
  float* stat;  // [slots][4]: reference, sum, sum of the weights before their rounding, -
  Begun* begun;   // (wide) [shares]
};

// The request of a unit and its sizes, each brought into range: whatever the device
// arrays hold, no access leaves the tensors.
struct Ragged {
  int row0, tokens, len, first;  // first: where row 0 stands (below 0: it sees nothing)
};
template <typename Args>
__device__ __forceinline__ Ragged ragged(const Args& a, int b) {
  Ragged r;
  const int lo = min(max(a.offsets[b], 0), a.rows);
  const int hi = min(max(a.offsets[b + 1], lo), a.rows);
  r.row0 = lo;
  r.tokens = min(hi - lo, a.max_tokens);
  const int64_t most = static_cast<int64_t>(a.cols) * a.bs;
  r.len = static_cast<int>(least(max(a.lens[b], 0), most));
  r.first = r.len - (hi - lo);
  return r;
}

// The tiles of T = 2^S keys that rows at pmin .. pmax see: some from the first on (sinks),
// then those of the windows.
struct Span {
  int sinks, from, tiles;  // sink tiles; the first of the windows; all
  __device__ __forceinline__ int tile(int i) const { return i < sinks ? i : from + i - sinks; }
};
template <int S, typename Args>
__device__ __forceinline__ Span span_of(const Args& a, int pmin, int pmax) {
  Span s{0, 0, 0};
  if (pmax < 0) return s;
  const int low = max(max(pmin, 0) - a.window + 1, 0);  // the first token of a window
  s.from = low >> S;
  s.sinks = (min(a.sinks, low) + (1 << S) - 1) >> S;
  if (s.sinks >= s.from) s.sinks = s.from = 0;  // (one piece)
  s.tiles = s.sinks + (pmax >> S) + 1 - s.from;
  return s;
}

// whether a row at p sees token j; low: p - window
__device__ __forceinline__ bool visible(int j, int p, int low, int sinks) { return j <= p && (j > low || j < sinks); }
// bits 0 .. n - 1 (none below 0, all from 32 on)
__device__ __forceinline__ uint32_t bits(int n) { return n >= 32 ? ~0u : (1u << max(n, 0)) - 1; }
// which of the keys key0 .. key0 + 31 it sees
__device__ __forceinline__ uint32_t visible32(int key0, int p, int low, int sinks) {
  return bits(p - key0 + 1) & (~bits(low < key0 ? 0 : low - key0 + 1) | bits(sinks - key0));
}
// (p - window for any p: where there is none p is below 0 and sees nothing anyhow)
__device__ __forceinline__ int low_of(int p, int window) { return max(p, -1) - window; }
// whether all rows at pmin .. pmax see all of the keys key0 .. last
template <typename Args>
__device__ __forceinline__ bool all_visible(const Args& a, int key0, int last, int pmin, int pmax) {
  return last <= pmin && (key0 > low_of(pmax, a.window) || last < a.sinks);
}

__device__ __forceinline__ float quad_sum(float v) {
  const uint32_t x = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const float s = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t y = __float_as_uint(s);
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ float low_bf16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_bf16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// eight codes -> eight values of the rows' type, exact
template <bool F16>
__device__ __forceinline__ u32x4 widen8(uint32_t d) {
  if constexpr (F16) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, 1.0f, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, 1.0f, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, 1.0f, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, 1.0f, 3))};
  } else {
    return __builtin_bit_cast(u32x4, fp4x8_to_bf16x8(d));
  }
}
// the pair of codes in byte S of d, in bf16
template <int S>
__device__ __forceinline__ uint32_t widen2(uint32_t d) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, 1.0f, S));
}

// The keys of one step of 32, half h: keys key0 + 16 h + l%16 as A operands of scores.
template <int D>
struct Keys16 {
  u32x4 k[2][D / 32];
};
template <int D>
struct Keys4 {
  uint32_t k[2][D / 32];
  uint32_t s[2][D / 16];  // scales of keys 4 (l/16) .. +3 of the half: of each D/32, in pairs
  // that of key i of the half and chunk c
  __device__ __forceinline__ float scale(int h, int i, int c) const {
    const uint32_t w = s[h][(i * (D / 32) + c) >> 1];
    return c & 1 ? high_bf16(w) : low_bf16(w);
  }
};
// Their values: keys 4 (l/16) .. +3 of both halves.
template <int D>
struct Values16 {
  uint32_t v[8][D / 32];  // dims (l%16) D/16 .. of key 4 h + i
};
template <int D>
struct Values4 {
  uint32_t v[2][D / 32];
  uint32_t s[2][D / 16];
  __device__ __forceinline__ float scale(int h, int i, int c) const {
    const uint32_t w = s[h][(i * (D / 32) + c) >> 1];
    return c & 1 ? high_bf16(w) : low_bf16(w);
  }
};

template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    const u32x2 x = *static_cast<const u32x2*>(p);
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 x = static_cast<const u32x4*>(p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
    }
  }
}

// Sixteen keys of key head kh, from `slot` on (a multiple of 16) of block blk.  All of
// them are in the block, written or not.
template <int D>
__device__ __forceinline__ void load_keys(const Window& a, int64_t blk, int slot, int kh, int li, int lg, u32x4 (&k)[D / 32]) {
  const uint16_t* p = static_cast<const uint16_t*>(a.kc) + blk * a.kc_block + static_cast<int64_t>(slot) * a.kc_slot +
                      kh * a.kc_head + static_cast<uint32_t>(li) * a.kc_slot + 8 * lg;
#pragma unroll
  for (int d = 0; d < D / 32; ++d) k[d] = ld16(p + 32 * d);
}
template <int D>
__device__ __forceinline__ void load_values(const Window& a, int64_t blk, int slot, int kh, int li, int lg,
                                            uint32_t (*v)[D / 32]) {
  const uint16_t* p = static_cast<const uint16_t*>(a.vc) + blk * a.vc_block + static_cast<int64_t>(slot) * a.vc_slot +
                      kh * a.vc_head + D / 16 * li;
#pragma unroll
  for (int e = 0; e < 4; ++e) load_words(p + static_cast<uint32_t>(4 * lg + e) * a.vc_slot, v[e]);
}
// (4-bit: the first of the sixteen is row `row` of [blocks * kv_heads * block_size])
__device__ __forceinline__ int64_t row_of(const Window& a, int64_t blk, int slot, int kh) {
  return (blk * a.kv_heads + kh) * a.bs + slot;
}
template <int D>
__device__ __forceinline__ void load_keys4(const Window& a, int64_t row, int li, int lg, uint32_t (&k)[D / 32],
                                           uint32_t (&s)[D / 16]) {
  load_words(static_cast<const uint8_t*>(a.kc) + (row + li) * (D / 2) + lg * (D / 8), k);
  load_words(a.ks + (row + 4 * lg) * (D / 32), s);
}
template <int D>
__device__ __forceinline__ void load_values4(const Window& a, int64_t row, int li, int lg, uint32_t (&v)[D / 32],
                                             uint32_t (&s)[D / 16]) {
  load_words(static_cast<const uint8_t*>(a.vc) + row * (D / 2) + (16 * lg + li) * (D / 8), v);
  load_words(a.vs + (row + 4 * lg) * (D / 32), s);
}

// Scores of a step's half h: lane l's keys 4 (l/16) + i of it, row l%16.  In 4 bits each
// chunk's sum is multiplied by its scale; nothing is rounded but in fp32.
template <int D, bool F16>
__device__ __forceinline__ f32x4 scores(const Keys16<D>& n, int h, const u32x4 (&q)[D / 32]) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D / 32; ++d) s = Elem<F16>::mfma(n.k[h][d], q[d], s);
  return s;
}
template <int D, bool F16>
__device__ __forceinline__ f32x4 scores(const Keys4<D>& n, int h, const u32x4 (&q)[D / 32]) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D / 32; ++d) {
    const f32x4 t = Elem<F16>::mfma(widen8<F16>(n.k[h][d]), q[d], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = fmaf(t[i], n.scale(h, i, d), s[i]);
  }
  return s;
}

// The same where columns r and r + 8 are row r, with its q of even chunks in one and of odd ones in
// the other (zeros elsewhere): one accumulator has two chunks' sums, each lane its own's scale
// (sel: the half of a word of two that it takes), and the two halves are added.
__device__ __forceinline__ uint32_t pair_half(int li) { return li < 8 ? 0x01000c0cu : 0x03020c0cu; }
__device__ __forceinline__ float half_of(uint32_t w, uint32_t sel) { return __uint_as_float(__builtin_amdgcn_perm(w, w, sel)); }
template <int D, bool F16>
__device__ __forceinline__ f32x4 pair_scores(const Keys4<D>& n, int h, const u32x4 (&q)[D / 32], uint32_t sel) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D / 64; ++d) {
    f32x4 t = Elem<F16>::mfma(widen8<F16>(n.k[h][2 * d]), q[2 * d], f32x4{0.f, 0.f, 0.f, 0.f});
    t = Elem<F16>::mfma(widen8<F16>(n.k[h][2 * d + 1]), q[2 * d + 1], t);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = fmaf(t[i], half_of(n.s[h][i * (D / 64) + d], sel), s[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    s[i] += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(s[i]), 0x128, 0xf, 0xf, true));  // (lanes 8 on in the row)
  return s;
}

// Host: the cache and the tables of a call, checked, into its arguments.  One of c and c4
// is given; values: whether the call reads them.
inline int take_cache(const char* fn, Window& a, const pgs_kv_cache* c, const pgs_kv_cache4* c4, bool values,
                      const int32_t* tables, int64_t table_stride, int64_t columns, int64_t requests) {
  if (!c == !c4) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: one cache, of 16 or of 4 bits", fn);
  const int64_t blocks = c ? c->blocks : c4->blocks, size = c ? c->block_size : c4->block_size;
  const int64_t heads = c ? c->kv_heads : c4->kv_heads, dim = c ? c->head_dim : c4->head_dim;
  if (dim != 64 && dim != 128) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: head_dim=%lld must be 64 or 128", fn, (long long)dim);
  if (heads < 1 || heads > 4096) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: kv_heads=%lld", fn, (long long)heads);
  if (blocks < 1 || blocks > 0x7fffffff || size < 16 || size > 0x10000 || size % 16 != 0)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: the cache needs blocks of a multiple of 16 tokens (block_size=%lld)", fn,
                (long long)size);
  // (a tile behind the last token still has a 32-bit number)
  if (columns < 0 || table_stride < columns || columns > 0x7fff0000 / size)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: bad block table", fn);
  if (columns > 0 && requests > 0 && !tables) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(tables, 4)) return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  if (c) {
    if (!c->k || (values && !c->v)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
    for (int64_t s : {c->k_block, c->k_slot, c->k_head, values ? c->v_block : 0, values ? c->v_slot : 0, values ? c->v_head : 0})
      if (s < 0 || s % 8 != 0) return fail(PGS_ERR_MISALIGNED, "%s: strides must be multiples of 8 elements", fn);
    // (16 rows' offsets from their first are 32-bit)
    if (c->k_slot > (1 << 26) || (values && c->v_slot > (1 << 26)))
      return fail(PGS_ERR_INVALID_ARGUMENT, "%s: rows are too far apart", fn);
    if (!aligned(c->k, 16) || (values && !aligned(c->v, 16)))
      return fail(PGS_ERR_MISALIGNED, "%s: the cache must be 16-byte aligned", fn);
    a.kc = c->k, a.vc = c->v;
    a.kc_block = c->k_block, a.kc_head = c->k_head, a.vc_block = c->v_block, a.vc_head = c->v_head;
    a.kc_slot = static_cast<uint32_t>(c->k_slot), a.vc_slot = static_cast<uint32_t>(c->v_slot);
  } else {
    if (!c4->k || !c4->k_scale || (values && (!c4->v || !c4->v_scale)))
      return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
    if (!aligned(c4->k, 16) || !aligned(c4->k_scale, 16) || (values && (!aligned(c4->v, 16) || !aligned(c4->v_scale, 16))))
      return fail(PGS_ERR_MISALIGNED, "%s: the cache must be 16-byte aligned", fn);
    a.kc = c4->k, a.vc = c4->v;
    a.ks = static_cast<const uint16_t*>(c4->k_scale), a.vs = static_cast<const uint16_t*>(c4->v_scale);
  }
  a.blocks = static_cast<int32_t>(blocks), a.bs = static_cast<int32_t>(size);
  a.bs_inv = static_cast<uint32_t>(((uint64_t{1} << 32) + a.bs - 1) / a.bs);
  a.tables = tables, a.tstride = table_stride, a.cols = static_cast<int32_t>(columns);
  a.kv_heads = static_cast<int32_t>(heads);
  return PGS_OK;
}

}  // namespace
}  // namespace pgs
