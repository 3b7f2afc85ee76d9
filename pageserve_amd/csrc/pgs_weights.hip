// What attention weights add up to for each cached token, and requests cut to the tokens of
// largest sums (gfx950; pgs_window.h).
//
//   w[slot of j] (+)= sum over the rows and query heads that see j of e^(scale q . k_j - lse)
//
// with the lse that the attention gave: 2^(c s - lse log2(e)), c = scale log2(e).
#include <algorithm>

#include "pgs_window.h"

namespace pgs {
namespace {

struct Weigh {
  Window w;
  float* weights;      // [blocks][block_size]
  const int32_t* fresh;  // [requests], or null: the last tokens whose sums start from 0
  int tiles;           // of kTile tokens: workgroups per request
};
constexpr int kTile = 128, kWaves = kTile / 32;

// A wave's 32 tokens stay in registers as A operands, one key head after the other; the rows
// pass by as B operands, sixteen (token, query head) at a time, and lane l adds up the
// weights of tokens 4 (l/16) + i for row l%16.  Every sum is one wave's: the order of the
// additions is fixed.
template <int D, bool F16, bool FP4>
__global__ __launch_bounds__(64 * kWaves) void weigh_kernel(Weigh g) {
  const Window& a = g.w;
  constexpr int DC = D / 32;
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int b = blockIdx.x / g.tiles;
  const Ragged rq = ragged(a, b);
  const int32_t* table = a.tables + b * a.tstride;
  const int fresh = rq.len - (g.fresh ? min(max(g.fresh[b], 0), rq.len) : 0);  // the first of them
  for (int64_t tile = blockIdx.x % g.tiles; tile * kTile + 32 * wave < rq.len; tile += g.tiles) {
    const int key0 = static_cast<int>(tile) * kTile + 32 * wave;
    // the rows that see some of them
    int t0 = max(0, key0 - rq.first), t1 = rq.tokens;
    if (key0 >= a.sinks) t1 = static_cast<int>(least(t1, static_cast<int64_t>(key0) + 31 + a.window - rq.first));
    if (t0 >= t1 && key0 + 32 <= fresh) continue;
    bool bad[2];
    int64_t blk[2];
    int slot[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // (a half behind the last token reads the other one's block, and is masked)
      const int id = uniform(table[block_of(a, key0 + (key0 + 16 * h < rq.len ? 16 * h : 0), slot[h])]);
      bad[h] = id < 0 || id >= a.blocks;
      blk[h] = bad[h] ? 0 : id;
    }
    float sum[2][4] = {};
    for (int kh = 0; t0 < t1 && kh < a.kv_heads; ++kh) {
      std::conditional_t<FP4, Keys4<D>, Keys16<D>> k;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (FP4) load_keys4<D>(a, row_of(a, blk[h], slot[h], kh), li, lg, k.k[h], k.s[h]);
        else load_keys<D>(a, blk[h], slot[h], kh, li, lg, k.k[h]);
      }
      for (int row0 = t0 * a.group; row0 < t1 * a.group; row0 += 16) {
        const int row = min(row0 + li, t1 * a.group - 1), t = row / a.group, head = kh * a.group + row - t * a.group;
        const uint16_t* p = a.q + (rq.row0 + t) * a.q_row + head * a.q_head + 8 * lg;
        u32x4 q[DC];
#pragma unroll
        for (int d = 0; d < DC; ++d) q[d] = ld16(p + 32 * d);
        const float lse = a.lse[static_cast<int64_t>(rq.row0 + t) * a.q_heads + head] * 1.44269504088896340736f;
        const int pos = rq.first + t, low = low_of(pos, a.window);
        const int first = rq.first + row0 / a.group, last = rq.first + (min(row0 + 16, t1 * a.group) - 1) / a.group;
        const bool masked = row0 + 16 > t1 * a.group || !all_visible(a, key0, key0 + 31, first, last);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 s = scores<D, F16>(k, h, q);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = __builtin_amdgcn_exp2f(fmaf(s[i], a.c, -lse));
            const bool in = !masked || (row0 + li < t1 * a.group && visible(key0 + 16 * h + 4 * lg + i, pos, low, a.sinks));
            sum[h][i] += in ? e : 0.f;
          }
        }
      }
    }
    // over the rows of the lanes: lane 16 lg then has tokens 4 lg + i
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) sum[h][i] += __shfl_xor(sum[h][i], x);
    if (li < 8) {
      const int h = li >> 2, i = li & 3, j = key0 + 16 * h + 4 * lg + i;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = li == e ? sum[e >> 2][e & 3] : s;
      if (j < rq.len && !(h ? bad[1] : bad[0])) {
        float* p = g.weights + (h ? blk[1] : blk[0]) * a.bs + (h ? slot[1] : slot[0]) + 4 * lg + i;
        *p = (j >= fresh ? 0.f : *p) + s;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------

struct Evict {
  float* weights;
  const int32_t *lens, *budget, *tables;
  int64_t tstride;
  int32_t cols, bs, blocks, requests, sinks, recent, most;  // most: tokens of a request at most
  uint32_t bs_inv;
  int32_t* kept;  // [requests]
  int32_t* from;  // [requests][most]: the token that moves to the i-th place
  int32_t* begin;  // [requests]: places before it keep their token
};

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kDigit = 11, kBins = 1 << kDigit;  // three digits: 11 + 11 + 10 bits

// a token's slot; below 0 where its block is absent
__device__ __forceinline__ int64_t slot_of(const Evict& a, const int32_t* table, int token) {
  int at;
  const int id = table[block_of(a, token, at)];
  return id < 0 || id >= a.blocks ? -1 : static_cast<int64_t>(id) * a.bs + at;
}
// A weight's place in the order: larger numbers stay first, a NaN before all, zeros alike, an
// absent token last.
__device__ __forceinline__ uint32_t order_of(const Evict& a, const int32_t* table, int token) {
  const int64_t s = slot_of(a, table, token);
  if (s < 0) return 0;
  const float x = a.weights[s] + 0.f;
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// One workgroup per request.  Of the tokens that may go, the place in the order of the last
// one that stays: its digits from the highest on, from counts of the tokens that agree with
// the digits so far.  Then the places of all that stay, in order, and their weights.
__global__ __launch_bounds__(kSelectThreads) void select_kernel(Evict a) {
  __shared__ int32_t bins[kBins], found[2], lowest;
  __shared__ int32_t count[2][kSelectWaves];
  const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6;
  const int b = blockIdx.x;
  const int64_t room = static_cast<int64_t>(a.cols) * a.bs;
  const int len = static_cast<int>(least(max(a.lens[b], 0), room));
  const int most = max(a.budget[b], 0);
  const int32_t* table = a.tables + b * a.tstride;
  if (len <= most || len > a.most) {
    if (thread == 0) a.kept[b] = len, a.begin[b] = len;
    return;
  }
  const int sinks = min(a.sinks, most), recent = min(a.recent, most - sinks);
  const int first = sinks, end = len - recent;  // those that may go
  int need = most - sinks - recent;             // of them stay
  uint32_t at = 0, mask = 0;                    // digits found
  if (need > 0) {
    for (int shift = 32 - kDigit; shift >= 0; shift = shift == 32 - kDigit ? shift - kDigit : shift - (kDigit - 1)) {
      const int digits = shift == 0 ? kDigit - 1 : kDigit;
      for (int i = thread; i < kBins; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
      for (int j = first + thread; j < end; j += kSelectThreads) {
        const uint32_t o = order_of(a, table, j);
        if ((o & mask) == at) atomicAdd(&bins[o >> shift & ((1u << digits) - 1)], 1);
      }
      __syncthreads();
      // the bin, from the highest on, in which the need is met
      if (wave == 0) {
        const int per = (1 << digits) / 64;
        int mine = 0;
        for (int i = 0; i < per; ++i) mine += bins[(63 - lane) * per + i];
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int o = __shfl_up(upto, d);
          if (lane >= d) upto += o;
        }
        if (upto >= need && upto - mine < need) {
          int left = need - (upto - mine), i = per - 1;
          while (bins[(63 - lane) * per + i] < left) left -= bins[(63 - lane) * per + i--];
          found[0] = (63 - lane) * per + i;
          found[1] = left;
        }
      }
      __syncthreads();
      at |= static_cast<uint32_t>(found[0]) << shift;
      mask |= ((1u << digits) - 1) << shift;
      need = found[1];
    }
  }
  // `need` of the tokens at `at` stay, the first ones, and all that lie above.  A wave counts
  // those of its part of the tokens, then knows where its first one goes.
  const int part = (len + kSelectThreads - 1) / kSelectThreads * 64, lo = min(wave * part, len), hi = min(lo + part, len);
  auto flags = [&](int j, bool& above, bool& equal) {
    above = equal = false;
    if (j >= hi) return;
    if (j < first || j >= end) {
      above = true;
    } else if (mask) {
      const uint32_t o = order_of(a, table, j);
      above = o > at;
      equal = o == at;
    }
  };
  int above_n = 0, equal_n = 0;
  for (int j0 = lo; j0 < hi; j0 += 64) {
    bool above, equal;
    flags(j0 + lane, above, equal);
    above_n += __popcll(__ballot(above));
    equal_n += __popcll(__ballot(equal));
  }
  if (lane == 0) count[0][wave] = above_n, count[1][wave] = equal_n;
  if (thread == 0) lowest = most;
  __syncthreads();
  int above_at = 0, equal_at = 0;  // of the waves before
  for (int w = 0; w < wave; ++w) above_at += count[0][w], equal_at += count[1][w];
  int32_t* from = a.from + static_cast<int64_t>(b) * a.most;
  for (int j0 = lo; j0 < hi; j0 += 64) {
    bool above, equal;
    flags(j0 + lane, above, equal);
    const unsigned long long am = __ballot(above), em = __ballot(equal), before = (1ull << lane) - 1;
    const int e = equal_at + __popcll(em & before), n = above_at + __popcll(am & before) + min(e, need);
    if (above || (equal && e < need)) {
      from[n] = j0 + lane;
      if (n != j0 + lane) atomicMin(&lowest, n);
    }
    above_at += __popcll(am);
    equal_at += __popcll(em);
  }
  __threadfence_block();
  __syncthreads();
  const int begin = lowest;
  if (thread == 0) a.kept[b] = most, a.begin[b] = begin;
  // the weights: a place takes that of a token further on, and is read before that
  for (int i0 = begin; i0 < most; i0 += kSelectThreads) {
    const int i = i0 + thread;
    float x = 0.f;
    int64_t to = -1;
    if (i < most) {
      const int64_t s = slot_of(a, table, from[i]);
      if (s >= 0) to = slot_of(a, table, i), x = a.weights[s];
    }
    __syncthreads();
    if (to >= 0) a.weights[to] = x;
    // (the next turn reads places that no earlier one writes)
  }
}

constexpr int kMoveThreads = 1024, kMaxCaches = 16;
struct MoveCache {
  void *k, *v, *ks, *vs;
  int64_t k_block, k_slot, k_head, v_block, v_slot, v_head;
};
struct Move {
  Evict e;
  int32_t heads, slices, caches;
  MoveCache c[kMaxCaches];
};

// What stays of a request, moved together: one workgroup per (request, cache, keys or values,
// head, slice of the token's pieces).  A place takes a token from further on, so a turn's
// tokens are read before any of its places is written, and the next turn's lie behind them.
// P pieces of type T of a token; piece(base of the block, slot, p): where one is.
template <typename T, int U, typename Where>
__device__ __forceinline__ void move_pieces(const Evict& e, int b, int p0, int pieces, Where where) {
  const int32_t* table = e.tables + b * e.tstride;
  const int32_t* from = e.from + static_cast<int64_t>(b) * e.most;
  const int begin = e.begin[b], kept = e.kept[b];
  const int64_t all = static_cast<int64_t>(kept - begin) * pieces;
  for (int64_t n0 = 0; n0 < all; n0 += U * kMoveThreads) {
    T x[U];
    T* to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * kMoveThreads + threadIdx.x;
      to[u] = nullptr;
      if (n >= all) continue;
      const int i = begin + static_cast<int>(n / pieces), p = p0 + static_cast<int>(n % pieces);
      int s, d;
      const int j = from[i], src = table[block_of(e, j, s)], dst = table[block_of(e, i, d)];
      if (j == i || src < 0 || src >= e.blocks || dst < 0 || dst >= e.blocks) continue;
      x[u] = *where(src, s, p);
      to[u] = where(dst, d, p);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u]) *to[u] = x[u];
  }
}

template <typename T>  // of 16 bytes, or of 2 where something is not aligned to 16
__global__ __launch_bounds__(kMoveThreads) void move_kernel(Move m, int pieces) {
  int u = blockIdx.x;
  const int slice = u % m.slices;
  u /= m.slices;
  const int h = u % m.heads;
  u /= m.heads;
  const bool values = u & 1;
  u >>= 1;
  const MoveCache& c = m.c[u % m.caches];
  const int b = u / m.caches;
  uint16_t* base = static_cast<uint16_t*>(values ? c.v : c.k) + h * (values ? c.v_head : c.k_head);
  const int64_t block = values ? c.v_block : c.k_block, step = values ? c.v_slot : c.k_slot;
  const int p0 = pieces * slice / m.slices, p1 = pieces * (slice + 1) / m.slices;
  move_pieces<T, 4>(m.e, b, p0, p1 - p0, [&](int blk, int slot, int p) {
    return reinterpret_cast<T*>(base + blk * block + slot * step) + p;
  });
}

// 4-bit: codes and scales as whole words of a token's own (values of 64 dims: 2 bytes each)
template <int D>
__global__ __launch_bounds__(kMoveThreads) void move4_kernel(Move m) {
  constexpr int C = D / 32;
  int u = blockIdx.x;
  const int h = u % m.heads;
  u /= m.heads;
  const int part = u & 3;
  u >>= 2;
  const MoveCache& c = m.c[u % m.caches];
  const int b = u / m.caches;
  auto row = [&](int blk, int slot) { return (static_cast<int64_t>(blk) * m.heads + h) * m.e.bs + slot; };
  if (part == 0) {
    typedef std::conditional_t<C == 4, u32x4, u32x2> T;
    move_pieces<T, 4>(m.e, b, 0, 4, [&](int blk, int slot, int p) { return static_cast<T*>(c.k) + row(blk, slot) * 4 + p; });
  } else if (part == 1) {
    typedef std::conditional_t<C == 4, uint32_t, uint16_t> T;
    move_pieces<T, 4>(m.e, b, 0, 16, [&](int blk, int slot, int p) {
      return static_cast<T*>(c.v) + row(blk, slot & ~15) * 16 + (16 * (slot >> 2 & 3) + p) * 4 + (slot & 3);
    });
  } else {
    typedef std::conditional_t<C == 4, u32x2, uint32_t> T;
    T* base = static_cast<T*>(part == 2 ? c.ks : c.vs);
    move_pieces<T, 4>(m.e, b, 0, 1, [&](int blk, int slot, int) { return base + row(blk, slot); });
  }
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" int pgs_accumulate_weights(const pgs_accumulate_weights_args* args, void* stream) {
  const char* fn = "pgs_accumulate_weights";
  if (!args) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null arguments", fn);
  const pgs_accumulate_weights_args& g = *args;
  if (g.dtype != PGS_DTYPE_BF16 && g.dtype != PGS_DTYPE_F16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: dtype %d must be bf16 or fp16", fn, g.dtype);
  Weigh w{};
  Window& a = w.w;
  if (int rc = take_cache(fn, a, g.cache, g.cache4, false, g.block_tables, g.table_stride, g.columns)) return rc;
  const int64_t dim = g.cache ? g.cache->head_dim : g.cache4->head_dim;
  if (g.rows < 0 || g.rows > 0x7fffffff / 64 || g.requests < 0 || g.requests > 0x100000 || g.q_heads < a.kv_heads ||
      g.q_heads % a.kv_heads != 0 || g.q_heads > 4096 || g.max_tokens < 1 || g.max_tokens > 0x7fffffff / 64 ||
      g.max_context < 0 || g.max_context > 0x7fffffff || g.window < 1 || g.window > 0x7fffffff || g.sinks < 0 ||
      g.sinks > 0x7fffffff || std::min(g.max_tokens, std::max<int64_t>(g.rows, 1)) * g.q_heads > 0x3fffffff)
    return fail(PGS_ERR_INVALID_ARGUMENT,
                "%s: rows=%lld requests=%lld q_heads=%lld kv_heads=%d max_tokens=%lld window=%lld sinks=%lld: q_heads is a "
                "multiple of kv_heads, max_tokens and window 1 at least, sinks 0 at least",
                fn, (long long)g.rows, (long long)g.requests, (long long)g.q_heads, a.kv_heads, (long long)g.max_tokens,
                (long long)g.window, (long long)g.sinks);
  for (int64_t s : {g.q_row, g.q_head})
    if (s < 0 || s % 8 != 0) return fail(PGS_ERR_MISALIGNED, "%s: strides must be multiples of 8 elements", fn);
  if (!(g.scale == g.scale)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: scale is NaN", fn);
  if (g.requests == 0) return PGS_OK;
  if (!g.lens || !g.offsets || !g.weights || (g.rows > 0 && (!g.q || !g.lse)))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(g.q, 16) || !aligned(g.lse, 4) || !aligned(g.weights, 4) || !aligned(g.lens, 4) || !aligned(g.offsets, 4) ||
      !aligned(g.new_lens, 4))
    return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  a.q = static_cast<const uint16_t*>(g.q);
  a.lse = const_cast<float*>(g.lse);
  a.q_row = g.q_row, a.q_head = g.q_head;
  a.lens = g.lens, a.offsets = g.offsets;
  a.rows = static_cast<int32_t>(g.rows), a.requests = static_cast<int32_t>(g.requests);
  a.q_heads = static_cast<int32_t>(g.q_heads), a.group = a.q_heads / a.kv_heads;
  a.max_tokens = static_cast<int32_t>(std::min(g.max_tokens, std::max<int64_t>(g.rows, 1)));
  a.window = static_cast<int32_t>(g.window), a.sinks = static_cast<int32_t>(g.sinks);
  a.c = g.scale * 1.44269504088896340736f;
  w.weights = g.weights, w.fresh = g.new_lens;
  // (a request that is longer than max_context takes further turns; grids are 32-bit)
  const int64_t context = std::min(g.max_context, g.columns * a.bs);
  w.tiles = static_cast<int>(std::max<int64_t>(1, std::min((context + kTile - 1) / kTile, 0x3fffffff / g.requests)));
  const dim3 grid(static_cast<unsigned>(g.requests * w.tiles)), block(64 * kWaves);
  auto go = [&](auto d, auto f16) {
    constexpr int D = decltype(d)::value;
    constexpr bool F = decltype(f16)::value;
    if (g.cache) hipLaunchKernelGGL((weigh_kernel<D, F, false>), grid, block, 0, st, w);
    else hipLaunchKernelGGL((weigh_kernel<D, F, true>), grid, block, 0, st, w);
  };
  const bool f16 = g.dtype == PGS_DTYPE_F16;
  if (dim == 64) f16 ? go(Int<64>{}, Int<1>{}) : go(Int<64>{}, Int<0>{});
  else f16 ? go(Int<128>{}, Int<1>{}) : go(Int<128>{}, Int<0>{});
  return check_launch("accumulate_weights kernel");
}

extern "C" size_t pgs_evict_tokens_workspace_bytes(int64_t requests, int64_t max_context) {
  if (requests < 1 || requests > 0x10000 || max_context < 0 || max_context > 0x7fffffff) return 0;
  return static_cast<size_t>(requests * (max_context + 1)) * 4;
}

extern "C" int pgs_evict_tokens(float* weights, const int32_t* lens, const int32_t* budget, const int32_t* block_tables,
                                int64_t table_stride, int64_t columns, int64_t blocks, int64_t block_size, int64_t requests,
                                int64_t sinks, int64_t recent, int64_t max_context, const pgs_kv_cache* caches, int64_t count,
                                const pgs_kv_cache4* caches4, int64_t count4, int32_t* kept, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* fn = "pgs_evict_tokens";
  if (requests < 0 || requests > 0x10000 || sinks < 0 || sinks > 0x7fffffff || recent < 0 || recent > 0x7fffffff ||
      max_context < 0 || max_context > 0x7fffffff || count < 0 || count4 < 0)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: requests=%lld (at most 65536) sinks=%lld recent=%lld max_context=%lld", fn,
                (long long)requests, (long long)sinks, (long long)recent, (long long)max_context);
  if (blocks < 0 || blocks > 0x7fffffff || block_size < 16 || block_size > 0x10000 || block_size % 16 != 0 || columns < 0 ||
      table_stride < columns || columns > 0x7fff0000 / block_size)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: bad block table, or block_size=%lld no multiple of 16", fn, (long long)block_size);
  if ((count > 0 && !caches) || (count4 > 0 && !caches4)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  bool vec = true;
  for (int64_t i = 0; i < count; ++i) {
    const pgs_kv_cache& c = caches[i];
    if (c.blocks != blocks || c.block_size != block_size || c.kv_heads != caches[0].kv_heads ||
        c.head_dim != caches[0].head_dim || c.kv_heads < 1 || c.kv_heads > 4096 || c.head_dim < 1 || c.head_dim > 0x4000)
      return fail(PGS_ERR_INVALID_ARGUMENT, "%s: caches must agree in their sizes, and with the weights in blocks", fn);
    for (int64_t s : {c.k_block, c.k_slot, c.k_head, c.v_block, c.v_slot, c.v_head}) {
      if (s < 0) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
      vec = vec && s % 8 == 0;
    }
    if (blocks > 0 && (!c.k || !c.v)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
    if (!aligned(c.k, 2) || !aligned(c.v, 2)) return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
    vec = vec && c.head_dim % 8 == 0 && aligned(c.k, 16) && aligned(c.v, 16);
  }
  for (int64_t i = 0; i < count4; ++i) {
    const pgs_kv_cache4& c = caches4[i];
    if (c.blocks != blocks || c.block_size != block_size || c.kv_heads != caches4[0].kv_heads ||
        c.head_dim != caches4[0].head_dim || c.kv_heads < 1 || c.kv_heads > 4096 || (c.head_dim != 64 && c.head_dim != 128))
      return fail(PGS_ERR_INVALID_ARGUMENT, "%s: caches must agree in their sizes, and with the weights in blocks", fn);
    if (blocks > 0 && (!c.k || !c.v || !c.k_scale || !c.v_scale)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_scale, 16) || !aligned(c.v_scale, 16))
      return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  }
  for (int64_t heads : {count ? caches[0].kv_heads : 1, count4 ? caches4[0].kv_heads : 1})  // (grids are 32-bit)
    if (requests * heads > 0x7fffffff / (kMaxCaches * 8)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: too many requests", fn);
  if (requests == 0) return PGS_OK;
  if ((blocks > 0 && !weights) || !lens || !budget || !kept || (columns > 0 && !block_tables))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(weights, 4) || !aligned(lens, 4) || !aligned(budget, 4) || !aligned(kept, 4) || !aligned(block_tables, 4))
    return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  const int64_t most = std::min(max_context, columns * block_size);
  if (!workspace || workspace_bytes < static_cast<size_t>(requests * (most + 1)) * 4 || !aligned(workspace, 4))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %zu bytes", fn,
                static_cast<size_t>(requests * (most + 1)) * 4);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  Move m{};
  Evict& e = m.e;
  e.weights = weights, e.lens = lens, e.budget = budget, e.tables = block_tables, e.tstride = table_stride;
  e.cols = static_cast<int32_t>(columns), e.bs = static_cast<int32_t>(block_size), e.blocks = static_cast<int32_t>(blocks);
  e.bs_inv = static_cast<uint32_t>(((uint64_t{1} << 32) + e.bs - 1) / e.bs);
  e.requests = static_cast<int32_t>(requests), e.sinks = static_cast<int32_t>(sinks), e.recent = static_cast<int32_t>(recent);
  e.most = static_cast<int32_t>(most), e.kept = kept;
  e.begin = static_cast<int32_t*>(workspace), e.from = e.begin + requests;
  hipLaunchKernelGGL(select_kernel, dim3(static_cast<unsigned>(requests)), dim3(kSelectThreads), 0, st, e);
  if (int rc = check_launch("evict_tokens kernel")) return rc;
  for (int64_t i0 = 0; i0 < count; i0 += kMaxCaches) {
    m.caches = static_cast<int32_t>(std::min<int64_t>(count - i0, kMaxCaches));
    m.heads = static_cast<int32_t>(caches[0].kv_heads);
    const int pieces = static_cast<int>(vec ? caches[0].head_dim / 8 : caches[0].head_dim);
    for (int i = 0; i < m.caches; ++i) {
      const pgs_kv_cache& c = caches[i0 + i];
      m.c[i] = MoveCache{c.k, c.v, nullptr, nullptr, c.k_block, c.k_slot, c.k_head, c.v_block, c.v_slot, c.v_head};
    }
    m.slices = 1;
    const int64_t units = requests * m.caches * 2 * m.heads;
    while (m.slices < 4 && units * m.slices < 512 && pieces % (2 * m.slices) == 0) m.slices *= 2;
    const dim3 grid(static_cast<unsigned>(units * m.slices));
    if (vec) hipLaunchKernelGGL(move_kernel<u32x4>, grid, dim3(kMoveThreads), 0, st, m, pieces);
    else hipLaunchKernelGGL(move_kernel<uint16_t>, grid, dim3(kMoveThreads), 0, st, m, pieces);
    if (int rc = check_launch("move kernel")) return rc;
  }
  for (int64_t i0 = 0; i0 < count4; i0 += kMaxCaches) {
    m.caches = static_cast<int32_t>(std::min<int64_t>(count4 - i0, kMaxCaches));
    m.heads = static_cast<int32_t>(caches4[0].kv_heads);
    for (int i = 0; i < m.caches; ++i) {
      const pgs_kv_cache4& c = caches4[i0 + i];
      m.c[i] = MoveCache{c.k, c.v, c.k_scale, c.v_scale, 0, 0, 0, 0, 0, 0};
    }
    const dim3 grid(static_cast<unsigned>(requests * m.caches * 4 * m.heads));
    if (caches4[0].head_dim == 64) hipLaunchKernelGGL(move4_kernel<64>, grid, dim3(kMoveThreads), 0, st, m);
    else hipLaunchKernelGGL(move4_kernel<128>, grid, dim3(kMoveThreads), 0, st, m);
    if (int rc = check_launch("move kernel")) return rc;
  }
  return PGS_OK;
}
