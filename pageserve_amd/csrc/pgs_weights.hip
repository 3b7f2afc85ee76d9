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
  float* weights;        // [blocks][block_size]
  const int32_t* fresh;  // [requests], or null: the last tokens whose sums start from 0
  uint32_t group_inv;    // 2^16 / group, rounded up
  int tiles, parts;      // of kTile tokens: workgroups per request; parts of the rows
  float* sums;           // (parts > 1) [requests][columns * block_size][parts]
};
constexpr int kWaves = 4, kTile = 32 * kWaves, kFewRows = 16;

// One workgroup per request, tile of 128 tokens and part of the rows (of all key heads, 32 (token,
// query head) at a time).  A wave's 32 tokens stay in registers as A operands of
// v_mfma_f32_32x32x16, 4-bit ones widened exactly (fp16: below 2^-16 to a multiple of
// 2^-24, which moves a score by 2^-25 sum |q| at most); the rows pass by through LDS as B operands,
// SUB tiles between two barriers (one: a key head has sixteen rows at most), shared by the waves,
// and lane l adds up the weights of tokens 8 b + 4 (l/32) + i for row l%32.  Every sum is one wave's, those
// of the parts are added in order: the order of all additions is fixed.
// Prompts are bound by issue: 512 rows over 4096 tokens and 256 over 8192 in 4 bits (64.5 M scores of
// 128 dims) 38 us, 1.7 T scores a second.  The products of all scores take 13 at a large product's
// rate, the exponentials, at a quarter of the vector units' rate, 8, a multiply-add and an addition a
// score 4; in a wave they follow one another, and only other waves' run beside them.  Single rows
// are bound by reading the keys, behind lengths and block numbers: 16-bit ones go through LDS too, in whole
// lines and a head ahead of the products, 16 requests of 4000 to 8000 tokens (49 MB) in 13.3 us, 3.7
// TB/s (straight into registers, a head after the other, 16).
template <int D, bool F16, bool FP4, int SUB>
__global__ __launch_bounds__(64 * kWaves, 4) void weigh_kernel(Weigh g) {
  const Window& a = g.w;
  typedef typename Elem<F16>::x8 x8;
  constexpr int DC = D / 16, P = D / 8, KI = 64 / P;
  constexpr int QR = SUB == 1 ? kFewRows : 32;             // rows of a tile
  constexpr int J = QR < kWaves * KI ? 1 : QR / kWaves / KI;  // loads of a wave for it (of too many waves some have none)
  constexpr bool STAGED = SUB == 1 && !FP4;                // the keys too go through LDS, a head ahead
  __shared__ __attribute__((aligned(256))) uint16_t lq[2][SUB][QR * D];
  __shared__ __attribute__((aligned(256))) uint16_t lk[STAGED ? kWaves : 1][STAGED ? 32 * D : 8];
  const int lane = threadIdx.x & 63, li = lane & 31, h = lane >> 5;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  // piece p of row r lies at p ^ turn: sixteen rows' pieces meet all banks
  auto turn = [](int r) { return r * P / 16 & (P - 1); };
  const uint32_t q_at = lds_address(lq) + li % QR * (2 * D) + 16 * (h ^ turn(li % QR));
  const int part = blockIdx.x % g.parts, unit = blockIdx.x / g.parts, b = unit / g.tiles;
  const Ragged rq = ragged(a, b);
  const int32_t* table = a.tables + b * a.tstride;
  const int fresh = rq.len - (g.fresh ? min(max(g.fresh[b], 0), rq.len) : 0);  // the first of them
  for (int64_t tile = unit % g.tiles; tile * kTile < rq.len; tile += g.tiles) {
    const int tile0 = static_cast<int>(tile) * kTile, key0 = tile0 + 32 * wave;
    // the tokens whose rows see some of them
    const int ta = max(0, tile0 - rq.first);
    int tb = rq.tokens;
    if (tile0 >= a.sinks) tb = static_cast<int>(least(tb, largest(static_cast<int64_t>(tile0) + kTile - 1 + a.window - rq.first, ta)));
    if (ta >= tb && tile0 + kTile <= fresh) continue;
    // the lane's key (one past the last is the last, and masked)
    int slot;
    const int id = table[block_of(a, min(key0 + li, rq.len - 1), slot)];
    const bool bad = id < 0 || id >= a.blocks;
    const int64_t blk = bad ? 0 : id;
    // the sum that this lane holds in the end: token `in`'s, and what it stood at
    const int e = li & 15, in = 8 * (e >> 2) + 4 * h + (e & 3), j = key0 + in;
    const bool bad_j = __shfl(static_cast<int>(bad), in);
    float* p = g.weights + static_cast<int64_t>(__shfl(static_cast<int>(blk), in)) * a.bs + __shfl(slot, in);
    const float old = g.parts == 1 && li < 16 && j < fresh && !bad_j ? *p : 0.f;
    const int rows = max(tb - ta, 0) * a.group, count = (rows + 32 * SUB - 1) / (32 * SUB);  // of a key head: rows, tiles of them
    const int64_t all = static_cast<int64_t>(count) * a.kv_heads;
    const bool whole = SUB == 1 && g.parts == 1;  // (the divisions cost a step)
    const int n0 = whole ? 0 : static_cast<int>(all * part / g.parts);
    const int n1 = static_cast<int>(whole ? all : all * (part + 1) / g.parts);
    float sum[16] = {};
    u32x4 k[DC];
    // Tiles follow one another: of key head kh from row0 on.  A lane keeps (token, query head of the
    // group) of the rows that it sends and of its own, and goes 32 rows on without a division.
    struct At {
      int t, r;
    };
    const int step_t = 32 / a.group, step_r = 32 - step_t * a.group, next_t = KI / a.group, next_r = KI - next_t * a.group;
    static_assert(J <= 2);
    int kh = SUB > 1 ? n0 / max(count, 1) : n0, row0 = (n0 - kh * count) * (32 * SUB);
    At sent, own;  // (the first of the rows that it sends)
    auto add = [&](At& x, int t, int r) {
      x.t += t, x.r += r;
      const bool over = x.r >= a.group;
      x.t += over, x.r -= over ? a.group : 0;
    };
    auto start = [&] {
      const int t = SUB > 1 ? row0 / a.group : 0, r = row0 - t * a.group;
      auto begin = [&](uint32_t row) {  // (below 32: exact)
        At x;
        x.t = __umul24(row, g.group_inv) >> 16;
        x.r = row - __umul24(x.t, a.group);
        add(x, t, r);
        return x;
      };
      sent = begin(wave * J * KI + lane / P);
      own = begin(li);
    };
    auto on = [&](At& x) { add(x, step_t, step_r); };
    // the tile into a buffer; the lane's rows of it: their lse and where they stand (rows past the
    // last repeat one of the last token's, and see nothing)
    float lse1[SUB];
    int pos1[SUB];
    const int tokens = tb - ta;
    auto send = [&](int to) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        if (row0 + 32 * u < rows) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            At x = sent;
            if (j) add(x, next_t, next_r);
            const int ln = here(lane), r = (wave * J + j) * KI + ln / P, t = min(x.t, tokens - 1);
            const uint16_t* p = a.q + static_cast<int64_t>(rq.row0 + ta + t) * a.q_row + (kh * a.group + x.r) * a.q_head +
                                8 * (ln % P ^ turn(r));
            if (QR >= kWaves * KI || wave < QR / KI)
              load_lds(p, lds_address(lq) + (to * SUB + u) * (QR * 2 * D) + (wave * J + j) * 1024);
          }
          if (SUB > 1) on(sent);
          lse1[u] = a.lse[static_cast<int64_t>(rq.row0 + ta + min(own.t, tokens - 1)) * a.q_heads + kh * a.group + own.r];
          pos1[u] = own.t < tokens ? rq.first + ta + own.t : -1;
          if (SUB > 1) on(own);
        }
      }
    };
    // The wave's keys of head kh into its part of lk: both sixteens whole (one behind the last token
    // is that with the last one again, and masked), piece p of a row at p ^ turn.
    auto fetch = [&] {
#pragma unroll
      for (int n = 0; n < 32 / KI; ++n) {
        const int ln = here(lane), r = n * KI + ln / P, from = n * KI & 16;
        const int64_t block = __builtin_amdgcn_readlane(static_cast<int>(blk), from);
        const int first = __builtin_amdgcn_readlane(slot, from) & ~15;
        const uint16_t* p = static_cast<const uint16_t*>(a.kc) + block * a.kc_block + static_cast<int64_t>(first) * a.kc_slot +
                            kh * a.kc_head + (r & 15) * a.kc_slot + 8 * (ln % P ^ turn(r));
        load_lds(p, lds_address(lk) + wave * (64 * D) + n * 1024);
      }
    };
    if (n0 < n1) {
      if constexpr (STAGED) fetch();
      start();
      send(0);
    }
    int head = -1;
    for (int n = n0; n < n1; ++n) {
      const int buf = (n - n0) & 1, row_a = row0;
      if (kh != head) {
        head = kh;
        if constexpr (FP4) {
          const int64_t at = row_of(a, blk, slot, kh);
          const uint8_t* p = static_cast<const uint8_t*>(a.kc) + at * (D / 2) + h * (D / 8);
          uint32_t w[2][D / 32], s[D / 64];
          load_words(p, w[0]);
          load_words(p + D / 4, w[1]);
          if constexpr (D == 128) load_words(a.ks + at * 4, s);
          else s[0] = *reinterpret_cast<const uint32_t*>(a.ks + at * 2);
#pragma unroll
          for (int d = 0; d < DC; ++d) {
            const float sc = d >> 1 & 1 ? high_bf16(s[d >> 2]) : low_bf16(s[d >> 2]);
            float f[8];
            fp4x8_to_f32(w[d & 1][d >> 1], f);
#pragma unroll
            for (int e = 0; e < 4; ++e) k[d][e] = Elem<F16>::pack(f[2 * e] * sc, f[2 * e + 1] * sc);
          }
        } else if constexpr (!STAGED) {
          const uint16_t* p = static_cast<const uint16_t*>(a.kc) + blk * a.kc_block + static_cast<int64_t>(slot) * a.kc_slot +
                              kh * a.kc_head + 8 * h;
#pragma unroll
          for (int d = 0; d < DC; ++d) k[d] = ld16(p + 16 * d);
        }
      }
      float lse[SUB];
      int pos[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) lse[u] = lse1[u] * 1.44269504088896340736f, pos[u] = pos1[u];
      arrived<0>();
      __syncthreads();  // (the rows are whole; the other buffer's have been read)
      if constexpr (STAGED) {
#pragma unroll
        for (int d = 0; d < DC; ++d)
          k[d] = *lds<const u32x4>((lds_address(lk) + wave * (64 * D) + li * (2 * D) + 16 * (h ^ turn(li))) ^ (32 * d));
#pragma unroll
        for (int d = 0; d < DC; ++d) asm volatile("" : "+v"(k[d]));  // (here: the next head's go there)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      if (n + 1 < n1) {
        row0 += 32 * SUB;
        if (row0 >= rows) {
          row0 = 0, ++kh;
          if (SUB > 1) start();
        }
        if constexpr (STAGED) fetch();
        send(buf ^ 1);
      }
#pragma unroll 1  // (a step's kernel waits for its instructions too)
      for (int u = 0; u < SUB; ++u) {
        const int row = row_a + 32 * u;
        if (row >= rows) break;
        const float lse_u = u ? lse[SUB - 1] : lse[0];
        const int pos_u = u ? pos[SUB - 1] : pos[0];
        f32x16 s{};
#pragma unroll
        for (int d = 0; d < DC; ++d) {
          const x8 q = __builtin_bit_cast(x8, *lds<const u32x4>((q_at ^ (32 * d)) + (buf * SUB + u) * (QR * 2 * D)));
          const x8 kd = __builtin_bit_cast(x8, k[d]);
          if constexpr (F16) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kd, q, s, 0, 0, 0);
          else s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kd, q, s, 0, 0, 0);
        }
        const int first = rq.first + ta + row / a.group, last = rq.first + ta + (min(row + 32, rows) - 1) / a.group;
        if (row + 32 <= rows && all_visible(a, key0, key0 + 31, first, last)) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sum[e] += __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -lse_u));
        } else {
          const uint32_t t = pos_u < 0 ? 0 : visible32(key0, pos_u, low_of(pos_u, a.window), a.sinks) >> (4 * h);
          const uint32_t ok = (t & 0xf) | (t >> 4 & 0xf0) | (t >> 8 & 0xf00) | (t >> 12 & 0xf000);
#pragma unroll
          for (int e = 0; e < 16; ++e) sum[e] += ok >> e & 1 ? __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -lse_u)) : 0.f;
        }
      }
    }
    __syncthreads();  // (the next tile's rows go where these were)
    // Over the rows of the lanes, halving the lanes and the tokens of each: lane l then has that of
    // element l%16 (b = l%16 / 4, i = l%4).
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[e] += __shfl_xor(sum[e], 16);
#pragma unroll
    for (int x = 8; x >= 1; x >>= 1)
#pragma unroll
      for (int e = 0; e < x; ++e) {
        const float mine = li & x ? sum[e + x] : sum[e], other = li & x ? sum[e] : sum[e + x];
        sum[e] = mine + __shfl_xor(other, x);
      }
    if (li < 16 && j < rq.len) {
      if (g.parts > 1) {
        g.sums[(static_cast<int64_t>(b) * a.cols * a.bs + j) * g.parts + part] = sum[0];
      } else if (!bad_j) {
        *p = old + sum[0];
      }
    }
  }
}

// (parts > 1) Behind it: the parts' sums, in order.
__global__ __launch_bounds__(256) void weigh_join_kernel(Weigh g) {
  const Window& a = g.w;
  const int per = (g.tiles * kTile + 255) / 256, b = blockIdx.x / per;
  const Ragged rq = ragged(a, b);
  const int fresh = rq.len - (g.fresh ? min(max(g.fresh[b], 0), rq.len) : 0);
  for (int64_t j = static_cast<int64_t>(blockIdx.x % per) * 256 + threadIdx.x; j < rq.len; j += static_cast<int64_t>(per) * 256) {
    const int tile0 = static_cast<int>(j) / kTile * kTile;
    const int ta = max(0, tile0 - rq.first);
    int tb = rq.tokens;
    if (tile0 >= a.sinks) tb = static_cast<int>(least(tb, largest(static_cast<int64_t>(tile0) + kTile - 1 + a.window - rq.first, ta)));
    if (ta >= tb && tile0 + kTile <= fresh) continue;  // (as above: nothing was left there)
    int slot;
    const int id = a.tables[b * a.tstride + block_of(a, static_cast<int>(j), slot)];
    if (id < 0 || id >= a.blocks) continue;
    const float* p = g.sums + (static_cast<int64_t>(b) * a.cols * a.bs + j) * g.parts;
    float s = 0.f;
    for (int i = 0; i < g.parts; ++i) s += p[i];
    float* w = g.weights + static_cast<int64_t>(id) * a.bs + slot;
    *w = (j >= fresh ? 0.f : *w) + s;
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
constexpr int kHeld = 32768;                      // a request's first tokens whose weights lie in LDS

// a token's slot; below 0 where its block is absent
__device__ __forceinline__ int64_t slot_of(const Evict& a, const int32_t* table, int token) {
  int at;
  const int id = table[block_of(a, token, at)];
  return id < 0 || id >= a.blocks ? -1 : static_cast<int64_t>(id) * a.bs + at;
}
// A token's weight as bits, kAbsent where its block is absent (a NaN of just these bits takes
// another's).
constexpr uint32_t kAbsent = 0xffffffffu;
__device__ __forceinline__ uint32_t weight_of(const Evict& a, const int32_t* table, int token) {
  const int64_t s = slot_of(a, table, token);
  if (s < 0) return kAbsent;
  return min(__float_as_uint(a.weights[s]), kAbsent - 1);
}
// Its place in the order: larger numbers stay first, a NaN before all, zeros alike, an absent
// token last.
__device__ __forceinline__ uint32_t order_of(uint32_t weight) {
  if (weight == kAbsent) return 0;
  const float x = __uint_as_float(weight) + 0.f;
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// One workgroup per request.  Its weights go into LDS (those of tokens from kHeld on are read
// again).  Of the tokens that may go, the place in the order of the last one that stays: its
// digits from the highest on, from counts of the tokens that agree with the digits so far, until
// all of them stay.  Then the places of all that stay, in order, and their weights.  Bound by
// latency (the blocks, the weights, and some ten waits of the workgroup): 8 requests of 6144 to 8192
// tokens 22 us, 4 of 825 to 1100 12.  With the weights read again for each digit they took 50 and 15.
__global__ __launch_bounds__(kSelectThreads) void select_kernel(Evict a) {
  __shared__ uint32_t held[kHeld];
  __shared__ int32_t ids[kHeld / 16];
  __shared__ int32_t bins[kBins], found[3], lowest;
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
  const int mine = min(len, kHeld);
  for (int i = thread; i * a.bs < mine; i += kSelectThreads) ids[i] = table[i];
  __syncthreads();
  for (int j0 = thread; j0 < mine; j0 += 8 * kSelectThreads) {
    uint32_t x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = weight_of(a, ids, min(j0 + u * kSelectThreads, mine - 1));
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (j0 + u * kSelectThreads < mine) held[j0 + u * kSelectThreads] = x[u];
  }
  // four tokens' weights, `step` apart from j on (behind the end: the last one's)
  auto weights4 = [&](int j, int step, int stop, uint32_t (&x)[4]) {
    if (stop <= kHeld) {
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = held[min(j + u * step, stop - 1)];
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = min(j + u * step, stop - 1);
        x[u] = t < kHeld ? held[t] : weight_of(a, table, t);
      }
    }
  };
  __syncthreads();
  const int sinks = min(a.sinks, most), recent = min(a.recent, most - sinks);
  const int first = sinks, end = len - recent;  // those that may go
  int need = most - sinks - recent;             // of them stay
  uint32_t at = 0, mask = 0;                    // digits found
  if (need > 0) {
    for (int shift = 32 - kDigit; shift >= 0; shift = shift == 32 - kDigit ? shift - kDigit : shift - (kDigit - 1)) {
      const int digits = shift == 0 ? kDigit - 1 : kDigit;
      for (int i = thread; i < kBins; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
      for (int j = first + thread; j < end; j += 4 * kSelectThreads) {
        uint32_t x[4];
        weights4(j, kSelectThreads, end, x);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t o = order_of(x[u]);
          if (j + u * kSelectThreads < end && (o & mask) == at) atomicAdd(&bins[o >> shift & ((1u << digits) - 1)], 1);
        }
      }
      __syncthreads();
      // the bin, from the highest on, in which the need is met: two for each thread
      const int top = kBins - 1 - 2 * thread, n0 = bins[top], n1 = bins[top - 1];
      int upto = n0 + n1;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      if (lane == 63) count[0][wave] = upto;
      __syncthreads();
      for (int w = 0; w < wave; ++w) upto += count[0][w];
      if (upto >= need && upto - n0 - n1 < need) {
        const int left = need - (upto - n0 - n1);
        const bool one = left <= n0;
        found[0] = one ? top : top - 1;
        found[1] = one ? left : left - n0;
        found[2] = one ? n0 : n1;
      }
      __syncthreads();
      at |= static_cast<uint32_t>(found[0]) << shift;
      mask |= ((1u << digits) - 1) << shift;
      need = found[1];
      if (need == found[2]) break;
    }
  }
  // `need` of the tokens at `at` stay, the first ones, and all that lie above.  A wave counts
  // those of its part of the tokens, then knows where its first one goes.
  const int part = (len + kSelectThreads - 1) / kSelectThreads * 64, lo = min(wave * part, len), hi = min(lo + part, len);
  auto flags = [&](int j, uint32_t weight, bool& above, bool& equal) {
    above = equal = false;
    if (j >= hi) return;
    if (j < first || j >= end) {
      above = true;
    } else if (mask) {
      const uint32_t o = order_of(weight) & mask;
      above = o > at;
      equal = o == at;
    }
  };
  int above_n = 0, equal_n = 0;
  for (int j0 = lo; j0 < hi; j0 += 256) {
    uint32_t x[4];
    weights4(j0 + lane, 64, hi, x);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bool above, equal;
      flags(j0 + 64 * u + lane, x[u], above, equal);
      above_n += __popcll(__ballot(above));
      equal_n += __popcll(__ballot(equal));
    }
  }
  __syncthreads();  // (the counts of the last digit have been read)
  if (lane == 0) count[0][wave] = above_n, count[1][wave] = equal_n;
  if (thread == 0) lowest = most;
  __syncthreads();
  int above_at = 0, equal_at = 0, low = most;  // of the waves before
  for (int w = 0; w < wave; ++w) above_at += count[0][w], equal_at += count[1][w];
  int32_t* from = a.from + static_cast<int64_t>(b) * a.most;
  for (int j0 = lo; j0 < hi; j0 += 256) {
    uint32_t x[4];
    weights4(j0 + lane, 64, hi, x);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + 64 * u + lane;
      bool above, equal;
      flags(j, x[u], above, equal);
      const unsigned long long am = __ballot(above), em = __ballot(equal), before = (1ull << lane) - 1;
      const int e = equal_at + __popcll(em & before), n = above_at + __popcll(am & before) + min(e, need);
      if (above || (equal && e < need)) {
        from[n] = j;
        if (n != j) {
          low = min(low, n);
          if (n < kHeld && x[u] != kAbsent) {  // (its own weight lies in LDS: nobody reads it any more)
            const int64_t to = slot_of(a, ids, n);
            if (to >= 0) a.weights[to] = __uint_as_float(x[u]);
          }
        }
      }
      above_at += __popcll(am);
      equal_at += __popcll(em);
    }
  }
  if (low < most) atomicMin(&lowest, low);
  __threadfence_block();
  __syncthreads();
  const int begin = lowest;
  if (thread == 0) a.kept[b] = most, a.begin[b] = begin;
  // the other places' weights: each takes that of a token further on, and is read before that
  for (int i0 = max(begin, kHeld); i0 < most; i0 += kSelectThreads) {
    const int i = i0 + thread;
    uint32_t x = kAbsent;
    if (i < most) x = weight_of(a, table, from[i]);
    const int64_t to = x == kAbsent ? -1 : slot_of(a, table, i);
    __syncthreads();
    if (to >= 0) a.weights[to] = __uint_as_float(x);
    // (the next turn reads places that no earlier one writes)
  }
}

constexpr int kMoveThreads = 1024, kMaxCaches = 16;
constexpr int64_t kMoveGroups = 0xffffffff / kMoveThreads;  // of a launch: its threads are fewer than 2^32
struct MoveCache {
  void *k, *v, *ks, *vs;
  int64_t k_block, k_slot, k_head, v_block, v_slot, v_head;
};
struct Move {
  Evict e;
  int32_t heads, slices, caches, first;  // first: request
  MoveCache c[kMaxCaches];
};

// What stays of a request, moved together: one workgroup per (request, cache, keys or values,
// head, slice of the token's pieces).  A place takes a token from further on, so a turn's
// tokens are read before any of its places is written, and while the turn before is written:
// that writes nothing that later turns read.  Bound by memory where there are many workgroups: 8
// requests of 6144 to 8192 tokens cut to 4096, in 4 layers of 2 x 128 dims (267 MB read and written), 70
// us, 3.8 TB/s.  By the turns' latency where there are few: one request of 32000 tokens cut to half, in one
// layer, has 32 (selection and move 107 us; in 4 bits, where a head's codes or scales have one each, 240).
// P pieces of type T of a token; piece(base of the block, slot, p): where one is.
template <typename T, int U, typename Where>
__device__ __forceinline__ void move_pieces(const Evict& e, int b, int p0, int pieces, Where where) {
  const int32_t* table = e.tables + b * e.tstride;
  const int32_t* from = e.from + static_cast<int64_t>(b) * e.most;
  const int begin = e.begin[b], kept = e.kept[b];
  const int64_t all = static_cast<int64_t>(kept - begin) * pieces;
  T x[U], next[U];
  T *to[U], *next_to[U];
  // the places of a turn two turns ahead, their tokens' blocks one ahead
  int token[U], src[U], dst[U], s[U], d[U];
  const int64_t mine = threadIdx.x;
  auto place = [&](int64_t n0, int u) {
    const int64_t n = n0 + u * kMoveThreads + mine;
    return n < all ? begin + static_cast<int>(n / pieces) : -1;
  };
  auto find = [&](int64_t n0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = place(n0, u);
      token[u] = i < 0 ? -1 : from[i];
    }
  };
  auto blocks = [&](int64_t n0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = place(n0, u);
      src[u] = -1;
      if (i < 0 || token[u] == i) continue;
      src[u] = table[block_of(e, token[u], s[u])];
      dst[u] = table[block_of(e, i, d[u])];
    }
  };
  auto load = [&](int64_t n0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      next_to[u] = nullptr;
      if (src[u] < 0 || src[u] >= e.blocks || dst[u] < 0 || dst[u] >= e.blocks) continue;
      const int p = p0 + static_cast<int>((n0 + u * kMoveThreads + mine) % pieces);
      next[u] = *where(src[u], s[u], p);
      next_to[u] = where(dst[u], d[u], p);
    }
  };
  constexpr int64_t N = U * kMoveThreads;
  find(0);
  blocks(0);
  find(N);
  load(0);
  blocks(N);
  find(2 * N);
  for (int64_t n0 = 0; n0 < all; n0 += N) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = next[u], to[u] = next_to[u];
      asm volatile("" : "+v"(x[u]));  // (here: they have arrived before the barrier)
    }
    __syncthreads();
    load(n0 + N);
    blocks(n0 + 2 * N);
    find(n0 + 3 * N);
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
  const int b = m.first + u / m.caches;
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
  const int b = m.first + u / m.caches;
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

namespace pgs {
namespace {
// Workgroups per request, and the parts that the rows are cut into while there are too few
// workgroups for all CUs: of 128 rows at least in a request of the batch's average.  (Not by
// max_tokens: the order of the additions, and so the last bits, are the same for any that is
// large enough.  A long prompt among single tokens gets no parts: 2048 rows beside 31 single ones, of 8000
// tokens each, take 819 us, in calls of their own 112 and 24.)
struct WeighPlan {
  int64_t tiles, parts;
};
constexpr int64_t kSums = int64_t{1} << 26;
WeighPlan weigh_plan(const pgs_accumulate_weights_args& g, int64_t block_size) {
  const int64_t context = std::min(g.max_context, g.columns * block_size);
  WeighPlan p;
  // (a request that is longer than its tiles takes further turns; a launch has fewer than 2^32 threads)
  constexpr int64_t most = 0xffffffff / (64 * kWaves);
  p.tiles = std::max<int64_t>(1, std::min((context + kTile - 1) / kTile, most / std::max<int64_t>(g.requests, 1)));
  const int64_t rows = g.rows * g.q_heads / std::max<int64_t>(g.requests, 1);
  // (and their sums, one for each token that the tables have room for, take kSums bytes at most)
  const int64_t each = std::max<int64_t>(1, g.requests * g.columns * block_size * 4);
  p.parts = std::max<int64_t>(1, std::min({1024 / (p.tiles * std::max<int64_t>(g.requests, 1)), rows / 128, kSums / each, int64_t{64}}));
  return p;
}
bool weigh_sizes_ok(const pgs_accumulate_weights_args& g, int64_t kv_heads) {
  return g.rows >= 0 && g.rows <= 0x7fffffff / 64 && g.requests >= 0 && g.requests <= 0x100000 && g.q_heads >= kv_heads &&
         kv_heads >= 1 && g.q_heads % kv_heads == 0 && g.q_heads <= 4096 && g.max_tokens >= 1 &&
         g.max_tokens <= 0x7fffffff / 64 && g.max_context >= 0 && g.max_context <= 0x7fffffff && g.window >= 1 &&
         g.window <= 0x7fffffff && g.sinks >= 0 && g.sinks <= 0x7fffffff &&
         std::min(g.max_tokens, std::max<int64_t>(g.rows, 1)) * g.q_heads <= 0x3fffffff;
}
size_t weigh_bytes(const pgs_accumulate_weights_args& g, const WeighPlan& p, int64_t block_size) {
  return p.parts == 1 ? 0 : static_cast<size_t>(g.requests * g.columns * block_size * p.parts) * 4;
}
}  // namespace
}  // namespace pgs

extern "C" size_t pgs_accumulate_weights_workspace_bytes(const pgs_accumulate_weights_args* args) {
  if (!args || !args->cache == !args->cache4) return 0;
  const pgs_accumulate_weights_args& g = *args;
  const int64_t size = g.cache ? g.cache->block_size : g.cache4->block_size;
  if (!weigh_sizes_ok(g, g.cache ? g.cache->kv_heads : g.cache4->kv_heads) || size < 16 || size > 0x10000 || g.columns < 0 ||
      g.columns > 0x7fff0000 / size || g.requests == 0)
    return 0;
  return weigh_bytes(g, weigh_plan(g, size), size);
}

extern "C" int pgs_accumulate_weights(const pgs_accumulate_weights_args* args, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const char* fn = "pgs_accumulate_weights";
  if (!args) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null arguments", fn);
  const pgs_accumulate_weights_args& g = *args;
  if (g.dtype != PGS_DTYPE_BF16 && g.dtype != PGS_DTYPE_F16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: dtype %d must be bf16 or fp16", fn, g.dtype);
  Weigh w{};
  Window& a = w.w;
  if (int rc = take_cache(fn, a, g.cache, g.cache4, false, g.block_tables, g.table_stride, g.columns, g.requests))
    return rc;
  const int64_t dim = g.cache ? g.cache->head_dim : g.cache4->head_dim;
  if (!weigh_sizes_ok(g, a.kv_heads))
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
  const WeighPlan p = weigh_plan(g, a.bs);
  const size_t need = weigh_bytes(g, p, a.bs);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 4)))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %zu bytes", fn, need);
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
  w.group_inv = (65536u + a.group - 1) / a.group;
  w.tiles = static_cast<int>(p.tiles), w.parts = static_cast<int>(p.parts);
  w.sums = static_cast<float*>(workspace);
  const dim3 grid(static_cast<unsigned>(g.requests * p.tiles * p.parts)), block(64 * kWaves);
  auto go = [&](auto d, auto f16) {
    constexpr int D = decltype(d)::value;
    constexpr bool F = decltype(f16)::value;
    const bool one = static_cast<int64_t>(a.max_tokens) * a.group <= kFewRows;
    if (g.cache) {
      if (one) hipLaunchKernelGGL((weigh_kernel<D, F, false, 1>), grid, block, 0, st, w);
      else hipLaunchKernelGGL((weigh_kernel<D, F, false, 2>), grid, block, 0, st, w);
    } else {
      if (one) hipLaunchKernelGGL((weigh_kernel<D, F, true, 1>), grid, block, 0, st, w);
      else hipLaunchKernelGGL((weigh_kernel<D, F, true, 2>), grid, block, 0, st, w);
    }
  };
  const bool f16 = g.dtype == PGS_DTYPE_F16;
  if (dim == 64) f16 ? go(Int<64>{}, Int<1>{}) : go(Int<64>{}, Int<0>{});
  else f16 ? go(Int<128>{}, Int<1>{}) : go(Int<128>{}, Int<0>{});
  if (int rc = check_launch("accumulate_weights kernel")) return rc;
  if (p.parts == 1) return PGS_OK;
  const int64_t per = (p.tiles * kTile + 255) / 256;
  hipLaunchKernelGGL(weigh_join_kernel, dim3(static_cast<unsigned>(g.requests * per)), dim3(256), 0, st, w);
  return check_launch("accumulate_weights join kernel");
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
  for (int64_t heads : {count ? caches[0].kv_heads : 1, count4 ? caches4[0].kv_heads : 1})
    if (requests * heads > 0x1000000)
      return fail(PGS_ERR_INVALID_ARGUMENT, "%s: requests=%lld x kv_heads=%lld is above 2^24", fn, (long long)requests, (long long)heads);
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
  // Caches and requests of a launch, `units` workgroups each.
  auto launches = [&](int64_t caches_left, int64_t units, auto launch) {
    m.caches = static_cast<int32_t>(std::min({caches_left, int64_t{kMaxCaches}, kMoveGroups / units}));
    const int64_t most_requests = kMoveGroups / (units * m.caches);
    int rc = PGS_OK;
    for (int64_t r = 0; r < requests && rc == PGS_OK; r += most_requests) {
      m.first = static_cast<int32_t>(r);
      launch(dim3(static_cast<unsigned>(std::min(requests - r, most_requests) * m.caches * units)));
      rc = check_launch("move kernel");
    }
    return rc;
  };
  for (int64_t i0 = 0; i0 < count; i0 += m.caches) {
    m.heads = static_cast<int32_t>(caches[0].kv_heads);
    const int pieces = static_cast<int>(vec ? caches[0].head_dim / 8 : caches[0].head_dim);
    const int64_t left = std::min<int64_t>(count - i0, kMaxCaches);
    for (int64_t i = 0; i < left; ++i) {
      const pgs_kv_cache& c = caches[i0 + i];
      m.c[i] = MoveCache{c.k, c.v, nullptr, nullptr, c.k_block, c.k_slot, c.k_head, c.v_block, c.v_slot, c.v_head};
    }
    // (a slice has whole lines of 128 bytes: of 64 the move of 8 requests above, 70 us, takes 134)
    m.slices = std::max(1, static_cast<int>(pieces * (vec ? 16 : 2)) / 128);
    while (pieces % m.slices) --m.slices;
    while (requests * left * 2 * m.heads * m.slices < 128 && pieces % (2 * m.slices) == 0 && pieces / m.slices > 2) m.slices *= 2;
    // (2 x 4096 heads x 256 slices at most: one cache of one request always fits)
    if (int rc = launches(left, int64_t{2} * m.heads * m.slices, [&](dim3 grid) {
          if (vec) hipLaunchKernelGGL(move_kernel<u32x4>, grid, dim3(kMoveThreads), 0, st, m, pieces);
          else hipLaunchKernelGGL(move_kernel<uint16_t>, grid, dim3(kMoveThreads), 0, st, m, pieces);
        }))
      return rc;
  }
  for (int64_t i0 = 0; i0 < count4; i0 += m.caches) {
    m.heads = static_cast<int32_t>(caches4[0].kv_heads);
    const int64_t left = std::min<int64_t>(count4 - i0, kMaxCaches);
    for (int64_t i = 0; i < left; ++i) {
      const pgs_kv_cache4& c = caches4[i0 + i];
      m.c[i] = MoveCache{c.k, c.v, c.k_scale, c.v_scale, 0, 0, 0, 0, 0, 0};
    }
    if (int rc = launches(left, int64_t{4} * m.heads, [&](dim3 grid) {
          if (caches4[0].head_dim == 64) hipLaunchKernelGGL(move4_kernel<64>, grid, dim3(kMoveThreads), 0, st, m);
          else hipLaunchKernelGGL(move4_kernel<128>, grid, dim3(kMoveThreads), 0, st, m);
        }))
      return rc;
  }
  return PGS_OK;
}
