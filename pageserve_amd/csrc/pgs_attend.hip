// Attention of drafted tokens (trees of at most 64 per request) over a paged cache
// (gfx950).  For row (t, h) of request b, over the cached tokens j < len_b and the
// drafted tokens j that are t or its ancestors:
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c s_j - m),  s_j = q . k_j,  c = scale log2(e)
//
// in one pass with a running maximum m and sum.
//
// One wave computes 16 R rows (the T tokens x G query heads of one key head) against
// 32 keys a step, with v_mfma_f32_16x16x32, keys as A and rows as B in both products,
// so that everything of one row -- scores, maximum, sum, output -- lies in the lanes
// l%16 = row and no transpose crosses lanes:
//
//   S^T [key][row]: A = K (lane l: key l%16, 8 dims from 8 (l/16) of each 32),
//                   B = Q^T; lane l then holds keys 4 (l/16) .. +3 of row l%16.
//   O^T [dim][row]: B = P^T: the lane's own eight scores of the two 16-key halves,
//                   i.e. MFMA index 8 (l/16) + e is key 4 (l/16) + e of the first
//                   half, or 4 (l/16) + e - 4 of the second; A = V^T with the same
//                   numbering: lane l loads D/16 dims (from (l%16) D/16) of its eight
//                   keys, whole 256-byte rows per 16 lanes, and transposes the 8 x
//                   D/16 piece in its registers; MFMA i covers the dims
//                   (l%16) D/16 + i.
//
// The row sums come from one more MFMA per step with ones as A, i.e. they add the
// rounded p that the output uses.  Keys and values go from memory straight to
// registers.  block_size is a multiple of 16, so a 16-key half lies in one block: its
// address is wave-uniform.
//
// Work: (request, key head, row group, part of the keys).  A workgroup's four waves
// are WR row tiles x 4/WR key slices, joined in LDS; parts are joined by a second
// kernel from fp32 partial outputs in the workspace.
#include <math.h>

#include "pgs_fp4.h"

namespace pgs {
namespace {

constexpr int kWaves = 4;
constexpr int kMaxTree = 64;

struct Attend {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  const uint16_t *kc, *vc;
  int64_t kc_block, kc_head, vc_block, vc_head;
  uint32_t kc_slot, vc_slot;
  int32_t blocks, bs;
  const int32_t* tables;
  int64_t tstride;
  int32_t cols;
  const int32_t *lens, *offsets, *parents;
  int32_t rows, requests, q_heads, kv_heads, group;  // group: q_heads / kv_heads
  int32_t max_tokens, row_groups, splits;
  float c;       // scale * log2(e)
  float* part;   // [rows * q_heads][splits][D] (splits > 1)
  float* stat;   // [rows * q_heads][splits][2]: m, l
};

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
    return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
  }
  static __device__ __forceinline__ float low(uint32_t v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v)));
  }
  static constexpr uint32_t kOnes = 0x3c003c00u, kExp = 0x7c00u;
};

// the maximum over lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// The request of a unit and its sizes, each brought into range: whatever the device
// arrays hold, no access leaves the tensors.
struct Request {
  int row0, tokens, len, len_tiles, tree_tiles;
};
__device__ __forceinline__ Request request(const Attend& a, int b) {
  Request r;
  const int lo = min(max(a.offsets[b], 0), a.rows);
  const int hi = min(max(a.offsets[b + 1], lo), a.rows);
  r.row0 = lo;
  r.tokens = min(hi - lo, a.max_tokens);
  const int64_t most = static_cast<int64_t>(a.cols) * a.bs;
  r.len = static_cast<int>(min<int64_t>(max(a.lens[b], 0), most));
  r.len_tiles = (r.len + 31) >> 5;
  r.tree_tiles = (r.tokens + 31) >> 5;
  return r;
}

template <int D, int R, int WR, bool F16>
__global__ __launch_bounds__(64 * kWaves) void attend_kernel(Attend a) {
  using E = Elem<F16>;
  constexpr int WK = kWaves / WR;  // key slices
  constexpr int DC = D / 32;       // 32-dim chunks of a key
  constexpr int DV = D / 16;       // dims of a value row per lane
  constexpr int VW = DV / 2;       // their dwords
  const int lane = threadIdx.x & 63;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int li = lane & 15, lg = lane >> 4;
  const int wr = wave % WR, wk = wave / WR;

  // unit: ((request, key head), part, row group); the row groups of one part are
  // neighbours on one XCD, whose L2 then holds the part's keys
  int unit = xcd_remap(blockIdx.x, gridDim.x);
  const int rg = unit % a.row_groups;
  unit /= a.row_groups;
  const int part = unit % a.splits;
  unit /= a.splits;
  const int kh = unit % a.kv_heads, b = unit / a.kv_heads;
  const Request rq = request(a, b);
  const int nrows = rq.tokens * a.group;
  const int wg_row0 = rg * (16 * R * WR);
  if (wg_row0 >= nrows) return;
  const int row0 = wg_row0 + wr * (16 * R);  // of this wave

  // the steps of this part: [t0, t1) of len_tiles + tree_tiles
  const int tiles = rq.len_tiles + rq.tree_tiles;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * part / a.splits);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / a.splits);

  // rows of this lane, one per R: token tk, head hd (rows past the last repeat it)
  int tk[R];
  u32x4 qf[R][DC];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = min(row0 + 16 * r + li, nrows - 1);
    tk[r] = row / a.group;
    const uint16_t* p = a.q + (rq.row0 + tk[r]) * a.q_row + (kh * a.group + row - tk[r] * a.group) * a.q_head + 8 * lg;
#pragma unroll
    for (int d = 0; d < DC; ++d) qf[r][d] = ld16(p + 32 * d);
  }

  // ancestors of each row's token as a bit mask over the request's drafted tokens:
  // lane t starts with bit t and its parent; each step adds the parent's mask and
  // takes the parent's parent, which doubles the distance covered
  unsigned long long sees[R];
  if (t1 > rq.len_tiles) {
    unsigned long long m = 1ull << lane;
    int par = -1;
    if (lane < rq.tokens) par = a.parents ? a.parents[rq.row0 + lane] : lane - 1;
    if (par >= lane || par < 0) par = -1;
    while (__ballot(par >= 0)) {
      const unsigned long long pm = __shfl(m, par & 63);
      const int pp = __shfl(par, par & 63);
      if (par >= 0) {
        m |= pm;
        par = pp;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) sees[r] = __shfl(m, tk[r]);
  }

  f32x4 o[R][DV], l[R];
  float mx[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mx[r] = -INFINITY;
    l[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DV; ++i) o[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* table = a.tables + b * a.tstride;
  const u32x4 ones = {E::kOnes, E::kOnes, E::kOnes, E::kOnes};

  for (int t = t0 + wk; t < t1; t += WK) {
    const bool tree = t >= rq.len_tiles;
    const int key0 = (tree ? t - rq.len_tiles : t) * 32;
    const int limit = (tree ? rq.tokens : rq.len);  // keys of this kind
    // each 16-key half: a uniform base and the last key of it that exists (a key
    // past the end reads that one instead and is masked)
    const uint16_t *kb[2], *vb[2];
    int last[2];
    bool bad[2];
    uint32_t ks, vs;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int first = min(key0 + 16 * h, limit - 1);
      if (tree) {
        kb[h] = a.k + (rq.row0 + first) * a.k_row + kh * a.k_head;
        vb[h] = a.v + (rq.row0 + first) * a.v_row + kh * a.v_head;
        bad[h] = false;
      } else {
        const int blk = first / a.bs;
        const int id = table[blk];
        bad[h] = id < 0 || id >= a.blocks;
        const int64_t at = bad[h] ? 0 : id, slot = first - blk * a.bs;
        kb[h] = a.kc + at * a.kc_block + slot * a.kc_slot + kh * a.kc_head;
        vb[h] = a.vc + at * a.vc_block + slot * a.vc_slot + kh * a.vc_head;
      }
      last[h] = limit - 1 - first;
    }
    ks = tree ? static_cast<uint32_t>(a.k_row) : a.kc_slot;
    vs = tree ? static_cast<uint32_t>(a.v_row) : a.vc_slot;

    u32x4 kf[2][DC];
    uint32_t vf[8][VW];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t* p = kb[h] + static_cast<uint32_t>(min(li, last[h])) * ks + 8 * lg;
#pragma unroll
      for (int d = 0; d < DC; ++d) kf[h][d] = ld16(p + 32 * d);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int h = e >> 2;
      const uint16_t* p = vb[h] + static_cast<uint32_t>(min(4 * lg + (e & 3), last[h])) * vs + DV * li;
      if constexpr (VW == 4) {
        const u32x4 x = ld16(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) vf[e][i] = x[i];
      } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
        for (int i = 0; i < 2; ++i) vf[e][i] = x[i];
      }
    }

    // scores: lane's keys key0 + 16 h + 4 lg + i
    f32x4 s[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[r][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DC; ++d) s[r][h] = E::mfma(kf[h][d], qf[r][d], s[r][h]);
      }
    const bool masked = tree || key0 + 32 > limit || bad[0] || bad[1];
    // values that no row may take must not meet p = 0 as an infinity or NaN: those
    // past the end and of absent blocks become zeros, and a drafted token's that
    // are not finite are left out of the products (bit of `odd`) and added below
    // for the rows that see it
    uint32_t odd = 0;
    if (masked) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool gone = key0 + 16 * (e >> 2) + 4 * lg + (e & 3) >= limit || bad[e >> 2];
        bool wild = false;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          if (gone) vf[e][i] = 0;
          wild = wild || (vf[e][i] & E::kExp) == E::kExp || (vf[e][i] & E::kExp << 16) == E::kExp << 16;
        }
        const unsigned long long w = tree ? __ballot(wild) : 0;
        if (w) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (w >> (16 * g) & 0xffff) odd |= 1u << (16 * (e >> 2) + 4 * g + (e & 3));
          if (w >> (16 * lg) & 0xffff)
#pragma unroll
            for (int i = 0; i < VW; ++i) vf[e][i] = 0;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (masked) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * h + 4 * lg + i;
            const bool ok = key < limit && !bad[h] && (!tree || ((sees[r] >> (key & 63)) & 1));
            s[r][h][i] = ok ? s[r][h][i] * a.c : -INFINITY;
          }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][h][i] *= a.c;
      }
      float top = s[r][0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, s[r][i >> 2][i & 3]);
      top = fmaxf(mx[r], quad_max(top));
      const float ref = top == -INFINITY ? 0.f : top;  // (nothing seen yet: every p is 0)
      const float f = __builtin_amdgcn_exp2f(mx[r] - ref);
      mx[r] = top;
#pragma unroll
      for (int i = 0; i < 4; ++i) l[r][i] *= f;
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[r][d][i] *= f;
      u32x4 p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(s[r][i >> 1][2 * (i & 1)] - ref);
        const float p1 = __builtin_amdgcn_exp2f(s[r][i >> 1][2 * (i & 1) + 1] - ref);
        p[i] = E::pack(p0, p1);
      }
      l[r] = E::mfma(ones, p, l[r]);
#pragma unroll
      for (int d = 0; d < DV; ++d) {
        u32x4 vt;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          vt[e] = __builtin_amdgcn_perm(vf[2 * e + 1][d >> 1], vf[2 * e][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
        o[r][d] = E::mfma(vt, p, o[r][d]);
      }
      for (uint32_t w = odd; w; w &= w - 1) {
        const int j = __builtin_ctz(w);
        const uint32_t lo = j & 2 ? p[1] : p[0], hi = j & 2 ? p[3] : p[2];
        const float pj = E::low(__shfl(j & 16 ? hi : lo, 16 * (j >> 2 & 3) + li) >> (16 * (j & 1)));
        if (!(sees[r] >> ((key0 + j) & 63) & 1)) continue;
        const uint16_t* x = (j & 16 ? vb[1] : vb[0]) + static_cast<uint32_t>(j & 15) * vs + 4 * lg * DV;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < DV; ++d) o[r][d][i] += pj * E::low(x[i * DV + d]);
      }
    }
  }

  // join the key slices: slice 0 adds the others' sums, brought to one maximum
  if constexpr (WK > 1) {
    __shared__ float lo_[(WK - 1) * WR][R][DV * 4][64];
    __shared__ float ls_[(WK - 1) * WR][R][2][64];
    if (wk > 0) {
      const int w = (wk - 1) * WR + wr;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ls_[w][r][0][lane] = mx[r];
        ls_[w][r][1][lane] = l[r][0];
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) lo_[w][r][4 * d + i][lane] = o[r][d][i];
      }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = mx[r];
#pragma unroll
      for (int s = 0; s < WK - 1; ++s) top = fmaxf(top, ls_[s * WR + wr][r][0][lane]);
      const float ref = top == -INFINITY ? 0.f : top;
      const float f = __builtin_amdgcn_exp2f(mx[r] - ref);
      mx[r] = top;
      l[r][0] *= f;
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[r][d][i] *= f;
#pragma unroll
      for (int s = 0; s < WK - 1; ++s) {
        const int w = s * WR + wr;
        const float g = __builtin_amdgcn_exp2f(ls_[w][r][0][lane] - ref);
        l[r][0] += g * ls_[w][r][1][lane];
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[r][d][i] += g * lo_[w][r][4 * d + i][lane];
      }
    }
  }

  // lane: row li, dims (4 lg + i) DV + d
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + 16 * r + li;
    if (row >= nrows) continue;
    const int head = kh * a.group + row - tk[r] * a.group;
    const int64_t token = rq.row0 + tk[r];
    if (a.splits == 1) {
      const float inv = l[r][0] > 0.f ? 1.f / l[r][0] : l[r][0] == 0.f ? 0.f : NAN;
      uint16_t* p = a.out + token * a.out_row + head * a.out_head + 4 * lg * DV;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[VW];
#pragma unroll
        for (int d = 0; d < VW; ++d) w[d] = E::pack(o[r][2 * d][i] * inv, o[r][2 * d + 1][i] * inv);
        if constexpr (VW == 4) *reinterpret_cast<u32x4*>(p + i * DV) = u32x4{w[0], w[1], w[2], w[3]};
        else *reinterpret_cast<u32x2*>(p + i * DV) = u32x2{w[0], w[1]};
      }
    } else {
      const int64_t at = (token * a.q_heads + head) * a.splits + part;
      float* p = a.part + at * D + 4 * lg * DV;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < DV; d += 4)
          *reinterpret_cast<f32x4*>(p + i * DV + d) = f32x4{o[r][d][i], o[r][d + 1][i], o[r][d + 2][i], o[r][d + 3][i]};
      if (lg == 0) {
        a.stat[2 * at] = mx[r];
        a.stat[2 * at + 1] = l[r][0];
      }
    }
  }
}

// One wave per (request, token, head): the parts' outputs brought to one maximum,
// added and divided by the joined sum.  Lane l owns D/64 neighbouring dims.
template <int D, bool F16>
__global__ __launch_bounds__(256) void join_kernel(Attend a) {
  constexpr int W = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + uniform(static_cast<int>(threadIdx.x >> 6));
  const int head = static_cast<int>(u % a.q_heads);
  const int64_t bt = u / a.q_heads;
  const int b = static_cast<int>(bt / a.max_tokens), t = static_cast<int>(bt % a.max_tokens);
  if (b >= a.requests) return;
  const Request rq = request(a, b);
  if (t >= rq.tokens) return;
  const int64_t token = rq.row0 + t;
  const int64_t at = (token * a.q_heads + head) * a.splits;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, a.stat[2 * (at + s)]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, o[W];
#pragma unroll
  for (int i = 0; i < W; ++i) o[i] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f(a.stat[2 * (at + s)] - ref);
    sum += f * a.stat[2 * (at + s) + 1];
    const float* p = a.part + (at + s) * D + W * lane;
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] += f * p[i];
  }
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
  uint16_t* p = a.out + token * a.out_row + head * a.out_head + W * lane;
  if constexpr (W == 2) {
    *reinterpret_cast<uint32_t*>(p) = Elem<F16>::pack(o[0] * inv, o[1] * inv);
  } else {
    *p = static_cast<uint16_t>(Elem<F16>::pack(o[0] * inv, 0.f));
  }
}

// The launch shape, a function of sizes the host knows (never of what the device
// arrays hold, so that a captured call replays with other lengths).
struct Plan {
  int r, wr, row_groups, splits;
};
Plan plan(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t max_tokens, int64_t max_context) {
  const int64_t rows = max_tokens * (q_heads / kv_heads);
  Plan p;
  p.r = rows <= 16 ? 1 : 2;
  p.wr = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.row_groups = static_cast<int>((rows + 16 * p.r * p.wr - 1) / (16 * p.r * p.wr));
  const int64_t units = requests * kv_heads * p.row_groups;
  const int64_t steps = (max_context + 31) / 32 + (max_tokens + 31) / 32;
  const int64_t most = steps / (4 * (kWaves / p.wr));  // at least four steps for each slice
  int64_t s = (1024 + units - 1) / units;
  s = s < most ? s : most;
  p.splits = static_cast<int>(s < 1 ? 1 : s > 256 ? 256 : s);
  return p;
}

size_t workspace_bytes(const Plan& p, int64_t rows, int64_t q_heads, int64_t head_dim) {
  return p.splits == 1 ? 0 : static_cast<size_t>(rows * q_heads * p.splits) * (head_dim + 2) * 4;
}

bool sizes_ok(int64_t rows, int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens,
              int64_t max_context) {
  return rows >= 0 && rows <= 0x7fffffff / 64 && requests >= 0 && requests <= 0x100000 && kv_heads >= 1 &&
         q_heads >= kv_heads && q_heads % kv_heads == 0 && q_heads <= 4096 && (head_dim == 64 || head_dim == 128) &&
         max_tokens >= 1 && max_tokens <= kMaxTree && max_context >= 0 && max_context <= 0x7fffffff;
}

template <int D, bool F16>
int launch(const Attend& a, const Plan& p, hipStream_t st) {
  const int64_t grid = static_cast<int64_t>(a.requests) * a.kv_heads * p.row_groups * p.splits;
  if (grid > 0x7fffffff || static_cast<int64_t>(a.requests) * a.max_tokens * a.q_heads > 0x7fffffff) return fail(PGS_ERR_INVALID_ARGUMENT, "pgs_tree_attention: too many requests");
  const dim3 g(static_cast<unsigned>(grid)), blk(64 * kWaves);
  if (p.r == 1) hipLaunchKernelGGL((attend_kernel<D, 1, 1, F16>), g, blk, 0, st, a);
  else if (p.wr == 1) hipLaunchKernelGGL((attend_kernel<D, 2, 1, F16>), g, blk, 0, st, a);
  else if (p.wr == 2) hipLaunchKernelGGL((attend_kernel<D, 2, 2, F16>), g, blk, 0, st, a);
  else hipLaunchKernelGGL((attend_kernel<D, 2, 4, F16>), g, blk, 0, st, a);
  if (int rc = check_launch("tree attention kernel")) return rc;
  if (p.splits == 1) return PGS_OK;
  const int64_t waves = static_cast<int64_t>(a.requests) * a.max_tokens * a.q_heads;
  hipLaunchKernelGGL((join_kernel<D, F16>), dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0, st, a);
  return check_launch("tree attention join kernel");
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" size_t pgs_tree_attention_workspace_bytes(int64_t rows, int64_t requests, int64_t q_heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_tokens, int64_t max_context) {
  if (!sizes_ok(rows, requests, q_heads, kv_heads, head_dim, max_tokens, max_context) || rows == 0 || requests == 0)
    return 0;
  return workspace_bytes(plan(requests, q_heads, kv_heads, max_tokens, max_context), rows, q_heads, head_dim);
}

extern "C" int pgs_tree_attention(const pgs_tree_attention_args* args, void* workspace, size_t workspace_bytes_given,
                                  void* stream) {
  const char* fn = "pgs_tree_attention";
  if (!args || !args->cache) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null arguments or cache", fn);
  const pgs_tree_attention_args& g = *args;
  const pgs_kv_cache& c = *g.cache;
  if (g.dtype != PGS_DTYPE_BF16 && g.dtype != PGS_DTYPE_F16)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: dtype %d must be bf16 or fp16", fn, g.dtype);
  if (!sizes_ok(g.rows, g.requests, g.q_heads, c.kv_heads, c.head_dim, g.max_tokens, g.max_context))
    return fail(PGS_ERR_INVALID_ARGUMENT,
                "%s: rows=%lld requests=%lld q_heads=%lld kv_heads=%lld head_dim=%lld max_tokens=%lld: head_dim is 64 or "
                "128, max_tokens 1..%d, q_heads a multiple of kv_heads",
                fn, (long long)g.rows, (long long)g.requests, (long long)g.q_heads, (long long)c.kv_heads,
                (long long)c.head_dim, (long long)g.max_tokens, kMaxTree);
  if (c.blocks < 1 || c.blocks > 0x7fffffff || c.block_size < 16 || c.block_size > 0x10000 || c.block_size % 16 != 0)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: the cache needs blocks of a multiple of 16 tokens (block_size=%lld)", fn,
                (long long)c.block_size);
  if (g.columns < 0 || g.table_stride < g.columns || g.columns * c.block_size > 0x7fffffff)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: bad block table", fn);
  const int64_t strides[] = {g.q_row, g.q_head, g.k_row, g.k_head, g.v_row, g.v_head, g.out_row, g.out_head,
                             c.k_block, c.k_slot, c.k_head, c.v_block, c.v_slot, c.v_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8 != 0)
      return fail(PGS_ERR_MISALIGNED, "%s: strides must be multiples of 8 elements", fn);
  // (16 rows' offsets from their first are 32-bit)
  if (g.k_row > (1 << 26) || g.v_row > (1 << 26) || c.k_slot > (1 << 26) || c.v_slot > (1 << 26))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: rows are too far apart", fn);
  if (!(g.scale == g.scale)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: scale is NaN", fn);
  if (g.rows == 0 || g.requests == 0) return PGS_OK;
  if (!g.q || !g.k || !g.v || !g.out || !c.k || !c.v || !g.lens || !g.offsets || (g.columns > 0 && !g.block_tables))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(g.q, 16) || !aligned(g.k, 16) || !aligned(g.v, 16) || !aligned(g.out, 16) || !aligned(c.k, 16) ||
      !aligned(c.v, 16) || !aligned(g.lens, 4) || !aligned(g.offsets, 4) || !aligned(g.parents, 4) ||
      !aligned(g.block_tables, 4))
    return fail(PGS_ERR_MISALIGNED, "%s: tensors must be 16-byte aligned", fn);
  const Plan p = plan(g.requests, g.q_heads, c.kv_heads, g.max_tokens, g.max_context);
  const size_t need = workspace_bytes(p, g.rows, g.q_heads, c.head_dim);
  if (need > 0 && (!workspace || workspace_bytes_given < need || !aligned(workspace, 256)))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: needs a 256-byte aligned workspace of %zu bytes", fn, need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  Attend a{};
  a.q = static_cast<const uint16_t*>(g.q);
  a.k = static_cast<const uint16_t*>(g.k);
  a.v = static_cast<const uint16_t*>(g.v);
  a.out = static_cast<uint16_t*>(g.out);
  a.q_row = g.q_row, a.q_head = g.q_head, a.k_row = g.k_row, a.k_head = g.k_head;
  a.v_row = g.v_row, a.v_head = g.v_head, a.out_row = g.out_row, a.out_head = g.out_head;
  a.kc = static_cast<const uint16_t*>(c.k);
  a.vc = static_cast<const uint16_t*>(c.v);
  a.kc_block = c.k_block, a.kc_head = c.k_head, a.vc_block = c.v_block, a.vc_head = c.v_head;
  a.kc_slot = static_cast<uint32_t>(c.k_slot), a.vc_slot = static_cast<uint32_t>(c.v_slot);
  a.blocks = static_cast<int32_t>(c.blocks), a.bs = static_cast<int32_t>(c.block_size);
  a.tables = g.block_tables, a.tstride = g.table_stride, a.cols = static_cast<int32_t>(g.columns);
  a.lens = g.lens, a.offsets = g.offsets, a.parents = g.parents;
  a.rows = static_cast<int32_t>(g.rows), a.requests = static_cast<int32_t>(g.requests);
  a.q_heads = static_cast<int32_t>(g.q_heads), a.kv_heads = static_cast<int32_t>(c.kv_heads);
  a.group = a.q_heads / a.kv_heads;
  a.max_tokens = static_cast<int32_t>(g.max_tokens), a.row_groups = p.row_groups, a.splits = p.splits;
  a.c = g.scale * 1.44269504088896340736f;
  a.part = static_cast<float*>(workspace);
  a.stat = a.part + g.rows * g.q_heads * p.splits * c.head_dim;
  if (c.head_dim == 64)
    return g.dtype == PGS_DTYPE_F16 ? launch<64, true>(a, p, st) : launch<64, false>(a, p, st);
  return g.dtype == PGS_DTYPE_F16 ? launch<128, true>(a, p, st) : launch<128, false>(a, p, st);
}
