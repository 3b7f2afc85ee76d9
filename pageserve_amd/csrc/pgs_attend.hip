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
// P is rounded to the tensors' type for that product (in two terms it would take twice the
// MFMAs, which bound the kernel for many rows), and the row sums, one more MFMA per step with
// ones as A, add the rounded p that the output uses: a weight is off by half a step of the
// type at most, the output by 1.3 to 1.4 times what it is with P in fp32.  block_size is a
// multiple of 16, so a 16-key half lies in one block: its address is wave-uniform.
//
// Work: (request, key head, row group, part of the keys).  A workgroup's waves are
// row tiles x key slices, joined in LDS; parts are joined by a second kernel from
// fp32 partial outputs in the workspace.
#include <math.h>

#include <algorithm>

#include "pgs_linear.h"

namespace pgs {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kMaxTree = 64;

struct Attend {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  const uint16_t *kc, *vc;
  int64_t kc_block, kc_head, vc_block, vc_head;
  uint32_t kc_slot, vc_slot;
  int32_t blocks, bs;
  uint32_t bs_inv;  // ceil(2^32 / bs)
  const int32_t* tables;
  int64_t tstride;
  int32_t cols;
  const int32_t *lens, *offsets, *parents;
  int32_t rows, requests, q_heads, kv_heads, group;  // group: q_heads / kv_heads
  int32_t max_tokens, splits, min_steps;
  float c;      // scale * log2(e)
  float* part;  // sums of the parts of rows: [slots][D], slots as Wave::store's caller numbers them
  float* stat;  // [slots][2]: m, l
  int64_t* sums;  // (wide) [requests]: counts of work up to and with each request
};

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
template <int N>
__device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The kernel's argument again, read from its segment at this point: for the parts of a
// kernel outside its inner loop, whose fields would otherwise all sit in scalar
// registers throughout (and push vector registers out to memory).
__device__ __forceinline__ Attend again() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  Attend a;
  __builtin_memcpy(&a, (const void*)p, sizeof(a));
  return a;
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

// token / bs without a division: the product's high half is the quotient or one more
// (bs_inv is too large by less than 1, token below 2^31), which the remainder's sign
// shows
__device__ __forceinline__ int block_of(const Attend& a, int token, int& slot) {
  int q = static_cast<int>(__umulhi(static_cast<uint32_t>(token), a.bs_inv));
  int r = token - q * a.bs;
  if (r < 0) --q, r += a.bs;
  slot = r;
  return q;
}

// 16 R rows of a wave and their running sums.  The output MFMA d covers the dims
// (4 lg + i) D/16 + d of its lanes (SPREAD: the direct kernel), or 16 d + 4 lg + i.
template <int D, int R, bool F16, bool SPREAD>
struct Wave {
  using E = Elem<F16>;
  static constexpr int DC = D / 32;  // 32-dim chunks of a key
  static constexpr int DV = D / 16;  // dims of a value row per lane
  static constexpr int VW = DV / 2;  // their dwords
  u32x4 q[R][DC];
  f32x4 o[R][DV], l[R];
  float mx[R];
  bool far;  // some row's reference is beyond kFar (the same in all lanes)

  __device__ __forceinline__ void load(const Attend& a, const Request& rq, int kh, int row0, int nrows, int li, int lg) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = min(row0 + 16 * r + li, nrows - 1), t = row / a.group;  // (rows past the last repeat it)
      const uint16_t* p = a.q + (rq.row0 + t) * a.q_row + (kh * a.group + row - t * a.group) * a.q_head + 8 * lg;
#pragma unroll
      for (int d = 0; d < DC; ++d) q[r][d] = ld16(p + 32 * d);
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
      l[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DV; ++i) o[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // see[t] (LDS, the wave's own): which of the request's drafted tokens token t attends
  // to, itself and its ancestors, as a bit mask.  Lane t starts with bit t and its
  // parent; each step adds the parent's mask and takes the parent's parent, which
  // doubles the distance covered.
  static __device__ __forceinline__ int parent(const Attend& a, const Request& rq, int lane) {
    if (lane >= rq.tokens) return -1;
    return a.parents ? a.parents[rq.row0 + lane] : lane - 1;
  }
  static __device__ __forceinline__ void trees(int par, int lane, unsigned long long* see) {
    unsigned long long m = 1ull << lane;
    if (par >= lane || par < 0) par = -1;
    while (__ballot(par >= 0)) {
      const unsigned long long pm = __shfl(m, par & 63);
      const int pp = __shfl(par, par & 63);
      if (par >= 0) {
        m |= pm;
        par = pp;
      }
    }
    see[lane] = m;
  }

  // One step: keys key0 .. key0 + 31 of `limit` (cached, or with tree drafted).
  // keys(h, d): A operand of the 16-key half h, 32-dim chunk d; values(d): that of
  // output MFMA d.  (SPREAD false: both are read here, from LDS, four at a time; left
  // to itself the compiler reads each just before its use and waits for it alone.)
  // masked: some key is past the limit, in an absent block (bad) or drafted.
  // odd: drafted keys whose values are not finite (v holds zeros for them); value(j)
  // is the row of key key0 + j.  see(r): which drafted tokens the lane's row r attends to.
  template <typename Keys, typename Values, typename See, typename Value>
  __device__ __forceinline__ void step(const Attend& a, Keys keys, Values values, int key0, int limit, bool tree,
                                       bool masked, bool bad0, bool bad1, uint32_t odd, See see, int li, int lg,
                                       Value value) {
    // lane's scores: keys key0 + 16 h + 4 lg + i
    f32x4 s[R][2];
    u32x4 k[2][DC], v[DV];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < DC; ++d) k[h][d] = keys(h, d);
    if (!SPREAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][h] = f32x4{0.f, 0.f, 0.f, 0.f};
    // (the four chains in turn: none waits for its own last product)
#pragma unroll
    for (int d = 0; d < DC; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][h] = E::mfma(k[h][d], q[r][d], s[r][h]);
    if constexpr (!SPREAD) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < DV; ++d) v[d] = values(d);
      __builtin_amdgcn_sched_barrier(0);
    }
    // exponents against the row's reference, and whether a row needs a new one
    float x[R][8];
    uint32_t ok[R];
    bool over = false;
    if (masked || far) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const unsigned long long sees = tree ? see(r) : ~0ull;
        ok[r] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + 16 * (e >> 2) + 4 * lg + (e & 3);
          const bool in = key < limit && !(e >> 2 ? bad1 : bad0) && (sees >> (key & 63) & 1);
          ok[r] |= in ? 1u << e : 0;
          x[r][e] = in ? exponent(s[r][e >> 2][e & 3], a.c, mx[r], far) : -INFINITY;
          over = over || x[r][e] > kSlack + E::kHead;
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ok[r] = 0xff;
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[r][e] = fmaf(s[r][e >> 2][e & 3], a.c, -mx[r]);
          top = fmaxf(top, x[r][e]);
        }
        over = over || top > kSlack + E::kHead;
      }
    }
    if (__ballot(over)) {
      // new references: the largest score of each row so far
      bool beyond = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float t = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) t = fmaxf(t, ok[r] >> e & 1 ? s[r][e >> 2][e & 3] * a.c : -INFINITY);
        t = quad_max(t);
        const float ref = fmaxf(fabsf(t) > kFar ? t : t - E::kHead, mx[r]), f = __builtin_amdgcn_exp2f(mx[r] - ref);
        mx[r] = ref;
        beyond = beyond || fabsf(ref) > kFar;
#pragma unroll
        for (int i = 0; i < 4; ++i) l[r][i] *= f;
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[r][d][i] *= f;
      }
      far = __ballot(beyond);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[r][e] = ok[r] >> e & 1 ? exponent(s[r][e >> 2][e & 3], a.c, mx[r], far) : -INFINITY;
    }
    u32x4 p[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[r][i] = E::pack(__builtin_amdgcn_exp2f(x[r][2 * i]), __builtin_amdgcn_exp2f(x[r][2 * i + 1]));
    const u32x4 ones = {E::kOnes, E::kOnes, E::kOnes, E::kOnes};
#pragma unroll
    for (int r = 0; r < R; ++r) l[r] = E::mfma(ones, p[r], l[r]);
#pragma unroll
    for (int d = 0; d < DV; ++d) {
      if constexpr (SPREAD) v[d] = values(d);
#pragma unroll
      for (int r = 0; r < R; ++r) o[r][d] = E::mfma(v[d], p[r], o[r][d]);
    }
    for (uint32_t w = odd; w; w &= w - 1) {
      const int j = __builtin_ctz(w);
      const uint16_t* row = value(j);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t lo = j & 2 ? p[r][1] : p[r][0], hi = j & 2 ? p[r][3] : p[r][2];
        const float pj = E::low(__shfl(j & 16 ? hi : lo, 16 * (j >> 2 & 3) + li) >> (16 * (j & 1)));
        if (!(see(r) >> ((key0 + j) & 63) & 1)) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < DV; ++d) o[r][d][i] += pj * E::low(row[SPREAD ? (4 * lg + i) * DV + d : 16 * d + 4 * lg + i]);
      }
    }
  }

  // The rows' outputs, or (whole false: other keys of theirs are elsewhere) their
  // sums.  slot(row, token, head): where to.
  template <typename Slot>
  __device__ __forceinline__ void store(const Attend& a, const Request& rq, int kh, int row0, int nrows, int li, int lg,
                                        bool whole, Slot slot) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = row0 + 16 * r + li;
      if (row >= nrows) continue;
      const int t = row / a.group, head = kh * a.group + row - t * a.group;
      const int64_t token = rq.row0 + t;
      if (whole) {
        const float inv = l[r][0] == 0.f ? 0.f : 1.f / l[r][0];
        uint16_t* d = a.out + token * a.out_row + head * a.out_head + 4 * lg * (SPREAD ? DV : 1);
        if constexpr (SPREAD) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[VW];
#pragma unroll
            for (int e = 0; e < VW; ++e) w[e] = E::pack(o[r][2 * e][i] * inv, o[r][2 * e + 1][i] * inv);
            if constexpr (VW == 4) *reinterpret_cast<u32x4*>(d + i * DV) = u32x4{w[0], w[1], w[2], w[3]};
            else *reinterpret_cast<u32x2*>(d + i * DV) = u32x2{w[0], w[1]};
          }
        } else {
#pragma unroll
          for (int e = 0; e < DV; ++e)
            *reinterpret_cast<u32x2*>(d + 16 * e) = u32x2{E::pack(o[r][e][0] * inv, o[r][e][1] * inv),
                                                          E::pack(o[r][e][2] * inv, o[r][e][3] * inv)};
        }
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
          for (int e = 0; e < DV; ++e) *reinterpret_cast<f32x4*>(d + 16 * e) = o[r][e];
        }
        if (lg == 0) {
          a.stat[2 * at] = mx[r];
          a.stat[2 * at + 1] = l[r][0];
        }
      }
    }
  }
};

// Parts that the keys of a request are cut into, of the `splits` that the grid has, by its
// 32-key steps (twice those where two waves share a step): none below kWholeSteps, else of
// min_steps at least.
constexpr int kWholeSteps = 32, kCoarseSteps = 16, kFineSteps = 8;
__device__ __forceinline__ int parts_of(const Attend& a, const Request& rq, int wr) {
  const int steps = (rq.len_tiles + rq.tree_tiles) * wr;
  return steps < kWholeSteps ? 1 : min(a.splits, steps / a.min_steps);
}

// Few rows (up to 64 per key head): bound by reading the keys and values once, and for
// short contexts by the chain of loads (lengths, block numbers, and a round of keys per step:
// only the next step's block numbers are loaded ahead).  A workgroup's NW waves are WR row
// tiles x NW/WR key slices; each wave loads the keys of its steps straight into registers.
// Measured in a replayed graph, 16 heads on two key heads of 128 dims: one token of 256
// requests of 512 keys 26.2 us (5.1 TB/s of keys and values), of 64 of 2048 29.1 (4.6), of
// one of 32768 with the join 17.9 (1.9); 4 tokens of 64 of 2048 32.0 (4.2).
template <int D, int R, int WR, int NW, bool F16>
__global__ __launch_bounds__(64 * NW, 2) void attend_kernel(Attend a) {
  using W = Wave<D, R, F16, true>;
  using E = Elem<F16>;
  constexpr int DC = W::DC, DV = W::DV, VW = W::VW;
  constexpr int WK = NW / WR;  // key slices
  const int lane = threadIdx.x & 63;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int li = lane & 15, lg = lane >> 4;
  const int wr = wave % WR, wk = wave / WR;
  // unit: ((request, key head), part)
  const int part = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int kh = unit % a.kv_heads, b = unit / a.kv_heads;
  const Request rq = request(a, b);
  const int parts = parts_of(a, rq, WR);
  const int nrows = rq.tokens * a.group;
  if (nrows == 0 || part >= parts) return;
  const int row0 = wr * (16 * R);  // of this wave

  // the steps of this part: [t0, t1) of len_tiles + tree_tiles
  const int tiles = rq.len_tiles + rq.tree_tiles;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * part / parts);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / parts);

  const int32_t* table = a.tables + b * a.tstride;
  // the block ids of a step's two halves, loaded a step ahead of its keys
  auto ids = [&](int t, int (&id)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int slot;
      // (not provably uniform: the value stays in a vector register, unwaited for, until
      // it is used)
      if (t < rq.len_tiles && t < t1)
        id[h] = table[block_of(a, min(t * 32 + 16 * h, rq.len - 1), slot) + (here(lane) >> 6)];
    }
  };
  struct Keys {
    u32x4 k[2][DC];
    uint32_t v[8][VW];
    bool bad[2];
  };
  auto load = [&](int t, const int (&id)[2], Keys& n) {
    const bool tree = t >= rq.len_tiles;
    const int key0 = (tree ? t - rq.len_tiles : t) * 32;
    const int limit = tree ? rq.tokens : rq.len;
    // each half: a uniform base and the last key of it that exists (a key past the
    // end reads that one instead and is masked)
    const uint32_t ks = tree ? static_cast<uint32_t>(a.k_row) : a.kc_slot;
    const uint32_t vs = tree ? static_cast<uint32_t>(a.v_row) : a.vc_slot;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int first = min(key0 + 16 * h, limit - 1), last = limit - 1 - first;
      const uint16_t *kb, *vb;
      n.bad[h] = false;
      if (tree) {
        kb = a.k + (rq.row0 + first) * a.k_row + kh * a.k_head;
        vb = a.v + (rq.row0 + first) * a.v_row + kh * a.v_head;
      } else {
        const int blk = uniform(id[h]);
        n.bad[h] = blk < 0 || blk >= a.blocks;
        int slot;
        block_of(a, first, slot);
        const int64_t at = n.bad[h] ? 0 : blk;
        kb = a.kc + at * a.kc_block + static_cast<int64_t>(slot) * a.kc_slot + kh * a.kc_head;
        vb = a.vc + at * a.vc_block + static_cast<int64_t>(slot) * a.vc_slot + kh * a.vc_head;
      }
      const uint16_t* p = kb + static_cast<uint32_t>(min(li, last)) * ks + 8 * lg;
#pragma unroll
      for (int d = 0; d < DC; ++d) n.k[h][d] = ld16(p + 32 * d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t* y = vb + static_cast<uint32_t>(min(4 * lg + e, last)) * vs + DV * li;
        if constexpr (VW == 4) {
          const u32x4 x = ld16(y);
#pragma unroll
          for (int i = 0; i < 4; ++i) n.v[4 * h + e][i] = x[i];
        } else {
          const u32x2 x = *reinterpret_cast<const u32x2*>(y);
#pragma unroll
          for (int i = 0; i < 2; ++i) n.v[4 * h + e][i] = x[i];
        }
      }
    }
  };

  // (the first block ids, the parents and the rows are on their way together)
  int id[2] = {0, 0};
  ids(t0 + wk, id);
  const int par = t1 > rq.len_tiles ? W::parent(a, rq, lane) : -1;
  W w;
  w.load(a, rq, kh, row0, nrows, li, lg);
  __shared__ unsigned long long lsee[NW][kMaxTree];
  int token[R];
#pragma unroll
  for (int r = 0; r < R; ++r) token[r] = min(row0 + 16 * r + li, nrows - 1) / a.group;
  if (t1 > rq.len_tiles) w.trees(par, lane, lsee[wave]);
  for (int t = t0 + wk; t < t1; t += WK) {
    Keys n;
    load(t, id, n);
    ids(t + WK, id);
    const bool tree = t >= rq.len_tiles;
    const int key0 = (tree ? t - rq.len_tiles : t) * 32;
    const int limit = tree ? rq.tokens : rq.len;
    const bool masked = tree || key0 + 32 > limit || n.bad[0] || n.bad[1];
    // values that no row may take must not meet p = 0 as an infinity or NaN: those
    // past the end and of absent blocks become zeros, and a drafted token's that
    // are not finite are left out of the products (bit of `odd`) and added for the
    // rows that see it
    uint32_t odd = 0;
    if (masked) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool gone = key0 + 16 * (e >> 2) + 4 * lg + (e & 3) >= limit || n.bad[e >> 2];
        bool wild = false;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          if (gone) n.v[e][i] = 0;
          wild = wild || (n.v[e][i] & E::kExp) == E::kExp || (n.v[e][i] & E::kExp << 16) == E::kExp << 16;
        }
        const unsigned long long m = tree ? __ballot(wild) : 0;
        if (m) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (m >> (16 * g) & 0xffff) odd |= 1u << (16 * (e >> 2) + 4 * g + (e & 3));
          if (m >> (16 * lg) & 0xffff)
#pragma unroll
            for (int i = 0; i < VW; ++i) n.v[e][i] = 0;
        }
      }
    }
    auto values = [&](int d) {
      u32x4 vt;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vt[e] = __builtin_amdgcn_perm(n.v[2 * e + 1][d >> 1], n.v[2 * e][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
      return vt;
    };
    w.step(a, [&](int h, int d) { return n.k[h][d]; }, values, key0, limit, tree, masked, n.bad[0], n.bad[1], odd,
           [&](int r) { return lsee[wave][token[r]]; }, li, lg,
           [&](int j) { return a.v + (rq.row0 + key0 + j) * a.v_row + kh * a.v_head; });
  }

  // join the key slices: slice 0 adds the others' sums, brought to one reference
  if constexpr (WK > 1) {
    __shared__ float lo_[(WK - 1) * WR][R][DV * 4][64];
    __shared__ float ls_[(WK - 1) * WR][R][2][64];
    if (wk > 0) {
      const int n = (wk - 1) * WR + wr;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        ls_[n][r][0][lane] = w.mx[r];
        ls_[n][r][1][lane] = w.l[r][0];
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
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[r][d][i] *= f;
#pragma unroll
      for (int s = 0; s < WK - 1; ++s) {
        const int n = s * WR + wr;
        const float g = __builtin_amdgcn_exp2f(ls_[n][r][0][lane] - ref);
        w.l[r][0] += g * ls_[n][r][1][lane];
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

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// The wide kernel's work: the tiles of all (request, key head, group of kGroup rows), in
// that order, cut into equal shares for the workgroups, whatever the requests' lengths
// are.  A group of at most half the rows has two key slices: half the arithmetic per tile,
// but the same loads.  A tile counts kFull, or kHalf there (`weight`), and a unit kUnit more
// for its rows' loads and its sums: fitted to the workgroups' times (4.6, 2.8 and 10 us).  A
// share has the tiles whose counts begin in it; of a unit that is not whole it leaves sums
// in slot 2 g (the unit began in an earlier share) or 2 g + 1.
// (all at 128 dims; 64 dims use the same.)
constexpr int kFull = 10, kHalf = 6, kUnit = 20;
constexpr int kShares = 256;      // workgroups: one per CU
static_assert(kHalf <= kFull);
constexpr int kMinShare = kFull;  // counts of a share at least (16 requests of 512 keys: 24 us, 3 kFull 32, 6 kFull 45)
constexpr int kWideRows = 2;      // row tiles of 16 per wave
constexpr int kWideWaves = 16 / kWideRows;
constexpr int kGroup = 16 * kWideRows * kWideWaves;
constexpr int kBuffers = 2;  // tiles in LDS: computed, on its way
constexpr int kTile = 128;   // keys of a tile

struct Groups {
  int tiles, n;     // of a request: tiles per group, groups
  int last;         // weight of the last group (the others': kFull)
  int64_t per_head; // counts of one key head
};
__device__ __forceinline__ Groups groups_of(const Attend& a, const Request& rq) {
  const int rows = rq.tokens * a.group;
  Groups g;
  g.tiles = (rq.len + kTile - 1) / kTile + (rq.tokens + kTile - 1) / kTile;
  g.n = (rows + kGroup - 1) / kGroup;
  g.last = rows - (g.n - 1) * kGroup > kGroup / 2 ? kFull : kHalf;
  g.per_head = g.n ? static_cast<int64_t>(g.tiles) * (kFull * (g.n - 1) + g.last) + kUnit * g.n : 0;
  return g;
}
__device__ __forceinline__ int shares_of(int64_t total) {
  // (not rounded up: a share between a unit's first and last has to have one of its tiles)
  return static_cast<int>(min<int64_t>(kShares, max<int64_t>(1, total / kMinShare)));
}
// where share g of n begins
__device__ __forceinline__ int64_t share_begin(int64_t total, int g, int n) { return g * total / n; }

struct Work {
  static constexpr int NT = 64 * kWideWaves;
  Attend a;
  int64_t* pre;   // LDS [NT]: counts up to and with request base + i
  int64_t* wsum;  // LDS [kWideWaves]
  int base;
  int64_t carry, total;
  struct Unit {
    Request rq;
    int b, kh, rg, tiles, cached, weight;
    int64_t begin;  // where its first tile's counts begin
  };

  // pre for the requests from `first` on; every thread must call it
  __device__ __forceinline__ void fill(int first, int64_t before) {
    const int thread = here(threadIdx.x), lane = thread & 63, wave = thread >> 6;
    base = first;
    carry = before;
    int64_t v = 0;
    if (first + thread < a.requests) v = groups_of(a, request(a, first + thread)).per_head * a.kv_heads;
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
  // the total; with `keep` the sums of all requests are left there for the join
  __device__ __forceinline__ void start(int64_t* keep) {
    const int thread = here(threadIdx.x);
    total = 0;
    for (int f = 0; f < a.requests; f += NT) {
      fill(f, total);
      if (keep && f + thread < a.requests) keep[f + thread] = pre[thread];
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
    const Request rq = request(a, u.b);
    u.rq = Request{uniform(rq.row0), uniform(rq.tokens), uniform(rq.len), 0, 0};
    const Groups g = groups_of(a, u.rq);
    const int64_t first = uniform64(lo ? pre[lo - 1] : carry);
    u.kh = uniform(static_cast<int>((pos - first) / g.per_head));
    const int64_t in = pos - first - u.kh * g.per_head;
    const int64_t full = static_cast<int64_t>(kFull) * g.tiles + kUnit;
    u.rg = uniform(static_cast<int>(min<int64_t>(in / full, g.n - 1)));
    u.tiles = g.tiles;
    u.cached = (u.rq.len + kTile - 1) / kTile;
    u.weight = u.rg == g.n - 1 ? g.last : kFull;
    u.begin = first + u.kh * g.per_head + u.rg * full + kUnit;
    return u;
  }
};

// Many rows: bound by the matrix units and the softmax, and a short group by its loads.
// Eight waves share tiles of 128 keys through LDS, 8 x 32 rows, or for a group of at most
// 128 rows 4 x 2 key slices (a wave then takes every second 32-key step of a tile, and the
// two are joined at the end of a unit).  A tile goes from memory to LDS past the registers,
// into the buffer that is not computed: one barrier per tile, and a load has a tile's
// arithmetic to arrive.
//
// LDS rows are D/8 pieces of 16 bytes.  A wave reads keys as A operands, 16 keys x one
// piece per access: piece p of key r lies at p ^ (r D / 128), so that the sixteen lanes
// of an access meet all banks.  Values are read transposed, 4 keys x 16 dims per 16 lanes
// (ds_read_b64_tr_b16: lane n gets dim n of the four keys), a pair of pieces of 16 keys per
// access: they are exchanged in pairs, p ^ 2 (r D / 128).
//
// Measured at 24 requests of up to 64 rows x 16 heads of 128 dims: 105 us with the join (106 to
// 114 and 9 in a trace of few calls), a full tile (256 rows x 128 keys) 4.6 us, 40% of the
// matrix units' rate: a step's scores, softmax and output follow one another in a wave, and the
// second wave of a SIMD covers a part of it.  Tiles through registers 133, of 64 keys 121.  The
// same: four waves per SIMD of 16 rows each, a higher priority for half of the waves, half of
// them starting a tile later (116), the next step's keys read during the softmax (and 131 for
// 123 across the barrier).
template <int D, bool F16>
__global__ __launch_bounds__(64 * kWideWaves, kWideWaves / 4) void attend_wide_kernel(Attend a) {
  constexpr int R = kWideRows, J = kTile * D / 512 / kWideWaves;  // J: loads per wave, tile and matrix
  using W = Wave<D, R, F16, false>;
  using E = Elem<F16>;
  constexpr int DV = W::DV;
  constexpr int NW = kWideWaves, TK = kTile;
  constexpr int P = D / 8;           // pieces per row
  constexpr int KI = 64 / P;         // keys of one wave-wide load
  constexpr int KW = J * KI;         // keys of a wave's loads
  static_assert(TK == NW * KW && 16 % KW == 0, "a wave's keys lie in one block");
  __shared__ __attribute__((aligned(256))) uint16_t lkv[kBuffers][2][TK * D];  // (whole rows aligned: k_at)
  __shared__ uint32_t lbad[kBuffers][NW];            // the wave's keys are of an absent block
  __shared__ unsigned long long lodd[kBuffers][NW];  // (drafted tile) keys whose values are not finite
  __shared__ unsigned long long lsee[NW][kMaxTree];
  __shared__ int64_t lpre[64 * NW], lsum[NW];
  const int lane = threadIdx.x & 63;
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  // LDS byte addresses of this lane's pieces of the first step: key li, piece lg; and
  // dims 4 (li % 4) .. +3 of key 4 lg + li / 4
  const int li = lane & 15, lg = lane >> 4, vkey = 4 * lg + (li >> 2);
  const uint32_t k_at = lds_address(lkv) + li * (2 * D) + 16 * (lg ^ (li * P / 16 & (P - 1)));
  const uint32_t v_at = lds_address(lkv) + TK * D * 2 + vkey * (2 * D) +
                        16 * ((li >> 1 & 1) ^ (2 * (vkey * P / 16) & (P - 1))) + 8 * (li & 1);
  Work work{again(), lpre, lsum, 0, 0, 0};
  work.start(blockIdx.x == 0 ? work.a.sums : nullptr);
  const int shares = shares_of(work.total), share = xcd_remap(blockIdx.x, gridDim.x);
  if (share >= shares) return;
  const int64_t begin = uniform64(share_begin(work.total, share, shares));
  const int64_t end = uniform64(share_begin(work.total, share + 1, shares));

  for (int64_t pos = begin; pos < end;) {
    work.a = again();
    const Work::Unit un = work.find(pos);
    const Request& rq = un.rq;
    const int nrows = rq.tokens * a.group;
    const int slices = un.weight == kHalf ? 2 : 1;  // of the keys
    const int wr = slices == 2 ? wave % (NW / 2) : wave, wk = slices == 2 ? wave / (NW / 2) : 0;
    const int row0 = un.rg * kGroup + wr * (16 * R);  // of this wave
    const bool active = row0 < nrows;
    const int kh = un.kh, cached = un.cached;

    // this share's tiles of the unit: cached ones, then the drafted tokens'
    const int t0 = uniform(static_cast<int>((max<int64_t>(pos - un.begin, 0) + un.weight - 1) / un.weight));
    const int t1 = uniform(static_cast<int>(min<int64_t>(un.tiles, (end - un.begin + un.weight - 1) / un.weight)));
    pos = un.begin + static_cast<int64_t>(un.tiles) * un.weight;  // the next unit's
    if (t0 >= t1) continue;

    const int32_t* table = a.tables + un.b * a.tstride;
    const uint16_t *kc = a.kc + kh * a.kc_head, *vc = a.vc + kh * a.vc_head;
    // Lane i: the block of this wave's keys of tile id0 + i.  (Waited for where it is
    // loaded: a wait for it further on would be one for the keys on their way too.)
    int id_lane = 0, id0 = t0 - 64;
    // tile t into buffer `to`; whether its keys are of an absent block
    auto load = [&](int t, int to) {
      const int ln = here(lane), kin = ln / P, piece = ln % P;
      const uint32_t at_k = lds_address(lkv) + to * (4 * TK * D) + wave * (1024 * J), at_v = at_k + 2 * TK * D;
      // (lane l fills piece l % P of its key's row in LDS: the exchange picks what it reads)
      if (t >= cached) {
        const Attend c = again();
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int key = wave * KW + j * KI + kin, turn = key * P / 16;
          const int64_t at = rq.row0 + min((t - cached) * TK + key, rq.tokens - 1);
          load_lds(c.k + at * c.k_row + kh * c.k_head + 8 * (piece ^ (turn & (P - 1))), at_k + 1024 * j);
          load_lds(c.v + at * c.v_row + kh * c.v_head + 8 * (piece ^ (2 * turn & (P - 1))), at_v + 1024 * j);
        }
        return false;
      }
      if (t >= id0 + 64) {
        id0 = t;
        int slot;
        const int64_t key = min<int64_t>(static_cast<int64_t>(t + ln) * TK + wave * KW, rq.len - 1);
        id_lane = table[block_of(a, static_cast<int>(key), slot)];
        asm volatile("" : "+v"(id_lane));
      }
      const int id = __builtin_amdgcn_readlane(id_lane, t - id0);
      const bool bad = id < 0 || id >= a.blocks;
      const int64_t blk = bad ? 0 : id;
      // (a key past the end reads the last one instead and is masked)
      const int first = min(t * TK + wave * KW, rq.len - 1);
      int slot;
      block_of(a, first, slot);
      const int64_t at0 = slot;
      const uint16_t *kb = kc + blk * a.kc_block + at0 * a.kc_slot, *vb = vc + blk * a.vc_block + at0 * a.vc_slot;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int64_t at = min(j * KI + kin, rq.len - 1 - first);
        const int turn = (wave * KW + j * KI + kin) * P / 16;
        load_lds(kb + at * a.kc_slot + 8 * (piece ^ (turn & (P - 1))), at_k + 1024 * j);
        load_lds(vb + at * a.vc_slot + 8 * (piece ^ (2 * turn & (P - 1))), at_v + 1024 * j);
      }
      return bad;
    };
    // This wave's part of tile t has arrived in buffer `in`: as in attend_kernel, no
    // infinity or NaN may meet p = 0.
    auto settle = [&](int t, int in, bool bad) {
      const bool tree = t >= cached;
      const int key0 = (tree ? t - cached : t) * TK + wave * KW, limit = tree ? rq.tokens : rq.len;
      const int ln = here(lane), kin = ln / P;
      if (tree || bad || key0 + KW > limit) {
        uint32_t odd = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          u32x4* const at = reinterpret_cast<u32x4*>(&lkv[in][1][(wave * J + j) * 512 + 8 * ln]);
          const bool gone = bad || key0 + j * KI + kin >= limit;
          bool wild = false;
          if (tree && !gone) {
            const u32x4 v = *at;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              wild = wild || (v[i] & E::kExp) == E::kExp || (v[i] & E::kExp << 16) == E::kExp << 16;
          }
          const unsigned long long m = __ballot(wild), one = P == 16 ? 0xffffull : 0xffull;
#pragma unroll
          for (int k = 0; k < KI; ++k)
            if (m >> (P * k) & one) odd |= 1u << (j * KI + k);
          if (gone || (m >> (P * kin) & one)) *at = u32x4{0, 0, 0, 0};
        }
        // (drafted tokens are 64 at most)
        if (ln == 0) lodd[in][wave] = static_cast<unsigned long long>(odd) << (wave * KW & 63);
      }
      if (ln == 0) lbad[in][wave] = bad;
    };

    // One barrier per tile.  Behind it, tile t is whole in its buffer and the one that held
    // tile t - 1 is free: tile t + 1 is sent for, t is computed, and each wave waits for its
    // part of t + 1.
    const bool bad0 = load(t0, 0);
    W w;
    if (active) {
      const Attend c = again();
      const int ln = here(lane);
      const int par = t1 > cached ? w.parent(c, rq, ln) : -1;
      w.load(c, rq, kh, row0, nrows, ln & 15, ln >> 4);
      if (t1 > cached) w.trees(par, ln, lsee[wave]);
    }
    arrived<0>();
    settle(t0, 0, bad0);
    __syncthreads();
    int buf = 0;
    for (int t = t0; t < t1; ++t) {
      const int next = buf == kBuffers - 1 ? 0 : buf + 1;
      bool bad1 = false;
      if (t + 1 < t1) bad1 = load(t + 1, next);
      if (active) {
        const bool tree = t >= cached;
        const int key0 = (tree ? t - cached : t) * TK, limit = tree ? rq.tokens : rq.len;
        const int ln = here(lane);
        const uint32_t bm = static_cast<uint32_t>(__ballot(ln < NW && lbad[buf][ln % NW]));
        const bool masked = tree || key0 + TK > limit || bm;
        unsigned long long odd = 0;
        if (tree)
#pragma unroll
          for (int i = 0; i < NW; ++i) odd |= lodd[buf][i];
#pragma unroll 1
        for (int h = wk; h < TK / 32; h += slices) {
          if (key0 + 32 * h >= limit) break;
          // a piece's exchange is an exclusive or of its row's address with 16 bytes times
          // the piece, halves of a step and steps are 16 and 32 whole rows apart
          const uint32_t kat = k_at + buf * (4 * TK * D) + 32 * h * (2 * D);
          const uint32_t vat = v_at + buf * (4 * TK * D) + 32 * h * (2 * D);
          auto keys = [&](int g, int d) { return *lds<const u32x4>((kat ^ (64 * d)) + 16 * g * (2 * D)); };
          auto values = [&](int d) {
            const u32x2 x = read_transposed((vat ^ (32 * d))), y = read_transposed((vat ^ (32 * d)) + 16 * (2 * D));
            return u32x4{x[0], x[1], y[0], y[1]};
          };
          const uint32_t odd32 = h < 2 ? static_cast<uint32_t>(odd >> (32 * h)) : 0;
          const int ln = here(lane);
          auto see = [&](int r) { return lsee[wave][min(row0 + 16 * r + (ln & 15), nrows - 1) / again().group]; };
          w.step(a, keys, values, key0 + 32 * h, limit, tree, masked, bm >> (32 * h / KW) & 1,
                 bm >> ((32 * h + 16) / KW) & 1, odd32, see, ln & 15, ln >> 4, [&](int j) {
                   const Attend c = again();
                   return c.v + (rq.row0 + key0 + 32 * h + j) * c.v_row + kh * c.v_head;
                 });
        }
      }
      if (t + 1 < t1) {
        arrived<0>();
        settle(t + 1, next, bad1);
      }
      buf = next;
      __syncthreads();
    }

    // (two slices) the second's sums are added to the first's, brought to one reference
    if (slices == 2) {
      float* lo = reinterpret_cast<float*>(lkv) + wr * (R * DV * 4 * 64);
      const int ln = here(lane);
      static_assert(sizeof(lkv) >= NW / 2 * R * DV * 4 * 64 * 4, "the sums fit the tiles' space");
      __shared__ float ls[NW / 2][R][2][64];
      if (active && wk == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          ls[wr][r][0][ln] = w.mx[r];
          ls[wr][r][1][ln] = w.l[r][0];
#pragma unroll
          for (int d = 0; d < DV; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) lo[(r * DV * 4 + 4 * d + i) * 64 + ln] = w.o[r][d][i];
        }
      }
      __syncthreads();
      if (active && wk == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float m = ls[wr][r][0][ln], ref = fmaxf(w.mx[r], m);
          const float f = __builtin_amdgcn_exp2f(w.mx[r] - ref), g = __builtin_amdgcn_exp2f(m - ref);
          w.mx[r] = ref;
          w.l[r][0] = f * w.l[r][0] + g * ls[wr][r][1][ln];
#pragma unroll
          for (int d = 0; d < DV; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w.o[r][d][i] = f * w.o[r][d][i] + g * lo[(r * DV * 4 + 4 * d + i) * 64 + ln];
        }
      }
      __syncthreads();
    }
    if (active && wk == 0) {
      const int64_t slot0 = static_cast<int64_t>(2 * share + (un.begin >= begin) - un.rg) * kGroup;
      const int ln = here(lane);
      w.store(again(), rq, kh, row0, nrows, ln & 15, ln >> 4, t0 == 0 && t1 == un.tiles,
              [&](int row, int64_t, int) { return slot0 + row; });
    }
  }
}

// Four rows' outputs from n parts' sums each: brought to one reference, added in order and
// divided by the joined sum.  Sixteen lanes per row, each with D/16 neighbouring dims;
// slot(i): where part i of the lane's row is; p: the lane's dims of the output, or null.
// WAVES: of the workgroup, each taking that share of the parts (all must call it), joined in
// LDS; or 1.  Bound by memory and, few rows of many parts, by its latency: up to eight
// parts' loads are on their way together.
template <int D, bool F16, int WAVES, typename Slot>
__device__ __forceinline__ void join_rows(const Attend& a, int n, int lane, int wave, uint16_t* p, Slot slot) {
  constexpr int W = D / 16;
  const int li = lane & 15;
  float ref = kLow, sum = 0.f, o[W];
#pragma unroll
  for (int d = 0; d < W; ++d) o[d] = 0.f;
  const int end = WAVES == 1 ? n : n * (wave + 1) / WAVES;
  auto batch = [&](int i0, auto count) {
    constexpr int U = decltype(count)::value;
    f32x2 st[U];
    f32x4 x[U][W / 4];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int64_t at = slot(min(i0 + e, end - 1));
      st[e] = *reinterpret_cast<const f32x2*>(a.stat + 2 * at);
#pragma unroll
      for (int d = 0; d < W / 4; ++d) x[e][d] = *reinterpret_cast<const f32x4*>(a.part + at * D + W * li + 4 * d);
    }
    float top = ref;
#pragma unroll
    for (int e = 0; e < U; ++e) top = fmaxf(top, st[e][0]);
    const float f = __builtin_amdgcn_exp2f(ref - top);
    ref = top;
    sum *= f;
#pragma unroll
    for (int d = 0; d < W; ++d) o[d] *= f;
#pragma unroll
    for (int e = 0; e < U; ++e) {
      if (i0 + e >= end) break;  // (a part read again)
      const float g = __builtin_amdgcn_exp2f(st[e][0] - ref);
      sum = fmaf(g, st[e][1], sum);
#pragma unroll
      for (int d = 0; d < W; ++d) o[d] = fmaf(g, x[e][d / 4][d % 4], o[d]);
    }
  };
  int i = WAVES == 1 ? 0 : n * wave / WAVES;
  for (; end - i > 4; i += 8) batch(i, Int<8>{});
  if (end - i > 2) batch(i, Int<4>{});
  else if (end > i) batch(i, Int<2>{});
  if constexpr (WAVES > 1) {
    __shared__ float lref[WAVES][64], lsum[WAVES][64], lo[WAVES][W][64];
    lref[wave][lane] = ref;
    lsum[wave][lane] = sum;
#pragma unroll
    for (int d = 0; d < W; ++d) lo[wave][d][lane] = o[d];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) ref = fmaxf(ref, lref[w][lane]);
    sum = 0.f;
#pragma unroll
    for (int d = 0; d < W; ++d) o[d] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float g = __builtin_amdgcn_exp2f(lref[w][lane] - ref);
      sum = fmaf(g, lsum[w][lane], sum);
#pragma unroll
      for (int d = 0; d < W; ++d) o[d] = fmaf(g, lo[w][d][lane], o[d]);
    }
  }
  if (!p) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t w[W / 2];
#pragma unroll
  for (int d = 0; d < W / 2; ++d) w[d] = Elem<F16>::pack(o[2 * d] * inv, o[2 * d + 1] * inv);
  if constexpr (W == 8) *reinterpret_cast<u32x4*>(p) = u32x4{w[0], w[1], w[2], w[3]};
  else *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
}

// Waves that join four rows: sixteen if those have eight parts and there are few of them, so
// that the parts' latency counts, else one (and four times four rows a workgroup).  Measured,
// the whole call in microseconds, sixteen/one, 16 heads on two key heads of 128 dims: one
// token of 32768 keys 17.0/32.0, of 4096 (8 parts) 14.4/15.8, of 2048 (4) 14.1/13.9; 64
// requests of 4 tokens and 4096 keys (8 parts, 1024 fours) 63.2/61.6; two requests of 64
// tokens and 4096 keys (32 parts, 512 fours) 38.2/39.5, four of 2048 (16, 1024) 44.6/36.4.
constexpr int kJoinWaves = 16;
inline bool join_by_many(int64_t parts, int64_t fours) { return parts >= 8 && fours <= 512; }
constexpr int join_threads(int waves) { return waves == 1 ? 256 : 64 * waves; }
// the four rows of a wave
template <int WAVES>
__device__ __forceinline__ int64_t join_quad(int wave) {
  return WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + wave : blockIdx.x;
}

// Behind attend_kernel: rows are (token, head) of a request.
template <int D, bool F16, int WAVES>
__global__ __launch_bounds__(join_threads(WAVES)) void join_kernel(Attend a, int wr) {
  const int lane = threadIdx.x & 63, li = lane & 15, wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int64_t u = join_quad<WAVES>(wave);
  const int quads = (a.max_tokens * a.q_heads + 3) >> 2;
  const int b = static_cast<int>(u / quads), first = static_cast<int>(u - static_cast<int64_t>(b) * quads) * 4;
  if (b >= a.requests) return;
  const Request rq = request(a, b);
  const int parts = parts_of(a, rq, wr), rows = rq.tokens * a.q_heads;
  if (first >= rows || parts == 1) return;
  const int row = min(first + (lane >> 4), rows - 1), t = row / a.q_heads;
  const int64_t at = (static_cast<int64_t>(rq.row0) * a.q_heads + row) * a.splits;
  uint16_t* p = a.out + (rq.row0 + t) * a.out_row + (row - t * a.q_heads) * a.out_head + D / 16 * li;
  join_rows<D, F16, WAVES>(a, parts, lane, wave, first + (lane >> 4) < rows ? p : nullptr, [&](int i) { return at + i; });
}

// Behind attend_wide_kernel: rows of a key head; those of whole units are already written.
template <int D, bool F16, int WAVES>
__global__ __launch_bounds__(join_threads(WAVES)) void join_wide_kernel(Attend a) {
  const int lane = threadIdx.x & 63, li = lane & 15, wave = uniform(static_cast<int>(threadIdx.x >> 6));
  int64_t u = join_quad<WAVES>(wave);
  const int quads = (a.max_tokens * a.group + 3) >> 2;
  const int first = static_cast<int>(u % quads) * 4;
  u /= quads;
  const int kh = static_cast<int>(u % a.kv_heads), b = static_cast<int>(u / a.kv_heads);
  if (b >= a.requests) return;
  const Request rq = request(a, b);
  const int rows = rq.tokens * a.group;
  if (first >= rows) return;
  const Groups g = groups_of(a, rq);
  const int64_t total = a.sums[a.requests - 1];
  const int n = shares_of(total), rg = first / kGroup;
  // the unit's first and last tile, and their shares: the largest that begin by then
  const int64_t s = (b ? a.sums[b - 1] : 0) + kh * g.per_head +
                    rg * (static_cast<int64_t>(kFull) * g.tiles + kUnit) + kUnit;
  const int64_t e = s + static_cast<int64_t>(g.tiles - 1) * (rg == g.n - 1 ? g.last : kFull);
  auto share = [&](int64_t at) {
    int k = static_cast<int>(at * n / total);
    while (k + 1 < n && share_begin(total, k + 1, n) <= at) ++k;
    return k;
  };
  const int g0 = share(s), g1 = share(e);
  if (g0 == g1) return;
  const int row = min(first + (lane >> 4), rows - 1), t = row / a.group;
  uint16_t* p = a.out + (rq.row0 + t) * a.out_row + (kh * a.group + row - t * a.group) * a.out_head + D / 16 * li;
  join_rows<D, F16, WAVES>(a, g1 - g0 + 1, lane, wave, first + (lane >> 4) < rows ? p : nullptr,
                    [&](int i) { return static_cast<int64_t>(2 * (g0 + i) + (i == 0) - rg) * kGroup + row; });
}

// The launch shape, a function of sizes the host knows (never of what the device
// arrays hold, so that a captured call replays with other lengths).
// Measured, microseconds, 16 query heads on two key heads of 128 dims:
// - Rows share tiles through LDS (wide) if they are more than 64, or more than 32 and the
//   cache's part is large; wide/else at 64 rows: 32 requests x 4096 keys 43.7/54.0, but
//   4 x 16384 33.6/29.3, 64 x 1024 34.8/29.6, 8 x 512 24/16.6 (its shares and joins cost
//   some 20 whatever the sizes), at 32 rows 32 x 4096 41.5/34.2.
// - Eight waves a workgroup if there is at most one workgroup per CU; eight/four: 4 requests
//   x 512 keys 11.1/12.2, 64 x 512 12.6/13.6, 32 x 2048 20.4/21.3, one of 32768 16.8/17.6,
//   but 64 x 2048 31.0/30.3, 256 x 512 27.6/26.7.  64 dims: 8 x 1024 of 32 rows 12.8/14.1.
//   Not for more than 16 rows of 128 dims, whose sums from eight waves take too much LDS:
//   24.2/13.8 at 8 x 512.
// - Parts of eight steps while parts of sixteen would leave half of the CUs idle; eight/sixteen:
//   one request of 1024 keys 12.3/13.3, of 8192 13.1/14.6, 8 x 1024 12.6/13.8, but 128 x 512
//   20.4/16.9, 8 x 4000 of 64 rows 24.7/22.3; of four 12.0, 13.2, 12.2, 24.4 and 33.9.  Below 32
//   steps the join costs more than two parts gain: 512 keys 11.6/10.8.
struct Plan {
  bool wide;
  int r, wr;   // else row tiles per wave, waves per key slice
  int waves;   // of a workgroup
  int splits, min_steps;  // of the keys, as parts_of takes them
};
Plan plan(int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens,
          int64_t max_context) {
  const int64_t rows = max_tokens * (q_heads / kv_heads), units = requests * kv_heads;
  Plan p{};
  p.wide = rows > 64 || (rows > 32 && units * max_context >= (24 << 20) / head_dim);
  p.splits = 1;
  if (p.wide) return p;
  p.r = rows <= 16 ? 1 : 2;
  p.wr = rows <= 32 ? 1 : 2;
  const int64_t steps = ((max_context + 31) / 32 + (max_tokens + 31) / 32) * p.wr;
  p.min_steps = units * (steps / kCoarseSteps) <= 128 ? kFineSteps : kCoarseSteps;
  if (steps >= kWholeSteps)
    p.splits = static_cast<int>(std::min<int64_t>({(1024 + units - 1) / units, steps / p.min_steps, 256}));
  p.waves = (p.r == 1 || head_dim == 64) && units * p.splits <= 256 ? 8 : 4;
  return p;
}

int64_t slots_of(const Plan& p, int64_t rows, int64_t q_heads) {
  return p.wide ? int64_t{2} * kShares * kGroup : p.splits == 1 ? 0 : rows * q_heads * p.splits;
}
size_t workspace_bytes(const Plan& p, int64_t rows, int64_t requests, int64_t q_heads, int64_t head_dim) {
  return static_cast<size_t>(slots_of(p, rows, q_heads)) * (head_dim + 2) * 4 + (p.wide ? 8 * requests : 0);
}

bool sizes_ok(int64_t rows, int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens,
              int64_t max_context) {
  return rows >= 0 && rows <= 0x7fffffff / 64 && requests >= 0 && requests <= 0x100000 && kv_heads >= 1 &&
         q_heads >= kv_heads && q_heads % kv_heads == 0 && q_heads <= 4096 && (head_dim == 64 || head_dim == 128) &&
         max_tokens >= 1 && max_tokens <= kMaxTree && max_context >= 0 && max_context <= 0x7fffffff &&
         requests * max_tokens * q_heads <= 0x3fffffff;  // (grids are 32-bit)
}

template <int D, bool F16>
int launch_wide(const Attend& a, hipStream_t st) {
  hipLaunchKernelGGL((attend_wide_kernel<D, F16>), dim3(kShares), dim3(64 * kWideWaves), 0, st, a);
  if (int rc = check_launch("tree attention kernel")) return rc;
  const int64_t quads = static_cast<int64_t>(a.requests) * a.kv_heads * ((a.max_tokens * a.group + 3) / 4);
  const int64_t units = static_cast<int64_t>(a.requests) * a.kv_heads * ((a.max_tokens * a.group + kGroup - 1) / kGroup);
  if (join_by_many(kShares / units, quads))
    hipLaunchKernelGGL((join_wide_kernel<D, F16, kJoinWaves>), dim3(static_cast<unsigned>(quads)),
                       dim3(join_threads(kJoinWaves)), 0, st, a);
  else
    hipLaunchKernelGGL((join_wide_kernel<D, F16, 1>), dim3(static_cast<unsigned>((quads + 3) / 4)), dim3(join_threads(1)),
                       0, st, a);
  return check_launch("tree attention join kernel");
}

// (variants that no plan has are not built)
template <int D, bool F16>
void launch_direct(const Attend& a, const Plan& p, hipStream_t st) {
  const dim3 g(static_cast<unsigned>(a.requests * a.kv_heads * p.splits)), blk(64 * p.waves);
  auto go = [&](auto r, auto wr, auto waves) {
    hipLaunchKernelGGL((attend_kernel<D, decltype(r)::value, decltype(wr)::value, decltype(waves)::value, F16>), g, blk, 0,
                       st, a);
  };
  if (p.waves == 8 && p.r == 1) return go(Int<1>{}, Int<1>{}, Int<8>{});
  if constexpr (D == 64) {
    if (p.waves == 8 && p.wr == 1) return go(Int<2>{}, Int<1>{}, Int<8>{});
    if (p.waves == 8) return go(Int<2>{}, Int<2>{}, Int<8>{});
  }
  if (p.r == 1) go(Int<1>{}, Int<1>{}, Int<4>{});
  else if (p.wr == 1) go(Int<2>{}, Int<1>{}, Int<4>{});
  else go(Int<2>{}, Int<2>{}, Int<4>{});
}

template <int D, bool F16>
int launch(const Attend& a, const Plan& p, hipStream_t st) {
  if (p.wide) return launch_wide<D, F16>(a, st);
  launch_direct<D, F16>(a, p, st);
  if (int rc = check_launch("tree attention kernel")) return rc;
  if (p.splits == 1) return PGS_OK;
  const int64_t quads = static_cast<int64_t>(a.requests) * ((a.max_tokens * a.q_heads + 3) / 4);
  if (join_by_many(p.splits, quads))
    hipLaunchKernelGGL((join_kernel<D, F16, kJoinWaves>), dim3(static_cast<unsigned>(quads)),
                       dim3(join_threads(kJoinWaves)), 0, st, a, p.wr);
  else
    hipLaunchKernelGGL((join_kernel<D, F16, 1>), dim3(static_cast<unsigned>((quads + 3) / 4)), dim3(join_threads(1)), 0,
                       st, a, p.wr);
  return check_launch("tree attention join kernel");
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" size_t pgs_tree_attention_workspace_bytes(int64_t rows, int64_t requests, int64_t q_heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t max_tokens, int64_t max_context) {
  if (!sizes_ok(rows, requests, q_heads, kv_heads, head_dim, max_tokens, max_context) || rows == 0 || requests == 0)
    return 0;
  const Plan p = plan(requests, q_heads, kv_heads, head_dim, max_tokens, max_context);
  return workspace_bytes(p, rows, requests, q_heads, head_dim);
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
  // (a tile behind the last token still has a 32-bit number)
  if (g.columns < 0 || g.table_stride < g.columns || g.columns > 0x7fff0000 / c.block_size)
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
  const Plan p = plan(g.requests, g.q_heads, c.kv_heads, c.head_dim, g.max_tokens, g.max_context);
  const size_t need = workspace_bytes(p, g.rows, g.requests, g.q_heads, c.head_dim);
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
  a.bs_inv = static_cast<uint32_t>(((uint64_t{1} << 32) + a.bs - 1) / a.bs);
  a.tables = g.block_tables, a.tstride = g.table_stride, a.cols = static_cast<int32_t>(g.columns);
  a.lens = g.lens, a.offsets = g.offsets, a.parents = g.parents;
  a.rows = static_cast<int32_t>(g.rows), a.requests = static_cast<int32_t>(g.requests);
  a.q_heads = static_cast<int32_t>(g.q_heads), a.kv_heads = static_cast<int32_t>(c.kv_heads);
  a.group = a.q_heads / a.kv_heads;
  a.max_tokens = static_cast<int32_t>(g.max_tokens), a.splits = p.splits, a.min_steps = p.min_steps;
  a.c = g.scale * 1.44269504088896340736f;
  a.part = static_cast<float*>(workspace);
  a.stat = a.part + slots_of(p, g.rows, g.q_heads) * c.head_dim;
  a.sums = reinterpret_cast<int64_t*>(a.stat + slots_of(p, g.rows, g.q_heads) * 2);
  if (c.head_dim == 64)
    return g.dtype == PGS_DTYPE_F16 ? launch<64, true>(a, p, st) : launch<64, false>(a, p, st);
  return g.dtype == PGS_DTYPE_F16 ? launch<128, true>(a, p, st) : launch<128, false>(a, p, st);
}
