// The paged cache's bookkeeping on the device: block tables extended and
// shortened by request lengths, the slot of every row, and rows stored at their
// slots (the reference does these in Python, one token at a time:
// engine/block_allocator.py:13-34, engine/paged_attention.py:62-79).
//
// Request b with len tokens cached and `add` to come, blocks of s tokens:
//   have = ceil(len / s), want = ceil((len + add) / s), need = want - have
//   upto_b = sum of the needs of requests 0 .. b (those whose table has the columns)
// It is served if need = 0 or upto_b <= the free count, so the served needs are a
// prefix; entry e = (upto_b - need) + j of them takes free[count - 1 - e].
#include <algorithm>

#include "pgs_linear.h"

namespace pgs {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kRowThreads = 256;
constexpr int kMaxRequests = 4096;  // per call: their prefix sums lie in LDS

// Inclusive prefix sum of v over the workgroup, plus `carry`; carry becomes the
// running total.  Every thread must call it.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& carry, int64_t (&wsum)[kScanThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  if (lane == 63) wsum[wave] = v;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kScanThreads / 64; ++w) {
    if (w < wave) before += wsum[w];
    total += wsum[w];
  }
  __syncthreads();  // (wsum is written again by the next call)
  v += before + carry;
  carry += total;
  return v;
}

// Number of entries of a[0 .. n) that are <= v (a does not decrease).
template <typename T>
__device__ __forceinline__ int upper_bound(const T* a, int n, T v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

struct Tables {
  int32_t* lens;
  int32_t* tables;
  int64_t stride;
  int cols;
  int32_t* free;
  int cap;
  int32_t* count;
  int bs;
  int requests;
};

struct Rows {
  const int32_t* offsets;
  const int32_t* index;  // or null
  int64_t rows;
  int64_t* slots;
};

// Bound by latency: 4.4 us for 8 requests, of which a launch without work is 2.5.
// One workgroup: the prefix sums, the table entries, and with ROWS the slots too
// (their blocks read from the free list where the table entry is new, so nothing
// waits for a write).
template <bool ROWS>
__global__ __launch_bounds__(kScanThreads) void append_kernel(Tables t, const int32_t* __restrict__ add, Rows rw,
                                                              int32_t* __restrict__ status) {
  extern __shared__ int32_t lds[];
  int32_t* start = lds;                   // entry number of the request's first new block
  int32_t* old = lds + t.requests;        // its length before, or -1 if it is not served
  int32_t* offs = lds + 2 * t.requests;   // (ROWS) the end of its rows
  __shared__ int64_t wsum[kScanThreads / 64];
  __shared__ int32_t used_s;
  const int c0 = min(max(*t.count, 0), t.cap);
  if (threadIdx.x == 0) used_s = 0;
  int64_t carry = 0;
  for (int b0 = 0; b0 < t.requests; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    int64_t len = 0, more = 0, need = 0;
    bool fits = false;
    if (b < t.requests) {
      len = t.lens[b];
      more = max(add[b], 0);
      const int64_t want = (len + more + t.bs - 1) / t.bs;
      fits = len >= 0 && want <= t.cols && len + more <= 0x7fffffff;
      need = fits ? want - (len + t.bs - 1) / t.bs : 0;
    }
    const int64_t upto = block_scan(need, carry, wsum);
    if (b < t.requests) {
      const bool served = fits && (need == 0 || upto <= c0);
      status[b] = served ? 0 : fits ? 1 : 2;
      // (an unserved request's start only has to keep the order: past every entry)
      start[b] = static_cast<int32_t>(min<int64_t>(upto - need, 0x7fffffff));
      old[b] = served ? static_cast<int32_t>(len) : -1;
      if constexpr (ROWS) offs[b] = rw.offsets[b + 1];
      if (served) {
        t.lens[b] = static_cast<int32_t>(len + more);
        if (need > 0) atomicMax(&used_s, static_cast<int32_t>(upto));
      }
    }
  }
  __syncthreads();
  const int used = used_s;
  for (int e = threadIdx.x; e < used; e += kScanThreads) {
    const int b = upper_bound(start, t.requests, e) - 1;
    const int col = static_cast<int>((static_cast<int64_t>(old[b]) + t.bs - 1) / t.bs) + e - start[b];
    t.tables[b * t.stride + col] = t.free[c0 - 1 - e];
  }
  if (threadIdx.x == 0) *t.count = c0 - used;
  if constexpr (ROWS) {
    for (int64_t i = threadIdx.x; i < rw.rows; i += kScanThreads) {
      const int b = upper_bound(offs, t.requests, static_cast<int32_t>(min<int64_t>(i, 0x7fffffff)));
      int64_t slot = -1;
      if (b < t.requests && old[b] >= 0) {
        const int64_t first = b ? offs[b - 1] : rw.offsets[0];
        const int64_t n = rw.index ? rw.index[i] : i - first;
        if (i >= first && n >= 0 && n < max(add[b], 0)) {
          const int64_t pos = old[b] + n;
          const int64_t blk = pos / t.bs, have = (static_cast<int64_t>(old[b]) + t.bs - 1) / t.bs;
          // (new_lens is read again here: whatever it holds by now, no entry that was not taken)
          const int64_t e = start[b] + blk - have;
          const int32_t id = blk < have ? t.tables[b * t.stride + blk] : e < used ? t.free[c0 - 1 - e] : -1;
          if (id >= 0) slot = static_cast<int64_t>(id) * t.bs + pos % t.bs;
        }
      }
      rw.slots[i] = slot;
    }
  }
}

// The slots alone, behind append_kernel<false>: lens are the new ones.
__global__ __launch_bounds__(kRowThreads) void slots_kernel(Tables t, const int32_t* __restrict__ add, Rows rw,
                                                            const int32_t* __restrict__ status) {
  extern __shared__ int32_t lds[];
  for (int b = threadIdx.x; b < t.requests; b += kRowThreads) lds[b] = rw.offsets[b + 1];
  __syncthreads();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  if (i >= rw.rows) return;
  const int b = upper_bound(lds, t.requests, static_cast<int32_t>(min<int64_t>(i, 0x7fffffff)));
  int64_t slot = -1;
  if (b < t.requests && status[b] == 0) {
    const int64_t first = b ? lds[b - 1] : rw.offsets[0];
    const int64_t n = rw.index ? rw.index[i] : i - first, more = max(add[b], 0);
    if (i >= first && n >= 0 && n < more) {
      const int64_t pos = t.lens[b] - more + n;
      const int32_t id = pos >= 0 ? t.tables[b * t.stride + pos / t.bs] : -1;  // (as in append_kernel)
      if (id >= 0) slot = static_cast<int64_t>(id) * t.bs + pos % t.bs;
    }
  }
  rw.slots[i] = slot;
}

// Shortens requests.  Of the table entries given up (in request order, then column order)
// those that name a block go to the stack, the last one first, so that append's lie where
// it took them from; an entry below 0 names none and is not counted.  Bound by latency:
// append and truncate together 9.9 us for 64 requests of 16 blocks each, 19 for 1000 of 4, 79 of 32.
__global__ __launch_bounds__(kScanThreads) void truncate_kernel(Tables t, const int32_t* __restrict__ keep) {
  extern __shared__ int32_t lds[];
  int32_t* start = lds;
  int32_t* left = lds + t.requests;  // blocks kept
  __shared__ int64_t wsum[kScanThreads / 64];
  const int c0 = min(max(*t.count, 0), t.cap);
  int64_t carry = 0;
  for (int b0 = 0; b0 < t.requests; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    int64_t give = 0;
    if (b < t.requests) {
      const int64_t len = t.lens[b], stay = min<int64_t>(max(keep[b], 0), max<int64_t>(len, 0));
      const int64_t have = min<int64_t>((max<int64_t>(len, 0) + t.bs - 1) / t.bs, t.cols);
      const int64_t l = min<int64_t>((stay + t.bs - 1) / t.bs, have);
      give = have - l;
      left[b] = static_cast<int32_t>(l);
      t.lens[b] = static_cast<int32_t>(stay);
    }
    const int64_t upto = block_scan(give, carry, wsum);
    if (b < t.requests) start[b] = static_cast<int32_t>(min<int64_t>(upto - give, 0x7fffffff));
  }
  __syncthreads();
  // Entries from the last on, U per thread and turn: a wave's are 64 U neighbours, counted by
  // ballots; the waves' counts are in one of two arrays in turn, so that one barrier will do.
  __shared__ int32_t found[2][kScanThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t total = carry;
  int64_t on = c0;  // blocks on the stack
  int turn = 0;
  auto give_back = [&](int64_t f, auto per) {
    constexpr int U = decltype(per)::value;
    int32_t* p[U];
    int32_t id[U];
    int at[U], mine = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = total - 1 - f - ((wave * U + u) * 64 + lane);
      p[u] = nullptr;
      if (e < 0) continue;
      const int b = upper_bound(start, t.requests, static_cast<int32_t>(min<int64_t>(e, 0x7fffffff))) - 1;
      p[u] = t.tables + b * t.stride + left[b] + (e - start[b]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = p[u] ? *p[u] : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned long long m = __ballot(id[u] >= 0);
      at[u] = mine + __popcll(m & ((1ull << lane) - 1));
      mine += __popcll(m);
    }
    if (lane == 0) found[turn][wave] = mine;
    __syncthreads();
    int64_t to = on;
#pragma unroll
    for (int w = 0; w < kScanThreads / 64; ++w) {
      if (w < wave) to += found[turn][w];
      on += found[turn][w];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p[u]) *p[u] = -1;
      if (id[u] >= 0 && to + at[u] < t.cap) t.free[to + at[u]] = id[u];
    }
    turn ^= 1;
  };
  int64_t f = 0;
  for (; total - f > kScanThreads; f += 4 * kScanThreads) give_back(f, Int<4>{});
  if (f < total) give_back(f, Int<1>{});
  if (threadIdx.x == 0) *t.count = static_cast<int32_t>(min<int64_t>(on, t.cap));
}

struct WriteArgs {
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_row, k_head, v_row, v_head;
  uint16_t* kc;
  uint16_t* vc;
  int64_t kc_block, kc_slot, kc_head, vc_block, vc_slot, vc_head;
  int64_t nslots;
  int bs, heads, pieces;  // pieces per head: head_dim / 8 (VEC) or head_dim
  const int64_t* slots;
  int64_t units;          // rows * heads * pieces
};

// One thread per piece (16 bytes, or one element where something is not aligned to
// 16 bytes) of a row of k and the same piece of v.  Memory bound: two reads and two
// writes of a row.  Measured: 8192 rows of two heads of 128 dims 4.4 us, 3.8 TB/s.
template <bool VEC>
__global__ __launch_bounds__(kRowThreads) void write_kv_kernel(WriteArgs a) {
  const int64_t u = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
  if (u >= a.units) return;
  const int per = a.heads * a.pieces;
  const int64_t row = u / per;
  const int in = static_cast<int>(u - row * per), h = in / a.pieces, p = (in - h * a.pieces) * (VEC ? 8 : 1);
  const int64_t slot = a.slots[row];
  const uint16_t* ks = a.k + row * a.k_row + h * a.k_head + p;
  const uint16_t* vs = a.v + row * a.v_row + h * a.v_head + p;
  if (slot < 0 || slot >= a.nslots) return;
  const int64_t b = slot / a.bs, s = slot - b * a.bs;
  uint16_t* kd = a.kc + b * a.kc_block + s * a.kc_slot + h * a.kc_head + p;
  uint16_t* vd = a.vc + b * a.vc_block + s * a.vc_slot + h * a.vc_head + p;
  if constexpr (VEC) {
    const u32x4 x = ld16_stream(ks), y = ld16_stream(vs);
    *reinterpret_cast<u32x4*>(kd) = x;
    *reinterpret_cast<u32x4*>(vd) = y;
  } else {
    *kd = *ks;
    *vd = *vs;
  }
}

int check_tables(const char* fn, const void* lens, const void* more, const void* tables, int64_t stride, int64_t columns,
                 const void* free_blocks, int64_t cap, const void* count, int64_t bs, int64_t requests) {
  if (requests < 0 || columns < 0 || cap < 0 || stride < columns)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: negative size, or table rows that overlap", fn);
  if (bs < 1 || bs > 0x10000) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: block_size=%lld must be 1..65536", fn, (long long)bs);
  if (requests > kMaxRequests)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: %lld requests; at most %d per call", fn, (long long)requests, kMaxRequests);
  if (columns > 0x7fffffff / kMaxRequests || cap > 0x7fffffff)  // (entry numbers are 32-bit)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: too large", fn);
  if (!count || (requests > 0 && (!lens || !more || (columns > 0 && !tables))) || (cap > 0 && !free_blocks))
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(lens, 4) || !aligned(more, 4) || !aligned(tables, 4) || !aligned(free_blocks, 4) || !aligned(count, 4))
    return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  return PGS_OK;
}

}  // namespace
}  // namespace pgs

using namespace pgs;

extern "C" int pgs_append_blocks(int32_t* lens, const int32_t* new_lens, int32_t* block_tables, int64_t table_stride,
                                 int64_t columns, const int32_t* free_blocks, int64_t free_capacity,
                                 int32_t* free_count, int64_t block_size, int64_t requests, const int32_t* offsets,
                                 const int32_t* index, int64_t rows, int64_t* slots, int32_t* status, void* stream) {
  const char* fn = "pgs_append_blocks";
  if (int rc = check_tables(fn, lens, new_lens, block_tables, table_stride, columns, free_blocks, free_capacity,
                            free_count, block_size, requests))
    return rc;
  if (rows < 0 || rows > 0xffffffff - kRowThreads)  // (threads of a launch)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: rows=%lld", fn, (long long)rows);
  if (!offsets || (requests > 0 && !status) || (rows > 0 && !slots)) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(offsets, 4) || !aligned(index, 4) || !aligned(slots, 8) || !aligned(status, 4))
    return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  if (requests == 0 && rows == 0) return PGS_OK;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const Tables t{lens, block_tables, table_stride, static_cast<int>(columns), const_cast<int32_t*>(free_blocks),
                 static_cast<int>(free_capacity), free_count, static_cast<int>(block_size), static_cast<int>(requests)};
  const Rows r{offsets, index, rows, slots};
  const size_t ints = 4 * static_cast<size_t>(requests);
  // One launch while the one workgroup is through the rows sooner than a second launch
  // starts.  Measured with a truncate behind each, microseconds one/two: 64 requests of
  // 256 rows in all 7.4/8.4, 2048 11.7/12.7, 4096 14.4/12.9, 16384 31.2/13.0.
  if (rows <= 2048) {
    hipLaunchKernelGGL(append_kernel<true>, dim3(1), dim3(kScanThreads), 3 * ints, st, t, new_lens, r, status);
    return check_launch("append kernel");
  }
  hipLaunchKernelGGL(append_kernel<false>, dim3(1), dim3(kScanThreads), 2 * ints, st, t, new_lens, r, status);
  if (int rc = check_launch("append kernel")) return rc;
  hipLaunchKernelGGL(slots_kernel, dim3(static_cast<unsigned>((rows + kRowThreads - 1) / kRowThreads)),
                     dim3(kRowThreads), ints, st, t, new_lens, r, status);
  return check_launch("slots kernel");
}

extern "C" int pgs_truncate_blocks(int32_t* lens, const int32_t* keep, int32_t* block_tables, int64_t table_stride,
                                   int64_t columns, int32_t* free_blocks, int64_t free_capacity, int32_t* free_count,
                                   int64_t block_size, int64_t requests, void* stream) {
  const char* fn = "pgs_truncate_blocks";
  if (int rc = check_tables(fn, lens, keep, block_tables, table_stride, columns, free_blocks, free_capacity, free_count,
                            block_size, requests))
    return rc;
  if (requests == 0) return PGS_OK;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  const Tables t{lens, block_tables, table_stride, static_cast<int>(columns), free_blocks,
                 static_cast<int>(free_capacity), free_count, static_cast<int>(block_size), static_cast<int>(requests)};
  hipLaunchKernelGGL(truncate_kernel, dim3(1), dim3(kScanThreads), 8 * static_cast<size_t>(requests), st, t, keep);
  return check_launch("truncate kernel");
}

extern "C" int pgs_write_kv(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                            const pgs_kv_cache* cache, const int64_t* slots, int64_t rows, void* stream) {
  const char* fn = "pgs_write_kv";
  if (!cache) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
  const pgs_kv_cache& c = *cache;
  if (rows < 0 || c.blocks < 0 || c.block_size < 1 || c.kv_heads < 1 || c.head_dim < 1 || k_row < 0 || k_head < 0 ||
      v_row < 0 || v_head < 0 || c.k_block < 0 || c.k_slot < 0 || c.k_head < 0 || c.v_block < 0 || c.v_slot < 0 ||
      c.v_head < 0)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: negative or empty size", fn);
  if (c.block_size > 0x10000 || c.kv_heads > 0x4000 || c.head_dim > 0x4000 || c.blocks > 0x7fffffff)
    return fail(PGS_ERR_INVALID_ARGUMENT, "%s: too large", fn);
  if (rows == 0 || c.blocks == 0) return PGS_OK;
  if (!k || !v || !c.k || !c.v || !slots) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned(k, 2) || !aligned(v, 2) || !aligned(c.k, 2) || !aligned(c.v, 2) || !aligned(slots, 8))
    return fail(PGS_ERR_MISALIGNED, "%s: misaligned", fn);
  const bool vec = (c.head_dim | k_row | k_head | v_row | v_head | c.k_block | c.k_slot | c.k_head | c.v_block |
                    c.v_slot | c.v_head) % 8 == 0 &&
                   aligned(k, 16) && aligned(v, 16) && aligned(c.k, 16) && aligned(c.v, 16);
  const int pieces = static_cast<int>(vec ? c.head_dim / 8 : c.head_dim);
  const int64_t per = c.kv_heads * pieces;
  if (rows > (int64_t{1} << 38) / per) return fail(PGS_ERR_INVALID_ARGUMENT, "%s: too large", fn);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = require_device(fn, st)) return rc;
  WriteArgs a{nullptr, nullptr, k_row, k_head, v_row, v_head,
              static_cast<uint16_t*>(c.k), static_cast<uint16_t*>(c.v), c.k_block, c.k_slot, c.k_head, c.v_block,
              c.v_slot, c.v_head, c.blocks * c.block_size, static_cast<int>(c.block_size),
              static_cast<int>(c.kv_heads), pieces, nullptr, 0};
  // (a launch has fewer than 2^32 threads, and larger counts are cut without an error)
  const int64_t most = (0xffffffff - kRowThreads) / per;  // of 2^28 units a row at most
  for (int64_t row = 0; row < rows; row += most) {
    a.k = static_cast<const uint16_t*>(k) + row * k_row, a.v = static_cast<const uint16_t*>(v) + row * v_row, a.slots = slots + row;
    a.units = std::min(rows - row, most) * per;
    const dim3 grid(static_cast<unsigned>((a.units + kRowThreads - 1) / kRowThreads)), block(kRowThreads);
    if (vec) hipLaunchKernelGGL(write_kv_kernel<true>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(write_kv_kernel<false>, grid, block, 0, st, a);
    if (int rc = check_launch("write_kv kernel")) return rc;
  }
  return PGS_OK;
}
