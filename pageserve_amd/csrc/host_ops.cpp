// Host fast path of the linear entry points for PyTorch callers.
//
// pageserve_amd/quantization.py's linear / linear_group / swiglu (and their
// rms_norm and residual forms) run once per projection per token step; the
// reference calls them through F.linear from a runner thread
// (engine/model.py:168-190, engine/runner.py:79).  This module does their
// argument checks, output allocation, device and stream selection and the
// C-ABI call (include/pageserve_amd.h) in C++, so that an eager call costs a
// few microseconds of host time: the same work in Python with ctypes cost
// 10-20 us per call, more than the decode kernels themselves.  It computes
// nothing itself; every result comes from the gfx950 kernels.  Error
// messages and exception types are those of the Python wrappers (ValueError,
// TypeError, RuntimeError).
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <initializer_list>
#include <string>
#include <vector>

#include "pageserve_amd.h"

namespace {

using Opt = c10::optional<at::Tensor>;

[[noreturn]] void value_error(const std::string& s) { throw pybind11::value_error(s); }
[[noreturn]] void type_error(const std::string& s) { throw pybind11::type_error(s); }

std::string dev_str(const at::Device& d) { return d.str(); }

void check_rc(int rc, const char* what) {
  if (rc == PGS_OK) return;
  std::string msg = std::string(what) + ": " + pgs_error_string(rc) + ": " + pgs_last_error();
  if (rc == PGS_ERR_INVALID_ARGUMENT || rc == PGS_ERR_MISALIGNED) value_error(msg);
  throw std::runtime_error(msg);
}

// contiguous, data pointer aligned to `align` bytes (copies only if needed)
at::Tensor aligned(const at::Tensor& t, uintptr_t align) {
  at::Tensor c = t.is_contiguous() ? t : t.contiguous();
  if (c.numel() && reinterpret_cast<uintptr_t>(c.data_ptr()) % align) c = c.clone();
  return c;
}

void* ptr(const at::Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }

// x: bf16 [..., k] on `dev` -> contiguous 16-byte aligned [m, k]
at::Tensor check_x(const at::Tensor& x, int64_t k, const at::Device& dev, const char* what) {
  if (x.device() != dev)
    value_error(std::string(what) + ": input on " + dev_str(x.device()) + " but weight on " + dev_str(dev));
  if (x.scalar_type() != at::kBFloat16)
    type_error(std::string(what) + ": the W8A16 kernels take bf16 activations, got " +
               std::string(c10::toString(x.scalar_type())));
  if (x.dim() < 1 || x.size(-1) != k)
    value_error(std::string(what) + ": input has " + std::to_string(x.dim() ? x.size(-1) : 0) +
                " features, weight expects " + std::to_string(k));
  // (a 2-D input is used as it is: each view op costs a few hundred ns of
  // host time per call)
  return aligned(x.dim() == 2 ? x : x.reshape({-1, k}), 16);
}

std::vector<int64_t> out_shape(const at::Tensor& x, int64_t n) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end() - 1);
  s.push_back(n);
  return s;
}

at::Tensor check_bias(const Opt& b, int64_t n, const at::Device& dev, const char* what) {
  if (!b.has_value() || !b->defined()) return at::Tensor();
  const at::Tensor& t = *b;
  if (t.device() != dev || t.scalar_type() != at::kBFloat16 || t.numel() != n)
    value_error(std::string(what) + ": bias must be a bf16 [" + std::to_string(n) + "] tensor on " + dev_str(dev));
  return aligned(t.dim() == 1 ? t : t.reshape({n}), 2);
}

at::Tensor check_norm(const Opt& w, int64_t k, const at::Device& dev, const char* what) {
  const at::Tensor& t = *w;
  if (t.scalar_type() != at::kBFloat16 || t.numel() != k || t.device() != dev)
    value_error(std::string(what) + ": norm weight must be a bf16 [" + std::to_string(k) + "] tensor on " +
                dev_str(dev));
  return aligned(t.reshape({k}), 16);
}

// RoPE of a q|k|v call's first two outputs: cos / sin bf16 [m, head_dim].
struct Rope {
  at::Tensor cos, sin;
  int64_t head_dim = 0;
};

// One or more projections of the same input (linear, linear_group, and with
// a single member the residual / out forms; norm_w: rms_norm fused in front;
// rope: with norm_w and three members, RoPE behind the first two).
std::vector<at::Tensor> linear_impl(const at::Tensor& x, const std::vector<at::Tensor>& qps,
                                    const std::vector<at::Tensor>& scales, const std::vector<Opt>& biases,
                                    const std::vector<int64_t>& ns, int64_t k, bool out_f32, const Opt& residual,
                                    const Opt& out, const Opt& norm_w, double eps, int64_t ws_ptr, int64_t ws_bytes,
                                    const Rope* rope) {
  const size_t g = qps.size();
  if (g < 1 || g > PGS_MAX_GROUP || scales.size() != g || biases.size() != g || ns.size() != g)
    value_error("linear_group takes 1.." + std::to_string(PGS_MAX_GROUP) + " weights");
  const at::Device dev = qps[0].device();
  const char* what = "linear";
  at::Tensor x2 = check_x(x, k, dev, what);
  const int64_t m = x2.size(0);
  at::Tensor nw;
  if (norm_w.has_value()) nw = check_norm(norm_w, k, dev, "rmsnorm_linear_group");
  const auto odt = out_f32 ? at::kFloat : at::kBFloat16;
  pgs_linear_out outs[PGS_MAX_GROUP];
  std::vector<at::Tensor> ys;
  ys.reserve(g);
  at::Tensor bias_keep[PGS_MAX_GROUP];
  at::Tensor res;
  // a group's outputs are contiguous pieces of one allocation (one call into
  // the caching allocator instead of one per member), each starting on a
  // 64-element boundary (the kernels' vector stores want aligned rows)
  auto piece = [&](size_t i) { return (m * ns[i] + 63) / 64 * 64; };
  at::Tensor flat;
  if (g > 1) {
    int64_t total = 0;
    for (size_t i = 0; i < g; ++i) total += piece(i);
    flat = at::empty({total}, x2.options().dtype(odt));
  }
  int64_t off = 0;
  for (size_t i = 0; i < g; ++i) {
    const int64_t n = ns[i];
    bias_keep[i] = check_bias(biases[i], n, dev, what);
    at::Tensor y;
    if (g > 1) {
      y = flat.as_strided({m, n}, {n, 1}, off);  // (a fresh allocation: storage offset 0)
      off += piece(i);
    } else if (out.has_value()) {
      const at::Tensor& o = *out;
      if (o.device() != dev || o.scalar_type() != odt || o.numel() != m * n || !o.is_contiguous())
        value_error("linear: out must be a contiguous " + std::string(c10::toString(odt)) + " tensor of " +
                    std::to_string(m * n) + " elements on " + dev_str(dev));
      y = o.view({m, n});
    } else {
      y = at::empty({m, n}, x2.options().dtype(odt));
    }
    outs[i] = pgs_linear_out{static_cast<const int8_t*>(ptr(qps[i])), static_cast<const float*>(ptr(scales[i])),
                             bias_keep[i].defined() ? bias_keep[i].data_ptr() : nullptr, ptr(y), n};
    ys.push_back(y);
  }
  if (residual.has_value()) {
    const at::Tensor& r = *residual;
    const int64_t n = ns[0];
    if (r.device() != dev || r.scalar_type() != at::kBFloat16 || r.dim() < 1 || r.size(-1) != n || r.numel() != m * n)
      value_error("linear: residual must be a bf16 [..., " + std::to_string(n) + "] tensor with " + std::to_string(m) +
                  " rows on " + dev_str(dev));
    res = r.reshape({m, n});
    if (!res.is_contiguous()) res = res.contiguous();
  }
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  void* ws = reinterpret_cast<void*>(static_cast<uintptr_t>(ws_ptr));
  const int ydt = out_f32 ? PGS_DTYPE_F32 : PGS_DTYPE_BF16;
  int rc;
  if (rope)
    rc = pgs_w8a16_rmsnorm_qkv_rope(ptr(x2), nw.data_ptr(), static_cast<float>(eps), outs, ptr(rope->cos),
                                    ptr(rope->sin), rope->head_dim, m, k, ws, static_cast<size_t>(ws_bytes), st);
  else if (nw.defined())
    rc = pgs_w8a16_rmsnorm_linear_group(ptr(x2), nw.data_ptr(), static_cast<float>(eps), outs, static_cast<int>(g), ydt,
                                        m, k, ws, static_cast<size_t>(ws_bytes), st);
  else if (res.defined() || out.has_value())
    rc = pgs_w8a16_linear_residual(ptr(x2), outs[0].qp, outs[0].scale, outs[0].bias, res.defined() ? ptr(res) : nullptr,
                                   outs[0].y, ydt, m, ns[0], k, ws, static_cast<size_t>(ws_bytes), st);
  else
    rc = pgs_w8a16_linear_group(ptr(x2), outs, static_cast<int>(g), ydt, m, k, ws, static_cast<size_t>(ws_bytes), st);
  check_rc(rc, "w8a16 linear");
  if (x.dim() != 2)
    for (size_t i = 0; i < g; ++i) ys[i] = ys[i].view(out_shape(x, ns[i]));
  return ys;
}

std::vector<at::Tensor> linear(const at::Tensor& x, const std::vector<at::Tensor>& qps,
                               const std::vector<at::Tensor>& scales, const std::vector<Opt>& biases,
                               const std::vector<int64_t>& ns, int64_t k, bool out_f32, const Opt& residual,
                               const Opt& out, const Opt& norm_w, double eps, int64_t ws_ptr, int64_t ws_bytes) {
  return linear_impl(x, qps, scales, biases, ns, k, out_f32, residual, out, norm_w, eps, ws_ptr, ws_bytes, nullptr);
}

// rms_norm, q|k|v and RoPE of q and k (one launch where the plan allows).
// cos / sin: bf16 [m, head_dim] on the weights' device (checked by the caller).
std::vector<at::Tensor> qkv_rope(const at::Tensor& x, const std::vector<at::Tensor>& qps,
                                 const std::vector<at::Tensor>& scales, const std::vector<Opt>& biases,
                                 const std::vector<int64_t>& ns, int64_t k, const at::Tensor& norm_w, double eps,
                                 const at::Tensor& cos, const at::Tensor& sin, int64_t head_dim, int64_t ws_ptr,
                                 int64_t ws_bytes) {
  if (qps.size() != 3) value_error("qkv_rope takes the q, k and v weights");
  const Rope rope{aligned(cos, 2), aligned(sin, 2), head_dim};
  return linear_impl(x, qps, scales, biases, ns, k, false, c10::nullopt, c10::nullopt, norm_w, eps, ws_ptr, ws_bytes,
                     &rope);
}

// One projection (linear and its residual / out forms): the group path
// without the four one-element lists a Python caller would build.
at::Tensor linear1(const at::Tensor& x, const at::Tensor& qp, const at::Tensor& scale, const Opt& bias, int64_t n,
                   int64_t k, bool out_f32, const Opt& residual, const Opt& out, int64_t ws_ptr, int64_t ws_bytes) {
  return linear(x, {qp}, {scale}, {bias}, {n}, k, out_f32, residual, out, c10::nullopt, 0.0, ws_ptr, ws_bytes)[0];
}

// gate / up / silu(gate) * up in one launch (norm_w: rms_norm fused in front)
at::Tensor swiglu(const at::Tensor& x, const at::Tensor& qg, const at::Tensor& sg, const at::Tensor& qu,
                  const at::Tensor& su, int64_t n, int64_t k, const Opt& norm_w, double eps, int64_t ws_ptr,
                  int64_t ws_bytes) {
  const at::Device dev = qg.device();
  at::Tensor x2 = check_x(x, k, dev, "swiglu");
  const int64_t m = x2.size(0);
  at::Tensor nw;
  if (norm_w.has_value()) nw = check_norm(norm_w, k, dev, "rmsnorm_swiglu");
  at::Tensor act = at::empty({m, n}, x2.options());
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  void* ws = reinterpret_cast<void*>(static_cast<uintptr_t>(ws_ptr));
  int rc;
  if (nw.defined())
    rc = pgs_w8a16_rmsnorm_swiglu(ptr(x2), nw.data_ptr(), static_cast<float>(eps), static_cast<const int8_t*>(ptr(qg)),
                                  static_cast<const float*>(ptr(sg)), static_cast<const int8_t*>(ptr(qu)),
                                  static_cast<const float*>(ptr(su)), ptr(act), m, n, k, ws,
                                  static_cast<size_t>(ws_bytes), st);
  else
    rc = pgs_w8a16_swiglu(ptr(x2), static_cast<const int8_t*>(ptr(qg)), static_cast<const float*>(ptr(sg)),
                          static_cast<const int8_t*>(ptr(qu)), static_cast<const float*>(ptr(su)), ptr(act), m, n, k,
                          ws, static_cast<size_t>(ws_bytes), st);
  check_rc(rc, "w8a16 swiglu");
  return x.dim() == 2 ? act : act.view(out_shape(x, n));
}

// ---------------------------------------------------------------------------
// 4-bit weights (pageserve_amd/quantization4.py)
// ---------------------------------------------------------------------------

// (codes, scales) of an fp32 or bf16 weight on a GPU, packed
std::vector<at::Tensor> quantize4(const at::Tensor& w, int64_t group) {
  const at::Device dev = w.device();
  at::Tensor w2 = aligned(w, 16);
  const int64_t n = w2.size(0), k = w2.size(1);
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  at::Tensor qp = at::empty({std::max<int64_t>(pgs_packed4_bytes(n, k), 0)}, w2.options().dtype(at::kByte));
  at::Tensor sp = at::empty({std::max<int64_t>(pgs_packed4_scales(n, k, group), 0)}, w2.options().dtype(at::kBFloat16));
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_rc(pgs_quantize4_packed(ptr(w2), w2.scalar_type() == at::kFloat ? PGS_DTYPE_F32 : PGS_DTYPE_BF16, n, k, group,
                                ptr(qp), ptr(sp), st),
           "quantize4");
  return {qp, sp};
}

at::Tensor dequantize4(const at::Tensor& qp, const at::Tensor& sp, int64_t n, int64_t k, int64_t group, int64_t dtype) {
  const at::Device dev = qp.device();
  const auto t = dtype == PGS_DTYPE_F32 ? at::kFloat : dtype == PGS_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  at::Tensor out = at::empty({n, k}, qp.options().dtype(t));
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_rc(pgs_dequantize4_packed(ptr(qp), ptr(sp), n, k, group, ptr(out), static_cast<int>(dtype), st), "dequantize4");
  return out;
}

// bytes from a tensor's first element to the end of its last
int64_t extent(const at::Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return (last + 1) * t.element_size();
}
// whether the memory of `o` and of `t` can overlap
bool overlap(const at::Tensor& o, const at::Tensor& t) {
  if (!o.numel() || !t.numel()) return false;
  const char *a = static_cast<const char*>(o.data_ptr()), *b = static_cast<const char*>(t.data_ptr());
  return a < b + extent(t) && b < a + extent(o);
}

at::Tensor linear4(const at::Tensor& x, const at::Tensor& qp, const at::Tensor& sp, const Opt& bias, int64_t n,
                   int64_t k, int64_t group, bool out_f32, const Opt& residual, const Opt& out) {
  const at::Device dev = qp.device();
  const char* what = "linear4";
  if (x.device() != dev)
    value_error("linear4: input on " + dev_str(x.device()) + " but weight on " + dev_str(dev));
  if (x.scalar_type() != at::kBFloat16)
    type_error("linear4: the W4A16 kernels take bf16 activations, got " + std::string(c10::toString(x.scalar_type())));
  if (x.dim() < 1 || x.size(-1) != k)
    value_error("linear4: input has " + std::to_string(x.dim() ? x.size(-1) : 0) + " features, weight expects " +
                std::to_string(k));
  int64_t m = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) m *= x.size(i);
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  at::Tensor x2 = aligned(x.dim() == 2 ? x : x.reshape({m, k}), 16);
  at::Tensor b = check_bias(bias, n, dev, what), res, y;
  const auto odt = out_f32 ? at::kFloat : at::kBFloat16;
  if (out.has_value()) {
    const at::Tensor& o = *out;
    if (o.device() != dev || o.scalar_type() != odt || o.numel() != m * n || !o.is_contiguous())
      value_error("linear4: out must be a contiguous " + std::string(c10::toString(odt)) + " tensor of " +
                  std::to_string(m * n) + " elements on " + dev_str(dev));
    if (overlap(o, x2)) value_error("linear4: out must not share memory with the input");
    if ((b.defined() && overlap(o, b)) || overlap(o, qp) || overlap(o, sp))
      value_error("linear4: out must not share memory with the weight or the bias");
    y = o.view({m, n});
  } else {
    y = at::empty({m, n}, x2.options().dtype(odt));
  }
  if (residual.has_value()) {
    const at::Tensor& r = *residual;
    if (r.device() != dev || r.scalar_type() != at::kBFloat16 || r.dim() < 1 || r.size(-1) != n || r.numel() != m * n)
      value_error("linear4: residual must be a bf16 [..., " + std::to_string(n) + "] tensor with " + std::to_string(m) +
                  " rows on " + dev_str(dev));
    res = r.reshape({m, n});
    if (!res.is_contiguous()) res = res.contiguous();
    if (overlap(y, res) && (y.data_ptr() != res.data_ptr() || out_f32))
      value_error("linear4: out may be the residual itself, but not share memory with a part of it");
  }
  const size_t need = pgs_w4a16_workspace_bytes(m, n, k);
  at::Tensor ws;  // (per call, as in tree_attention)
  if (need) ws = at::empty({static_cast<int64_t>(need)}, x2.options().dtype(at::kByte));
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_rc(pgs_w4a16_linear(ptr(x2), ptr(qp), ptr(sp), b.defined() ? ptr(b) : nullptr,
                            res.defined() ? ptr(res) : nullptr, ptr(y), out_f32 ? PGS_DTYPE_F32 : PGS_DTYPE_BF16, m, n, k,
                            group, need ? ws.data_ptr() : nullptr, need, st),
           "w4a16 linear");
  return x.dim() == 2 ? y : y.view(out_shape(x, n));
}

// ---------------------------------------------------------------------------
// the paged cache (pageserve_amd/paged.py)
// ---------------------------------------------------------------------------

void need_gpu(const at::Tensor& t, const char* what, const char* name) {
  if (!t.is_cuda()) throw std::runtime_error(std::string(what) + ": " + name + " must be on a ROCm GPU");
}

// an int32 tensor of `n` elements (any count: -1), contiguous, on dev
const int32_t* ints(const at::Tensor& t, int64_t n, const at::Device& dev, const char* what, const char* name) {
  if (t.device() != dev)
    value_error(std::string(what) + ": " + name + " on " + dev_str(t.device()) + " but the batch is on " + dev_str(dev));
  if (t.scalar_type() != at::kInt) type_error(std::string(what) + ": " + name + " must be int32");
  if (!t.is_contiguous() || (n >= 0 && t.numel() != n))
    value_error(std::string(what) + ": " + name + " must be contiguous" +
                (n >= 0 ? " with " + std::to_string(n) + " elements" : ""));
  return static_cast<const int32_t*>(ptr(t));
}
int32_t* ints_out(const at::Tensor& t, int64_t n, const at::Device& dev, const char* what, const char* name) {
  return const_cast<int32_t*>(ints(t, n, dev, what, name));
}

// block tables: int32 [requests, columns], columns contiguous
int32_t* table(const at::Tensor& t, int64_t requests, const at::Device& dev, const char* what, int64_t& stride) {
  if (t.device() != dev)
    value_error(std::string(what) + ": block_tables on " + dev_str(t.device()) + " but the batch is on " + dev_str(dev));
  if (t.scalar_type() != at::kInt) type_error(std::string(what) + ": block_tables must be int32");
  if (t.dim() != 2 || t.size(0) != requests || (t.size(1) > 1 && t.stride(1) != 1) ||
      (requests > 1 && t.stride(0) < t.size(1)))
    value_error(std::string(what) + ": block_tables must be [" + std::to_string(requests) +
                ", columns] with contiguous rows that do not overlap");
  stride = requests > 1 ? t.stride(0) : t.size(1);
  return static_cast<int32_t*>(ptr(t));
}

// Whether two int32 arrays share an element: rows of `cols` contiguous elements, `stride` apart.
struct Ints {
  const char* name;
  const int32_t* p;
  int64_t rows, cols, stride;
};
bool share(const Ints& a, const Ints& b) {
  if (b.rows > 1) return a.rows > 1 ? share(a, {b.name, b.p, 1, (b.rows - 1) * b.stride + b.cols, 0}) : share(b, a);
  if (!a.rows || !a.cols || !b.rows || !b.cols) return false;
  // b is [d, d + cols) in elements from a's first (everything here is 4-byte aligned)
  const int64_t d = (reinterpret_cast<intptr_t>(b.p) - reinterpret_cast<intptr_t>(a.p)) / 4, end = d + b.cols;
  if (a.rows == 1) return d < a.cols && end > 0;
  const int64_t r = d < 0 ? 0 : std::min(d / a.stride, a.rows - 1);  // the last row that begins by d
  return (d < r * a.stride + a.cols && end > r * a.stride) || (r + 1 < a.rows && end > (r + 1) * a.stride);
}
// `written` share no element with one another nor with `read`
void check_apart(const char* what, std::initializer_list<Ints> written, std::initializer_list<Ints> read) {
  for (const Ints* w = written.begin(); w != written.end(); ++w) {
    for (const Ints* o = w + 1; o != written.end(); ++o)
      if (share(*w, *o)) value_error(std::string(what) + ": " + w->name + " and " + o->name + " must not share memory");
    for (const Ints& r : read)
      if (share(*w, r)) value_error(std::string(what) + ": " + w->name + " and " + r.name + " must not share memory");
  }
}
constexpr int64_t kMaxRequests = 4096;  // (more are refused by the kernels' entry, first)

std::vector<at::Tensor> append_blocks(const at::Tensor& lens, const at::Tensor& new_lens, const at::Tensor& offsets,
                                      const at::Tensor& block_tables, const at::Tensor& free_blocks,
                                      const at::Tensor& free_count, int64_t block_size, int64_t rows, const Opt& index) {
  const char* what = "append_blocks";
  need_gpu(lens, what, "lens");
  const at::Device dev = lens.device();
  const int64_t n = lens.numel();
  int64_t stride = 0;
  int32_t* lp = ints_out(lens, n, dev, what, "lens");
  const int32_t* np = ints(new_lens, n, dev, what, "new_lens");
  const int32_t* op = ints(offsets, n + 1, dev, what, "offsets");
  int32_t* tp = table(block_tables, n, dev, what, stride);
  const int32_t* fp = ints(free_blocks, -1, dev, what, "free_blocks");
  int32_t* cp = ints_out(free_count, 1, dev, what, "free_count");
  if (rows < 0) value_error("append_blocks: rows must not be negative");
  const int32_t* ip = index.has_value() ? ints(*index, rows, dev, what, "index") : nullptr;
  if (n <= kMaxRequests)
    check_apart(what,
                {{"lens", lp, 1, n, 0}, {"block_tables", tp, n, block_tables.size(1), stride}, {"free_count", cp, 1, 1, 0}},
                {{"new_lens", np, 1, n, 0}, {"offsets", op, 1, n + 1, 0}, {"free_blocks", fp, 1, free_blocks.numel(), 0},
                 {"index", ip, 1, ip ? rows : 0, 0}});
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  at::Tensor slots = at::empty({rows}, lens.options().dtype(at::kLong)), status = at::empty({n}, lens.options());
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_rc(pgs_append_blocks(lp, np, tp, stride, block_tables.size(1), fp, free_blocks.numel(), cp, block_size, n, op, ip,
                             rows, static_cast<int64_t*>(ptr(slots)), static_cast<int32_t*>(ptr(status)), st),
           what);
  return {slots, status};
}

void truncate_blocks(const at::Tensor& lens, const at::Tensor& keep, const at::Tensor& block_tables,
                     const at::Tensor& free_blocks, const at::Tensor& free_count, int64_t block_size) {
  const char* what = "truncate_blocks";
  need_gpu(lens, what, "lens");
  const at::Device dev = lens.device();
  const int64_t n = lens.numel();
  int64_t stride = 0;
  int32_t* lp = ints_out(lens, n, dev, what, "lens");
  const int32_t* kp = ints(keep, n, dev, what, "keep");
  int32_t* tp = table(block_tables, n, dev, what, stride);
  int32_t* fp = ints_out(free_blocks, -1, dev, what, "free_blocks");
  int32_t* cp = ints_out(free_count, 1, dev, what, "free_count");
  if (n <= kMaxRequests)  // (keep may be lens itself: nothing to shorten)
    check_apart(what,
                {{"lens", lp, 1, n, 0}, {"block_tables", tp, n, block_tables.size(1), stride},
                 {"free_blocks", fp, 1, free_blocks.numel(), 0}, {"free_count", cp, 1, 1, 0}},
                {{"keep", kp, 1, kp == lp ? 0 : n, 0}});
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_rc(pgs_truncate_blocks(lp, kp, tp, stride, block_tables.size(1), fp, free_blocks.numel(), cp, block_size, n, st),
           what);
}

int code_of(const at::Tensor& t, const char* what) {
  if (t.scalar_type() == at::kBFloat16) return PGS_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return PGS_DTYPE_F16;
  type_error(std::string(what) + ": tensors must be bf16 or fp16, got " + std::string(c10::toString(t.scalar_type())));
}

// the step of dimension d (0 where it has one index: never multiplied by another)
int64_t step(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// k and v caches [blocks, block_size, kv_heads, head_dim] of one dtype on one device
pgs_kv_cache check_cache(const at::Tensor& kc, const at::Tensor& vc, const char* what) {
  for (const at::Tensor* t : {&kc, &vc}) {
    need_gpu(*t, what, "the cache");
    if (t->dim() != 4 || (t->size(3) > 1 && t->stride(3) != 1))
      value_error(std::string(what) + ": k_cache and v_cache must be (blocks, block_size, kv_heads, head_dim) with a "
                                      "contiguous head_dim");
  }
  if (kc.sizes() != vc.sizes() || kc.scalar_type() != vc.scalar_type() || kc.device() != vc.device())
    value_error(std::string(what) + ": k_cache and v_cache must agree in shape, dtype and device");
  return pgs_kv_cache{ptr(kc), ptr(vc), kc.size(0), kc.size(1), kc.size(2), kc.size(3), step(kc, 0), step(kc, 1),
                      step(kc, 2), step(vc, 0), step(vc, 1), step(vc, 2)};
}

// rows [rows, heads, head_dim] of the cache's dtype, head_dim contiguous
at::Tensor check_rows(const at::Tensor& t, int64_t rows, int64_t heads, const at::Tensor& kc, const char* what,
                      const char* name) {
  if (t.device() != kc.device())
    value_error(std::string(what) + ": " + name + " on " + dev_str(t.device()) + " but the cache is on " +
                dev_str(kc.device()));
  if (t.scalar_type() != kc.scalar_type())
    type_error(std::string(what) + ": " + name + " must have the cache's dtype");
  if (t.dim() != 3 || t.size(0) != rows || (heads >= 0 && t.size(1) != heads) || t.size(2) != kc.size(3))
    value_error(std::string(what) + ": " + name + " must be (" + std::to_string(rows) + ", " +
                (heads >= 0 ? std::to_string(heads) : std::string("heads")) + ", " + std::to_string(kc.size(3)) + ")");
  return t.size(2) > 1 && t.stride(2) != 1 ? t.contiguous() : t;
}

// every element of a cache that is written has a place of its own: each step is past all
// that the smaller ones span
void check_places(const at::Tensor& c, const char* what, const char* name) {
  std::array<int64_t, 4> order{0, 1, 2, 3};
  std::sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return c.stride(a) < c.stride(b); });
  int64_t span = 1;
  for (int64_t d : order) {
    if (c.size(d) < 2) continue;
    if (c.stride(d) < span)
      value_error(std::string(what) + ": " + name + " must not overlap itself (strides of its dimensions)");
    span += (c.size(d) - 1) * c.stride(d);
  }
}

void write_kv(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
              const at::Tensor& slots) {
  const char* what = "write_kv";
  const pgs_kv_cache c = check_cache(k_cache, v_cache, what);
  code_of(k_cache, what);
  const int64_t rows = slots.numel();
  const at::Device dev = k_cache.device();
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  at::Tensor kr = check_rows(k, rows, c.kv_heads, k_cache, what, "k");
  at::Tensor vr = check_rows(v, rows, c.kv_heads, k_cache, what, "v");
  check_places(k_cache, what, "k_cache");
  check_places(v_cache, what, "v_cache");
  // rows of the cache itself (moved to other slots) are read before any is written
  if (overlap(kr, k_cache) || overlap(kr, v_cache)) kr = kr.clone();
  if (overlap(vr, k_cache) || overlap(vr, v_cache)) vr = vr.clone();
  if (slots.device() != dev)
    value_error("write_kv: slots on " + dev_str(slots.device()) + " but the cache is on " + dev_str(dev));
  if (slots.scalar_type() != at::kLong) type_error("write_kv: slots must be int64");
  if (!slots.is_contiguous()) value_error("write_kv: slots must be contiguous");
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_rc(pgs_write_kv(ptr(kr), step(kr, 0), step(kr, 1), ptr(vr), step(vr, 0), step(vr, 1), &c,
                        static_cast<const int64_t*>(ptr(slots)), rows, st),
           what);
}

// rows usable by 16-byte accesses as they are, else a contiguous copy
at::Tensor pieces(const at::Tensor& t) {
  const bool ok = step(t, 0) % 8 == 0 && step(t, 1) % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                          const at::Tensor& v_cache, const at::Tensor& block_tables, const at::Tensor& lens,
                          const at::Tensor& offsets, const Opt& parents, int64_t max_tokens, int64_t max_context,
                          const c10::optional<double>& scale, const Opt& out) {
  const char* what = "tree_attention";
  const pgs_kv_cache c = check_cache(k_cache, v_cache, what);
  pgs_tree_attention_args a{};
  a.dtype = code_of(k_cache, what);
  const at::Device dev = k_cache.device();
  at::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  if (q.dim() != 3) value_error("tree_attention: q must be (rows, q_heads, head_dim)");
  a.rows = q.size(0);
  a.q_heads = q.size(1);
  at::Tensor qr = pieces(check_rows(q, a.rows, -1, k_cache, what, "q"));
  at::Tensor kr = pieces(check_rows(k, a.rows, c.kv_heads, k_cache, what, "k"));
  at::Tensor vr = pieces(check_rows(v, a.rows, c.kv_heads, k_cache, what, "v"));
  a.requests = lens.numel();
  a.lens = ints(lens, a.requests, dev, what, "lens");
  a.offsets = ints(offsets, a.requests + 1, dev, what, "offsets");
  if (parents.has_value()) {
    a.parents = ints(*parents, a.rows, dev, what, "parents");
  }
  a.block_tables = table(block_tables, a.requests, dev, what, a.table_stride);
  a.columns = block_tables.size(1);
  at::Tensor o;
  if (out.has_value()) {
    o = *out;
    if (o.device() != dev || o.scalar_type() != k_cache.scalar_type() || o.sizes() != q.sizes() || !o.is_contiguous() ||
        reinterpret_cast<uintptr_t>(o.data_ptr()) % 16)
      value_error("tree_attention: out must be a contiguous 16-byte aligned tensor of q's shape, dtype and device");
    if (overlap(o, qr) && (o.data_ptr() != qr.data_ptr() || !qr.is_contiguous()))
      value_error("tree_attention: out may be q itself, but not share memory with a part of it");
    if (overlap(o, kr) || overlap(o, vr) || overlap(o, k_cache) || overlap(o, v_cache))
      value_error("tree_attention: out must not share memory with k, v or the cache");
  } else {
    o = at::empty(q.sizes(), k_cache.options());
  }
  a.q = ptr(qr), a.k = ptr(kr), a.v = ptr(vr), a.out = ptr(o);
  a.q_row = step(qr, 0), a.q_head = step(qr, 1);
  a.k_row = step(kr, 0), a.k_head = step(kr, 1);
  a.v_row = step(vr, 0), a.v_head = step(vr, 1);
  a.out_row = step(o, 0), a.out_head = step(o, 1);
  a.cache = &c;
  // No request has more rows than the batch, and the kernels are chosen by the bound: plain
  // decoding with the default of 64 is planned as what it is.  Microseconds with the bound at 64
  // and cut, 16 heads on two key heads of 128 dims: one token of 100 keys 16.8 and 8.0, of 2000
  // 19.0 and 12.5, of eight requests of 2000 20.9 and 13.0.  (A bound out of range is refused below.)
  a.max_tokens = max_tokens <= 64 ? std::min(max_tokens, std::max<int64_t>(a.rows, 1)) : max_tokens;
  a.max_context = max_context >= 0 ? max_context : a.columns * c.block_size;
  a.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(c.head_dim)));
  const size_t need = pgs_tree_attention_workspace_bytes(a.rows, a.requests, a.q_heads, c.kv_heads, c.head_dim,
                                                         a.max_tokens, a.max_context);
  // (a fresh workspace per call, from torch's caching allocator: ordered on this
  // stream, and inside a capture the graph's own)
  at::Tensor ws;
  if (need) ws = at::empty({static_cast<int64_t>(need)}, k_cache.options().dtype(at::kByte));
  void* st = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_rc(pgs_tree_attention(&a, need ? ws.data_ptr() : nullptr, need, st), what);
  return o;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  mod.doc() = "C++ host path of pageserve_amd's linear entry points (calls the gfx950 C ABI)";
  mod.def("abi_version", &pgs_abi_version);
  mod.def("linear", &linear, "one or more W8A16 projections of the same input");
  mod.def("linear1", &linear1, "one W8A16 projection");
  mod.def("qkv_rope", &qkv_rope, "rms_norm, q|k|v projections and RoPE of q and k");
  mod.def("swiglu", &swiglu, "fused gate/up/silu*up");
  mod.def("quantize4", &quantize4, "4-bit codes and group scales of a weight, packed");
  mod.def("dequantize4", &dequantize4, "the dense weight of packed 4-bit codes");
  mod.def("linear4", &linear4, "one W4A16 projection");
  mod.def("append_blocks", &append_blocks, "block tables extended, slots of the new rows");
  mod.def("truncate_blocks", &truncate_blocks, "requests shortened, their blocks given back");
  mod.def("write_kv", &write_kv, "key and value rows stored at their slots");
  mod.def("tree_attention", &tree_attention, "attention of drafted tokens over a paged cache");
}
