/*
 * pageserve_amd: C ABI of the MI355X (gfx950) INT8 weight-only linear path.
 *
 * Every entry point takes plain device pointers, element counts and an opaque
 * hipStream_t (passed as void*; NULL means the default stream).  All launches
 * are asynchronous on that stream; no entry point synchronises the host and
 * none allocates device memory.  Buffers are owned by the caller.
 *
 * Workspace (linear entry points): some shapes split the reduction over K
 * across workgroups and combine the partial results through a
 * caller-provided device buffer.  pgs_w8a16_workspace_bytes() gives the size
 * a call needs (0 = none).  The buffer must be 256-byte aligned and
 * zero-filled before its first use; every call leaves it valid for the next
 * one (its leading slots are left zeroed), so one buffer of the largest size
 * needed can serve all calls.  Calls that share a workspace must be ordered
 * (same stream, or synchronised); overlapping calls on one workspace race.
 * Passing NULL disables the split (always correct, slower for short-N shapes).
 * Under HIP graph capture a graph replays with the workspace it was captured
 * with: give each captured graph a workspace that it alone uses and zero it
 * inside the capture (a kernel fill, recorded in the graph), so that every
 * replay starts from empty slots whatever else used that memory meanwhile.
 *
 * Return value: PGS_OK (0) or one of the PGS_ERR_* codes below.  A call that
 * returns an error has launched nothing.  pgs_last_error() gives a
 * human-readable message for the calling thread's most recent failure.
 *
 * Layouts (no leading-dimension argument):
 *   weight w   [n, k]  fp32 or bf16   row-major (out_features, in_features)
 *   q          [n, k]  int8           row-major, per-output-row symmetric
 *                                     quantization (QuantizedWeight.q)
 *   qp         packed  int8           the same values in "MFMA tile" order,
 *                                     pgs_packed_bytes(n, k) bytes: 16-row x
 *                                     64-column blocks of 1 KiB, stored
 *                                     [ceil(n/16)][ceil(k/64)]; inside a block
 *                                     byte 16*l + b (l = 0..63, b = 0..15) is
 *                                     q[16*blk_row + l%16][64*blk_col +
 *                                     16*(l/16) + b]; padding is zero.  The
 *                                     linear entry points read weights only in
 *                                     this layout (one contiguous KiB per
 *                                     wavefront load).
 *   scale      [n]     fp32           (the reference stores it as [n, 1])
 *   x          [m, k]  bf16           row-major activations
 *   bias       [n]     bf16           optional (NULL = none)
 *   y          [m, n]  bf16 or fp32   row-major, y = x . (q * scale)^T + bias
 *
 * Reference interface (Rakshit-gen/pageserve, a Python package with no FFI):
 * each entry point below names the Python function or call site it replaces.
 */
#ifndef PAGESERVE_AMD_H
#define PAGESERVE_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element type codes */
#define PGS_DTYPE_F32 0
#define PGS_DTYPE_BF16 1
#define PGS_DTYPE_F16 2

/* return codes */
#define PGS_OK 0
#define PGS_ERR_INVALID_ARGUMENT 1 /* bad size, null pointer, bad dtype code */
#define PGS_ERR_MISALIGNED 2       /* pointer not aligned to its element size */
#define PGS_ERR_LAUNCH 3           /* the HIP runtime rejected a kernel launch */
#define PGS_ERR_NO_DEVICE 4        /* no HIP device, or the stream's device is not a gfx950 */
#define PGS_ERR_TIMEOUT 5          /* a bounded device-side wait gave up (pgs_w8a16_decode_span_status) */

/* ABI version: bumped whenever a signature below changes. */
int pgs_abi_version(void);

/* Static string for a return code. */
const char* pgs_error_string(int code);

/* Detail of the calling thread's most recent failed call ("" if none). */
const char* pgs_last_error(void);

/*
 * Diagnostic, no counterpart in the reference: the kernel instance (with its
 * template arguments), grid size and K split of the calling thread's most
 * recent launch by a linear entry point ("" if none).  Lets tests and
 * profiles name the launch plan a shape takes.
 */
const char* pgs_last_plan(void);

/*
 * Whether `stream` is being captured into a HIP graph: *capturing = 1 and
 * *capture_id = the capture's id while a capture is active (2 if it was
 * invalidated), else 0 and 0.  No counterpart in the reference; hosts use it
 * to give each captured graph its own workspace (see the workspace notes
 * above).
 */
int pgs_stream_capture_state(void* stream, int* capturing, unsigned long long* capture_id);

/*
 * Replaces quantize_per_channel(weight) -- engine/quantization.py:16-23.
 *   absmax[r] = max(max_j |w[r,j]|, 1e-8f)
 *   scale[r]  = absmax[r] / 127.0f                 (IEEE fp32 division)
 *   q[r,j]    = clamp(rint(w[r,j] / scale[r]), -127, 127)   (ties to even)
 * Bit-exact with the reference's CPU arithmetic.  w_dtype: PGS_DTYPE_F32 or
 * PGS_DTYPE_BF16 (a bf16 weight widens exactly, as weight.float() does).
 * Non-finite weights follow the reference's CPU arithmetic: a row holding a
 * NaN gets a NaN scale (torch's amax and clamp keep NaN), a row holding an
 * infinity and no NaN gets an infinite scale, and every quotient that is NaN
 * (NaN / s, inf / inf, w / NaN) becomes q = 0, the value torch's CPU
 * conversion of NaN to int8 gives; finite / inf is 0.
 */
int pgs_quantize_per_channel(const void* w, int w_dtype, int64_t n, int64_t k,
                             int8_t* q, float* scale, void* stream);

/*
 * quantize_per_channel with the int8 result written in the packed layout
 * (same values as pgs_quantize_per_channel; padding zeroed).  This is how
 * QuantizedWeight(weight) stores its weight (engine/quantization.py:36-38).
 */
int pgs_quantize_per_channel_packed(const void* w, int w_dtype, int64_t n,
                                    int64_t k, int8_t* qp, float* scale,
                                    void* stream);

/* Bytes of the packed layout of an [n, k] int8 matrix (-1 for bad sizes). */
int64_t pgs_packed_bytes(int64_t n, int64_t k);

/*
 * Row-major q -> packed qp (padding written as zero), and back.  No
 * counterpart in the reference, which only has the row-major form
 * (QuantizedWeight.q, engine/quantization.py:38): unpack is how that form
 * is produced from the packed storage.
 */
int pgs_pack_weight(const int8_t* q, int64_t n, int64_t k, int8_t* qp,
                    void* stream);
int pgs_unpack_weight(const int8_t* qp, int64_t n, int64_t k, int8_t* q,
                      void* stream);

/*
 * Replaces dequantize(q, scale, dtype) -- engine/quantization.py:26-27.
 *   out[r,j] = dtype(float(q[r,j]) * scale[r])  (fp32 product, then one
 *   round-to-nearest-even conversion to out_dtype).  Bit-exact.
 * out_dtype: PGS_DTYPE_F32, PGS_DTYPE_BF16 or PGS_DTYPE_F16.
 */
int pgs_dequantize(const int8_t* q, const float* scale, int64_t n, int64_t k,
                   void* out, int out_dtype, void* stream);

/* dequantize from the packed layout; row-major [n, k] output, bit-exact. */
int pgs_dequantize_packed(const int8_t* qp, const float* scale, int64_t n,
                          int64_t k, void* out, int out_dtype, void* stream);

/*
 * Replaces F.linear(x, _resolve(W), b) for a QuantizedWeight W --
 * engine/model.py:25-26 (_resolve -> QuantizedWeight.get -> dequantize) feeding
 * the projections at engine/model.py:168-170 (q/k/v, with bias), :184 (o),
 * :188-190 (gate, up, down) and, with y_dtype = PGS_DTYPE_F32, the lm_head
 * at engine/model.py:193.
 *   y[i,r] = sum_j x[i,j] * q[r,j] * scale[r] (+ bias[r]),  fp32 accumulate,
 * with the weight given packed (qp).  The dense weight is never materialised.  y_dtype: PGS_DTYPE_BF16 or
 * PGS_DTYPE_F32.  Dispatches on m: the skinny kernel for m <= 32, the
 * MFMA tile kernel above.
 */
int pgs_w8a16_linear(const void* x, const int8_t* qp, const float* scale,
                     const void* bias, void* y, int y_dtype, int64_t m,
                     int64_t n, int64_t k, void* workspace,
                     size_t workspace_bytes, void* stream);

/*
 * pgs_w8a16_linear for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  No counterpart in the reference.  Same arguments, launch plan
 * and results as pgs_w8a16_linear with a workspace, but the K-split scratch
 * (pair slots, partial tiles) is a fixed 64 MiB device array inside the
 * library, one per GPU, held until the process ends; the call allocates
 * nothing and frees nothing.  A shape whose plan needs more scratch than that
 * returns PGS_ERR_INVALID_ARGUMENT (every projection of a 2048-hidden /
 * 11008-intermediate model up to 2048 tokens needs at most 60.5 MiB).  Every
 * call on one GPU shares the array: calls that overlap on one GPU (other
 * streams, concurrently replayed graphs) race; stream-ordered calls do not.
 * The first call on a device must have that device current.
 */
int pgs_w8a16_linear_noalloc(const void* x, const int8_t* qp, const float* scale,
                             const void* bias, void* y, int y_dtype, int64_t m,
                             int64_t n, int64_t k, void* stream);

/*
 * Replaces x = residual + F.linear(h, _resolve(W)) -- engine/model.py:184
 * (o_proj) and :190 (down_proj) -- with one launch: the residual add runs in
 * the linear's epilogue, with the reference's roundings,
 *   y = bf16( residual + bf16( x . (q * scale)^T + bias ) )
 * (fp32 output: y = residual + x . (q * scale)^T + bias).  residual: bf16
 * [m, n]; y may be the residual buffer itself (in place).  Otherwise as
 * pgs_w8a16_linear.
 */
int pgs_w8a16_linear_residual(const void* x, const int8_t* qp, const float* scale,
                              const void* bias, const void* residual, void* y,
                              int y_dtype, int64_t m, int64_t n, int64_t k,
                              void* workspace, size_t workspace_bytes,
                              void* stream);

/*
 * Replaces rms_norm(x, weight, eps) -- engine/model.py:29-34, applied before
 * the q|k|v (engine/model.py:166) and gate|up (:187) projections -- with one
 * kernel:
 *   r = 1 / sqrt(mean_j x[i,j]^2 + eps)   (fp32)
 *   h[i,j] = bf16( weight[j] * bf16( x[i,j] * r ) )
 * x, weight, h: bf16 ([m, k], [k], [m, k]); h may not alias x.
 */
int pgs_rmsnorm(const void* x, const void* weight, float eps, void* h,
                int64_t m, int64_t k, void* stream);

/*
 * Replaces q = apply_rope(q, cos, sin); k = apply_rope(k, cos, sin) --
 * engine/model.py:53-56 (apply_rope, rotate_half at :37-39), applied at
 * :172-173 -- with one kernel for both tensors.  With h = head_dim / 2, per
 * (token, head) and i < h, the reference's bf16 op chain
 * x * cos + rotate_half(x) * sin with its roundings:
 *   out[i]     = bf16( bf16(x[i]     * cos[i])     + bf16(-x[i + h] * sin[i]) )
 *   out[i + h] = bf16( bf16(x[i + h] * cos[i + h]) + bf16( x[i]     * sin[i + h]) )
 * q, q_out: bf16 [m, q_heads, head_dim]; k, k_out: bf16 [m, k_heads, head_dim]
 * (k_heads = 0: q only); cos, sin: bf16 [m, head_dim], the rows of the
 * reference's cos_cache / sin_cache for the m tokens.  Outputs may alias
 * their inputs (in place).  head_dim even.
 */
int pgs_rope(const void* q, void* q_out, int64_t q_heads, const void* k, void* k_out,
             int64_t k_heads, const void* cos, const void* sin, int64_t m,
             int64_t head_dim, void* stream);

/*
 * One output of a grouped linear: several quantized weights that read the
 * same activations (the q/k/v triple of engine/model.py:168-170).
 */
typedef struct pgs_linear_out {
  const int8_t* qp;    /* [n, k] int8, packed layout */
  const float* scale;  /* [n] fp32 */
  const void* bias;    /* [n] bf16 or NULL */
  void* y;             /* [m, n] of y_dtype */
  int64_t n;           /* rows of this weight */
} pgs_linear_out;

#define PGS_MAX_GROUP 4

/*
 * Replaces the three F.linear calls of engine/model.py:168-170 (q, k, v
 * projections of the same normalised hidden state) with one launch.  Each
 * output is what pgs_w8a16_linear computes for it, up to the order of the
 * fp32 summation over K (the K split is planned for the whole group, so a
 * member may be split differently than on its own).
 * 1 <= n_outs <= PGS_MAX_GROUP.
 */
int pgs_w8a16_linear_group(const void* x, const pgs_linear_out* outs,
                           int n_outs, int y_dtype, int64_t m, int64_t k,
                           void* workspace, size_t workspace_bytes,
                           void* stream);

/*
 * Replaces gate = F.linear(h, Wg); up = F.linear(h, Wu); F.silu(gate) * up
 * -- engine/model.py:188-190 -- with one fused launch:
 *   act[i,r] = silu(g) * u,  g = sum_j x[i,j] q_gate[r,j] * s_gate[r],
 *                            u = sum_j x[i,j] q_up[r,j] * s_up[r]
 * (both weights packed)
 * computed in fp32 and rounded once to bf16.  act: bf16 [m, n].
 * The down projection is a separate pgs_w8a16_linear call on act.
 */
int pgs_w8a16_swiglu(const void* x, const int8_t* qp_gate, const float* s_gate,
                     const int8_t* qp_up, const float* s_up, void* act,
                     int64_t m, int64_t n, int64_t k, void* workspace,
                     size_t workspace_bytes, void* stream);

/*
 * Replaces h = rms_norm(x, weight, eps) followed by the q/k/v projections of
 * h -- engine/model.py:166 (rms_norm at :29-34) and :168-170 -- with one
 * launch where the plan allows (K % 64 == 0, no K split, bf16 outputs, 16-byte
 * aligned norm weight, and m <= 4 tokens, or m <= 16 with K <= 2048 and few
 * enough output rows that the workgroups repeating the norm cost less than its
 * launch: at K <= 1024 16384 rows for m <= 8 and 8192 above, at longer K 4096 and
 * none): the kernel normalises the activations it loads, with the reference's roundings
 * (h = bf16(weight * bf16(x * r)), r = 1/sqrt(mean(x^2) + eps) in fp32);
 * otherwise pgs_rmsnorm into the workspace, then pgs_w8a16_linear_group.
 * The fp32 sum of squares is formed in a fixed order (deterministic) that
 * differs from pgs_rmsnorm's, so h may differ from it in the last bf16 bit.
 * workspace: pgs_w8a16_rmsnorm_workspace_bytes() bytes.
 */
int pgs_w8a16_rmsnorm_linear_group(const void* x, const void* norm_weight, float eps,
                                   const pgs_linear_out* outs, int n_outs, int y_dtype,
                                   int64_t m, int64_t k, void* workspace,
                                   size_t workspace_bytes, void* stream);

/*
 * Replaces h = rms_norm(x, weight, eps); silu(F.linear(h, Wg)) * F.linear(h,
 * Wu) -- engine/model.py:187-189 -- with one launch where the plan allows
 * (m <= 4 tokens; the other conditions and the roundings of
 * pgs_w8a16_rmsnorm_linear_group), otherwise pgs_rmsnorm into the workspace, then pgs_w8a16_swiglu.
 */
int pgs_w8a16_rmsnorm_swiglu(const void* x, const void* norm_weight, float eps,
                             const int8_t* qp_gate, const float* s_gate,
                             const int8_t* qp_up, const float* s_up, void* act,
                             int64_t m, int64_t n, int64_t k, void* workspace,
                             size_t workspace_bytes, void* stream);

/*
 * pgs_w8a16_rmsnorm_linear_group for q, k and v (outs[0..2], bf16 outputs),
 * then RoPE of q and k (engine/model.py:166-173): the outputs are
 * apply_rope(q), apply_rope(k) and v, with the reference's roundings (the bf16
 * projection, then pgs_rope's three).  cos / sin: bf16 [m, head_dim]; outs[0].n
 * and outs[1].n are whole heads of head_dim.  One launch at up to 32 tokens
 * where the norm runs inside the projection (above 4 tokens K <= 2048 and, since
 * the rotation's launch is saved too, up to 16384 / 8192 output rows for m <= 8 / 16
 * at K <= 1024, 8192 / 4096 at longer K, and 4096 for m <= 32) and head_dim % 32 == 0
 * (the two halves of a head are then computed side by side); the separate
 * kernels otherwise.  Workspace: pgs_w8a16_rmsnorm_workspace_bytes of the three.
 */
int pgs_w8a16_rmsnorm_qkv_rope(const void* x, const void* norm_weight, float eps,
                               const pgs_linear_out* outs, const void* cos,
                               const void* sin, int64_t head_dim, int64_t m, int64_t k,
                               void* workspace, size_t workspace_bytes, void* stream);

/*
 * Workspace bytes a linear call needs (0 = none): n[0..n_outs-1] are the
 * out_features of its members (one member for pgs_w8a16_linear; for
 * pgs_w8a16_swiglu pass swiglu = 1 and n[0] = intermediate size).  The value
 * is fixed by the sizes and never smaller than the plan needs.
 * No counterpart in the reference, whose dense F.linear needs no workspace.
 */
size_t pgs_w8a16_workspace_bytes(int64_t m, const int64_t* n, int n_outs,
                                 int64_t k, int swiglu);

/*
 * Workspace bytes of pgs_w8a16_rmsnorm_linear_group / pgs_w8a16_rmsnorm_swiglu
 * (same arguments as pgs_w8a16_workspace_bytes): always room for the
 * normalised activations ([m, k] bf16, used when the norm cannot run inside
 * the linear kernel) after the linear's own workspace and after the pair
 * slots at its start (kept empty for later calls sharing the workspace).  No
 * counterpart in the reference.
 */
size_t pgs_w8a16_rmsnorm_workspace_bytes(int64_t m, const int64_t* n, int n_outs,
                                         int64_t k, int swiglu);

/*
 * Replaces the greedy next token of server.py:51 (int(logits[-1].argmax()),
 * also app.py:87-93 and engine/runner.py:79) after the lm_head projection of
 * engine/model.py:193, without writing the logits: for each of the m rows of
 * x, idx[t] = argmax over r of y[t, r] = x[t] . (q[r] * scale[r]) (+ bias[r])
 * in fp32 -- torch.argmax's choice: the first index of the maximum, a NaN
 * counting as the maximum, -0.0 equal to +0.0 -- and, if vmax is not NULL,
 * vmax[t] = y[t, idx[t]] (bit-equal to pgs_w8a16_linear's fp32 output; a
 * canonical quiet NaN for a NaN maximum).  1 <= m <= 32 (pass only the rows
 * whose argmax is needed, e.g. the last prompt row).  idx: int64 [m];
 * vmax: fp32 [m].  workspace: pgs_w8a16_argmax_workspace_bytes(m, n, k)
 * bytes (per-workgroup partial maxima, fully rewritten by every call; no
 * zero-fill needed), 8-byte aligned.  Two launches (the projection with a
 * per-workgroup maximum in its epilogue, then one workgroup per row).
 */
int pgs_w8a16_linear_argmax(const void* x, const int8_t* qp, const float* scale,
                            const void* bias, int64_t* idx, float* vmax, int64_t m,
                            int64_t n, int64_t k, void* workspace,
                            size_t workspace_bytes, void* stream);

/* Workspace bytes of pgs_w8a16_linear_argmax (0 for unsupported sizes). */
size_t pgs_w8a16_argmax_workspace_bytes(int64_t m, int64_t n, int64_t k);

/* One decoder layer's weights after its attention (engine/model.py:184-190). */
typedef struct pgs_span_weights {
  const int8_t* qp_o;    const float* s_o;     /* o_proj [hidden, hidden], packed */
  const void* ln_post;                         /* post_attention_layernorm weight, bf16 [hidden] */
  const int8_t* qp_gate; const float* s_gate;  /* gate_proj [inter, hidden] */
  const int8_t* qp_up;   const float* s_up;    /* up_proj [inter, hidden] */
  const int8_t* qp_down; const float* s_down;  /* down_proj [hidden, inter] */
} pgs_span_weights;

/* The next layer's part before its attention (engine/model.py:165-173). */
typedef struct pgs_span_next {
  const void* ln_in;                 /* input_layernorm weight, bf16 [hidden] */
  pgs_linear_out q, k, v;            /* q/k/v projections: weight, scale, bias (or NULL), output [m, n] bf16 */
  const void* cos; const void* sin;  /* bf16 [m, head_dim] rows of the RoPE tables (applied to q and k), or NULL */
  int64_t head_dim;
} pgs_span_next;

/*
 * Replaces everything one decode step runs between two attention calls --
 * engine/model.py:184-190 of layer l, then :165-173 of layer l + 1 -- with
 * one launch:
 *   x1 = residual + o_proj(attn)          (pgs_w8a16_linear_residual)
 *   h  = rms_norm(x1, ln_post, eps)       (pgs_rmsnorm)
 *   a  = silu(gate(h)) * up(h)            (pgs_w8a16_swiglu)
 *   x_out = x1 + down(a)                  (pgs_w8a16_linear_residual)
 *   h' = rms_norm(x_out, next->ln_in, eps)
 *   q, k, v = projections of h' (+ bias); RoPE of q and k with cos/sin
 * each with the rounding of the entry point named beside it (results equal
 * those of the chain of those entry points up to the order of the fp32 sums).
 * next = NULL: the last layer (no q/k/v).  The weights stream from HBM once,
 * in one persistent launch of one workgroup per CU whose stages meet through
 * tagged exchanges in the workspace, so the device must not run other work
 * meanwhile.  Compiled configurations: pgs_w8a16_decode_span_supported().
 * attn, residual, x_out: bf16 [m, hidden]; x_out may not alias residual.
 * workspace: pgs_w8a16_decode_span_workspace_bytes() bytes, 256-byte
 * aligned, zero-filled before its first use; calls sharing it must be
 * stream-ordered.  The waits inside the launch are bounded: a launch that
 * gives up (a workgroup that never ran, another kernel occupying CUs) leaves
 * an error word in the workspace and returns; later launches on that
 * workspace then do nothing until pgs_w8a16_decode_span_status() clears it.
 * No counterpart in the reference (its forward_step runs these as separate
 * torch calls).
 */
int pgs_w8a16_decode_span(const void* attn, const void* residual, void* x_out,
                          const pgs_span_weights* w, const pgs_span_next* next,
                          float eps, int64_t m, int64_t hidden, int64_t inter,
                          void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes of pgs_w8a16_decode_span (0 for unsupported sizes). */
size_t pgs_w8a16_decode_span_workspace_bytes(int64_t m, int64_t hidden, int64_t inter);

/* 1 if pgs_w8a16_decode_span has a compiled configuration for these sizes. */
int pgs_w8a16_decode_span_supported(int64_t m, int64_t hidden, int64_t inter,
                                    int64_t nq, int64_t nkv, int64_t head_dim);

/*
 * Synchronises `stream` and reads the workspace's error word: PGS_OK, or
 * PGS_ERR_TIMEOUT if a launch gave up since the workspace was cleared; with
 * reset != 0 the workspace header and exchange buffers are then zero-filled
 * (a kernel on `stream`) so the next launch can run.
 */
int pgs_w8a16_decode_span_status(void* workspace, int reset, void* stream);

/*
 * Test hook, no counterpart in the reference: the number of polls after
 * which a decode span launch gives up (0 = the default), and force_giveup
 * != 0 makes every launch wait for a tag that no workgroup writes, so that
 * the give-up path runs.  Process-wide; affects later launches.
 */
int pgs_w8a16_decode_span_test_hooks(int spin_limit, int force_giveup);

/*
 * Tracing aid, no counterpart in the reference: with a device buffer set,
 * every later decode span launch writes per-workgroup stage timestamps
 * (s_memrealtime, a constant 100 MHz clock) into it, laid out
 * [slots][256 workgroups][16] uint64 with slots = bytes / 32768 (at most
 * 65535) and slot = launch tag % slots (the tag advances by one per launch
 * on a workspace).  Entries 0..12: launch start, end of the prologue, end of
 * o_proj's stream, o_proj's result published, x1 gathered (RMSNorm done),
 * end of gate|up's stream, activations published, activations gathered,
 * end of down_proj's stream, x2 published, x2 gathered (next RMSNorm done),
 * end of q|k|v's stream, end of the launch; 13..15: polls of the three
 * gathers (wave 0's).  NULL turns it off.  Process-wide; the buffer must outlive the
 * launches that write it, including every replay of a graph captured while
 * it was set (the launch holds its address).
 */
int pgs_w8a16_decode_span_trace(void* buffer, size_t bytes);

/*
 * ---------------------------------------------------------------------------
 * 4-bit weights with group scales.  No counterpart in the reference, whose one
 * quantized form is the 8-bit one above; same rules: symmetric, absmax, the
 * weight stored once in the layout the matmul streams.
 *
 * A group is `group` (32, 64 or 128) consecutive columns of a row, the last
 * one of a row possibly shorter.  Values of a code c (0..15): 0, 0.5, 1, 1.5,
 * 2, 3, 4, 6 for c % 8 = 0..7, negative for c >= 8 (the E2M1 values gfx950
 * widens to bf16 in hardware, exactly).
 *   scale  = bf16( max(max_j |w[r,j]| over the group, 1e-8f) / 6.0f )
 *   code   = the value nearest to w / scale, a tie to the even code (decided
 *            by exact products of scale, without a division; a weight that
 *            rounds to zero has code 0); weight = value * scale
 * A group holding a NaN gets a NaN scale and codes 0; one holding an infinity
 * an infinite scale (its finite weights' codes 0).
 *
 *   qp   packed codes, pgs_packed4_bytes(n, k): 16-row x 128-column blocks of
 *        1 KiB, [ceil(n/16)][ceil(k/128)]; inside a block, dword j of the 16
 *        bytes of lane l (0..63) holds columns 32*j + 8*(l/16) .. +7 of row
 *        l%16, column 32*j + 8*(l/16) + i in bits 4*i .. 4*i+3
 *   sp   packed scales, pgs_packed4_scales(n, k, group) bf16 values: per block
 *        [16 rows][128/group groups]
 * Padding codes and scales are zero.  k must be a multiple of 16.
 */
int64_t pgs_packed4_bytes(int64_t n, int64_t k);
int64_t pgs_packed4_scales(int64_t n, int64_t k, int64_t group);

/* w [n, k] fp32 or bf16, row-major, 16-byte aligned -> qp, sp (padding included). */
int pgs_quantize4_packed(const void* w, int w_dtype, int64_t n, int64_t k,
                         int64_t group, void* qp, void* sp, void* stream);

/* out[r,j] = dtype(value * scale): the fp32 product (exact), rounded once. */
int pgs_dequantize4_packed(const void* qp, const void* sp, int64_t n, int64_t k,
                           int64_t group, void* out, int out_dtype, void* stream);

/*
 * y = x . (value * scale)^T (+ bias) for 4-bit weights: x bf16 [m, k] (rows
 * contiguous, 16-byte aligned), bias bf16 [n] or NULL, y bf16 or fp32 [m, n];
 * fp32 accumulation.  With residual (bf16 [m, n], else NULL) the output is
 * residual + the linear's output rounded to y_dtype, as in
 * pgs_w8a16_linear_residual; y may be the residual buffer.  Made for the few
 * tokens of a drafting step; above 64 rows the weights are read once per 64.
 * The workspace holds the partial sums of a K that is split over workgroups
 * (0 bytes: none is needed, and it may be NULL); it must be 16-byte aligned.
 */
size_t pgs_w4a16_workspace_bytes(int64_t m, int64_t n, int64_t k);
int pgs_w4a16_linear(const void* x, const void* qp, const void* sp,
                     const void* bias, const void* residual, void* y,
                     int y_dtype, int64_t m, int64_t n, int64_t k,
                     int64_t group, void* workspace, size_t workspace_bytes,
                     void* stream);

/*
 * ---------------------------------------------------------------------------
 * The paged cache of keys and values (the reference's engine/paged_attention.py
 * and engine/block_allocator.py run these on the CPU or as torch calls, one
 * sequence at a time; here a batch of requests per launch).
 *
 * Block tables: int32 [requests, columns], row stride `table_stride`; column c
 * of request b names the block that holds its tokens c*block_size .. +
 * block_size - 1.  lens: int32 [requests], tokens cached.  free_blocks: int32
 * [free_capacity], a stack of the blocks in no table, *free_count of them.
 * offsets: int32 [requests + 1]: rows offsets[b] .. offsets[b+1] - 1 of a
 * batch belong to request b; rows behind offsets[requests] to none.
 * Everything is read on the device: nothing here waits for the host, and every
 * call can be captured in a HIP graph.
 */

/*
 * Extends each request by new_lens[b] tokens (a negative count is 0), in
 * request order: the blocks it needs are taken from the top of the stack into
 * its next table columns, lens and free_count are updated.  status[b] = 0 if
 * request b was served; 1 if it needs blocks and the requests up to it need
 * more than the stack holds; 2 if its length is negative or its table has too
 * few columns.  A request that is not served is left as it was.
 * slots[i], i < rows: the slot (block * block_size + place in the block) of row
 * i of the batch: token lens[b] (before the call) + n of its request, where n =
 * index[i], or i - offsets[b] without an index; -1 if n is not in
 * 0..new_lens[b]-1, the request was not served, the row belongs to none, or the
 * table's column for it (an older one) holds a negative number.
 * No array that is written (here and in pgs_truncate_blocks) may share memory
 * with another.
 */
int pgs_append_blocks(int32_t* lens, const int32_t* new_lens, int32_t* block_tables,
                      int64_t table_stride, int64_t columns, const int32_t* free_blocks,
                      int64_t free_capacity, int32_t* free_count, int64_t block_size,
                      int64_t requests, const int32_t* offsets, const int32_t* index,
                      int64_t rows, int64_t* slots, int32_t* status, void* stream);

/*
 * Shortens each request to keep[b] tokens (0: it is finished; a count above its
 * length keeps all; a negative length becomes 0): blocks no longer needed go back
 * to the stack, their table columns become -1.  Undoes pgs_append_blocks exactly.
 * A column that holds a negative number names no block and gives none back; other
 * numbers are not checked (nothing here says how many blocks there are).  Blocks
 * beyond the stack's capacity are dropped.
 */
int pgs_truncate_blocks(int32_t* lens, const int32_t* keep, int32_t* block_tables,
                        int64_t table_stride, int64_t columns, int32_t* free_blocks,
                        int64_t free_capacity, int32_t* free_count, int64_t block_size,
                        int64_t requests, void* stream);

/* Keys and values of one layer: element strides of [blocks, block_size,
 * kv_heads, head_dim] (the last dimension contiguous). */
typedef struct pgs_kv_cache {
  void* k;
  void* v;
  int64_t blocks, block_size, kv_heads, head_dim;
  int64_t k_block, k_slot, k_head;
  int64_t v_block, v_slot, v_head;
} pgs_kv_cache;

/*
 * Rows i of k and v (bf16 or fp16 [rows, kv_heads, head_dim], element strides
 * of row and head given) into slot slots[i] of the cache; a slot outside the
 * cache is left out.  The slots of the rows must differ: of two rows with one
 * slot, either may stay.  The rows must not lie in the cache, nor two of its
 * elements in one place.
 */
int pgs_write_kv(const void* k, int64_t k_row, int64_t k_head, const void* v,
                 int64_t v_row, int64_t v_head, const pgs_kv_cache* cache,
                 const int64_t* slots, int64_t rows, void* stream);

/* The arguments of pgs_tree_attention. */
typedef struct pgs_tree_attention_args {
  const void* q;               /* [rows, q_heads, head_dim] */
  const void* k;               /* [rows, kv_heads, head_dim]: the drafted tokens' own */
  const void* v;
  void* out;                   /* [rows, q_heads, head_dim] */
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head; /* element strides */
  const pgs_kv_cache* cache;
  const int32_t* block_tables; /* [requests, columns] */
  int64_t table_stride, columns;
  const int32_t* lens;         /* [requests]: cached tokens */
  const int32_t* offsets;      /* [requests + 1] */
  const int32_t* parents;      /* [rows], or NULL: each token's parent is the one before it */
  int64_t rows, requests, q_heads;
  int64_t max_tokens;          /* rows per request, at most 64; the kernels are chosen by it */
  int64_t max_context;         /* the longest lens expected: sizes the split, not the result */
  float scale;
  int dtype;                   /* PGS_DTYPE_BF16 or PGS_DTYPE_F16, of all tensors */
} pgs_tree_attention_args;

/*
 * Attention of drafted tokens over a paged cache.  Token t of request b (row
 * offsets[b] + t) attends to the request's lens[b] cached tokens, to itself and
 * to its ancestors among the drafted tokens: parents[row] names a token of the
 * same request before t (any other value: none), so that the drafted tokens form
 * trees.  Query heads share key heads in groups of q_heads / kv_heads.
 *   out = sum_j softmax_j(scale * q . k_j) v_j     (softmax in fp32)
 * head_dim 64 or 128; block_size a multiple of 16, columns * block_size at most
 * 2^31 - 65536; strides multiples of 8 elements and pointers 16-byte aligned.
 * Lengths beyond the table's columns are cut to them; tokens in a block outside
 * the cache are left out; rows of no request, and a request's rows from max_tokens
 * on, are not written.
 * workspace: pgs_tree_attention_workspace_bytes() bytes, 256-byte aligned, no
 * fill needed.
 */
int pgs_tree_attention(const pgs_tree_attention_args* args, void* workspace,
                       size_t workspace_bytes, void* stream);

/* Workspace bytes of pgs_tree_attention (0: none needed). */
size_t pgs_tree_attention_workspace_bytes(int64_t rows, int64_t requests, int64_t q_heads,
                                          int64_t kv_heads, int64_t head_dim,
                                          int64_t max_tokens, int64_t max_context);

/*
 * ---------------------------------------------------------------------------
 * Long texts in a bounded cache.  No counterpart in the reference, whose
 * attention reads every cached token of a sequence in its own type
 * (engine/paged_attention.py:16-50).
 *
 * Row t of a request of n rows and len cached tokens, the rows' own among them,
 * stands at p = len - n + t and sees token j if
 *   j <= p  and  (j > p - window  or  j < sinks)
 * A window past every text (2^31 - 1) sees them all.
 */

/* A layer's keys and values in 4 bits, heads in front of slots, contiguous:
 *   k, v              uint8 [blocks, kv_heads, block_size, head_dim / 2]
 *   k_scale, v_scale  bf16 [blocks, kv_heads, block_size, head_dim / 32]
 * Per 32 dims of a token and head one scale, max(absmax, 1e-8) / 6 cut to its
 * first 6 significant bits, and a code per dim (the values and the rounding are
 * those of the 4-bit weights above), so that value * scale is a bf16 number.  A
 * group that holds an infinity or a NaN gets it as its scale, and its finite
 * numbers codes 0.
 * With C = head_dim / 32: byte 4 (C a + c) + i of a key's row (a, i < 4, c < C)
 * holds dims 32 c + 8 a + 2 i (low half) and the next one.  Of 16 tokens' values,
 * token 4 a + b has its dims m, 16 + m, 32 + m, ... (m < 16) in the C bytes from
 * byte C (4 (16 a + m) + b) of the sixteen on, low halves first. */
typedef struct pgs_kv_cache4 {
  void* k;
  void* k_scale;
  void* v;
  void* v_scale;
  int64_t blocks, block_size, kv_heads, head_dim;
} pgs_kv_cache4;

/*
 * Rows i of k and v (bf16 or fp16 [rows, kv_heads, head_dim], element strides of
 * row and head given) in 4 bits into slot slots[i] of the cache; a slot outside
 * the cache is left out.  The slots of the rows must differ (of two rows with one
 * slot, pieces of either may stay).  head_dim 64 or 128, block_size a multiple
 * of 16, the cache 16-byte aligned; rows * kv_heads * head_dim at most 2^34 - 1024.
 */
int pgs_write_kv4(const void* k, int64_t k_row, int64_t k_head, const void* v,
                  int64_t v_row, int64_t v_head, int dtype,
                  const pgs_kv_cache4* cache, const int64_t* slots, int64_t rows,
                  void* stream);

/* The rows at slots[i] back: k, v [rows, kv_heads, head_dim] (bf16, fp16 or
 * fp32, contiguous, 16-byte aligned); zeros for a slot outside the cache.  As many
 * rows as above. */
int pgs_read_kv4(const pgs_kv_cache4* cache, const int64_t* slots, int64_t rows,
                 void* k, void* v, int dtype, void* stream);

/* The arguments of pgs_window_attention. */
typedef struct pgs_window_attention_args {
  const void* q;               /* [rows, q_heads, head_dim] */
  void* out;                   /* [rows, q_heads, head_dim] */
  float* lse;                  /* [rows, q_heads], or NULL */
  int64_t q_row, q_head, out_row, out_head; /* element strides */
  const pgs_kv_cache* cache;   /* of the rows' dtype, or NULL: cache4 */
  const pgs_kv_cache4* cache4;
  const int32_t* block_tables; /* [requests, columns] */
  int64_t table_stride, columns;
  const int32_t* lens;         /* [requests]: cached tokens, the rows' own among them */
  const int32_t* offsets;      /* [requests + 1] */
  int64_t rows, requests, q_heads;
  int64_t max_tokens;          /* rows per request; the kernels are chosen by it */
  int64_t max_context;         /* the longest lens expected: sizes the split, not the result */
  int64_t window, sinks;
  float scale;
  int dtype;                   /* PGS_DTYPE_BF16 or PGS_DTYPE_F16, of q and out */
} pgs_window_attention_args;

/*
 * out = sum_j softmax_j(scale * q . k_j) v_j and lse = ln sum_j e^(scale q . k_j)
 * over the tokens that a row sees (softmax in fp32); a row that sees none gets
 * zeros and -inf.  Query heads share key heads in groups of q_heads / kv_heads.
 * head_dim 64 or 128; block_size a multiple of 16, columns * block_size at most
 * 2^31 - 65536; strides multiples of 8 elements and pointers 16-byte aligned.
 * Lengths beyond the table's columns are cut to them; tokens in a block outside
 * the cache are left out; rows of no request, and a request's rows from max_tokens
 * on, are not written.  With fp16 rows, 4-bit keys and values beyond fp16's range
 * may count as infinite.
 * workspace: pgs_window_attention_workspace_bytes() bytes, 256-byte aligned, no
 * fill needed.
 */
int pgs_window_attention(const pgs_window_attention_args* args, void* workspace,
                         size_t workspace_bytes, void* stream);

/* Workspace bytes of a call with these arguments (0: none needed); its pointers, but
 * for the cache's sizes, are not looked at. */
size_t pgs_window_attention_workspace_bytes(const pgs_window_attention_args* args);

/* The arguments of pgs_accumulate_weights; those with a name of
 * pgs_window_attention_args mean the same. */
typedef struct pgs_accumulate_weights_args {
  const void* q;
  int64_t q_row, q_head;
  const pgs_kv_cache* cache;   /* (its values are not read and may be NULL) */
  const pgs_kv_cache4* cache4;
  const int32_t* block_tables;
  int64_t table_stride, columns;
  const int32_t* lens;
  const int32_t* offsets;
  const float* lse;            /* [rows, q_heads], as pgs_window_attention gave it */
  const int32_t* new_lens;     /* [requests], or NULL: as many last tokens of a request start from 0 */
  float* weights;              /* [blocks, block_size] */
  int64_t rows, requests, q_heads, max_tokens, max_context, window, sinks;
  float scale;
  int dtype;
} pgs_accumulate_weights_args;

/*
 * Adds to weights[slot of token j] the attention weights of the rows and query
 * heads that see j: sum of e^(scale q . k_j - lse).  Sums are fp32, in a fixed
 * order.  Tokens in a block outside the cache are left out; no block may be in two
 * requests' tables, or twice in one (an addition may be lost).
 */
int pgs_accumulate_weights(const pgs_accumulate_weights_args* args, void* workspace,
                           size_t workspace_bytes, void* stream);

/* Workspace bytes of a call with these arguments (0: none needed), 4-byte aligned, no
 * fill needed. */
size_t pgs_accumulate_weights_workspace_bytes(const pgs_accumulate_weights_args* args);

/*
 * Cuts each request of more than budget[b] tokens to budget[b] (below 0: 0): the
 * first `sinks`, the last `recent` and, of those between, the ones of largest
 * weight stay (of equal ones the first; a NaN is the largest, a token in a block
 * outside the cache the smallest), in their order, moved together to the front.
 * sinks come before recent where the budget does not hold both.  kept[b]: the
 * tokens that stay; lens and the tables are left as they are (pgs_truncate_blocks
 * with kept shortens them).  weights [blocks, block_size] and the rows of every
 * cache (of one layer each: `count` in 16 bits, `count4` in 4, each kind of one
 * size) move alike; what lies behind the kept tokens is left as it is, and so is
 * a place whose token, or which itself, is in a block outside the cache.  A
 * request of more than max_context tokens is left as it is.  No block may be in
 * two requests' tables, no two caches may share an element, and no array that is
 * written may share memory with another.
 * requests at most 65536, requests * kv_heads at most 2^24.
 * workspace: pgs_evict_tokens_workspace_bytes() bytes, no fill needed.
 */
int pgs_evict_tokens(float* weights, const int32_t* lens, const int32_t* budget,
                     const int32_t* block_tables, int64_t table_stride, int64_t columns,
                     int64_t blocks, int64_t block_size, int64_t requests, int64_t sinks,
                     int64_t recent, int64_t max_context, const pgs_kv_cache* caches,
                     int64_t count, const pgs_kv_cache4* caches4, int64_t count4,
                     int32_t* kept, void* workspace, size_t workspace_bytes, void* stream);
size_t pgs_evict_tokens_workspace_bytes(int64_t requests, int64_t max_context);

#ifdef __cplusplus
}
#endif

#endif /* PAGESERVE_AMD_H */
