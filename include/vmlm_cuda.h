/*
 * vmlm_cuda.h -- C ABI of the B200 (sm_100a) implementation of the VMLM
 * quantised-linear path: the Q8 (int8 weight, per-output-row f32 scale) and
 * bf16-weight GEMM/GEMV kernels that the VM's OP_GEMM dispatches to.
 *
 * Reference interfaces replaced (paths inside the shouzugzs-AI/Sparrow tree):
 *   vmlm_gemm_nt_int8  <- vmlm_ops::kernels::gemm_nt_int8  ops/src/kernels.rs:1256-1261
 *   vmlm_gemm_nt_bf16  <- vmlm_ops::kernels::gemm_nt_bf16  ops/src/kernels.rs:1200-1204
 * Both are called from the OP_GEMM arm of Vm::run (core/src/interp.rs:764, 801)
 * and from Rust generated by the Sparrow DSL (sparrow/src/libgen.rs:649-657).
 *
 * Semantics kept from the reference:
 *   - row-major, contiguous K, no strides: A[m,k], W[n,k] (nn.Linear), C[m,n];
 *   - C is overwritten (the reference bf16/int8 kernels have no accumulate);
 *   - gemm_nt_int8: C[i][j] = (sum_k A[i][k]*f32(q[j][k])) * scale[j];
 *   - gemm_nt_bf16: C[i][j] =  sum_k A[i][k]*widen(b[j][k]).
 * Differences: every entry point returns a status (the Rust kernels return
 * `()` and the VM prints and calls exit(9) on misuse, core/src/interp.rs:752-806);
 * the Rust shim (crate vmlm-ops-cuda) maps a non-zero status to that convention.
 *
 * All buffers are owned by the caller. Host-pointer entry points are
 * synchronous. Device-pointer entry points (suffix _dev) are ordered on the
 * given CUDA stream (NULL = the library stream of the current device) and
 * return before the GPU finishes.
 *
 * Threading: calls are serialised by the library per device. Device-pointer
 * calls share one workspace per device, so calls on different streams of the
 * same device must not overlap on the GPU.
 *
 * Stream capture: a _dev call can be captured into a CUDA graph once an eager
 * call of at least its size has sized the workspace; a call that would have to
 * allocate cannot be captured. A workspace that captured calls use is kept until
 * vmlm_shutdown when a later, larger call replaces it, so their graphs can still be
 * replayed (and must not be replayed after vmlm_shutdown).
 *
 * Aliasing: C must not overlap A (some calls clear C before they read A).
 *
 * Programmatic dependent launch: the library's GEMM kernels let the next
 * kernel in the stream be scheduled before they finish. A kernel the caller
 * launches right after a _dev call with the programmatic stream
 * serialization attribute must execute griddepcontrol.wait
 * (cudaGridDependencySynchronize) before it touches the call's buffers;
 * kernels launched without that attribute are ordered as usual.
 */
#ifndef VMLM_CUDA_H
#define VMLM_CUDA_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define VMLM_API __attribute__((visibility("default")))
#else
#define VMLM_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum vmlm_status {
  VMLM_OK = 0,
  VMLM_ERR_ARG = 1,            /* null pointer, zero size where data is required, bad value */
  VMLM_ERR_SHAPE = 2,          /* size outside what the kernels support (e.g. int32 range) */
  VMLM_ERR_CUDA = 3,           /* a CUDA runtime/driver call failed; see vmlm_last_error() */
  VMLM_ERR_NO_DEVICE = 4,      /* no usable sm_100 device */
  VMLM_ERR_STATE = 5,          /* call out of order (e.g. not initialised) */
  VMLM_ERR_OOM = 6,            /* device allocation failed */
  VMLM_ERR_DEVICE_TIMEOUT = 7, /* a kernel gave up a bounded wait; results are invalid */
  VMLM_ERR_OPERATOR = 8        /* an OP_GEMM misuse the VM reports by printing and exit(9) */
};

/* Library version, major*10000 + minor*100 + patch. */
VMLM_API int vmlm_version(void);

/* Select the device used by the host-pointer entry points and create its
 * context (stream, workspace). Safe to call again; device < 0 keeps the
 * current CUDA device. No reference counterpart (the reference has no device). */
VMLM_API int vmlm_init(int device);

/* Release every device context, registered weight and workspace. */
VMLM_API int vmlm_shutdown(void);

/* Human-readable description of the last error on the calling thread. */
VMLM_API const char *vmlm_last_error(void);

/* ---------------------------------------------------------------- weights
 * Weights are immutable constants in the VM (core/src/interp.rs:241-345 forbids
 * any non-GEMM op on bf16/i8 constants), so a device copy can be kept per host
 * address range. A host-pointer call whose weight (or scale) lies inside a
 * registered range uses the resident copy; otherwise it uploads the bytes for
 * that call only. Sub-ranges resolve too (OP_LAYERB offsets, interp.rs:438-475). */
VMLM_API int vmlm_register_weight(const void *host_ptr, size_t bytes);
VMLM_API int vmlm_unregister_weight(const void *host_ptr);
VMLM_API int vmlm_unregister_all(void);

/* --------------------------------------------------- host-pointer GEMMs
 * Drop-in for vmlm_ops::kernels::gemm_nt_int8 (ops/src/kernels.rs:1256-1261). */
VMLM_API int vmlm_gemm_nt_int8(const float *a, const int8_t *q, const float *scale, float *c, size_t m, size_t n,
                      size_t k);

/* Drop-in for vmlm_ops::kernels::gemm_nt_bf16 (ops/src/kernels.rs:1200-1204). */
VMLM_API int vmlm_gemm_nt_bf16(const float *a, const uint16_t *b, float *c, size_t m, size_t n, size_t k);

/* int8 activations x int8 weights, exact int32 accumulation, then
 * C = f32(acc) * scale[n]; c and/or acc may be NULL. No reference kernel
 * exists (the VM has no int8-activation GEMM); this is the exact integer
 * definition used by the large prefill FFN configuration. */
VMLM_API int vmlm_gemm_i8i8(const int8_t *x, const int8_t *w, const float *scale, float *c, int32_t *acc, size_t m,
                   size_t n, size_t k);

/* f32 GEMMs, the rest of the VM's OP_GEMM: C[m,n] = A[m,k] . B^T (+ C when
 * acc != 0). Drop-in for vmlm_ops::kernels::gemm_nt (ops/src/kernels.rs:987-1015:
 * B is [n,k], row-major) and vmlm_ops::kernels::gemm (ops/src/kernels.rs:407-419,
 * gemm_scalar :381-403: B is [k,n], row-major, C = A . B). With acc the
 * product is added to C's old value (one f32 add per element, as the
 * reference's `s += c`). Both operands are split exactly into three bf16 terms
 * and multiplied on the tensor cores in f32: results are within f32 rounding of
 * the reference's (which itself differs between its AVX2, packed and scalar
 * kernels in summation order); NaN / Inf propagate as in the reference.
 * k == 0 gives C = 0 (acc == 0) or leaves C unchanged. */
VMLM_API int vmlm_gemm_nt_f32(const float *a, const float *b, float *c, size_t m, size_t n, size_t k, int acc);
VMLM_API int vmlm_gemm_f32(const float *a, const float *b, float *c, size_t m, size_t n, size_t k, int acc);

/* ------------------------------------------- decode-step neighbours
 * RMSNorm fused into the Q8 linear layer: C = gemm_nt_int8(rmsnorm(a, g,
 * eps), q, scale), rmsnorm as vmlm_ops::kernels::rmsnorm
 * (ops/src/kernels.rs:1346-1370: per row x * 1/sqrt(mean(x^2) + eps) * g,
 * same rounding steps; the mean of squares is summed in another order), then
 * the Q8 GEMM of vmlm_gemm_nt_int8. The norm is computed inside the
 * activation encoding (no separate pass over a, no normalised copy for the
 * caller). g has k values. */
VMLM_API int vmlm_rmsnorm_gemm_nt_int8(const float *a, const float *g, float eps, const int8_t *q, const float *scale,
                                       float *c, size_t m, size_t n, size_t k);
VMLM_API int vmlm_rmsnorm_gemm_nt_int8_dev(const float *a, const float *g, float eps, const int8_t *q,
                                           const float *scale, float *c, size_t m, size_t n, size_t k, void *stream);

/* OP_GEMV (core/src/interp.rs:815-827): c[i] = sum_p a[i*k + p] * b[p], a
 * [m, k] row-major f32, b [k] f32, c [m] f32 (the sum in another order). */
VMLM_API int vmlm_gemv_f32(const float *a, const float *b, float *c, size_t m, size_t k);
VMLM_API int vmlm_gemv_f32_dev(const float *a, const float *b, float *c, size_t m, size_t k, void *stream);

/* OP_EMB (core/src/interp.rs:1351-1420) for m indices at once: out[t, :] =
 * f32(table[idx[t], :]), table [rows, cols] of VMLM_DT_BF16 (widened exactly)
 * or VMLM_DT_F32. Each idx[t] is an f32 that must be an integer in
 * [0, rows); otherwise VMLM_ERR_OPERATOR with the VM's message ("EMB: row
 * index out of range" / "EMB: row index is not an integer"): the host call
 * checks before any device work, the device call on the device (reported by
 * vmlm_sync; rows with a bad index are not written). A host table that is not
 * registered has just the m rows uploaded. */
VMLM_API int vmlm_emb(const void *table, int dtype, size_t rows, size_t cols, const float *idx, size_t m, float *out);
VMLM_API int vmlm_emb_dev(const void *table, int dtype, size_t rows, size_t cols, const float *idx, size_t m,
                          float *out, void *stream);

/* A batch of independent Q8 calls (device pointers) on one stream, e.g. the q, k, v projections of a decode
 * step or a layer's set of linears: the results of calling vmlm_gemm_nt_int8_dev for each in turn, up to the
 * Q8 activation rounding (a grouped launch forms a token's digit planes over the whole K, a single call may
 * form them per K range of a cluster). The calls must be independent: no call's c may overlap another call's
 * a, q, scale or c.
 * Calls that share m and fit the decode kernel run as one grouped launch, a CTA per 128-row tile of every
 * call, so the per-call launch and start-up latency is paid once; the others run one by one. A batch with
 * more tiles than the GPU has SMs at m <= 32 (e.g. a decoder layer's seven linears) runs instead as one CTA
 * per SM, each streaming an equal share of the batch's weight bytes; tiles split between CTAs are summed in
 * f64 through library workspace. */
typedef struct vmlm_q8_call {
  const float *a;
  const int8_t *q;
  const float *scale;
  float *c;
  size_t m, n, k;
} vmlm_q8_call;
VMLM_API int vmlm_gemm_nt_int8_batch_dev(const vmlm_q8_call *calls, size_t count, void *stream);

/* ---------------------------------------------- quantisation variants
 * int4 weights with a scale per group of columns: gemm_nt_int4_gs of
 * tests/src/quant.rs:298-362 (and gemm_nt_int4, :210-286, which is the same
 * with group = k). packed [n, (k+1)/2] as quant_int4_grouped writes it
 * (:114-152: column p in the low nibble of byte p/2 when p is even, the high
 * nibble when odd, two's complement); scale [n, ceil(k/group)] f32;
 * c[i][j] = sum over groups g of scale[j][g] * sum_{p in g} a[i][p] * v(j, p).
 * order 0 takes v from the packed order. order 1 reproduces the reference's
 * AVX2 step as shipped (:316-333), which reads other nibbles: in a 32-column
 * step at column kk inside a group, column kk+t uses the nibble of byte
 * kk/2 + (t&16)/2 + (t&7)/2, the high one when t is even. group >= 1 and
 * order in {0, 1}, else VMLM_ERR_ARG. f32 sums in another order. */
VMLM_API int vmlm_gemm_nt_int4_gs(const float *a, const uint8_t *packed, const float *scale, float *c, size_t m,
                                  size_t n, size_t k, size_t group, int order);
VMLM_API int vmlm_gemm_nt_int4_gs_dev(const float *a, const uint8_t *packed, const float *scale, float *c, size_t m,
                                      size_t n, size_t k, size_t group, int order, void *stream);

/* int8 with outlier input columns added back in f32 (LLM.int8):
 * gemm_nt_int8_outlier of tests/src/quant.rs:524-565. q/scale as
 * quant_int8_with_outliers writes them (:458-515: outlier columns of q are 0),
 * idx the n_idx outlier column indices, w the f32 weight [n, k]:
 * c = gemm_nt_int8(a, q, scale), then c[i][j] += a[i][idx[t]] * w[j][idx[t]]
 * for t = 0 .. n_idx-1 in that order (product rounded, then added). Every
 * idx[t] must be < k (VMLM_ERR_ARG). The host call uploads only the outlier
 * columns of w unless w is registered. The device call reads w[j * k + idx[t]]
 * when compact = 0, or wo[j * n_idx + t] of a compact matrix when compact = 1
 * (vmlm_gather_columns_dev builds it once per weight); a bad index there is
 * reported by vmlm_sync. */
VMLM_API int vmlm_gemm_nt_int8_outlier(const float *a, const int8_t *q, const float *scale, const float *w,
                                       const uint32_t *idx, size_t n_idx, float *c, size_t m, size_t n, size_t k);
VMLM_API int vmlm_gemm_nt_int8_outlier_dev(const float *a, const int8_t *q, const float *scale, const float *w,
                                           int compact, const uint32_t *idx, size_t n_idx, float *c, size_t m,
                                           size_t n, size_t k, void *stream);
/* wo[j][t] = w[j][idx[t]] for j < n, t < n_idx (device pointers). */
VMLM_API int vmlm_gather_columns_dev(const float *w, const uint32_t *idx, size_t n_idx, size_t n, size_t k,
                                     float *wo, void *stream);

/* ------------------------------------------------------ the OP_GEMM operator
 * A VM slot as the OP_GEMM arm reads it (slot_dtype / slot_shape / slot_mut,
 * core/src/interp.rs:481-500): a row-major [rows, cols] array of `dtype`
 * elements at ptr. dtype codes are the .vmb ones (core/src/format.rs:73-79);
 * the flag bits those of trans/src/opcode.rs:303-304. */
#define VMLM_DT_F32 0
#define VMLM_DT_F16 1
#define VMLM_DT_I8 2
#define VMLM_DT_I32 3
#define VMLM_DT_BF16 4
#define VMLM_FL_ACC 1     /* C += A . op(B) */
#define VMLM_FL_TRANS_B 2 /* set: NN, B is [K,N]; clear: NT, B is [N,K] */
typedef struct vmlm_slot {
  void *ptr;
  size_t rows;
  size_t cols;
  int dtype;
} vmlm_slot;

/* The OP_GEMM arm of Vm::run (core/src/interp.rs:734-812): C = A . op(B) with
 * m, k from A's shape and N = rows(B) (NT) or cols(B) (NN), dispatched on B's
 * dtype to vmlm_gemm_nt_bf16 / vmlm_gemm_nt_int8 / vmlm_gemm_nt_f32 /
 * vmlm_gemm_f32 (same arithmetic). `scale` is the slot the instruction's dt
 * field names (int8 B only; may be NULL otherwise). Where the VM prints and
 * exits 9 this returns VMLM_ERR_OPERATOR with the VM's message in
 * vmlm_last_error(): "bf16 NN gemm unimplemented", "bf16 acc gemm
 * unimplemented", "int8 NN gemm unimplemented", "int8 acc gemm
 * unimplemented", "int8 gemm: scale slot must be f32", "int8 gemm: scale
 * shorter than N rows", "gemm operand dtype unsupported". Added here, because
 * the reference reads out of bounds instead: A and C must be f32, the K of B
 * must equal cols(A), and C must hold m * N elements (also VMLM_ERR_OPERATOR).
 * vmlm_op_gemm takes host slots (synchronous, registered weights resolve);
 * vmlm_op_gemm_dev device slots on `stream` (as the _dev entry points). */
VMLM_API int vmlm_op_gemm(unsigned fl, const vmlm_slot *d, const vmlm_slot *a, const vmlm_slot *b,
                          const vmlm_slot *scale);
VMLM_API int vmlm_op_gemm_dev(unsigned fl, const vmlm_slot *d, const vmlm_slot *a, const vmlm_slot *b,
                              const vmlm_slot *scale, void *stream);

/* ---------------------------------------------- device constant pool (.vmb)
 * A .vmb program's constants, scratch regions and slot table on the device:
 * the load half of Vm::load / load_weights_mapped (core/src/interp.rs:123-220)
 * and bind_slots (:351-397), container layout of core/src/format.rs. The CONST
 * section (or `weights`, the separate weights file of load_weights_mapped,
 * when non-NULL) is copied to device memory once; the activation, state and
 * gradient regions are allocated and zeroed as the VM does. Checks before any
 * device work: "bad magic" (VMLM_ERR_ARG; the VM exits 3), "const has unknown
 * dtype" (VMLM_ERR_OPERATOR; the VM exits 9), VMLM_ERR_SHAPE for a header,
 * table or slot outside the image or its region (the VM reads such bytes), and
 * the VM's load-time dtype audit of the program text (audit_const_dtypes,
 * core/src/interp.rs:241-345; VMLM_ERR_OPERATOR with its message, e.g. "op 3
 * uses bf16 const at slot 5 (only a GEMM may read a non-f32 operand)" or
 * "gemm B has no kernel for this dtype"). The
 * program text is not run: the caller's interpreter runs it and hands OP_GEMM
 * instructions to vmlm_pool_gemm. The pool belongs to the current device. */
typedef struct vmlm_pool vmlm_pool;
#define VMLM_SLOT_CONST 0
#define VMLM_SLOT_ACT 1
#define VMLM_SLOT_STATE 2
#define VMLM_SLOT_GRAD 3
#define VMLM_SLOT_PARAM 4
VMLM_API int vmlm_pool_load(const void *vmb, size_t len, const void *weights, size_t weights_len, vmlm_pool **out);
VMLM_API int vmlm_pool_free(vmlm_pool *pool);
/* Counts and region sizes: region_bytes[4] = const, act, state, grad bytes (any pointer may be NULL). */
VMLM_API int vmlm_pool_info(const vmlm_pool *pool, size_t *n_const, size_t *n_slots, size_t *region_bytes);
/* Device base of region 0 (const), 1 (act), 2 (state) or 3 (grad). */
VMLM_API int vmlm_pool_region(const vmlm_pool *pool, int region, void **base);
/* Slot i as a device vmlm_slot (ptr, rows, cols, dtype) and its kind (VMLM_SLOT_*). CONSTANT slots
 * move with the OP_LAYERB base and are bound-checked as const_ptr_based does (core/src/interp.rs:453-479):
 * VMLM_ERR_OPERATOR "layer base walks past the constant pool: off=.. base=.. bytes=.. limit=..". */
VMLM_API int vmlm_pool_slot(const vmlm_pool *pool, size_t slot, vmlm_slot *out, int *kind);
/* OP_LAYERB (core/src/interp.rs:1019-1045): base += delta (saturating) for delta >= 0, base -= -delta
 * (saturating at 0) otherwise; float-to-integer as Rust casts (truncate, NaN -> 0). */
VMLM_API int vmlm_pool_layerb(vmlm_pool *pool, float delta);
VMLM_API int vmlm_pool_layer_base(const vmlm_pool *pool, size_t *base);
/* Vm::find / Vm::find_slot (core/src/interp.rs:399-424): FNV-1a name hash lookup; VMLM_ERR_ARG "const
 * not found" / "slot not found" where the VM exits 4 / 7. */
VMLM_API int vmlm_pool_find_const(const vmlm_pool *pool, const char *name, size_t *idx);
VMLM_API int vmlm_pool_find_slot(const vmlm_pool *pool, const char *name, size_t *idx);
/* Run one 16-byte OP_GEMM instruction (op u8 = 10, fl u8, dt u16, dst, a, b u32; trans/src/ins.rs:24-33)
 * on the pool's device slots: vmlm_op_gemm_dev with scale = slot dt when dt < n_slots. */
VMLM_API int vmlm_pool_gemm(vmlm_pool *pool, const void *ins, void *stream);

/* --------------------------------------- a 4-bit key/value cache for decode
 * What a decode step needs between its q/k/v projections and its output
 * projection, no reference counterpart: the norm and rotation of queries and
 * keys, a cache that holds keys and values in 4 bits, attention over it, and
 * eviction from it. Device pointers only (a cache lives on the device); all
 * activations f32, in rows of heads * d values with a row stride ld (in
 * values), so q, k and v may be slices of one projection's output. Rows whose
 * pointer or stride is not a multiple of 16 bytes are read value by value.
 * Lengths and positions are device arrays, so that a captured step can be
 * replayed; what cannot be checked on the host is checked on the device and
 * reported by vmlm_sync (VMLM_ERR_OPERATOR).
 *
 * A cache holds [n_seq][n_kv][cap] rows (slots) of d = 64, 128 or 256 values,
 * keys and values alike: codes d/2 bytes (column p in byte p/2, the low nibble
 * when p is even), and for every 32 columns two halves (step, base). A code c
 * stands for half(step * (16 + c) + base). A group x of 32 columns becomes, in
 * f32 operations rounded one by one, after |x| is clamped to 16384:
 *   step = half((max - min) * (1/15)), base = half(min - 16 * step),
 *   c = clamp(rint((x - base) * (1 / step)) - 16, 0, 15), or 0 where step = 0.
 * A NaN makes its whole group NaN. Buffers belong to the caller (16-byte
 * aligned): k and v n_seq * n_kv * cap * d/2 bytes, ks and vs
 * n_seq * n_kv * cap * d/32 * 4 bytes; cap is at most 2^31 - 8192. Slots at or
 * behind a sequence's length are never read: they may hold anything. */
typedef struct vmlm_kv4 {
  void *k, *v;   /* codes */
  void *ks, *vs; /* (step, base) */
  size_t n_seq, n_kv, cap, d;
} vmlm_kv4;

/* The rotation of a head's first `rot` columns (a multiple of 16, at most d):
 * (a, b) -> (a cos - b sin, b cos + a sin) on the pairs (i, i + rot/2), or
 * (2i, 2i + 1) when interleaved != 0, with row pos[token] of the tables
 * [n_pos][rot/2]. A position outside [0, n_pos) leaves the token's rows
 * unwritten and is reported by vmlm_sync. */
typedef struct vmlm_rope {
  const float *cos_t, *sin_t;
  const int32_t *pos;
  size_t n_pos, rot;
  int interleaved;
} vmlm_rope;

/* Queries and keys after their projections: for each head
 * y = x * (1 / sqrt(sum(x^2) / d + eps)) * g (g = gq or gk, [d]; NULL: no
 * norm), then the rotation (rope NULL: none). qo and ko may be q and k (same
 * stride) and may share no other memory with them. n_q = 0 or n_kv = 0 leaves
 * that part out. */
VMLM_API int vmlm_qk_norm_rope_dev(const float *q, size_t ldq, const float *k, size_t ldk, const float *gq,
                                   const float *gk, float eps, const vmlm_rope *rope, float *qo, size_t ldqo,
                                   float *ko, size_t ldko, size_t tokens, size_t n_q, size_t n_kv, size_t d,
                                   void *stream);

/* The same for q (n_q = 0: none) and k, and the m new tokens of each sequence
 * (rows b * m + t) written to slots len[b] + t in 4 bits, v as it is. len is
 * not changed; len[b] < 0 marks an idle sequence, for which nothing is
 * written to the cache; its queries are written where their positions lie in the
 * table, and no position outside it is reported. A slot behind cap is not written and is reported by
 * vmlm_sync. qo may be q (same stride) and may share no other memory with q, k
 * or v. */
VMLM_API int vmlm_kv4_append_dev(const vmlm_kv4 *cache, const float *q, size_t ldq, float *qo, size_t ldqo,
                                 size_t n_q, const float *k, size_t ldk, const float *v, size_t ldv, const float *gq,
                                 const float *gk, float eps, const vmlm_rope *rope, const int32_t *len, size_t m,
                                 void *stream);

/* Values of `count` rows from slot start[b] of each sequence and kv head, as
 * halves (bits): k, v [n_seq][n_kv][count][d], 16-byte aligned. Rows at or
 * behind end[b] read as zeros; a row before end[b] outside the cache reads as
 * zeros and is reported by vmlm_sync. */
VMLM_API int vmlm_kv4_read_dev(const vmlm_kv4 *cache, const int32_t *start, const int32_t *end, size_t count,
                               uint16_t *k, uint16_t *v, void *stream);

/* Attention of the m newest tokens of each sequence (rows b * m + t of q and
 * out, n_q heads, n_q / n_kv of them to a kv head): token t sees the slots
 * j < len[b] - (m - 1 - t), len[b] counting the m tokens themselves.
 * A slot that a token does not see has no part in its output, whatever bits it
 * holds; a NaN or an infinity in a value reaches the tokens that see it, as
 * one of the two.
 *   out = sum_j p_j v_j, p = softmax(scale * q . k_j); no visible slot: zeros.
 * With w_out ([n_seq][n_kv][cap]), the weight that each slot received is
 * accumulated: w_out[j] = w_in[j] + the sum of p_j over the tokens and the kv
 * head's query heads for j < len[b] (w_in counts as 0 for the m newest slots
 * and where it is NULL; w_in and w_out may be the same). Other slots of w_out
 * are not written. out may not overlap q. A len above cap is taken as cap and reported by vmlm_sync.
 * Sums are f32. Queries are held as two halves (22 bits of a row's largest
 * value), softmax weights as two (21 bits, and down to 2^-38 of a row's
 * largest); products of these with cached values are exact. With w_out the call
 * holds n_seq * n_kv * cap scores a query row of a kv head in workspace (f32;
 * rows rounded up to even chunks of a multiple of 4, for 25 rows and more of
 * d = 256 to chunks of 32, 48, 64 or 80): a prompt's last tokens are a cheaper
 * source of weights than all of them. Every chunk of rows walks all slots of
 * its sequence, those that none of its tokens sees too. */
VMLM_API int vmlm_kv4_attn_dev(const vmlm_kv4 *cache, const float *q, size_t ldq, const int32_t *len, float *out,
                               size_t ldo, size_t m, size_t n_q, float scale, const float *w_in, float *w_out,
                               void *stream);

/* Keep `keep` slots of each sequence and kv head and copy them, in slot order,
 * to slots 0 .. of another cache with the same n_seq, n_kv and d: the first
 * `first` and the last `recent` slots, and of the others those with the
 * largest w ([n_seq][n_kv][cap]; of equal ones the lower slots, a NaN last). A
 * sequence with len[b] <= keep keeps all. idx [n_seq][n_kv][keep] receives the
 * kept slots (-1 behind them), w_out (may be NULL) their weights (0 behind
 * them), len_out[b] = min(len[b], keep) (0 for a negative len). src is not
 * changed. No output may overlap an input (len_out is not len) or another
 * output. */
VMLM_API int vmlm_kv4_evict_dev(const vmlm_kv4 *src, const vmlm_kv4 *dst, const float *w, const int32_t *len,
                                size_t keep, size_t first, size_t recent, int32_t *idx, float *w_out,
                                int32_t *len_out, void *stream);

/* ------------------------------------------------- device-pointer GEMMs
 * Same arithmetic as the host entry points; pointers are device memory of the
 * current CUDA device; `stream` is a cudaStream_t. NULL selects the library's
 * own stream, so the legacy default stream must be passed as cudaStreamLegacy
 * ((void *)1). */
VMLM_API int vmlm_gemm_nt_int8_dev(const float *a, const int8_t *q, const float *scale, float *c, size_t m, size_t n,
                          size_t k, void *stream);
VMLM_API int vmlm_gemm_nt_bf16_dev(const float *a, const uint16_t *b, float *c, size_t m, size_t n, size_t k,
                          void *stream);
VMLM_API int vmlm_gemm_i8i8_dev(const int8_t *x, const int8_t *w, const float *scale, float *c, int32_t *acc, size_t m,
                       size_t n, size_t k, void *stream);
VMLM_API int vmlm_gemm_nt_f32_dev(const float *a, const float *b, float *c, size_t m, size_t n, size_t k, int acc,
                                  void *stream);
VMLM_API int vmlm_gemm_f32_dev(const float *a, const float *b, float *c, size_t m, size_t n, size_t k, int acc,
                               void *stream);

/* Allocation-free variant of vmlm_gemm_nt_int8_dev; it has no counterpart in
 * the reference. Same arithmetic and arguments, but every byte of scratch the
 * call needs comes from one fixed array of device memory inside the library
 * (about 4.7 MB, held on each GPU that loads the library until the process
 * exits), so the call never allocates or frees device memory. It is meant for
 * callers that must not allocate while they run, such as an engine that
 * reserves all of its device memory at start-up and cannot let a kernel call
 * fail or stall on cudaMalloc inside its per-token loop.
 *   Limits: m <= 16, n <= 131072, k <= 16384; larger sizes return
 *   VMLM_ERR_SHAPE and do nothing.
 *   The first call on a device performs one-time set-up on that device (looks
 *   up the array's device address, clears it, sets the kernel's shared-memory
 *   limit); make that first call before any stream capture.
 *   All calls share the array and it keeps the last call's contents, so calls
 *   that overlap on the GPU (different streams, or different host threads on
 *   the same device) race; order them on one stream.
 *   Streams: NULL here means the CUDA legacy default stream, NOT the library
 *   stream that NULL selects in the other _dev entry points (a library stream
 *   would need the per-device context, which allocates). Pass the caller's
 *   stream explicitly to order these calls with the caller's other work.
 *   Errors: a kernel that gives up a bounded wait records it in the array's
 *   own error word. vmlm_sync reads that word (after waiting for the whole
 *   device), returns VMLM_ERR_DEVICE_TIMEOUT, and clears the word with the
 *   split-tile counters and slots an aborted launch can leave behind, so the
 *   next call starts clean; on a device that has only seen allocation-free
 *   calls, vmlm_sync allocates nothing either. */
VMLM_API int vmlm_gemm_nt_int8_dev_noalloc(const float *a, const int8_t *q, const float *scale, float *c, size_t m,
                                           size_t n, size_t k, void *stream);

/* Wait for the given stream (NULL = library stream), then read and clear the
 * device error word of the current device: VMLM_OK or VMLM_ERR_DEVICE_TIMEOUT
 * (or the operator / argument error a device-side check recorded). After an
 * error the library's split-tile counters and slots are cleared too. If the
 * allocation-free entry point has been used on this device, its own error word
 * is read as well, after waiting for the whole device. */
VMLM_API int vmlm_sync(void *stream);

/* Host-pointer calls over many activation rows (at least two chunks of 128 or
 * 256 rows, 2 MB of input and output) run as a pipeline of row chunks: the
 * copy in of one chunk, the GEMM of the previous one and the copy out of the
 * one before overlap. At most max_chunks chunks per call (2..8); 1 turns the
 * pipeline off; 0 restores the default (4). Results do not depend on it.
 * VMLM_ERR_ARG outside [0, 8]. */
VMLM_API int vmlm_set_host_pipeline(int max_chunks);

/* Number of kernels this library has launched since vmlm_init (diagnostics). */
VMLM_API uint64_t vmlm_launch_count(void);

/* ------------------------------------------------------------------------
 * Multi-GPU, row-sharded calls (no reference counterpart; the reference is
 * single-process CPU code). For a weight too large or too slow for one GPU
 * (the LM head, an FFN projection), each of `world` ranks (one process per
 * GPU of one node) holds rows [rank*R, rank*R + R) of W, R = ceil(n / world),
 * and computes those output columns; the all-gather is part of the call, and
 * C is complete on every rank in stream order after it:
 *   - small outputs (under 16 MB sent to the peers per call): the GEMM
 *     epilogue stores every output value straight into every rank's full
 *     C[m][n] over NVLink, and the kernel ends once all ranks' outputs have
 *     landed in its C;
 *   - larger outputs on two GPUs: the GEMM writes this rank's column slice of
 *     its own C (int8 x int8: in row chunks) and the copy engines send each
 *     finished block to the peer over NVLink while the next chunk computes; a
 *     small kernel then waits until every rank's copies into this C are done;
 *   - larger int8 x int8 outputs on more than two GPUs: as on two, but a
 *     kernel beside the GEMM pushes each finished row chunk to every peer;
 *     Q8 calls on more than two GPUs use the fused epilogue stores.
 *   c_peers[q]     rank q's C [m][n] row-major, mapped into this process
 *                  (c_peers[rank] is this rank's own C)
 *   inbox_peers[q] rank q's inbox: one 4-byte device word, reset with
 *                  vmlm_sharded_reset before its first call, mapped here
 * Every rank makes the same calls in the same order, each on one stream. A
 * rank waits at most 5 s for the others; then the call reports
 * VMLM_ERR_DEVICE_TIMEOUT from vmlm_sync and every rank must call
 * vmlm_sharded_reset on its inbox (after a host barrier) before the next call.
 * Requirements: 1 <= world <= 8, k % 16 == 0, k <= 131072, every rank gets
 * at least one row. */
VMLM_API int vmlm_sharded_gemm_nt_int8_dev(const float *a, const int8_t *q_shard, const float *scale_shard,
                                          float *const *c_peers, unsigned *const *inbox_peers, int rank, int world,
                                          size_t m, size_t n, size_t k, void *stream);
VMLM_API int vmlm_sharded_gemm_i8i8_dev(const int8_t *x, const int8_t *w_shard, const float *scale_shard,
                                       float *const *c_peers, unsigned *const *inbox_peers, int rank, int world,
                                       size_t m, size_t n, size_t k, void *stream);
/* Zero this rank's inbox and forget its call count: before the first call on
 * a newly allocated inbox word (the library counts calls per inbox address),
 * and after an error. */
VMLM_API int vmlm_sharded_reset(unsigned *inbox);

/* Sharing device buffers between the ranks' processes. vmlm_ipc_handle
 * writes VMLM_IPC_HANDLE_BYTES bytes naming the allocation that holds dptr
 * and dptr's offset in it; vmlm_ipc_open maps it in another process of the
 * same node (each allocation once, however often it is opened) and returns
 * the same address there; vmlm_ipc_close undoes one open. */
#define VMLM_IPC_HANDLE_BYTES 72
VMLM_API int vmlm_ipc_handle(const void *dptr, void *handle);
VMLM_API int vmlm_ipc_open(const void *handle, void **dptr);
VMLM_API int vmlm_ipc_close(void *dptr);

/* Diagnostics, no reference counterpart: when enabled, every tensor-core GEMM
 * launch is bracketed by a CUDA event pair on its stream (programmatic
 * dependent launch is then not used). vmlm_profile_take waits for the
 * recorded launches and returns their summed device time and count. */
VMLM_API int vmlm_profile_enable(int on);
VMLM_API int vmlm_profile_take(double *gemm_ms, uint64_t *launches);
/* The kernel and tile plan of the last profiled launch, as text (empty before
 * the first), truncated to n bytes with a terminating zero. */
VMLM_API int vmlm_profile_kernel(char *buf, size_t n);

/* Diagnostics, no reference counterpart: the dense tensor-core rate of this
 * device. One CTA per SM issues iters x 4 back-to-back tcgen05.mma of
 * 128 x 256 x (32 bytes of K) on operands held in shared memory (no memory
 * traffic): kind 0 = kind::f16 with bf16 operands (f32 accumulate), kind 1 =
 * kind::i8 (s32 accumulate). Returns the rate in 10^12 dense multiply-adds x 2
 * per second (TFLOP/s or TOP/s) and the kernel's event time in ms. iters in
 * [1, 200000]. */
VMLM_API int vmlm_probe_mma_peak(int kind, int iters, double *tops, double *ms);

/* Diagnostics, no reference counterpart: when enabled (max_ctas > 0), every
 * tensor-core GEMM launch of up to max_ctas CTAs records 16 values per CTA:
 * 8 globaltimer stamps in ns (start, producer past the wait for the previous
 * kernel, TMA issue done, first stage consumed, last accumulator committed,
 * first accumulator in the epilogue, epilogue done, TMEM released), 4 summed
 * waits in ns (producer for free stages, MMA for loaded stages, MMA for a
 * free accumulator, epilogue for a finished accumulator), 3 summed epilogue
 * phases in ns (split tiles: publishing partials, counting arrivals,
 * finishing; whole tiles: TMEM loads, finishing and storing, unused)
 * and the count of work items * 65536 + tiles finished. Each launch
 * overwrites the previous one. 0 disables and frees. */
VMLM_API int vmlm_trace_enable(int max_ctas);
VMLM_API int vmlm_trace_take(uint64_t *stamps, size_t n_values);

#ifdef __cplusplus
}
#endif

#endif /* VMLM_CUDA_H */
