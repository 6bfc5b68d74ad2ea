/*
 * libsupra_attn — C ABI of the B200 (sm_100a) fused attention operator of Supra2-Img.
 *
 * The operator surface mirrors the reference's JavaScript entry point
 *   attention(gpu, {q, k, v, Lq, Lk, H, D, ldq, ldk, ldv, qOff, kOff, vOff, oOff, scale, bias, out})
 * (app/gpu/ops.js:103-149) and the runtime it records into (app/gpu/device.js:41-269):
 *
 *   - q is [Lq, ldq] row-major fp32; head h of query row i is q[qOff + i*ldq + h*D + 0..D).
 *     k / v likewise with ldk / ldv and kOff / vOff, over Lk key rows.
 *   - The output row i is written at out[oOff + i*(H*D) + h*D + 0..D): row stride H*D.
 *   - scale multiplies the scores; the reference's default is 1/sqrt(D) (app/gpu/ops.js:109).
 *   - bias, when present, is an additive score bias laid out [H, Lq, Lk] (T5 relative
 *     positions, app/models/t5.js:55-65); it is added after scaling (app/gpu/kernels.js:34).
 *   - All offsets, strides and sizes are in ELEMENTS (floats), never bytes.
 *
 * Execution model ("record now, submit at flush", app/gpu/device.js:1-5,207-253):
 *   supra_attn_enqueue() validates a problem synchronously and records it; nothing runs yet.
 *   supra_attn_flush() groups every recorded problem by kernel configuration and issues one
 *   grouped launch per group on the context's stream; supra_attn_sync() waits and reports
 *   device-side failures (the reference surfaces asynchronous errors at read/sync,
 *   app/gpu/device.js:186,258,262-268). A recorded problem that reads memory written by an
 *   earlier recorded problem (or writes memory an earlier one touches) flushes the queue
 *   first, so results never depend on grouping.
 *
 * Every function returns a status code (SUPRA_ATTN_OK on success) and never throws or aborts.
 * supra_attn_last_error() returns the message of the most recent failure on a context.
 * A context is bound to one device and is not thread-safe (one context per host thread),
 * like the reference's single-threaded GPU object.
 */
#ifndef SUPRA_ATTN_H
#define SUPRA_ATTN_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define SUPRA_ATTN_API __attribute__((visibility("default")))
#else
#define SUPRA_ATTN_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---------------------------------------------------------------------- */
#define SUPRA_ATTN_OK 0
#define SUPRA_ATTN_EINVAL 1   /* bad argument: sizes, alignment, bounds, aliasing, unknown flag */
#define SUPRA_ATTN_ENOMEM 2   /* device or pinned host allocation failed                      */
#define SUPRA_ATTN_ECUDA 3    /* a CUDA runtime/driver call failed                            */
#define SUPRA_ATTN_ETIMEOUT 4 /* a device-side bounded wait ran out (reported at sync)        */
#define SUPRA_ATTN_EDEVICE 5  /* the device reported an error status (reported at sync)       */
#define SUPRA_ATTN_ESTATE 6   /* call not allowed in the context's current state              */

/* ---- numeric variants -------------------------------------------------------------------- */
#define SUPRA_ATTN_FP32 0 /* FFMA kernel, fp32 throughout: matches torch CPU fp32 to <=1e-5 */
/* tcgen05 tensor-core kernel with TF32 operands, fp32 accumulate. Covers head dim 64 with
 * whole-row, 16-byte aligned buffers (fused kernel, with or without a bias), and head dims above
 * 128 without a bias and with Lk >= 32 (Q K^T and P V on the tensor-core linear, the row softmax
 * between them); other requests run the FP32 kernels. */
#define SUPRA_ATTN_TF32 1
/* tcgen05 kernels with every operand split x = hi + lo (hi = TF32(x), lo = x - hi) and each
 * product formed as lo*hi + hi*lo + hi*hi ("3xTF32"): fp32-class accuracy on the tensor cores.
 * Same coverage as SUPRA_ATTN_TF32; other requests run the FP32 kernels. */
#define SUPRA_ATTN_TF32X3 2

/* ---- descriptor flags -------------------------------------------------------------------- */
#define SUPRA_ATTN_F_DEFAULT_SCALE 0x1u /* ignore .scale, use 1/sqrt(D) (ops.js:109 default) */
/* .bias is T5's relative-attention-bias TABLE, not an expanded bias: bias points at
 * bias_size >= buckets*H floats laid out [buckets, H] (encoder.block.0...relative_attention_bias
 * .weight, app/models/t5.js:44), and the kernels form the score bias themselves as
 *   bias[h, i, j] = table[relativeBucket(j - i)*H + h]   (app/models/t5.js:14-23,55-65)
 * with the bidirectional bucket of supra_attn_relative_bucket. .bias_param carries the bucket
 * parameters: buckets in bits 0-15, max_distance in bits 16-31. Not in the reference: its T5
 * builds the [H, L, L] bias on the host and uploads it per encode (app/models/t5.js:73); this
 * saves those 4*H*L*L bytes per prompt and the host loop. */
#define SUPRA_ATTN_F_T5_TABLE 0x2u

typedef struct supra_attn_ctx supra_attn_ctx;

/*
 * One attention problem: all H heads of one call of ops.attention (app/gpu/ops.js:109).
 * The *_size fields give the number of floats the caller owns at each pointer; every
 * element the problem reads or writes is checked against them at enqueue, so an
 * out-of-range offset is an EINVAL instead of a device fault. Pass 0 only for bias when
 * bias is NULL.
 */
typedef struct supra_attn_desc {
  const float* q;
  const float* k;
  const float* v;
  float* out;
  const float* bias; /* NULL, [H, Lq, Lk] additive score bias, or a T5 table (SUPRA_ATTN_F_T5_TABLE) */
  int64_t q_size, k_size, v_size, out_size, bias_size;
  int64_t ldq, ldk, ldv;
  int64_t q_off, k_off, v_off, o_off;
  int32_t Lq, Lk, H, D;
  float scale;
  int32_t variant; /* SUPRA_ATTN_FP32, SUPRA_ATTN_TF32 or SUPRA_ATTN_TF32X3 */
  uint32_t flags;  /* SUPRA_ATTN_F_* */
  uint32_t bias_param; /* with SUPRA_ATTN_F_T5_TABLE: buckets | max_distance << 16; else 0 */
} supra_attn_desc;

/* ---- context ----------------------------------------------------------------------------- */
/* Replaces GPU.create (app/gpu/device.js:92-118): binds a context to a CUDA device and
 * creates its stream, descriptor ring and device status word. Its first attention flush adds a
 * device table of TMA tensor maps (2 MiB, kept for the context's life; larger only if one flush
 * needs more than 16384 maps). */
SUPRA_ATTN_API int supra_attn_create(int device, supra_attn_ctx** out);
/* Flushes, synchronises and frees everything the context owns. NULL is a no-op. */
SUPRA_ATTN_API int supra_attn_destroy(supra_attn_ctx* ctx);
/* Runs subsequent launches and copies on a caller-owned cudaStream_t (NULL = the context's
 * own non-blocking stream; pass cudaStreamLegacy, (void*)1, for the legacy default stream).
 * Flushes and waits for pending work on the previous stream first. */
SUPRA_ATTN_API int supra_attn_set_stream(supra_attn_ctx* ctx, void* cuda_stream);
SUPRA_ATTN_API const char* supra_attn_last_error(const supra_attn_ctx* ctx);
/* Message for a status code. */
SUPRA_ATTN_API const char* supra_attn_status_string(int status);

/* ---- tensors (the Tensor/BufferPool surface, app/gpu/device.js:41-88,144-191) ------------ */
/* gpu.empty(shape): a pooled device buffer of n floats (size-bucketed like BufferPool.round). */
SUPRA_ATTN_API int supra_attn_tensor_alloc(supra_attn_ctx* ctx, int64_t n, float** dptr);
/* Tensor.release(): flushes recorded work, then returns the buffer to the pool. */
SUPRA_ATTN_API int supra_attn_tensor_free(supra_attn_ctx* ctx, float* dptr);
/* fromArray / write: flushes, then copies n floats host->device (stream-ordered). */
SUPRA_ATTN_API int supra_attn_upload(supra_attn_ctx* ctx, float* dst, const float* src, int64_t n);
/* The same for n bytes at any address: tensors of other element types. */
SUPRA_ATTN_API int supra_attn_upload_bytes(supra_attn_ctx* ctx, void* dst, const void* src, int64_t n);
/* read(): flushes, copies n floats device->host and waits for them. */
SUPRA_ATTN_API int supra_attn_download(supra_attn_ctx* ctx, float* dst, const float* src, int64_t n);
/* Page-locked host memory for fast upload/download (freed with supra_attn_host_free). */
SUPRA_ATTN_API int supra_attn_host_alloc(supra_attn_ctx* ctx, int64_t n, float** hptr);
SUPRA_ATTN_API int supra_attn_host_free(supra_attn_ctx* ctx, float* hptr);

/* ---- the operator (app/gpu/ops.js:103-149) ------------------------------------------------ */
/* Validates and records one problem. Synchronous EINVAL mirrors the reference's synchronous
 * throw (app/gpu/ops.js:122, app/gpu/device.js:208). */
SUPRA_ATTN_API int supra_attn_enqueue(supra_attn_ctx* ctx, const supra_attn_desc* desc);
/* Validates a descriptor exactly as supra_attn_enqueue does, without a context or a device
 * (pure host function). Writes the message of a failure into msg (cap bytes, may be NULL). */
SUPRA_ATTN_API int supra_attn_check_desc(const supra_attn_desc* desc, char* msg, int32_t cap);
/* Records n problems (an explicit varlen batch); all or none are recorded. */
SUPRA_ATTN_API int supra_attn_enqueue_batch(supra_attn_ctx* ctx, const supra_attn_desc* descs, int32_t n);
/* GPU.flush (app/gpu/device.js:243-253): one grouped launch per kernel configuration. */
SUPRA_ATTN_API int supra_attn_flush(supra_attn_ctx* ctx);
/* GPU.sync (app/gpu/device.js:255-259): flush, wait, and check the device status word.
 * *device_status (may be NULL) receives the raw device status (0 = clean). */
SUPRA_ATTN_API int supra_attn_sync(supra_attn_ctx* ctx, int32_t* device_status);
/* Number of problems recorded and not yet flushed. */
SUPRA_ATTN_API int supra_attn_pending(const supra_attn_ctx* ctx, int32_t* n);

/* ---- T5 relative-position bias (app/models/t5.js:14-23,55-65) ----------------------------- */
/* relativeBucket(rel, buckets, maxDistance) (app/models/t5.js:14-23), bidirectional, with the
 * same float32 rounding steps. Pure host function. Returns the bucket, or -1 on bad input. */
SUPRA_ATTN_API int32_t supra_attn_relative_bucket(int32_t rel, int32_t buckets, int32_t max_distance);
/* T5Encoder.positionBias(L) (app/models/t5.js:55-65) computed on the device:
 *   out[(h*L + i)*L + j] = table[relativeBucket(j - i)*H + h]
 * table is a DEVICE pointer to table_size >= buckets*H floats laid out [buckets, H]
 * (encoder.block.0...relative_attention_bias.weight, app/models/t5.js:44); out is a device
 * pointer to out_size >= H*L*L floats. Stream-ordered with the context's other work
 * (recorded attention is flushed first). */
SUPRA_ATTN_API int supra_attn_position_bias(supra_attn_ctx* ctx, const float* table, int64_t table_size,
                                            int32_t buckets, int32_t max_distance, int32_t H, int32_t L,
                                            float* out, int64_t out_size);

/* ---- linear: the projections beside the attention (ops.linear, app/gpu/ops.js:35-43) -------- */
/* One y = x W^T (+ bias) problem, recorded like an attention problem (same queue, same hazard
 * tracking, one grouped launch per flush). x: M rows of K floats, row stride ldx, first row at
 * x_off; w: [N, K] row-major with row stride ldw >= K (the reference's weight layout, x @ W^T);
 * bias: N floats or NULL; y: M rows of N floats, row stride ldy >= N, first row at y_off. All
 * counts in floats. SUPRA_ATTN_FP32: fp32 FFMA. SUPRA_ATTN_TF32 / SUPRA_ATTN_TF32X3 with K >= 32: on
 * the tensor cores, TF32 products or the split form (three TF32 products per product, held to the
 * FP32 tolerance); operands are read through tensor maps, in place for the TF32 products when
 * 16-byte aligned with row strides of a multiple of 4 floats, else (and always for the split
 * form) first copied as hi / lo parts, x normalised when asked, into a context-owned buffer.
 * Shallower products run the FFMA kernel.
 * Two optional fusions (the VAE mid-block attention, app/models/vae.js:77-94):
 *   - gn != NULL: x is GroupNorm-ed on the way in (ops.groupnorm, app/gpu/ops.js:82-92,
 *     app/gpu/kernels.js:117-162): x rows form images of gn->rows_per_image rows; per image and
 *     group of K / gn->groups channels the library computes (mean, 1/sqrt(var + eps)) in an extra
 *     launch, and the product uses (x - mean) * rstd * gamma[k] + beta[k] (then SiLU if
 *     gn->silu) in place of x. Needs x_off == 0 and ldx == K.
 *   - resid != NULL: y = resid + (x W^T + bias), resid rows of stride ldr at r_off (the residual
 *     add of app/models/vae.js:91). resid may be y itself (same rows: r_off == y_off and
 *     ldr == ldy), which is the reference's in-place `out: x, resid: true` (app/models/dit.js:
 *     175,187,193); otherwise it may not overlap y.
 *   - gate != NULL (needs resid): y = resid + gate[g_off + n] * (x W^T + bias), the gated
 *     residual of the DiT blocks (app/gpu/gemm.js:10,135, app/models/dit.js:175,193).
 *   - ln != NULL (not with gn): x is LayerNorm-ed on the way in, each row over its K channels
 *     (ops.layernorm, app/gpu/ops.js:71-79, app/gpu/kernels.js:87-114): the library computes
 *     (mean, 1/sqrt(var + eps)) per row in an extra launch, and the product uses
 *     (x - mean) * rstd, times (1 + mod[scale_off + k]) plus mod[shift_off + k] when ln->mod is
 *     set (adaLN modulation; app/models/dit.js:164,179,189). Needs x_off == 0 and ldx == K.
 *   With gn or ln on the FFMA kernel, a product whose x is read by two or more column tiles
 *   first writes the normalised x once into a context-owned buffer (one more launch), which the
 *   product then reads; products with one column tile normalise each staged x tile.
 *   - act: SUPRA_ATTN_ACT_NONE, _GELU (erf form), _GELU_TANH or _SILU, applied to x W^T + bias
 *     before the gate and the residual (ops.linear's act, app/gpu/gemm.js:9,28-36,130-135).
 * flags must be 0.
 * Cross-attention K/V preparation (app/models/dit.js:137-144) is two calls: ctx_proj, then ONE
 * product with the 14 blocks' kv weights stacked [14*1152, 576]; block b's cross attention then
 * reads K at column 1152*b and V at 1152*b + 576 of rows of stride 14*1152, without a copy. */
typedef struct supra_attn_groupnorm {
  const float* gamma; /* K floats */
  const float* beta;  /* K floats */
  int32_t groups;     /* K % groups == 0 */
  int32_t rows_per_image; /* M % rows_per_image == 0 */
  float eps;          /* the reference uses 1e-6 */
  int32_t silu;       /* nonzero: SiLU after the affine (ops.groupnorm's silu flag) */
} supra_attn_groupnorm;

enum { SUPRA_ATTN_ACT_NONE = 0, SUPRA_ATTN_ACT_GELU = 1, SUPRA_ATTN_ACT_GELU_TANH = 2, SUPRA_ATTN_ACT_SILU = 3 };

typedef struct supra_attn_layernorm {
  const float* mod;   /* NULL: plain LayerNorm; else the modulation vector (mod_size floats) */
  int64_t mod_size;
  int64_t shift_off;  /* LN(x) * (1 + mod[scale_off + k]) + mod[shift_off + k] */
  int64_t scale_off;
  float eps;          /* the reference uses 1e-6 */
  int32_t reserved;   /* 0 */
} supra_attn_layernorm;

typedef struct supra_attn_linear_desc {
  const float* x;
  const float* w;
  const float* bias;
  float* y;
  int64_t x_size, w_size, bias_size, y_size;
  int64_t ldx, ldw, ldy;
  int64_t x_off, y_off;
  int32_t M, N, K;
  int32_t variant;
  uint32_t flags;
  uint32_t act;                   /* SUPRA_ATTN_ACT_* */
  const supra_attn_groupnorm* gn; /* NULL, or GroupNorm x on the way in (copied at enqueue) */
  const float* resid;             /* NULL, or y = resid + ... (rows of stride ldr at r_off) */
  int64_t resid_size, ldr, r_off;
  const float* gate;              /* NULL, or the product is scaled by gate[g_off + n] */
  int64_t gate_size, g_off;
  const supra_attn_layernorm* ln; /* NULL, or LayerNorm x on the way in (copied at enqueue) */
} supra_attn_linear_desc;
SUPRA_ATTN_API int supra_attn_enqueue_linear(supra_attn_ctx* ctx, const supra_attn_linear_desc* desc);
/* Validates a linear descriptor as supra_attn_enqueue_linear does (pure host function). */
SUPRA_ATTN_API int supra_attn_check_linear_desc(const supra_attn_linear_desc* desc, char* msg, int32_t cap);

/* ---- norm and rotation of query and key heads ----------------------------------------------- */
/* Element types of the buffers of the calls below. Strides and offsets count elements of the type. */
enum { SUPRA_ATTN_T_F32 = 0, SUPRA_ATTN_T_F16 = 1, SUPRA_ATTN_T_BF16 = 2 };

/* One operand of a qk_norm call: H heads of D channels in each row, head h of row i at
 * x[x_off + i*ldx + h*D + 0..D), written to y[y_off + i*ldy + h*D + 0..D). y may be x itself with
 * the same offset and stride (in place); otherwise they may not overlap. */
typedef struct supra_attn_qk_operand {
  const void* x;
  void* y;
  const float* w; /* D channel weights shared by the heads, or NULL (ones) */
  int64_t x_size, y_size, w_size;
  int64_t ldx, ldy, x_off, y_off;
  int32_t H;
  int32_t reserved; /* 0 */
} supra_attn_qk_operand;

/* Flags of a qk_norm call. */
#define SUPRA_ATTN_QK_NO_NORM 0x1u     /* rotate only: no RMS norm and no weights */
#define SUPRA_ATTN_QK_INTERLEAVED 0x2u /* pairs (2i, 2i+1) instead of (i, i + rot/2) */

/* RMS norm of every head of the queries and of the keys, with the position rotation in the same
 * pass (not in the reference, whose DiT normalises whole rows and adds its positions):
 *   n = x / sqrt(mean(x^2) + eps) * w                    over the D channels of one head
 *   (y_a, y_b) = (n_a cos - n_b sin, n_b cos + n_a sin)  for the rot/2 channel pairs (a, b) of
 *                                                        the first rot channels; the others stay n
 * with cos = turns[position*rot + i], sin = turns[position*rot + rot/2 + i] for pair i: the caller
 * lays the table out once for its positions (n_turns rows), which may stand for one axis or for
 * a patch grid. position = positions[row], or the row index when positions is NULL. A position
 * outside [0, n_turns) leaves its row unwritten and is reported at sync (SUPRA_ATTN_EDEVICE).
 * Sums and products are held in 32 bits (heads whose squares leave that range come out as such arithmetic has
 * them); the result is rounded once, to `type`.
 * 1 <= D <= 256, even; 0 <= rot <= D, even (0: no rotation, turns and positions NULL). k.H = 0:
 * no keys. Recorded like an attention problem (same queue and hazard tracking). */
typedef struct supra_attn_qk_norm_desc {
  supra_attn_qk_operand q, k;
  const float* turns;
  const int32_t* positions;
  int64_t turns_size, positions_size;
  int32_t M, D, rot, n_turns;
  int32_t type;   /* SUPRA_ATTN_T_* of x and y */
  uint32_t flags; /* SUPRA_ATTN_QK_* */
  float eps;
  int32_t reserved; /* 0 */
} supra_attn_qk_norm_desc;
SUPRA_ATTN_API int supra_attn_enqueue_qk_norm(supra_attn_ctx* ctx, const supra_attn_qk_norm_desc* desc);
/* Validates as supra_attn_enqueue_qk_norm does (pure host function). */
SUPRA_ATTN_API int supra_attn_check_qk_norm_desc(const supra_attn_qk_norm_desc* desc, char* msg, int32_t cap);

/* ---- the paged 8-bit K/V cache ---------------------------------------------------------------- */
/* Keys and values of many sequences (prompts) held in 8 bits, the reference's cached FP32 K/V
 * (app/models/dit.js:137-144, app/pipeline.js:97-117) in a quarter of the bytes. The pool is split into blocks of block_tokens tokens, and each block has one scale per head, for K and
 * for V: value = code * scale[block*H + head]. Codes of one block and head are contiguous:
 *   codes[((block*H + head)*block_tokens + slot)*D + channel]
 * SUPRA_ATTN_CACHE_INT8: signed bytes in [-127, 127]; SUPRA_ATTN_CACHE_E4M3: 8-bit floats with 4
 * exponent and 3 mantissa bits (the two bytes that stand for NaN are no codes, and no write makes them: what one
 * gives at a token in use may also reach rows of its sequence that do not see the token). D is a multiple of 16 up to 128, block_tokens 16, 32, 64 or 128;
 * k and v are 16-byte aligned. All four arrays are the caller's. */
enum { SUPRA_ATTN_CACHE_INT8 = 0, SUPRA_ATTN_CACHE_E4M3 = 1 };
typedef struct supra_attn_cache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t k_size, v_size;             /* bytes, >= blocks*H*block_tokens*D */
  int64_t k_scale_size, v_scale_size; /* floats, >= blocks*H */
  int32_t blocks, block_tokens, H, D;
  int32_t format;   /* SUPRA_ATTN_CACHE_* */
  int32_t reserved; /* 0 */
} supra_attn_cache;

/* The sequences of one call. All arrays are device memory, read when the call runs: their contents
 * may change between calls, and between replays of a captured one. Token t of sequence b sits in
 * block table[b*ld_table + t / block_tokens], slot t % block_tokens. The call's rows (queries, or
 * K/V rows to write or read) of sequence b are rows row_start[b] .. row_start[b+1]-1 of its
 * operands, or b*max_rows .. (b+1)*max_rows-1 when row_start is NULL; with n rows, row i stands
 * at token lengths[b] - n + i (lengths count the tokens that the call writes).
 * rows bounds row_start[B] (with row_start NULL it is B*max_rows), max_rows the rows of one
 * sequence and max_len its length; operand rows at and after row_start[B] are neither read nor
 * written. A sequence outside these bounds is left out (its output rows stay as they are), tokens
 * in a block outside [0, blocks) are left out, and either is reported at sync
 * (SUPRA_ATTN_EDEVICE). Table entries past a sequence's last block are not read. */
typedef struct supra_attn_cache_batch {
  const int32_t* lengths;   /* B */
  const int32_t* table;     /* B rows of ld_table block numbers */
  const int32_t* row_start; /* B + 1, ascending, or NULL */
  int64_t lengths_size, table_size, row_start_size;
  int64_t rows;
  int32_t B, ld_table;
  int32_t max_rows, max_len;
} supra_attn_cache_batch;

/* K/V rows beside the cache: row r of the keys at k[k_off + r*ldk + h*D + 0..D), values likewise. */
typedef struct supra_attn_cache_rows_desc {
  supra_attn_cache cache;
  supra_attn_cache_batch seqs;
  void* k; /* cache_write reads them, cache_read writes them */
  void* v;
  int64_t k_size, v_size, ldk, ldv, k_off, v_off;
  int32_t type;   /* SUPRA_ATTN_T_* */
  uint32_t flags; /* 0 */
} supra_attn_cache_rows_desc;

/* Quantises rows into the cache: the last n tokens of each sequence are written, and the tokens
 * before them in the first touched block keep their values. Per block and head, over the block's
 * written tokens,
 *   s = max(amax|x|, 2^-100) * (1/qmax)         qmax 127 (INT8) or 448 (E4M3)
 *   s = max(s, old scale)                       if the block already held earlier tokens
 *   code = nearest (ties to even) to x * (1/s); the held codes become the nearest to
 *   code * (old scale / s) when the scale grew
 * s, 1/qmax, 1/s and the ratio are fp32; each product is rounded once, to the code. A value that is not
 * finite makes its block's scale NaN (and its codes 0): the block then reads as NaN. Slots after a
 * sequence's last token keep their bytes and stand for nothing. Blocks written by one call have to
 * be distinct: a block given to two written tokens ranges of one call gets unspecified values. */
SUPRA_ATTN_API int supra_attn_enqueue_cache_write(supra_attn_ctx* ctx, const supra_attn_cache_rows_desc* desc);
SUPRA_ATTN_API int supra_attn_check_cache_write_desc(const supra_attn_cache_rows_desc* desc, char* msg, int32_t cap);
/* Reads the last n tokens of each sequence back: code * scale, rounded to `type`. */
SUPRA_ATTN_API int supra_attn_enqueue_cache_read(supra_attn_ctx* ctx, const supra_attn_cache_rows_desc* desc);
SUPRA_ATTN_API int supra_attn_check_cache_read_desc(const supra_attn_cache_rows_desc* desc, char* msg, int32_t cap);

/* Flags of a cache_attention call. */
#define SUPRA_ATTN_CA_DEFAULT_SCALE 0x1u /* ignore .scale, use 1/sqrt(D) */
#define SUPRA_ATTN_CA_CAUSAL 0x2u        /* row i of n sees tokens 0 .. length - n + i */

/* Attention of query rows over the cache: softmax(scale * q k^T) v per head, over the sequence's
 * tokens (causal: up to the row's own token). H query heads, a multiple of cache.H: heads
 * g*H/cache.H .. (g+1)*H/cache.H-1 read the cache's head g. Row r, head h of the queries at
 * q[q_off + r*ldq + h*D], of the result at out[o_off + r*ldo + h*D]. A row that sees no token
 * (an empty sequence, or a causal row before the first token) is 0. blocks*H*block_tokens is below 2^31.
 * The codes enter the products exactly; scores, softmax statistics and the sums over tokens are held in 32
 * bits. For the products on the tensor cores SUPRA_ATTN_T_F16 and _BF16 requests round each probability to 11
 * bits (their queries keep all of theirs, but for BF16 channels below 2^-27 of a head's largest);
 * SUPRA_ATTN_T_F32 requests hold queries and probabilities as two such parts, 22 bits: errors of about 4e-7 where
 * sums in FP32 throughout have 1e-7 to 3e-7. */
typedef struct supra_attn_cache_attn_desc {
  supra_attn_cache cache;
  supra_attn_cache_batch seqs;
  const void* q;
  void* out;
  int64_t q_size, out_size, ldq, ldo, q_off, o_off;
  int32_t H;
  int32_t type; /* SUPRA_ATTN_T_* of q and out */
  float scale;
  uint32_t flags; /* SUPRA_ATTN_CA_* */
} supra_attn_cache_attn_desc;
SUPRA_ATTN_API int supra_attn_enqueue_cache_attention(supra_attn_ctx* ctx, const supra_attn_cache_attn_desc* desc);
SUPRA_ATTN_API int supra_attn_check_cache_attention_desc(const supra_attn_cache_attn_desc* desc, char* msg,
                                                         int32_t cap);
/* The launches of these four calls take their descriptors as kernel arguments and use no memory of
 * the context but its status word and, for cache_attention where few rows meet a long cache, a
 * workspace ordered on the context's stream, which inside a stream capture belongs to the graph. So a
 * flush of them alone (profiling off) may be captured into a CUDA graph on the context's stream, a
 * context's first flush among them, and graphs captured from one context may run at the same time where
 * their own operands allow it. Release such graphs before the context. */

/* ---- profiling (the reference's Profiler, app/gpu/device.js:91-99,222-233,272-325) -------- */
/* When on, every grouped launch is bracketed by CUDA events on the launching stream and
 * aggregated by kernel name with its algorithmic FLOPs (4*Lq*Lk*D*H, app/gpu/ops.js:116) and
 * bytes (Q+K+V+O read/written once, plus the bias). */
SUPRA_ATTN_API int supra_attn_profile_enable(supra_attn_ctx* ctx, int32_t on);
typedef struct supra_attn_profile_entry {
  char name[48];
  int64_t launches;
  double ms;    /* summed device time */
  double flops; /* summed algorithmic FLOPs */
  double bytes; /* summed algorithmic bytes */
} supra_attn_profile_entry;
/* Synchronises, then copies up to cap entries (sorted by time) and sets *n. */
SUPRA_ATTN_API int supra_attn_profile_report(supra_attn_ctx* ctx, supra_attn_profile_entry* entries,
                              int32_t cap, int32_t* n);
SUPRA_ATTN_API int supra_attn_profile_reset(supra_attn_ctx* ctx);
/* Total kernels this context has launched since creation, all kinds: every flushed group is one
 * descriptor-staging kernel plus its attention kernel(s). */
SUPRA_ATTN_API int supra_attn_launch_count(const supra_attn_ctx* ctx, int64_t* n);

/* ---- attention without allocation ---------------------------------------------------------- */
/* No counterpart in the reference: this entry point exists for callers that cannot allocate
 * device memory when they need attention, such as a host whose allocator reserves the GPU's
 * memory up front and sub-allocates from it, or code on a latency-critical path that must not
 * call cudaMalloc/cudaFree (those can synchronise the device).
 *
 * Runs ONE problem (validated exactly as supra_attn_enqueue validates it, any head dim) on
 * `cuda_stream` through the score-materialising kernels (QK^T GEMM, row softmax, PV GEMM),
 * without a context and without any allocation: the score scratch is a 16 MiB array of static
 * device memory inside the library, used chunk by chunk, and the chunk's unit table sits in a
 * second static array of about 62 KB, written on the device by a small kernel from values passed
 * as kernel arguments (no host buffer is read after the call returns). Every GPU on which the
 * library's kernels are loaded holds both until the process exits. Limit: one row of scores
 * must fit the scratch, i.e. Lk <= 4,194,304; larger Lk is rejected with SUPRA_ATTN_EINVAL and a
 * message. The arithmetic is always FP32 FFMA, whatever desc->variant asks for: a TF32 or
 * TF32X3 request gets the FP32 result, which lies inside their tolerances.
 *
 * The caller passes inputs and outputs as for supra_attn_enqueue. The work is enqueued on
 * cuda_stream and the call returns without waiting for it. The first call on each device looks
 * up the arrays' device addresses (cudaGetSymbolAddress) with that device current; make that
 * first call before any stream capture. All calls share the two arrays, which keep the last
 * call's contents: every call writes each score and unit entry it reads before reading it, so
 * nothing needs to start at zero. Calls that overlap on the GPU (different streams, or different
 * host threads on one device) race on the arrays; serialise them, e.g. on one stream.
 * msg (cap bytes, may be NULL) receives the message of a failure. */
SUPRA_ATTN_API int supra_attn_attention_noalloc(const supra_attn_desc* desc, void* cuda_stream, char* msg,
                                                int32_t cap);

#ifdef __cplusplus
}
#endif

#endif /* SUPRA_ATTN_H */
