/*
 * libcqhip: go-whistle's CQ quantized-matrix path and int8 KV numerics on
 * AMD Instinct MI355X (gfx950), behind a plain C ABI.
 *
 * Each entry point replaces one method of the reference's Go API (cited as
 * file:line in the go-whistle repository); a Go caller binds them through
 * cgo (the stub a maintainer would add is in INTEGRATION.md). Host-slice
 * entry points copy their operands to and from the device within the call,
 * as cgo requires of Go memory; the _dev entry points take device pointers
 * and a HIP stream for device-resident pipelines.
 *
 * Errors: every call returns CQ_OK or a status; cq_last_error() returns the
 * failing call's message on the calling thread. Construction errors carry
 * the reference's "cq: ..." text (the Go API returns them as error values);
 * misuse that the Go API answers with a panic (lengths that do not match
 * the shape, rows out of range) returns CQ_ERR_MISUSE.
 *
 * Threads: matrices are immutable after construction and safe for
 * concurrent use from any thread (internal/cq/matrix.go:22-24). Host-slice
 * calls run on a per-thread stream with per-thread staging buffers.
 *
 * Workspaces: the table and split forms of a batched product keep tables
 * or float terms in device memory between their two launches. They lease
 * it from one pool per process for the length of the call and return it
 * with an event behind their launches; a workspace is reused at once on the
 * stream that last used it, on another stream only once that work has
 * completed. Products queued at the same time on several streams, from one
 * thread or many, therefore never share one. A product queued while its
 * stream is captured into a graph gets a workspace that only its capture
 * sequence uses and that is held until the process ends (the graph replays
 * it at that address); such a first product of a shape may itself be
 * captured. cq_workspace_held and cq_workspace_trim report and release the
 * pool's memory.
 */
#ifndef CQHIP_H
#define CQHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    CQ_OK = 0,
    CQ_ERR_ARG = 1,         /* construction rejected: the Go API's error result */
    CQ_ERR_MISUSE = 2,      /* shape misuse: the Go API panics */
    CQ_ERR_DEVICE = 3,      /* HIP runtime failure or no device */
    CQ_ERR_UNSUPPORTED = 4, /* a geometry this library does not run */
};

/* Message of the last failing call on this thread ("" if none). */
const char *cq_last_error(void);

/* Library version string and the device it runs on (cf. `whistle doctor`,
 * cmd/whistle/doctor.go:349-370, which names the active kernels). */
const char *cq_version(void);
int cq_device_info(char *buf, size_t len);

typedef struct cq_matrix cq_matrix;

/* cq.New (internal/cq/matrix.go:46-55) when gather == 0, cq.NewGather
 * (matrix.go:60-96) when gather != 0: validates the packed form of
 * cact.Packed (internal/cact/packed.go:18-29) with the reference's checks and
 * messages, widens nothing on the host, and uploads the index and FP16 norms
 * to the device in the product layout. No host pointer is kept. */
int cq_new(int out, int in, int group, int bits, int width, const float *codebook, size_t codebook_len,
           const uint8_t *index, size_t index_len, const uint8_t *norms_fp16, size_t norms_len, int gather,
           cq_matrix **m);

/* Releases a matrix or a view; the storage goes with the last of them (the
 * Go shim calls it from a runtime.AddCleanup, as *cq.Matrix has no Close). */
void cq_free(cq_matrix *m);

int cq_out(const cq_matrix *m);  /* Matrix.Out  (matrix.go:99) */
int cq_in(const cq_matrix *m);   /* Matrix.In   (matrix.go:102) */
int cq_bits(const cq_matrix *m); /* Matrix.Bits (matrix.go:105) */
/* Matrix.Prepare (matrix.go:111-115). */
int cq_prepare(cq_matrix *m);
/* Matrix.Bytes (matrix.go:121-129): the reference's accounting. */
long long cq_bytes(const cq_matrix *m);
/* Device memory the matrix's storage holds (no reference counterpart). */
long long cq_device_bytes(const cq_matrix *m);
/* Matrix.Rows (matrix.go:133-145): a view of rows [lo, hi) sharing storage. */
int cq_rows(const cq_matrix *m, int lo, int hi, cq_matrix **view);
/* Matrix.Exact (matrix.go:152-157): a view whose products use the float
 * nibble tables (kernel.go:239-374) instead of the lut kernel. */
int cq_exact(const cq_matrix *m, cq_matrix **view);
/* A view sharing m's storage whose products of 16 or more activations run
 * Exact's semantics as a dense fp32 MFMA contraction: the activations
 * rotated as Exact rotates them (kernel.go:203-217), times W[r][k] =
 * norm[r][k/G] * codebook[index(r, k)] dequantized tile by tile into LDS, on
 * v_mfma_f32_32x32x2_f32. The sums run in the MFMA's order, so results are
 * within float32 rounding of Exact's (tests hold them within 1e-5 of the
 * largest |y| of each activation), not bit for bit; fewer activations,
 * and groups outside 32..1024, run Exact's nibble kernels. No counterpart in the
 * reference: for batched encoder-frame products that take Exact's
 * arithmetic at matrix-core rates. Rows views keep the setting; cq_exact
 * of it is a plain Exact view. */
int cq_dense(const cq_matrix *m, cq_matrix **view);
/* Name of the kernel the matrix's products run: "lut", "nibble4" or, for a
 * Dense view, "dense-f32" (kernel.go:30-43, 92-98). */
const char *cq_kernel_name(const cq_matrix *m);

/* Matrix.Row (matrix.go:161-181): row r dequantised as cact.CQ does, bit
 * for bit; dst holds In floats (host). */
int cq_row(const cq_matrix *m, float *dst, size_t dst_len, int r);
/* Matrix.GEMM (kernel.go:85-87); GEMV (kernel.go:78-80) is rows = 1.
 * x is [rows][In], dst [rows][Out], host row-major. */
int cq_gemm(const cq_matrix *m, float *dst, size_t dst_len, const float *x, size_t x_len, int rows);
/* cq.GEMMs (kernel.go:134-158): dsts[k] = ms[k].GEMM of the same x. */
int cq_gemms(int n, cq_matrix *const *ms, float *const *dsts, const size_t *dst_lens, const float *x, size_t x_len,
             int rows);

/* Device-pointer forms of GEMM, GEMMs and Row: every pointer is device
 * memory, work is queued on `stream` (a hipStream_t; NULL = the null
 * stream) and the call returns without waiting. */
int cq_gemm_dev(const cq_matrix *m, float *dst, const float *x, int rows, void *stream);
/* The same product, always in the MFMA form of the lut kernel (one-hot
 * indices times int8 table planes on v_mfma_i32_32x32x32_i8, exact int32
 * sums, the lut fold), bit for bit cq_gemm_dev's result. No counterpart in
 * the reference: the encoder's batched products (many frames at once) call
 * it; cq_gemm_dev picks it by itself when its grid is large enough. Group
 * 128, 2 or 4 bits, not an Exact view; else CQ_ERR_UNSUPPORTED. */
int cq_gemm_mfma_dev(const cq_matrix *m, float *dst, const float *x, int rows, void *stream);
/* The kernel cq_gemm_dev runs for `rows` activations: "lut", "lut-mfma",
 * "lut-mfma-tab" (the table pre-pass and its MFMA product), "lut-mfma-split",
 * "dense-f32" (a Dense view's fp32 MFMA form) or "nibble4". */
const char *cq_gemm_path(const cq_matrix *m, int rows);
int cq_gemms_dev(int n, cq_matrix *const *ms, float *const *dsts, const float *x, int rows, void *stream);
/* Bytes of device memory the workspace pool holds on every device (leased,
 * idle and held for graphs). No reference counterpart (the Go code's
 * scratch comes from a sync.Pool, internal/cq/kernel.go:59-74). */
long long cq_workspace_held(void);
/* Frees the idle workspaces whose work has completed, on every device;
 * returns the bytes still held. No reference counterpart. */
long long cq_workspace_trim(void);
/* cq_gemms_dev with the decode step's neighbours fused into the product
 * (no reference counterpart: one launch instead of three, results bit for
 * bit those of the separate steps). norm_gain non-null: every input row is
 * first ZCRMSNorm.Apply'd with that gain (internal/needle/norm.go:53-109).
 * resid non-null (n = 1): dst = resid + product, the residual add of the
 * decoder's layer body (resid may be dst). act 1 (no resid): dst =
 * silu(product), the synthetic decoder's FFN activation (as nd_silu_dev).
 * lut matrices only. */
int cq_gemms_fused_dev(int n, cq_matrix *const *ms, float *const *dsts, const float *x, int rows,
                       const float *norm_gain, const float *resid, int act, void *stream);
/* The gated attention's output projection: dst = product of (x * gate')
 * with gate' = sigmoid(gate) elementwise, sigmoid float32(1 / (1 +
 * exp(-float64(g)))) -- Attention.output (internal/needle/attention.go:
 * 242-260) and the cross-attention's gate (internal/decoder/cross.go:
 * 231-252) followed by outProj.Apply, one launch instead of two, bit for bit
 * nd_sigmoid_gate_dev then cq_gemms_dev. gate has x's layout (rows of the
 * matrices' input width) and is only read. resid non-null (n = 1): dst =
 * resid + product (resid may be dst). lut matrices only. */
int cq_gemms_gated_dev(int n, cq_matrix *const *ms, float *const *dsts, const float *x, const float *gate, int rows,
                       const float *resid, void *stream);
/* cq_gemms_fused_dev (norm_gain only) whose outputs are also appended to
 * int8 row caches: the decoder's K and V projections followed by
 * Int8Rows.Append (internal/needle/int8.go:36-55; Attention.Extend's
 * projections, RoPE and append, internal/needle/cache.go:90-125), one launch instead of
 * three, results bit for bit kv_append_rope_dev's. No reference
 * counterpart. For k with kv_q[k] non-null, activation b's product row is
 * quantized per 64-wide head into row pos[b] of stream b's cache (codes
 * kv_q[k] + b*q_stride + pos[b]*out, scales kv_s[k] + b*s_stride +
 * pos[b]*out/64; no append where pos[b] is outside [0, cap)), after RoPE
 * at pos[b] with the half-width tables cos_t[k], sin_t[k] when cos_t and
 * cos_t[k] are non-null (internal/needle/rope.go:69-81). dsts[k] still
 * receives the product. Matrix k's view must cover whole 64-row blocks;
 * at most 8 lut matrices of one group size and index width (else
 * CQ_ERR_MISUSE / CQ_ERR_UNSUPPORTED). */
int cq_gemms_append_dev(int n, cq_matrix *const *ms, float *const *dsts, const float *x, int rows,
                        const float *norm_gain, int8_t *const *kv_q, float *const *kv_s, long long q_stride,
                        long long s_stride, const int32_t *pos, int cap, const float *const *cos_t,
                        const float *const *sin_t, void *stream);
/* A product chained to the next one through its tables (no reference
 * counterpart: the decoder's layer body, internal/decoder/decoder.go:
 * 446-505, runs each projection on the previous one's output; here the
 * previous product's launch also builds the next product's lookup tables,
 * lut.go:158-282, which that product would otherwise build in a launch of
 * its own). Results bit for bit those of the unchained calls.
 *
 * cq_tables_bytes: bytes of the tables of the product over next[0..n) at
 * `rows` activations, or 0 when that product takes no tables from a buffer
 * (it then runs as cq_gemms_fused_dev / cq_gemms_append_dev would). */
size_t cq_tables_bytes(int n, cq_matrix *const *next, int rows);
/* dst = [resid +] product of m and (x [* sigmoid(gate)]), as
 * cq_gemms_gated_dev (gate may be null: no gate); and, where the product
 * runs one workgroup per activation over all of m's rows, the tables of
 * the next product over next[0..n_next) of ZCRMSNorm(dst; next_gain)
 * (next_gain null: dst itself) into `tables`, tables_bytes =
 * cq_tables_bytes(n_next, next, rows) (0: none asked). *built = 1 when the
 * tables were built, else 0: then the next product runs unchained. The
 * next matrices take m's outputs as inputs. Calls that overlap on one
 * table buffer race. */
int cq_gemm_tables_dev(const cq_matrix *m, float *dst, const float *x, const float *gate, int rows, const float *resid,
                       int n_next, cq_matrix *const *next, const float *next_gain, void *tables, size_t tables_bytes,
                       int *built, void *stream);
/* The product over ms[0..n) of the activations whose tables
 * cq_gemm_tables_dev built (with `next` ms, or matrices of the same
 * codebook and geometry, and the same rows), with the epilogues of
 * cq_gemms_fused_dev (resid, act) and cq_gemms_append_dev (kv_q null: no
 * appends). The norm and the input are those the tables were built from.
 * CQ_ERR_MISUSE where cq_tables_bytes(n, ms, rows) is 0 or differs from
 * tables_bytes (tables of the other index width always differ). */
int cq_gemms_tables_dev(int n, cq_matrix *const *ms, float *const *dsts, int rows, const float *resid, int act,
                        int8_t *const *kv_q, float *const *kv_s, long long q_stride, long long s_stride,
                        const int32_t *pos, int cap, const float *const *cos_t, const float *const *sin_t,
                        const void *tables, size_t tables_bytes, void *stream);
int cq_row_dev(const cq_matrix *m, float *dst, int r, void *stream);
/* Rows gathered by index: dst[i] = scale * Row(rows[i]) for i < n, rows a
 * device int32 array: the decoder's scaled token-embedding lookup for
 * several streams (internal/decoder/decoder.go:269-275) in one launch. A
 * listed row outside the matrix gives zeros. */
int cq_row_gather_dev(const cq_matrix *m, float *dst, const int32_t *rows, int n, float scale, void *stream);

/* Batch plans (no reference counterpart; the device-resident form of many
 * independent Matrix.GEMM calls): job k multiplies ms[k] by rows[k]
 * activations at device xs[k] into device ys[k], as cq_gemm_dev would, bit
 * for bit. cq_batch_new validates the jobs and uploads a device job table
 * once; cq_batch_run queues one lut-kernel launch per kernel geometry (index
 * width and group size) on `stream`, and can be captured in a HIP graph. The
 * matrices and buffers must outlive the plan's runs. Jobs on Exact views or
 * on groups the lut kernel does not hold in LDS return CQ_ERR_UNSUPPORTED. */
typedef struct cq_batch cq_batch;
int cq_batch_new(int n, cq_matrix *const *ms, float *const *ys, const float *const *xs, const int *rows,
                 cq_batch **plan);
int cq_batch_run(const cq_batch *plan, void *stream);
int cq_batch_launches(const cq_batch *plan);
void cq_batch_free(cq_batch *plan);

/* ---- int8 KV numerics (internal/needle/int8.go) ------------------------- */

/* QuantizeRows (int8.go:116-121, Append :125-141): x is rows of cols
 * floats; each chunk of width values gets its codes and one scale as
 * QuantizeRow (int8.go:36-55) gives them, bit for bit. Host and device
 * forms. */
int kv_quantize_rows(int8_t *q, float *s, const float *x, int rows, int cols, int width);
int kv_quantize_rows_dev(int8_t *q, float *s, const float *x, int rows, int cols, int width, void *stream);
/* KVCache.Fork for many streams at once (internal/needle/cache.go:62-67,
 * Int8Rows.Clip int8.go:155-161; the beams of internal/search/beam.go):
 * stream b of the int8 cache (codes q, scales s; streams of cap rows of
 * cols codes, width codes per scale) becomes the first len[b] rows of
 * stream parent[b], after which every stream extends on its own. parent
 * and len are device int32 arrays of `streams`; rows past len[b] are left
 * as they were. The reference shares the rows until one side appends
 * (copy on write); here they are copied, through the caller's temporaries
 * tmp_q, tmp_s of the cache's size. No reference counterpart as one call. */
int kv_reorder_dev(int8_t *q, float *s, int8_t *tmp_q, float *tmp_s, const int32_t *parent, const int32_t *len,
                   int streams, int cap, int cols, int width, void *stream);
/* kv_reorder_dev without the temporaries and without any allocation: the
 * temporaries live in a device array of 16 MiB that the library holds on
 * each GPU it runs on until the process ends. No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under HIP graph capture, a serving loop's beam reorder, harnesses that
 * forbid hipMalloc). A reorder whose temporaries (streams * cap * cols
 * codes, 256-byte aligned, plus streams * cap * cols/width float scales)
 * exceed 16 MiB returns CQ_ERR_MISUSE. Every call on one GPU uses that
 * GPU's one array: calls that overlap on one GPU race. */
int kv_reorder_noalloc_dev(int8_t *q, float *s, const int32_t *parent, const int32_t *len, int streams, int cap,
                           int cols, int width, void *stream);

/* AttendInt8Spans (int8.go:208-272) on device memory for `batch`
 * independent streams (beam hypotheses, internal/search/beam.go:508-521).
 * Stream b reads q + b*q_stride (t rows of heads*qk floats), its keys and
 * values at kq + b*kv_stride codes (nk rows of k_cols / v_cols) with scales
 * at ks/vs + b*s_stride, its spans at spans + b*t*4 (per query row the
 * two ascending disjoint key spans {lo0, hi0, lo1, hi1}), and writes t rows
 * of heads*vd floats at out + b*out_stride (out_stride and q_stride 0 mean
 * dense streams; kv_stride and s_stride 0 share one cache). nk_max is the
 * number of key rows each stream's arrays hold: spans outside [0, nk_max),
 * or of more than nk_max keys together, leave that output untouched. quant_q chooses the int8 query
 * (int8Logits, int8.go:278-285) or the float32 query (dotsF32I8,
 * int8.go:289-300). The softmax is softmaxInPlace (load.go:128-138) with
 * the amd64 kernel's exponent (exp_amd64.s:68-124). */
int kv_attend_int8_dev(float *out, long long out_stride, const float *q, long long q_stride, int t, int heads,
                       const int8_t *kq, const float *ks, int k_cols, int qk, const int8_t *vq, const float *vs,
                       int v_cols, int vd, long long kv_stride, long long s_stride, const int32_t *spans, int nk_max,
                       float scale, int quant_q, int batch, void *stream);
/* The same with the query heads first rotated by RoPE (Rope.apply,
 * internal/needle/rope.go:69-81) at row qpos[b*t + i] of the (positions x
 * qk/2) cos/sin tables: Attention.Extend's rotated query
 * (internal/needle/attention.go:345-415) without a separate pass. */
int kv_attend_int8_rope_dev(float *out, long long out_stride, const float *q, long long q_stride, int t, int heads,
                            const int8_t *kq, const float *ks, int k_cols, int qk, const int8_t *vq, const float *vs,
                            int v_cols, int vd, long long kv_stride, long long s_stride, const int32_t *spans,
                            int nk_max, float scale, int quant_q, int batch, const float *cos_t, const float *sin_t,
                            const int32_t *qpos, void *stream);
/* kv_attend_int8_dev over caches that streams share: stream b reads the
 * keys and values of cache kv_index[b] (a device int32 array of `batch`),
 * one of kv_streams caches kv_stride codes / s_stride scales apart; an
 * index outside [0, kv_streams) leaves stream b's output untouched. The
 * beams of one utterance after State.Fork (internal/decoder/decoder.go:
 * 223-240) share its cross-attention memory, which is never copied. */
int kv_attend_int8_shared_dev(float *out, long long out_stride, const float *q, long long q_stride, int t, int heads,
                              const int8_t *kq, const float *ks, int k_cols, int qk, const int8_t *vq, const float *vs,
                              int v_cols, int vd, long long kv_stride, long long s_stride, const int32_t *spans,
                              int nk_max, float scale, int quant_q, int batch, const int32_t *kv_index, int kv_streams,
                              void *stream);

/* Int8Rows.Append (int8.go:125-141) on a device KV cache for `batch`
 * streams: stream b's row x + b*cols is quantised per chunk of width
 * (QuantizeRow, bit for bit) into codes q + b*q_stride + pos[b]*cols and
 * scales s + b*s_stride + pos[b]*(cols/width); pos is a device array, and a
 * position outside [0, cap) is skipped. */
int kv_append_dev(int8_t *q, float *s, const float *x, int batch, int cols, int width, long long q_stride,
                  long long s_stride, const int32_t *pos, int cap, void *stream);
/* The same with each chunk (a key head) first rotated by RoPE (rope.go:
 * 69-81) at row pos[b] of the (positions x width/2) cos/sin tables: the
 * rotated key appended (attention.go:345-415). width <= 256, even. */
int kv_append_rope_dev(int8_t *q, float *s, const float *x, int batch, int cols, int width, long long q_stride,
                       long long s_stride, const int32_t *pos, int cap, const float *cos_t, const float *sin_t,
                       void *stream);

/* ---- float blocks of a decode step, on device memory -------------------- */

/* ZCRMSNorm.Apply (internal/needle/norm.go:53-66, meanSquare :91-109):
 * dst = gain * x / sqrt(mean(x^2) + 1e-6) per row of dim, mean in float64
 * as the reference sums it; gain = 1 + scale (NewZCRMSNorm, norm.go:22-30).
 * dst may be x. */
int nd_zcrmsnorm_dev(float *dst, const float *x, const float *gain, int rows, int dim, void *stream);
/* Rope.apply (internal/needle/rope.go:69-81) in place on rows of heads
 * vectors of head_dim: row r uses position pos[r / rows_per_pos] of the
 * (positions x head_dim/2) cos/sin tables (NewRope, rope.go:17-44). A row
 * whose position is outside [0, positions) is left unchanged (the
 * reference's table slice would panic there). */
int nd_rope_dev(float *x, int rows, int heads, int head_dim, const float *cos_t, const float *sin_t, int positions,
                const int32_t *pos, int rows_per_pos, void *stream);
/* argmax (internal/decoder/greedy.go:181-191) of each row of n: the first
 * index of the largest value. */
int nd_argmax_dev(int32_t *out, const float *v, int rows, int n, void *stream);
/* nd_argmax_dev that also advances each stream's decode position, the end
 * of Decoder.Extend's step (internal/decoder/decoder.go:252-302, greedy.go:
 * 31-69): pos[r] += 1, and span_hi[r * span_stride] = pos[r] + 1, the key
 * bound of the next step's self-attention after its append. No reference
 * counterpart as one call: the device decode step's bookkeeping without
 * launches of its own. */
int nd_argmax_advance_dev(int32_t *out, const float *v, int rows, int n, int32_t *pos, int32_t *span_hi,
                          int span_stride, void *stream);
/* nd_argmax_advance_dev with greedy decoding's stop (internal/decoder/
 * greedy.go:50-66): a stream whose done[r] is nonzero is left as it is (its
 * token, position and key bound); otherwise, after the argmax and the
 * advance, done[r] = 1 when the token is eos. Streams of one batch stop one
 * by one, each after its own EOS, as GreedyMemory stops each hypothesis. */
int nd_argmax_advance_eos_dev(int32_t *out, const float *v, int rows, int n, int32_t *pos, int32_t *span_hi,
                              int span_stride, int32_t *done, int eos, void *stream);
/* x = x * sigmoid(x), sigmoid from the amd64 exponent kernel's arithmetic
 * (exp_amd64.s:84-112) on non-positive arguments. No reference
 * counterpart: the synthetic decoder's FFN activation. */
int nd_silu_dev(float *x, long long n, void *stream);
/* fakeQuant (internal/needle/int8.go:57-75): rows of cols values, each
 * chunk of width through QuantizeRow and back, dst = float32(q) * s; the
 * input of a Linear WithInt8Input (quantInput, int8.go:81-88;
 * internal/needle/linear.go:82-86). dst may be x. */
int nd_fake_quant_dev(float *dst, const float *x, long long rows, int cols, int width, void *stream);
/* x += y elementwise (the residual adds). */
int nd_add_dev(float *x, const float *y, long long n, void *stream);
/* HadamardMLP.Forward (internal/needle/hadamard.go:172-294), Whistle's
 * Monarch FFN, on rows of dim values: cond = 1 + softmax(x cond_v) cond_u;
 * z1 = kron(d1 x; w1a, w1b)[p1]; z2 = kron(silu(d2 cond z1 + b2); w2a,
 * w2b)[p2]; out = d4 kron(d3 z2; w3a, w3b), kron(z; a, b) = a^T Z b with Z
 * the na x nb matrix of z (kronApply, hadamard.go:296-310); x zero-padded
 * to n = na * nb >= dim, out cut back to dim (LoadHadamardMLP's padding,
 * hadamard.go:19-24). vecs = {d1, d2, b2, d3, d4} (n each), factors =
 * {w1a, w1b, w2a, w2b, w3a, w3b} row-major, cond_v dim x rank, cond_u
 * rank x n, p1 and p2 permutations of n (hada_p1/p2). n <= 1024, rank <= 32.
 * Float32, within 1e-5 of the float64 form (hadamard_test.go:152-191); the
 * reference's GEMMs sum in their library's own order. The order here follows
 * na and nb alone: a row's result is the same in every call. */
int nd_hadamard_mlp_dev(float *out, const float *x, int rows, int dim, int na, int nb, int rank,
                        const float *const *vecs, const float *const *factors, const float *cond_v,
                        const float *cond_u, const int32_t *p1, const int32_t *p2, void *stream);
/* RMSUnit (internal/needle/norm.go:68-81): each row of dim times
 * float32(1 / sqrt(float64(meanSquare + 1e-6))), meanSquare in float64 as
 * ZCRMSNorm's; mHC's nx of the lane stream (rows of lanes * dim). */
int nd_rms_unit_dev(float *dst, const float *x, int rows, int dim, void *stream);
/* MHC.forward's heads and block input (internal/needle/mhc.go:204-219,
 * 246-263) from the φ products' logits (rows x lanes, rows x lanes x
 * lanes): with affine non-null (device floats {a_pre, a_post, a_res,
 * b_pre[lanes], pre_off[lanes], b_post[lanes], post_off[lanes],
 * b_res[lanes^2]}) the logits are first a * logit + b (+ off) as MHC.logits
 * rounds them; h_pre = sigmoid, h_post = 2 sigmoid, h_res = sinkhorn of 20
 * iterations (mhc.go:301-417), u[i] = sum_k h_pre[k] stream[i, k] in k
 * order (stream rows x lanes x dim, u rows x dim). lanes <= 8. */
int nd_mhc_heads_dev(float *h_pre, float *h_post, float *h_res, float *u, const float *pre_logits,
                     const float *post_logits, const float *res_logits, const float *stream_rows, int rows, int lanes,
                     int dim, const float *affine, void *stream);
/* nd_mhc_heads_dev with the three φ products' logits in one array, rows x
 * (2 lanes + lanes^2): pre, post, then res of each row, as one product of
 * the three φ matrices stacked row-wise gives them (the same outputs bit
 * for bit; one table build per activation instead of three). */
int nd_mhc_heads_stacked_dev(float *h_pre, float *h_post, float *h_res, float *u, const float *logits,
                             const float *stream_rows, int rows, int lanes, int dim, const float *affine,
                             void *stream);
/* MHC.forward's output (internal/needle/mhc.go:229-234, 266-299): y =
 * block_out - u, out[i, a] = sum_b h_res[i, a, b] stream[i, b] (b in order)
 * + h_post[i, a] y. out must not be the stream. */
int nd_mhc_mix_dev(float *out, const float *stream_rows, const float *h_res, const float *h_post,
                   const float *block_out, const float *u, int rows, int lanes, int dim, void *stream);
/* AttendInt8Spans over paged int8 caches: the arrays kq/ks/vq/vs are one
 * pool of pool_pages pages of page_rows rows (a power of two; codes k_cols /
 * v_cols per row, scales per head), and key j of stream b is row
 * pages[b*page_stride + j/page_rows]*page_rows + j%page_rows. Otherwise
 * kv_attend_int8_rope_dev (cos_t null: no RoPE of the query). Forked
 * streams share their full pages without a copy, as KVCache.Fork shares the
 * rows so far until one side appends (internal/needle/cache.go:62-67). An
 * entry outside [0, pool_pages) reads page 0. */
int kv_attend_int8_paged_dev(float *out, long long out_stride, const float *q, long long q_stride, int t, int heads,
                             const int8_t *kq, const float *ks, int k_cols, int qk, const int8_t *vq, const float *vs,
                             int v_cols, int vd, const int32_t *spans, int nk_max, float scale, int quant_q, int batch,
                             const float *cos_t, const float *sin_t, const int32_t *qpos, const int32_t *pages,
                             int page_stride, int page_rows, int pool_pages, void *stream);
/* Attention.Extend's steps between the projections and the attention for
 * one token per stream (internal/needle/cache.go:88-125): q, k, v are batch
 * rows of dim (heads of 64) at positions pos[b]. In order: the causal taps
 * (taps > 0; applyTaps on extendTaps' rows, attention.go:597-613,
 * cache.go:143-154): out = sum_j taps_w[z][j] * row(pos - j) over j <= pos,
 * from 0 in j order, products rounded; hist [batch][taps][3][dim] holds the
 * raw rows of the last positions at slot position mod taps and is updated
 * (slot pos[b] mod taps, which the step does not read: running a position
 * again gives the same result); the per-head ZCRMSNorm of q and k (q_gain / k_gain of 64; null:
 * none; normRotate, attention.go:298-330); RoPE of k at pos[b] (cos_t null:
 * none; tables of 32 per row, `positions` rows); then k and v quantized per
 * head and appended at row pos[b] (< cap) through the page table (as
 * kv_attend_int8_paged_dev reads them; an entry outside the pool skips the
 * append). q is written back, normed and not rotated (the attention rotates
 * it). dim a multiple of 64 up to 1024. No reference counterpart as one call. */
int nd_qkv_prep_dev(float *q, const float *k, const float *v, int batch, int dim, float *hist, const float *taps_w,
                    int taps, const float *q_gain, const float *k_gain, const float *cos_t, const float *sin_t,
                    int positions, const int32_t *pos, int cap, int8_t *kq, float *ks, int8_t *vq, float *vs,
                    const int32_t *pages, int page_stride, int page_rows, int pool_pages, void *stream);
/* h = resid + float32(scale * ZCRMSNorm(y)) per row of dim (resid null or
 * h: h += ...): the attention's post norm and residual factor, h +=
 * float32(gate * postNorm(a)) (internal/needle/block.go:183-188), and the
 * cross branch's (internal/decoder/cross.go:255-263 with the hook's add,
 * decoder.go:461-465). y is only read. dim a multiple of 256 up to 4096. */
int nd_norm_scaled_add_dev(float *h, const float *resid, const float *y, const float *gain, float scale, int rows,
                           int dim, void *stream);
/* RMSUnit (internal/needle/norm.go:68-81) of each row of dim, then its
 * fakeQuant as one chunk (int8.go:57-75): the mHC phi products' int8 input
 * (mhc.go:99-106 with Linear.WithInt8Input, linear.go:80-87), one launch,
 * bit for bit nd_rms_unit_dev then nd_fake_quant_dev. dim a multiple of 256
 * up to 4096; dst may be x. */
int nd_rms_unit_quant_dev(float *dst, const float *x, int rows, int dim, void *stream);
/* ExpandLanes / CollapseLanes (internal/needle/mhc.go:137-170): each row of
 * x to `lanes` equal lanes of the stream (rows x lanes x dim), and back as
 * the lane mean (lanes summed in order from 0, then divided by lanes). */
int nd_expand_lanes_dev(float *stream_rows, const float *x, int rows, int lanes, int dim, void *stream);
int nd_collapse_lanes_dev(float *x, const float *stream_rows, int rows, int lanes, int dim, void *stream);
/* Page dst[j] of a paged int8 cache (page_rows rows of cols codes, cols/width
 * scales) becomes a copy of page src[j], j < n: the copy-on-write of a
 * forked stream's partly filled page. Pairs outside [0, pool_pages) are
 * skipped. No reference counterpart (its Fork copies on the next append). */
int kv_page_copy_dev(int8_t *q, float *s, const int32_t *src, const int32_t *dst, int n, int page_rows, int cols,
                     int width, int pool_pages, void *stream);
/* dst row r = src row idx[r] (idx null: r), rows of width floats: a fork's
 * tap history (State.Fork shares it, decoder.go:218-240). dst must not
 * overlap src. */
int nd_gather_rows_dev(float *dst, const float *src, const int32_t *idx, int rows, long long width, void *stream);
/* The attention's output gate (internal/needle/attention.go:245-249):
 * gate[i] = sigmoid(gate[i]), out[i] *= gate[i], sigmoid being jax.nn.sigmoid
 * in float32 as the reference writes it, float32(1 / (1 + exp(-float64(x))))
 * (internal/needle/load.go:120-123; internal/decoder/cross.go:240-248). */
int nd_sigmoid_gate_dev(float *out, float *gate, long long n, void *stream);

/* ---- float and int8 caches of any length, and what a step answers with ---- */

/* Types of the values the calls below read and write. */
enum {
    ND_F32 = 0,
    ND_F16 = 1,
    ND_BF16 = 2,
    ND_I8 = 3, /* caches only: codes with one float32 scale a row and head, as QuantizeRow gives them (int8.go:36-55) */
    /* caches only: codes with one float32 scale a page and head, the largest
     * |x| that the page has held over 127 (int8) or 448 (e4m3, the OCP 8-bit
     * float without infinities) */
    ND_I8_PAGES = 5,
    ND_E4M3_PAGES = 6,
};

/* Paged key and value caches: pools of pool_pages pages of page_rows rows (a
 * power of two) of kv_heads keys of qk and values of vd of one type, scales
 * [row][kv_heads] beside ND_I8 ones, [page][kv_heads] beside ND_I8_PAGES and
 * ND_E4M3_PAGES (else null). Row j of stream b is row
 * pages[b*page_stride + j/page_rows]*page_rows + j%page_rows of the pools, as
 * kv_attend_int8_paged_dev reads them. Device pointers; the pools 16-byte
 * aligned. qk and vd are multiples of 16 up to 256; pool_pages * page_rows
 * is below 2^31. */
typedef struct kv_paged {
    void *k, *v;
    float *ks, *vs;
    const int32_t *pages;
    int type, kv_heads, qk, vd;
    int page_stride, page_rows, pool_pages;
} kv_paged;

/* Rows of keys and values appended to paged caches of any type: Int8Rows.
 * Append and its float counterpart (internal/needle/int8.go:125-141,
 * cache.go:88-125) for t rows of each of `batch` streams. Row i < rows[b]
 * (null: t; counts outside [0, t] append nothing) of stream b goes to row
 * pos[b] + i of its cache; rows outside [0, cap), and rows in pages outside
 * the pool, are skipped. k and v hold values of `type` (ND_F32, ND_F16 or
 * ND_BF16): row i of stream b is kv_heads*qk (kv_heads*vd) values at element
 * b*k_stream + i*k_row (b*v_stream + i*v_row). Rounded to the cache's type to
 * the nearest even; int8 rows are quantized per head as QuantizeRow does, bit
 * for bit. acc non-null ([batch][kv_heads][acc_cap], acc_cap >= cap): the
 * appended rows' accumulated weights become 0. Rows of one call that land in
 * the same place race.
 * Caches with a scale a page: the page of the first appended row keeps its
 * rows before it and, for them, a scale that does not fall; rows that raise it
 * have those rows' codes rounded anew, from their float32 values, under the new
 * one. A page that the appended rows begin, and every page behind, takes its
 * scale from them alone; rows behind the last appended one stand for nothing. Codes
 * are the nearest (ties to the even one) to float32(x / scale). So a row is off
 * by up to half a step for each scale that its page has had since (int8: half
 * of each scale; e4m3: 2^-4 of the value, at least 2^-10 of the scale): once for
 * a page appended whole, up to page_rows times for one that grows token by token while
 * its rows do, and the errors may add up. Rows that are appended over (refused
 * drafts) leave the scale of a begun page where they raised it. The scale goes
 * by the finite values: infinities are held as the largest code of their sign,
 * NaN as 0 (int8) or NaN (e4m3); a page of zeros has the scale 0. Streams of one
 * call that append into one page race, also in different rows of it: a shared
 * page is copied first (kv_page_copy_dev with rows of a page's head each:
 * page_rows 1, cols page_rows * kv_heads * width, width page_rows * width). */
int kv_append_paged_dev(const kv_paged *c, const void *k, long long k_stream, long long k_row, const void *v,
                        long long v_stream, long long v_row, int type, int batch, int t, const int32_t *rows,
                        const int32_t *pos, int cap, float *acc, long long acc_cap, void *stream);
/* Attention of one new token a stream over its paged cache, the work split
 * over the cache's length and joined where there are few streams: the float
 * form of kv_attend_int8_paged_dev (AttendInt8Spans with a float query,
 * internal/needle/int8.go:208-300) for caches of any type and length. Logits
 * are q.k / scale (scale > 0); the softmax, its sums and the products' sums
 * are float32: weights of at most 1 times the values, of all keys, whose sum has
 * to be in float32's range (half of it where the work is split).
 * q and out hold values of `type`: batch streams of heads*qk (heads*vd),
 * q_stride (out_stride, at least heads*vd) elements apart (0: dense). Query head h reads key
 * head h / (heads/kv_heads). spans are [batch][4] as kv_attend_int8_dev
 * takes them for t = 1: {lo0, hi0, lo1, hi1}, ascending, disjoint and inside
 * [0, nk_max); others leave the stream's output as it was, and spans with no
 * key give zeros. A page outside the pool reads page 0. Rows outside the spans
 * may hold anything.
 * acc_out non-null ([batch][kv_heads][acc_cap], acc_cap >= nk_max): for
 * each row j of the spans, acc_out[j] = acc[j] (null: 0) + the sum over the
 * key head's query heads of their softmax weights; other entries are left
 * as they were. acc_out may be acc; otherwise the two share no memory, and
 * out and q share none. */
int kv_attend_paged_dev(const kv_paged *c, void *out, long long out_stride, const void *q, long long q_stride,
                        int type, int batch, int heads, const int32_t *spans, int nk_max, float scale,
                        const float *acc, float *acc_out, long long acc_cap, void *stream);
/* Eviction from paged caches by accumulated attention weight (acc of
 * kv_attend_paged_dev): of stream b's len[b] rows every key head keeps the
 * first `sink`, the last `recent`, and of the others those of the largest
 * weights, `keep` in all (every row where len[b] <= keep); among equal
 * weights the lowest row; a NaN weight counts as the least. The kept rows
 * are written in their order to the front of the cache that dst_pages
 * ([batch][dst_stride] of the same pool, dst_stride * page_rows >= keep)
 * names, whose pages are none that any stream's rows are read from (so not
 * c->pages). The source pages are only read, so streams that share them after a
 * fork may be evicted apart. kept ([batch][kv_heads][keep]) gets the kept rows'
 * numbers, -1 past the last; acc_out ([batch][kv_heads][acc_out_cap],
 * acc_out_cap >= keep, apart from acc) their weights; len_out[b] = min(len[b],
 * keep) (len_out may be len, or lies apart from it). A stream whose len is
 * outside [0, nk_max] is left as it was, len_out too. A source page outside the
 * pool reads page 0, and rows of a destination page outside it are not
 * written. sink + recent <= keep. Caches with a scale a page, whose rows cannot
 * move without their page, are not taken (CQ_ERR_UNSUPPORTED). */
int kv_evict_paged_dev(const kv_paged *c, const int32_t *dst_pages, int dst_stride, const float *acc,
                       long long acc_cap, float *acc_out, long long acc_out_cap, const int32_t *len, int32_t *len_out,
                       int32_t *kept, int batch, int nk_max, int keep, int sink, int recent, void *stream);

/* Rows of paged caches of any type read back: row pos[b] + i of stream b's
 * cache, i < rows[b] (null: t; counts outside [0, t] read nothing), as values of
 * `type` (ND_F32, ND_F16 or ND_BF16; codes times their scale in float32, then
 * rounded to the nearest even) to element b*k_stream + i*k_row of k and b*v_stream +
 * i*v_row of v, kv_heads*qk and kv_heads*vd values each. Rows that the table does
 * not hold (below 0, at or past page_stride * page_rows), and rows in pages
 * outside the pool, are left as they were in the outputs. The written rows share
 * no element, keys' with values' either (refused where the host sees it). */
int kv_read_paged_dev(const kv_paged *c, void *k, long long k_stream, long long k_row, void *v, long long v_stream,
                      long long v_row, int type, int batch, int t, const int32_t *rows, const int32_t *pos,
                      void *stream);
/* Causal attention of many rows a stream over its paged cache of any type: the
 * prompt's rows after their append, and drafted tokens'. Row i < rows[b] (null:
 * t) of stream b is at position p = pos[b] + i and attends the cache's rows j
 * <= p, of which with window > 0 only j > p - window and j < sink (the last
 * `window` rows, its own among them, and the first `sink`); logits q.k / scale (>
 * 0). Streams whose count is outside [1, t], or whose rows are not inside [0,
 * nk_max), and rows past the count leave their outputs as they were. q and out
 * hold values of `type` (ND_F32, ND_F16, ND_BF16): row i of stream b is
 * heads*qk values at element b*q_stream + i*q_row (heads*vd at b*out_stream +
 * i*out_row).
 * Query head h reads key head h / (heads/kv_heads). A page outside the pool
 * reads page 0. Cache rows that no row attends may hold anything. The written
 * output rows share no element, and none with q (refused where the host sees it).
 * 16-bit queries over caches of their type, and over codes, take 16-bit
 * products: the operands as they are (codes exactly), the softmax weights in
 * two parts (22 bits with float16 caches, 16 else). Everything else is
 * float32; sums and softmax are float32 throughout, and as
 * kv_attend_paged_dev's past the range of values. */
int kv_attend_rows_paged_dev(const kv_paged *c, void *out, long long out_stream, long long out_row, const void *q,
                             long long q_stream, long long q_row, int type, int batch, int t, int heads,
                             const int32_t *rows, const int32_t *pos, int nk_max, int window, int sink, float scale,
                             void *stream);

/* Where the rows of nd_cross_attend_dev's operands are, in elements: row i
 * of stream b's queries at b*q_stream + i*q_row (heads side by side, qk
 * apart), outputs likewise (vd apart); row j of memory m, key head h at
 * m*k_stream + j*k_row + h*k_head, values likewise. The output rows that are
 * written share no element. */
typedef struct nd_cross_layout {
    long long q_stream, q_row, out_stream, out_row;
    long long k_stream, k_row, k_head, v_stream, v_row, v_head;
} nd_cross_layout;

/* Cross-attention to encoder states of other lengths, in floats: the float
 * form of cross.attend (internal/decoder/cross.go:273-320) for one or many
 * query rows of many streams. q, k, v and out hold values of `type` (ND_F32,
 * ND_F16, ND_BF16). Row i < q_len[b] (null: t; clamped to [0, t]) of stream b
 * attends the first k_len[m] (null: frames; clamped to [0, frames]) of the
 * `frames` rows of memory m = index[b] (null: b), logits q.k / scale (> 0); rows
 * past q_len, and streams whose index is outside [0, memories), leave their
 * outputs as they were; an empty memory gives zeros. Query head h reads key
 * head h / (heads/kv_heads). layout null: dense [batch][t][heads][width] and
 * [memories][frames][kv_heads][width]. qk and vd are multiples of 16 up to
 * 256; k, v and their strides (of dimensions past 1) are multiples of 16 bytes.
 * ND_F32 products are float32; with 16-bit types the products take them as they
 * are, and the softmax weights are float32 or, for many rows, two parts of the
 * type (16 bits in bfloat16, 22 in float16); sums and softmax are float32, and as
 * kv_attend_paged_dev's past the range of values. */
int nd_cross_attend_dev(void *out, const void *q, const void *k, const void *v, int type,
                        const nd_cross_layout *layout, int batch, int t, int heads, int kv_heads, int qk, int vd,
                        int memories, int frames, const int32_t *q_len, const int32_t *k_len, const int32_t *index,
                        float scale, void *stream);
/* What a step or a teacher-forced hypothesis answers with, from rows of n
 * logits of `type`, `stride` elements apart, in one pass: lp[r] the log
 * probability of tokens[r] under the row's softmax (a negative token, a
 * padded row, gives 0; one past n NaN), ent[r] the softmax's entropy in nats,
 * and top_idx / top_lp [rows][top] the `top` likeliest tokens, the lowest
 * index first among equals, with their log probabilities (top <= 64, <= n).
 * lp, ent and the pair of tops may each be null. The log probabilities of
 * internal/search's beams (beam.go:501-540) and the alternatives of
 * greedy's argmax (greedy.go:181-191). Sums are float32. A row of -inf
 * alone has lp -inf and entropy 0; a NaN or +inf makes the row's values
 * NaN, a NaN ranking as -inf. */
int nd_logprobs_dev(float *lp, float *ent, int32_t *top_idx, float *top_lp, const void *logits, long long stride,
                    int type, int rows, int n, const int32_t *tokens, int top, void *stream);
/* Where the rows of nd_qk_norm_rope_dev's operands are, in elements: row i of
 * stream b's queries at b*q_stream + i*q_row (heads side by side, `width`
 * apart), keys, and the outputs of both likewise. */
typedef struct nd_heads_layout {
    long long q_stream, q_row, k_stream, k_row;
    long long q_out_stream, q_out_row, k_out_stream, k_out_row;
} nd_heads_layout;

/* The norms of the query and key heads and their rotation in one pass
 * (normRotate, internal/needle/attention.go:298-330; Rope.apply,
 * rope.go:69-81), for rows of any count: row i < rows[b] (null: t; counts
 * outside [0, t] are none) of stream b has `heads` query and kv_heads key heads
 * of `width` values of `type` (ND_F32, ND_F16, ND_BF16). Each head is
 * ZCRMSNorm'ed (norm.go:53-109) with q_gain or k_gain (float32 [width]; null: no
 * norm of those), then rotated by row pos[b] + i of the (positions x width/2)
 * float32 tables (cos_t null: no rotation, and pos may be null; positions outside the
 * tables: that row is not rotated), and rounded once, to q_out and k_out. Rows past
 * the count are left as they were. ND_F32 arithmetic is ZCRMSNorm's and
 * Rope.apply's but for the order of the float64 squares' sum; 16-bit types
 * compute in float32. The outputs may be the inputs in place (same pointer and
 * strides); else they share no element with an input. Written rows share none.
 * Rows may lie between each other in any order (where q, k and outputs do so at
 * different strides and more than a million steps do not tell their rows
 * apart, the call is refused). heads or kv_heads may be 0. width is a multiple of 16 up to 256. layout null:
 * dense [batch][t][heads][width]. */
int nd_qk_norm_rope_dev(void *q_out, void *k_out, const void *q, const void *k, int type, const nd_heads_layout *layout,
                        int batch, int t, int heads, int kv_heads, int width, const float *q_gain, const float *k_gain,
                        const float *cos_t, const float *sin_t, int positions, const int32_t *pos, const int32_t *rows,
                        void *stream);
/* Drafted tokens verified against the target's probabilities, from given random
 * numbers. target holds t + 1 rows of n logits of `type` (ND_F32, ND_F16,
 * ND_BF16) a stream, row i at element b*target_stream + i*target_row: what the
 * target gives before drafts[b][i] (i < drafted[b]; null: t; clamped to [0, t]), row
 * drafted[b] behind the last. draft: the t rows of logits that the drafts were
 * drawn from (null: each was chosen for sure). With p = softmax(target /
 * temperature) and q = softmax(draft / temperature) of a row (q = 1 for the
 * draft without them), draft d of row i is kept while u[b][i] * q(d) < p(d). At
 * the first that is not, the stream's next token is the least j at which the
 * running sum of max(p - q, 0) passes u_next[b] times its total (without draft: p
 * without d), behind the last draft that of p; where rounding leaves none, or
 * u_next is 1 or more, the last j of any weight; where the whole residual is 0
 * or not a number, p is sampled. temperature 0 is greedy: a draft is kept if it
 * is the first of its row's largest logits, the next token is that, and u, u_next
 * and draft are not read. accepted[b] is the number of drafts kept; tokens
 * ([batch][t + 1]) the kept drafts, the next token, then -1; lp (null or
 * [batch][t + 1]) their log probabilities under softmax(target / temperature),
 * of temperature 1 where it is 0, then 0. A draft outside [0, n) is not kept.
 * A target row that holds NaN or +inf, or -inf alone, keeps nothing, and its
 * next token is -1 with the log probability 0; a draft row of that kind keeps
 * nothing. Exponentials and sums are float64. The outputs lie apart from the
 * inputs. What internal/search's steps of one token (beam.go:501-540) take
 * one by one. */
int nd_verify_drafts_dev(int32_t *accepted, int32_t *tokens, float *lp, const void *target, long long target_stream,
                         long long target_row, const void *draft, long long draft_stream, long long draft_row, int type,
                         int batch, int t, int n, const int32_t *drafts, const int32_t *drafted, const float *u,
                         const float *u_next, double temperature, void *stream);

#ifdef __cplusplus
}
#endif

#endif
