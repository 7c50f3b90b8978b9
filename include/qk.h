/*
 * qk.h - C ABI of the MI355X (gfx950) Q4_K / Q6_K dequant-GEMV library.
 *
 * Drop-in boundary for inferencer.cu's quantized matrix path.  The reference
 * has no plugin layer: its kernels are launched from FastGPU / FastRunner.
 * Each entry point below names the reference code it replaces.  Conventions
 * shared by every call:
 *
 *  - Weights are GGUF/GGML super-block bytes, rows contiguous, row stride
 *    (cols/256) * 144 B for Q4_K (type 12) and (cols/256) * 210 B for Q6_K
 *    (type 14) (inferencer.cu:252-259, 652).  cols = dims[0] is a multiple
 *    of 256, rows = dims[1] (inferencer.cu:184-185).
 *  - Activations and outputs are fp32.  Outputs are overwritten, never
 *    accumulated (inferencer.cu:660); inputs and outputs must not alias.
 *  - Device pointers only.  Weight bases must be 16-byte aligned (GGUF tensor
 *    data is aligned to general.alignment, default 32: inferencer.cu:270-272);
 *    fp32 activation bases and leading dimensions must keep 16-byte alignment.
 *  - stream is a hipStream_t (NULL selects the null stream).  Calls are
 *    asynchronous, allocate nothing and keep no per-call state: they are
 *    reentrant and may be issued from several host threads.
 *  - Every call validates its arguments on the host before any launch and
 *    returns a qk status (QK_OK = 0).  Nothing throws across the ABI; the
 *    reference's runtime_error texts (inferencer.cu:126-128, 1157-1158) map
 *    to the status plus qk_last_error(), a thread-local message.
 */
#ifndef QK_H
#define QK_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Storage type ids: the GGUF type numbers of storage_name (inferencer.cu:194-202). */
#define QK_TYPE_F32 0
#define QK_TYPE_F16 1
#define QK_TYPE_Q4_K 12
#define QK_TYPE_Q6_K 14
/* A Q6_K matrix in the split layout made by qk_q6k_split (no reference
   counterpart): the same 210 bytes per super-block, each row of nb =
   cols/256 blocks stored as four streams -- ql [nb][128], qh [nb][64],
   scales [nb][16], d [nb] (fp16) -- and padded to a multiple of 16 bytes,
   so every field a kernel reads is 16-byte aligned (in the GGUF layout a
   Q6_K block is only 2-byte aligned at odd block indices).  Accepted
   wherever Q6_K is. */
#define QK_TYPE_Q6_K_SPLIT 114
/* Types of paged cache rows (besides QK_TYPE_F16); no weights have them. */
#define QK_TYPE_I8 24
#define QK_TYPE_F8_E4M3 120
#define QK_TYPE_I4 121

/* Status codes. */
#define QK_OK 0
#define QK_ERR_INVALID_ARG 1   /* null pointer, negative count, bad leading dimension */
#define QK_ERR_SHAPE 2         /* cols not a positive multiple of 256, rows < 1 */
#define QK_ERR_TYPE 3          /* storage type other than Q4_K / Q6_K / Q6_K split */
#define QK_ERR_ALIGN 4         /* base pointer or leading dimension misaligned */
#define QK_ERR_DEVICE 5        /* HIP runtime error at launch */
#define QK_ERR_LIMIT 6         /* size beyond what the kernels index */
#define QK_ERR_FORMAT 7        /* malformed or unsupported GGUF file */
#define QK_ERR_IO 8            /* file cannot be opened or mapped */

typedef void *qk_stream;

/* ------------------------------------------------------------ utility -- */

/* Status text; replaces the cuda_check / runtime_error messages
   (inferencer.cu:126-128). */
const char *qk_status_string(int status);
/* Detail of the last failing call on this host thread ("" if none). */
const char *qk_last_error(void);
/* Bytes per 256-value super-block (144 / 210; 0 for other types) and bytes of
   a cols x rows tensor: the size rule of inferencer.cu:252-259 (split Q6_K
   rows rounded up to 16 bytes). */
int qk_block_bytes(int type);
int64_t qk_tensor_bytes(int type, int64_t cols, int64_t rows);

/* ------------------------------------------------ FP32 dequant-GEMV -- */

/* Precision of the FP32 entry points (this section, the FP32 step kernels
   that feed them and the FP32 decode drivers): x is carried as 22-bit block
   fixed point per 16 consecutive values, X = rint(x * 2^(21-e)) with e =
   ilogb of the group's largest |x|, so each value is rounded to within
   2^(e-22) -- relative 2^-22 for the group's largest value, coarser for
   values far below it -- and the products and sums that follow are exact
   integer dots plus fp32 combines.  An output therefore differs from the
   reference's fp32 products by at most sum_c |W[r][c]| 2^(e_c - 22) plus
   fp32 rounding (tests/test_gpu_gemv.py pins both terms); on N(0, 1)-like
   activations that is within 1e-6 rel-L2 of an fp64 product.  The
   multi-token forms carry the same 22 bits per 256-column block as fp16
   high / low halves.  The INT8 entry points below follow the reference's
   INT8 arithmetic instead. */

/* y[r] = sum_c W[r][c] * x[c] for r < rows.
   Replaces FastGPU::matvec's FP32 branch (inferencer.cu:1156-1171) and the
   gemv_quant<12|14> kernel (inferencer.cu:645-661) it launches. */
int qk_gemv_f32(int type, const void *w, const float *x, float *y, int cols, int rows,
                qk_stream stream);

/* One matrix of a fused launch. */
typedef struct qk_matrix {
    int type;          /* QK_TYPE_Q4_K or QK_TYPE_Q6_K */
    int rows;
    const void *w;
    float *y;          /* rows outputs */
} qk_matrix;

/* Several matrices that share x and cols, in one launch: y_m = W_m x.
   Replaces qkv_cuda (inferencer.cu:753-784: Q, K and a Q4_K or Q6_K V) and
   gate_up_cuda (inferencer.cu:786-804).  At most QK_MAX_FUSED matrices. */
#define QK_MAX_FUSED 8
int qk_gemv_multi_f32(const qk_matrix *mats, int n_mats, const float *x, int cols,
                      qk_stream stream);

/* Device workspace a multi-token call needs: cols activations, `rows` output
   rows in total (the sum over the matrices of a fused call) and n_tokens
   tokens.  From 8 tokens on it holds the activations packed for the matrix
   cores (4.1 KiB per token and 256 columns, tokens rounded up to 32) and,
   when one row group's blocks are split over several workgroups, their
   partial sums; below 8 tokens it is 0 and the pointer may be NULL.  It
   plays the part of the reference's preallocated batch buffers
   (inferencer.cu:1237-1238) and never needs clearing.  Base alignment 256
   bytes.  With this many bytes or more, what a call adds in which order
   depends on the call alone; from 33 tokens on, a smaller buffer that holds
   what the call cannot do without is accepted too and may get fewer splits
   (the same sums, rounded in another order).  The same holds for the queries
   of the feed-forward block and of the INT8 products below. */
size_t qk_gemv_batched_workspace_bytes(int cols, int rows, int n_tokens);

/* Multi-token variant: y[t*ldy + r] = sum_c W[r][c] * x[t*ldx + c] for
   t < n_tokens (token-major like inferencer.cu:698).  The FP32 arithmetic
   above (22-bit block fixed point per 256-column block) applied to the
   reference's batched path FastRunner::batch_matvec +
   gemv_batch_dp4a (inferencer.cu:1265-1278, 678-699), without its 32-token
   cap; n_tokens = 0 is a no-op.  workspace holds at least
   qk_gemv_batched_workspace_bytes(cols, rows, n_tokens) device bytes and
   must not be shared by calls in flight at the same time. */
int qk_gemv_batched_f32(int type, const void *w, const float *x, int ldx, float *y, int ldy,
                        int cols, int rows, int n_tokens, void *workspace,
                        size_t workspace_bytes, qk_stream stream);

/* Fused multi-token launch over matrices sharing x: y_m[t*rows_m + r].
   Replaces qkv_batch_cuda (inferencer.cu:701-731) and gate_up_batch_cuda
   (inferencer.cu:733-751). */
int qk_gemv_multi_batched_f32(const qk_matrix *mats, int n_mats, const float *x, int ldx,
                              int cols, int n_tokens, void *workspace, size_t workspace_bytes,
                              qk_stream stream);

/* The feed-forward block of n_tokens tokens: y[t*ldy + r] (+)= (W_down
   (SiLU(W_gate x_t) * (W_up x_t)))[r] -- gate and up are hidden x dim (cols
   dim), down dim x hidden; `accumulate` adds into y (the residual; y may be
   x).  Replaces the reference's batched FFN sequence gate_up_batch_cuda +
   silu_cuda + the down projection (inferencer.cu:733-751, 1043-1056,
   1362-1380) with FP32 semantics.  From 8 tokens on it runs as five
   launches on the matrix cores: the gate / up reduction packs SiLU(gate) *
   up straight into the down projection's input records, so neither gate,
   up nor their product is stored as fp32; below 8 tokens, the fused GEMV pair
   of qk_gemv_multi_f32 and a down GEMV staging SiLU * up, or, where that is
   estimated to take less time (2 to 7 tokens, gate and up of one type), one
   read of their weights on the matrix cores that writes SiLU * up, and a down
   launch over it.  workspace:
   qk_ffn_batched_workspace_bytes(dim, hidden, n_tokens) bytes (256-byte
   aligned; also enough for fewer tokens), not shared by calls in flight at
   the same time.  dim and hidden multiples of 256.  No reference
   counterpart as one call. */
size_t qk_ffn_batched_workspace_bytes(int dim, int hidden, int n_tokens);
int qk_ffn_batched_f32(int gate_type, const void *gate, int up_type, const void *up, int down_type, const void *down,
                       const float *x, int ldx, float *y, int ldy, int dim, int hidden, int n_tokens, int accumulate,
                       void *workspace, size_t workspace_bytes, qk_stream stream);

/* ------------------------------------------------------------ dequant -- */

/* out[r*cols + c] = W[row0 + r][c] as fp32, bit-exact with q4_value /
   q6_value (inferencer.cu:454-487). */
int qk_dequant_rows(int type, const void *w, float *out, int cols, int row0, int nrows,
                    qk_stream stream);

/* Copy a cols x rows Q6_K matrix (GGUF block bytes at src) into the split
   layout of QK_TYPE_Q6_K_SPLIT at dst (qk_tensor_bytes(QK_TYPE_Q6_K_SPLIT,
   cols, rows) bytes, 16-byte aligned, not overlapping src).  A load-time
   step: the block bytes are moved, never decoded. */
int qk_q6k_split(const void *src, void *dst, int cols, int rows, qk_stream stream);

/* out[t*cols + c] = W[tokens[t]][c]; tokens is a device array of n_tokens
   ids in [0, vocab).  Replaces embedding_cuda / embedding_batch_cuda
   (inferencer.cu:806-819); any Q4_K, Q6_K or split Q6_K table. */
int qk_embedding(int type, const void *w, const int32_t *tokens, int n_tokens, float *out,
                 int cols, int vocab, qk_stream stream);

/* y = W x as qk_gemv_f32, and out[0] = the lowest row index among the
   maxima of y (NaN never wins; 0 when no value exceeds -inf): the LM head and
   the greedy pick of argmax_blocks_cuda / argmax_final_cuda
   (inferencer.cu:1414, 1523-1526, 1063-1099) in two launches -- each GEMV
   workgroup keeps the best of the rows it stores, one small kernel reduces
   those partials.  workspace: qk_gemv_argmax_workspace_bytes() bytes, 4-byte
   aligned; calls sharing it must not overlap. */
size_t qk_gemv_argmax_workspace_bytes(void);
int qk_gemv_argmax_f32(int type, const void *w, const float *x, float *y, int cols, int rows, int32_t *out,
                       void *workspace, qk_stream stream);

/* qk_gemv_argmax_f32 without a workspace argument and without any device
   allocation: the partials live in a 128 KiB array compiled into the library
   (one per GPU, held until the process ends).  No reference counterpart: it
   serves callers that cannot allocate or pass a workspace (code under HIP
   graph capture, tight serving loops).  Any rows / cols that
   qk_gemv_argmax_f32 accepts fit the array (the GEMV keeps at most 16384
   partials); the call otherwise fails with QK_ERR_LIMIT before its
   argmax launch.  Every call on one GPU shares the array and leaves its
   partials there: calls that overlap on one GPU (two streams, two host
   threads) race and must be serialised by the caller. */
int qk_gemv_argmax_f32_noalloc(int type, const void *w, const float *x, float *y, int cols, int rows,
                               int32_t *out, qk_stream stream);

/* ---------------------------------------------------------- INT8 mode -- */

/* Per 32 values: scale = amax/127 (1 if amax == 0), xq = clamp(rne(x/scale),
   -127, 127).  Token t reads x + t*ldx and writes xq + t*ldxq, xscale +
   t*ldscale (the reference's fixed strides are 8192 and 256,
   inferencer.cu:687-688).  Replaces quantize_x32_cuda (inferencer.cu:544-556)
   and quantize_batch_cuda (inferencer.cu:891-904). */
int qk_quantize_x32(const float *x, int ldx, int8_t *xq, int ldxq, float *xscale, int ldscale,
                    int cols, int n_tokens, qk_stream stream);

/* RMSNorm and the per-32 quantization in one launch: out = x * 1/sqrt(
   mean(x^2) + eps) * weight exactly as qk_rmsnorm_f32 (out may be NULL to
   skip the fp32 copy), then xq / xscale of those values exactly as
   qk_quantize_x32 -- bit-identical to the two calls in sequence.  Token t
   reads x + t*ldx and writes out + t*ldout, xq + t*ldxq, xscale + t*ldscale.
   cols % 32 == 0 (QK_ERR_SHAPE); x, weight and out 16-byte aligned with ldx,
   ldout multiples of 4, xq 4-byte aligned with ldxq a multiple of 4
   (QK_ERR_ALIGN).  Replaces rmsnorm_quantize_cuda and
   rmsnorm_quantize_batch_cuda (inferencer.cu:839-889; the reference's batch
   strides are 8192 and 256). */
int qk_rmsnorm_quantize_x32(const float *x, int ldx, const float *weight, float *out, int ldout,
                            int8_t *xq, int ldxq, float *xscale, int ldscale, int cols, int n_tokens,
                            float eps, qk_stream stream);

/* INT8-activation GEMV for n_tokens tokens (1 = decode): exact integer
   sub-block dots, fp32 combine.  Replaces gemv_q4_dp4a / gemv_q6_dp4a
   (inferencer.cu:558-569, 663-674) and gemv_batch_dp4a
   (inferencer.cu:678-699). */
int qk_gemv_i8(int type, const void *w, const int8_t *xq, int ldxq, const float *xscale,
               int ldscale, float *y, int ldy, int cols, int rows, int n_tokens,
               qk_stream stream);

/* qk_gemv_i8 for a batch of tokens: y[t*ldy + r] for t < n_tokens, the
   reference's INT8 multi-token semantics (gemv_batch_dp4a, inferencer.cu:
   678-699; its default batched mode, inferencer.cu:1611) without the
   32-token cap and without re-reading the weights per token.  From 8 tokens
   on the exact integer sub-block dots run on the integer matrix cores
   (v_mfma_i32_32x32x32_i8 per Q4_K sub-block of 32 columns,
   v_mfma_i32_32x32x16_i8 per Q6_K sub-block of 16) for 32 tokens x 32 rows
   at a time, and each sub-block is combined in fp32 as the reference does:
   (d*sc*dot - dmin*m*sum(xq)) * xscale (Q4_K, inferencer.cu:520-542) and
   d*scale*dot*xscale (Q6_K, 613-643; two sub-blocks sharing an xscale are
   added in integers first); below 8 tokens it is qk_gemv_i8.  A workgroup
   takes 32 rows x 32 tokens x up to 12 or 16 blocks of the row, one per
   wave.  Each launch's plan, chosen from the kernels' occupancy on the
   device, may split rows over workgroups, whose sums a second launch adds
   in split order (deterministic), and a launch larger than the chip holds
   at once lets resident workgroups walk the row tiles or, with enough
   tokens, takes 128 rows x 64 tokens a workgroup with the integer scales
   folded into fp16 operands (the same exact sub-block sums, scaled per 32
   columns and then by d).  The workspace
   holds the split sums of any plan:
   qk_gemv_batched_i8_workspace_bytes(cols, rows, n_tokens) bytes, 16-byte
   aligned (0, and NULL allowed, below 8 tokens or at 256 columns; a plan
   without splits ignores it). */
size_t qk_gemv_batched_i8_workspace_bytes(int cols, int rows, int n_tokens);
int qk_gemv_batched_i8(int type, const void *w, const int8_t *xq, int ldxq, const float *xscale, int ldscale,
                       float *y, int ldy, int cols, int rows, int n_tokens, void *workspace, size_t workspace_bytes,
                       qk_stream stream);

/* Fused INT8 GEMV over 1..QK_MAX_FUSED matrices sharing one token's
   quantized activations (xq: cols int8, xscale: cols/32): the dp4a branch of
   qkv_cuda / gate_up_cuda (inferencer.cu:753-804) for any mix of Q4_K and
   Q6_K (either layout).  Each matrix's rows go to its own y. */
int qk_gemv_multi_i8(const qk_matrix *mats, int n_mats, const int8_t *xq, const float *xscale, int cols,
                     qk_stream stream);

/* The fused form of qk_gemv_batched_i8 (qkv_batch_cuda, gate_up_batch_cuda,
   inferencer.cu:701-751): 1..QK_MAX_FUSED matrices (any mix of Q4_K, Q6_K
   and split Q6_K) of cols columns read the same n_tokens quantized rows (xq
   + t*ldxq, xscale + t*ldscale); mats[m].y receives [n_tokens][rows_m].
   One launch from 8 tokens on (two when the plan splits the rows);
   workspace qk_gemv_batched_i8_workspace_bytes(cols, sum of the rows,
   n_tokens). */
int qk_gemv_multi_batched_i8(const qk_matrix *mats, int n_mats, const int8_t *xq, int ldxq, const float *xscale,
                             int ldscale, int cols, int n_tokens, void *workspace, size_t workspace_bytes,
                             qk_stream stream);

/* The feed-forward block in the reference's INT8 batched arithmetic for
   n_tokens quantized rows of dim values: gate / up (gate_up_batch_cuda,
   inferencer.cu:733-751), SiLU(gate) * up (silu_batch_cuda) quantized per 32
   values (quantize_batch_cuda, 891-904), down (gemv_batch_dp4a), into
   y[t*ldy + c] (overwritten, or added with accumulate: add_batch_cuda).
   From 8 tokens on, the gate / up product forms SiLU * up and its
   quantization in its own epilogue (or its reduction launch when the plan
   splits its rows), then down.  gate and up have one storage type.  The workspace
   holds the quantized hidden rows and the split sums:
   qk_ffn_batched_i8_workspace_bytes(dim, hidden, n_tokens), 256-byte
   aligned (also enough for fewer tokens). */
size_t qk_ffn_batched_i8_workspace_bytes(int dim, int hidden, int n_tokens);
int qk_ffn_batched_i8(int gate_type, const void *gate, int up_type, const void *up, int down_type, const void *down,
                      const int8_t *xq, int ldxq, const float *xscale, int ldscale, float *y, int ldy, int dim,
                      int hidden, int n_tokens, int accumulate, void *workspace, size_t workspace_bytes,
                      qk_stream stream);

/* -------------------------------------------------------- step kernels -- */

/* out = x * 1/sqrt(mean(x^2) + eps) * weight per token of n values.
   Replaces rmsnorm_cuda (inferencer.cu:821-834). */
int qk_rmsnorm_f32(const float *x, const float *weight, float *out, int n, int n_tokens,
                   float eps, qk_stream stream);

/* Rotates q (heads*head_dim) and k (kv_heads*head_dim) in adjacent pairs at
   position pos, writes rotated k and v into the caches at
   [(layer*context + pos)*kv_dim].  Tables are [context][head_dim/2].
   Replaces rope_cache_cuda / rope_cuda + cache_cuda (inferencer.cu:906-951),
   generalised from head_dim 128. */
int qk_rope_kv_write(float *q, const float *k, const float *v, const float *cosine,
                     const float *sine, float *key_cache, float *value_cache, int layer, int pos,
                     int context, int heads, int kv_heads, int head_dim, qk_stream stream);

/* GQA attention of one query token over cache positions 0..pos of a layer
   (caches and out 16-byte aligned).  Replaces attention_cuda
   (inferencer.cu:981-1009), generalised head_dim. */
int qk_attention_f32(const float *q, const float *key_cache, const float *value_cache,
                     float *out, int layer, int pos, int context, int heads, int kv_heads,
                     int head_dim, qk_stream stream);

/* x += y (add_cuda, inferencer.cu:1043-1046). */
int qk_add_f32(float *x, const float *y, int n, qk_stream stream);

/* gate = gate / (1 + exp(-gate)) * up (silu_cuda, inferencer.cu:1053-1056). */
int qk_silu_mul_f32(float *gate, const float *up, int n, qk_stream stream);

/* Index of the maximum of v[0..n), lowest index among equal maxima, into
   *out (device).  workspace holds qk_argmax_workspace_bytes(n) device bytes.
   Replaces argmax_blocks_cuda + argmax_final_cuda (inferencer.cu:1063-1099). */
size_t qk_argmax_workspace_bytes(int n);
int qk_argmax_f32(const float *v, int n, int32_t *out, void *workspace, qk_stream stream);

/* ----------------------------------------------- ragged decode batches -- */

/* One token of a ragged batch: the position of the token in its sequence
   and the first row of that sequence in the packed KV caches
   ([layer][cache_rows][kv_dim]; a sequence owns rows kv_row .. kv_row +
   capacity - 1).  The token's key / value go to row kv_row + pos and it
   attends to rows kv_row .. kv_row + pos.  The nearest reference code serves
   one sequence at contiguous positions (start_pos + token,
   inferencer.cu:956-959, 1012-1016); this descriptor lets the tokens of a
   batch come from any mix of sequences -- one decode token each, or a chunk
   of consecutive positions of one sequence (prefill). */
typedef struct qk_batch_token {
    int32_t pos;
    int32_t seq;       /* sequence id; informational (kv_row identifies the rows) */
    int64_t kv_row;
} qk_batch_token;

/* RoPE of token t's q (heads*head_dim at q + t*heads*head_dim, in place) and
   k at its own position, k and v written to row kv_row + pos of `layer`.
   desc is a device array of n_tokens entries; tokens outside the cache
   (pos >= context or kv_row + pos >= cache_rows) are skipped.  Replaces
   rope_cache_batch_cuda (inferencer.cu:953-979). */
int qk_rope_kv_write_batched(float *q, const float *k, const float *v, const float *cosine, const float *sine,
                             float *key_cache, float *value_cache, int layer, int64_t cache_rows,
                             const qk_batch_token *desc, int n_tokens, int context, int heads, int kv_heads,
                             int head_dim, qk_stream stream);

/* GQA attention of every token of a ragged batch over rows kv_row ..
   kv_row + pos of its sequence; out is [n_tokens][heads*head_dim] (16-byte
   aligned, like the caches).  max_pos bounds every pos; a token beyond it or
   beyond the cache gets NaN outputs.  Replaces attention_batch_cuda
   (inferencer.cu:1011-1041). */
int qk_attention_batched_f32(const float *q, const float *key_cache, const float *value_cache, float *out, int layer,
                             int64_t cache_rows, const qk_batch_token *desc, int n_tokens, int max_pos, int heads,
                             int kv_heads, int head_dim, qk_stream stream);

/* qk_attention_batched_f32 with every token's rows spread over several
   workgroups: rows 0..pos of a token are cut into splits of split_rows rows
   (0: chosen from the batch), each split leaves a partial (max, sum of exp,
   output) in workspace and a second kernel merges them in split order.  A
   token whose rows fit one split is written directly.  workspace holds
   qk_attention_split_workspace_bytes(n_tokens, ..., max_pos) bytes for the
   chosen split; with less (or none) the call takes fewer, longer splits.
   Calls sharing a workspace must not overlap.  No reference counterpart:
   attention_cuda (inferencer.cu:981-1009) runs one block per head over the
   whole context, which one CU reads at a few tens of GB/s. */
size_t qk_attention_split_workspace_bytes(int n_tokens, int heads, int kv_heads, int head_dim, int max_pos,
                                          int split_rows);
int qk_attention_split_f32(const float *q, const float *key_cache, const float *value_cache, float *out, int layer,
                           int64_t cache_rows, const qk_batch_token *desc, int n_tokens, int max_pos, int heads,
                           int kv_heads, int head_dim, int split_rows, void *workspace, size_t workspace_size,
                           qk_stream stream);

/* Greedy token of each of `rows` rows of n values (row r at v + r*ldv), the
   lowest index among equal maxima; out is a device array of rows ints.
   workspace holds qk_argmax_rows_workspace_bytes(n, rows) bytes.  The
   per-token form of argmax_blocks_cuda + argmax_final_cuda. */
size_t qk_argmax_rows_workspace_bytes(int n, int rows);
int qk_argmax_rows_f32(const float *v, int n, int64_t ldv, int rows, int32_t *out, void *workspace,
                       qk_stream stream);

/* ------------------------------------- paged cache of a serving step -- */

/* No reference counterpart (its one fp32 cache holds one sequence).  A step
   over a paged cache: qk_rope_tables_f32 once, then per layer
   qk_rope_paged_write and qk_paged_attention_f32, and qk_sample_rows_f32 over
   the logits. */

/* One layer's cache: a pool of pages.  Row `slot` of page `page` of KV head h
   is the head_dim values from ((page * kv_heads + h) * page_rows + slot) *
   head_dim of key (and of value), and the fp32 scale at (page * kv_heads + h)
   * page_rows + slot of key_scale (value_scale):
     QK_TYPE_F16      fp16, rounded to nearest even; no scales (NULL).
     QK_TYPE_I8       int8 code * scale; written with scale = max|x| / 127 and
                      code = x / scale rounded to nearest, ties to even.
     QK_TYPE_F8_E4M3  float8 (4-bit exponent, 3-bit mantissa, no infinities)
                      code * scale; written with scale the least power of two
                      that keeps the row within 448, code = x / scale to
                      nearest even.
     QK_TYPE_I4       4-bit code * multiplier * scale.  Codes are of two's
                      complement, two a byte, the earlier value in the low half:
                      a row is head_dim / 2 bytes.  A row's entry of key_scale
                      (value_scale) is 8 bytes: the fp32 scale, then a multiplier
                      (one byte, 1 to 255) for each quarter of the row's values.
                      Written with scale the least number of 13 significant bits
                      with 1785 scale >= max|x| (and finite), the multiplier the
                      least with 7 multiplier scale >= its quarter's max|x|, code
                      = x / (multiplier scale) to nearest even, -7 to 7: a value
                      as written is an fp32 number.
   A row whose largest magnitude is below 2^-100 is written as zeros with scale
   1 (multipliers 1), one that holds a value that is not finite as zeros with
   scale NaN (I8, I4, E4M3).  head_dim 64, 96, 128 or 256; page_rows a power of two, 16 to 1024;
   every base 16-byte aligned. */
typedef struct qk_paged_kv {
    int type;
    int kv_heads, head_dim, page_rows;
    int64_t pages;
    void *key, *value;
    float *key_scale, *value_scale;
} qk_paged_kv;

/* One sequence of a call: its new tokens are rows first .. first + count - 1
   of q, k, v and out (rows of no other sequence), at positions pos .. pos +
   count - 1; its row r lies in page page_table[table * table_stride + r /
   page_rows]. */
typedef struct qk_paged_seq {
    int32_t first, count, pos, table;
} qk_paged_seq;

/* The sequences of a call.  page_table is a device array [table_rows]
   [table_stride]; an entry outside [0, pages) is a page that is absent.  seqs
   is a device array of n_seqs entries, n_tokens the token rows of q, k, v and
   out, max_count and max_rows bounds of count and of pos + count: a call may
   take time and workspace by them.  A sequence with count < 1 or a negative
   entry, with more than max_count tokens or max_rows rows, with tokens beyond
   n_tokens, with rows beyond the table's stride or a table row beyond
   table_rows is left out: nothing of it is read or written. */
typedef struct qk_paged_batch {
    const int32_t *page_table;
    int table_rows, table_stride;
    const qk_paged_seq *seqs;
    int n_seqs, n_tokens, max_count, max_rows;
} qk_paged_batch;

/* How the rotary frequencies of rot_dim / 2 pairs, theta^(-2 i / rot_dim), are
   scaled for contexts longer than the trained one:
     QK_ROPE_NONE    as they are
     QK_ROPE_LINEAR  / factor
     QK_ROPE_LLAMA3  / factor where they turn less than low_freq_factor times
                     over original_context, as they are from high_freq_factor
                     turns on, in between mixed by the turns
     QK_ROPE_YARN    from pair low to pair high a linear ramp from unscaled to
                     / factor, low and high the pairs that turn beta_fast and
                     beta_slow times over original_context (rounded outwards,
                     within 0 .. rot_dim - 1); cosines and sines times
                     attention_factor (0: 0.1 ln(factor) + 1) */
#define QK_ROPE_NONE 0
#define QK_ROPE_LINEAR 1
#define QK_ROPE_LLAMA3 2
#define QK_ROPE_YARN 3
typedef struct qk_rope_scaling {
    int type;
    float factor, low_freq_factor, high_freq_factor, original_context, beta_fast, beta_slow, attention_factor;
} qk_rope_scaling;

/* cosine[p * rot_dim / 2 + i] and sine[...] of (first_pos + p) * f_i for p <
   positions, in 64 bits, rounded once: the tables that qk_rope_kv_write* and
   qk_rope_paged_write take.  (The decode drivers build their own from rope_theta
   and take none.)  scaling may be NULL (QK_ROPE_NONE); freq_factors (device,
   rot_dim / 2 values, or NULL) divide the frequencies before the scaling (a GGUF
   file's rope_freqs.weight).  rot_dim even, at most 512; at most 2^30 positions;
   cosine and sine share nothing. */
int qk_rope_tables_f32(float theta, int rot_dim, const qk_rope_scaling *scaling, const float *freq_factors,
                       int first_pos, int positions, float *cosine, float *sine, qk_stream stream);

/* Rotates every new token's q and k at its position and writes k and v into
   the pages.  q is [n_tokens] rows of heads * head_dim values, ldq apart, its
   rotation goes to q_out (which may be q with ldq_out = ldq, but share nothing
   else with q, k or v; or NULL with q NULL: no queries); k and v are rows of
   kv_heads * head_dim.  The first rot_dim values of a head rotate (0: none, and
   no tables), in pairs (2 i, 2 i + 1) or, with `half`, (i, i + rot_dim / 2), by
   the tables' row of the token's position, in 64 bits, rounded once.  Tables
   have `positions` rows of rot_dim / 2 values; a sequence that reaches beyond
   them is left out.  A token whose page is absent writes no row (its q is
   rotated).  No two tokens of a call may have the same row.  q, q_out, k, v
   16-byte aligned with leading dimensions multiples of 4. */
int qk_rope_paged_write(const qk_paged_kv *kv, const qk_paged_batch *batch, const float *q, int ldq, float *q_out,
                        int ldq_out, const float *k, int ldk, const float *v, int ldv, int heads, const float *cosine,
                        const float *sine, int positions, int rot_dim, int half, qk_stream stream);

/* The rows of every sequence's count tokens as fp32: row pos + i of a sequence
   goes to row first + i of key_out and value_out (rows of kv_heads * head_dim,
   ldk and ldv apart, that share nothing; either may be NULL).  Rows of absent
   pages are 0.  16-byte aligned, leading dimensions multiples of 4. */
int qk_paged_read_f32(const qk_paged_kv *kv, const qk_paged_batch *batch, float *key_out, int ldk, float *value_out,
                      int ldv, qk_stream stream);

/* GQA attention of every new token over its sequence's rows 0 .. its own
   position (which hold them already): out = softmax(scale q K^T) V, scale 1 /
   sqrt(head_dim) when 0.  q and out are [n_tokens] rows of heads * head_dim,
   ldq and ldout apart; out may be q with ldout = ldq, or shares nothing with it.
   Rows of absent pages take no part; a token that sees no row gets zeros.
   Products keep every bit of the cache, 22 bits of q, and of a token's
   probabilities times value scales 22 bits or 2^-32 of the largest, whatever the
   scales of rows that it does not see or gives no weight (value scales of a
   sequence within 2^100 of each other).  A key or value that is not finite makes
   the outputs of the tokens that see it not finite, and reaches no other.
   workspace holds partial results when a sequence's rows are split over
   workgroups; with less than the queried bytes (or none) the call takes fewer
   splits.  Calls sharing a workspace must not overlap.  Base alignments 16 bytes,
   leading dimensions multiples of 4. */
size_t qk_paged_attention_workspace_bytes(const qk_paged_batch *batch, int heads, int kv_heads, int head_dim);
int qk_paged_attention_f32(const qk_paged_kv *kv, const qk_paged_batch *batch, const float *q, int ldq, float *out,
                           int ldout, int heads, float scale, void *workspace, size_t workspace_bytes,
                           qk_stream stream);

/* What a model adds to the scores of attention and which rows its tokens see.  Of
   a token at position p and a row r, with s = scale q k:
     cap     s = cap tanh(s / cap); 0: not.  From 2^-64 to 2^64.
     slopes  s - slopes[head] |p - r| (after the cap); a device array of `heads`
             finite values, or NULL.
     window  rows with p - r < window alone; 0: all.
     prefix  besides rows 0 .. p, those below prefix[sequence] (a device array of
             n_seqs values, in the order of seqs; or NULL) that the sequence has
             by the end of the call: its first rows see each other.
   All zeros: none. */
typedef struct qk_attention_terms {
    float cap;
    int window;
    const float *slopes;
    const int32_t *prefix;
} qk_attention_terms;

/* qk_paged_attention_f32 with terms (NULL: none).  A row that a token does not see
   takes no part in it, whatever it holds; rows that no token of a call sees are
   not read beyond the tile (32 or 64 rows) that a seen one shares with them. */
size_t qk_paged_attention_terms_workspace_bytes(const qk_paged_batch *batch, int heads, int kv_heads, int head_dim,
                                                int window);
int qk_paged_attention_terms_f32(const qk_paged_kv *kv, const qk_paged_batch *batch, const float *q, int ldq, float *out,
                                 int ldout, int heads, float scale, const qk_attention_terms *terms, void *workspace,
                                 size_t workspace_bytes, qk_stream stream);

/* A pool of pages and the table of the sequences that hold them: page_table
   [table_rows][table_stride] (what qk_paged_batch takes) and refs, of each page the
   number of table entries that name it; both on the device, with all entries -1 and
   all refs 0 an empty pool.  layers is a host array of n_layers caches of these pages
   (0: none; contents then stay where they are).  At most 2^30 pages and table
   entries, refs 16-byte aligned.  The calls below keep refs right; entries that name
   no page count as absent.  They run on the device alone (no value comes back to the
   host) and give the same result for the same table and refs. */
typedef struct qk_page_pool {
    int32_t *page_table;
    int table_rows, table_stride;
    int32_t *refs;
    int64_t pages;
    int page_rows;
    const qk_paged_kv *layers;
    int n_layers;
} qk_page_pool;

/* Workspace of the three calls below, 16-byte aligned; calls sharing it, or the
   pool, must not overlap.  What a call writes (table, refs, its number, workspace)
   may share no memory with its other arguments. */
size_t qk_pages_workspace_bytes(const qk_page_pool *pool);

/* Every table row r with lengths[r] >= 0 comes to hold the pages of its rows
   begins[r] .. lengths[r] - 1 (begins NULL: from 0) and no others: entries before
   begins[r] / page_rows and from ceil(lengths[r] / page_rows) on give their pages
   back (0: the whole row), absent ones between take free pages, in order of table
   rows and entries the lowest page first.  Pages that the call takes back are free for
   it.  lengths and begins are device arrays of table_rows values.  (Before a step
   through a window of w rows begins[r] is its first new token's position less w - 1:
   that token sees the rows from there on.)  missing (device, or NULL) receives the
   number of entries that got no page (and stay absent), those beyond the table's
   stride included. */
int qk_pages_resize(const qk_page_pool *pool, const int32_t *begins, const int32_t *lengths, int32_t *missing,
                    void *workspace, size_t workspace_bytes, qk_stream stream);

/* Every table row c whose parents[c] is another table row becomes a fork of that row
   as it was before the call, of its first lengths[c] rows: it gives its own pages back,
   shares the pages that these rows fill, and the contents of the last page, where they
   fill a part of it, are copied in every layer into a page that was free before the
   call (lowest first, in order of c).  Other rows (parents[c] out of range, or c
   itself) stay as they are.  Entries absent in the parent are absent.  Rows may be
   forked from rows that are forked themselves.  missing as above: forks without a
   page for the last part.
   Rows that follow a fork's or its parent's lie in pages of their own.  A row that is
   cut back (qk_pages_resize) into a page that others hold too still shares it: before
   new rows are written there, it is to be forked from one of those that hold it. */
int qk_pages_fork(const qk_page_pool *pool, const int32_t *parents, const int32_t *lengths, int32_t *missing,
                  void *workspace, size_t workspace_bytes, qk_stream stream);

/* Of n pages that are held, those numbered n and more move to the free ones below, in
   order: contents in every layer, table entries and refs.  moved (device, or NULL)
   receives their number. */
int qk_pages_compact(const qk_page_pool *pool, int32_t *moved, void *workspace, size_t workspace_bytes,
                     qk_stream stream);

/* The contents of page source[i] into page target[i], i < n, in every layer (device
   arrays; pairs that name no page are left out).  No page is a target twice, or a
   target and a source. */
int qk_pages_copy(const qk_paged_kv *layers, int n_layers, const int32_t *source, const int32_t *target, int n,
                  qk_stream stream);

/* The next token of each of `rows` rows of n logits (row r at logits + r *
   ldv).  Of row r, with w_i = exp((logit_i - max) / temperature[r]) held to 2^-30
   of itself and 2^-45 (a token below that may have no weight), tokens in
   descending order of their logits (equal ones by index):
     top_k[r]  keeps the first top_k (<= 0: all),
     top_p[r]  of those the shortest run whose weights reach top_p of their sum
               (1: all),
     min_p[r]  of those the tokens with w_i >= min_p (0: all),
   and the first always; out[r] is the first token in index order at which the
   running sum of the kept weights exceeds uniform[r] (in [0, 1)) of their sum.
   prob (or NULL) receives its share of that sum.  temperature[r] <= 0, or a
   parameter that is NaN, keeps the first alone.  NaN logits count as -inf;
   where a logit is +inf, those that are share the weight.  A row without a
   logit above -inf gives 0 with prob 0.  A row's token does not depend on the
   other rows.  All arrays are on the device; temperature, top_k, top_p and min_p
   hold `rows` values, or are NULL: 1, and no filter.  At most 2^19 logits.  A row
   with thousands of tokens of like weight at the cut, with 16384 aligned logits
   that are all finite but far from its others (|logit / temperature| above some
   2800) or with a temperature of 2^60 takes ten to thirty times as long as others.
   workspace: qk_sample_rows_workspace_bytes(n, rows) bytes, 256-byte aligned;
   calls sharing it must not overlap. */
size_t qk_sample_rows_workspace_bytes(int n, int rows);
int qk_sample_rows_f32(const float *logits, int n, int64_t ldv, int rows, const float *temperature,
                       const int32_t *top_k, const float *top_p, const float *min_p, const float *uniform,
                       int32_t *out, float *prob, void *workspace, size_t workspace_bytes, qk_stream stream);

/* ---------------------------------------------------- decode-step driver -- */

/* Llama configuration (the llama.* GGUF keys read at inferencer.cu:1205-1214). */
typedef struct qk_llama_config {
    int dim, layers, heads, kv_heads, hidden, vocab, context;
    float eps, rope_theta;
} qk_llama_config;

/* Device pointers to one layer's tensors (blk.N.* names of inferencer.cu:1434-1502). */
typedef struct qk_llama_layer {
    int q_type, k_type, v_type, o_type, gate_type, up_type, down_type;
    const void *q, *k, *v, *o, *gate, *up, *down;
    const float *attn_norm, *ffn_norm;
} qk_llama_layer;

typedef struct qk_llama_weights {
    int embd_type;
    const void *token_embd;
    int output_type;
    const void *output;            /* NULL: tied to token_embd (inferencer.cu:1521-1522) */
    const float *output_norm;
    const qk_llama_layer *layers;  /* host array of cfg.layers entries */
} qk_llama_weights;

typedef struct qk_llama qk_llama;

/* Allocates the step buffers, KV cache and RoPE tables once (the FastGPU /
   FastRunner constructors, inferencer.cu:1115-1142, 1196-1249).  Every Q6_K
   tensor is copied once into the split layout (QK_TYPE_Q6_K_SPLIT, owned by
   the handle, freed by destroy); create returns after those copies, so the
   caller's Q6_K buffers may be released then.  Q4_K, split Q6_K and norm
   tensors are read in place at every step and stay owned by the caller.
   Like the reference's upload (inferencer.cu:329-333), create first checks
   that everything it allocates (caches, split copies, activation buffers,
   logits, workspaces) fits in free device memory with a 64 MiB margin
   (QK_ERR_DEVICE otherwise). */
int qk_llama_create(const qk_llama_config *cfg, const qk_llama_weights *w, qk_stream stream,
                    qk_llama **out);

/* Device bytes a decode handle holds: the split-layout Q6_K copies, the two
   KV caches, and every other buffer (activations, logits, workspaces, RoPE
   tables).  The copies cost as much as the model's Q6_K tensors (449 MB for
   the Llama-3.2-1B Q4_K_M-style mix). */
typedef struct qk_llama_memory {
    uint64_t weight_copies;
    uint64_t kv_cache;
    uint64_t buffers;
} qk_llama_memory;
int qk_llama_memory_bytes(const qk_llama *m, qk_llama_memory *out);
int qk_llama_destroy(qk_llama *m);
/* The reference's INT8 GEMV modes (FastGPU's use_dp4a for Q4_K and
   use_q6_dp4a for Q6_K, inferencer.cu:1159-1166, 1611; both on by default
   there, both off here): enabled types run their GEMVs on per-32 int8
   activations -- RMSNorm and quantization in one launch before QKV, gate/up
   and the LM head (--fused-norm-quant), the attention output quantized
   before o, SiLU * up and its quantization in one launch before down, and
   the residual adds in the o / down GEMVs' epilogues -- and the other types
   stay FP32.  (With both types enabled the driver folds the quantizations
   into the GEMVs and the attention, with the same codes.)  Takes effect at
   the next qk_llama_forward. */
int qk_llama_set_int8(qk_llama *m, int q4k_int8, int q6k_int8);
/* Device pointers to the fp32 caches, [layer][kv_heads][context][head_dim]:
   the drivers keep each KV head's rows contiguous, so the attention
   workgroup of a (token, KV head) streams one run of memory (the reference's
   FastGPU caches are [layer][context][kv_dim]; the Python load_kv and
   cache-row helpers convert). */
int qk_llama_kv_cache(qk_llama *m, float **key_cache, float **value_cache);
/* Device pointer to the fp32 logits of the last step with need_logits. */
int qk_llama_logits(qk_llama *m, const float **logits);
/* Device pointer to the fp32 residual stream x (dim values) after the last
   step: the state --compare-prefill downloads from FastGPU::x
   (inferencer.cu:1744).  Ask again after each step: a greedy INT8 step fed
   the previous step's token swaps in the embedding row that step's final
   pick wrote into a second buffer, so x moves between two buffers, and the
   other one is overwritten by the next pick. */
int qk_llama_residual(qk_llama *m, const float **x);
/* Quantized matrix products the handle has issued since create: seven per
   layer and step (q, k, v, o, gate, up, down) plus one per LM head, the
   count FastGPU::calls keeps for the --stats line "GPU pipeline ... across
   N quantized matrix calls" (inferencer.cu:1170, 1457, 1500, 1909-1910). */
int qk_llama_matrix_calls(const qk_llama *m, uint64_t *calls);
/* The per-layer state --compare-prefill reads (FastRunner::forward's
   layer_trace and quant_trace, inferencer.cu:1424-1531): while set, every
   step copies the residual stream after each layer to residuals
   [layer][dim] and, for the products that run in an INT8 mode, their
   quantized inputs to quantized [layer][4][max(dim, hidden)] -- QKV,
   attention output (o), gate / up, down; the first dim (down: hidden)
   bytes of each slot.  Both are device buffers the caller owns (either may
   be NULL); the copies run on the handle's stream. */
int qk_llama_set_trace(qk_llama *m, float *residuals, int8_t *quantized);
/* One decode step at position pos (FastRunner::forward, inferencer.cu:1424-1531).
   With need_logits, *next_token receives the greedy token (synchronises the
   stream like the reference's 4-byte copy, inferencer.cu:1529); otherwise
   the step stays asynchronous and *next_token is -1. */
int qk_llama_forward(qk_llama *m, int token, int pos, int need_logits, int *next_token);

/* ------------------------------------------- batched decode-step driver -- */

/* A step for a ragged batch of up to max_tokens tokens -- decode tokens of
   different sequences, prefill chunks of consecutive positions of one
   sequence, or any mix (a continuous batch) -- with packed KV caches of
   cache_rows rows per layer ([layer][kv_heads][cache_rows][head_dim], fp32,
   as qk_llama_kv_cache).  The
   multi-sequence counterpart of FastRunner::prefill's batched path
   (inferencer.cu:1279-1423), which serves one sequence; every projection
   runs through qk_gemv_multi_batched_f32 / qk_gemv_batched_f32 (matrix cores
   from 8 tokens on).  Buffers, caches and workspaces are allocated once at
   create; weights are handled as by qk_llama_create (Q6_K copied into the
   split layout, the rest read in place). */
typedef struct qk_llama_batch qk_llama_batch;

int qk_llama_batch_create(const qk_llama_config *cfg, const qk_llama_weights *w, int max_tokens,
                          int64_t cache_rows, qk_stream stream, qk_llama_batch **out);
int qk_llama_batch_destroy(qk_llama_batch *m);
/* The handle's device bytes, as qk_llama_memory_bytes. */
int qk_llama_batch_memory_bytes(const qk_llama_batch *m, qk_llama_memory *out);
/* Device pointers to the fp32 caches, [layer][kv_heads][cache_rows][head_dim]. */
int qk_llama_batch_kv_cache(qk_llama_batch *m, float **key_cache, float **value_cache);
/* Device pointer to the fp32 logits of the last step with need_logits,
   [n_tokens][vocab]. */
int qk_llama_batch_logits(qk_llama_batch *m, const float **logits);
/* Device pointer to the fp32 residual streams after the last step,
   [n_tokens][dim] in the step's token order (inferencer.cu:1744). */
int qk_llama_batch_residual(qk_llama_batch *m, const float **x);
/* Quantized matrix products issued since create: seven per layer and token,
   one per logit row (FastRunner::prefill's counts, inferencer.cu:1277, 1321,
   1368). */
int qk_llama_batch_matrix_calls(const qk_llama_batch *m, uint64_t *calls);
/* qk_llama_set_trace for the batched driver (FastRunner::prefill's
   all_layer_trace and quant_trace, inferencer.cu:1279-1423): per token of
   the step, residuals [token][layer][dim] and, in the INT8 mode, quantized
   [token][layer][4][max(dim, hidden)]; sized for the step's n_tokens. */
int qk_llama_batch_set_trace(qk_llama_batch *m, float *residuals, int8_t *quantized);
/* The reference's INT8 batched arithmetic for the steps that follow
   (FastRunner::prefill with use_dp4a and use_q6_dp4a, inferencer.cu:
   1279-1423; its batched prefill requires both, 1662-1663): per layer
   RMSNorm and per-32 quantization of x, the fused QKV product, attention,
   the attention output quantized, o added into x, RMSNorm and quantization,
   gate / up with SiLU(gate) * up quantized, down added into x; the LM head
   over the RMSNorm of x quantized.  Products run as qk_gemv_multi_batched_i8
   (exact integer sub-block dots).  q4k_int8 and q6k_int8 must be equal
   (QK_ERR_INVALID_ARG otherwise); the first enable allocates the quantized
   activation buffers (QK_ERR_DEVICE when they do not fit). */
int qk_llama_batch_set_int8(qk_llama_batch *m, int q4k_int8, int q6k_int8);
/* One step for n_tokens tokens: tokens[t] (host) at desc[t] (host).  Every
   token writes its key / value row kv_row + pos before any token's
   attention reads the cache, so a token sees the rows of earlier positions
   of its sequence written in the same step (causal within a prefill chunk,
   rope_cache_batch_cuda before attention_batch_cuda, inferencer.cu:953-1041).
   Two tokens writing the same row is QK_ERR_INVALID_ARG.  With need_logits,
   next_tokens[t] (host) receives each token's greedy successor and the call
   synchronises the stream; otherwise it stays asynchronous. */
int qk_llama_batch_forward(qk_llama_batch *m, const int32_t *tokens, const qk_batch_token *desc, int n_tokens,
                           int need_logits, int32_t *next_tokens);
/* The same step with the LM head run only for the n_rows tokens listed in
   logit_rows (host, token indices in [0, n_tokens), any order): logits are
   [n_rows][vocab] in list order and next_tokens[i] (host) is the greedy
   successor of token logit_rows[i].  The reference's prefill computes the
   logits of a chunk's last token only (inferencer.cu:1410-1414); a
   continuous batch needs them for each chunk end and each decode token.
   n_rows = 0 runs no LM head and stays asynchronous. */
int qk_llama_batch_forward_rows(qk_llama_batch *m, const int32_t *tokens, const qk_batch_token *desc, int n_tokens,
                                const int32_t *logit_rows, int n_rows, int32_t *next_tokens);

/* --------------------------------------------------------------- GGUF -- */

/* A GGUF v3 model file, mapped read-only (the reference's GGUF struct,
   inferencer.cu:204-340).  Scalar metadata is kept as doubles, string values
   as strings, tokenizer.ggml.tokens / merges as string arrays; other arrays
   are skipped.  Tensors may be FP32 (0), FP16 (1), Q4_K (12) or Q6_K (14).
   Stricter than the reference: every tensor's offset + bytes must lie inside
   the data section (the reference checks offset < size, inferencer.cu:282),
   offsets must be multiples of general.alignment, and names must be unique;
   each violation is QK_ERR_FORMAT. */
typedef struct qk_gguf qk_gguf;

typedef struct qk_gguf_tensor {
    const char *name;      /* valid until qk_gguf_close */
    int type;              /* 0 FP32, 1 FP16, 12 Q4_K, 14 Q6_K */
    int n_dims;            /* 1..4 */
    int64_t dims[4];       /* dims[0] is contiguous (cols); unused dims are 1 */
    uint64_t offset;       /* from the start of the data section */
    uint64_t bytes;
    const void *host;      /* inside the mapping */
    const void *device;    /* after qk_gguf_upload, else NULL */
} qk_gguf_tensor;

/* QK_ERR_IO if the file cannot be opened or mapped, QK_ERR_FORMAT with the
   reason in qk_last_error() if it is not a valid GGUF v3 file. */
int qk_gguf_open(const char *path, qk_gguf **out);
/* Unmaps the file and frees the device copy. */
int qk_gguf_close(qk_gguf *g);
/* A scalar metadata value (GGUF::param, inferencer.cu:290-294); missing keys
   are QK_ERR_INVALID_ARG. */
int qk_gguf_param(const qk_gguf *g, const char *key, double *value);
/* A string metadata value, or NULL. */
const char *qk_gguf_string(const qk_gguf *g, const char *key);
int64_t qk_gguf_tensor_count(const qk_gguf *g);
/* Tensors in file order. */
int qk_gguf_tensor_at(const qk_gguf *g, int64_t index, qk_gguf_tensor *out);
/* GGUF::tensor (inferencer.cu:317-321); missing names are QK_ERR_INVALID_ARG. */
int qk_gguf_find_tensor(const qk_gguf *g, const char *name, qk_gguf_tensor *out);
/* which = 0: tokenizer.ggml.tokens, 1: tokenizer.ggml.merges. */
int64_t qk_gguf_token_count(const qk_gguf *g, int which);
/* The bytes of entry i (not NUL-terminated; *length receives the size). */
const char *qk_gguf_token(const qk_gguf *g, int which, int64_t i, int64_t *length);
/* The mapped data section, its size and the alignment in effect. */
int qk_gguf_data(const qk_gguf *g, const void **host, uint64_t *bytes, uint64_t *alignment);
/* Copies the data section into one device buffer owned by the handle
   (GGUF::upload, inferencer.cu:322-339: same free-memory margin) and sets
   every tensor's device pointer.  Synchronises the stream. */
int qk_gguf_upload(qk_gguf *g, qk_stream stream);
/* The llama.* hyper-parameters and every tensor of a Llama model by its GGUF
   name (FastRunner's constructor, inferencer.cu:1196-1214, any shape the
   decode drivers support), ready for qk_llama_create: matrices Q4_K or Q6_K
   with dims {cols, rows}, norms FP32 of dims {dim}; output.weight optional
   (tied to token_embd.weight).  llama.vocab_size when present, else the
   embedding's row count.  Requires qk_gguf_upload; layers receives
   cfg.layers entries (at most max_layers); w->layers points at it. */
int qk_gguf_llama(const qk_gguf *g, int context, qk_llama_config *cfg, qk_llama_weights *w,
                  qk_llama_layer *layers, int max_layers);

#ifdef __cplusplus
}
#endif

#endif
