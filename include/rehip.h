/*
 * librehip: MI355X (gfx950) fused GGUF dequant-matmul behind a C ABI.
 *
 * Drop-in for the quantized projection path of platinoff/rusty-engine:
 *   QMat::matvec  src/qmat.rs:80     -> re_qmat_matvec
 *   QMat::matmul  src/qmat.rs:169    -> re_qmat_matmul
 *   QMat::from_bytes / from_model    -> re_qmat_create   (src/qmat.rs:52-59, 312-330)
 *   quant::dequant src/quant.rs:363  -> re_dequant        (bit-exact, quant and float types)
 *   moe expert FFN + combine          -> re_moe_forward    (src/moe.rs:288-300, 360-388)
 *
 * Conventions (from the reference):
 *   - W is m x n row-major; each row is a run of GGUF blocks (kernel.rs:51, 329). GGUF dims
 *     are [n, m] (qmat.rs:310-311).
 *   - X is rows x n row-major f32; Y is rows x m row-major f32, Y[row*m + r] (kernel.rs:1508).
 *   - ggml types: 2 Q4_0, 6 Q5_0, 8 Q8_0, 12 Q4_K, 13 Q5_K, 14 Q6_K (quant.rs:75-88).
 *   - n must be a multiple of 32. When n is not a multiple of the type's block size (the
 *     K-quants at n = 896), each row holds ceil(n/256) whole super-blocks and the elements
 *     past n are ignored.
 *
 * Every entry point returns 0 on success or an RE_ERR_* code; re_last_error() gives the
 * message of the calling thread's last failure. Nothing panics or throws across the ABI.
 * Host-pointer entry points are synchronous and thread-safe (calls on one matrix serialize).
 * Device-pointer entry points (*_dev) enqueue on the caller's HIP stream and return at once;
 * calls on the same matrix object must not overlap in time (they share its split scratch).
 */
#ifndef REHIP_H
#define REHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RE_OK 0
#define RE_ERR_TYPE 1      /* unknown / unsupported ggml type (kernel.rs:2006, 2027 panic) */
#define RE_ERR_SIZE 2      /* byte count or shape mismatch (quant.rs:402-447) */
#define RE_ERR_ARG 3       /* null pointer or invalid argument */
#define RE_ERR_HIP 4       /* HIP runtime failure */
#define RE_ERR_NODEV 5     /* no usable gfx950 device */

#define RE_MODE_BF16 0     /* GEMM: bf16 MFMA, f32 accumulate (|err| <= 1e-2 rel-to-norm) */
#define RE_MODE_F32 1      /* GEMM: f32-accurate mode (|err| <= 2^-10 sum|w*x|): GEMMs run bf16 MFMAs on
                              split operands (hi*hi + hi*lo + lo*hi; two MFMAs for BF16 weights, whose
                              low part is zero); REHIP_GEMM_SP=0 keeps f32 MFMAs above 64 rows */

typedef struct re_qmat re_qmat;
typedef struct re_moe re_moe;

/* Library state. re_init selects the current HIP device; it is called implicitly. */
int re_init(void);
const char *re_last_error(void);
const char *re_version(void);

/* ---- layout (host only; no GPU needed) ------------------------------------------------ */
/* Bytes of one padded GGUF row: ceil(n/QK) * block_bytes (kernel.rs:1983-1993, padded). */
int re_row_bytes(uint32_t ggml_type, size_t n, size_t *out);
/* Size of the GPU-resident tiled layout of an m x n matrix. */
int re_tiled_bytes(uint32_t ggml_type, size_t m, size_t n, size_t *out);
/* Repack GGUF rows into the tiled layout on the host (out holds re_tiled_bytes bytes). */
int re_repack(uint32_t ggml_type, const uint8_t *bytes, size_t nbytes, size_t m, size_t n,
              uint8_t *out, size_t out_len);

/* ---- QMat (src/qmat.rs:30-42) ---------------------------------------------------------- */
/* Upload and repack once. nbytes must equal m * re_row_bytes(type, n). F32 (0), F16 (1) and
 * BF16 (30) bytes are QMat::F32 / the no-fused-kernel arms (qmat.rs:45-49, 128-151): kept
 * row-major, nbytes = m * n * element size; they do not stack. Below 16 activation rows their
 * products are f32 in every mode; from 16 rows (n a multiple of 8) an MFMA GEMM, with bf16
 * operands in bf16 mode and f32 ones in f32 mode. re_qmat_matvec_ex_dev's RMS-norm runs as its own
 * launch into a buffer the matrix owns, and re_ffn_create pairs two dense matrices of one type. */
int re_qmat_create(uint32_t ggml_type, const uint8_t *bytes, size_t nbytes, size_t m, size_t n,
                   re_qmat **out);
/* A stack of `count` same-type, same-shape matrices (nbytes = count * m * row bytes, one after
 * the other, as ExpertWeights holds experts, moe.rs:349-353); every other entry point works on
 * matrix 0, re_qmat_matvec_stacked_dev on any range of them in one launch. */
int re_qmat_create_stacked(uint32_t ggml_type, const uint8_t *bytes, size_t nbytes, size_t m, size_t n,
                           size_t count, re_qmat **out);
size_t re_qmat_count(const re_qmat *q);
void re_qmat_destroy(re_qmat *q);
size_t re_qmat_rows(const re_qmat *q);   /* m (qmat.rs:62-66) */
size_t re_qmat_cols(const re_qmat *q);   /* n (qmat.rs:69-73) */
uint32_t re_qmat_type(const re_qmat *q);

/* y[m] = W x[n] (qmat.rs:80). Host pointers, synchronous. f32 accumulation. */
int re_qmat_matvec(re_qmat *q, const float *x, float *y);
/* Y[rows x m] = X[rows x n] W^T (qmat.rs:169). Host pointers, synchronous. rows == 1 runs
 * the GEMV; otherwise the MFMA GEMM in the given mode. */
int re_qmat_matmul(re_qmat *q, const float *x, size_t rows, float *y, int mode);

/* Device-pointer variants; `stream` is a hipStream_t (NULL = default stream). re_qmat_matmul_dev
 * allocates on first use: up to 32 MiB per matrix for K-split partial tiles and, for the calls of many
 * rows that run on packed bf16 operands, workspaces shared by all matrices of a GPU (at most 4 of
 * 64 .. 512 MiB, ordered between streams by events, freed with the last matrix). Under stream capture, or
 * without memory for a workspace, such calls run the unpacked GEMM: results that differ by the order of
 * the sums. */
int re_qmat_matvec_dev(re_qmat *q, const float *d_x, float *d_y, void *stream);
int re_qmat_matmul_dev(re_qmat *q, const float *d_x, size_t rows, float *d_y, int mode,
                       void *stream);
/* re_qmat_matmul_dev that allocates nothing, for callers that cannot allocate device memory
 * (code under HIP graph capture, serving loops, harnesses that forbid hipMalloc). It has no
 * counterpart in the reference. The GEMM's K-split partial tiles and packed operands go to a static
 * device scratch of 64 MiB per GPU instead of buffers allocated on first use; the same plan, kernels
 * and results as re_qmat_matmul_dev, except where packed operands exceed the scratch: they are then packed
 * and multiplied in pieces (the same results) or, if the pieces would be too small to fill the GPU, the
 * unpacked GEMM runs (results that differ by the order of the sums). A plan whose partials exceed the
 * scratch fails with RE_ERR_SIZE (the planned splits of every shape fit: the planner caps partial tiles
 * at 32 MiB). The scratch is shared by every call on a GPU. Outside stream capture, a call first waits for
 * the launches of the previous call on that GPU (an event set up once per device), so calls from several
 * streams or threads stay ordered. Inside stream capture no ordering is added: replays of captured graphs
 * that use the scratch must not overlap in time. Those are the graphs of quantized calls with K slices;
 * dense weights and single-slice calls are captured as the unpacked GEMM, without the scratch. */
int re_qmat_matmul_noalloc_dev(re_qmat *q, const float *d_x, size_t rows, float *d_y, int mode, void *stream);
/* Dequantize the resident weights to d_out[m x n] f32, bit-exact with quant::dequant. */
int re_qmat_dequant_dev(re_qmat *q, float *d_out, void *stream);

/* Flat-stream dequant on the GPU (quant::dequant, src/quant.rs:363-453) for the six quant
 * types and F32/F16/BF16: out receives nbytes / block_bytes * QK floats (nbytes / element size
 * for the float types). Same length errors as the reference. */
int re_dequant(uint32_t ggml_type, const uint8_t *bytes, size_t nbytes, float *out, size_t out_len);

/* ---- MoE expert FFN (src/moe.rs:288-300, 360-388) ------------------------------------- */
/* Experts stored like a GGUF expert tensor: gate/up are n_experts x inter x hidden, down is
 * n_experts x hidden x inter, each expert's rows as GGUF blocks. */
int re_moe_create(uint32_t gate_type, const uint8_t *gate, size_t gate_bytes,
                  uint32_t up_type, const uint8_t *up, size_t up_bytes,
                  uint32_t down_type, const uint8_t *down, size_t down_bytes,
                  size_t n_experts, size_t hidden, size_t inter, re_moe **out);
void re_moe_destroy(re_moe *e);
/* out[t] = sum_j weights[t*k+j] * down_e(silu(gate_e x_t) * up_e x_t), e = ids[t*k+j], summed
 * in routing order j = 0..k-1 (moe.rs:376-383). Routing comes from the host router
 * (moe.rs:75-125). Host pointers, synchronous. */
int re_moe_forward(re_moe *e, const float *x, size_t tokens, size_t top_k, const uint32_t *ids,
                   const float *weights, float *out, int mode);
/* Device x/out; ids and weights stay on the host (they shape the grouped launch). */
int re_moe_forward_dev(re_moe *e, const float *d_x, size_t tokens, size_t top_k,
                       const uint32_t *ids, const float *weights, float *d_out, int mode,
                       void *stream);
/* Shared expert (moe_layer_forward's `shared`, moe.rs:380-385 and 424-429; combine, moe.rs:339-343):
 * a dense SwiGLU FFN (gate and up inter x hidden, down hidden x inter, each of any type QMat takes)
 * run on every token and added after the routed sum, out[t] = sum_j w_j expert_j(x_t) +
 * down(silu(gate x_t) * up x_t). Once set, every forward call of e adds it (re_moe_forward, _dev,
 * _routed_dev, re_moe_layer_dev). All three pointers NULL removes it. It takes e's lock (held
 * by re_moe_forward) and waits for the device to drain before freeing the previous shared
 * matrices, so forwards queued before the call finish with them; device-pointer forwards that
 * another thread enqueues while it runs are not ordered with it. */
int re_moe_set_shared(re_moe *e, uint32_t gate_type, const uint8_t *gate, size_t gate_bytes,
                      uint32_t up_type, const uint8_t *up, size_t up_bytes,
                      uint32_t down_type, const uint8_t *down, size_t down_bytes, size_t inter);

/* ---- MoE layer with the routing on the device (moe.rs:75-125, 360-388): no host round trip --
 * re_moe_router_logits_dev: logits[t][e] = router_w[e] . x[t] (router_w f32, n_experts x hidden;
 *   the matvec of moe.rs:367).
 * re_moe_route_dev: top_k experts per token (ties to the lower expert index, as the reference's
 *   stable descending sort) and their weights: RE_GATE_SOFTMAX = softmax over the chosen logits
 *   (top_k, moe.rs:75-93), RE_GATE_SIGMOID = per-expert sigmoid renormalised over the chosen
 *   (top_k_sigmoid, moe.rs:98-118). n_experts <= 1024. NaN logits rank as -inf.
 * re_moe_forward_routed_dev: re_moe_forward_dev with device ids/weights (tokens x top_k); the
 *   grouping by expert and the task lists are built by a kernel; tokens * top_k <= 8192. An id
 *   outside [0, n_experts) contributes nothing.
 * re_moe_layer_dev: the three in one stream (scratch for logits/ids/weights is kept by e).
 * re_moe_route_group_dev: the bias-corrected group routers (moe.rs:126-268): scores
 *   sigmoid(logit + bias[e]) (bias entries past bias_len count as 0; d_bias may be NULL with
 *   bias_len 0), experts in n_groups contiguous groups (expert e in group e * ng / n_experts,
 *   ng = n_groups clamped to 1 ..= n_experts), only the top_k_group best groups eligible
 *   (0 = every group), the top_k best eligible experts renormalised over their scores.
 *   RE_GATE_GROUP scores a group by its summed scores (route_group, moe.rs:132-194),
 *   RE_GATE_NOAUX_TC by its two best (route_noaux_tc, moe.rs:196-268, DeepSeek-V3 / Qwen3).
 *   Ties go to the lower group / expert index. When the eligible groups hold fewer than top_k
 *   experts, the remaining slots get id -1 and weight 0 (they contribute nothing downstream).
 * re_moe_layer_group_dev: router logits, group routing and the FFN in one stream. */
#define RE_GATE_SOFTMAX 0
#define RE_GATE_SIGMOID 1
#define RE_GATE_GROUP 2
#define RE_GATE_NOAUX_TC 3
int re_moe_router_logits_dev(const float *d_x, const float *d_router_w, size_t tokens, size_t hidden,
                             size_t n_experts, float *d_logits, void *stream);
int re_moe_route_dev(const float *d_logits, size_t tokens, size_t n_experts, size_t top_k, int gate,
                     int *d_ids, float *d_weights, void *stream);
int re_moe_forward_routed_dev(re_moe *e, const float *d_x, size_t tokens, size_t top_k, const int *d_ids,
                              const float *d_weights, float *d_out, int mode, void *stream);
int re_moe_layer_dev(re_moe *e, const float *d_x, size_t tokens, const float *d_router_w, size_t top_k,
                     int gate, float *d_out, int mode, void *stream);
int re_moe_route_group_dev(const float *d_logits, size_t tokens, size_t n_experts, size_t top_k, int gate,
                           const float *d_bias, size_t bias_len, size_t n_groups, size_t top_k_group,
                           int *d_ids, float *d_weights, void *stream);
int re_moe_layer_group_dev(re_moe *e, const float *d_x, size_t tokens, const float *d_router_w, size_t top_k,
                           int gate, const float *d_bias, size_t bias_len, size_t n_groups,
                           size_t top_k_group, float *d_out, int mode, void *stream);

/* ---- device-resident transformer steps (src/forward.rs, src/infer.rs, src/runner.rs) ------
 * Device pointers, enqueued on `stream`. Positions come from a device int (*d_pos) so that a
 * captured graph serves every decode step; re_pos_add_dev advances it on the stream. */
typedef struct re_ffn re_ffn;

/* y = W norm(x) + add, with the pieces of the transformer block around a projection folded in:
 *   d_norm_w  NULL, or x is RMS-normalised first, x * (1/sqrt(mean(x^2) + eps)) * norm_w
 *             (the attention/FFN/output norms, infer.rs:72-82, forward.rs:432, 479, runner.rs:275);
 *   d_add     NULL, or added to the result (may equal y): the residual adds (forward.rs:472-485);
 *   d_best    NULL, or RE_ARGMAX_SLOTS uint64 slots that keep the maximum of key(y[r], r) over
 *             the rows, the key ordering by value and then by index, so the low 32 bits of the
 *             largest slot end as the greedy token (infer.rs:217-223: the last index among equal
 *             maxima). The slots must start at 0 (re_decode_advance_dev clears them).
 * x and norm_w are 16-byte aligned. */
/* y_b = W_b x_b for the matrices b = first .. first + count - 1 of a stack, in one launch:
 * x_b = d_x + (b - first) * x_stride (x_stride 0: one shared x), y_b = d_y + (b - first) *
 * y_stride. Each result is the GEMV of re_qmat_matvec_dev (qmat.rs:80) up to summation order:
 * the launch shape is planned for the whole stack. */
int re_qmat_matvec_stacked_dev(re_qmat *q, size_t first, size_t count, const float *d_x, size_t x_stride,
                               float *d_y, size_t y_stride, void *stream);
/* Launch shape the GEMV of re_qmat_matvec_dev (count = 1) or of a re_qmat_matvec_stacked_dev call
 * over `count` matrices would use, for tests and profiles (no counterpart in the reference, whose
 * GEMV has one shape): kernel RE_GEMV_TILE (one 64-row tile per workgroup), RE_GEMV_ROWS (row
 * groups of 4/8/16 rows), RE_GEMV_SPLIT (rows split over workgroups + a reduce) or RE_GEMV_DENSE
 * (F32/F16/BF16 weights); waves per workgroup; half = 1 when super-blocks stream half blocks. */
#define RE_GEMV_SPLIT 0
#define RE_GEMV_ROWS 1
#define RE_GEMV_TILE 2
#define RE_GEMV_DENSE 3
int re_qmat_gemv_plan(const re_qmat *q, size_t count, int *kernel, int *rows_per_group, int *waves, int *half);
int re_qmat_matvec_ex_dev(re_qmat *q, const float *d_x, const float *d_norm_w, float eps, const float *d_add,
                          float *d_y, unsigned long long *d_best, void *stream);
/* out[r] = x[r] * (1 / sqrt(mean(x[r]^2) + eps)) * w for rows x d (infer.rs:72-82). */
int re_rmsnorm_dev(const float *d_x, const float *d_w, size_t rows, size_t d, float eps, float *d_out,
                   void *stream);
/* NeoX rotate-half of rows x heads x head_dim in place, row r at position *d_pos + pos_offset + r
 * (infer.rs:90-139, angle = pos * theta^(-2i/head_dim)). */
int re_rope_dev(float *d_x, size_t rows, size_t heads, size_t head_dim, float theta, const int *d_pos,
                int pos_offset, void *stream);
/* Append rows x kv_dim of K and V at cache rows *d_pos + r (the rotated-key cache of
 * forward.rs:347-363). The caches hold max_seq rows; rows that would land at or past max_seq
 * are not stored (the caller keeps *d_pos + rows <= max_seq). */
int re_kv_append_dev(const float *d_k, const float *d_v, size_t rows, size_t kv_dim, float *d_kcache,
                     float *d_vcache, size_t max_seq, const int *d_pos, void *stream);
/* Causal GQA attention of rows x n_heads x head_dim queries at positions *d_pos + r over cache
 * rows 0..position (forward.rs:232-277, 437-470); max_seq <= 32768 cache rows, positions are
 * clamped to them. Output rows x n_heads x head_dim. Rows >= 8 with head_dim 32, 64, 96 or 128 run as
 * f32 MFMA flash attention, except that up to 400, 600 and 900 (row, head) pairs of head_dim 32, 96 and
 * 128, like fewer rows, use d_work (re_attention_work_bytes bytes; NULL = no such exception, and fewer
 * rows run one workgroup per head and row, slower for long caches) to split the cache over workgroups.
 * Buffers are 16-byte aligned. */
size_t re_attention_work_bytes(size_t rows, size_t n_heads, size_t head_dim, size_t max_seq);
int re_attention_dev(const float *d_q, const float *d_kcache, const float *d_vcache, size_t rows,
                     size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t max_seq,
                     const int *d_pos, float *d_work, size_t work_bytes, float *d_ctx, void *stream);
/* NeoX RoPE table (infer.rs:90-139): d_table[(p * head_dim/2 + i) * 2 + {0, 1}] = cos, sin of pair
 * i's angle at position p, for p < rows (rows * head_dim floats), computed exactly as the rotation
 * kernels compute them, so a rotation read from the table has the same bits. head_dim even. */
int re_rope_table_dev(float theta, size_t head_dim, size_t rows, float *d_table, void *stream);
/* One decode row's attention with the q/k/v epilogue folded in (forward.rs:347-363, 437-470):
 * d_q / d_k / d_v are the raw projection outputs of the row (no bias, not rotated); q and k get
 * their biases and NeoX RoPE at *d_pos, v its bias, k and v are appended at cache row *d_pos
 * (not stored at or past max_seq), and attention over rows 0..*d_pos is written to d_ctx
 * (n_heads x head_dim). Same results as re_qkv_rope_append_dev followed by re_attention_dev with
 * rows = 1, in two kernels instead of three. d_rope: NULL, or re_rope_table_dev's table for theta
 * and head_dim with max_seq rows; with it (head_dim % 8 == 0 and q, k, v, biases and table 16-byte
 * aligned) the rotation reads its cosines and sines instead of computing them (same results,
 * shorter critical path). d_work: re_attention_work_bytes(1, ...) bytes. */
int re_attention_decode_dev(const float *d_q, const float *d_k, const float *d_v, const float *d_bq,
                            const float *d_bk, const float *d_bv, size_t n_heads, size_t n_kv_heads,
                            size_t head_dim, float theta, const float *d_rope, const int *d_pos, float *d_kcache,
                            float *d_vcache, size_t max_seq, float *d_work, size_t work_bytes, float *d_ctx,
                            void *stream);
/* The q/k/v projections' epilogue (forward.rs:347-363, 437-449): q = q + bq and k = k + bk
 * rotated (NeoX, as re_rope_dev) at position *d_pos + r, v = v + bv; rotated q written to
 * d_qout (rows x n_heads x head_dim), k and v appended at cache rows *d_pos + r (rows past
 * max_seq are not stored). The three inputs are row-strided (ldq/ldk/ldv floats), so they may
 * be slices of one fused q|k|v projection. Biases may be NULL. */
int re_qkv_rope_append_dev(const float *d_q, size_t ldq, const float *d_k, size_t ldk, const float *d_v,
                           size_t ldv, const float *d_bq, const float *d_bk, const float *d_bv, size_t rows,
                           size_t n_heads, size_t n_kv_heads, size_t head_dim, float theta, const int *d_pos,
                           float *d_qout, float *d_kcache, float *d_vcache, size_t max_seq, void *stream);
/* End of a greedy step (runner.rs:262-282): *d_tok = the token in the largest of the
 * RE_ARGMAX_SLOTS slots at d_best (low 32 bits), *d_pos += delta, d_hist[*d_pos] = *d_tok when
 * d_hist is given and *d_pos < hist_len, and the slots cleared for the next step. */
#define RE_ARGMAX_SLOTS 8
int re_decode_advance_dev(unsigned long long *d_best, int *d_tok, int *d_pos, int delta, int *d_hist,
                          size_t hist_len, void *stream);
/* out[i] = a[i] + b[i % nb] (residual add for nb == n, per-column bias for nb | n). */
int re_add_dev(const float *d_a, const float *d_b, size_t n, size_t nb, float *d_out, void *stream);
/* h = silu(g) * u elementwise (moe.rs:44-51, 280-283). */
int re_swiglu_dev(const float *d_g, const float *d_u, float *d_h, size_t n, void *stream);
/* *d_idx = index of the largest of n values; the last one among equal maxima (infer.rs:217-223). */
int re_argmax_dev(const float *d_x, size_t n, int *d_idx, void *stream);
/* out[r] = table[tok[r]] for rows tokens of an n_vocab x d f32 table (runner.rs:105-122); a token
 * outside [0, n_vocab) gives a zero row (the host checks prompt ids before upload). */
int re_embed_dev(const float *d_table, size_t n_vocab, size_t d, const int *d_tok, size_t rows, float *d_out,
                 void *stream);
/* *d_pos += delta on the stream. */
int re_pos_add_dev(int *d_pos, int delta, void *stream);
/* A gate/up pair (same type and shape, inter x hidden) read side by side for one activation row:
 * h = silu(gate x) * (up x) in one launch (the SwiGLU FFN input, forward.rs:100-105). Dense
 * (F32/F16/BF16) pairs run the norm, the two products and SwiGLU as four launches through a buffer
 * the pair owns. The pair keeps references to the two matrices, which must outlive it. */
int re_ffn_create(re_qmat *gate, re_qmat *up, re_ffn **out);
void re_ffn_destroy(re_ffn *f);
/* d_norm_w: NULL, or x is RMS-normalised first (the FFN norm, forward.rs:479). */
int re_ffn_forward_dev(re_ffn *f, const float *d_x, const float *d_norm_w, float eps, float *d_h, void *stream);
/* A whole FFN over several rows (prefill): y = add + down(silu(gate x) * up x), x `rows` rows of gate's
 * columns (already normalised), add NULL or `rows` rows of down's rows (may be y: the residual). The
 * results of the two products, SwiGLU, the down product and the addition as calls of their own; from a
 * few hundred rows of quantized weights the products and SwiGLU are one GEMM. d_work: at least
 * re_ffn_block_work_bytes(f, down, rows) bytes of device memory. */
size_t re_ffn_block_work_bytes(const re_ffn *f, const re_qmat *down, size_t rows);
int re_ffn_block_dev(re_ffn *f, re_qmat *down, const float *d_x, size_t rows, const float *d_add, float *d_y,
                     float *d_work, size_t work_bytes, int mode, void *stream);

/* ---- batched serving over a paged int8 K/V cache ------------------------------------------
 * No counterpart on the reference's forward path, which holds one sequence's f32 K and V
 * (forward.rs:347-363); the reference's own page table over requests is infer.rs:328-527. Device
 * pointers, enqueued on `stream`; nothing is allocated and no value is read back, so every call may
 * be captured into a graph (with buffers of its own, or replayed one after the other). The stream's
 * device is the current one, and all buffers are on it.
 *
 * A ragged batch: request b's rows are row_start[b] .. row_start[b] + row_count[b] - 1 of the row
 * arrays (q, k, v, ctx, positions), ranges ascending and disjoint, row_start[b + 1] >= row_start[b] +
 * row_count[b]; rows between and behind them are left as they were. kv_len[b] counts the request's
 * tokens, its new rows included: row i stands at position kv_len[b] - row_count[b] + i. Token t of
 * it lies in page d_table[b * table_ld + t / page] at place t % page; an entry outside 0 .. n_pages - 1
 * holds no page, nor does what is behind the table's columns. A request's pages are distinct, and a page
 * that is being appended to belongs to one request; full pages may be shared.
 *
 * The cache: d_kcodes and d_vcodes hold n_pages x n_kv_heads x page x head_dim int8 codes (page and
 * head_dim multiples of 32 up to 256; 16-byte aligned), d_kscale and d_vscale n_pages x n_kv_heads f32
 * scales; a code c stands for c * scale. The codes of one page and head are blocks of 32 tokens x 32
 * dimensions, 1 KiB each, [page / 32][head_dim / 32], with token t and dimension d of a block at byte
 *   K: 256 (d / 8) + 16 (t % 16) + 8 (t / 16) + d % 8
 *   V: 256 (t / 4 % 4) + 16 (d % 16) + 8 (d / 16) + 4 (t / 16) + t % 4
 * (the order in which a wave's lanes hold matrix operands). A page needs no preparation; scales that are
 * written by other means are finite and not negative. */

/* The plan of a step from the requests' lengths. Request b holds d_kv_len[b] tokens and brings
 * d_new_len[b] more (0: none this time; up to 262144); a negative number ends it: its pages go back to
 * the pool, request after request, and its length becomes 0 (so not a request that shares pages). d_free
 * is a stack of free pages, n_pages entries of which the first *d_n_free are set; the step's new pages are
 * taken from its top in request order and written to d_table (other entries are left). A request whose pages, with those of the requests
 * before it, exceed the free ones, or whose tokens exceed table_ld * page, is refused: row_count 0,
 * length and pages unchanged. Outputs: d_kv_len_out and d_n_free_out (may be d_kv_len and d_n_free);
 * d_row_start (rows packed in request order, refused ones included, as the caller packed them from
 * new_len) and d_row_count; for rows 0 .. row_cap - 1 the request, the position and the slot
 * (page * page size + place), -1 for rows of refused requests and behind the last; d_status[0] refused
 * requests, d_status[1] rows. Up to 4096 requests, requests * table_ld up to 2^30. */
int re_kv_plan_dev(size_t requests, size_t page, const int *d_new_len, const int *d_kv_len, int *d_table,
                   size_t table_ld, int *d_free, size_t n_pages, const int *d_n_free, int *d_kv_len_out,
                   int *d_n_free_out, int *d_row_start, int *d_row_count, size_t row_cap, int *d_row_seq,
                   int *d_row_pos, int *d_row_slot, int *d_status, void *stream);

/* Rotary frequencies on the host: freqs[i] radians per position of pair i < rot_dim / 2, theta^(-2i/rot_dim)
 * scaled for contexts longer than the trained ones, and the factor of the rotated vectors in *mscale
 * (1 except for RE_ROPE_YARN):
 *   RE_ROPE_LINEAR  all divided by factor;
 *   RE_ROPE_NTK     theta * factor^(d / (d - 2)) in theta's place, d = rot_dim;
 *   RE_ROPE_YARN    pairs from the one that makes p0 turns over trained_len positions (fast, e.g. 32)
 *                   to the one that makes p1 (slow, e.g. 1) move from theirs to theirs / factor along a
 *                   ramp; mscale = 0.1 ln(factor) + 1;
 *   RE_ROPE_BANDS   pairs of up to p0 turns over trained_len are divided by factor, of p1 or more kept,
 *                   between them mixed linearly in the number of turns (p0 < p1, e.g. 1 and 4). */
#define RE_ROPE_NONE 0
#define RE_ROPE_LINEAR 1
#define RE_ROPE_NTK 2
#define RE_ROPE_YARN 3
#define RE_ROPE_BANDS 4
int re_rope_freqs(double theta, size_t rot_dim, int scaling, double factor, double trained_len, double p0, double p1,
                  double *freqs, float *mscale);
/* Rotary positions of rows x heads x head_dim (row strides ldx and ldo floats): the first rot_dim
 * dimensions of each head of row r turn by d_pos[r] * d_freqs[i] (angles in 64 bits, so far positions
 * keep theirs) and are scaled by mscale, pair i being (x[i], x[i + rot_dim / 2]) (RE_ROPE_HALF, as
 * infer.rs:90-139) or (x[2i], x[2i + 1]) (RE_ROPE_INTERLEAVED); the other dimensions are copied. d_out
 * may be d_x (with ldo = ldx), and then holds q and k of a fused projection rotated in one call; other
 * overlaps are not allowed. Rows at negative positions are left as they were. d_freqs: rot_dim / 2 doubles. */
#define RE_ROPE_HALF 0
#define RE_ROPE_INTERLEAVED 1
int re_rope_rows_dev(const float *d_x, size_t ldx, size_t rows, size_t heads, size_t head_dim, size_t rot_dim,
                     int layout, const double *d_freqs, float mscale, const int *d_pos, float *d_out, size_t ldo,
                     void *stream);

/* Append the batch's K and V rows (strides ldk, ldv floats, multiples of 4 up to 2^22; 16-byte aligned) to the cache.
 * A page and head's scale is the largest finite magnitude of what it holds / 127 (0 where that is below the
 * smallest normal float), a code round(x / scale), ties to even; +-inf are stored as +-127 and NaN as 0.
 * Rows that raise the scale of a page with earlier rows of the request in it round those rows' codes
 * to the new one, round(c * (old / new)); a page that the new rows begin starts a scale of its own. A
 * request's kv_len may have been set back before: the codes behind it are overwritten, the scale of a
 * page that keeps rows is kept. Requests with kv_len < row_count or beyond the table are skipped. */
int re_kv8_append_dev(const float *d_k, size_t ldk, const float *d_v, size_t ldv, size_t rows, size_t requests,
                      const int *d_row_start, const int *d_row_count, const int *d_kv_len, const int *d_table,
                      size_t table_ld, size_t page, size_t n_pages, int8_t *d_kcodes, int8_t *d_vcodes,
                      float *d_kscale, float *d_vscale, size_t n_kv_heads, size_t head_dim, void *stream);

/* Causal GQA attention of the batch's q rows (stride ldq floats, a multiple of 4; after their k and v are
 * appended): row at position p sees the tokens max(0, p - window + 1) .. p (window 0: all up to p) that lie
 * in a page, ctx = softmax(scale * q . k) v, rows x n_heads x head_dim; a row that sees nothing gets zeros.
 * Products and sums are f32-accurate (the codes are exact in f16; q and the probabilities are split into two
 * f16 parts of 22 bits). max_rows: no request has more rows (rows past it are left). max_len: the largest
 * kv_len to plan for (longer ones are computed too, only slower). d_work: re_attention_kv8_work_bytes bytes,
 * 16-byte aligned (NULL where that is 0); calls that may run at the same time, replays of captured graphs
 * among them, each need their own. */
size_t re_attention_kv8_work_bytes(size_t rows, size_t requests, size_t max_rows, size_t max_len, size_t n_heads,
                                   size_t n_kv_heads, size_t head_dim);
int re_attention_kv8_dev(const float *d_q, size_t ldq, size_t rows, size_t requests, const int *d_row_start,
                         const int *d_row_count, const int *d_kv_len, const int *d_table, size_t table_ld, size_t page,
                         size_t n_pages, const int8_t *d_kcodes, const int8_t *d_vcodes, const float *d_kscale,
                         const float *d_vscale, size_t max_rows, size_t max_len, size_t n_heads, size_t n_kv_heads,
                         size_t head_dim, float scale, size_t window, float *d_ctx, void *d_work, size_t work_bytes,
                         void *stream);

/* The same with a few first tokens that stay visible behind the window: row at position p sees the tokens t <= p with
 * t > p - window or t < sinks (up to 1024; of no effect with window 0). A row costs window + sinks tokens however long its
 * request is; pages that no row sees any more are not read. d_lse: NULL, or rows x n_heads, the natural logarithm of each
 * row and head's sum of exp(scale * q . k) (-inf where it sees nothing). The workspace is re_attention_kv8_work_bytes' too. */
int re_attention_kv8_sinks_dev(const float *d_q, size_t ldq, size_t rows, size_t requests, const int *d_row_start,
                               const int *d_row_count, const int *d_kv_len, const int *d_table, size_t table_ld,
                               size_t page, size_t n_pages, const int8_t *d_kcodes, const int8_t *d_vcodes,
                               const float *d_kscale, const float *d_vscale, size_t max_rows, size_t max_len,
                               size_t n_heads, size_t n_kv_heads, size_t head_dim, float scale, size_t window,
                               size_t sinks, float *d_ctx, float *d_lse, void *d_work, size_t work_bytes, void *stream);

/* The weight that a step's attention gives each cached token, added to what it has: d_mass holds n_pages x n_kv_heads x
 * page f32, d_mass[page][head][place] += the sum over the request's rows that see the token and over the query heads of that
 * KV head of exp(scale * q . k - lse), with the q, window and sinks of the attention call and the d_lse that it gave. A
 * token that the step brought starts from 0, so pages need no preparation. A row whose q or lse is not finite adds
 * nothing. Every row of the batch adds its weights: made right behind attention, before drafts are verified, those of drafts that are
 * rejected stay in the masses of the tokens before them, and eviction ranks by them. To count only the rows that stay, keep each
 * layer's q and lse and make the call behind re_kv_rewind_dev and before re_kv_evict_plan_dev, with row_count - back in row_count's
 * place and the lengths that the rewind left: rows then have the positions that they had. Accurate to about 2^-23 |lse| of a weight. Here a page belongs to one request. No workspace; d_q and d_mass
 * 16-byte aligned. */
int re_kv8_mass_dev(const float *d_q, size_t ldq, const float *d_lse, size_t rows, size_t requests,
                    const int *d_row_start, const int *d_row_count, const int *d_kv_len, const int *d_table,
                    size_t table_ld, size_t page, size_t n_pages, const int8_t *d_kcodes, const float *d_kscale,
                    size_t max_rows, size_t max_len, size_t n_heads, size_t n_kv_heads, size_t head_dim, float scale,
                    size_t window, size_t sinks, float *d_mass, void *stream);

/* Eviction: requests that hold more than `limit` tokens are cut to `keep` (1 .. limit) of them, in fresh pages, so that one
 * plan serves the caches of all layers. re_kv_evict_plan_dev, once a step: each cut request, in request order, takes
 * ceil(keep / page) pages from the top of the stack and then gives its old ones back (behind the free ones, entries that
 * hold no page left out); one whose new pages are not there is left as it is. Outputs: lengths, table, stack and its height
 * (d_kv_len_out, d_table_out, d_free_out, d_n_free_out may be the inputs; entries of d_table_out behind a cut request's
 * pages are -1); d_from_len: a cut request's old length, 0 for the others; d_from_table (requests x table_ld): a cut
 * request's old entries (may be d_table if d_table_out is another buffer; never d_table_out); d_dropped: NULL, or per
 * request += the tokens it lost, 0 where it holds none (re_kv_positions_dev adds them to its rows' positions; a request number that
 * passes to another conversation with no such call between keeps the old one's, and is set to 0 by the caller);
 * d_status[0] requests over the limit that were left, d_status[1] cut ones. d_from_len is neither of the lengths' buffers. Not
 * for requests that share pages: a cut one gives all of its pages back. Up to 4096 requests.
 *
 * re_kv8_evict_dev, for each layer: of a cut request's tokens the first `first`, the last `recent` and the heaviest of
 * those between them stay, `keep` in all, KV head by KV head (ties to the earlier token; a NaN counts as -inf, a token
 * without a page below that), and move to the new pages in their order, K, V and mass. A new page's scale is the largest of
 * the pages that its tokens come from, a code round(c * (old / new)), ties to even; places behind the last token get code
 * and mass 0. d_kept: requests x n_kv_heads x keep, the old places of what stayed (of cut requests). d_mass (16-byte
 * aligned) may be NULL if first + recent = keep. Old pages are only read: they must not be given out before the last layer's call. max_len: the
 * largest d_from_len to plan for (longer ones are computed too, only slower). */
int re_kv_evict_plan_dev(size_t requests, size_t page, size_t limit, size_t keep, const int *d_kv_len,
                         const int *d_table, size_t table_ld, const int *d_free, size_t n_pages, const int *d_n_free,
                         int *d_kv_len_out, int *d_table_out, int *d_free_out, int *d_n_free_out, int *d_from_len,
                         int *d_from_table, int *d_dropped, int *d_status, void *stream);
int re_kv8_evict_dev(size_t requests, const int *d_from_len, const int *d_from_table, const int *d_table,
                     size_t table_ld, size_t page, size_t n_pages, int8_t *d_kcodes, int8_t *d_vcodes, float *d_kscale,
                     float *d_vscale, float *d_mass, size_t n_kv_heads, size_t head_dim, size_t keep, size_t first,
                     size_t recent, size_t max_len, int *d_kept, void *stream);

/* Rotary positions of a step's rows after evictions: d_out[r] = d_row_pos[r] + d_dropped[d_row_seq[r]], -1 for rows without a
 * request (of the plan's d_row_seq and d_row_pos, which count what the cache holds). d_out may be d_row_pos. Positions go on with
 * the conversation, and tokens that stay keep the rotation of theirs: what an eviction bounds is memory, not the range of
 * positions, so a conversation longer than the trained one needs frequencies scaled for it (re_rope_freqs). */
int re_kv_positions_dev(size_t rows, const int *d_row_seq, const int *d_row_pos, size_t requests, const int *d_dropped,
                        int *d_out, void *stream);

/* Drafted tokens against the target's probabilities. Request b has d_row_count[b] rows of logits from d_row_start[b] on
 * (ranges ascending and disjoint, as above; 0: none): row i is the target's after token d_tokens[row i], d_tokens[row i + 1] the
 * token drafted there, and the last row has no draft behind it, so that a request of one row just draws a token. p =
 * softmax(logits / T), T = d_temperature[b] (NULL: 1). d_probs (stride ldp), or NULL: the distributions q that the drafts were
 * drawn from, row by row; finite, not negative. Of d_probs and d_accept_u a request's last row is not read, of d_tokens its first:
 * buffers may end before them. A draft d is accepted if d_accept_u[row] * q(d) < p(d) (without d_probs:
 * q(d) = 1). In the place of the first that is not, a token is drawn from max(0, p - q) over its sum (without d_probs: from
 * p without d; where nothing is left, from p), behind the last from p. Drawn: the lowest token t with sum over j <= t
 * of the weights > d_sample_u[b] * their sum; both random numbers from [0, 1). T <= 0 or NaN: greedy, a draft is accepted
 * if it is the largest logit (ties to the lower id), and the token behind is the largest. Exponentials are good to
 * 3.6e-11 of their value and sums are taken in 64 bits: a random number that close to a token's border may draw its neighbour. A
 * draft outside 0 .. vocab - 1 is not accepted. A row with NaN or +inf among its logits, or nothing above -inf, has no
 * distribution: its draft is not accepted, and the token in its place is -1. Outputs: d_accepted[b] drafts, d_back[b] = the
 * others (for re_kv_rewind_dev), d_out_tokens[row i]: the accepted drafts, the token behind them, -1 after that; rows
 * outside the requests' are left. The outputs are buffers of their own (d_out_tokens over d_tokens is refused).
 * d_work: re_draft_verify_work_bytes bytes (never fewer for more rows, requests or tokens: the largest step's serve all), 16-byte
 * aligned; as above. */
size_t re_draft_verify_work_bytes(size_t rows, size_t requests, size_t vocab);
int re_draft_verify_dev(const float *d_logits, size_t ld, size_t rows, size_t vocab, size_t requests,
                        const int *d_row_start, const int *d_row_count, const int *d_tokens, const float *d_probs,
                        size_t ldp, const float *d_temperature, const float *d_accept_u, const float *d_sample_u,
                        int *d_accepted, int *d_back, int *d_out_tokens, void *d_work, size_t work_bytes, void *stream);

/* Takes d_back[b] tokens (negative: none; more than there are: all) off the ends of the requests' lengths; pages that hold
 * none of the rest go back to the stack, behind the free ones in request order. d_kv_len_out and d_n_free_out may be
 * d_kv_len and d_n_free; the table is left. Lengths outside 0 .. table_ld * page stay. Such pages belong to one request. A
 * part-filled page keeps the scale that the tokens behind had raised, and the tokens that are left keep the weights that
 * the rows taken back had added to their masses (re_kv8_mass_dev says how to leave those out). Up to 4096 requests. */
int re_kv_rewind_dev(size_t requests, size_t page, const int *d_back, const int *d_kv_len, const int *d_table,
                     size_t table_ld, int *d_free, size_t n_pages, const int *d_n_free, int *d_kv_len_out,
                     int *d_n_free_out, void *stream);

/* Of rows x vocab logits (row stride ld): d_logprob[r] = log softmax of logit d_targets[r] (a target outside
 * 0 .. vocab - 1: 0, so that a sum over rows skips it), d_entropy[r] in nats, and the top_k (up to 64)
 * largest logits' ids and log probabilities in descending order, ties to the lower id; rows x top_k. d_logprob
 * (with d_targets) and d_entropy may be NULL, top_k 0. A logit of -inf has probability 0 and adds nothing to the
 * entropy. A row with NaN or +inf among its logits, or with nothing above -inf, has no distribution: its log
 * probabilities and entropy are NaN; ids rank NaN as -inf. d_work: re_logprobs_work_bytes bytes, as above. */
size_t re_logprobs_work_bytes(size_t rows, size_t vocab, size_t top_k);
int re_logprobs_dev(const float *d_logits, size_t ld, size_t rows, size_t vocab, const int *d_targets, size_t top_k,
                    float *d_logprob, float *d_entropy, int *d_top_ids, float *d_top_logprobs, void *d_work,
                    size_t work_bytes, void *stream);

/* ---- int8 activations (src/kernel.rs:70-166) ------------------------------------------
 * re_quantize_q8_act[_dev]: Q8Activation::from_f32 (kernel.rs:88-105) of `rows` activation rows
 * of n values (n a multiple of 32): scales rows x n/32 f32 (d = max|x|/127 per block) and qs
 * rows x n i8 (round half away from zero of x/d, clamped to [-127, 127]), each row laid out like
 * one Q8Activation. The _dev form needs x and qs 16-byte aligned. Bit-identical to the reference.
 * re_qmat_matmul_i8[_dev]: matvec_q8_0_i8 / matmul_q8_0_i8 (kernel.rs:145-166) of a Q8_0 QMat
 * against such rows: y (rows x m) = per block the exact i32 dot of weight and activation i8,
 * folded as s += ((f32)isum * dw) * dx in block order; bit-identical to dot_q8_0_i8
 * (kernel.rs:123-142). RE_ERR_TYPE for a matrix that is not Q8_0. */
int re_quantize_q8_act(const float *x, size_t rows, size_t n, float *scales, int8_t *qs);
int re_quantize_q8_act_dev(const float *d_x, size_t rows, size_t n, float *d_scales, int8_t *d_qs, void *stream);
int re_qmat_matmul_i8(re_qmat *q, const float *scales, const int8_t *qs, size_t rows, float *y);
int re_qmat_matmul_i8_dev(re_qmat *q, const float *d_scales, const int8_t *d_qs, size_t rows, float *d_y,
                          void *stream);

/* ---- GGUF model files (src/gguf.rs:17-392, src/loader.rs:17-130) ----
 * re_gguf_open maps the file read-only and parses its header: magic "GGUF", version 2 (u32
 * counts) or 3 (u64 counts), metadata of every value kind (nested arrays included), up to 8 dims
 * per tensor, data start = header end rounded up to general.alignment (U32 or U64; default 32).
 * Parse failures return RE_ERR_ARG with "gguf parse error at <offset>: <message>" (gguf.rs:60-70).
 * Strings and tensor data returned below point into the mapping and live until re_gguf_close. */
typedef struct re_gguf re_gguf;
int re_gguf_open(const char *path, re_gguf **out);               /* MmapModel::open (loader.rs:30-50) */
void re_gguf_close(re_gguf *g);
uint32_t re_gguf_version(const re_gguf *g);
size_t re_gguf_kv_count(const re_gguf *g);
size_t re_gguf_tensor_count(const re_gguf *g);
uint64_t re_gguf_alignment(const re_gguf *g);                  /* GgufFile::alignment (gguf.rs:143-150) */
size_t re_gguf_data_offset(const re_gguf *g);                  /* header end, before alignment */
size_t re_gguf_data_start(const re_gguf *g);                   /* aligned_start (loader.rs:17-21) */
/* i-th metadata key (NUL-terminated copy) and its value kind (0 U8 .. 12 F64, gguf.rs:274-312). */
int re_gguf_kv(const re_gguf *g, size_t i, const char **key, uint32_t *kind);
/* First value under `key` (gguf.rs:139-141): integers and Bool widened to int64, F32/F64 to
 * double, strings as (pointer, length) without a NUL, arrays as element kind and count. */
int re_gguf_get_int(const re_gguf *g, const char *key, int64_t *v);
int re_gguf_get_float(const re_gguf *g, const char *key, double *v);
int re_gguf_get_str(const re_gguf *g, const char *key, const char **s, size_t *len);
int re_gguf_get_array(const re_gguf *g, const char *key, uint32_t *elem_kind, uint64_t *count);
/* Tensor i: name, ggml type, dims (dims[0..7], zero past n_dims) and byte offset past data start. */
int re_gguf_tensor_info(const re_gguf *g, size_t i, const char **name, uint32_t *type, uint32_t *n_dims,
                        uint64_t *dims, uint64_t *offset);
int re_gguf_find_tensor(const re_gguf *g, const char *name, size_t *index);
/* MmapModel::tensor_bytes (loader.rs:95-101): [data_start + offset, + nbytes) of the mapping,
 * nbytes from the type and element count (quant.rs:75-101); RE_ERR_TYPE for an unsized type or
 * a count that is not whole blocks, RE_ERR_SIZE when the range leaves the file. */
int re_gguf_tensor_data(const re_gguf *g, size_t i, const uint8_t **data, size_t *nbytes);
/* QMat::from_model (qmat.rs:310-330): W[m x n] from the tensor with dims [n, m] (or [n, m, count]:
 * a stacked QMat of count matrices). The mapped bytes are copied to the device unchanged and
 * repacked there. Errors: "QMat: tensor '<name>' missing" / "... bytes out of bounds". */
int re_qmat_from_gguf(const re_gguf *g, const char *name, size_t m, size_t n, re_qmat **out);
/* One MoE layer's stacked experts (model.rs:372-389): gate and up tensors with dims
 * [hidden, inter, n_experts], down with [inter, hidden, n_experts]. */
int re_moe_from_gguf(const re_gguf *g, const char *gate, const char *up, const char *down, size_t n_experts,
                     size_t hidden, size_t inter, re_moe **out);

#ifdef __cplusplus
}
#endif
#endif /* REHIP_H */
