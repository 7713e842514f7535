/*
 * tkmi.h -- C ABI of libtkmi.so, the MI355X (gfx950) kernels of the
 * transformer-layer forward path.
 *
 * Conventions
 *   - Every entry point is extern "C", returns int: 0 on success, a negative
 *     TK_ERR_* code on a rejected argument, or TK_ERR_HIP when the HIP runtime
 *     reported an error at launch.  tk_last_error_string() describes the last
 *     failure on the calling thread.
 *   - All buffers are DEVICE pointers owned by the caller (the Python side
 *     allocates them with torch.empty).  No entry point allocates device or
 *     host memory, none synchronizes; each enqueues on `stream` (a
 *     hipStream_t passed as void*; NULL = the legacy default stream).
 *   - tk_half is IEEE binary16 storage.  Row-major layouts; leading
 *     dimensions (ld*) and strides are in ELEMENTS.
 *
 * The reference (danielfodgaard/transformer-kernel) exposes this path as
 * Python functions on torch tensors; each entry point below names the
 * reference interface it replaces (paths relative to the reference repo).
 */
#ifndef TKMI_H
#define TKMI_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TKMI_ABI_VERSION 7

typedef uint16_t tk_half;

enum tk_status {
  TK_OK = 0,
  TK_ERR_ARG = -1,         /* null pointer, bad size, bad stride, bad enum */
  TK_ERR_UNSUPPORTED = -2, /* valid request outside the kernels' envelope  */
  TK_ERR_HIP = -3          /* the HIP runtime rejected the launch          */
};

enum tk_dtype { TK_F32 = 0, TK_F16 = 1, TK_BF16 = 2 /* the serving calls at the end only */ };

/*
 * Padding masks.  `row_valid` arguments are nullable [rows] byte arrays
 * (nonzero = valid token; a torch bool tensor's storage); NULL means every
 * row is valid and the kernels take their unmasked path.  The row modes give
 * what an invalid row of a residual update becomes, following the baseline
 * block (src/torch_transformer_benchmark.py:119-120,141-142,170-171):
 */
enum tk_row_mode {
  TK_ROWS_KEEP_RESID = 1, /* s = resid: the attention output of a padded row is 0 */
  TK_ROWS_ZERO = 2,       /* s = 0: the block output of a padded row is 0           */
  TK_ROWS_ZERO_ALL = 3    /* s = 0 and the normalised output h = 0 (final norm)     */
};

enum tk_epilogue {
  TK_EPI_BIAS = 0,      /* C(f16)  = A.W^T + bias                          */
  TK_EPI_BIAS_GELU = 1, /* C(f16)  = gelu_erf(A.W^T + bias)                */
  TK_EPI_BIAS_RESID = 2 /* C(f32)  = resid + (A.W^T + bias); C may alias resid */
};

/* ABI version (TKMI_ABI_VERSION) of the loaded library. */
int tk_version(void);

/* Message for the last non-zero status returned on this thread ("" if none). */
const char *tk_last_error_string(void);

/*
 * LayerNorm over the last dim + cast.
 *   out[r, :] = (x[r,:] - mean) * rsqrt(var_pop + eps) * w + b   (fp32 math)
 * x: [rows, cols] f32 contiguous; w, b: [cols] f32; out: [rows, cols] of
 * out_dtype (TK_F16 or TK_F32).  cols in [1, 8192].  row_valid (nullable):
 * rows marked invalid are written as zeros (the final norm of a padded row,
 * src/torch_transformer_benchmark.py:170-171).
 * Replaces fused_kernels.ln_fwd / _ln_kernel (src/fused_kernels.py:164-193,
 * :80-112).
 */
int tk_ln_cast(const float *x, const float *w, const float *b, void *out,
               int out_dtype, int64_t rows, int64_t cols, float eps,
               const uint8_t *row_valid, void *stream);

/*
 * Residual add + LayerNorm + cast.
 *   s = x + y (added in fp32);  h = LN(s) (statistics of the fp32 sum) cast
 *   to h_dtype;  s stored in x's dtype.
 * x has x_dtype and y has y_dtype (TK_F16 or TK_F32 each); sum_out, when not
 * NULL, is [rows, cols] of x_dtype and may alias x (NULL: s not stored).
 * cols in [1, 8192].
 * Replaces fused_kernels.add_ln_fwd / _add_ln_kernel
 * (src/fused_kernels.py:196-238, :114-161; s = empty_like(x) at :216).
 */
int tk_add_ln_cast(const void *x, int x_dtype, const void *y, int y_dtype,
                   const float *w, const float *b, void *sum_out, void *h_out,
                   int h_dtype, int64_t rows, int64_t cols, float eps,
                   void *stream);

/*
 * GEMM  C[m, n] = epilogue( sum_k A[m, k] * W[n, k] + bias[n] )
 * A: [m, k] f16 (lda), W: [n, k] f16 (ldw) -- the nn.Linear weight layout,
 * bias: [n] f32 (may be NULL = 0), fp32 accumulation on MFMA.
 * epilogue TK_EPI_BIAS / TK_EPI_BIAS_GELU: C is f16 (ldc).
 * epilogue TK_EPI_BIAS_RESID: C is f32 (ldc), resid is f32 (ldr), C may
 * equal resid (in-place residual stream update).
 * Any k >= 0 with lda, ldw >= k; A and W 2-byte aligned.  When k, lda and
 * ldw are multiples of 8 and A, W 16-byte aligned the operands are read in
 * 16-byte vectors (the fast path); otherwise by element (odd d_model /
 * ffn_dim, which the reference's config validation accepts).
 * row_valid / row_mode (TK_EPI_BIAS_RESID only; row_valid nullable, m bytes):
 * an invalid row m is written as resid (TK_ROWS_KEEP_RESID) or 0
 * (TK_ROWS_ZERO, TK_ROWS_ZERO_ALL).
 * Replaces torch F.linear (+ F.gelu) in src/optimized.py:572,627,632-636.
 */
int tk_gemm(const tk_half *a, int64_t lda, const tk_half *w, int64_t ldw,
            const float *bias, const float *resid, int64_t ldr, void *c,
            int64_t ldc, int64_t m, int64_t n, int64_t k, int epilogue,
            const uint8_t *row_valid, int row_mode, void *stream);

/*
 * GEMM, residual add, LayerNorm and cast:
 *   s = resid + A.W^T + bias (fp32);  h = LN(s; ln_w, ln_b, eps) -> h_dtype
 * sum_out (may be NULL, may alias resid) receives s.  Given, it is the
 * residual GEMM's output and a LayerNorm launch reads it; NULL, one kernel
 * keeps whole rows on chip, so n must fit one tile: n in {128, 256, 512}
 * (tk_gemm_ln_supported) in both cases.
 * row_valid (nullable, m bytes) / row_mode: an invalid row takes s per
 * row_mode (tk_row_mode); h = LN(s), or 0 under TK_ROWS_ZERO_ALL.
 * Replaces F.linear followed by fused_kernels.add_ln_fwd
 * (src/optimized.py:523-553 with :627 / :636).
 */
int tk_gemm_bias_add_ln(const tk_half *a, int64_t lda, const tk_half *w,
                        int64_t ldw, const float *bias, const float *resid,
                        const float *ln_w, const float *ln_b, float *sum_out,
                        void *h_out, int h_dtype, int64_t m, int64_t n,
                        int64_t k, float eps, const uint8_t *row_valid,
                        int row_mode, void *stream);

/* 1 when tk_gemm_bias_add_ln handles rows of n elements, else 0. */
int tk_gemm_ln_supported(int64_t n);

/*
 * tk_gemm and tk_gemm_bias_add_ln with one order of sums for every m: an output
 * row's bits do not depend on how many others the call has.  (Those two split
 * the k sums of launches that would leave most of the chip idle.)
 */
int tk_gemm_invariant(const tk_half *a, int64_t lda, const tk_half *w,
                      int64_t ldw, const float *bias, const float *resid,
                      int64_t ldr, void *c, int64_t ldc, int64_t m, int64_t n,
                      int64_t k, int epilogue, const uint8_t *row_valid,
                      int row_mode, void *stream);
int tk_gemm_bias_add_ln_invariant(const tk_half *a, int64_t lda,
                                  const tk_half *w, int64_t ldw,
                                  const float *bias, const float *resid,
                                  const float *ln_w, const float *ln_b,
                                  float *sum_out, void *h_out, int h_dtype,
                                  int64_t m, int64_t n, int64_t k, float eps,
                                  const uint8_t *row_valid, int row_mode,
                                  void *stream);

/*
 * FlashAttention-2-style forward (online softmax, scores never stored).
 * q, k, v: logical [batch, heads, seq, head_dim] f16 with element strides
 * {b, h, s} given in *_strides[3] (head_dim stride is 1).  out: logical
 * [batch, heads, seq, head_dim] written through o_strides (pass
 * {S*H*hd, hd, H*hd} for the [B, S, H*hd] layout).
 * scores = (q.k^T) * scale in fp32, causal masks key > query, fp32 softmax,
 * fp16 P on MFMA for P.V, fp32 accumulation.
 * key_valid (nullable): key validity bytes, key s of batch b at
 * key_valid[b * key_valid_stride + s]; invalid keys are masked with -inf
 * like future keys (src/torch_transformer_benchmark.py:104-107).  A query
 * row with no valid key yields non-finite output (the baseline's NaN row);
 * callers zero such padded rows downstream.
 * Any head_dim <= 256 (tk_attention_supported) and any element strides;
 * q/k/v/out 2-byte aligned.  Head dims 16/32/64/128/256 with rows that are
 * 16-byte vectors (q, k; v too except at 128) and 8-byte vectors (out; v
 * at 128) take the tuned kernels; every other head dim or view runs on the
 * tile of the next power of two >= max(head_dim, 16) with element loads and
 * the head-dim tail read as zeros (src/kernels.py:262-263 pads the same way).
 * Replaces kernels.flash_attention / _flash_attn_fwd_kernel
 * (src/kernels.py:250-294, :137-247) and F.scaled_dot_product_attention
 * (src/optimized.py:615-626).
 */
int tk_flash_attn_fwd(const tk_half *q, const tk_half *k, const tk_half *v,
                      tk_half *out, int64_t batch, int64_t heads, int64_t seq,
                      int64_t head_dim, const int64_t *q_strides,
                      const int64_t *k_strides, const int64_t *v_strides,
                      const int64_t *o_strides, float scale, int causal,
                      const uint8_t *key_valid, int64_t key_valid_stride,
                      void *stream);

/* tk_flash_attn_fwd with kernels whose choice does not depend on batch * heads:
 * a sequence's bits do not depend on what else the call has.  (That call splits
 * the keys of launches that would leave most of the chip idle.) */
int tk_flash_attn_fwd_invariant(const tk_half *q, const tk_half *k,
                                const tk_half *v, tk_half *out, int64_t batch,
                                int64_t heads, int64_t seq, int64_t head_dim,
                                const int64_t *q_strides,
                                const int64_t *k_strides,
                                const int64_t *v_strides,
                                const int64_t *o_strides, float scale,
                                int causal, const uint8_t *key_valid,
                                int64_t key_valid_stride, void *stream);

/* 1 when tk_flash_attn_fwd handles head_dim, else 0: the reference's rule
 * next_pow2(max(head_dim, 16)) <= 256, i.e. head_dim <= 256.
 * Replaces kernels.attention_supported (src/kernels.py:96-103). */
int tk_attention_supported(int64_t head_dim);

/*
 * Masked softmax over rows of materialised scores.
 * scores: [groups, seq, seq] f32 (query-major, one group per (b, h));
 * probs: same shape, f16.  causal masks key > query with -inf before the
 * fp32 softmax; key_len (may be NULL) gives per-batch valid key counts
 * (group g belongs to batch g / heads_per_batch) -- keys >= key_len masked.
 * A row whose keys are all masked yields zeros.
 * Replaces the masked softmax of the baseline attention
 * (src/torch_transformer_benchmark.py:99-111; src/optimized.py:658-666).
 */
int tk_masked_softmax(const float *scores, tk_half *probs, int64_t groups,
                      int64_t seq, int causal, const int32_t *key_len,
                      int64_t heads_per_batch, void *stream);

/*
 * The whole dense forward of a narrow model in one launch: for each of the
 * batch's sequences, every layer of
 *   h = LN1(x); qkv = h.W_qkv^T + b; ctx = attention(q, k, v);
 *   x += ctx.W_o^T + b_o; h = LN2(x); u = gelu(h.W_1^T + b_1);
 *   x += u.W_2^T + b_2
 * then out = LN_final(x), with the numerics of the layer-by-layer path
 * (fp16 operands, fp32 accumulation, residual and statistics).
 * x, out: [batch, seq, d_model] f32 (out may not alias x).
 * Weights stacked over the layers, each layer's block as the layer-by-layer
 * calls take it: w_qkv [L][3*heads*hd][d] f16 (head rows zero-padded to hd =
 * head_dim_padded), b_qkv [L][3*heads*hd] f32, w_o [L][d][heads*hd] f16,
 * b_o [L][d], w_1 [L][ffn][d] f16, b_1 [L][ffn], w_2 [L][d][ffn] f16,
 * b_2 [L][d], n1_w, n1_b, n2_w, n2_b [L][d] f32, nf_w, nf_b [d] f32; all
 * 16-byte aligned.
 * scale: the attention scale (1/sqrt(unpadded head_dim)).  Dense inputs only
 * (no padding mask).  Shapes: tk_small_forward_supported.
 * Causal sequences of more than 32 tokens run one 32-row block per
 * workgroup when batch * ceil(seq/32) workgroups fit on the device's CUs at
 * once and batch * layers * 4 <= 4096: the blocks of a sequence hand each
 * layer's K and V rows to one another through a workspace the library
 * allocates on the device the first time a call needs it (and replaces by a
 * larger one, keeping the old, when a call needs more; 16 KB per sequence,
 * layer and block, plus 16 KB), with
 * the same results bit for bit as one workgroup per sequence.  Calls that
 * overlap on one device share that workspace and must not run concurrently;
 * a call made while its stream is being captured into a graph, with no
 * workspace yet large enough, runs one workgroup per sequence instead.
 * Replaces the layer loop of OptimizedTransformer._run_layers_fused
 * (src/optimized.py:488-554) for the narrow configs (reference config 1 and
 * the appendix cases of src/configs/shapes.json with d_model 128).
 */
int tk_small_forward(const float *x, float *out, int64_t batch, int64_t seq,
                     int64_t d_model, int64_t heads, int64_t head_dim_padded,
                     int64_t ffn_dim, int64_t layers, int causal,
                     const tk_half *w_qkv, const float *b_qkv,
                     const tk_half *w_o, const float *b_o,
                     const tk_half *w_1, const float *b_1,
                     const tk_half *w_2, const float *b_2,
                     const float *n1_w, const float *n1_b,
                     const float *n2_w, const float *n2_b,
                     const float *nf_w, const float *nf_b, float n1_eps,
                     float n2_eps, float nf_eps, float scale, void *stream);

/* tk_small_forward without any allocation: the same arguments, work and
 * results (bit for bit), but a split launch hands its K/V rows through a
 * fixed per-device scratch array (16 MB + 16 KB, in the library's code
 * object: each device holds it from the library's load until the process
 * ends) instead of the library's allocated workspace, and its count table is
 * cleared by a small kernel at each call.  Returns TK_ERR_UNSUPPORTED when a
 * split launch would need more than 1024 hand-off slots (batch * layers * 4
 * row blocks, e.g. C1's B64 L4); shapes that run unsplit use no scratch.
 * Calls that overlap on one device share that device's array and race.
 * No counterpart in the reference: for callers that cannot allocate device
 * memory (code under graph capture, tight serving loops, harnesses that
 * forbid hipMalloc).
 */
int tk_small_forward_noalloc(const float *x, float *out, int64_t batch,
                             int64_t seq, int64_t d_model, int64_t heads,
                             int64_t head_dim_padded, int64_t ffn_dim,
                             int64_t layers, int causal, const tk_half *w_qkv,
                             const float *b_qkv, const tk_half *w_o,
                             const float *b_o, const tk_half *w_1,
                             const float *b_1, const tk_half *w_2,
                             const float *b_2, const float *n1_w,
                             const float *n1_b, const float *n2_w,
                             const float *n2_b, const float *nf_w,
                             const float *nf_b, float n1_eps, float n2_eps,
                             float nf_eps, float scale, void *stream);

/* tk_small_forward on weights packed once into the kernel's fragment order
 * (tk_small_pack, from the stacked weights above): the same work and results
 * bit for bit, with one contiguous kilobyte per weight load instead of 32
 * rows.  packed: tk_small_pack_halves(layers) f16 elements, 16-byte aligned.
 * d_model = ffn = 128. */
int64_t tk_small_pack_halves(int64_t layers);
int tk_small_pack(const tk_half *w_qkv, const tk_half *w_o, const tk_half *w_1,
                  const tk_half *w_2, tk_half *packed, int64_t layers,
                  void *stream);
int tk_small_forward_packed(const float *x, float *out, int64_t batch,
                            int64_t seq, int64_t heads,
                            int64_t head_dim_padded, int64_t layers,
                            int causal, const tk_half *packed,
                            const float *b_qkv, const float *b_o,
                            const float *b_1, const float *b_2,
                            const float *n1_w, const float *n1_b,
                            const float *n2_w, const float *n2_b,
                            const float *nf_w, const float *nf_b, float n1_eps,
                            float n2_eps, float nf_eps, float scale,
                            void *stream);

/* Fused QKV projection + attention for one-key-tile sequences:
 *   ctx[t, h*64 + :64] = attention_h( h . W_qkv^T + b_qkv )
 * i.e. tk_gemm(h, w_qkv, b_qkv) into a [T, 3*d_model] q|k|v buffer followed
 * by tk_flash_attn_fwd on its strided views, without the buffer: q, k and v
 * of one head for two sequences stay in LDS.  h: [batch*seq, ldh] fp16;
 * w_qkv: [3*d_model, ldw] fp16 (rows q, k, v, each head's 64 rows
 * contiguous); b_qkv: [3*d_model] fp32; ctx: [batch*seq, ldc] fp16;
 * d_model = heads * head_dim.  Dense inputs only.  Shapes:
 * tk_qkv_attention_supported (seq = 64, head_dim = 64, batch*seq a multiple
 * of 128).  Replaces F.linear + scaled_dot_product_attention of
 * OptimizedTransformer._attention_block (src/optimized.py:572-626) for those
 * shapes (the reference's config 2). */
int tk_qkv_attention(const tk_half *h, int64_t ldh, const tk_half *w_qkv,
                     int64_t ldw, const float *b_qkv, tk_half *ctx,
                     int64_t ldc, int64_t batch, int64_t seq, int64_t heads,
                     int64_t head_dim, float scale, int causal, void *stream);

/* 1 when tk_qkv_attention takes the shape, else 0.  No counterpart in the
 * reference (its attention block always materialises q, k, v). */
int tk_qkv_attention_supported(int64_t batch, int64_t seq, int64_t heads,
                               int64_t head_dim);

/* 1 when tk_small_forward takes the shape (seq <= 128, d_model = ffn_dim =
 * 128, heads * head_dim_padded = 128, head_dim_padded in {16, 32, 64, 128}),
 * else 0.  No counterpart in the reference (its narrow configs run the
 * layer loop). */
int tk_small_forward_supported(int64_t seq, int64_t d_model, int64_t heads,
                               int64_t head_dim_padded, int64_t ffn_dim);

/*
 * The row-local parts of a block of width 128 (tk_narrow_supported: d_model and
 * attention width 128, ffn_dim a multiple of 128 up to 1024), fused:
 *   tk_narrow_qkv:  qkv[rows][384] f16 = LN(x) . W_qkv^T + b
 *   tk_narrow_tail: s = resid + ctx . W_o^T + b_o;
 *                   s += gelu(LN(s; n2) . W_1^T + b_1) . W_2^T + b_2;
 *                   out = LN(s; next) (out_dtype), sum_out (nullable) = s
 * ctx [rows][128] f16, resid and sum_out [rows][128] f32 (sum_out may alias
 * resid).  A weight W[N][K] f16 is given in fragment order: [K/128][N/32] blocks
 * of 8 fragments of 64 lanes of 8 values, lane l of fragment kk holding row
 * l & 31, columns 16 kk + 8 (l >> 5) .. + 8 of its block.  row_valid (nullable,
 * rows bytes): an invalid row keeps its residual after attention and is 0 after
 * the FFN (row_mode TK_ROWS_ZERO), its normalised output too with
 * TK_ROWS_ZERO_ALL (f32 output).  All buffers 16-byte aligned.
 * Replaces add_ln_fwd and F.linear / F.gelu between two attention calls
 * (src/optimized.py:523-553,572,627-636) at that width.
 */
int tk_narrow_supported(int64_t d_model, int64_t attn_width, int64_t ffn_dim);
int tk_narrow_qkv(const float *x, const float *ln_w, const float *ln_b,
                  float eps, const tk_half *w_packed, const float *b_qkv,
                  tk_half *qkv, int64_t rows, void *stream);
int tk_narrow_tail(const tk_half *ctx, const float *resid, const tk_half *w_o,
                   const float *b_o, const float *n2_w, const float *n2_b,
                   float n2_eps, const tk_half *w_1, const float *b_1,
                   const tk_half *w_2, const float *b_2, int64_t ffn_dim,
                   const float *next_w, const float *next_b, float next_eps,
                   float *sum_out, void *out, int out_dtype, int64_t rows,
                   const uint8_t *row_valid, int row_mode, void *stream);

/*
 * The layer loop of the forward: every launch of a dense or padded forward of
 * any width, enqueued by one call with the arguments the entry points above
 * take (no other work, so the results are those of the separate calls).
 *
 * tk_layer / tk_model hold device pointers to packed weights, laid out as
 * the separate calls take them: w_qkv [3*heads*head_dim][d_model] (each
 * head's rows zero-padded to head_dim), w_o [d_model][heads*head_dim], w_1
 * [ffn][d_model], w_2 [d_model][ffn] f16; biases, norms f32.  The structs
 * themselves are host memory, read during the call only.
 */
typedef struct tk_layer {
  const float *n1_w, *n1_b;
  const tk_half *w_qkv;
  const float *b_qkv;
  const tk_half *w_o;
  const float *b_o;
  const float *n2_w, *n2_b;
  const tk_half *w_1;
  const float *b_1;
  const tk_half *w_2;
  const float *b_2;
  /* The four projections in fragment order (tk_narrow_qkv, tk_narrow_tail); NULL: not used. */
  const tk_half *w_qkv_packed, *w_o_packed, *w_1_packed, *w_2_packed;
  float n1_eps, n2_eps;
} tk_layer;

typedef struct tk_model {
  int64_t d_model, heads, head_dim, ffn_dim, num_layers; /* head_dim as padded */
  const tk_layer *layers;                                /* [num_layers] */
  const float *nf_w, *nf_b;
  float nf_eps;
  float scale; /* 1/sqrt(unpadded head_dim) */
  int causal;
} tk_model;

enum tk_forward_flags {
  TK_FWD_FUSED_NORM = 1,    /* tk_narrow_qkv / tk_narrow_tail where they take the shape and every layer's
                              packed weights are given, else tk_gemm_bias_add_ln (with sum_out: a residual
                              GEMM and a LayerNorm launch, timed as one step) where tk_gemm_ln_supported */
  TK_FWD_QKV_ATTENTION = 2, /* tk_qkv_attention where it takes the shape (dense inputs) */
  TK_FWD_BATCH_INVARIANT = 4, /* no kernel whose choice and order of sums depend on the batch size: a
                                 sequence's output bits are the same in every batch */
  TK_FWD_IO_F16 = 8,          /* x and out are fp16 ... */
  TK_FWD_IO_BF16 = 16         /* ... or bf16 instead of fp32; without TK_FWD_FUSED_NORM only */
};

/* Bytes of the workspace that tk_forward needs; negative: a tk_status. */
int64_t tk_forward_workspace(const tk_model *model, int64_t batch, int64_t seq, int dense, int flags);

/* Launches of one forward, and the name of launch `step` (NULL past the end). */
int64_t tk_forward_steps(const tk_model *model, int64_t batch, int64_t seq, int dense, int flags);
const char *tk_forward_step_name(const tk_model *model, int64_t batch, int64_t seq, int dense, int flags,
                                 int64_t step);

/*
 * x, out: [batch, seq, d_model] f32, or 16-bit as the flags say (out may not
 * alias x).  valid (nullable):
 * [batch, seq] validity bytes, NULL = dense.  workspace: 256-byte aligned
 * device memory of at least tk_forward_workspace bytes, this call's own until
 * its launches have run.  Runs launches [first_step, first_step + num_steps);
 * num_steps < 0: all that follow.
 * Replaces the layer loop of OptimizedTransformer._run_layers_fused
 * (src/optimized.py:488-554).
 */
int tk_forward(const tk_model *model, const void *x, void *out, int64_t batch, int64_t seq,
               const uint8_t *valid, void *workspace, int64_t workspace_bytes, int flags,
               int64_t first_step, int64_t num_steps, void *stream);

/*
 * Serving: attention over a window of keys, a paged key/value cache, and attention of one
 * new token over it.  All of them take 16-bit tensors of one dtype (TK_F16 or TK_BF16),
 * head_dim a multiple of 8 up to 256, and rows of 16-byte vectors (base 16-byte aligned,
 * strides multiples of 8 elements; out: 8-byte in tk_window_attn, any in tk_paged_attn).
 * heads is a multiple of kv_heads; head h reads key head h / (heads / kv_heads).  scale is
 * positive and at most 2.3e38.
 * No counterpart in the reference, which recomputes whole sequences with full causal
 * attention (src/kernels.py:250-294).
 */

/*
 * Causal attention of the last q_len of k_len positions (q_len <= k_len): query i sits at
 * position p = k_len - q_len + i and sees key j when j <= p, and j > p - window or
 * j < sinks, and key_valid[b * key_valid_stride + j] (nullable) is set.  window >= 1; one of
 * k_len or more is plain causal attention.  A query that sees nothing gets 0.
 * q [batch, heads, q_len, head_dim], k and v [batch, kv_heads, k_len, head_dim], out as q:
 * element strides {b, h, s} in *_strides[3].  What K and V hold at keys that
 * are not valid has no effect; at valid ones it must be finite.
 * Launches with few query rows split their keys over workgroups; batch_invariant: not so, a
 * sequence's bits do not depend on the rest of the batch.  workspace:
 * tk_window_attn_workspace bytes, 16-byte aligned, this call's own until its launches have
 * run (0 bytes: may be NULL).
 */
int64_t tk_window_attn_workspace(int64_t batch, int64_t heads,
                                 int64_t kv_heads, int64_t q_len,
                                 int64_t k_len, int64_t head_dim,
                                 int64_t window, int64_t sinks,
                                 int batch_invariant);
int tk_window_attn(const void *q, const int64_t *q_strides, const void *k,
                   const int64_t *k_strides, const void *v,
                   const int64_t *v_strides, void *out,
                   const int64_t *o_strides, int dtype, int64_t batch,
                   int64_t heads, int64_t kv_heads, int64_t q_len,
                   int64_t k_len, int64_t head_dim, float scale,
                   int64_t window, int64_t sinks, const uint8_t *key_valid,
                   int64_t key_valid_stride, int batch_invariant,
                   void *workspace, int64_t workspace_bytes, void *stream);

/*
 * The cache: k and v pages [layers][pages][kv_heads][page_size][head_dim] (any strides with
 * 16-byte rows; page_size a power of two from 16 to 1024) and three int32 arrays on the
 * device: table [rows][table_width], row stride table_stride; lengths [rows]; refs [pages].
 * A sequence of n tokens holds the first ceil(n / page_size) entries of its row, token j in
 * row j % page_size of page table[j / page_size].  refs counts the sequences that hold a
 * page; it is free at refs <= 0.  Entries that are no page of the cache are never followed.
 */

/*
 * out[b, h] = attention of the token at position lengths[b] - 1 over sequence b: q
 * [batch, heads, head_dim], strides {b, h}; pages of one layer, strides {page, head, row}.
 * It sees key j when j >= lengths[b] - window or j < sinks; window 0: every key.  Keys whose
 * table entry is no page of the cache are not seen; a sequence that sees nothing gets 0.
 * max_length: the longest length to be expected; it only sizes the split of the keys over
 * workgroups, longer sequences are attended whole.  batch_invariant: a sequence's bits do
 * not depend on the rest of the batch, table_width or max_length, which then counts (in the
 * workspace's size too) as at least table_width * page_size.  workspace: tk_paged_attn_workspace bytes, 16-byte
 * aligned, this call's own until its launches have run (0 bytes: may be NULL).  Fewer than 2^24
 * rows (batch * heads) and at most 2^34 tokens (batch * table_width * page_size) in all.
 */
int64_t tk_paged_attn_workspace(int64_t batch, int64_t heads, int64_t kv_heads,
                                int64_t head_dim, int64_t max_length,
                                int64_t window, int64_t sinks,
                                int batch_invariant);
int tk_paged_attn(const void *q, const int64_t *q_strides, const void *k_pages,
                  const int64_t *k_strides, const void *v_pages,
                  const int64_t *v_strides, void *out,
                  const int64_t *o_strides, int dtype, int64_t batch,
                  int64_t heads, int64_t kv_heads, int64_t head_dim,
                  int64_t pages, int64_t page_size, const int32_t *table,
                  int64_t table_stride, int64_t table_width,
                  const int32_t *lengths, int64_t max_length, float scale,
                  int64_t window, int64_t sinks, int batch_invariant,
                  void *workspace, int64_t workspace_bytes, void *stream);

/*
 * Writes the last added[b] tokens (nullable: n; at most n) of every sequence into its pages:
 * row i < added[b] of k and v [batch, n, kv_heads, head_dim], strides {b, token, head}, goes
 * to position lengths[b] - added[b] + i.  Positions before 0, past the table, or on an entry
 * that is no page of the cache are left out.  Pages of one layer, strides {page, head, row}.
 * A reservation that was refused has left lengths as they were, so its tokens would be written
 * over the newest ones of every sequence: tk_cache_append_reserved takes the reservation's status
 * (device) and writes nothing where it is not 0.
 */
int tk_cache_append(const void *k, const int64_t *k_strides, const void *v,
                    const int64_t *v_strides, void *k_pages,
                    const int64_t *k_page_strides, void *v_pages,
                    const int64_t *v_page_strides, int64_t batch, int64_t n,
                    int64_t kv_heads, int64_t head_dim, int64_t pages,
                    int64_t page_size, const int32_t *table,
                    int64_t table_stride, int64_t table_width,
                    const int32_t *lengths, const int32_t *added, void *stream);
int tk_cache_append_reserved(const void *k, const int64_t *k_strides,
                             const void *v, const int64_t *v_strides,
                             void *k_pages, const int64_t *k_page_strides,
                             void *v_pages, const int64_t *v_page_strides,
                             int64_t batch, int64_t n, int64_t kv_heads,
                             int64_t head_dim, int64_t pages,
                             int64_t page_size, const int32_t *table,
                             int64_t table_stride, int64_t table_width,
                             const int32_t *lengths, const int32_t *added,
                             const int32_t *status, void *stream);

/*
 * Page bookkeeping, decided on the device.  An operation that cannot be done whole changes
 * nothing and leaves the reason in *status (device): the number of pages that were missing,
 * or -1 for a row, length or count that cannot be taken; 0 when done.  Free pages are taken
 * from the lowest id on.  workspace: tk_cache_workspace bytes (rows, pages, and n children;
 * n = 0 but for a fork), 4-byte aligned, this call's own until its launches have run.
 *
 * reserve: lengths[b] += added[b] >= 0 for every row, with the pages that this needs.
 * fork:    child i (an empty row, named once) becomes a copy of parent i as it was before the
 *          call: it shares the parent's whole pages and gets a page of its own with the rows
 *          of the one that is begun, in every layer (strides {layer, page, head, row}).  At most
 *          2^18 rows.
 * free:    every listed row gives up its pages (-1 in the table) and has length 0; rows that
 *          are not in the table are passed over, a row listed twice is freed once.
 * compact: with `used` live pages in all, the i-th live page of those with id >= used moves
 *          into the i-th free one below, ascending, in every layer; table and refs follow.
 *          *used (device): their number, so that pages [used, pages) are free afterwards.
 */
int64_t tk_cache_workspace(int64_t rows, int64_t pages, int64_t n);
int tk_cache_reserve(int32_t *table, int64_t table_stride, int64_t table_width,
                     int64_t rows, int32_t *lengths, int32_t *refs,
                     int64_t pages, int64_t page_size, const int32_t *added,
                     int32_t *status, void *workspace, int64_t workspace_bytes,
                     void *stream);
int tk_cache_fork(void *k_pages, const int64_t *k_strides, void *v_pages,
                  const int64_t *v_strides, int64_t layers, int64_t kv_heads,
                  int64_t head_dim, int32_t *table, int64_t table_stride,
                  int64_t table_width, int64_t rows, int32_t *lengths,
                  int32_t *refs, int64_t pages, int64_t page_size,
                  const int32_t *parents, const int32_t *children, int64_t n,
                  int32_t *status, void *workspace, int64_t workspace_bytes,
                  void *stream);
int tk_cache_free(int32_t *table, int64_t table_stride, int64_t table_width,
                  int64_t rows, int32_t *lengths, int32_t *refs, int64_t pages,
                  int64_t page_size, const int32_t *list, int64_t n,
                  void *stream);
int tk_cache_compact(void *k_pages, const int64_t *k_strides, void *v_pages,
                     const int64_t *v_strides, int64_t layers,
                     int64_t kv_heads, int64_t head_dim, int32_t *table,
                     int64_t table_stride, int64_t table_width, int64_t rows,
                     const int32_t *lengths, int32_t *refs, int64_t pages,
                     int64_t page_size, int32_t *used, void *workspace,
                     int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TKMI_H */
