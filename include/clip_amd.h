/* clip_amd.h — C ABI of libclip_amd.so, the MI355X (gfx950) engine for the bulk BERT(+Context)
 * sentence-scoring path of asappresearch/clip.
 *
 * The reference has no FFI/plugin layer on this path: the boundary it sits behind is the Python
 * nn.Module contract (from_pretrained / load_state_dict / set_* / forward -> (loss, logits)) plus
 * the inline numpy epilogue of the driver.  Each entry point below cites the reference lines whose
 * work it takes over; clip_amd/bert_model.py and clip_amd/scoring.py are the host mirrors that
 * bind these symbols with ctypes (INTEGRATION.md shows the stub a reference maintainer would add).
 *
 * Conventions: plain pointers and sizes only; every function returns 0 (CLIP_OK) or a negative
 * clip_status; no C++ exception crosses the ABI; clip_last_error() gives the message of the last
 * failure on the calling thread.  Pointers named dev_* are device (HIP) pointers owned by the
 * caller (e.g. torch tensors' data_ptr()), host_* are host pointers.  `stream` is a hipStream_t
 * passed as void* (NULL = default stream).  One engine per device per process; an engine is not
 * re-entrant (its workspace is shared by all calls on it).
 */
#ifndef CLIP_AMD_H
#define CLIP_AMD_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum clip_status {
  CLIP_OK = 0,
  CLIP_ERR_ARG = -1,       /* bad argument (null pointer, unsupported shape, unknown name) */
  CLIP_ERR_HIP = -2,       /* a HIP runtime call failed */
  CLIP_ERR_STATE = -3,     /* call order: weights missing / not finalized */
  CLIP_ERR_CAPACITY = -4,  /* n_seqs / total_tokens beyond the engine's workspace */
  CLIP_ERR_SEP_COUNT = -5  /* a row does not hold exactly 2n+1 [SEP] (bert_model.py:51-55) */
} clip_status;

typedef struct clip_engine clip_engine; /* opaque */

/* Encoder geometry = the transformers.BertConfig fields the reference reads
 * (sentclf/apply_bert_unlabeled.py:55-62; sentclf/bert_model.py:13-19). */
typedef struct clip_config {
  int32_t vocab_size, hidden_size, num_layers, num_heads, intermediate_size;
  int32_t max_position, type_vocab_size, num_labels;
  float layer_norm_eps;
  int32_t max_tokens; /* workspace capacity: packed tokens per forward call */
  int32_t max_seqs;   /* workspace capacity: sequences per forward call */
} clip_config;

/* Replaces model construction + model.to(device) (apply_bert_unlabeled.py:65-72; test_load.py:21).
 * Binds the engine to `device_id`; device weights and the activation workspace are allocated by
 * clip_finalize_weights. */
int clip_create(const clip_config* cfg, int device_id, clip_engine** out);
int clip_destroy(clip_engine* e);

/* Replaces model.load_state_dict(sd) (apply_bert_unlabeled.py:78-79), one tensor per call, using
 * the reference's 201 state-dict key names; host_data is fp32, row-major, `numel`
 * elements.  "bert.embeddings.position_ids" and other unknown buffers return CLIP_ERR_ARG and may
 * be skipped by the caller.  clip_finalize_weights() fails with CLIP_ERR_STATE if a key is missing;
 * it builds the fused bf16 QKV weight (1/sqrt(head_dim) folded into the query rows). */
int clip_load_weight(clip_engine* e, const char* name, const float* host_data, int64_t numel);
int clip_finalize_weights(clip_engine* e);

/* Numerics setting of the engine, chosen before clip_finalize_weights (which rounds the GEMM weights
 * and sizes the activation workspace accordingly).  The reference runs fp32 torch
 * (apply_bert_unlabeled.py:72 moves an fp32 model to the device); BASELINE.json asks for bf16 with an
 * fp32 check mode:
 *   CLIP_PRECISION_BF16 (default): bf16 GEMM / attention operands, fp32 accumulation, fp32
 *     LayerNorm statistics and softmax — logits within 2e-2 of the reference;
 *   CLIP_PRECISION_FP32: the same kernel templates instantiated on fp32 operands
 *     (v_mfma_f32_16x16x4_f32, fp32 activations end to end; attention in plain fp32 FMAs; every layer
 *     whole, no last-layer trimming) — logits within 1e-4 of the reference.  ~1/16 of the MFMA rate:
 *     a checker for the bf16 path, not a production setting;
 *   CLIP_PRECISION_F16: the same kernels compiled for fp16 operands (v_mfma_*_f16: the same MFMA rate as
 *     bf16, 11 significant bits instead of 8, fp32 accumulation / LayerNorm / softmax as in the bf16
 *     setting).  For checkpoints whose logits reach beyond +-2: operand rounding is ~1/8 of bf16's, so the
 *     2e-2 budget holds on weights with trained-like statistics (tests/test_gpu_parity_gates.py), where
 *     bf16 operands cannot (their rounding alone is ~0.5 % of the logit spread).  The price is fp16's
 *     RANGE: a weight beyond +-65504 is refused at load; an activation beyond it becomes inf and the
 *     logits NaN (never silently wrong).  BERT-base activations stay far inside it.  In this setting the
 *     LayerNorm output is kept ONCE (fp16, row-major: GEMM operand and residual are the same bits), where
 *     the bf16 setting keeps a bf16 operand copy and an fp16 residual copy;
 *   CLIP_PRECISION_F16R: fp16 operands as above with the RESIDUAL STREAM IN FP32: the fused-LayerNorm GEMMs
 *     read and rewrite an fp32 copy of every LayerNorm output (clip_gemm_f16_lnout_res32) beside the fp16
 *     operand copy — the residual never passes through a 16-bit type.  (Hidden sizes that are not a multiple
 *     of 256, or clip_set_fused_layernorm(e, 0): fp32 pre-LayerNorm rows + (mean, rstd), the residual
 *     recomputed in the GEMM epilogue — clip_gemm_bf16_lnres's form on fp16 operands.)  Measured on the
 *     trained-like stress goldens: rms logit error 3.8e-3 -> 2.6e-3, max 2.14e-2 -> below the 2e-2 budget;
 *     more bytes per token than CLIP_PRECISION_F16 (7.5 KB instead of 3 KB per fused GEMM). */
enum { CLIP_PRECISION_BF16 = 0, CLIP_PRECISION_FP32 = 1, CLIP_PRECISION_F16 = 2, CLIP_PRECISION_F16R = 3 };
int clip_set_precision(clip_engine* e, int32_t precision);

/* Replaces _collect_focus_repr's index search (bert_model.py:52): for each packed sequence the
 * token index of its (n_ctx+1)-th `sep_id`; n_ctx < 0 selects the first token ([CLS], the pooler
 * row of bert_model.py:234).  dev_err[0] gets bit 0 set when a sequence does not hold exactly
 * 2*n_ctx+1 separators. */
int clip_focus_index(const int32_t* dev_ids, const int32_t* dev_cu_seqlens, int32_t n_seqs,
                     int32_t sep_id, int32_t n_ctx, int32_t* dev_focus, int32_t* dev_err,
                     void* stream);

/* Replaces the per-batch tensor building of the collators for PACKED rows, on the device, from the
 * token ids alone: token-type ids exactly as sentclf/bert.py:168-176 assigns them (type 0 on the
 * [SEP] before the focus and on the focus tokens, 1 elsewhere; all 0 when n_ctx <= 0 as
 * sentclf/bert.py:44-68 passes none), position ids 0..len-1 (modeling_bert.py:65,83) and the focus
 * index of clip_focus_index (n_ctx <= 0: the row's first token).  dev_err as clip_focus_index. */
int clip_prepare_packed(const int32_t* dev_ids, const int32_t* dev_cu_seqlens, int32_t n_seqs,
                        int32_t sep_id, int32_t n_ctx, int32_t* dev_type_ids, int32_t* dev_pos_ids,
                        int32_t* dev_focus, int32_t* dev_err, void* stream);

/* Replaces model(**inputs) (apply_bert_unlabeled.py:110; test_load.py:36; bert_model.py:66-103
 * and :210-251) on PACKED rows: token t of sequence s sits at dev_ids[cu_seqlens[s] + t]; the
 * key-padding mask of the reference (modeling_bert.py:688-708) is replaced by the packing.
 *   head_kind 0: hidden state at dev_focus[s] -> classifier           (context model)
 *   head_kind 1: tanh pooler on dev_focus[s] (= [CLS]) -> classifier  (sentence-only model)
 * dev_type_ids may be NULL (all zero).  dev_logits is fp32 [n_seqs, num_labels]. */
int clip_forward_packed(clip_engine* e, const int32_t* dev_ids, const int32_t* dev_type_ids,
                        const int32_t* dev_pos_ids, const int32_t* dev_cu_seqlens,
                        const int32_t* dev_focus, int32_t n_seqs, int32_t total_tokens,
                        int32_t max_seqlen, int32_t head_kind, float* dev_logits, void* stream);

/* Replaces model(**inputs) on the reference's own PADDED tensors (apply_bert_unlabeled.py:110;
 * test_load.py:36; bert_model.py:66-103): int64 [B, S] row-major device arrays as the HF tokenizer
 * and the collators produce them (sentclf/bert.py:57,152).  attention_mask (NULL = all ones) selects
 * the tokens (modeling_bert.py:688-708); token_type_ids may be NULL (all zero); position_ids may be
 * NULL (the padded column index, modeling_bert.py:65,83), else `position_row_stride` is 0 for one
 * broadcast row or S for B rows.  The engine packs the rows on the device into its own workspace
 * (one wait for the token count, returned in *total_tokens when not NULL), finds the focus index
 * (sep_id, n_ctx as clip_focus_index; ignored for head_kind 1) and runs clip_forward_packed.  A row
 * with a wrong [SEP] count sets bit 0 of the engine's error word, a row without any unmasked token
 * (or longer than max_position) bit 2.  error_flags NULL: the call returns with the forward queued;
 * poll with clip_poll_errors.  error_flags not NULL: the call returns when the forward has finished,
 * with the error word (bits of clip_poll_errors; cleared when set) in *error_flags.  Both waits spin
 * on words the device writes into mapped host memory (no copy back, no stream wait; after 2 s without
 * the word the call falls back to a stream wait and reports CLIP_ERR_HIP if it is still missing).
 * Because it waits on the host in its middle, this entry point cannot be captured into a HIP graph.
 * (clip_forward_packed has no host wait, but in the fused-LayerNorm flow every launch carries an epoch
 * numbered on the host: a captured forward must not be REPLAYED in that flow either — the replay
 * would meet its own flags.  Only clip_gemm_bf16_lnout_noalloc is built and tested for replay.) */
int clip_forward_padded(clip_engine* e, const int64_t* dev_input_ids, const int64_t* dev_attention_mask,
                        const int64_t* dev_token_type_ids, const int64_t* dev_position_ids,
                        int64_t position_row_stride, int32_t batch, int32_t width, int32_t sep_id,
                        int32_t n_ctx, int32_t head_kind, float* dev_logits, int32_t* total_tokens,
                        int32_t* error_flags, void* stream);

/* Replaces the numpy epilogue of the driver (apply_bert_unlabeled.py:111-124) and the per-label
 * decision of test_load.py:37-38: probs = sigmoid(logits) (fp32); labels[i,j] = (double)p > t_j
 * (strict, fp64 thresholds); keep[i] = any_j(p > any_thresh) (fp32 compare, as numpy does for a
 * float32 array against a Python float); max_score[i] = max_j p.  Any output pointer may be NULL;
 * dev_label_thresh may be NULL when dev_labels is NULL. */
int clip_epilogue(const float* dev_logits, const double* dev_label_thresh, float any_thresh,
                  int32_t n, int32_t num_labels, float* dev_probs, float* dev_max_score,
                  uint8_t* dev_labels, uint8_t* dev_keep, void* stream);

/* Replaces F.binary_cross_entropy_with_logits(logits, labels) (bert_model.py:97): mean over all
 * `count` elements, written to dev_loss[0]. */
int clip_bce_loss(const float* dev_logits, const float* dev_targets, int32_t count,
                  float* dev_loss, void* stream);

/* The LM prediction head + CrossEntropyLoss of BertContextMLMSwitch.forward (bert_model.py:113,165,
 * 175-179; transformers BertLMPredictionHead: dense H->H + erf-GELU + LayerNorm, decoder H->vocab + bias),
 * for task-targeted pre-training's evaluation pass (weights mlm_predictions.* loaded
 * with clip_load_weight).  Works on the last hidden state the LATEST clip_forward_packed on this engine left
 * behind, which must have run with clip_set_trim_last_layer(e, 0).  dev_rows[i] is a packed token index
 * whose MLM label dev_labels[i] is a vocabulary id: CrossEntropyLoss ignores label -100, so the caller
 * passes only the labelled positions and the decoder runs on those rows alone.
 *   dev_loss[0] = (accumulate ? dev_loss[0] : 0) + mean_i(logsumexp(scores_i) - scores_i[label_i])
 * (NaN for n_rows == 0, as torch's mean over no elements); dev_scores_out (optional) receives the fp32
 * scores [n_rows, vocab] (mlm_scores of bert_model.py:165 at those positions).  The head's workspace
 * (n_rows x padded vocabulary of fp32) is allocated on first use and grows with n_rows. */
int clip_mlm_head(clip_engine* e, const int32_t* dev_rows, const int32_t* dev_labels, int32_t n_rows,
                  float* dev_scores_out, float* dev_loss, int32_t accumulate, void* stream);
/* CrossEntropyLoss(logits [n, n_classes] fp32, labels int32) as bert_model.py:182 applies it to the switch
 * logits: dev_row_loss[i] = logsumexp(logits_i) - logits_i[label_i]; dev_loss[0] (+)= their mean. */
int clip_ce_loss(const float* dev_logits, const int32_t* dev_labels, int32_t n, int32_t n_classes,
                 float* dev_row_loss, float* dev_loss, int32_t accumulate, void* stream);

/* ---- losses of the vocabulary decoder with their gradients, the scores never kept ----
 * The reference trains BertContextMLMSwitch's LM head with CrossEntropyLoss over scores = decoder(hidden)
 * (bert_model.py:165,175-179; its loop is pretrain_tasks.py:333-466); clip_mlm_head evaluates that loss and keeps
 * [n_rows, vocab] fp32 scores.  The entry points below take any hidden rows and any decoder and give the loss AND the
 * gradients with a workspace that does not grow as n x vocab: of the order of n x hidden (and n x k), 64 bytes per vocabulary entry
 * for a distillation's gradients, and one piece of the vocabulary, at most 1 GiB of 16-bit score gradients, or of (max, sum) pairs
 * for a loss.  Stateless: no engine, all
 * memory is the caller's, all work is queued on `stream` of the current device, nothing waits on the host, and calls can be
 * captured into HIP graphs (after one eager call of the same sizes) and replayed; calls that run at the same time need workspaces
 * of their own. */
typedef struct clip_linear {
  int32_t operand;               /* CLIP_PRECISION_BF16 or CLIP_PRECISION_F16: type of hidden, weight and their gradients */
  int32_t n;                     /* hidden rows, 0 <= n < 2^21, (n + 256) hidden_size < 2^31 */
  int32_t hidden_size;           /* a multiple of 64, <= 8192 */
  int64_t vocab;                 /* decoder rows, 1 .. 2^30; n x vocab < 2^45 */
  const uint16_t* dev_hidden;    /* [n, hidden_size], row stride ld_hidden (elements, >= hidden_size) */
  int64_t ld_hidden;
  const uint16_t* dev_weight;    /* [vocab, hidden_size], row stride ld_weight (a multiple of 8), 16-byte aligned */
  int64_t ld_weight;             /* <= 2^22 */
  const float* dev_bias;         /* [vocab] fp32 (4-byte aligned), or NULL; -inf leaves an entry out of the softmax */
} clip_linear;

/* Bytes of workspace (16-byte aligned) of the calls below for these sizes: k = 0 for the cross entropy, else the teacher's
 * entries per row; grad = 0 for the loss, 1 for the gradients. */
int clip_linear_loss_workspace(const clip_linear* d, int32_t k, int32_t grad, int64_t* bytes);

/* z = hidden weight^T + bias;  row_loss[i] = logsumexp(z_i) - z_i[labels[i]] (CrossEntropyLoss, bert_model.py:175-179),
 * 0 where labels[i] == ignore_index; NaN (with NaN gradients) where a label is neither that nor in [0, vocab).
 *   reduction 0: rows only;  1: loss[0] = mean over the rows that are not ignored (NaN when there is none, as torch);
 *   2: loss[0] = sum.   dev_loss may be NULL for 0.
 * dev_lse [n, 2] (m, s, with logsumexp(z_i) = ln 2 m + ln s; 8-byte aligned) and dev_target [n] (z_i[labels[i]]) are what the gradient
 * call needs of the forward. */
int clip_linear_ce(const clip_linear* d, const int64_t* dev_labels, int64_t ignore_index, int32_t reduction,
                   float* dev_row_loss, float* dev_lse, float* dev_target, float* dev_loss, void* dev_work,
                   int64_t work_bytes, void* stream);
/* Gradients of the same loss: dz_i = g_i (softmax(z_i) - onehot(labels[i])), dhidden = dz weight, dweight = dz^T hidden,
 * dbias = column sums of dz; g_i = dev_grad[i] for reduction 0, dev_grad[0] / count for 1, dev_grad[0] for 2 (fp32).  Ignored
 * rows get zero dhidden rows and reach nothing else, whatever they hold.  Any of the three outputs may be NULL.  dz is rounded
 * once to the operand type for the two products (a relative 2^-8 or 2^-11; for fp16 no finer than 2^-40 of the call's largest |g_i| T:
 * with V 30 522 the dhidden rows of a g_i down to 2^-20 of the largest are as exact as the others', of 2^-24 off by 0.2 % and of 2^-27 by
 * 1.3 %, and bf16 is the type for a wider range), but the label's entry reaches dhidden with the
 * rounding's residual added back, calls of at most 64 rows form dweight from two such parts of dz, and dbias is summed from
 * unrounded values.  dweight must be 8-byte aligned with a row stride that is a multiple of 4.  Every call that asks for the
 * same outputs gives the same bits. */
int clip_linear_ce_grad(const clip_linear* d, const int64_t* dev_labels, int64_t ignore_index, int32_t reduction,
                        const float* dev_lse, const float* dev_target, const float* dev_grad, uint16_t* dev_dhidden,
                        int64_t ld_dhidden, uint16_t* dev_dweight, int64_t ld_dweight, float* dev_dbias, void* dev_work,
                        int64_t work_bytes, void* stream);
/* Distillation from a teacher's top scores at `temperature` T (1e-6 <= T <= 1e6): row i lists k scores teacher_values[i, :] with their
 * vocabulary ids teacher_index[i, :]; p_i = softmax of the listed values / T, q_i = softmax(z_i / T) over the vocabulary,
 *   row_loss[i] = T^2 sum_j p_ij (log p_ij - log q_i[index_ij]).
 * An entry with a negative id or the value -inf is left out; a row with none left contributes nothing (loss 0, no gradient,
 * not counted by the mean).  Ids may repeat within a row.  An id >= vocab, a NaN or a +inf makes the row's loss NaN (and the
 * gradients).  Scores / T are good up to 2^30 (beyond, fp32 has no digits left for their differences: infinite or NaN).  1 <= k <= 1024.
 * dev_target [n (2 k + 1)] is what the gradient call needs of the lists, which it does not read again.  No counterpart in the
 * reference. */
int clip_linear_distill(const clip_linear* d, const float* dev_teacher_values, const int64_t* dev_teacher_index, int32_t k,
                        float temperature, int32_t reduction, float* dev_row_loss, float* dev_lse, float* dev_target,
                        float* dev_loss, void* dev_work, int64_t work_bytes, void* stream);
/* Its gradients, dz_i = g_i T (q_i - p_i), as clip_linear_ce_grad (residuals for the teacher's ids with |q - p| >= 1/16). */
int clip_linear_distill_grad(const clip_linear* d, const int64_t* dev_teacher_index, int32_t k, float temperature,
                             int32_t reduction, const float* dev_lse,
                             const float* dev_target, const float* dev_grad, uint16_t* dev_dhidden, int64_t ld_dhidden,
                             uint16_t* dev_dweight, int64_t ld_dweight, float* dev_dbias, void* dev_work,
                             int64_t work_bytes, void* stream);
/* The k largest scores of every row with their ids, largest first, ties to the lowest id, NaN above everything (torch.topk's
 * order with its ties settled): what a teacher hands to clip_linear_distill.  `type` CLIP_PRECISION_BF16 / FP32 / F16 is that
 * of dev_scores [n, vocab] (row stride ld) and dev_values [n, k]; 1 <= k <= min(vocab, 1024).  The last step before it in the
 * reference's terms is the decoder's scores, bert_model.py:165 (clip_mlm_head's dev_scores_out). */
int clip_topk_scores(int32_t type, const void* dev_scores, int64_t ld, int32_t n, int32_t vocab, int32_t k,
                     void* dev_values, int64_t* dev_index, void* stream);

/* ---- single-kernel entry points (parity tests drive each kernel through the ABI) ---- */
/* out[M,N] = epi(A[M,K] W[N,K]^T + bias): epi 0 bias, 1 bias+erf-GELU, 2 bias+residual, 3 bias+tanh
 * (modeling_bert.py:175-177, 289-293, 334-337, 347-351, 457-463). A, W, res are bf16; out bf16 or
 * fp32 (out_f32). Leading dimensions in elements. tile: 0 = choose, 128 / 256 = force that
 * workgroup tile edge, 2 = ping-pong persistent kernel (M, N multiples of 256, K of 128). */
int clip_gemm_bf16(const uint16_t* dev_A, const uint16_t* dev_W, const float* dev_bias,
                   const uint16_t* dev_res, void* dev_out, int32_t M, int32_t N, int32_t K,
                   int32_t lda, int32_t ldw, int32_t ldo, int32_t ldres, int32_t epi,
                   int32_t out_f32, int32_t tile, void* stream);
/* clip_gemm_bf16 on fp16 operands (A, W, res fp16; out fp16 or fp32): the k_f16 kernel set */
int clip_gemm_f16(const uint16_t* dev_A, const uint16_t* dev_W, const float* dev_bias,
                  const uint16_t* dev_res, void* dev_out, int32_t M, int32_t N, int32_t K,
                  int32_t lda, int32_t ldw, int32_t ldo, int32_t ldres, int32_t epi,
                  int32_t out_f32, int32_t tile, void* stream);
/* The residual form the engine uses in the bf16 setting: out_f32[m,n] = A W^T + bias + LN(pre)[r,n]
 * with r = res_index ? res_index[m] : m, where LN(pre) is the fp32 LayerNorm output
 * (modeling_bert.py:292,350: what the reference adds as the residual) recomputed in the epilogue from
 * the producer's fp32 pre-LayerNorm rows `dev_res_pre`, their (mean, rstd) pairs `dev_ln_stats`
 * (clip_layernorm_stats) and the affine — so the residual stream never passes through bf16.
 * tile as clip_gemm_bf16; res_index only with the one-tile kernels (0, 128, 256). */
int clip_gemm_bf16_lnres(const uint16_t* dev_A, const uint16_t* dev_W, const float* dev_bias,
                         const float* dev_res_pre, const float* dev_ln_stats,
                         const float* dev_ln_gamma, const float* dev_ln_beta,
                         const int32_t* dev_res_index, float* dev_out, int32_t M, int32_t N,
                         int32_t K, int32_t lda, int32_t ldw, int32_t ldo, int32_t ldres,
                         int32_t tile, void* stream);
/* The fused form (ping-pong kernel; M, N multiples of 256, N <= 2048, K a multiple of 128):
 *   v = A W^T + bias + res16[m, :] (fp16);  x_out (bf16), xres_out (fp16) = LayerNorm_{gamma,beta,eps}(v)
 * over the N columns of each row (BertSelfOutput / BertOutput, modeling_bert.py:289-293, 347-351, in
 * one kernel, no pre-LayerNorm tensor in HBM).  The N/256 workgroups computing the column tiles of a
 * 256-row panel run side by side and exchange per-row sums through dev_part ((M/256)*(N/256)*256
 * float pairs) and dev_flags ((M/256)*(N/256) uint32, zero before first use); `epoch` must differ from
 * every earlier call on the same flags; dev_err |= 2 if a partner never published (clip_poll_errors).
 * xres_out is TILED for the kernel's accumulator layout: element (row, col) at
 *   ((tile*8 + wave)*8 + blk)*1024 + nh*512 + lane*8 + i*4 + e,  tile = (row>>8)*(N/256) + (col>>8),
 *   r = row&255, c = col&255, wave = ((r>>6)&1)*4 + (c>>6), blk = (r>>7)*4 + ((r>>4)&3),
 *   lane = ((c>>2)&3)*16 + (r&15), nh = (c>>5)&1, i = (c>>4)&1, e = c&3
 * (whole 1-KiB wave stores, and whole 1-KiB loads when the next call takes it as its residual).
 * res_tiled != 0: dev_res16 is such a tiled tensor and may be xres_out itself (a workgroup rewrites
 * exactly the elements it read); 0: row-major fp16 with row stride ldres, not aliasing xres_out. */
int clip_gemm_bf16_lnout(const uint16_t* dev_A, const uint16_t* dev_W, const float* dev_bias,
                         const uint16_t* dev_res16, int32_t res_tiled, const float* dev_gamma, const float* dev_beta,
                         float eps, uint16_t* dev_x_out, uint16_t* dev_xres_out, float* dev_part,
                         uint32_t* dev_flags, uint32_t epoch, int32_t* dev_err, int32_t M, int32_t N,
                         int32_t K, int32_t lda, int32_t ldw, int32_t ldo, int32_t ldres, void* stream);
/* The f16 setting's form of clip_gemm_bf16_lnout (fp16 operands, CLIP_PRECISION_F16; same reference math,
 * modeling_bert.py:289-293 / :347-351): operand copy and residual copy would hold the same fp16 bits, so there is
 * ONE buffer.  x_inout [M, N] (row stride ldx, fp16) holds the residual on entry and LayerNorm(A W^T + bias +
 * residual) on return; every workgroup reads exactly the elements it rewrites.  A must not alias x_inout.
 * part / flags / epoch / err as clip_gemm_bf16_lnout. */
int clip_gemm_f16_lnout_inplace(const uint16_t* dev_A, const uint16_t* dev_W, const float* dev_bias,
                                const float* dev_gamma, const float* dev_beta, float eps, uint16_t* dev_x_inout,
                                float* dev_part, uint32_t* dev_flags, uint32_t epoch, int32_t* dev_err, int32_t M,
                                int32_t N, int32_t K, int32_t lda, int32_t ldw, int32_t ldx, void* stream);
/* The F16R setting's form (fp16 operands, FP32 residual stream; same reference math, modeling_bert.py:289-293 /
 * :347-351): xres32_inout [M, N] fp32 holds the residual on entry and the fp32 LayerNorm output on return — the
 * residual never passes through a 16-bit type — and x_out (fp16, row stride ldx) receives the same values rounded
 * once, as the next GEMM's operand.  xres32_inout is TILED in the order of clip_gemm_bf16_lnout's xres_out with the
 * two 16-column blocks of a lane stored one after the other (16-byte accesses):
 *   ((tile*8 + wave)*8 + blk)*1024 + nh*512 + i*256 + lane*4 + e      (tile, wave, blk, lane, nh, i, e as above);
 * a workgroup rewrites exactly the elements it read.  part / flags / epoch / err as clip_gemm_bf16_lnout. */
int clip_gemm_f16_lnout_res32(const uint16_t* dev_A, const uint16_t* dev_W, const float* dev_bias,
                              const float* dev_gamma, const float* dev_beta, float eps, uint16_t* dev_x_out,
                              float* dev_xres32_inout, float* dev_part, uint32_t* dev_flags, uint32_t epoch,
                              int32_t* dev_err, int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldw,
                              int32_t ldx, void* stream);

/* clip_gemm_bf16_lnout for callers that CANNOT ALLOCATE (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc).  No counterpart in the reference.  Same arguments, kernel and
 * result bits as clip_gemm_bf16_lnout, minus dev_part / dev_flags / epoch: the exchange buffers live in
 * a static device array inside the library (4.2 MB per GPU, held until the process ends).  Calls no
 * hipMalloc / hipFree or allocating routine.  Every call enqueues, on `stream`, a clear of the flags of the
 * tiles it uses followed by the kernel (which waits for the constant 1): nothing in the kernel arguments
 * depends on a host-side counter, so a call recorded into a HIP graph replays correctly any number of
 * times (tests/test_zz_no_alloc.py captures one call and replays it on changed inputs).  The FIRST call on
 * a device resolves the array's address (hipGetSymbolAddress) and the kernel's launch attributes: make
 * one eager call per device before capturing.
 * Limit: (M/256)*(N/256) <= CLIP_NOALLOC_MAX_TILES, else CLIP_ERR_CAPACITY.  All calls on one GPU share
 * that GPU's array: calls that overlap in time on one GPU (two streams, two threads, two graphs in
 * flight) race on it — serialise them; calls on different GPUs are independent.  Runs on the current device. */
#define CLIP_NOALLOC_MAX_TILES 2048
int clip_gemm_bf16_lnout_noalloc(const uint16_t* dev_A, const uint16_t* dev_W, const float* dev_bias,
                                 const uint16_t* dev_res16, int32_t res_tiled, const float* dev_gamma,
                                 const float* dev_beta, float eps, uint16_t* dev_x_out, uint16_t* dev_xres_out,
                                 int32_t* dev_err, int32_t M, int32_t N, int32_t K, int32_t lda, int32_t ldw,
                                 int32_t ldo, int32_t ldres, void* stream);
/* fp32 check mode of the same GEMM kernel: fp32 operands, residual and output, exact-fp32 MFMA
 * (v_mfma_f32_16x16x4_f32 = a k-ordered fmaf chain).  K a multiple of 32. */
int clip_gemm_f32(const float* dev_A, const float* dev_W, const float* dev_bias,
                  const float* dev_res, float* dev_out, int32_t M, int32_t N, int32_t K,
                  int32_t lda, int32_t ldw, int32_t ldo, int32_t ldres, int32_t epi, void* stream);
/* softmax(q k^T) v per packed sequence and head (modeling_bert.py:111-136), q pre-scaled;
 * qkv bf16 [T, 3*hidden], ctx bf16 [T, hidden], head_dim 64. */
int clip_attention_varlen(const uint16_t* dev_qkv, const int32_t* dev_cu_seqlens,
                          uint16_t* dev_ctx, int32_t n_seqs, int32_t max_seqlen, int32_t n_heads,
                          int32_t hidden, void* stream);
/* the same on fp16 q/k/v and ctx (k_f16 kernel set) */
int clip_attention_varlen_f16(const uint16_t* dev_qkv, const int32_t* dev_cu_seqlens,
                              uint16_t* dev_ctx, int32_t n_seqs, int32_t max_seqlen, int32_t n_heads,
                              int32_t hidden, void* stream);
/* out_bf16[t] = LayerNorm(x_f32[t]) (modeling_bert.py:292,350) */
int clip_layernorm(const float* dev_x, const float* dev_gamma, const float* dev_beta, float eps,
                   uint16_t* dev_out, int32_t T, int32_t H, void* stream);
/* the same, also writing dev_stats[t] = (mean, rstd) for clip_gemm_bf16_lnres consumers */
int clip_layernorm_stats(const float* dev_x, const float* dev_gamma, const float* dev_beta, float eps,
                         uint16_t* dev_out, float* dev_stats, int32_t T, int32_t H, void* stream);
/* BertEmbeddings.forward (modeling_bert.py:68-108): tables fp32, out bf16 [T,H] */
int clip_embed_layernorm(const int32_t* dev_ids, const int32_t* dev_type_ids,
                         const int32_t* dev_pos_ids, const float* dev_word, const float* dev_pos,
                         const float* dev_type, const float* dev_gamma, const float* dev_beta,
                         float eps, uint16_t* dev_out, int32_t T, int32_t H, int32_t vocab,
                         int32_t max_pos, int32_t type_vocab, void* stream);

/* The reference's heads read ONE hidden row per sentence (bert_model.py:52-58, :234).  With the
 * switch on (default) the last layer computes attention, both dense blocks and both LayerNorms for
 * that row only (M = n_seqs instead of total_tokens); off = every token through every layer, as
 * transformers BertModel does.  Same result up to rounding (tests compare both). */
int clip_set_trim_last_layer(clip_engine* e, int32_t on);

/* The bf16 setting fuses each LayerNorm into the GEMM that feeds it when hidden_size is a multiple of
 * 256 (default on): the column-tile workgroups of a 256-row panel exchange per-row sums through
 * device memory and write the LayerNorm output themselves, as the bf16 GEMM operand and as an fp16
 * residual copy (clip_gemm_bf16_lnout).  Off = GEMM -> fp32 pre-LayerNorm rows -> LayerNorm kernel,
 * the residual recomputed in fp32; same result to within bf16 rounding (tests compare both).  The
 * choice never depends on the batch, so a row's logits do not either. */
int clip_set_fused_layernorm(clip_engine* e, int32_t on);
/* Packed tokens per forward call that fill the GPU in whole rounds of the fused-LayerNorm GEMMs
 * (<= max_tokens; = max_tokens when that flow is not in use).  The bulk driver sizes its steps by it. */
int clip_preferred_step_tokens(clip_engine* e, int32_t* tokens);
/* Device-side error word of the engine since the last poll (read behind the latest forward on that
 * forward's stream, then cleared):
 *   bit 0 (1) = clip_forward_padded only: a row did not hold exactly 2*n_ctx+1 separators (the reference
 *               prints and fails in its classifier: bert_model.py:51-55,91);
 *   bit 1 (2) = a fused-LayerNorm tile's partner statistics did not arrive within the spin bound (a GPU
 *               shared with work that kept a workgroup from being scheduled; the fused flow needs its
 *               3 column-tile workgroups co-resident).  Sticky on the device: while it is set no later
 *               tile waits, so a void job ends quickly;
 *   bit 2 (4) = the row table of a forward was inconsistent (cu_seqlens[0] != 0, a row of < 1 or
 *               > max_seqlen tokens, cu_seqlens[n_seqs] != total_tokens);
 *   bit 3 (8) = a forward produced a non-finite logit (an fp16 activation beyond +-65504 in the F16 / F16R
 *               settings, a NaN weight): `score > threshold` is False for NaN, so without this bit the
 *               sentence would silently be missing from the output files.
 * While the word is non-zero every clip_forward_packed writes NaN logits: results of those calls are
 * void whether or not the caller polls. */
int clip_poll_errors(clip_engine* e, int32_t* host_flags);

/* HIP-event timing of the kernels inside clip_forward_packed, for bench.py's roofline figure (no
 * counterpart in the reference, which has no profiling: SURVEY.md 5).  Bit k of kind_mask turns
 * kind k on; events are recorded on the forward's stream around each launch of that kind.
 * clip_profile_read() waits for the recorded events and returns summed milliseconds and launch
 * counts per kind (arrays of CLIP_N_KINDS). */
enum {
  CLIP_KIND_EMBED_LN = 0, CLIP_KIND_GEMM_QKV = 1, CLIP_KIND_ATTENTION = 2,
  CLIP_KIND_GEMM_ATTN_OUT = 3, CLIP_KIND_LAYERNORM = 4, CLIP_KIND_GEMM_FFN_UP = 5,
  CLIP_KIND_GEMM_FFN_DOWN = 6, CLIP_KIND_HEAD = 7, CLIP_KIND_LAST_LAYER_ROWS = 8, CLIP_N_KINDS = 9
};
int clip_profile_enable(clip_engine* e, uint32_t kind_mask);
int clip_profile_read(clip_engine* e, double* ms_per_kind, int64_t* launches_per_kind, int32_t reset);

/* Sustained MFMA peak of the current device (no counterpart in the reference; SURVEY.md 8d: measure the
 * peak before quoting a fraction of it): a register-only v_mfma_f32_16x16x32 loop on random operands of
 * type `operand` (CLIP_PRECISION_BF16 or CLIP_PRECISION_F16), one 8-wave workgroup per CU (2 waves per
 * SIMD), `iters` x 16 MFMAs per wave (12000 iters ~ 3 ms), launched `repeats` times after one warm-up
 * launch on the null stream.  Returns the best and the mean TFLOP/s and the mean launch time. */
int clip_mfma_peak(int32_t operand, int32_t iters, int32_t repeats, double* tflops_best,
                   double* tflops_mean, double* ms_mean);

/* message of the last failing call on this thread ("" if none) */
const char* clip_last_error(void);
/* ABI version of this header */
int clip_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* CLIP_AMD_H */
