/*
 * rac_llm.h — attention over packed prompts and over trees of drafted tokens,
 * and log probabilities of given tokens, in librac_amd.so (MI355X, gfx950).
 * No counterpart in the reference, whose attention (rac.h:323-335) takes one
 * length for a batch and equal heads, and whose decoder
 * (bench/bench_rac_transformer.c:557-616) one new token a step.
 *
 * Conventions of rac_ext.h: device buffers, work enqueued on `stream`, which
 * belongs to the current device; 0 or a negative RAC_ERR_* code (message in
 * rac_last_error()), arguments checked before any device work.  dtype: 0 fp32,
 * 1 bf16, 2 fp16, the type of every `void *` tensor of the call; sums, softmax
 * statistics and the float outputs are fp32.  Products run on the matrix cores
 * (the FAST MAC) and exponentials on the hardware's 2^x: the CORDIC iteration
 * and mode knobs have no part here.
 *
 * Strides count elements; d_head values of a head are contiguous.  Rows that
 * start on 16-byte boundaries and whose d_head is a multiple of 16 bytes are
 * read 16 bytes at a time, others value by value, with the same results.
 * Outputs and workspaces overlap no input.
 */
#ifndef RAC_LLM_H
#define RAC_LLM_H

#ifdef __cplusplus
extern "C" {
#endif

/* Largest d_head, and tokens of a tree, and alternatives of a row. */
#define RAC_LLM_MAX_HEAD 256
#define RAC_TREE_MAX_TOKENS 256
#define RAC_LOGPROB_MAX_TOP 64

/* Causal attention within each of n_seqs sequences packed one behind the
 * other: sequence i is rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1 of `total`
 * (n_seqs + 1 non-decreasing ints in [0, total], in device memory; a sequence
 * may be empty).  q [total, n_heads, d_head], k and v [total, n_kv_heads,
 * d_head] with element strides per row and per head; query head h reads key /
 * value head h / (n_heads / n_kv_heads).  out[t, h] = sum_{j <= t} p_j v_j,
 * p = softmax(scale q_t . k_j), contiguous [total, n_heads, d_head]; lse
 * [n_heads, total] (may be null) receives log sum_j exp(scale q_t . k_j), out_lo
 * (out's shape and type, may be null; the 16-bit types) what the rounding of out
 * took away, for the backward pass.
 * Rows of out outside every sequence become 0 with zero_rest and stay as they
 * are without; their lse stays as it is.  A row whose scores are all -inf gives
 * 0; values at positions a row does not see never reach it, NaN included.
 * scale > 0; total <= 2^30 and (total / 32 + n_seqs + 2) * n_heads < 2^24. */
int rac_packed_attention_dev(const void *q, const void *k, const void *v, void *out, void *out_lo, float *lse,
                             const int *cu_seqlens, int n_seqs, int total, int n_heads, int n_kv_heads, int d_head,
                             long q_stride, long q_head_stride, long k_stride, long k_head_stride, long v_stride,
                             long v_head_stride, float scale, int zero_rest, int dtype, void *stream);

/* Its gradients: grad_out, out, dq [total, n_heads, d_head], dk and dv [total,
 * n_kv_heads, d_head] contiguous, lse and out_lo (may
 * be null: the gradients of q and k are then about half again as far off in the
 * 16-bit types) as the forward pass left them.  dk and dv
 * are sums over the query heads that share a head, taken in a fixed order: the
 * same call gives the same bits.  workspace:
 * rac_packed_attention_backward_workspace_bytes bytes on a 16-byte boundary, the
 * call's own while it runs. */
long rac_packed_attention_backward_workspace_bytes(int n_seqs, int total, int n_heads, int n_kv_heads, int d_head);
int rac_packed_attention_backward_dev(const void *q, const void *k, const void *v, const void *out,
                                      const void *out_lo, const void *grad_out, const float *lse, const int *cu_seqlens, void *dq,
                                      void *dk, void *dv, float *workspace, int n_seqs, int total, int n_heads,
                                      int n_kv_heads, int d_head, long q_stride, long q_head_stride, long k_stride,
                                      long k_head_stride, long v_stride, long v_head_stride, float scale,
                                      int zero_rest, int dtype, void *stream);

/* Attention of `tokens` drafted tokens of each of `batch` sequences over their
 * caches.  Sequence b's cache holds lengths[b] tokens, and at the next
 * positions, lengths[b] + t, the keys and values of its drafted tokens, which
 * form a tree: token t continues token parents[b * parents_stride + t] < t, or
 * the cache itself (-1; any value not below t counts as -1).  A token sees the
 * cache, its ancestors and itself.  q [batch, tokens, n_heads, d_head], caches
 * [batch, n_kv_heads, t_cap, d_head], element strides; out contiguous [batch,
 * tokens, n_heads, d_head].  lengths and parents (ints) are read when the
 * kernels run, so a recorded graph replays with new ones.  A sequence whose
 * lengths[b] is not in [0, t_cap - tokens] gives NaN and reads no cache.
 * parents_stride 0: one tree for all.  1 <= tokens <= 256; batch * n_kv_heads
 * <= 65535, and times the 32-row blocks of a key head's queries below 2^24 -
 * 4096.  workspace: rac_tree_attention_workspace_bytes bytes (null when
 * that is 0), the call's own while it runs. */
long rac_tree_attention_workspace_bytes(int batch, int tokens, int n_heads, int n_kv_heads, int d_head, long t_cap,
                                        int dtype);
int rac_tree_attention_dev(const void *q, const void *k_cache, const void *v_cache, void *out, const int *lengths,
                           const int *parents, float *workspace, int batch, int tokens, int n_heads, int n_kv_heads,
                           int d_head, long t_cap, long parents_stride, long q_stride_b, long q_stride_t,
                           long q_stride_h, long k_stride_b, long k_stride_h, long k_stride_t, long v_stride_b,
                           long v_stride_h, long v_stride_t, float scale, int dtype, void *stream);

/* Of each row of logits [rows, vocab] (row_stride elements apart):
 * logprob[r] = log softmax(x)_token, entropy[r] = -sum p log p, lse[r] (may be
 * null) = log sum exp x, and, with top > 0, the `top` likeliest tokens, best
 * first and equal logits by the lower token (NaN counts as -inf), with their
 * log probabilities [rows, top].  tokens (64-bit): a negative one stands for
 * none (logprob 0), one >= vocab gives NaN.  A row of nothing but -inf has log
 * probabilities -inf and entropy 0; NaN or +inf in a row makes its results NaN.
 * rows < 2^24, vocab < 2^31 - 64; top <= min(64, vocab).  workspace:
 * rac_token_logprobs_workspace_bytes bytes (null when that is 0). */
long rac_token_logprobs_workspace_bytes(long rows, long vocab, int top, int dtype);
int rac_token_logprobs_dev(const void *logits, long row_stride, const long *tokens, float *logprob, float *entropy,
                           float *lse, float *top_logprob, long *top_token, float *workspace, long rows, long vocab,
                           int top, int dtype, void *stream);

/* grad_logits [rows, vocab] (contiguous, the logits' type) =
 *   grad_logprob ([j = token] - p_j) - grad_entropy p_j (log p_j + entropy),
 * from the forward pass's lse and entropy; grad_logprob or grad_entropy (not
 * both) may be null.  A row without a token has no grad_logprob part. */
int rac_token_logprobs_backward_dev(const void *logits, long row_stride, const long *tokens, const float *lse,
                                    const float *entropy, const float *grad_logprob, const float *grad_entropy,
                                    void *grad_logits, long rows, long vocab, int dtype, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RAC_LLM_H */
