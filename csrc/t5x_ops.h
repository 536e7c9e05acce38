/* Entry points that the compiled host path (host/host_ops.cpp) calls beside those of t5x_b200.h. The
 * sources that define them include this file too, so that a changed argument list does not
 * compile on one side only. */
#ifndef T5X_OPS_H_
#define T5X_OPS_H_

#ifdef __cplusplus
extern "C" {
#endif

int t5x_rmsnorm_fwd(const void* x, const void* scale, void* y, void* rstd, int rows, int d, float eps,
                    void* stream);
long long t5x_rmsnorm_bwd_partial(int rows, int d);
int t5x_rmsnorm_bwd(const void* dy, const void* x, const void* scale, const void* rstd,
                    const void* dres, void* dx, void* dscale, void* partial, int rows, int d,
                    void* stream);
int t5x_attention_fwd(const void* q, const void* k, const void* v, void* o, void* lse, int B, int H,
                      int Lq, int Lk, long long q_sb, long long q_sl, long long q_sh, long long k_sb,
                      long long k_sl, long long k_sh, long long v_sb, long long v_sl, long long v_sh,
                      long long o_sb, long long o_sl, long long o_sh, const void* rel_bias,
                      const void* rel_bucket, int num_buckets, int nrel, int rel_off,
                      const void* key_mask, const void* q_seg, const void* kv_seg, int causal,
                      int causal_off, void* stream);
int t5x_attention_fwd_few(const void* q, const void* k, const void* v, void* o, void* lse, int B, int H,
                          int Lq, int Lk, long long q_sb, long long q_sl, long long q_sh, long long k_sb,
                          long long k_sl, long long k_sh, long long v_sb, long long v_sl, long long v_sh,
                          long long o_sb, long long o_sl, long long o_sh, const void* rel_bias,
                          const void* rel_bucket, int num_buckets, int nrel, int rel_off,
                          const void* key_mask, const void* q_seg, const void* kv_seg, int causal,
                          int causal_off, void* stream);
int t5x_attention_fwd_stream(const void* q, const void* k, const void* v, void* o, void* lse, int B,
                             int H, int Lq, int Lk, int D, long long q_sb, long long q_sl,
                             long long q_sh, long long k_sb, long long k_sl, long long k_sh,
                             long long v_sb, long long v_sl, long long v_sh, long long o_sb,
                             long long o_sl, long long o_sh, const void* rel_bias,
                             const void* rel_bucket, int num_buckets, int nrel, int rel_off,
                             const void* key_mask, const void* q_seg, const void* kv_seg, int causal,
                             int causal_off, void* stream);
int t5x_attention_bwd(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                      const void* lse, void* delta, void* dq_f32, void* dk, void* dv, int B, int H,
                      int Lq, int Lk, int D, long long q_sb, long long q_sl, long long q_sh,
                      long long k_sb, long long k_sl, long long k_sh, long long v_sb, long long v_sl,
                      long long v_sh, long long o_sb, long long o_sl, long long o_sh, long long do_sb,
                      long long do_sl, long long do_sh, long long dk_sb, long long dk_sl,
                      long long dk_sh, const void* rel_bias, const void* rel_bucket, void* d_rel_bias,
                      int num_buckets, int nrel, int rel_off, const void* key_mask, const void* q_seg,
                      const void* kv_seg, int causal, int causal_off, void* stream);
int t5x_attention_bwd_head_covers(int B, int H, int Lq, int Lk, int D, int num_buckets);
int t5x_attention_bwd_head(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                           const void* lse, void* dq, void* dk, void* dv, void* dk32, void* dv32, int B,
                           int H, int Lq, int Lk, long long q_sb, long long q_sl, long long q_sh,
                           long long k_sb, long long k_sl, long long k_sh, long long v_sb, long long v_sl,
                           long long v_sh, long long o_sb, long long o_sl, long long o_sh, long long do_sb,
                           long long do_sl, long long do_sh, long long dq_sb, long long dq_sl, long long dq_sh,
                           long long dk_sb, long long dk_sl, long long dk_sh, const void* rel_bias,
                           const void* rel_bucket, void* d_rel_bias, int num_buckets, int nrel,
                           int rel_off, const void* key_mask, const void* q_seg, const void* kv_seg,
                           int causal, int causal_off, void* stream);
int t5x_gemm_gated_grad_covers(int M, int N);
int t5x_gemm_relu_covers(int M, int N);
int t5x_gemm_relu(const void* A, const void* B, void* C, const void* positive, int M, int N, int K, long long lda,
                  long long ldb, long long ldc, long long ldp, int b_mn_major, void* stream);
int t5x_gemm_gated_grad(const void* dy, const void* B, void* h0, void* h1, int M, int N, int K, long long ld_dy,
                        long long ldb, long long ldh, int b_mn_major, void* stream);
int t5x_gated_gelu_bwd(void* dg, void* h, long long rows, int dff, long long ldh, long long ldg,
                       int write_g, void* stream);

/* One parameter of t5x_adamw_group: n fp32 values p and gradients g, the moments mu and nu (fp32, or
 * e4m3 codes with the largest magnitude of each 256 values in mu_absmax / nu_absmax), and the bf16
 * working copy or null. No two items may share memory. */
typedef struct {
  void* p;
  const void* g;
  void* mu;
  void* nu;
  void* out;
  void* mu_absmax;
  void* nu_absmax;
  long long n;
} t5x_adamw_item;
/* One AdamW step of all items. state_bits: 32 or 8 (seed: of the rounding). step >= 1 is the count after
 * this update. clip_scale: device float that multiplies the gradients, or null. */
int t5x_adamw_group(const t5x_adamw_item* items, int count, int state_bits, float lr, double b1, double b2,
                    float eps, float eps_root, float weight_decay, int step, unsigned int seed,
                    const void* clip_scale, void* stream);
/* *clip_scale = min(1, max_norm / (norm + 1e-16)), norm over the items' gradients (the other pointers
 * are not read). scratch: t5x_grad_clip_scratch_bytes bytes, 8-byte aligned. */
long long t5x_grad_clip_scratch_bytes(const t5x_adamw_item* items, int count);
int t5x_grad_clip_scale(const t5x_adamw_item* items, int count, void* scratch, float max_norm,
                        void* clip_scale, void* stream);

/* Losses over logits [batch, length, vocab] (fp32 or bf16; strides in values, last dimension contiguous)
 * with their gradient in `grad` (of the strides of t5x_loss_gradient_strides, that is the logits' own where their
 * rows lie side by side, and at the same place of 16 bytes; or null), and over
 * log-probabilities [batch, length] (fp32) with theirs in `slope` (or null): see token_losses.cu.
 * targets int64, weights fp32 (or null: all 1), other inputs fp32. normalizer: device scalar that divides
 * the loss, or null: `scale` multiplies it. scratch: the stated bytes, 16-byte aligned. policy: out = loss,
 * kl, clipped, weight. preference: scores [batch], margins [batch / 2], out = loss, pairs. */
/* strides: of batch and length */
void t5x_loss_gradient_strides(int length, int vocab, int fp32, long long stride_b, long long stride_t,
                               long long* strides);
long long t5x_policy_loss_scratch_bytes();
int t5x_policy_loss(const void* logits, int fp32, void* grad, long long batch, int length, int vocab,
                    long long stride_b, long long stride_t, const void* targets, const void* weights,
                    const void* old_scores, const void* ref_scores, const void* advantages, long long adv_b,
                    long long adv_t, float clip_low, float clip_high, float kl_weight, float scale,
                    const void* normalizer, void* scratch, void* out, void* stream);
int t5x_policy_loss_tokens(const void* logp, void* slope, long long batch, int length, const void* weights,
                           const void* old_scores, const void* ref_scores, const void* advantages,
                           long long adv_b, long long adv_t, float clip_low, float clip_high, float kl_weight,
                           float scale, const void* normalizer, void* scratch, void* out, void* stream);
long long t5x_preference_loss_scratch_bytes(long long batch, int length, int vocab, int fp32);
int t5x_preference_loss(const void* logits, int fp32, void* grad, long long batch, int length, int vocab,
                        long long stride_b, long long stride_t, const void* targets, const void* weights,
                        const void* reference, float beta, float smoothing, float scale, const void* normalizer,
                        void* scratch, void* scores, void* margins, void* out, void* stream);
int t5x_preference_loss_tokens(const void* logp, void* slope, long long batch, int length, const void* weights,
                               const void* reference, float beta, float smoothing, float scale,
                               const void* normalizer, void* scratch, void* scores, void* margins, void* out,
                               void* stream);
/* dst = src * *factor (dst may be src; nothing is done where the factor is 1 then) */
int t5x_scale_gradient(const void* src, void* dst, long long n, int fp32, const void* factor, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* T5X_OPS_H_ */
