/* mogt_lm_loss.h — C ABI of the post-training losses of libmogt_scan.so:
 * label log-probabilities of logits rows, the clipped policy loss with a KL
 * term, and the paired preference loss, each with its gradient.
 *
 * Conventions are those of mogt_scan.h.  logits are [B, L, V] with batch and
 * row strides in elements and dense rows, of MOGT_DTYPE_F32, _BF16 or _F16;
 * dlogits likewise with strides of its own.  labels int64 [B, L]; mask uint8
 * [B, L] (nonzero = the token counts) or NULL.  A token counts when its mask
 * is set and its label is not negative; rows that do not count are never read,
 * their log-probability and loss are 0 and their gradient rows are zero.  A
 * counting label >= V gives NaN.  Statistics are f32; the sums over tokens and
 * pairs are f64, in a fixed order.
 *
 * The reference's only loss is cross-entropy (chunked_lm_loss.py:5-80); these
 * have no counterpart there.
 */
#ifndef MOGT_LM_LOSS_H_
#define MOGT_LM_LOSS_H_

#include "mogt_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* logprobs[r] = logits[r, label] - log sum exp(logits[r]).  stats [B, L, 2] (or
 * NULL) receives the row's maximum m and s = sum exp(logits[r] - m), which
 * mogt_logprob_bwd takes (log sum exp alone would lose the bits that
 * exp(logit - m) needs when the logits are large). */
int mogt_logprob_fwd(const void* logits, int64_t sb, int64_t sl, const int64_t* labels,
                     const uint8_t* mask, int64_t B, int64_t L, int64_t V, int dtype,
                     float* logprobs, float* stats, void* stream);
/* dlogits[r] = coef[r / coef_div] * (onehot(label) - softmax(logits[r])),
 * coef f32, times *scale when scale is not NULL.  unless_one: leave dlogits as
 * it is when *scale is 1 (read on the device). */
int mogt_logprob_bwd(const void* logits, int64_t sb, int64_t sl, const int64_t* labels,
                     const uint8_t* mask, const float* stats, const float* coef, int64_t coef_div,
                     const float* scale, int unless_one, void* dlogits, int64_t d_sb,
                     int64_t d_sl, int64_t B, int64_t L, int64_t V, int dtype, void* stream);

/* Clipped policy loss over the n counting tokens, lp = their log-probability,
 * r = exp(lp - old), d = ref - lp:
 *   loss = 1/max(n, 1) sum [ -min(r adv, clip(r, 1-clip_low, 1+clip_high) adv)
 *                            + kl_coef (exp(d) - d - 1) ]
 * adv[b * adv_sb + l * adv_sl]; old, ref (or NULL) f32 [B, L] dense.
 * Writes loss (one f32), logprobs, stats, coef ([B, L], d loss / d lp), and,
 * when dlogits is not NULL, coef * (onehot - softmax) in the same pass over
 * the logits.  scratch: mogt_policy_loss_scratch_bytes(B, L). */
size_t mogt_policy_loss_scratch_bytes(int64_t B, int64_t L);
int mogt_policy_loss(const void* logits, int64_t sb, int64_t sl, const int64_t* labels,
                     const uint8_t* mask, const float* old_logprobs, const float* ref_logprobs,
                     const float* adv, int64_t adv_sb, int64_t adv_sl, float clip_low,
                     float clip_high, float kl_coef, float* loss, float* logprobs, float* stats,
                     float* coef, void* dlogits, int64_t d_sb, int64_t d_sl, int64_t B, int64_t L,
                     int64_t V, int dtype, void* scratch, size_t scratch_bytes, void* stream);

/* Paired preference loss from per-token log-probabilities [2P, L] (sequences
 * 0..P-1 preferred over P..2P-1): s = their sums over each sequence,
 *   x_p = beta ((s_p - ref_p) - (s_{P+p} - ref_{P+p}))
 *   loss = mean_p [ -(1 - eps) log sigmoid(x_p) - eps log sigmoid(-x_p) ]
 * Writes loss, seq (the sums) and coef[2P] = d loss / d s.  logit gradients:
 * mogt_logprob_bwd with coef_div = L. */
int mogt_preference_pairs(const float* logprobs, const float* ref, int64_t P, int64_t L, float beta,
                          float eps, float* loss, float* seq, float* coef, void* stream);
/* The same with reference sums in f64: at a sum of -30000 one unit of f32 is
 * 2e-3, far more than the kernel's own f64 sums are off. */
int mogt_preference_pairs_f64(const float* logprobs, const double* ref, int64_t P, int64_t L,
                              float beta, float eps, float* loss, float* seq, float* coef,
                              void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MOGT_LM_LOSS_H_ */
