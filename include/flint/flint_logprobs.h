/* libflint: log probabilities of given tokens, with each row's entropy and its
 * most likely alternatives, and the gradient of the logits.
 *
 * No counterpart in the reference's ABI (flint_softmax_cross_entropy gives the
 * loss and its gradient at once): additive entry points, for scoring, for
 * serving log probabilities, and for losses whose gradient by a token's log
 * probability is known only after the forward pass.
 *
 * logits: rows x cols FP16, of which the first vocab columns count; cols a
 * multiple of 8 up to 65,536. targets: rows uint16 values. Per row, over
 * j < vocab: x_j = scale l_j, p_j = exp(x_j) / sum exp(x). */
#ifndef FLINT_FLINT_LOGPROBS_H
#define FLINT_FLINT_LOGPROBS_H

#include "flint/flint.h"

#ifdef __cplusplus
extern "C" {
#endif

/* logprob[r] = log p_target (+0 where the target is not below vocab: a row
 * without one); entropy[r] = -sum p log p (p log p is 0 where p is). stats[r]
 * (2 FP32 values) is what the backward pass needs: the row's largest logit and
 * log(sum exp(x - its x)). top_ids and top_logprobs (rows x top, int32 and
 * FP32): the top largest logits' columns, largest first, the lower column first
 * among equal ones (-0 equals +0; NaN counts as the largest), and their log
 * probabilities; null with top 0. top up to 64 and up to vocab. scale is
 * positive and finite. A logit of -inf is a word of probability 0; a row whose
 * every logit is -inf, or that holds NaN or +inf, gives NaN. */
FLINT_API flint_status flint_logprobs_forward(void* logprob, void* entropy, void* stats,
                                              void* top_ids, void* top_logprobs,
                                              const void* logits, const void* targets, float scale,
                                              size_t rows, size_t vocab, size_t cols, size_t top,
                                              flint_stream stream);

/* dlogits (rows x cols FP16) of sum_r dlogprob[r] logprob[r] + dentropy[r]
 * entropy[r]:
 *   scale (dlogprob ([j = target] - p_j) - dentropy p_j (log p_j + entropy))
 * and +0 at j >= vocab. A row without a target takes dlogprob as 0. dentropy may
 * be null (0 everywhere), and entropy then too. stats and entropy come from the
 * forward pass on these logits and this scale. dlogits may be logits. */
FLINT_API flint_status flint_logprobs_backward(void* dlogits, const void* dlogprob,
                                               const void* dentropy, const void* logits,
                                               const void* targets, const void* entropy,
                                               const void* stats, float scale, size_t rows,
                                               size_t vocab, size_t cols, flint_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* FLINT_FLINT_LOGPROBS_H */
