/* libflint: the gated feed-forward product, forward and backward.
 *
 * No counterpart in the reference's ABI (GPT-2's MLP is not gated): additive entry
 * points beside flint_gemm_nt_bias_gelu and flint_gemm_nn_dgelu.
 *
 * A gated block of width k and n hidden values is h = act(x w_gate^T) * (x
 * w_up^T), out = h w_down^T. w holds both projections, 2n x k: rows 0 .. n - 1 the
 * gate's, n .. 2n - 1 the up's. Forward: flint_gemm_nt_gated, then flint_gemm_nt with
 * w_down (k x n). Backward, from dout:
 *   dpre = flint_gemm_nn_dgated(dout, w_down, pre);
 *   dw_down = flint_gemm_tn(dout, h), dx = flint_gemm_nn(dpre, w),
 *   dw = flint_gemm_tn(dpre, x), dbias = flint_bias_gradient(dpre).
 *
 * Conventions and limits are flint.h's GEMM functions'; n is a multiple of 8, and
 * m n up to 2^34. m or n of 0 is a no-op that checks nothing. */
#ifndef FLINT_FLINT_GATED_H
#define FLINT_FLINT_GATED_H

#include "flint/flint.h"

#ifdef __cplusplus
extern "C" {
#endif

/* act: s / (1 + exp(-s)), or GPT-2's tanh GELU. */
enum { FLINT_GATE_SILU = 0, FLINT_GATE_GELU = 1 };

/* s = x(m x k) w(2n x k)^T + bias (2n FP32, or null for none) in FP32; y(m x n) =
 * RN16(act(s[:, :n]) s[:, n:]); pre(m x 2n) = RN16(s), or null: not kept. k a positive
 * multiple of 8. act(-inf) is NaN. */
FLINT_API flint_status flint_gemm_nt_gated(void* y, void* pre, const void* x, const void* w,
                                           const void* bias, size_t m, size_t n, size_t k,
                                           int activation, flint_stream stream);

/* s = x(m x k) w(k x n) in FP32, the gradient of y; dpre(m x 2n) = RN16(s u act'(g))
 * then RN16(s act(g)), g = pre[:, :n] and u = pre[:, n:]. act and act' are 0 at -inf
 * and act' is 1 at +inf (pre may have overflowed FP16); NaN at NaN. */
FLINT_API flint_status flint_gemm_nn_dgated(void* dpre, const void* x, const void* w,
                                            const void* pre, size_t m, size_t n, size_t k,
                                            int activation, flint_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* FLINT_FLINT_GATED_H */
