// C-ABI entry points of the token log probabilities
// (include/flint/flint_logprobs.h): a Checker chain and the launches of
// kernels/logprobs.hip.
#include <cmath>

#include "common/args.h"
#include "flint/flint_logprobs.h"
#include "kernels/kernels.h"

namespace {

using flint::Checker;
using flint::Span;

Checker& logprobs_sizes(Checker& c, float scale, size_t rows, size_t vocab, size_t cols) {
    return c
        .require(cols != 0 && cols % 8 == 0 && cols <= flint::kCrossEntropyMaxCols,
                 "cols (%zu) must be a multiple of 8 from 8 to %zu", cols,
                 flint::kCrossEntropyMaxCols)
        .require(vocab != 0 && vocab <= cols, "vocab (%zu) must be from 1 to cols (%zu)", vocab,
                 cols)
        .require(rows <= flint::kCrossEntropyMaxRows, "rows (%zu) can be up to %zu", rows,
                 flint::kCrossEntropyMaxRows)
        .require(std::isfinite(scale) && scale > 0.0f, "scale (%g) must be positive and finite",
                 double(scale));
}

}  // namespace

extern "C" {

FLINT_API flint_status flint_logprobs_forward(void* logprob, void* entropy, void* stats,
                                              void* top_ids, void* top_logprobs,
                                              const void* logits, const void* targets, float scale,
                                              size_t rows, size_t vocab, size_t cols, size_t top,
                                              flint_stream stream) {
    Checker c("flint_logprobs_forward");
    logprobs_sizes(c, scale, rows, vocab, cols)
        .require(top <= flint::kLogprobsMaxTop && top <= vocab,
                 "top (%zu) can be up to %zu and up to vocab (%zu)", top, flint::kLogprobsMaxTop,
                 vocab);
    if (!c.ok() || rows == 0) return c.status();
    const Span spans[] = {{"logprob", logprob, rows * 4},
                          {"entropy", entropy, rows * 4},
                          {"stats", stats, rows * 8},
                          {"logits", logits, rows * cols * 2},
                          {"targets", targets, rows * 2},
                          {"top_ids", top_ids, rows * top * 4},
                          {"top_logprobs", top_logprobs, rows * top * 4}};
    if (top == 0) {
        c.buffers(spans, 5, 3);
    } else {
        const Span all[] = {spans[0], spans[1], spans[2], spans[5], spans[6], spans[3], spans[4]};
        c.buffers(all, 7, 5);
    }
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_logprobs_forward(logprob, entropy, stats, top_ids, top_logprobs,
                                                   logits, targets, scale, rows, vocab, cols, top,
                                                   flint::to_hip(stream)));
    return FLINT_OK;
}

FLINT_API flint_status flint_logprobs_backward(void* dlogits, const void* dlogprob,
                                               const void* dentropy, const void* logits,
                                               const void* targets, const void* entropy,
                                               const void* stats, float scale, size_t rows,
                                               size_t vocab, size_t cols, flint_stream stream) {
    Checker c("flint_logprobs_backward");
    if (!logprobs_sizes(c, scale, rows, vocab, cols).ok() || rows == 0) return c.status();
    const Span out{"dlogits", dlogits, rows * cols * 2};
    const Span in{"logits", logits, rows * cols * 2};
    c.buffers({out,
               {"dlogprob", dlogprob, rows * 4},
               {"targets", targets, rows * 2},
               {"stats", stats, rows * 8}},
              1);
    if (dentropy != nullptr)
        c.buffers({out, {"dentropy", dentropy, rows * 4}, {"entropy", entropy, rows * 4}}, 1);
    // In place is the one overlap allowed: a value is read before its
    // gradient is written there.
    if (dlogits == logits) c.buffers({in}, 0);
    else c.buffers({out, in}, 1);
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_logprobs_backward(dlogits, dlogprob, dentropy, logits, targets,
                                                    dentropy == nullptr ? nullptr : entropy, stats,
                                                    scale, rows, vocab, cols,
                                                    flint::to_hip(stream)));
    return FLINT_OK;
}

}  // extern "C"
