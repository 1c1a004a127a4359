// C-ABI entry points of the rotary positions (include/flint/flint_rotary.h): a
// Checker chain and the launches of kernels/rotary.hip.
#include <cmath>

#include "common/args.h"
#include "flint/flint_rotary.h"
#include "kernels/kernels.h"

namespace {

using flint::Checker;
using flint::Span;
using flint::View;

Checker& rotary_width(Checker& c, size_t width) {
    return c.require(width != 0 && width % 2 == 0 && width <= flint::kRotaryMaxWidth,
                     "width (%zu) must be even, from 2 to %zu", width, flint::kRotaryMaxWidth);
}

Checker& rotary_sizes(Checker& c, const flint_rotary_shape* s) {
    if (!c.require(s != nullptr, "shape is null").ok()) return c;
    c.require(s->head_width != 0 && s->head_width % 8 == 0 &&
                  s->head_width <= flint::kRotaryMaxWidth,
              "head_width (%zu) must be a multiple of 8 from 8 to %zu", s->head_width,
              flint::kRotaryMaxWidth);
    rotary_width(c, s->width)
        .require(s->width <= s->head_width, "width (%zu) can be up to head_width (%zu)", s->width,
                 s->head_width)
        .require(s->layout == FLINT_ROTARY_HALVES || s->layout == FLINT_ROTARY_PAIRS,
                 "layout (%d) must be 0 or 1", s->layout)
        .require(s->tokens <= flint::kPackedMaxTokens, "tokens (%zu) can be up to %zu", s->tokens,
                 flint::kPackedMaxTokens)
        .require(s->heads <= flint::kHeadsMax, "heads (%zu) can be up to %zu", s->heads,
                 flint::kHeadsMax)
        .require(s->kv_heads <= flint::kHeadsMax, "kv_heads (%zu) can be up to %zu", s->kv_heads,
                 flint::kHeadsMax);
    const struct {
        const char* name;
        size_t stride, heads;
    } strides[] = {{"q_stride", s->q_stride, s->heads},
                   {"k_stride", s->k_stride, s->kv_heads},
                   {"q_out_stride", s->q_out_stride, s->heads},
                   {"k_out_stride", s->k_out_stride, s->kv_heads}};
    for (const auto& t : strides) {
        const size_t least = t.heads * s->head_width;
        c.require(t.heads == 0 ||
                      (t.stride % 8 == 0 && t.stride >= least && t.stride <= flint::kStrideMax),
                  "%s (%zu) must be a multiple of 8 from %zu to %zu", t.name, t.stride, least,
                  flint::kStrideMax);
    }
    return c;
}

}  // namespace

extern "C" {

FLINT_API flint_status flint_rotary_plan_bytes(size_t width, size_t* bytes) {
    Checker c("flint_rotary_plan_bytes");
    if (!rotary_width(c.require(bytes != nullptr, "bytes is null"), width).ok()) return c.status();
    *bytes = (1 + width / 2) * sizeof(double);
    return FLINT_OK;
}

FLINT_API flint_status flint_rotary_plan(void* plan, const flint_rotary_angles* angles,
                                         flint_stream stream) {
    Checker c("flint_rotary_plan");
    if (!c.require(angles != nullptr, "angles is null").ok()) return c.status();
    const flint_rotary_angles& a = *angles;
    rotary_width(c, a.width)
        .require(std::isfinite(a.base) && a.base > 1.0, "base (%g) must be finite and above 1", a.base)
        .require(std::isfinite(a.factor) && a.factor > 0.0,
                 "factor (%g) must be positive and finite", a.factor)
        .require(std::isfinite(a.original) && a.original >= 0.0,
                 "original (%g) must be 0 or positive and finite", a.original)
        .require(a.original == 0.0 || (std::isfinite(a.low) && std::isfinite(a.high) && a.low < a.high),
                 "low (%g) must be below high (%g)", a.low, a.high)
        .require(std::isfinite(a.magnitude), "magnitude (%g) must be finite", a.magnitude)
        .buffers({{"plan", plan, (1 + a.width / 2) * sizeof(double)}}, 1);
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_rotary_plan(plan, a, flint::to_hip(stream)));
    return FLINT_OK;
}

FLINT_API flint_status flint_rotary(void* q_out, void* k_out, const void* q, const void* k,
                                    const void* positions, const void* plan,
                                    const flint_rotary_shape* shape, int backward,
                                    flint_stream stream) {
    Checker c("flint_rotary");
    if (!rotary_sizes(c, shape).ok()) return c.status();
    const flint_rotary_shape& s = *shape;
    if (s.tokens == 0 || s.heads + s.kv_heads == 0) return FLINT_OK;
    const size_t qw = s.heads * s.head_width, kw = s.kv_heads * s.head_width;
    const View outs[2] = {{"q_out", q_out, s.tokens, qw, s.q_out_stride, 2},
                          {"k_out", k_out, s.tokens, kw, s.k_out_stride, 2}};
    const View ins[2] = {{"q", q, s.tokens, qw, s.q_stride, 2},
                         {"k", k, s.tokens, kw, s.k_stride, 2}};
    const View maps[2] = {{"positions", positions, 1, s.tokens, 0, 4},
                          {"plan", plan, 1, 1 + s.width / 2, 0, 8}};
    const bool used[2] = {s.heads != 0, s.kv_heads != 0};
    for (const View* both : {outs, ins})
        for (int i = 0; i < 2; ++i)
            if (used[i]) c.buffers({both[i].span()}, 0);
    c.buffers({maps[0].span(), maps[1].span()}, 0);
    if (used[0] && used[1]) c.require(!outs[0].meets(outs[1]), "q_out and k_out overlap");
    for (int i = 0; i < 2; ++i) {
        if (!used[i]) continue;
        for (int j = 0; j < 2; ++j) {
            // In place: the same rows. (An item is read whole before it is written.)
            const bool same = i == j && outs[i].at == ins[j].at && outs[i].stride == ins[j].stride;
            if (used[j])
                c.require(same || !outs[i].meets(ins[j]), "%s and %s overlap", outs[i].name,
                          ins[j].name);
        }
        for (const View& m : maps)
            c.require(!outs[i].meets(m), "%s and %s overlap", outs[i].name, m.name);
    }
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_rotary(q_out, k_out, q, k, positions, plan, s, backward != 0,
                                         flint::to_hip(stream)));
    return FLINT_OK;
}

}  // extern "C"
