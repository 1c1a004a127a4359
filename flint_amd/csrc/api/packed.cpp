// C-ABI entry points of the attention over packed sequences
// (include/flint/flint_packed.h): a Checker chain and the launches of
// kernels/packed.hip.
#include <cmath>

#include "common/args.h"
#include "flint/flint_packed.h"
#include "kernels/kernels.h"

namespace {

using flint::Checker;
using flint::View;

Checker& scale_in_range(Checker& c, float scale) {
    return c
        .require(std::isfinite(scale), "scale (%g) must be finite", double(scale))
        .require(std::fabs(scale) <= flint::kAttentionMaxScale, "scale (%g) can be up to %g in size",
                 double(scale), double(flint::kAttentionMaxScale));
}

// The shape itself; every later check reads it only once these have passed.
Checker& packed_sizes(Checker& c, const flint_packed_shape* s) {
    if (!c.require(s != nullptr, "shape is null").ok()) return c;
    c.require(s->head_width == 64 || s->head_width == 128, "head_width (%zu) must be 64 or 128",
              s->head_width)
        .require(s->heads != 0 && s->heads <= flint::kHeadsMax, "heads (%zu) must be from 1 to %zu",
                 s->heads, flint::kHeadsMax)
        .require(s->kv_heads != 0 && s->kv_heads <= s->heads && s->heads % s->kv_heads == 0,
                 "kv_heads (%zu) must divide heads (%zu)", s->kv_heads, s->heads)
        .require(s->tokens <= flint::kPackedMaxTokens, "tokens (%zu) can be up to %zu", s->tokens,
                 flint::kPackedMaxTokens)
        .require(s->sequences <= flint::kPackedMaxSequences, "sequences (%zu) can be up to %zu",
                 s->sequences, flint::kPackedMaxSequences);
    if (!c.ok()) return c;
    c.require(flint::packed_items(*s) * s->heads <= flint::kPackedMaxBlocks,
              "(tokens / 128 + sequences) x heads (%zu) can be up to %zu",
              flint::packed_items(*s) * s->heads, flint::kPackedMaxBlocks);
    const struct {
        const char* name;
        size_t stride, width;
    } strides[] = {{"q_stride", s->q_stride, s->heads * s->head_width},
                   {"kv_stride", s->kv_stride, s->kv_heads * s->head_width},
                   {"o_stride", s->o_stride, s->heads * s->head_width}};
    for (const auto& t : strides)
        c.require(t.stride % 8 == 0 && t.stride >= t.width && t.stride <= flint::kStrideMax,
                  "%s (%zu) must be a multiple of 8 from %zu to %zu", t.name, t.stride, t.width,
                  flint::kStrideMax);
    return c;
}

bool empty(const flint_packed_shape& s) { return s.tokens == 0 || s.sequences == 0; }

View q_view(const char* name, const void* at, const flint_packed_shape& s) {
    return {name, at, s.tokens, s.heads * s.head_width, s.q_stride, 2};
}
View kv_view(const char* name, const void* at, const flint_packed_shape& s) {
    return {name, at, s.tokens, s.kv_heads * s.head_width, s.kv_stride, 2};
}
View o_view(const char* name, const void* at, const flint_packed_shape& s) {
    return {name, at, s.tokens, s.heads * s.head_width, s.o_stride, 2};
}
View bytes_view(const char* name, const void* at, size_t bytes) {
    return {name, at, 1, bytes, 0, 1};
}
View lse_view(const void* at, const flint_packed_shape& s) {
    return bytes_view("lse", at, s.heads * s.tokens * 4);
}
View plan_view(const void* at, const flint_packed_shape& s) {
    return bytes_view("plan", at, flint::packed_plan_bytes(s));
}

}  // namespace

extern "C" {

FLINT_API flint_status flint_attention_packed_plan_bytes(const flint_packed_shape* shape,
                                                         size_t* bytes) {
    Checker c("flint_attention_packed_plan_bytes");
    if (!packed_sizes(c.require(bytes != nullptr, "bytes is null"), shape).ok()) return c.status();
    *bytes = flint::packed_plan_bytes(*shape);
    return FLINT_OK;
}

FLINT_API flint_status flint_attention_packed_plan(void* plan, const void* offsets,
                                                   const flint_packed_shape* shape,
                                                   flint_stream stream) {
    Checker c("flint_attention_packed_plan");
    if (!packed_sizes(c, shape).ok() || empty(*shape)) return c.status();
    c.views({plan_view(plan, *shape), bytes_view("offsets", offsets, (shape->sequences + 1) * 4)},
            1);
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_packed_plan(plan, offsets, *shape, flint::to_hip(stream)));
    return FLINT_OK;
}

FLINT_API flint_status flint_attention_packed_forward(void* o, void* lse, const void* q,
                                                      const void* k, const void* v,
                                                      const void* plan,
                                                      const flint_packed_shape* shape, float scale,
                                                      flint_stream stream) {
    Checker c("flint_attention_packed_forward");
    if (!scale_in_range(packed_sizes(c, shape), scale).ok() || empty(*shape)) return c.status();
    c.views({o_view("o", o, *shape), lse_view(lse, *shape), q_view("q", q, *shape),
             kv_view("k", k, *shape), kv_view("v", v, *shape), plan_view(plan, *shape)},
            2);
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_packed_forward(o, lse, q, k, v, plan, *shape, scale,
                                                 flint::to_hip(stream)));
    return FLINT_OK;
}

FLINT_API flint_status flint_attention_packed_backward_workspace(const flint_packed_shape* shape,
                                                                 size_t* bytes) {
    Checker c("flint_attention_packed_backward_workspace");
    if (!packed_sizes(c.require(bytes != nullptr, "bytes is null"), shape).ok()) return c.status();
    *bytes = flint::packed_backward_workspace(*shape);
    return FLINT_OK;
}

FLINT_API flint_status flint_attention_packed_backward(
    void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k, const void* v,
    const void* o, const void* lse, const void* plan, const flint_packed_shape* shape, float scale,
    void* workspace, size_t workspace_bytes, flint_stream stream) {
    Checker c("flint_attention_packed_backward");
    if (!scale_in_range(packed_sizes(c, shape), scale).ok() || empty(*shape)) return c.status();
    const flint_packed_shape& s = *shape;
    const size_t needed = flint::packed_backward_workspace(s);
    c.require(workspace_bytes >= needed, "needs %zu bytes of workspace, given %zu", needed,
              workspace_bytes)
        .views({q_view("dq", dq, s), kv_view("dk", dk, s), kv_view("dv", dv, s),
                bytes_view("workspace", workspace, needed), o_view("dout", dout, s),
                q_view("q", q, s), kv_view("k", k, s), kv_view("v", v, s), o_view("o", o, s),
                lse_view(lse, s), plan_view(plan, s)},
               4);
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_packed_backward(dq, dk, dv, dout, q, k, v, o, lse, plan, s, scale,
                                                  workspace, flint::to_hip(stream)));
    return FLINT_OK;
}

}  // extern "C"
