// C-ABI entry points of the attention over a paged cache
// (include/flint/flint_paged.h): a Checker chain and the launches of
// kernels/paged.hip.
#include <cmath>

#include "common/args.h"
#include "flint/flint_paged.h"
#include "kernels/kernels.h"

namespace {

using flint::Checker;
using flint::View;

Checker& paged_sizes(Checker& c, const flint_paged_shape* s) {
    if (!c.require(s != nullptr, "shape is null").ok()) return c;
    const size_t columns = flint::kPagedMaxPositions / (s->page_size == 0 ? 1 : s->page_size);
    c.require(s->head_width == 64 || s->head_width == 128, "head_width (%zu) must be 64 or 128",
              s->head_width)
        .require(s->heads != 0 && s->heads <= flint::kHeadsMax, "heads (%zu) must be from 1 to %zu",
                 s->heads, flint::kHeadsMax)
        .require(s->kv_heads != 0 && s->kv_heads <= s->heads && s->heads % s->kv_heads == 0,
                 "kv_heads (%zu) must divide heads (%zu)", s->kv_heads, s->heads)
        .require(s->tokens <= flint::kPagedMaxTokens, "tokens (%zu) can be up to %zu", s->tokens,
                 flint::kPagedMaxTokens)
        .require(s->sequences <= flint::kPagedMaxSequences, "sequences (%zu) can be up to %zu",
                 s->sequences, flint::kPagedMaxSequences)
        .require(s->max_new <= flint::kPagedMaxTokens, "max_new (%zu) can be up to %zu", s->max_new,
                 flint::kPagedMaxTokens)
        .require(s->page_size != 0 && s->page_size % 8 == 0 &&
                     s->page_size <= flint::kPagedMaxPageSize,
                 "page_size (%zu) must be a multiple of 8 from 8 to %zu", s->page_size,
                 flint::kPagedMaxPageSize)
        .require(s->pages != 0 && s->pages <= 0x7fffffffu, "pages (%zu) must be from 1 to %zu",
                 s->pages, size_t{0x7fffffff})
        .require(s->max_pages != 0 && s->max_pages <= columns, "max_pages (%zu) must be from 1 to %zu",
                 s->max_pages, columns);
    if (c.ok())
        c.require(s->pages <= flint::kPagedMaxPool / (s->page_size * s->kv_heads * s->head_width),
                  "pages (%zu) x page_size x kv_heads x head_width can be up to %zu", s->pages,
                  flint::kPagedMaxPool)
            .require(s->tokens * s->heads <= flint::kPagedMaxRows,
                     "tokens x heads (%zu) can be up to %zu", s->tokens * s->heads,
                     flint::kPagedMaxRows)
            .require(s->sequences * s->kv_heads <= flint::kPagedMaxRows / 8,
                     "sequences x kv_heads (%zu) can be up to %zu", s->sequences * s->kv_heads,
                     flint::kPagedMaxRows / 8);
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

bool empty(const flint_paged_shape& s) {
    return s.tokens == 0 || s.sequences == 0 || s.max_new == 0;
}

}  // namespace

extern "C" {

FLINT_API flint_status flint_attention_paged_workspace(const flint_paged_shape* shape,
                                                       size_t* bytes) {
    Checker c("flint_attention_paged_workspace");
    if (!paged_sizes(c.require(bytes != nullptr, "bytes is null"), shape).ok()) return c.status();
    *bytes = empty(*shape) ? 0 : flint::paged_workspace(*shape);
    return FLINT_OK;
}

FLINT_API flint_status flint_attention_paged(void* o, void* k_pages, void* v_pages, const void* q,
                                             const void* k, const void* v, const void* offsets,
                                             const void* cached, const void* table,
                                             const flint_paged_shape* shape, float scale,
                                             void* workspace, size_t workspace_bytes,
                                             flint_stream stream) {
    Checker c("flint_attention_paged");
    paged_sizes(c, shape)
        .require(std::isfinite(scale), "scale (%g) must be finite", double(scale))
        .require(std::fabs(scale) <= flint::kAttentionMaxScale, "scale (%g) can be up to %g in size",
                 double(scale), double(flint::kAttentionMaxScale));
    if (!c.ok() || empty(*shape)) return c.status();
    const flint_paged_shape& s = *shape;
    const size_t needed = flint::paged_workspace(s);
    c.workspace(workspace, workspace_bytes, needed);
    const size_t qw = s.heads * s.head_width, kw = s.kv_heads * s.head_width;
    const size_t pool = s.pages * s.page_size * kw;
    auto run = [](const char* name, const void* at, size_t count, size_t value) {
        return View{name, at, 1, count, 0, value};
    };
    c.views({{"o", o, s.tokens, qw, s.o_stride, 2},
             run("k_pages", k_pages, pool, 2),
             run("v_pages", v_pages, pool, 2),
             {"q", q, s.tokens, qw, s.q_stride, 2},
             {"k", k, s.tokens, kw, s.kv_stride, 2},
             {"v", v, s.tokens, kw, s.kv_stride, 2},
             run("offsets", offsets, s.sequences + 1, 4),
             run("cached", cached, s.sequences, 4),
             run("table", table, s.sequences * s.max_pages, 4)},
            3);
    if (needed != 0 && c.ok()) {
        const flint::Span ws{"workspace", workspace, needed};
        c.apart(ws, {{"o", o, ((s.tokens - 1) * s.o_stride + qw) * 2},
                     {"k_pages", k_pages, pool * 2},
                     {"v_pages", v_pages, pool * 2},
                     {"q", q, ((s.tokens - 1) * s.q_stride + qw) * 2},
                     {"k", k, ((s.tokens - 1) * s.kv_stride + kw) * 2},
                     {"v", v, ((s.tokens - 1) * s.kv_stride + kw) * 2},
                     {"offsets", offsets, (s.sequences + 1) * 4},
                     {"cached", cached, s.sequences * 4},
                     {"table", table, s.sequences * s.max_pages * 4}});
    }
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_attention_paged(o, k_pages, v_pages, q, k, v, offsets, cached,
                                                  table, s, scale, workspace,
                                                  flint::to_hip(stream)));
    return FLINT_OK;
}

}  // extern "C"
