// Checks shared by the entry points of the attention over a paged cache (paged.cpp,
// paged8.cpp).
#pragma once

#include <cmath>

#include "common/args.h"
#include "flint/flint_paged.h"
#include "kernels/kernels.h"

namespace flint {

inline Checker& paged_sizes(Checker& c, const flint_paged_shape* s) {
    if (!c.require(s != nullptr, "shape is null").ok()) return c;
    const size_t columns = kPagedMaxPositions / (s->page_size == 0 ? 1 : s->page_size);
    c.require(s->head_width == 64 || s->head_width == 128, "head_width (%zu) must be 64 or 128",
              s->head_width)
        .require(s->heads != 0 && s->heads <= kHeadsMax, "heads (%zu) must be from 1 to %zu",
                 s->heads, kHeadsMax)
        .require(s->kv_heads != 0 && s->kv_heads <= s->heads && s->heads % s->kv_heads == 0,
                 "kv_heads (%zu) must divide heads (%zu)", s->kv_heads, s->heads)
        .require(s->tokens <= kPagedMaxTokens, "tokens (%zu) can be up to %zu", s->tokens,
                 kPagedMaxTokens)
        .require(s->sequences <= kPagedMaxSequences, "sequences (%zu) can be up to %zu",
                 s->sequences, kPagedMaxSequences)
        .require(s->max_new <= kPagedMaxTokens, "max_new (%zu) can be up to %zu", s->max_new,
                 kPagedMaxTokens)
        .require(s->page_size != 0 && s->page_size % 8 == 0 &&
                     s->page_size <= kPagedMaxPageSize,
                 "page_size (%zu) must be a multiple of 8 from 8 to %zu", s->page_size,
                 kPagedMaxPageSize)
        .require(s->pages != 0 && s->pages <= 0x7fffffffu, "pages (%zu) must be from 1 to %zu",
                 s->pages, size_t{0x7fffffff})
        .require(s->max_pages != 0 && s->max_pages <= columns, "max_pages (%zu) must be from 1 to %zu",
                 s->max_pages, columns);
    if (c.ok())
        c.require(s->pages <= kPagedMaxPool / (s->page_size * s->kv_heads * s->head_width),
                  "pages (%zu) x page_size x kv_heads x head_width can be up to %zu", s->pages,
                  kPagedMaxPool)
            .require(s->tokens * s->heads <= kPagedMaxRows,
                     "tokens x heads (%zu) can be up to %zu", s->tokens * s->heads,
                     kPagedMaxRows)
            .require(s->sequences * s->kv_heads <= kPagedMaxRows / 8,
                     "sequences x kv_heads (%zu) can be up to %zu", s->sequences * s->kv_heads,
                     kPagedMaxRows / 8);
    const struct {
        const char* name;
        size_t stride, width;
    } strides[] = {{"q_stride", s->q_stride, s->heads * s->head_width},
                   {"kv_stride", s->kv_stride, s->kv_heads * s->head_width},
                   {"o_stride", s->o_stride, s->heads * s->head_width}};
    for (const auto& t : strides)
        c.require(t.stride % 8 == 0 && t.stride >= t.width && t.stride <= kStrideMax,
                  "%s (%zu) must be a multiple of 8 from %zu to %zu", t.name, t.stride, t.width,
                  kStrideMax);
    return c;
}

inline Checker& scale_in_range(Checker& c, float scale) {
    return c.require(std::isfinite(scale), "scale (%g) must be finite", double(scale))
        .require(std::fabs(scale) <= kAttentionMaxScale, "scale (%g) can be up to %g in size",
                 double(scale), double(kAttentionMaxScale));
}

inline bool empty(const flint_paged_shape& s) {
    return s.tokens == 0 || s.sequences == 0 || s.max_new == 0;
}

}  // namespace flint
