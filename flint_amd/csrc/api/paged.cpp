// C-ABI entry points of the attention over a paged cache
// (include/flint/flint_paged.h): a Checker chain and the launches of
// kernels/paged.hip.
#include "api/paged_args.h"
#include "flint/flint_paged.h"
#include "kernels/kernels.h"

namespace {

using flint::Checker;
using flint::View;
using flint::empty;
using flint::paged_sizes;
using flint::scale_in_range;

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
    scale_in_range(paged_sizes(c, shape), scale);
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
