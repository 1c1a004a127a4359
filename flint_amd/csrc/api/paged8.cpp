// C-ABI entry points of the attention over a paged cache of 8-bit values
// (include/flint/flint_paged8.h): a Checker chain and the launches of
// kernels/paged8.hip.
#include "api/paged_args.h"
#include "flint/flint_paged8.h"

namespace {

using flint::Checker;
using flint::View;

Checker& paged8_sizes(Checker& c, const flint_paged_shape* s, size_t block) {
    if (!flint::paged_sizes(c, s).ok()) return c;
    return c.require(block != 0 && (block & (block - 1)) == 0 && block <= flint::kPaged8MaxBlock &&
                         s->page_size % block == 0,
                     "block (%zu) must be a power of two up to %zu that divides page_size (%zu)",
                     block, flint::kPaged8MaxBlock, s->page_size);
}

}  // namespace

extern "C" {

FLINT_API flint_status flint_attention_paged8_workspace(const flint_paged_shape* shape, size_t block,
                                                        size_t* bytes) {
    Checker c("flint_attention_paged8_workspace");
    if (!paged8_sizes(c.require(bytes != nullptr, "bytes is null"), shape, block).ok())
        return c.status();
    *bytes = flint::empty(*shape) ? 0 : flint::paged8_workspace(*shape);
    return FLINT_OK;
}

FLINT_API flint_status flint_attention_paged8(void* o, void* k_pages, void* k_scales, void* v_pages,
                                              void* v_scales, const void* q, const void* k,
                                              const void* v, const void* offsets, const void* cached,
                                              const void* table, const flint_paged_shape* shape,
                                              size_t block, float scale, void* workspace,
                                              size_t workspace_bytes, flint_stream stream) {
    Checker c("flint_attention_paged8");
    flint::scale_in_range(paged8_sizes(c, shape, block), scale);
    if (!c.ok() || flint::empty(*shape)) return c.status();
    const flint_paged_shape& s = *shape;
    const size_t needed = flint::paged8_workspace(s);
    c.workspace(workspace, workspace_bytes, needed);
    const size_t qw = s.heads * s.head_width, kw = s.kv_heads * s.head_width;
    const size_t pool = s.pages * s.page_size * kw;
    const size_t scales = s.pages * s.kv_heads * (s.page_size / block);
    auto run = [](const char* name, const void* at, size_t count, size_t value) {
        return View{name, at, 1, count, 0, value};
    };
    const View views[] = {{"o", o, s.tokens, qw, s.o_stride, 2},
                          run("k_pages", k_pages, pool, 1),
                          run("k_scales", k_scales, scales, 1),
                          run("v_pages", v_pages, pool, 1),
                          run("v_scales", v_scales, scales, 1),
                          {"q", q, s.tokens, qw, s.q_stride, 2},
                          {"k", k, s.tokens, kw, s.kv_stride, 2},
                          {"v", v, s.tokens, kw, s.kv_stride, 2},
                          run("offsets", offsets, s.sequences + 1, 4),
                          run("cached", cached, s.sequences, 4),
                          run("table", table, s.sequences * s.max_pages, 4)};
    c.views({views[0], views[1], views[2], views[3], views[4], views[5], views[6], views[7], views[8],
             views[9], views[10]},
            5);
    if (needed != 0 && c.ok())
        for (const View& v : views) c.apart({"workspace", workspace, needed}, {v.span()});
    if (!c.ok()) return c.status();
    FLINT_HIP_CHECK(flint::launch_attention_paged8(o, k_pages, k_scales, v_pages, v_scales, q, k, v,
                                                   offsets, cached, table, s, block, scale, workspace,
                                                   flint::to_hip(stream)));
    return FLINT_OK;
}

}  // extern "C"
