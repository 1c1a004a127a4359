// Attention of new tokens over a paged cache for gfx950: each new token sees the
// cached positions of its sequence and the sequence's new tokens up to itself;
// the new rows of k and v go into their pages in the same launch, and are read
// from k and v here, so no workgroup waits for another's store.
#include <hip/hip_runtime.h>

#include "common/common.h"
#include "kernels/attention_tiles.h"
#include "kernels/kernels.h"

namespace flint {
namespace {

struct PagedArgs {
    _Float16 *o, *k_pages, *v_pages;
    const _Float16 *q, *k, *v;
    const int *offsets, *cached, *table;
    int tokens, sequences, max_new, heads, kv_heads;
    int q_stride, kv_stride, o_stride;
    int pages, page_size, max_pages;
    float c;   // scale log2 e
};

// Sequence s: its new tokens' first row and count, and its cached positions.
struct Sequence {
    int first, count, cached;
};
__device__ __forceinline__ Sequence sequence_of(const PagedArgs& a, int s) {
    Sequence q;
    q.first = min(max(a.offsets[s], 0), a.tokens);
    q.count = min(min(max(a.offsets[s + 1], q.first), a.tokens) - q.first, a.max_new);
    q.cached = min(max(a.cached[s], 0), a.max_pages * a.page_size);
    return q;
}

// The page of position p of sequence s, or -1.
__device__ __forceinline__ int page_of(const PagedArgs& a, int s, int p) {
    const int column = p / a.page_size;
    if (column >= a.max_pages) return -1;
    const int page = a.table[size_t(s) * a.max_pages + column];
    return page >= 0 && page < a.pages ? page : -1;
}
template <int HD>
__device__ __forceinline__ size_t row_in_pages(const PagedArgs& a, int page, int head, int p) {
    return ((size_t(page) * a.kv_heads + head) * a.page_size + p % a.page_size) * HD;
}

// One wave a token and head: a lane takes a key of each 64, then a column of V.
template <int HD>
__global__ void __launch_bounds__(256) paged_rows(PagedArgs a) {
    const int lane = threadIdx.x & 63;
    const int head = (blockIdx.x * 4 + (threadIdx.x >> 6)) % a.heads;
    const int place = (blockIdx.x * 4 + (threadIdx.x >> 6)) / a.heads;
    const int s = blockIdx.y;
    const Sequence sq = sequence_of(a, s);
    if (place >= sq.count) return;
    const int group = a.heads / a.kv_heads, kv = head / group;
    const _Float16* qr = a.q + size_t(sq.first + place) * a.q_stride + size_t(head) * HD;
    if (head % group == 0) {
        const int page = page_of(a, s, sq.cached + place);
        const size_t from = size_t(sq.first + place) * a.kv_stride + size_t(kv) * HD;
        if (page >= 0) {
            const size_t to = row_in_pages<HD>(a, page, kv, sq.cached + place);
            for (int d = lane; d < HD; d += 64) {
                a.k_pages[to + d] = a.k[from + d];
                a.v_pages[to + d] = a.v[from + d];
            }
        }
    }
    const int keys = sq.cached + place + 1;
    float m = -3e38f, l = 0.0f, acc[HD / 64] = {};
    for (int base = 0; base < keys; base += 64) {
        const int p = base + lane;
        const _Float16 *kr = nullptr, *vr = nullptr;
        if (p < keys) {
            if (p >= sq.cached) {
                const size_t at = size_t(sq.first + p - sq.cached) * a.kv_stride + size_t(kv) * HD;
                kr = a.k + at;
                vr = a.v + at;
            } else if (const int page = page_of(a, s, p); page >= 0) {
                const size_t at = row_in_pages<HD>(a, page, kv, p);
                kr = a.k_pages + at;
                vr = a.v_pages + at;
            }
        }
        float x = -INFINITY;
        if (kr != nullptr) {
            float dot = 0.0f;
            for (int d = 0; d < HD; d += 8) {
                const f16x8 kv8 = *reinterpret_cast<const f16x8*>(kr + d);
                const f16x8 qv8 = *reinterpret_cast<const f16x8*>(qr + d);
                for (int e = 0; e < 8; ++e) dot = __builtin_fmaf(float(kv8[e]), float(qv8[e]), dot);
            }
            x = dot * a.c;
        }
        float mx = x;
        for (int d = 32; d > 0; d /= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float m_new = fmaxf(m, mx);
        const float alpha = __builtin_amdgcn_exp2f(m - m_new);
        const float pr = __builtin_amdgcn_exp2f(x - m_new);
        float sum = pr;
        for (int d = 32; d > 0; d /= 2) sum += __shfl_xor(sum, d);
        l = l * alpha + sum;
        m = m_new;
        for (int i = 0; i < HD / 64; ++i) acc[i] *= alpha;
        for (int j = 0; j < 64; ++j) {
            const auto row = reinterpret_cast<const _Float16*>(
                __shfl(reinterpret_cast<unsigned long long>(vr), j));
            if (row == nullptr) continue;
            const float pj = __shfl(pr, j);
            for (int i = 0; i < HD / 64; ++i)
                acc[i] = __builtin_fmaf(pj, float(row[64 * i + lane]), acc[i]);
        }
    }
    _Float16* orow = a.o + size_t(sq.first + place) * a.o_stride + size_t(head) * HD;
    for (int i = 0; i < HD / 64; ++i) orow[64 * i + lane] = _Float16(acc[i] / l);
}

}  // namespace

size_t paged_workspace(const flint_paged_shape&) { return 0; }

hipError_t launch_attention_paged(void* o, void* k_pages, void* v_pages, const void* q,
                                  const void* k, const void* v, const void* offsets,
                                  const void* cached, const void* table,
                                  const flint_paged_shape& s, float scale, void*,
                                  hipStream_t stream) {
    PagedArgs a{static_cast<_Float16*>(o), static_cast<_Float16*>(k_pages),
                static_cast<_Float16*>(v_pages), static_cast<const _Float16*>(q),
                static_cast<const _Float16*>(k), static_cast<const _Float16*>(v),
                static_cast<const int*>(offsets), static_cast<const int*>(cached),
                static_cast<const int*>(table), int(s.tokens), int(s.sequences),
                int(s.max_new < s.tokens ? s.max_new : s.tokens), int(s.heads), int(s.kv_heads),
                int(s.q_stride), int(s.kv_stride), int(s.o_stride), int(s.pages),
                int(s.page_size), int(s.max_pages), scale * kLog2e};
    const dim3 grid(unsigned((size_t(a.max_new) * s.heads + 3) / 4), unsigned(s.sequences));
    auto* const kernel = s.head_width == 64 ? paged_rows<64> : paged_rows<128>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace flint
