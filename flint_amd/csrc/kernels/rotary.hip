// Rotary positions for gfx950: pairs of a head's values turned by position x
// frequency.
//
// Bound by HBM: every value is read and written once, 4 bytes against some 3
// operations. An angle is shared by all heads of its token, so a workgroup takes
// the sines and cosines of a few tokens first (one a thread, in LDS) and then the
// tokens' heads, 32 bytes an item: 8 values of either half of the pairs, or 8
// neighbouring pairs. A thread's first items load before the sines are taken, since a
// workgroup's only other loads, positions and frequencies, stand in a chain in front of
// them (16,411 tokens, 32 + 8 heads of 128, half turned: 87 -> 71 us, 4.7 TB/s; a copy of
// the same bytes takes 56). Recomputing the angles for every head, or reading a table of
// them a layer, would cost more than this sharing. 8,192 tokens of 12 + 12 heads of 64
// take 12.7 us (4.0 TB/s; 10.1 to 13 in the kernel), one to 512 tokens a launch's 5.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common/common.h"
#include "kernels/kernels.h"

namespace flint {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;   // items of a thread that load before the angles are there
constexpr unsigned kMaxGrid = 1u << 20;
constexpr size_t kMostTurns = 1024;   // sines and cosines in LDS, of a workgroup

template <int N>
struct Vec {
    typedef _Float16 T __attribute__((ext_vector_type(N)));
};
template <>
struct Vec<1> {
    typedef _Float16 T;
};

__global__ void __launch_bounds__(kThreads) rotary_plan(double* plan, flint_rotary_angles a) {
    constexpr double kTau = 6.283185307179586476925286766559;
    for (int i = threadIdx.x; i <= int(a.width / 2); i += kThreads) {
        if (i == 0) {
            plan[0] = a.magnitude;
            continue;
        }
        const double turns = pow(a.base, -2.0 * (i - 1) / double(a.width)) / kTau;
        double keep = 0.0;
        if (a.original > 0.0)
            keep = fmin(fmax((a.original * turns - a.low) / (a.high - a.low), 0.0), 1.0);
        plan[i] = turns * (keep + (1.0 - keep) / a.factor);
    }
}

struct RotaryArgs {
    _Float16 *q_out, *k_out;
    const _Float16 *q, *k;
    const int* positions;
    const double* plan;
    unsigned tokens, heads, kv_heads, head_width, width;
    unsigned q_stride, k_stride, q_out_stride, k_out_stride;
    unsigned block;    // tokens a workgroup takes at a time
    unsigned chunks;   // work items of a head: the turned ones, then the copied
    unsigned turned;
    int backward;
};

// HALVES: an item turns V pairs (V values of either half), else V neighbouring
// pairs, in two vectors of V. V is the widest that the width's alignment allows; the
// values that do not turn are copied 2 V at a time.
template <bool HALVES, int V>
__global__ void __launch_bounds__(kThreads) rotary(RotaryArgs a) {
    using H = typename Vec<V>::T;
    extern __shared__ float2 turns[];   // [token][pair]: cos, sin
    const unsigned pairs = a.width / 2, heads = a.heads + a.kv_heads;
    const float magnitude = float(a.plan[0]);
    const unsigned items = heads * a.chunks;
    // An item: 2 V values of a row, V at `to` and V `gap` further on (the pairs' halves, or
    // their neighbours), and where its token's angles lie; copied with `turn` kCopied.
    struct Item {
        _Float16* to;
        unsigned turn;
        H u, v;
    };
    constexpr unsigned kCopied = ~0u;
    const unsigned half = HALVES ? pairs : V;
    auto load = [&](unsigned t0, unsigned i) __attribute__((always_inline)) {
        const unsigned t = i / items, in = i - t * items;
        const unsigned head = in / a.chunks, chunk = in - head * a.chunks;
        const bool is_q = head < a.heads, turned = chunk < a.turned;
        const unsigned at = (is_q ? head : head - a.heads) * a.head_width +
                            (turned ? chunk * (HALVES ? V : 2 * V)
                                    : a.width + (chunk - a.turned) * 2 * V);
        const _Float16* from =
            (is_q ? a.q : a.k) + size_t(t0 + t) * (is_q ? a.q_stride : a.k_stride) + at;
        Item x;
        x.to = (is_q ? a.q_out : a.k_out) +
               size_t(t0 + t) * (is_q ? a.q_out_stride : a.k_out_stride) + at;
        x.turn = turned ? t * pairs + chunk * V : kCopied;
        x.u = *reinterpret_cast<const H*>(from);
        x.v = *reinterpret_cast<const H*>(from + (turned ? half : V));
        return x;
    };
    auto finish = [&](const Item& it) __attribute__((always_inline)) {
        H u = it.u, v = it.v;
        if (it.turn != kCopied) {
            // The 2 V values, in the order of their pairs.
            float x[2 * V];
            auto value = [&](int i) -> float {
                if constexpr (V == 1) return float(i == 0 ? it.u : it.v);
                else return float(i < V ? it.u[i % V] : it.v[i % V]);
            };
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int first = HALVES ? e : 2 * e, second = HALVES ? V + e : 2 * e + 1;
                const float a0 = value(first), b0 = value(second);
                const float c = turns[it.turn + e].x, s = turns[it.turn + e].y;
                x[first] = __builtin_fmaf(a0, c, -b0 * s);
                x[second] = __builtin_fmaf(a0, s, b0 * c);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (V == 1) u = _Float16(x[0]), v = _Float16(x[1]);
                else u[e] = _Float16(x[e]), v[e] = _Float16(x[V + e]);
            }
        }
        *reinterpret_cast<H*>(it.to) = u;
        *reinterpret_cast<H*>(it.to + (it.turn != kCopied ? half : V)) = v;
    };
    for (unsigned t0 = blockIdx.x * a.block; t0 < a.tokens; t0 += gridDim.x * a.block) {
        const unsigned block = min(a.block, a.tokens - t0), n = block * items;
        // The first items of a thread are on their way under the sines.
        Item ahead[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (threadIdx.x + j * kThreads < n) ahead[j] = load(t0, threadIdx.x + j * kThreads);
        for (unsigned i = threadIdx.x; i < block * pairs; i += kThreads) {
            const unsigned t = i / pairs, pair = i - t * pairs;
            // Whole turns drop out in FP64; what is left is off by 2^-26 turns in FP32.
            double turn = double(a.positions[t0 + t]) * a.plan[1 + pair];
            turn -= rint(turn);
            float s, c;
            sincospif(2.0f * float(turn), &s, &c);
            turns[i] = float2{c * magnitude, (a.backward ? -s : s) * magnitude};
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (threadIdx.x + j * kThreads < n) finish(ahead[j]);
        for (unsigned i = threadIdx.x + kAhead * kThreads; i < n; i += kThreads)
            finish(load(t0, i));
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_rotary_plan(void* plan, const flint_rotary_angles& angles, hipStream_t stream) {
    hipLaunchKernelGGL(rotary_plan, dim3(1), dim3(kThreads), 0, stream, static_cast<double*>(plan),
                       angles);
    return hipGetLastError();
}

hipError_t launch_rotary(void* q_out, void* k_out, const void* q, const void* k,
                         const void* positions, const void* plan, const flint_rotary_shape& s,
                         bool backward, hipStream_t stream) {
    const bool halves = s.layout == FLINT_ROTARY_HALVES;
    // Vectors of V values, aligned to their size.
    const size_t v = s.width % 16 == 0 && s.head_width % 16 == 0 ? 8
                     : s.width % 8 == 0                          ? 4
                     : s.width % 4 == 0                          ? 2
                                                                 : 1;
    RotaryArgs a{static_cast<_Float16*>(q_out), static_cast<_Float16*>(k_out),
                 static_cast<const _Float16*>(q), static_cast<const _Float16*>(k),
                 static_cast<const int*>(positions), static_cast<const double*>(plan),
                 unsigned(s.tokens), unsigned(s.heads), unsigned(s.kv_heads),
                 unsigned(s.head_width), unsigned(s.width), unsigned(s.q_stride),
                 unsigned(s.k_stride), unsigned(s.q_out_stride), unsigned(s.k_out_stride)};
    a.turned = unsigned(s.width / 2 / v);
    // In place nothing is copied.
    const bool copies = (s.heads != 0 && q_out != q) || (s.kv_heads != 0 && k_out != k);
    a.chunks = a.turned + (copies ? unsigned((s.head_width - s.width) / (2 * v)) : 0u);
    // As many tokens as the threads' first items hold; fewer where that leaves CUs without.
    const size_t items = (s.heads + s.kv_heads) * a.chunks;
    const size_t block = std::min(kAhead * kThreads / items, kMostTurns / (s.width / 2));
    a.block = unsigned(std::clamp<size_t>(std::min(block, s.tokens / 1024), 1, kMostTurns));
    a.backward = backward;
    const unsigned grid =
        unsigned(std::min<size_t>(kMaxGrid, (s.tokens + a.block - 1) / a.block));
    auto pick = [v](auto form) {
        constexpr bool kHalves = decltype(form)::value;
        return v == 8   ? rotary<kHalves, 8>
               : v == 4 ? rotary<kHalves, 4>
               : v == 2 ? rotary<kHalves, 2>
                        : rotary<kHalves, 1>;
    };
    auto* const kernel = halves ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), a.block * (s.width / 2) * sizeof(float2),
                       stream, a);
    return hipGetLastError();
}

}  // namespace flint
