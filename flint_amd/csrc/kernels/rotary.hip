// Rotary positions for gfx950: pairs of a head's values turned by position x
// frequency.
//
// Bound by HBM: every value is read and written once, 4 bytes against some 3
// operations. An angle is shared by all heads of its token, so a workgroup takes
// the sines and cosines of a few tokens first (one a thread, in LDS) and then the
// tokens' heads in 16-byte chunks: 8 values of either half of the pairs, or 4
// neighbouring pairs.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common/common.h"
#include "kernels/kernels.h"

namespace flint {
namespace {

constexpr int kThreads = 256;
constexpr unsigned kMaxGrid = 1u << 20;

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
// pairs. V is the widest that the width's alignment allows; the values that do
// not turn are copied 2 V at a time.
template <bool HALVES, int V>
__global__ void __launch_bounds__(kThreads) rotary(RotaryArgs a) {
    using H = typename Vec<V>::T;
    using W = typename Vec<2 * V>::T;
    extern __shared__ float2 turns[];   // [token][pair]: cos, sin
    const unsigned pairs = a.width / 2, heads = a.heads + a.kv_heads;
    const float magnitude = float(a.plan[0]);
    const unsigned items = heads * a.chunks;
    for (unsigned t0 = blockIdx.x * a.block; t0 < a.tokens; t0 += gridDim.x * a.block) {
        const unsigned block = min(a.block, a.tokens - t0);
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
        for (unsigned i = threadIdx.x; i < block * items; i += kThreads) {
            const unsigned t = i / items, in = i - t * items;
            const unsigned head = in / a.chunks, chunk = in - head * a.chunks;
            const bool is_q = head < a.heads;
            const unsigned at = (is_q ? head : head - a.heads) * a.head_width;
            const _Float16* from = (is_q ? a.q : a.k) +
                                   size_t(t0 + t) * (is_q ? a.q_stride : a.k_stride) + at;
            _Float16* to = (is_q ? a.q_out : a.k_out) +
                           size_t(t0 + t) * (is_q ? a.q_out_stride : a.k_out_stride) + at;
            if (chunk >= a.turned) {
                const unsigned d = a.width + (chunk - a.turned) * 2 * V;
                *reinterpret_cast<W*>(to + d) = *reinterpret_cast<const W*>(from + d);
                continue;
            }
            const float2* turn = turns + t * pairs + chunk * V;
            float x[V], y[V];
            if constexpr (HALVES) {
                const H u = *reinterpret_cast<const H*>(from + chunk * V);
                const H v = *reinterpret_cast<const H*>(from + pairs + chunk * V);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if constexpr (V == 1) x[e] = float(u), y[e] = float(v);
                    else x[e] = float(u[e]), y[e] = float(v[e]);
                }
            } else {
                const W w = *reinterpret_cast<const W*>(from + chunk * 2 * V);
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = float(w[2 * e]), y[e] = float(w[2 * e + 1]);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float c = turn[e].x, s = turn[e].y;
                const float re = __builtin_fmaf(x[e], c, -y[e] * s);
                y[e] = __builtin_fmaf(x[e], s, y[e] * c);
                x[e] = re;
            }
            if constexpr (HALVES) {
                H u, v;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if constexpr (V == 1) u = _Float16(x[e]), v = _Float16(y[e]);
                    else u[e] = _Float16(x[e]), v[e] = _Float16(y[e]);
                }
                *reinterpret_cast<H*>(to + chunk * V) = u;
                *reinterpret_cast<H*>(to + pairs + chunk * V) = v;
            } else {
                W w;
#pragma unroll
                for (int e = 0; e < V; ++e) w[2 * e] = _Float16(x[e]), w[2 * e + 1] = _Float16(y[e]);
                *reinterpret_cast<W*>(to + chunk * 2 * V) = w;
            }
        }
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
    // V values of both halves, aligned to their size; or 4 pairs, 16 bytes.
    const size_t v = halves ? (s.width % 16 == 0 ? 8 : s.width % 8 == 0 ? 4 : 1)
                            : (s.width % 8 == 0 ? 4 : 1);
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
    // A sine and a cosine a thread; fewer tokens where that leaves CUs without any.
    a.block = unsigned(std::max<size_t>(1, kThreads / (s.width / 2)));
    a.block = unsigned(std::min<size_t>(a.block, std::max<size_t>(1, s.tokens / 1024)));
    a.backward = backward;
    const unsigned grid =
        unsigned(std::min<size_t>(kMaxGrid, (s.tokens + a.block - 1) / a.block));
    auto* const kernel = halves ? (v == 8 ? rotary<true, 8> : v == 4 ? rotary<true, 4> : rotary<true, 1>)
                                : (v == 4 ? rotary<false, 4> : rotary<false, 1>);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), a.block * (s.width / 2) * sizeof(float2),
                       stream, a);
    return hipGetLastError();
}

}  // namespace flint
