// Log probabilities of given tokens for gfx950, with entropy and top
// alternatives, and the gradient of the logits.
//
// Per row, with mx its largest logit and g_j = scale (l_j - mx) <= 0:
//   S = sum exp g,  logprob_j = g_j - log S,  entropy = log S - sum(g exp g) / S
// (both terms of the entropy are at least 0, so nothing cancels; log S is
// log1p of the sum without one largest term, which a peaked row would lose
// beside it), and
//   dlogits_j = scale (dlp ([j = t] - p_j) - dH p_j (logprob_j + entropy)).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common/common.h"
#include "kernels/kernels.h"
#include "kernels/reduce_common.h"

namespace flint {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// The order of the alternatives as distinct whole numbers: the FP16 value's
// place among all values (-0 with +0, NaN above +inf), then the lower column.
__device__ __forceinline__ unsigned rank_key(_Float16 v, int column) {
    unsigned x = __builtin_bit_cast(unsigned short, v);
    if ((x & 0x7fff) == 0) x = 0;
    x = (x & 0x7fff) > 0x7c00 ? 0xffffu : (x & 0x8000) ? 0xffffu - x : x | 0x8000u;
    return x << 16 | (0xffffu - unsigned(column));
}

template <class T, class Op>
__device__ T block_reduce(T v, T* shared, Op op) {
    for (int d = 32; d > 0; d /= 2) v = op(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
    for (int w = 1; w < kThreads / 64; ++w) v = op(v, shared[w]);
    return v;
}

// One workgroup a row: the maximum, the sums, then the alternatives one by one,
// each the largest key below the last one's.
__global__ void __launch_bounds__(kThreads)
logprobs_forward(float* __restrict__ logprob, float* __restrict__ entropy,
                 float* __restrict__ stats, int* __restrict__ top_ids,
                 float* __restrict__ top_logprobs, const _Float16* __restrict__ logits,
                 const uint16_t* __restrict__ targets, float scale, int vocab, int cols, int top) {
    __shared__ float red[kThreads / 64];
    __shared__ unsigned red_key[kThreads / 64];
    const size_t row = blockIdx.x;
    const _Float16* l = logits + row * cols;
    const int tid = threadIdx.x;
    float mx = -INFINITY;
    for (int j = tid; j < vocab; j += kThreads) mx = __builtin_elementwise_maximum(mx, float(l[j]));
    mx = block_reduce(mx, red, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
    float rest = 0.0f, largest = 0.0f, weighted = 0.0f;   // the terms below 1, how many are 1
    for (int j = tid; j < vocab; j += kThreads) {
        const float gap = float(l[j]) - mx, g = scale * gap;
        const float e = __builtin_amdgcn_exp2f(g * kLog2e);
        if (gap == 0.0f) largest += 1.0f;
        else rest += e;
        weighted += e * fmaxf(g, -3e38f);
    }
    auto add = [](float a, float b) { return a + b; };
    rest = block_reduce(rest, red, add);
    largest = block_reduce(largest, red, add);
    weighted = block_reduce(weighted, red, add);
    const float sum = largest + rest, log_sum = log1pf(largest - 1.0f + rest);
    if (tid == 0) {
        const int t = targets[row];
        logprob[row] = t < vocab ? scale * (float(l[t]) - mx) - log_sum : 0.0f;
        entropy[row] = log_sum - weighted / sum;
        stats[2 * row] = mx;
        stats[2 * row + 1] = log_sum;
    }
    unsigned last = 0xffffffffu;
    for (int i = 0; i < top; ++i) {
        unsigned best = 0;
        for (int j = tid; j < vocab; j += kThreads) {
            const unsigned key = rank_key(l[j], j);
            // The first pass takes every key (a NaN in column 0 has the largest).
            if ((i == 0 || key < last) && key > best) best = key;
        }
        best = block_reduce(best, red_key, [](unsigned a, unsigned b) { return max(a, b); });
        last = best;
        if (tid == 0) {
            const int j = int(0xffffu - (best & 0xffffu));
            top_ids[row * top + i] = j;
            top_logprobs[row * top + i] = scale * (float(l[j]) - mx) - log_sum;
        }
    }
}

__global__ void __launch_bounds__(kThreads)
logprobs_backward(h8* __restrict__ dlogits, const float* __restrict__ dlogprob,
                  const float* __restrict__ dentropy, const h8* __restrict__ logits,
                  const uint16_t* __restrict__ targets, const float* __restrict__ entropy,
                  const float* __restrict__ stats, float scale, int vocab, int chunks) {
    const size_t row = blockIdx.x;
    const int t = targets[row];
    const float mx = stats[2 * row], log_sum = stats[2 * row + 1];
    const float dlp = t < vocab ? dlogprob[row] : 0.0f;
    const float dh = dentropy != nullptr ? dentropy[row] : 0.0f;
    const float ent = dentropy != nullptr ? entropy[row] : 0.0f;
    for (int c = threadIdx.x; c < chunks; c += kThreads) {
        const h8 l = logits[row * chunks + c];
        h8 d;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int j = 8 * c + i;
            const float lp = scale * (float(l[i]) - mx) - log_sum;
            const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
            float g = -p * (dlp + dh * (fmaxf(lp, -3e38f) + ent));
            if (j == t) g += dlp;
            d[i] = j < vocab ? _Float16(scale * g) : _Float16(0.0f);
        }
        dlogits[row * chunks + c] = d;
    }
}

}  // namespace

hipError_t launch_logprobs_forward(void* logprob, void* entropy, void* stats, void* top_ids,
                                   void* top_logprobs, const void* logits, const void* targets,
                                   float scale, size_t rows, size_t vocab, size_t cols, size_t top,
                                   hipStream_t stream) {
    for (size_t done = 0; done < rows;) {
        const size_t n = std::min<size_t>(rows - done, size_t{1} << 22);
        hipLaunchKernelGGL(logprobs_forward, dim3(unsigned(n)), dim3(kThreads), 0, stream,
                           static_cast<float*>(logprob) + done, static_cast<float*>(entropy) + done,
                           static_cast<float*>(stats) + 2 * done,
                           static_cast<int*>(top_ids) + done * top,
                           static_cast<float*>(top_logprobs) + done * top,
                           static_cast<const _Float16*>(logits) + done * cols,
                           static_cast<const uint16_t*>(targets) + done, scale, int(vocab),
                           int(cols), int(top));
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        done += n;
    }
    return hipSuccess;
}

hipError_t launch_logprobs_backward(void* dlogits, const void* dlogprob, const void* dentropy,
                                    const void* logits, const void* targets, const void* entropy,
                                    const void* stats, float scale, size_t rows, size_t vocab,
                                    size_t cols, hipStream_t stream) {
    for (size_t done = 0; done < rows;) {
        const size_t n = std::min<size_t>(rows - done, size_t{1} << 22);
        const auto* dh = static_cast<const float*>(dentropy);
        const auto* ent = static_cast<const float*>(entropy);
        hipLaunchKernelGGL(logprobs_backward, dim3(unsigned(n)), dim3(kThreads), 0, stream,
                           static_cast<h8*>(dlogits) + done * (cols / 8),
                           static_cast<const float*>(dlogprob) + done,
                           dh == nullptr ? nullptr : dh + done,
                           static_cast<const h8*>(logits) + done * (cols / 8),
                           static_cast<const uint16_t*>(targets) + done,
                           ent == nullptr ? nullptr : ent + done,
                           static_cast<const float*>(stats) + 2 * done, scale, int(vocab),
                           int(cols / 8));
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        done += n;
    }
    return hipSuccess;
}

}  // namespace flint
