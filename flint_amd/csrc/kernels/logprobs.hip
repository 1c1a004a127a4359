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
constexpr float kLn2 = 0.69314718055994531f;
// Chunks (of 8 columns) and words that may hold an alternative, as LDS keeps
// them. Rows with more take the words above the border and then the first of those
// at it, or find the exact border first.
constexpr int kChunkList = 512, kWordList = 512;

// The place of an FP16 value among all values: -0 with +0, NaN above +inf.
__device__ __forceinline__ unsigned order_of(_Float16 v) {
    unsigned x = __builtin_bit_cast(unsigned short, v);
    if ((x & 0x7fff) == 0) x = 0;
    return (x & 0x7fff) > 0x7c00 ? 0xffffu : (x & 0x8000) ? 0xffffu - x : x | 0x8000u;
}
__device__ __forceinline__ float value_of(unsigned order) {
    if (order == 0xffffu) return __builtin_nanf("");
    const unsigned short x = (unsigned short)(order & 0x8000u ? order ^ 0x8000u : 0xffffu - order);
    return float(__builtin_bit_cast(_Float16, x));
}

__device__ __forceinline__ _Float16 max_of(const h8& v) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h4 a = __builtin_elementwise_maximum(__builtin_shufflevector(v, v, 0, 1, 2, 3),
                                               __builtin_shufflevector(v, v, 4, 5, 6, 7));
    const h2 b = __builtin_elementwise_maximum(__builtin_shufflevector(a, a, 0, 1),
                                               __builtin_shufflevector(a, a, 2, 3));
    return __builtin_elementwise_maximum(b[0], b[1]);
}

// An empty asm on a chunk: what one pass formed from it is formed again in the
// next rather than kept (8 registers or more a chunk, which cost the rows in
// flight).
__device__ __forceinline__ void keep_packed(h8& v) { asm volatile("" : "+v"(v)); }

// One workgroup of THREADS a row, which it reads once into registers (thread t
// holds the 16-byte chunks t, t + THREADS, ...: at most CPT). Reading bounds it:
// 7 VALU slots a word against 2 bytes. 8,192 rows of 50,257 words: 133 to 149 us
// on different cards, 5.5 to 6.2 TB/s; with 5 alternatives 170.
//
// Alternatives: the row falls into 64 groups of threads, or 256 where many are
// asked (a wave that has a row of its own: into its chunks). The top-th largest of
// the n groups' maxima is a border that at least `top` words reach, and few more
// do: n (1 / (n - top + 1) + ... + 1 / n) on average of words in no order. The
// chunks holding them go to a list in LDS, from there the words, and a word's place
// in the answer is the number of listed words before it. The 64 groups' maxima are a
// step of the row's maximum anyway (16 rows of 50,257 words and 33 alternatives: 9.4
// us, and 10.1 with 256), but 64 of 64 are 304 words on average, and past the list
// in 1 row of 50: 64 rows took 193 us so, 11 with 256.
constexpr int kFewTop = 40;
template <int THREADS, int CPT>
__global__ void __launch_bounds__(THREADS)
logprobs_forward(float* __restrict__ logprob, float* __restrict__ entropy,
                 float* __restrict__ stats, int* __restrict__ top_ids,
                 float* __restrict__ top_logprobs, const h8* __restrict__ logits,
                 const uint16_t* __restrict__ targets, float scale, int vocab, int chunks, int top) {
    constexpr int kWaves = THREADS / 64;
    __shared__ unsigned group_max[64], fine_max[256];
    __shared__ __attribute__((aligned(16))) h8 list[kChunkList];
    __shared__ int list_chunk[kChunkList];
    __shared__ unsigned words[kWordList];
    __shared__ int counts[2];
    __shared__ float red[3][kWaves];
    __shared__ int red_count[kWaves];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const h8* lr = logits + row * chunks;
    const int held = (vocab + 7) >> 3, last = held - 1, last_count = vocab - last * 8;
    const _Float16 lowest = -__builtin_huge_valf16();
    const int target = targets[row];
    float at_target = 0.0f;
    if (tid == 0 && target < vocab) at_target = float(reinterpret_cast<const _Float16*>(lr)[target]);

    h8 raw[CPT];
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
        const int c = tid + i * THREADS;
        raw[i] = c < held ? load_stream(lr + c) : h8(lowest);
    }
    if (last_count < 8 && last >= tid && (last - tid) % THREADS == 0) {
#pragma unroll
        for (int i = 0; i < CPT; ++i)
            if (i == (last - tid) / THREADS) {
#pragma unroll
                for (int j = 1; j < 8; ++j)
                    if (j >= last_count) raw[i][j] = lowest;
            }
    }
    if (tid < 2) counts[tid] = 0;

    // The groups' maxima, the row's, and the border.
    h8 m8 = raw[0];
#pragma unroll
    for (int i = 1; i < CPT; ++i) m8 = __builtin_elementwise_maximum(m8, raw[i]);
    const unsigned own = order_of(max_of(m8));
    unsigned group = own;
    if constexpr (THREADS > 64) {   // groups of THREADS / 64 neighbouring lanes
        constexpr int kGroup = THREADS / 64, kFine = THREADS / 256;
        const bool fine = top > kFewTop && lane % kFine == 0;
        if (kFine == 1 && fine) fine_max[tid] = group;
        group = max(group, unsigned(__builtin_amdgcn_update_dpp(0, int(group), 0xB1, 0xF, 0xF, false)));
        if (kFine == 2 && fine) fine_max[tid / 2] = group;
        group = max(group, unsigned(__builtin_amdgcn_update_dpp(0, int(group), 0x4E, 0xF, 0xF, false)));
        if (kFine == 4 && fine) fine_max[tid / 4] = group;
        if constexpr (kGroup >= 8)
            group = max(group, unsigned(__builtin_amdgcn_update_dpp(0, int(group), 0x141, 0xF, 0xF, false)));
        if constexpr (kGroup >= 16)
            group = max(group, unsigned(__builtin_amdgcn_update_dpp(0, int(group), 0x140, 0xF, 0xF, false)));
        if (lane % kGroup == 0) group_max[tid / kGroup] = group;
        __syncthreads();
        group = group_max[lane];
    } else {
        __syncthreads();
    }
    unsigned border = 0;
    constexpr int kFineOfLane = THREADS > 64 ? 4 : CPT;   // (one wave: its chunks)
    if (kFineOfLane > 1 && top > kFewTop) {
        unsigned f[kFineOfLane];
#pragma unroll
        for (int k = 0; k < kFineOfLane; ++k) {
            if constexpr (THREADS > 64) f[k] = fine_max[lane + 64 * k];
            else f[k] = order_of(max_of(raw[k]));
        }
        for (int bit = 15; bit >= 0; --bit) {
            const unsigned higher = border | 1u << bit;
            int n = 0;
#pragma unroll
            for (int k = 0; k < kFineOfLane; ++k) n += __popcll(__ballot(f[k] >= higher));
            if (n >= top) border = higher;
        }
    } else {
        const int wanted = max(top, 1);
#pragma unroll
        for (int bit = 15; bit >= 0; --bit) {
            const unsigned higher = border | 1u << bit;
            if (__popcll(__ballot(group >= higher)) >= wanted) border = higher;
        }
    }
    unsigned top_order = group;
#pragma unroll
    for (int d = 32; d > 0; d /= 2) top_order = max(top_order, unsigned(__shfl_xor(int(top_order), d)));
    const float mx = value_of(top_order);

    if (top > 0) {
        // (Not below the border's value, so that NaN passes; the words of the chunks
        // are compared by their order.)
        const auto least = _Float16(value_of(border));
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
            keep_packed(raw[i]);
            if (own >= border && !(max_of(raw[i]) < least)) {
                const int at = atomicAdd(&counts[0], 1);
                if (at < kChunkList) {
                    list[at] = raw[i];
                    list_chunk[at] = tid + i * THREADS;
                }
            }
        }
        __syncthreads();
        const int listed = min(counts[0], kChunkList);
        for (int e = tid; e < 8 * listed; e += THREADS) {
            const unsigned order = order_of(list[e >> 3][e & 7]);
            const int column = list_chunk[e >> 3] * 8 + (e & 7);
            if (column < vocab && order >= border) {
                const int at = atomicAdd(&counts[1], 1);
                if (at < kWordList) words[at] = order << 16 | (0xffffu - unsigned(column));
            }
        }
        __syncthreads();
        bool full = counts[0] > kChunkList || counts[1] > kWordList;
        if (full) {
            // Many words equal to the border (a mask that leaves fewer than are
            // asked, say): the words above it, then the lowest columns of those at
            // it, a slice of THREADS chunks at a time until there are enough. (64
            // rows of 50,257 words with 3 left take 14 us so, 192 by halving.)
            __syncthreads();
            if (tid < 2) counts[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < CPT; ++i) {
                keep_packed(raw[i]);
                if (order_of(max_of(raw[i])) <= border) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned order = order_of(raw[i][j]);
                    if (order <= border) continue;
                    const int at = atomicAdd(&counts[1], 1);
                    if (at < kWordList)
                        words[at] = order << 16 | (0xffffu - unsigned((tid + i * THREADS) * 8 + j));
                }
            }
            __syncthreads();
            int have = counts[1];
            full = have > kWordList;
            if (!full && have < top) {
#pragma unroll
                for (int i = 0; i < CPT; ++i) {
                    if (have >= top) continue;   // for all threads alike
                    const int first = (tid + i * THREADS) * 8;
                    unsigned equal = 0;   // bit j: word j of the chunk
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        equal |= unsigned(order_of(raw[i][j]) == border && first + j < vocab) << j;
                    int upto = __popc(equal);
#pragma unroll
                    for (int d = 1; d < 64; d *= 2) {
                        const int v = __shfl_up(upto, d);
                        upto += lane >= d ? v : 0;
                    }
                    if (lane == 63) red_count[wave] = upto;
                    __syncthreads();
                    int at = have + upto - __popc(equal);
                    for (int w = 0; w < kWaves; ++w) {
                        at += w < wave ? red_count[w] : 0;
                        have += red_count[w];
                    }
                    for (; equal != 0 && at < top; equal &= equal - 1, ++at)
                        words[at] = border << 16 | (0xffffu - unsigned(first + __ffs(equal) - 1));
                    __syncthreads();
                }
                if (tid == 0) counts[1] = top;
                __syncthreads();
            }
        }
        if (full) {
            // The exact border by halving: the value, then among the words of
            // that value the column, counting over the whole row each time. (What
            // pads the row is -inf behind its last column: after every word.)
            auto count = [&](auto in) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < CPT; ++i) {
                    keep_packed(raw[i]);
                    unsigned first = unsigned(tid + i * THREADS) * 8;
                    asm volatile("" : "+v"(first));
#pragma unroll
                    for (int j = 0; j < 8; ++j) n += in(order_of(raw[i][j]), first + j);
                }
#pragma unroll
                for (int d = 32; d > 0; d /= 2) n += __shfl_xor(n, d);
                __syncthreads();
                if (lane == 0) red_count[wave] = n;
                __syncthreads();
                n = 0;
                for (int w = 0; w < kWaves; ++w) n += red_count[w];
                return n;
            };
            border = 0;
            for (int bit = 15; bit >= 0; --bit) {
                const unsigned higher = border | 1u << bit;
                if (count([&](unsigned o, unsigned) { return o >= higher; }) >= top) border = higher;
            }
            const int more = top - count([&](unsigned o, unsigned) { return o > border; });
            unsigned below = 0;   // fewer than `more` of them lie before this column
            for (int bit = 15; bit >= 0; --bit) {
                const unsigned higher = below | 1u << bit;
                if (count([&](unsigned o, unsigned c) { return o == border && c < higher; }) < more)
                    below = higher;
            }
            // Words now, without the chunks: exactly `top`.
            if (tid < 2) counts[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < CPT; ++i) {
                keep_packed(raw[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned order = order_of(raw[i][j]);
                    const unsigned column = unsigned(tid + i * THREADS) * 8 + j;
                    if (order > border || (order == border && column <= below))
                        words[atomicAdd(&counts[1], 1)] = order << 16 | (0xffffu - column);
                }
            }
            __syncthreads();
        }
    }

    // The largest words leave the sum (each is 1) and are counted.
    float largest = 0.0f;
    if (__any(own == top_order)) {
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
            keep_packed(raw[i]);
            if (order_of(max_of(raw[i])) != top_order) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (float(raw[i][j]) == mx) {
                    raw[i][j] = lowest;
                    largest += 1.0f;
                }
        }
    }
    // e = 2^(x - mx c), c = scale log2 e: one fma of the exact product, and the
    // rounding of mx c (common to every word) put right in the sums below.
    // -1e4 keeps words of probability 0 out of 0 x inf.
    // Large scales: FP16 values are 2^-24 apart at least, so from c = 2^32 on every
    // e is 0, and c stops at 2^40, where mx c is finite. Values next to mx differ
    // from it by 2^-11 of its size at least and `off` is at most 2^-24 of mx c, so
    // where off passes 1 every e is 0 too, and off stops there: 2^-off is finite.
    const float c = fminf(scale * kLog2e, 0x1p40f), shift = mx * c;
    const float off = fminf(fmaxf(__builtin_fmaf(mx, c, -shift), -1.0f), 1.0f);
    float rest = 0.0f, weighted = 0.0f;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
        keep_packed(raw[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float g = fmaxf(__builtin_fmaf(float(raw[i][j]), c, -shift), -1e4f);
            const float e = __builtin_amdgcn_exp2f(g);
            rest += e;
            weighted = __builtin_fmaf(e, g, weighted);
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        rest += __shfl_xor(rest, d);
        weighted += __shfl_xor(weighted, d);
        largest += __shfl_xor(largest, d);
    }
    if constexpr (kWaves > 1) {
        if (lane == 0) {
            red[0][wave] = rest;
            red[1][wave] = weighted;
            red[2][wave] = largest;
        }
        __syncthreads();
        rest = weighted = largest = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            rest += red[0][w];
            weighted += red[1][w];
            largest += red[2][w];
        }
    }
    // Every g is off by `off`: weighted is the sum of e (g - off), in units of 1.
    const float unit = __builtin_amdgcn_exp2f(-off);
    weighted = __builtin_fmaf(-off, rest, weighted) * unit;
    rest *= unit;
    // (A row without a finite largest logit has no distribution.)
    float log_sum = log1pf(largest - 1.0f + rest);
    if (!(fabsf(mx) < __builtin_huge_valf())) log_sum = __builtin_nanf("");
    if (tid == 0) {
        logprob[row] = target < vocab ? scale * (at_target - mx) - log_sum : 0.0f;
        entropy[row] = log_sum - kLn2 * (weighted / (largest + rest));
        stats[2 * row] = mx;
        stats[2 * row + 1] = log_sum;
    }
    if (top > 0) {
        const int n = counts[1];
        for (int i = tid; i < n; i += THREADS) {
            const unsigned word = words[i];
            int place = 0;
            for (int k = 0; k < n; ++k) place += words[k] > word;
            if (place < top) {
                top_ids[row * top + place] = int(0xffffu - (word & 0xffffu));
                top_logprobs[row * top + place] = scale * (value_of(word >> 16) - mx) - log_sum;
            }
        }
    }
}

// A streaming pass (log p of a word of probability 0 is -1e4: no 0 x inf, however
// large dH is): a workgroup takes kAhead chunks a thread of a row, all read before
// the first is written (dlogits may be logits, so the compiler keeps that order).
// HBM bounds it: 8,192 rows of 50,257 words 311 us, 5.3 TB/s. Shares of a row
// instead of whole ones are for few rows: 16 of 50,257 words take 5.0 us, and 10.1
// in one workgroup each.
constexpr int kAhead = 9;
__global__ void __launch_bounds__(kThreads)
logprobs_backward(h8* dlogits, const float* __restrict__ dlogprob,
                  const float* __restrict__ dentropy, const h8* logits,
                  const uint16_t* __restrict__ targets, const float* __restrict__ entropy,
                  const float* __restrict__ stats, float scale, int vocab, int chunks) {
    const size_t row = blockIdx.x;
    const int t = targets[row];
    const float mx = stats[2 * row], log_sum = stats[2 * row + 1];
    const float dlp = t < vocab ? dlogprob[row] : 0.0f;
    const float dh = dentropy != nullptr ? dentropy[row] : 0.0f;
    const float ent = dentropy != nullptr ? entropy[row] : 0.0f;
    const h8* from = logits + row * chunks;
    h8* to = dlogits + row * chunks;
    const int c0 = int(blockIdx.y) * kThreads * kAhead + int(threadIdx.x);
    h8 l[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (c0 + k * kThreads < chunks) l[k] = from[c0 + k * kThreads];
    auto logprob_of = [&](_Float16 v) { return __builtin_fmaf(scale, float(v) - mx, -log_sum); };
    auto by_probability = [&](float lp, float by) {   // -p (by + dH (log p + H))
        return -__builtin_amdgcn_exp2f(lp * kLog2e) * __builtin_fmaf(dh, fmaxf(lp, -1e4f) + ent, by);
    };
    // The target's, by the thread that has it: 1 - p as -expm1(log p). Of a word
    // that takes most of its row, the difference of 1 and p keeps the rounding of p
    // (2^-24 of 1) and little else: at log p = -1e-6 it is 10% off.
    float d_target = 0.0f;
    const int ahead = (t >> 3) - c0;
    if (t < vocab && ahead >= 0 && ahead % kThreads == 0 && ahead < kThreads * kAhead) {
        _Float16 v{};
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (ahead == k * kThreads && (t & 7) == i) v = l[k][i];
        const float lp = logprob_of(v);
        d_target = __builtin_fmaf(-dlp, expm1f(lp), by_probability(lp, 0.0f));
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const int c = c0 + k * kThreads;
        if (c >= chunks) break;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = by_probability(logprob_of(l[k][i]), dlp);
        if (c == t >> 3 || c == (vocab - 1) >> 3 || c > (vocab - 1) >> 3) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 8 * c + i;
                if (j == t) d[i] = d_target;
                if (j >= vocab) d[i] = 0.0f;
            }
        }
        h8 out;
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = _Float16(scale * d[i]);
        store_stream(to + c, out);
    }
}

}  // namespace

hipError_t launch_logprobs_forward(void* logprob, void* entropy, void* stats, void* top_ids,
                                   void* top_logprobs, const void* logits, const void* targets,
                                   float scale, size_t rows, size_t vocab, size_t cols, size_t top,
                                   hipStream_t stream) {
    // A wave a row while it holds at most 4 chunks a lane (8,192 rows of 997 words:
    // 10.3 us, and 21.8 with 256 threads), else 256 threads, or 1,024 where the rows
    // leave CUs idle and are long (16 rows of 50,257 words and 5 alternatives: 8.7
    // us, and 13.0 with 256; 1,024 rows the other way 33 and 24), or 512 up to 4
    // rows a CU, which hold more of them at once so (512 rows 16.1 us, and 17.9 with
    // 256; 8,192 rows without alternatives the other way 168 and 149).
    const size_t held = (vocab + 7) / 8;
    const bool few = rows <= 256 && held > 1024, some = rows <= 1024 && held > 4096;
    for (size_t done = 0; done < rows;) {
        const size_t n = std::min<size_t>(rows - done, size_t{1} << 22);
#define FLINT_LP(TAKE, THREADS, CPT)                                                            \
    if (TAKE && held <= size_t{THREADS} * CPT)                                                  \
        hipLaunchKernelGGL((logprobs_forward<THREADS, CPT>), dim3(unsigned(n)), dim3(THREADS),  \
                           0, stream, static_cast<float*>(logprob) + done,                      \
                           static_cast<float*>(entropy) + done,                                 \
                           static_cast<float*>(stats) + 2 * done,                               \
                           static_cast<int*>(top_ids) + done * top,                             \
                           static_cast<float*>(top_logprobs) + done * top,                      \
                           static_cast<const h8*>(logits) + done * (cols / 8),                  \
                           static_cast<const uint16_t*>(targets) + done, scale, int(vocab),     \
                           int(cols / 8), int(top))
        FLINT_LP(true, 64, 1);
        else FLINT_LP(true, 64, 2);
        else FLINT_LP(true, 64, 4);
        else FLINT_LP(few, 1024, 2);
        else FLINT_LP(few, 1024, 4);
        else FLINT_LP(few, 1024, 7);
        else FLINT_LP(few, 1024, 8);
        else FLINT_LP(some, 512, 13);
        else FLINT_LP(some, 512, 16);
        else FLINT_LP(true, 256, 2);
        else FLINT_LP(true, 256, 4);
        else FLINT_LP(true, 256, 8);
        else FLINT_LP(true, 256, 16);
        else FLINT_LP(true, 256, 25);
        else FLINT_LP(true, 256, 32);
#undef FLINT_LP
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        done += n;
    }
    return hipSuccess;
}

hipError_t launch_logprobs_backward(void* dlogits, const void* dlogprob, const void* dentropy,
                                    const void* logits, const void* targets, const void* entropy,
                                    const void* stats, float scale, size_t rows, size_t vocab,
                                    size_t cols, hipStream_t stream) {
    constexpr size_t kShare = kThreads * kAhead;
    const auto shares = unsigned((cols / 8 + kShare - 1) / kShare);
    for (size_t done = 0; done < rows;) {
        const size_t n = std::min<size_t>(rows - done, size_t{1} << 22);
        const auto* dh = static_cast<const float*>(dentropy);
        const auto* ent = static_cast<const float*>(entropy);
        hipLaunchKernelGGL(logprobs_backward, dim3(unsigned(n), shares), dim3(kThreads), 0, stream,
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
