// Causal attention over packed sequences for gfx950: sequences of different
// lengths one after another in the token rows, grouped heads, head widths 64
// and 128; forward, and backward to dQ, dK and dV.
//
// Per query t of a sequence, over its keys t' <= t: S = c q k^T (c = scale
// log2 e), P = 2^(S - m) / l with the running maximum m and sum l, O = P V,
// lse = (m + log2 l) ln 2. Backward, with P recomputed from lse and D = sum
// dO O: dV = P^T dO, dS = P (dO V^T - D), dQ = scale dS K, dK = scale dS^T Q.
//
// A workgroup owns 128 queries (dK/dV: keys) of one sequence and head and walks
// the sequence's tiles of 64 keys (queries). Which, the plan says: a list of
// blocks, longest first, made once a batch on the device. The work of a block
// grows with its place in its sequence, so the list's order is what balances
// the GPU; the kernels' grids are the largest number of blocks that tokens and
// sequences allow, and workgroups past the list's end leave at once.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "common/common.h"
#include "kernels/attention_tiles.h"
#include "kernels/kernels.h"

namespace flint {
namespace {

constexpr int kThreads = 256;   // of the joining launch

// A workgroup's waves: four over its 128 queries (keys), times `turns` groups
// that take the 64-row tiles in turn and join their sums in LDS at the end. Two
// turns halve the longest block's time, which bounds batches of different
// lengths (one head of one 3,913-token sequence: forward 53 -> 41 us, backward
// 163 -> 110; the forward of 12 heads and 24 sequences up to that length 59 ->
// 53), and cost batches of equal short ones some of their second round of
// workgroups (8 x 1,024 tokens, 12 heads: forward 24 -> 29, since then 27). Two
// waves over 64 queries and four turns shorten that block more (25 us), but read
// each tile for half the rows (one 8,192-token sequence 127 -> 182). dK and dV at
// 128-wide heads take a wave's 512 registers: one turn (two waves and two turns:
// 616 -> 634).
constexpr int kRowWaves = kPackedBlock / 32;
constexpr int kForwardTurns = 2, kQueryTurns = 2;
template <int HD>
constexpr int kKeyTurns = HD == 64 ? 2 : 1;
constexpr int threads_of(int turns) { return 64 * kRowWaves * turns; }

// The kernels that load tiles ahead keep all of a workgroup's LDS in one array:
// with others beside it the compiler cannot tell the loads under way from what it
// reads, and waits for them before every tile (the forward pass of 24 ragged
// sequences, 12 heads of 64: 53 us instead of 46).

// ---------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024;
constexpr int kBuckets = 1024;

// One workgroup. The blocks of a sequence of n blocks have places 0 .. n - 1;
// bucket b holds the places b << shift .. and comes before bucket b - 1. A
// counting sort: full[b] counts the sequences whose last, partly filled bucket
// is b, part[b] their places in it; the items of b are part[b] + (full[b + 1] +
// full[b + 2] + ...) << shift. Within a bucket the order is the arrival's: it
// changes which workgroup takes which block and no result. More blocks than the
// plan holds, which takes offsets that decrease, make it empty: their number is
// not bounded by tokens, nor the time to write them.
__global__ void __launch_bounds__(kPlanThreads)
packed_plan(int4* __restrict__ plan, const int* __restrict__ offsets, int sequences, int tokens,
            int capacity, int shift) {
    __shared__ int full[kBuckets], part[kBuckets], next[kBuckets], filled, blocks;
    const int tid = threadIdx.x;
    full[tid] = part[tid] = 0;
    if (tid == 0) blocks = 0;
    __syncthreads();
    auto rows_of = [&](int s, int* begin) {
        const int a = min(max(offsets[s], 0), tokens), b = min(max(offsets[s + 1], a), tokens);
        *begin = a;
        return b;
    };
    const int low = (1 << shift) - 1;
    int own = 0;   // this thread's blocks, and a wave's: at most capacity + 1
    for (int s = tid; s < sequences; s += kPlanThreads) {
        int begin;
        const int end = rows_of(s, &begin);
        const int n = (end - begin + kPackedBlock - 1) / kPackedBlock;
        if (n == 0) continue;
        own = min(own + n, capacity + 1);
        atomicAdd(&full[n >> shift], 1);
        atomicAdd(&part[n >> shift], n & low);
    }
    own = min(wave_sum(own), capacity + 1);
    if (tid % 64 == 0) atomicAdd(&blocks, own);
    __syncthreads();
    if (blocks > capacity) {
        for (int i = tid; i < capacity; i += kPlanThreads) plan[i] = int4{0, 0, 0, 0};
        return;
    }
    // Sums over the buckets after this thread's, the last bucket first: a scan
    // in each wave and of the waves' totals.
    __shared__ int totals[kPlanThreads / 64];
    const int lane = tid & 63, wave = tid >> 6, bucket = kBuckets - 1 - tid;
    auto before = [&](int own) {
        const int upto = wave_scan(own);
        if (lane == 63) totals[wave] = upto;
        __syncthreads();
        const int others = wave_scan(lane < kPlanThreads / 64 ? totals[lane] : 0);
        const int sum = upto - own + (wave == 0 ? 0 : __builtin_amdgcn_readlane(others, max(wave - 1, 0)));
        __syncthreads();
        return sum;
    };
    const int items = part[bucket] + (before(full[bucket]) << shift);
    const int first = before(items);
    next[bucket] = first;
    // Entries past the last block are empty: a workgroup reads its own alone.
    if (bucket == 0) filled = first + items;
    __syncthreads();
    for (int i = filled + tid; i < capacity; i += kPlanThreads) plan[i] = int4{0, 0, 0, 0};
    // A sequence of many blocks is written by its whole wave.
    for (int base = 0; base < sequences; base += kPlanThreads) {
        const int s = base + tid;
        int begin = 0, end = 0;
        if (s < sequences) end = rows_of(s, &begin);
        const int n = (end - begin + kPackedBlock - 1) / kPackedBlock;
        auto put = [&](int b0, int e0, int block) {
            const int at = atomicAdd(&next[min(block >> shift, kBuckets - 1)], 1);
            if (at < capacity) plan[at] = int4{b0, e0, block, 0};
        };
        if (n <= 16)
            for (int b = 0; b < n; ++b) put(begin, end, b);
        for (unsigned long long many = __ballot(n > 16); many != 0; many &= many - 1) {
            const int from = __ffsll(many) - 1;
            const int b0 = __shfl(begin, from), e0 = __shfl(end, from), n0 = __shfl(n, from);
            for (int b = lane; b < n0; b += 64) put(b0, e0, b);
        }
    }
}

// The block and head that workgroup `id` works on; false past the list. Blocks
// go longest first, heads side by side: workgroup id runs on XCD id % 8, so with
// 8 heads an XCD's L2 holds one head's rows. (Every other run of 256 workgroups
// backwards, to put short blocks beside long ones, breaks that: 8 heads of 128
// over 8,192 tokens 158 -> 197 us, and the ragged batch gained nothing. Nor did
// cutting the longest blocks into parts of their tiles, joined by another
// launch: blocks that start together read the same tiles of K and V at the same
// time, out of L2, which parts do not; 8 heads of 128 over 8,192 tokens 165 ->
// 191.) A plan of other sequences gives wrong rows, but none outside the tokens.
struct Work {
    int begin, length, block, head;
};
__device__ __forceinline__ bool work_of(const int4* plan, int id, int heads, int tokens,
                                        Work* w) {
    const int item = id / heads;
    const int4 it = plan[item];
    w->begin = min(max(it.x, 0), tokens);
    w->length = min(max(it.y, w->begin), tokens) - w->begin;
    w->block = it.z;
    w->head = id - item * heads;
    return it.z >= 0 && it.z <= (w->length - 1) / kPackedBlock && w->length > 0;
}

// A block's 128 rows of one head into two tiles, shared out over WAVES waves.
// Read by the lanes straight into their fragments, 16 bytes of 32 rows at a time
// and by both turns, they come slower: over 8 x 1,024 tokens of 8 heads of 128
// the forward pass takes 34.9 us so and 33.3 through LDS, dQ 47.8 and 43.0.
template <int HD, int WAVES>
__device__ __forceinline__ void load_block(_Float16* tiles, const _Float16* from, int left,
                                           int stride, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        load_tile<HD, WAVES>(tiles + i * Tile<HD>::kHalves, from + size_t(64 * i) * stride,
                             left - 64 * i, stride, wave, lane);
}
// The fragments of wave `wave`'s 32 of them.
template <int HD>
__device__ __forceinline__ void block_frags(f16x8 (&f)[HD / 16], const _Float16* tiles,
                                            const Frags<HD>& fo, int wave) {
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
        f[kk] = fo.row(tiles + (wave >> 1) * Tile<HD>::kHalves, wave & 1, kk);
}

// Fragments of row `row` of a head's matrix from memory (zeros from `left` on).
template <int HD>
__device__ __forceinline__ void load_frags(f16x8 (&f)[HD / 16], const _Float16* base, int row,
                                           int left, int stride, int h) {
    const _Float16* at = base + size_t(row) * stride + 8 * h;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
        f[kk] = row < left ? *reinterpret_cast<const f16x8*>(at + 16 * kk) : f16x8{};
}

struct Strides {
    int q, kv, o;
};

// Whether a wave of the 32 queries from q0 on leaves the tile of keys from kbase on
// out: every key after every query, or no query in the sequence. What it takes is
// a tile that was loaded: kbase is a multiple of 64 and q0 of 32, so kbase is in the
// tile of q0 or before. (Past the sequence a turn may have no tile at all, and LDS
// holds what was there before: not a number, mostly.)
__device__ __forceinline__ bool unseen(int kbase, int q0, int length) {
    return kbase > q0 + 31 || q0 >= length;
}

// The backward kernels form 2^kUp P and with it 2^kUp dS, and take the factor
// out of their sums again: over thousands of keys, or from a small dO, dS is
// often below FP16's normal values (one head over 3,000 tokens, dO of 0.01: dQ
// 3.2e-4 off relative to its size without the factor, 3.0e-4 with it, 2.1e-4
// from storing it alone). A block whose sums overflow by it is done again
// without it.
constexpr float kUp = 8.0f;
__device__ __forceinline__ float down_by(float up) { return up == 0.0f ? 1.0f : 0x1p-8f; }

template <int DB>
__device__ __forceinline__ bool non_finite(const f32x16 (&acc)[DB]) {
    float zero = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) zero = __builtin_fmaf(acc[db][r], 0.0f, zero);
    return !(zero == 0.0f);
}

// The turns' sums of one result added in LDS, in order, into the first's; false
// in the others.
template <int HD, int W, int G>
__device__ __forceinline__ bool join_turns(float* lds, f32x16* acc, int wave, int turn, int lane) {
    __syncthreads();
    if constexpr (G == 1) return true;
    const int fr = lane & 31, h = lane >> 5;
    auto theirs = [&](int g) { return lds + ((g - 1) * W + wave) * HD * 32; };
    if (turn != 0) {
#pragma unroll
        for (int db = 0; db < HD / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                theirs(turn)[(32 * db + result_row(r, h)) * 32 + fr] = acc[db][r];
    }
    __syncthreads();
    if (turn != 0) return false;
#pragma unroll
    for (int g = 1; g < G; ++g)
#pragma unroll
        for (int db = 0; db < HD / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[db][r] += theirs(g)[(32 * db + result_row(r, h)) * 32 + fr];
    return true;
}

// ---------------------------------------------------------------- forward

template <int HD>
__global__ void __launch_bounds__(threads_of(kForwardTurns), HD == 64 ? 4 : 2)
packed_forward(_Float16* __restrict__ out, float* __restrict__ lse, const _Float16* __restrict__ q,
               const _Float16* __restrict__ k, const _Float16* __restrict__ v,
               const int4* __restrict__ plan, int tokens, int heads, int group, Strides st,
               float c, bool negative) {
    constexpr int kTile = Tile<HD>::kHalves, KK = HD / 16, DB = HD / 32;
    constexpr int W = kRowWaves, G = kForwardTurns;
    // [buf][group][K, V]; behind them the turns' maxima and sums.
    constexpr int kTiles = 2 * G * 2 * kTile;
    __shared__ __attribute__((aligned(16))) _Float16 lds[kTiles + G * W * 32 * 4];
    float2(*sums)[W][32] = reinterpret_cast<float2(*)[W][32]>(lds + kTiles);
    Work w;
    if (!work_of(plan, int(blockIdx.x), heads, tokens, &w)) return;
    const int row0 = w.block * kPackedBlock;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W;
    const int turn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / W;
    const int fr = lane & 31, h = lane >> 5;
    const Frags<HD> fo(lane);
    const int length = w.length;
    const _Float16* qb = q + size_t(w.begin) * st.q + size_t(w.head) * HD;
    const _Float16* kb = k + size_t(w.begin) * st.kv + size_t(w.head / group) * HD;
    const _Float16* vb = v + size_t(w.begin) * st.kv + size_t(w.head / group) * HD;
    const int q0 = row0 + wave * 32;
    const int qi = q0 + fr;

    float m = kFloor, l = 0.0f;
    bool started = false;
    f32x16 acc[DB] = {};
    const int q_last = min(row0 + 32 * W, length) - 1;
    const int tiles = q_last / 64 + 1, steps = (tiles + G - 1) / G;
    auto load = [&](int i) {
        const int j = G * i + turn;
        if (j >= tiles) return;
        _Float16* t = lds + ((i & 1) * G + turn) * 2 * kTile;
        const size_t at = size_t(64 * j) * st.kv;
        load_tile<HD, W>(t, kb + at, length - 64 * j, st.kv, wave, lane);
        load_tile<HD, W>(t + kTile, vb + at, length - 64 * j, st.kv, wave, lane);
    };
    // The queries go through the buffers of the second step.
    _Float16* block = lds + 2 * G * kTile;
    load_block<HD, W * G>(block, qb + size_t(row0) * st.q, length - row0, st.q,
                          wave + W * turn, lane);
    load(0);
    wait_vmcnt<0>();
    block_sync();
    f16x8 qf[KK];
    block_frags<HD>(qf, block, fo, wave);
    if (negative)   // c is positive: the scale's sign goes into q
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[kk] = -qf[kk];
    for (int i = 0; i < steps; ++i) {
        wait_vmcnt<0>();
        block_sync();
        const _Float16* kt = lds + ((i & 1) * G + turn) * 2 * kTile;
        const _Float16* vt = kt + kTile;
        if (i + 1 < steps) load(i + 1);
        const int kbase = 64 * (G * i + turn);
        if (unseen(kbase, q0, length)) continue;
        // Scores are scaled by c inside the exponent's FMA; where the tile holds
        // keys after a query (a uniform branch), before it, and masked.
        auto scores = [&](f32x16 (&s)[2], unsigned zero) __attribute__((always_inline)) {
            s[0] = s[1] = f32x16{};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int hb = 0; hb < 2; ++hb) s[hb] = mfma(fo.row(kt + zero, hb, kk), qf[kk], s[hb]);
            if (kbase + 63 <= q0) return c;
            const int seen = qi - kbase - 4 * h + int(zero);   // a register's key: a constant + 4h
#pragma unroll
            for (int hb = 0; hb < 2; ++hb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[hb][r] = 32 * hb + result_row(r, 0) <= seen ? s[hb][r] * c : -INFINITY;
            return 1.0f;
        };
        f16x8 pf[4];
        l += probabilities<2>(pf, scores, &m, &started, [&](float by) __attribute__((always_inline)) {
            l *= by;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= by;
        });
        // O^T += V^T P^T, a 16-key slice at a time (two for 64-wide heads).
        constexpr int kSlices = HD == 64 ? 2 : 1;
#pragma unroll
        for (int cs = 0; cs < 4; cs += kSlices) {
            TrFrag vf[kSlices][DB];
#pragma unroll
            for (int i = 0; i < kSlices; ++i)
#pragma unroll
                for (int db = 0; db < DB; ++db) vf[i][db] = fo.transposed(vt, cs + i, db);
            wait_lds();
#pragma unroll
            for (int i = 0; i < kSlices; ++i)
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    acc[db] = mfma(as_f16x8(vf[i][db]), pf[cs + i], acc[db]);
        }
    }
    l += xor32(l);
    // The turns' sums join in LDS: each but the first leaves its O^T [HD][32] a
    // wave.
    __syncthreads();
    auto theirs = [&](int g) { return reinterpret_cast<float*>(lds) + ((g - 1) * W + wave) * HD * 32; };
    if (turn != 0) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                theirs(turn)[(32 * db + result_row(r, h)) * 32 + fr] = acc[db][r];
        if (h == 0) sums[turn][wave][fr] = float2{m, l};
    }
    __syncthreads();
    _Float16* rows = lds + (G - 1) * W * HD * 32 * 2;   // behind theirs
    if (turn == 0) {
#pragma unroll
        for (int g = 1; g < G; ++g) {
            const float2 other = sums[g][wave][fr];
            const float most = fmaxf(m, other.x);
            const float by = __builtin_amdgcn_exp2f(m - most);
            const float other_by = __builtin_amdgcn_exp2f(other.x - most);
            m = most;
            l = __builtin_fmaf(other.y, other_by, l * by);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[db][r] = __builtin_fmaf(theirs(g)[(32 * db + result_row(r, h)) * 32 + fr],
                                                other_by, acc[db][r] * by);
        }
        write_rows<HD>(rows, acc, 1.0f / l, wave * 32 + fr, h);
        if (qi < length && h == 0)
            lse[size_t(w.head) * tokens + w.begin + qi] =
                (m + kBelow + __builtin_amdgcn_logf(l * kBelowFactor)) * kLn2;
    }
    __syncthreads();
    copy_rows<HD, threads_of(kForwardTurns)>(rows, length - row0, [&](int row) {
        return out + size_t(w.begin + row0 + row) * st.o + size_t(w.head) * HD;
    });
}

// ---------------------------------------------------------------- backward: dQ (and D)

template <int HD>
__global__ void __launch_bounds__(threads_of(kQueryTurns), 2)
packed_backward_dq(_Float16* __restrict__ dq, float* __restrict__ dsum,
                   const _Float16* __restrict__ q, const _Float16* __restrict__ k,
                   const _Float16* __restrict__ v, const _Float16* __restrict__ o,
                   const _Float16* __restrict__ dout, const float* __restrict__ lse,
                   const int4* __restrict__ plan, int tokens, int heads, int group, Strides st,
                   float c, float scale) {
    constexpr int kTile = Tile<HD>::kHalves, KK = HD / 16, DB = HD / 32;
    constexpr int W = kRowWaves, G = kQueryTurns;
    // [buf][group][K, V]; behind them the turns' rests and the overflow flag.
    constexpr int kTiles = 2 * G * 2 * kTile;
    __shared__ __attribute__((aligned(16))) _Float16 lds[kTiles + (G * W * 32 + 4) * 2];
    float(*rests)[W][32] = reinterpret_cast<float(*)[W][32]>(lds + kTiles);
    int& overflow = *reinterpret_cast<int*>(lds + kTiles + G * W * 32 * 2);
    Work w;
    if (!work_of(plan, int(blockIdx.x), heads, tokens, &w)) return;
    if (threadIdx.x == 0) overflow = 0;
    const int row0 = w.block * kPackedBlock;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W;
    const int turn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / W;
    const int fr = lane & 31, h = lane >> 5;
    const Frags<HD> fo(lane);
    const int length = w.length;
    const size_t o_at = size_t(w.begin) * st.o + size_t(w.head) * HD;
    const size_t kv_at = size_t(w.begin) * st.kv + size_t(w.head / group) * HD;
    const size_t q_at = size_t(w.begin) * st.q + size_t(w.head) * HD;
    const int q0 = row0 + wave * 32;
    const int qi = q0 + fr;

    const int q_last = min(row0 + 32 * W, length) - 1;
    const int tiles = q_last / 64 + 1, steps = (tiles + G - 1) / G;
    auto load = [&](int i) {
        const int j = G * i + turn;
        if (j >= tiles) return;
        _Float16* t = lds + ((i & 1) * G + turn) * 2 * kTile;
        const size_t at = kv_at + size_t(64 * j) * st.kv;
        load_tile<HD, W>(t, k + at, length - 64 * j, st.kv, wave, lane);
        load_tile<HD, W>(t + kTile, v + at, length - 64 * j, st.kv, wave, lane);
    };
    // Q and dO go through the buffers of the second step.
    _Float16* block = lds + 2 * G * kTile;
    load_block<HD, W * G>(block, q + q_at + size_t(row0) * st.q, length - row0, st.q,
                          wave + W * turn, lane);
    load_block<HD, W * G>(block + 2 * kTile, dout + o_at + size_t(row0) * st.o, length - row0,
                          st.o, wave + W * turn, lane);
    load(0);
    f16x8 of[KK];
    load_frags<HD>(of, o + o_at, qi, length, st.o, h);
    wait_vmcnt<0>();
    block_sync();
    f16x8 qf[KK], df[KK];
    block_frags<HD>(qf, block, fo, wave);
    block_frags<HD>(df, block + 2 * kTile, fo, wave);
    float dd = 0.0f;
    {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                dd = __builtin_fmaf(float(df[kk][e]), float(of[kk][e]), dd);
    }
    dd += xor32(dd);
    const size_t row_at = size_t(w.head) * tokens + w.begin + qi;
    const float lse2 = qi < length ? lse[row_at] * kLog2e : 0.0f;

    f32x16 acc[DB];   // 2^up dQ^T[d][q]
    float up = kUp;
    for (;;) {
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
        const float l2 = lse2 - up;
        float rest = 0.0f;   // 2^up times the sum of dS over the keys
        for (int i = 0; i < steps; ++i) {
            wait_vmcnt<0>();
            block_sync();
            const _Float16* kt = lds + ((i & 1) * G + turn) * 2 * kTile;
            const _Float16* vt = kt + kTile;
            if (i + 1 < steps) load(i + 1);
            const int kbase = 64 * (G * i + turn);
            if (unseen(kbase, q0, length)) continue;
            const bool masked = kbase + 63 > q0;
            // Two halves of 32 keys, each through all of its products before the
            // next (fewer registers live at once).
#pragma unroll
            for (int hb = 0; hb < 2; ++hb) {
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    s = mfma(fo.row(kt, hb, kk), qf[kk], s);
                    dp = mfma(fo.row(vt, hb, kk), df[kk], dp);
                }
                f16x8 sf[2];
                auto form = [&](auto mask) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float p = __builtin_amdgcn_exp2f(s[r] * c - l2);
                        if constexpr (mask)
                            if (kbase + 32 * hb + result_row(r, h) > qi) p = 0.0f;
                        const float ds = p * (dp[r] - dd);
                        rest += ds;
                        sf[r >> 3][r & 7] = _Float16(ds);
                    }
                };
                if (masked) form(std::true_type{});
                else form(std::false_type{});
                // dQ^T += K^T dS^T.
#pragma unroll
                for (int cs = 0; cs < 2; ++cs) {
                    TrFrag kf[DB];
#pragma unroll
                    for (int db = 0; db < DB; ++db) kf[db] = fo.transposed(kt, 2 * hb + cs, db);
                    wait_lds();
#pragma unroll
                    for (int db = 0; db < DB; ++db) acc[db] = mfma(as_f16x8(kf[db]), sf[cs], acc[db]);
                }
            }
        }
        // dS adds up to 0 over a query's keys where D is what it should be. D from
        // an FP16 O is not quite; dK, in the next launch, gets it put right.
        rest += xor32(rest);
        if (h == 0) rests[turn][wave][fr] = rest;
        if (__any(non_finite(acc)) && lane == 0) overflow = 1;
        __syncthreads();
        if (up == 0.0f || overflow == 0) break;
        up = 0.0f;
        load(0);
    }
    const float down = down_by(up);
    if (qi < length && h == 0 && turn == 0) {
        float rest = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) rest += rests[g][wave][fr];
        dsum[row_at] = __builtin_fmaf(rest, down, dd);
    }
    _Float16* rows = lds + (G - 1) * W * HD * 32 * 2;   // behind the turns' sums
    if (join_turns<HD, W, G>(reinterpret_cast<float*>(lds), acc, wave, turn, lane))
        write_rows<HD>(rows, acc, scale * down, wave * 32 + fr, h);
    __syncthreads();
    copy_rows<HD, threads_of(kQueryTurns)>(rows, length - row0, [&](int row) {
        return dq + q_at + size_t(row0 + row) * st.q;
    });
}

// ---------------------------------------------------------------- backward: dK, dV

// 128 keys (32 a wave) of one head of k and v; walks the 64-query tiles at or
// after its first key, of the group's query heads in turn. A lane holds one key
// and 16 queries per 32-query half, whose lse and D come from LDS.
//
// With parts > 1 a workgroup takes `share` of the group's heads and leaves FP32
// sums ([part][token][kv head][HD], dK then dV) for packed_backward_join: heads
// of k and v are few where groups are large, and so are workgroups then.
template <int HD>
__global__ void __launch_bounds__(threads_of(kKeyTurns<HD>), HD == 64 ? 2 : 1)
packed_backward_dkdv(_Float16* __restrict__ dk, _Float16* __restrict__ dv,
                     const _Float16* __restrict__ q, const _Float16* __restrict__ k,
                     const _Float16* __restrict__ v, const _Float16* __restrict__ dout,
                     const float* __restrict__ lse, const float* __restrict__ dsum,
                     const int4* __restrict__ plan, float* __restrict__ sums, int tokens,
                     int kv_heads, int group, int share, Strides st, float c, float scale) {
    constexpr int kTile = Tile<HD>::kHalves, KK = HD / 16, DB = HD / 32;
    constexpr int W = kRowWaves, G = kKeyTurns<HD>;
    // [buf][group][Q, dO]; behind them [buf][group][lse, D] and the overflow flag.
    constexpr int kTiles = 2 * G * 2 * kTile, kStats = 2 * G * 2 * 64;
    __shared__ __attribute__((aligned(16))) _Float16 lds[kTiles + (kStats + 4) * 2];
    float(*rowstat)[2][64] = reinterpret_cast<float(*)[2][64]>(lds + kTiles);
    int& overflow = *reinterpret_cast<int*>(lds + kTiles + kStats * 2);
    Work w;
    const int parts = group / share;
    if (!work_of(plan, int(blockIdx.x), kv_heads * parts, tokens, &w)) return;
    if (threadIdx.x == 0) overflow = 0;
    const int part = w.head % parts;
    w.head /= parts;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W;
    const int turn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / W;
    const int fr = lane & 31, h = lane >> 5;
    const Frags<HD> fo(lane);
    const int length = w.length;
    // The list's long blocks are the last of their sequences; as keys the first
    // ones have the most queries.
    const int block = (length + kPackedBlock - 1) / kPackedBlock - 1 - w.block;
    const int row0 = block * kPackedBlock;
    const size_t kv_at = size_t(w.begin) * st.kv + size_t(w.head) * HD;
    const int k0 = row0 + wave * 32;
    const int ki = k0 + fr;

    f32x16 dka[DB], dva[DB];   // 2^up dK^T, dV^T [d][key]
    float up = kUp;
    const int first = row0 / 64;
    const int per_head = (length + 63) / 64 - first;
    const int tiles = per_head * share, steps = (tiles + G - 1) / G;
    // A step's lse and D, of wave 0's lanes, go to LDS at the step's start, when
    // its tiles are there as well.
    float lv = 0.0f, dv0 = 0.0f;
    auto note = [&](int i) {
        if (wave != 0) return;
        const int buf = (i & 1) * G + turn;
        rowstat[buf][0][lane] = __builtin_fmaf(lv, kLog2e, -up);
        rowstat[buf][1][lane] = dv0;
    };
    auto stage = [&](int i) {
        const int at_tile = G * i + turn;
        if (at_tile >= tiles) return;
        const int buf = (i & 1) * G + turn, g = at_tile / per_head;
        const int tile = first + at_tile - g * per_head;
        const int head = w.head * group + part * share + g;
        _Float16* t = lds + buf * 2 * kTile;
        const int qq = 64 * tile + lane;
        lv = dv0 = 0.0f;
        if (wave == 0 && qq < length) {
            const size_t at = size_t(head) * tokens + w.begin + qq;
            lv = lse[at];
            dv0 = dsum[at];
        }
        const size_t row = size_t(w.begin) + 64 * tile;
        load_tile<HD, W>(t, q + row * st.q + size_t(head) * HD, length - 64 * tile, st.q, wave, lane);
        load_tile<HD, W>(t + kTile, dout + row * st.o + size_t(head) * HD, length - 64 * tile, st.o,
                         wave, lane);
    };
    // K and V go through the buffers: the second step's, and the first's for
    // want of room with one turn.
    _Float16* keys = lds + 2 * G * kTile;
    _Float16* values = G == 1 ? lds : keys + 2 * kTile;
    load_block<HD, W * G>(keys, k + kv_at + size_t(row0) * st.kv, length - row0, st.kv,
                          wave + W * turn, lane);
    load_block<HD, W * G>(values, v + kv_at + size_t(row0) * st.kv, length - row0, st.kv,
                          wave + W * turn, lane);
    if constexpr (G > 1) stage(0);
    wait_vmcnt<0>();
    block_sync();
    f16x8 kf[KK], vf[KK];
    block_frags<HD>(kf, keys, fo, wave);
    block_frags<HD>(vf, values, fo, wave);
    if constexpr (G == 1) {
        block_sync();
        stage(0);
    }
    for (;;) {
#pragma unroll
        for (int db = 0; db < DB; ++db) dka[db] = dva[db] = f32x16{};
        int tile = first + turn % per_head;
        for (int i = 0; i < steps; ++i) {
            const int buf = (i & 1) * G + turn;
            wait_vmcnt<0>();
            note(i);
            __syncthreads();
            const _Float16* qt = lds + buf * 2 * kTile;
            const _Float16* gt = qt + kTile;
            const float* l2 = rowstat[buf][0];
            const float* dd = rowstat[buf][1];
            if (i + 1 < steps) stage(i + 1);
            const int qbase = 64 * tile;
            tile += G;
            while (tile >= first + per_head) tile -= per_head;
            if (G * i + turn >= tiles) break;
            if (qbase + 63 < k0) continue;        // every query before every key of the wave
            const bool masked = qbase < k0 + 31 || qbase + 63 >= length;
#pragma unroll
            for (int qh = 0; qh < 2; ++qh) {
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    s = mfma(fo.row(qt, qh, kk), kf[kk], s);
                    dp = mfma(fo.row(gt, qh, kk), vf[kk], dp);
                }
                f16x8 pf[2], sf[2];
                auto form = [&](auto mask) {
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const int qr = 32 * qh + 8 * a + 4 * h;   // query row in the tile, + e
                        const f32x4 l4 = *reinterpret_cast<const f32x4*>(l2 + qr);
                        const f32x4 d4 = *reinterpret_cast<const f32x4*>(dd + qr);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = 4 * a + e;
                            float p = __builtin_amdgcn_exp2f(s[r] * c - l4[e]);
                            if constexpr (mask) {
                                if (ki > qbase + qr + e || qbase + qr + e >= length) p = 0.0f;
                            }
                            pf[a >> 1][4 * (a & 1) + e] = _Float16(p);
                            sf[a >> 1][4 * (a & 1) + e] = _Float16(p * (dp[r] - d4[e]));
                        }
                    }
                };
                if (masked) form(std::true_type{});
                else form(std::false_type{});
                // dV^T += dO^T P^T and dK^T += Q^T dS^T, a 16-query slice at a time.
#pragma unroll
                for (int cs = 0; cs < 2; ++cs) {
                    TrFrag gf[DB], tf[DB];
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        gf[db] = fo.transposed(gt, 2 * qh + cs, db);
                        tf[db] = fo.transposed(qt, 2 * qh + cs, db);
                    }
                    wait_lds();
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        dva[db] = mfma(as_f16x8(gf[db]), pf[cs], dva[db]);
                        dka[db] = mfma(as_f16x8(tf[db]), sf[cs], dka[db]);
                    }
                }
            }
        }
        if (up == 0.0f) break;
        if (__any(non_finite(dka)) && lane == 0) overflow = 1;
        __syncthreads();
        if (overflow == 0) break;
        up = 0.0f;
        stage(0);
    }
    const float down = down_by(up);
    const size_t at = kv_at + size_t(row0) * st.kv;
    _Float16* rows = lds + (G - 1) * W * HD * 32 * 2;   // behind the turns' sums
    bool mine = false;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        f32x16* acc = which == 0 ? dka : dva;
        mine = join_turns<HD, W, G>(reinterpret_cast<float*>(lds), acc, wave, turn, lane);
        if (parts > 1) continue;
        if (mine) write_rows<HD>(rows, acc, which == 0 ? scale * down : down, wave * 32 + fr, h);
        __syncthreads();
        copy_rows<HD, threads_of(kKeyTurns<HD>)>(rows, length - row0, [&](int row) {
            return (which == 0 ? dk : dv) + at + size_t(row) * st.kv;
        });
    }
    if (parts == 1 || !mine || ki >= length) return;
    float* to = sums + ((size_t(part) * tokens + w.begin + ki) * kv_heads + w.head) * HD;
    const size_t dv_at = size_t(parts) * tokens * kv_heads * HD;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int d = 32 * db + 8 * a + 4 * h;
            auto four = [&](const f32x16& acc) {
                return f32x4{acc[4 * a], acc[4 * a + 1], acc[4 * a + 2], acc[4 * a + 3]} * down;
            };
            *reinterpret_cast<f32x4*>(to + d) = four(dka[db]);
            *reinterpret_cast<f32x4*>(to + dv_at + d) = four(dva[db]);
        }
}

// The parts' sums in order, of kJoinRows of a block's rows and one head: 8
// values a thread and step. (All 128 rows a workgroup leave most CUs idle:
// 16 heads on 2 of width 128 over 4,133 tokens 47 -> 11.6 us.)
constexpr int kJoinRows = 16;
template <int HD>
__global__ void __launch_bounds__(kThreads)
packed_backward_join(_Float16* __restrict__ dk, _Float16* __restrict__ dv,
                     const float* __restrict__ sums, const int4* __restrict__ plan, int tokens,
                     int kv_heads, int parts, int stride, float scale) {
    Work w;
    if (!work_of(plan, int(blockIdx.x), kv_heads, tokens, &w)) return;
    const int row0 = w.block * kPackedBlock + int(blockIdx.y) * kJoinRows;
    const int rows = min(w.length - row0, kJoinRows);
    const size_t step = size_t(tokens) * kv_heads * HD, dv_at = step * parts;
    for (int i = threadIdx.x; i < rows * (HD / 8); i += kThreads) {
        const size_t token = size_t(w.begin) + row0 + i / (HD / 8);
        const int d = i % (HD / 8) * 8;
        const float* from = sums + (token * kv_heads + w.head) * HD + d;
        const size_t to = token * stride + size_t(w.head) * HD + d;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            f32x4 low = {}, high = {};
            for (int p = 0; p < parts; ++p) {
                const float* at = from + which * dv_at + p * step;
                low += *reinterpret_cast<const f32x4*>(at);
                high += *reinterpret_cast<const f32x4*>(at + 4);
            }
            const float by = which == 0 ? scale : 1.0f;
            f16x8 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = _Float16(low[e] * by);
                v[4 + e] = _Float16(high[e] * by);
            }
            *reinterpret_cast<f16x8*>((which == 0 ? dk : dv) + to) = v;
        }
    }
}

// How many parts the heads of a group go into for dK and dV: the fewest equal
// ones that give the GPU two workgroups a CU (256 CUs).
size_t group_parts(const flint_packed_shape& s) {
    const size_t group = s.heads / s.kv_heads, blocks = packed_items(s) * s.kv_heads;
    size_t parts = 1;
    while (parts < group && (blocks * parts < 512 || group % parts != 0)) ++parts;
    return parts;
}

// D, one FP32 value a query and head (padded to 16 bytes).
size_t dsum_values(const flint_packed_shape& s) { return (s.heads * s.tokens + 3) / 4 * 4; }

template <int HD>
hipError_t forward(void* o, void* lse, const void* q, const void* k, const void* v,
                   const void* plan, const flint_packed_shape& s, float scale,
                   hipStream_t stream) {
    hipLaunchKernelGGL(packed_forward<HD>, dim3(unsigned(packed_items(s) * s.heads)),
                       dim3(threads_of(kForwardTurns)), 0, stream, static_cast<_Float16*>(o),
                       static_cast<float*>(lse),
                       static_cast<const _Float16*>(q), static_cast<const _Float16*>(k),
                       static_cast<const _Float16*>(v), static_cast<const int4*>(plan),
                       int(s.tokens), int(s.heads), int(s.heads / s.kv_heads),
                       Strides{int(s.q_stride), int(s.kv_stride), int(s.o_stride)},
                       std::fabs(scale) * kLog2e, scale < 0.0f);
    return hipGetLastError();
}

template <int HD>
hipError_t backward(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k,
                    const void* v, const void* o, const void* lse, const void* plan,
                    const flint_packed_shape& s, float scale, void* workspace, hipStream_t stream) {
    const Strides st{int(s.q_stride), int(s.kv_stride), int(s.o_stride)};
    auto* dsum = static_cast<float*>(workspace);
    const int group = int(s.heads / s.kv_heads);
    hipLaunchKernelGGL(packed_backward_dq<HD>, dim3(unsigned(packed_items(s) * s.heads)),
                       dim3(threads_of(kQueryTurns)), 0, stream, static_cast<_Float16*>(dq), dsum,
                       static_cast<const _Float16*>(q), static_cast<const _Float16*>(k),
                       static_cast<const _Float16*>(v), static_cast<const _Float16*>(o),
                       static_cast<const _Float16*>(dout), static_cast<const float*>(lse),
                       static_cast<const int4*>(plan), int(s.tokens), int(s.heads), group, st,
                       scale * kLog2e, scale);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const size_t parts = group_parts(s), blocks = packed_items(s) * s.kv_heads;
    float* sums = dsum + dsum_values(s);
    hipLaunchKernelGGL(packed_backward_dkdv<HD>, dim3(unsigned(blocks * parts)),
                       dim3(threads_of(kKeyTurns<HD>)), 0, stream, static_cast<_Float16*>(dk),
                       static_cast<_Float16*>(dv),
                       static_cast<const _Float16*>(q), static_cast<const _Float16*>(k),
                       static_cast<const _Float16*>(v), static_cast<const _Float16*>(dout),
                       static_cast<const float*>(lse), static_cast<const float*>(dsum),
                       static_cast<const int4*>(plan), sums, int(s.tokens), int(s.kv_heads), group,
                       group / int(parts), st, scale * kLog2e, scale);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || parts == 1) return e;
    hipLaunchKernelGGL(packed_backward_join<HD>, dim3(unsigned(blocks), kPackedBlock / kJoinRows),
                       dim3(kThreads), 0, stream,
                       static_cast<_Float16*>(dk), static_cast<_Float16*>(dv),
                       static_cast<const float*>(sums), static_cast<const int4*>(plan),
                       int(s.tokens), int(s.kv_heads), int(parts), int(s.kv_stride), scale);
    return hipGetLastError();
}

}  // namespace

size_t packed_backward_workspace(const flint_packed_shape& s) {
    const size_t parts = group_parts(s);
    const size_t sums = parts == 1 ? 0 : 2 * parts * s.tokens * s.kv_heads * s.head_width;
    return (dsum_values(s) + sums) * 4;
}

hipError_t launch_packed_plan(void* plan, const void* offsets, const flint_packed_shape& s,
                              hipStream_t stream) {
    // The longest possible sequence's blocks fit the buckets.
    int shift = 0;
    while (((s.tokens / kPackedBlock + 1) >> shift) >= size_t(kBuckets)) ++shift;
    hipLaunchKernelGGL(packed_plan, dim3(1), dim3(kPlanThreads), 0, stream,
                       static_cast<int4*>(plan), static_cast<const int*>(offsets),
                       int(s.sequences), int(s.tokens), int(packed_items(s)), shift);
    return hipGetLastError();
}

hipError_t launch_packed_forward(void* o, void* lse, const void* q, const void* k, const void* v,
                                 const void* plan, const flint_packed_shape& s, float scale,
                                 hipStream_t stream) {
    return s.head_width == 64 ? forward<64>(o, lse, q, k, v, plan, s, scale, stream)
                              : forward<128>(o, lse, q, k, v, plan, s, scale, stream);
}

hipError_t launch_packed_backward(void* dq, void* dk, void* dv, const void* dout, const void* q,
                                  const void* k, const void* v, const void* o, const void* lse,
                                  const void* plan, const flint_packed_shape& s, float scale,
                                  void* workspace, hipStream_t stream) {
    return s.head_width == 64
               ? backward<64>(dq, dk, dv, dout, q, k, v, o, lse, plan, s, scale, workspace, stream)
               : backward<128>(dq, dk, dv, dout, q, k, v, o, lse, plan, s, scale, workspace, stream);
}

}  // namespace flint
