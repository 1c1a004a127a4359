// Shared by the attention kernels over a paged cache (paged.hip, and paged8.hip for a
// cache of 8-bit values): how the work is cut into items, a tile's softmax and
// products for 32 rows, the joining of waves and parts, and the sizes that follow.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common/common.h"
#include "kernels/attention_tiles.h"
#include "kernels/kernels.h"

namespace flint {
namespace {

constexpr int kThreads = 256;   // 4 waves
constexpr int kFewWaves = 2, kFewThreads = 64 * kFewWaves;
constexpr int kGroups = 2;      // of 4 waves, where rows are many
constexpr int kFewRows = 32, kManyRows = 128;
// Workgroups aimed at: what the GPU holds at once at width 64 (few rows: four a
// CU, or six over 8-bit values; many: two), half of it at 128; and the fewest tiles that
// a part of a sequence takes. With 1,024 and with 1,536 over 8-bit values, one new token:
// 64 sequences to 8,192 positions, 8 heads of K and V of 128, 170 and 136 us, 64 to 1,023,
// 12 of 64, 24.7 and 22.1; 17 to 32 rows (32 heads on 8): 64 sequences of 8 new tokens to
// 4,096 at width 128 108 and 97, at 64 53 and 50, 16 of 5 at 128 37 and 33, but 200 of 2 to
// 1,000, 32 heads on 2 of 128, 31 and 38.
constexpr int kFewTarget = 1024, kFewOwnTarget = 1536, kManyTarget = 512;
constexpr int kFewTiles = 4, kManyTiles = 4;
// From this many tiles a workgroup on, few rows are cut for two rounds of
// workgroups, the second of which evens out what the first did not. 64 ragged
// sequences, 309,000 positions with 8 heads of K and V of 128 (150 tiles each),
// take 258 us in two rounds and 309 in one; 32 of 3,000 positions, 12 heads of 64
// (35 tiles), 65 and 62.
constexpr int kTwoRounds = 64;
// Many rows over 8-bit values are cut for two rounds where one would leave a sixth of its
// time idle and take this many tiles: a block's parts are equal, and seldom as many as the
// workgroups. 3,000 new tokens over 30,000, 12 heads on 4 of 64 (one round of 284 workgroups
// for 512), take 704 us in one round and 475 in two, 2,000 over 16,384, 12 of 64, 213 and
// 185; where a round is full, two cost their joins: 64 over 131,072, 32 on 8 of 128, 197 and
// 215; and at 21 tiles 53 and 58.
constexpr int kManyTwoRounds = 32;

template <int HD, bool MANY>
struct Plan {
    static constexpr int kRows = MANY ? kManyRows : kFewRows;
    static constexpr int kKeys = MANY ? 64 : 32;   // of a tile
    static constexpr int kLeast = MANY ? kManyTiles : kFewTiles;
};

struct PagedArgs {
    _Float16 *o, *k_pages, *v_pages;
    const _Float16 *q, *k, *v;
    const int *offsets, *cached, *table;
    int tokens, sequences, max_new, heads, kv_heads, group;
    int q_stride, kv_stride, o_stride;
    int pages, page_size, max_pages;
    unsigned magic;   // column of position p: p / 8 times magic, high word >> shift
    int shift;
    int page_rows;    // kv_heads x page_size
    float c;       // |scale| log2 e
    int negative;  // scale < 0: q enters negated
    int target;    // items a kv head aimed at
    int slots;     // parts that the workspace holds, a kv head
    int rows;      // of a part there
    int2* splits;  // [sequences]: first slot, parts
    float2* sums;  // [slots][kv_heads][rows]: maximum (log2 units), sum
    float* parts;  // [slots][kv_heads][rows][HD]
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

// The table column of a position: an exact division of p / 8 (below 2^28) by
// page_size / 8 = d, as the high word of a product. With 2^shift < d <=
// 2^(shift + 1) and magic = floor(2^(32 + shift) / d) + 1, magic d - 2^(32 +
// shift) is at most d, and 2^28 d at most 2^(29 + shift). d = 1 has magic 0.
__device__ __forceinline__ int column_of(const PagedArgs& a, int p) {
    const unsigned n = unsigned(p) >> 3;
    return int(a.magic == 0 ? n : __umulhi(n, a.magic) >> a.shift);
}

// Item `idx` of a kv head. Every item takes about the same number of tiles,
// total / target: the sequences' lengths are known only here, so each wave adds
// them up (64 sequences a step) and finds its item by a prefix sum. (Four
// sequences a lane, which saves 256 of them three chains of loads, cost as much in
// divisions: 256 sequences of 200 positions stayed at 58 us, 64 of 512 took 32
// instead of 29.)
struct Item {
    Sequence seq;
    int s, block, part, parts, slot;   // slot of the block's part 0 (parts > 1)
};
// OWN: the new rows lie in tiles of their own.
template <int HD, bool MANY, bool OWN = false>
__device__ __forceinline__ bool find_item(const PagedArgs& a, int idx, int lane, Item* it) {
    using P = Plan<HD, MANY>;
    auto blocks_of = [&](const Sequence& q) { return (q.count * a.group + P::kRows - 1) / P::kRows; };
    auto tiles_of = [&](const Sequence& q) {
        if (q.count == 0) return 0;
        if (OWN)
            return int(unsigned(q.cached + P::kKeys - 1) / P::kKeys +
                       unsigned(q.count + P::kKeys - 1) / P::kKeys);
        return int(unsigned(q.cached + q.count + P::kKeys - 1) / P::kKeys);
    };
    long long total = 0;
    Sequence q{};
    for (int s0 = 0; s0 < a.sequences; s0 += 64) {
        q = Sequence{};
        if (s0 + lane < a.sequences) q = sequence_of(a, s0 + lane);
        total += (long long)(blocks_of(q)) * tiles_of(q);
    }
    // In two words of 24 bits: the rows' blocks add up to at most 2^21 and tiles
    // to 2^26, and only offsets that decrease pass that.
    total = min(total, 1ll << 48);
    total = ((long long)(wave_sum(int(total >> 24))) << 24) + wave_sum(int(total & 0xffffff));
    constexpr long long kMost = 1 << 30;   // more tiles than any sequence has
    const bool twice = !MANY && total >= (long long)(kTwoRounds) * a.target;
    int target = twice ? 2 * a.target : a.target;
    int each = max(P::kLeast, int(min(kMost, (total + target - 1) / target)));
    // The target is what the GPU holds at once: parts that round up past it would
    // run behind the others. (One step of sequences only; the parts of more are
    // many anyway.)
    auto fit = [&] {
        for (int i = 0; i < 8 && a.sequences <= 64; ++i) {
            const int parts = (tiles_of(q) + each - 1) / each;
            if (wave_sum(blocks_of(q) * parts) <= target || __ballot(parts > 1) == 0) break;
            each += (each + 7) / 8;
        }
    };
    fit();
    if (MANY && OWN && total >= (long long)(kManyTwoRounds) * target &&
        6 * total < 5 * (long long)(each) * target) {
        target *= 2;
        each = int(min(kMost, (total + target - 1) / target));
        fit();
    }
    int before = 0, slots = 0;
    for (int s0 = 0; s0 < a.sequences; s0 += 64) {
        if (a.sequences > 64) {
            q = Sequence{};
            if (s0 + lane < a.sequences) q = sequence_of(a, s0 + lane);
        }
        const int parts = (tiles_of(q) + each - 1) / each;
        const int items = blocks_of(q) * parts;
        const int upto = wave_scan(items);
        const int held = wave_scan(parts > 1 ? items : 0);
        const unsigned long long past = __ballot(before + upto > idx);
        if (past != 0) {
            const int at = __ffsll(past) - 1;
            auto get = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
            it->s = s0 + at;
            it->seq = {get(q.first), get(q.count), get(q.cached)};
            it->parts = get(parts);
            const int in = idx - before - get(upto - items);
            it->block = in / it->parts;
            it->part = in - it->block * it->parts;
            it->slot = slots + get(held) - get(parts > 1 ? items : 0) + it->block * it->parts;
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(held, 63);
    }
    return false;
}

// One tile of KEYS keys for a wave's 32 rows: scores, probabilities and sum,
// O^T += V^T P^T. valid: bit u for load u's pages.
template <int HD, int KEYS>
struct Rows {
    static constexpr int KK = HD / 16, DB = HD / 32, HB = KEYS / 32;
    f16x8 q[KK];
    float m = kFloor, l = 0.0f;
    bool started = false;
    f32x16 acc[DB] = {};

    __device__ __forceinline__ void tile(const _Float16* kt, const _Float16* vt,
                                         const Frags<HD>& fo, int kbase, unsigned valid, int cached,
                                         int last, float c, int h) {
        constexpr unsigned kAll = unsigned((1ull << (KEYS / Tile<HD>::kLoadRows)) - 1);
        auto scores = [&](f32x16 (&s)[HB], unsigned zero) __attribute__((always_inline)) {
#pragma unroll
            for (int hb = 0; hb < HB; ++hb) s[hb] = f32x16{};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int hb = 0; hb < HB; ++hb) s[hb] = mfma(fo.row(kt + zero, hb, kk), q[kk], s[hb]);
            if (kbase + KEYS <= cached && valid == kAll) return c;
            // Keys after the query: the register's key is a constant plus 4h.
            const int seen = last - kbase - 4 * h + int(zero);
#pragma unroll
            for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[hb][r] = 32 * hb + result_row(r, 0) <= seen ? s[hb][r] * c : -INFINITY;
            if (valid != kAll) {
                const int fresh = cached - kbase - 4 * h;
                const unsigned paged = HD == 64 ? valid : valid >> h;
#pragma unroll
                for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        constexpr int kRows = Tile<HD>::kLoadRows;
                        const int in = 32 * hb + result_row(r, 0);
                        if (!(paged >> (in / kRows) & 1) && in < fresh) s[hb][r] = -INFINITY;
                    }
            }
            return 1.0f;
        };
        take(vt, fo, scores);
    }

    // O^T and the sum by a tile whose scores and their factor scores(s, zero) gives,
    // as probabilities() takes it.
    template <class Scores>
    __device__ __forceinline__ void take(const _Float16* vt, const Frags<HD>& fo,
                                         const Scores& scores) {
        f16x8 p[2 * HB];
        l += probabilities<HB>(p, scores, &m, &started, [&](float by) __attribute__((always_inline)) {
            l *= by;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= by;
        });
#pragma unroll
        for (int cs = 0; cs < 2 * HB; ++cs) {
            TrFrag vf[DB];
#pragma unroll
            for (int db = 0; db < DB; ++db) vf[db] = fo.transposed(vt, cs, db);
            wait_lds();
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = mfma(as_f16x8(vf[db]), p[cs], acc[db]);
        }
    }

    // The keys' halves of a row, in lanes l and l ^ 32, become one.
    __device__ __forceinline__ void finish() { l += xor32(l); }

    // Rows `row` of the sequence (32 from the wave's first), zeros from `rows` on.
    __device__ __forceinline__ void load_q(const PagedArgs& a, const Item& it, int head, int row,
                                           int rows, int h) {
        const int place = row / a.group;
        const _Float16* at = a.q + size_t(it.seq.first + place) * a.q_stride +
                             size_t(head * a.group + row - place * a.group) * HD + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            q[kk] = row < rows ? *reinterpret_cast<const f16x8*>(at + 16 * kk) : f16x8{};
            if (a.negative) q[kk] = -q[kk];
        }
    }
};

// The tiles of a block's part: the keys up to its last row's own position.
__device__ __forceinline__ void part_of(const PagedArgs& a, const Item& it, int rows_of_block,
                                        int keys, int* from, int* to) {
    const int rows = it.seq.count * a.group;
    const int place = (min((it.block + 1) * rows_of_block, rows) - 1) / a.group;
    const int tiles = (it.seq.cached + place) / keys + 1;
    *from = int((long long)(tiles) * it.part / it.parts);
    *to = int((long long)(tiles) * (it.part + 1) / it.parts);
}

// Where the joining launch finds a sequence's parts.
__device__ __forceinline__ void store_splits(const PagedArgs& a, const Item& it, int head) {
    if (a.slots > 0 && head == 0 && it.block == 0 && it.part == 0 && threadIdx.x == 0)
        a.splits[it.s] = int2{it.slot, it.parts};
}

// Few rows: joins the workgroup's waves, which left O^T [HD][32], kWaveHalves halves
// after the one's before, and their maxima and sums; stores the rows, or the part's.
template <int HD, int kWaveHalves>
__device__ __forceinline__ void few_joined(const PagedArgs& a, const Item& it, int head,
                                           const _Float16* lds, const float2 (*wave_sums)[32]) {
    constexpr int kW = kFewWaves;
    constexpr int kOut = HD * kFewRows / kFewThreads;   // values of a thread
    static_assert(kWaveHalves >= HD * 32 * 2, "O^T of a wave");
    const int rows = it.seq.count * a.group, first_row = it.block * kFewRows;
    __syncthreads();
    const int row = threadIdx.x & 31, d0 = (threadIdx.x >> 5) * kOut;
    if (first_row + row < rows) {
        float m = kFloor, l = 0.0f, by[kW], sum[kOut] = {};
#pragma unroll
        for (int i = 0; i < kW; ++i) m = fmaxf(m, wave_sums[i][row].x);
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            by[i] = __builtin_amdgcn_exp2f(wave_sums[i][row].x - m);
            l = __builtin_fmaf(wave_sums[i][row].y, by[i], l);
        }
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            const float* part = reinterpret_cast<const float*>(lds + i * kWaveHalves);
#pragma unroll
            for (int d = 0; d < kOut; ++d)
                sum[d] = __builtin_fmaf(part[(d0 + d) * 32 + row], by[i], sum[d]);
        }
        if (it.parts == 1) {
            const int place = (first_row + row) / a.group;
            _Float16* o = a.o + size_t(it.seq.first + place) * a.o_stride +
                          size_t(head * a.group + first_row + row - place * a.group) * HD + d0;
            const float inv = 1.0f / l;
#pragma unroll
            for (int d = 0; d < kOut; d += 8) {
                f16x8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = _Float16(sum[d + e] * inv);
                *reinterpret_cast<f16x8*>(o + d) = v;
            }
        } else if (it.slot + it.part < a.slots) {
            const size_t at = (size_t(it.slot + it.part) * a.kv_heads + head) * a.rows + row;
            if (d0 == 0) a.sums[at] = float2{m, l};
#pragma unroll
            for (int d = 0; d < kOut; d += 4)
                *reinterpret_cast<f32x4*>(a.parts + at * HD + d0 + d) =
                    f32x4{sum[d], sum[d + 1], sum[d + 2], sum[d + 3]};
        }
    }
}


template <int HD, int kWaveHalves>
__device__ __forceinline__ void few_result(const PagedArgs& a, const Item& it, int head,
                                           const Rows<HD, Plan<HD, false>::kKeys>& w, _Float16* lds,
                                           float2 (*wave_sums)[32], int wave, int fr, int h) {
    // Each wave leaves O^T in its own tiles.
    float* own = reinterpret_cast<float*>(lds + wave * kWaveHalves);
#pragma unroll
    for (int db = 0; db < HD / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) own[(32 * db + result_row(r, h)) * 32 + fr] = w.acc[db][r];
    if (h == 0) wave_sums[wave][fr] = float2{w.m, w.l};
    few_joined<HD, kWaveHalves>(a, it, head, lds, wave_sums);
}

// Many rows: joins the two groups of waves and stores the rows, or the part's.
template <int HD>
__device__ __forceinline__ void many_result(const PagedArgs& a, const Item& it, int head,
                                            Rows<HD, Plan<HD, true>::kKeys>& w, _Float16* lds,
                                            float2 (*sums)[32], int wave, int turn, int fr, int h) {
    const int rows = it.seq.count * a.group, first_row = it.block * kManyRows + wave * 32;
    // The second group's sums join the first's in LDS, as in packed.hip.
    float* theirs = reinterpret_cast<float*>(lds) + wave * HD * 32;
    __syncthreads();
    if (turn != 0) {
#pragma unroll
        for (int db = 0; db < HD / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                theirs[(32 * db + result_row(r, h)) * 32 + fr] = w.acc[db][r];
        if (h == 0) sums[wave][fr] = float2{w.m, w.l};
    }
    __syncthreads();
    if (turn == 0) {
        const float2 other = sums[wave][fr];
        const float most = fmaxf(w.m, other.x);
        const float by = __builtin_amdgcn_exp2f(w.m - most);
        const float other_by = __builtin_amdgcn_exp2f(other.x - most);
        w.m = most;
        w.l = __builtin_fmaf(other.y, other_by, w.l * by);
#pragma unroll
        for (int db = 0; db < HD / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                w.acc[db][r] = __builtin_fmaf(theirs[(32 * db + result_row(r, h)) * 32 + fr],
                                              other_by, w.acc[db][r] * by);
    }
    if (it.parts == 1) {
        _Float16* block = lds + 4 * HD * 32 * 2;   // behind theirs
        if (turn == 0) write_rows<HD>(block, w.acc, 1.0f / w.l, wave * 32 + fr, h);
        __syncthreads();
        const int row0 = it.block * kManyRows;
        copy_rows<HD, kThreads * kGroups>(block, rows - row0, [&](int i) {
            const int place = (row0 + i) / a.group;
            return a.o + size_t(it.seq.first + place) * a.o_stride +
                   size_t(head * a.group + row0 + i - place * a.group) * HD;
        });
        return;
    }
    // (Offsets that decrease can make more blocks, and parts, than there are slots.)
    if (turn != 0 || first_row + fr >= rows || it.slot + it.part >= a.slots) return;
    const size_t slot =
        (size_t(it.slot + it.part) * a.kv_heads + head) * a.rows + wave * 32 + fr;
    if (h == 0) a.sums[slot] = float2{w.m, w.l};
#pragma unroll
    for (int db = 0; db < HD / 32; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(a.parts + slot * HD + 32 * db + 8 * i + 4 * h) =
                f32x4{w.acc[db][4 * i], w.acc[db][4 * i + 1], w.acc[db][4 * i + 2],
                      w.acc[db][4 * i + 3]};
}

// The sequence that token t belongs to, or -1: 64 offsets a step.
__device__ __forceinline__ int sequence_at(const PagedArgs& a, int t, int lane) {
    int low = 0, count = a.sequences;   // among low .. low + count - 1
    while (count > 1) {
        const int step = (count + 63) / 64;
        const int s = low + lane * step;
        const bool starts = lane * step < count && min(max(a.offsets[s], 0), a.tokens) <= t;
        const int at = __popcll(__ballot(starts)) - 1;
        if (at < 0) return -1;
        low += at * step;
        count = min(step, count - at * step);
    }
    const Sequence q = sequence_of(a, low);
    return t >= q.first && t < q.first + q.count ? low : -1;
}

__device__ __forceinline__ void store_joined(_Float16* o, const f32x4& sum, float by) {
    *reinterpret_cast<f16x4*>(o) = f16x4{_Float16(sum[0] * by), _Float16(sum[1] * by),
                                         _Float16(sum[2] * by), _Float16(sum[3] * by)};
}

// A row's parts in the workspace: false where it has none to join.
struct Parts {
    size_t at, step;   // of the first part's row, in rows
    int count;
};
__device__ __forceinline__ bool parts_of_row(const PagedArgs& a, const Sequence& q, int2 split,
                                             int t, int head, Parts* p) {
    const int kv = head / a.group, row = (t - q.first) * a.group + head - kv * a.group;
    // Offsets that decrease make more blocks than the grid has workgroups. A
    // sequence that got none has what lay in the workspace as its split: any two
    // numbers, so the parts are looked for in 64 bits, inside the slots alone.
    const int block = row / a.rows;
    const long long first = split.x + (long long)(block) * split.y;
    if (split.y <= 1 || split.y > a.slots || first < 0 || first > a.slots - split.y) return false;
    p->step = size_t(a.kv_heads) * a.rows;
    p->at = (size_t(first) * a.kv_heads + kv) * a.rows + (row - block * a.rows);
    p->count = split.y;
    return true;
}

// The parts' results, weighted by their maxima's distance; HD / 4 lanes (a set)
// take 4 columns of a row each.
//
// Few rows: four waves a row, whose sets take the parts in turn (a sequence may
// have a thousand) and then add up. The grid is sequences x heads and places, so
// that no search stands before the parts (16 sequences of 100: 8.0 -> 7.5 us).
template <int HD>
__device__ __forceinline__ void join_few(const PagedArgs& a, int s, int head, int place) {
    constexpr int kLanes = HD / 4, kSets = 64 / kLanes, kWaves = kThreads / 64;
    __shared__ __attribute__((aligned(16))) f32x4 wave_parts[kWaves][kLanes];
    __shared__ float wave_sums[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = lane % kLanes * 4;
    const int set = wave * kSets + lane / kLanes;
    const Sequence q = sequence_of(a, s);
    const int2 split = a.splits[s];
    if (place >= q.count) return;
    const int t = q.first + place;
    Parts p;
    if (!parts_of_row(a, q, split, t, head, &p)) return;
    float m = kFloor;
    for (int i = lane; i < p.count; i += 64) m = fmaxf(m, a.sums[p.at + i * p.step].x);
#pragma unroll
    for (int i = 32; i > 0; i /= 2) m = fmaxf(m, __shfl_xor(m, i));
    float l = 0.0f;
    f32x4 sum = {};
#pragma unroll 4
    for (int i = set; i < p.count; i += kSets * kWaves) {
        const float2 part = a.sums[p.at + i * p.step];
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.parts + (p.at + i * p.step) * HD + d);
        const float by = __builtin_amdgcn_exp2f(part.x - m);
        l = __builtin_fmaf(part.y, by, l);
        sum += v * by;
    }
#pragma unroll
    for (int i = kLanes; i < 64; i *= 2) {
        l += __shfl_xor(l, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], i);
    }
    if (lane < kLanes) wave_parts[wave][lane] = sum;
    if (lane == 0) wave_sums[wave] = l;
    __syncthreads();
    if (set != 0) return;
    l = 0.0f;
    sum = f32x4{};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        l += wave_sums[w];
        sum += wave_parts[w][lane];
    }
    store_joined(a.o + size_t(t) * a.o_stride + size_t(head) * HD + d, sum, 1.0f / l);
}

// Many rows, of few parts each: a set a row, a wave on heads of one token, since
// finding the token's sequence is a chain of loads.
template <int HD>
__device__ __forceinline__ void join_many(const PagedArgs& a, unsigned block) {
    constexpr int kLanes = HD / 4, kSets = 64 / kLanes;
    const int lane = threadIdx.x & 63, d = lane % kLanes * 4;
    const unsigned id = block * (kThreads / 64) + (threadIdx.x >> 6);
    const unsigned runs = unsigned(a.heads + kSets - 1) / kSets;   // of kSets heads
    const int t = int(id / runs), head = int(id % runs) * kSets + lane / kLanes;
    if (t >= a.tokens) return;
    const int s = sequence_at(a, t, lane);
    if (s < 0 || head >= a.heads) return;
    Parts p;
    if (!parts_of_row(a, sequence_of(a, s), a.splits[s], t, head, &p)) return;
    float m = kFloor;
#pragma unroll 4
    for (int i = 0; i < p.count; ++i) m = fmaxf(m, a.sums[p.at + i * p.step].x);
    float l = 0.0f;
    f32x4 sum = {};
#pragma unroll 4
    for (int i = 0; i < p.count; ++i) {
        const float2 part = a.sums[p.at + i * p.step];
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.parts + (p.at + i * p.step) * HD + d);
        const float by = __builtin_amdgcn_exp2f(part.x - m);
        l = __builtin_fmaf(part.y, by, l);
        sum += v * by;
    }
    store_joined(a.o + size_t(t) * a.o_stride + size_t(head) * HD + d, sum, 1.0f / l);
}

inline bool many_rows(const flint_paged_shape& s) {
    return std::min(s.max_new, s.tokens) * (s.heads / s.kv_heads) > kFewRows;
}

// What the kernels' grids and the workspace follow from. A block of rows may
// have as many parts as the longest sequence has runs of kLeast tiles; a
// sequence in p > 1 parts of `each` tiles has fewer than 2 tiles / each of them,
// so the parts of all are below twice the items aimed at. Few rows are one block
// of a sequence, and its parts hold no more rows than it can have.
struct Sizes {
    size_t target, most, blocks, slots, rows;
};
inline Sizes sizes_of(const flint_paged_shape& s, bool own = false) {
    const bool many = many_rows(s);
    const size_t group = s.heads / s.kv_heads, new_rows = std::min(s.max_new, s.tokens) * group;
    Sizes z;
    z.rows = many ? kManyRows : new_rows;
    const size_t keys = many ? 64 : 32, least = many ? kManyTiles : kFewTiles;
    const size_t target =
        (many ? kManyTarget : own ? kFewOwnTarget : kFewTarget) * 64 / s.head_width;
    z.target = std::max<size_t>(1, target / s.kv_heads);
    z.most = many && !own ? z.target : 2 * z.target;
    z.blocks = many ? std::min(s.sequences * ((new_rows + z.rows - 1) / z.rows),
                               s.tokens * group / z.rows + s.sequences)
                    : s.sequences;
    // (New rows in tiles of their own make one more at most.)
    const size_t longest =
        (s.max_pages * s.page_size + s.max_new + keys - 1) / keys + (own ? 1 : 0);
    const size_t parts = (longest + least - 1) / least;
    z.slots = parts > 1 ? std::min(2 * z.most, z.blocks * parts) : 0;
    return z;
}

// The workspace: the sequences' splits, the parts' sums, the parts.
struct Space {
    size_t sums, parts, bytes;
};
inline Space space_of(const flint_paged_shape& s, const Sizes& z) {
    const size_t rows = z.slots * s.kv_heads * z.rows;
    Space w;
    w.sums = (s.sequences * sizeof(int2) + 15) / 16 * 16;
    w.parts = w.sums + rows * sizeof(float2);
    w.bytes = z.slots == 0 ? 0 : w.parts + rows * s.head_width * 4;
    return w;
}

// A call's arguments, with k_pages and v_pages left null.
inline PagedArgs paged_args(void* o, const void* q, const void* k, const void* v,
                            const void* offsets, const void* cached, const void* table,
                            const flint_paged_shape& s, float scale, const Sizes& z, const Space& w,
                            void* workspace) {
    auto* ws = static_cast<char*>(workspace);
    const size_t eighths = s.page_size / 8;
    int shift = 0;
    while ((size_t{2} << shift) < eighths) ++shift;
    const unsigned magic = eighths == 1 ? 0u : unsigned((size_t{1} << (32 + shift)) / eighths + 1);
    return {static_cast<_Float16*>(o), nullptr, nullptr, static_cast<const _Float16*>(q),
            static_cast<const _Float16*>(k), static_cast<const _Float16*>(v),
            static_cast<const int*>(offsets), static_cast<const int*>(cached),
            static_cast<const int*>(table), int(s.tokens), int(s.sequences),
            int(std::min(s.max_new, s.tokens)), int(s.heads), int(s.kv_heads),
            int(s.heads / s.kv_heads), int(s.q_stride), int(s.kv_stride), int(s.o_stride),
            int(s.pages), int(s.page_size), int(s.max_pages), magic, shift,
            int(s.kv_heads * s.page_size), std::fabs(scale) * kLog2e, scale < 0.0f, int(z.target),
            int(z.slots), int(z.rows), reinterpret_cast<int2*>(ws),
            reinterpret_cast<float2*>(ws + w.sums), reinterpret_cast<float*>(ws + w.parts)};
}

}  // namespace
}  // namespace flint
