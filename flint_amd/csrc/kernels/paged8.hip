// Attention of new tokens over a paged cache of 8-bit values for gfx950, and their
// storing: paged.hip's work items and tiles, with the cached rows decoded on the chip.
//
// A value of the cache is an e4m3 number times a power of two from 2^-15 to 2^8, which
// FP16 holds exactly: its subnormals reach 2^-24 = 2^-9 2^-15, and rows are stored with
// nothing past 240 at 2^8. So a decoded tile is the FP16 tile that packed.hip's and
// paged.hip's products read, and only the cache's own rounding is left.
//
// Reading the cache bounds few rows, at half of paged.hip's bytes. Codes go to LDS
// directly, two tiles ahead of their use (held in registers so long they spilled), and
// are decoded as they become operands, V's behind a transposing read of bytes. Where
// rows are many, a tile's four waves decode a quarter of it each, to halves in LDS. The
// new rows, FP16 as they were given, lie in tiles of their own in front of the cached
// ones, so that no tile mixes the two. Measured, one new token a sequence: 64 sequences to
// 8,192 positions, 32 heads on 8 of 128, 136 us (4.65 TB/s; the FP16 cache 259), 3 of 50,000
// to 131,072, 12 heads of 64, 82 us (164), 64 to 1,023, 12 of 64, 21 to 22.5 (32 to 33). With
// K and V decoded to halves in LDS and 32-row products (one wave a SIMD) the first took 238.
//
// Probabilities enter the product with V as FP16, as in paged.hip; their sum is of the FP32
// values. o is then 2.9e-4 of itself from float64 (root mean squares), where storing it in
// FP16 alone leaves 2.1e-4; the cache's e4m3 values are off by up to 2^-4 of theirs. A
// second product, with what the rounding left of each probability, brings 2.1e-4 and takes
// the first of these from 136 to 138 us, the last from 22.1 to 23.4, 8 new tokens each over
// to 4,096 positions, 32 heads on 8 of 128, from 97 to 104, and where rows are many chunks of
// 500 over to 4,096, 12 heads on 4 of 64, from 39 to 52, 2,000 over 16,384, 12 of 64, from 181
// to 278 (it spills there): left out for all, so that a token's result is as exact in a batch
// of either kind.
//
// The rows are stored behind the attention by the launch that joins the parts: a block's
// scale may grow with a new row, which rewrites rows that the attention reads.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "kernels/paged_parts.h"

namespace flint {
namespace {

constexpr int kLeastByte = 112, kMostByte = 135;   // a scale of 2^(byte - 127)

struct Paged8Args {
    PagedArgs p;
    unsigned char *k_pages, *v_pages, *k_scales, *v_scales;
    int block_shift;   // 2^block_shift positions share a scale
    int blocks;        // of a page and head
};

typedef __attribute__((address_space(3))) unsigned char lds_byte;

__device__ __forceinline__ int scale_byte(int b) { return min(max(b, kLeastByte), kMostByte); }
__device__ __forceinline__ float scale_of(int b) {
    return __builtin_bit_cast(float, scale_byte(b) << 23);
}

// 8 codes' values, at one scale or at one each.
__device__ __forceinline__ f16x8 decode(const i32x2& codes, float scale) {
    f16x8 out;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale, false);
        const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale, true);
        out[4 * j] = a[0];
        out[4 * j + 1] = a[1];
        out[4 * j + 2] = b[0];
        out[4 * j + 3] = b[1];
    }
    return out;
}
__device__ __forceinline__ f16x8 decode(const i32x2& codes, const float (&scale)[8]) {
    f16x8 out;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        out[4 * j] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale[4 * j], false)[0];
        out[4 * j + 1] =
            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale[4 * j + 1], false)[1];
        out[4 * j + 2] =
            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale[4 * j + 2], true)[0];
        out[4 * j + 3] =
            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale[4 * j + 3], true)[1];
    }
    return out;
}

// Four transposing reads of bytes: of 16 lanes, 2i and 2i + 1 address the halves of row i,
// 16 bytes, of 8; lane c gets column c of them. (The builtin waits for every load under way
// into LDS. The wait stands in the same asm, so that no register is touched before it is
// filled.)
template <int OFFSET>
__device__ __forceinline__ void read_transposed(unsigned a, unsigned b, unsigned c, unsigned d,
                                                i32x2* to) {
    i32x2 r0, r1, r2, r3;
    asm volatile(
        "ds_read_b64_tr_b8 %0, %4 offset:%8\n"
        "ds_read_b64_tr_b8 %1, %5 offset:%8\n"
        "ds_read_b64_tr_b8 %2, %6 offset:%8\n"
        "ds_read_b64_tr_b8 %3, %7 offset:%8\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
        : "v"(a), "v"(b), "v"(c), "v"(d), "i"(OFFSET));
    to[0] = r0;
    to[1] = r1;
    to[2] = r2;
    to[3] = r3;
}

// Reads the cached rows of one sequence and kv head in tiles of KEYS positions. Codes
// lie in LDS as rows of HD bytes, 16-byte chunk c of row r at position c ^ key(r). Two
// reads have to spread over the banks, 32 lanes at a time: one chunk of 16 consecutive
// rows (V), and one of the 16 rows whose bit 2 is the same (K).
template <int HD, int KEYS>
struct Cached {
    static constexpr int kLanes = HD / 16;           // of a row in a load
    static constexpr int kRows = 64 / kLanes;        // of a load
    static constexpr int kLoads = KEYS / kRows;      // of a tile, of K and of V
    static constexpr int kRuns = KEYS / 8;           // runs of 8 positions, one page each
    const Paged8Args& a;
    const int* table;
    int head, cached, lane;

    __device__ __forceinline__ Cached(const Paged8Args& args, const Item& it, int kv, int lane_)
        : a(args), table(args.p.table + size_t(it.s) * args.p.max_pages), head(kv),
          cached(it.seq.cached), lane(lane_) {}

    static __device__ __forceinline__ int key(int row) {
        const int top = (row >> 4 ^ row >> 2) & 1;
        return HD == 64 ? top << 1 | (row >> 3 & 1) : top << 2 | (row >> 3 & 1) << 1 | (row >> 1 & 1);
    }
    // The row, and the first column of the 16, that this lane has of load u.
    __device__ __forceinline__ int row_of(int u) const { return u * kRows + lane / kLanes; }
    __device__ __forceinline__ int column_at(int row) const {
        return ((lane % kLanes) ^ key(row)) * 16;
    }

    // The page of the run at position p: an entry of the table, or -1 past the cache.
    __device__ __forceinline__ int entry(int p) const {
        return p < cached ? table[column_of(a.p, p)] : -1;   // cached ends inside the table
    }
    __device__ __forceinline__ bool held(int page) const { return page >= 0 && page < a.p.pages; }

    // Where position p lies: its row in the pool, its scale. Rows that hold nothing read
    // something of a page, the first where they have none, which counts for nothing.
    struct Place {
        size_t row, scale;
    };
    __device__ __forceinline__ Place place(int page, int p) const {
        const unsigned in = unsigned(p - column_of(a.p, p) * a.p.page_size);
        const size_t at =
            size_t(unsigned(held(page) ? page : 0)) * unsigned(a.p.kv_heads) + unsigned(head);
        return {at * unsigned(a.p.page_size) + in, at * unsigned(a.blocks) + (in >> a.block_shift)};
    }

    // Load u of tile t, of K and of V, 1 KB each; the lane's row lies in `page`.
    __device__ __forceinline__ void load(unsigned char* k, unsigned char* v, int page, int t,
                                         int u) const {
        const int row = row_of(u);
        const size_t from = place(page, t * KEYS + row).row * HD + column_at(row);
        auto into = [](unsigned char* lds, const unsigned char* src) {
            __builtin_amdgcn_global_load_lds(
                (__attribute__((address_space(1))) void*)const_cast<unsigned char*>(src),
                (__attribute__((address_space(3))) void*)(lds_byte*)lds, 16, 0, 0);
        };
        into(k, a.k_pages + from);
        into(v, a.v_pages + from);
    }

    // This lane's codes of load u of a tile of values as a tile of halves.
    __device__ __forceinline__ void put(const unsigned char* codes, _Float16* tile, int u, bool ok,
                                        float scale) const {
        using T = Tile<HD>;
        const int row = row_of(u), chunk = column_at(row) / 8;
        i32x4 c = *reinterpret_cast<const i32x4*>(codes + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = ok ? c[j] : 0;
        const f16x8 low = decode(i32x2{c[0], c[1]}, scale), high = decode(i32x2{c[2], c[3]}, scale);
        *reinterpret_cast<f16x8*>(tile + row * HD + (chunk ^ T::key(row)) * 8) = low;
        *reinterpret_cast<f16x8*>(tile + row * HD + ((chunk + 1) ^ T::key(row)) * 8) = high;
    }
};

// New rows `from` .. of a sequence (count in all) into a tile of KEYS rows, zeros
// behind the last: loads first, first + step, ...
template <int HD, int KEYS>
__device__ __forceinline__ void load_new(const PagedArgs& a, const Item& it, int head, int from,
                                         _Float16* kt, _Float16* vt, int first, int step, int lane) {
    using T = Tile<HD>;
    const size_t start = size_t(it.seq.first + from) * a.kv_stride + size_t(head) * HD;
    const int rows = min(it.seq.count - from, KEYS);
    const unsigned bytes = unsigned((rows - 1) * a.kv_stride + HD) * 2;
#pragma unroll
    for (int i = 0; i < KEYS / T::kLoadRows; ++i) {
        const int u = first + step * i;
        if (u >= KEYS / T::kLoadRows) break;
        const int row = u * T::kLoadRows + lane / T::kChunks;
        const unsigned at =
            unsigned(row * a.kv_stride + ((lane % T::kChunks) ^ T::key(row)) * 8) * 2;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc_of(a.k + start, bytes),
            (__attribute__((address_space(3))) void*)(lds_half*)(kt + u * 512), 16, at, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc_of(a.v + start, bytes),
            (__attribute__((address_space(3))) void*)(lds_half*)(vt + u * 512), 16, at, 0, 0, 0);
    }
}

// A tile of halves whose keys up to `limit` (the lane's own) are seen, of the runs of 8
// in `valid`; all of them where `whole` says so.
template <int HD, int KEYS>
__device__ __forceinline__ void tile(Rows<HD, KEYS>& w, const _Float16* kt, const _Float16* vt,
                                     const Frags<HD>& fo, bool whole, int limit, unsigned valid,
                                     float c, int h) {
    using R = Rows<HD, KEYS>;
    auto scores = [&](f32x16 (&s)[R::HB], unsigned zero) __attribute__((always_inline)) {
#pragma unroll
        for (int hb = 0; hb < R::HB; ++hb) s[hb] = f32x16{};
#pragma unroll
        for (int kk = 0; kk < R::KK; ++kk)
#pragma unroll
            for (int hb = 0; hb < R::HB; ++hb)
                s[hb] = mfma(fo.row(kt + zero, hb, kk), w.q[kk], s[hb]);
        if (whole) return c;
        const int seen = limit - 4 * h + int(zero);
#pragma unroll
        for (int hb = 0; hb < R::HB; ++hb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[hb][r] = 32 * hb + result_row(r, 0) <= seen && (valid >> (4 * hb + (r >> 2)) & 1)
                               ? s[hb][r] * c
                               : -INFINITY;
        return 1.0f;
    };
    w.take(vt, fo, scores);
}

// The tiles of a block's part: new rows' tiles, up to the one of the block's last row,
// then the cached ones.
__device__ __forceinline__ void part_of8(const PagedArgs& a, const Item& it, int rows_of_block,
                                         int keys, int* fresh, int* from, int* to) {
    const int rows = it.seq.count * a.group;
    const int place = (min((it.block + 1) * rows_of_block, rows) - 1) / a.group;
    *fresh = place / keys + 1;
    const int tiles = *fresh + int(unsigned(it.seq.cached + keys - 1) / unsigned(keys));
    *from = int((long long)(tiles) * it.part / it.parts);
    *to = int((long long)(tiles) * (it.part + 1) / it.parts);
}

// RB blocks of 16 rows and tiles of 32 keys: up to 16 rows (one token of up to 16 heads on
// one) take half the registers and exponentials of 32. The 16 rows of K that an MFMA takes
// are keys 8 i + 4 kb + 0 .. 3, i < 4: lane group g (of 16) then has the scores of keys
// 8g .. 8g + 7 of its query, in order, which is what the product with V wants of it, and
// one page and, from 8 positions a block on, one scale of V.
template <int HD, int RB>
struct FewRows {
    static constexpr int KK = HD / 32, DB = HD / 16;
    f16x8 q[RB][KK];
    float m[RB], l[RB];
    bool started = false;
    f32x4 acc[RB][DB] = {};

    __device__ __forceinline__ FewRows() {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) m[rb] = kFloor, l[rb] = 0.0f;
    }

    __device__ __forceinline__ void load_q(const PagedArgs& a, const Item& it, int head, int lane) {
        const int first = it.block * kFewRows, rows = it.seq.count * a.group;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int row = first + 16 * rb + (lane & 15), place = row / a.group;
            const _Float16* at = a.q + size_t(it.seq.first + place) * a.q_stride +
                                 size_t(head * a.group + row - place * a.group) * HD +
                                 8 * (lane >> 4);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                q[rb][kk] = row < rows ? *reinterpret_cast<const f16x8*>(at + 32 * kk) : f16x8{};
                if (a.negative) q[rb][kk] = -q[rb][kk];
            }
        }
    }

    // One tile: keys(kb, kk) and values(db) are operands of K and V; key 8g + i of the
    // lane's group is seen where i <= seen[rb]. (The softmax is attention_tiles.h's: the
    // reference moves at a wave's first tile and where a lane's sum passes kSumLimit.)
    template <class Keys, class Values>
    __device__ __forceinline__ void tile(const Keys& keys, const Values& values, bool whole,
                                         const int (&seen)[RB], float c) {
        f16x8 p[RB];
        for (;;) {
            // Two blocks of rows read K's operands again where the tile is done again: kept for
            // it, they took 32 registers through the softmax and others went to scratch, whose
            // loads wait for the tiles on their way (64 sequences of 8 new tokens over 4,096,
            // 32 heads on 8 of 128: 192 -> 130 us; 64-wide heads 71 -> 55).
            if constexpr (RB > 1) asm volatile("" ::: "memory");
            f32x4 s[RB][2] = {};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const f16x8 k = keys(kb, kk);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
                        s[rb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[rb][kk], s[rb][kb],
                                                                           0, 0, 0);
                }
            float by = c;
            if (!whole) {
                by = 1.0f;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        s[rb][i >> 2][i & 3] = i <= seen[rb] ? s[rb][i >> 2][i & 3] * c : -INFINITY;
            }
            const bool move = !started;
            if (move) {
                started = true;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    float mx = s[rb][0][0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[rb][i >> 2][i & 3]);
                    mx *= by;
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    const float m_new = fmaxf(m[rb], fmaxf(mx, xor32(mx)) - kBelow);
                    const float scale = __builtin_amdgcn_exp2f(m[rb] - m_new);
                    l[rb] *= scale;
#pragma unroll
                    for (int db = 0; db < DB; ++db) acc[rb][db] *= scale;
                    m[rb] = m_new;
                }
            }
            float sum[RB] = {};
            bool past = false;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float e = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(s[rb][i >> 2][i & 3], by, -m[rb]));
                    p[rb][i] = _Float16(e);
                    sum[rb] += e;
                }
                past |= sum[rb] > kSumLimit;
            }
            if (move || !__any(past)) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) l[rb] += sum[rb];
                break;
            }
            started = false;
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const f16x8 v = values(db);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                acc[rb][db] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[rb], acc[rb][db], 0, 0, 0);
        }
    }

    // Leaves O^T [HD][32] and the maxima and sums for few_joined.
    __device__ __forceinline__ void leave(float* own, float2* sums, int lane) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            l[rb] += __shfl_xor(l[rb], 16);
            l[rb] += xor32(l[rb]);
            const int row = 16 * rb + (lane & 15);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    own[(16 * db + 4 * (lane >> 4) + r) * 32 + row] = acc[rb][db][r];
            if (lane < 16) sums[row] = float2{m[rb], l[rb]};
        }
    }
};

// Few rows. A wave's LDS: kRing tiles of codes, K and V each; the new rows, as halves,
// take the place of the last two. FINE: blocks of fewer than 8 positions, so that each
// of a lane's 8 keys may have its own scale of V.
template <int HD, int RB, bool FINE>
__global__ void __launch_bounds__(kFewThreads, HD == 64 ? 4 / RB : 2) paged8_few(Paged8Args a) {
    using P = Plan<HD, false>;
    constexpr int kKeys = P::kKeys, kW = kFewWaves, kRing = 3;
    using C = Cached<HD, kKeys>;
    using R = FewRows<HD, RB>;
    constexpr int kCodes = kKeys * HD;                      // bytes of a tile of K
    constexpr int kWave = kRing * 2 * kCodes;               // bytes of a wave
    constexpr int kBatch = 64 / C::kRuns;                   // tiles of a load of the table
    constexpr unsigned kAll = (1u << C::kRuns) - 1;
    // One LDS object: with several the compiler waits for the loads under way.
    __shared__ __attribute__((aligned(16))) unsigned char lds[kW * kWave + kW * 32 * sizeof(float2)];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i16 = lane & 15;
    const int head = int(blockIdx.x % unsigned(a.p.kv_heads));
    Item it;
    if (!find_item<HD, false, true>(a.p, int(blockIdx.x / unsigned(a.p.kv_heads)), lane, &it))
        return;
    store_splits(a.p, it, head);
    const int cached = it.seq.cached;
    R w;
    const C reader(a, it, head, lane);
    int fresh, from, to;
    part_of8(a.p, it, kFewRows, kKeys, &fresh, &from, &to);
    unsigned char* const mine = lds + wave * kWave;
    auto codes_at = [&](int slot) { return mine + slot * 2 * kCodes; };
    // Tile 0 of the list is the new rows' (few rows are at most 32 new ones); the wave's
    // n-th cached tile is first + kW n, up to `end`. Past it the loads take the last one
    // again, so that every wait counts the same loads.
    const bool takes_new = from + wave == 0;
    const int first = (takes_new ? kW : from + wave) - 1, end = to - 1;
    const int count = first < end ? (end - first + kW - 1) / kW : 0;
    auto tile_of = [&](int n) { return first + kW * min(n, count - 1); };
    // Lane l has run l % kRuns of the tile l / kRuns after the batch's first.
    auto look = [&](int n) {
        return reader.entry(tile_of(n + lane / C::kRuns) * kKeys + lane % C::kRuns * 8);
    };
    _Float16* const new_k = reinterpret_cast<_Float16*>(codes_at(kRing - 2));
    _Float16* const new_v = reinterpret_cast<_Float16*>(codes_at(kRing - 1));
    if (takes_new) load_new<HD, kKeys>(a.p, it, head, 0, new_k, new_v, 0, 1, lane);
    int entries = 0, ahead = 0;        // of this batch of tiles, of the next
    int scales[kRing];                 // of a tile: lane l K's row l, or V's row l - 32
    unsigned valid[kRing];
    auto issue = [&](int n, int slot) __attribute__((always_inline)) {
        const int t = tile_of(n), batch = n % kBatch * C::kRuns;
        const unsigned runs = unsigned(__ballot(reader.held(entries)) >> batch) & kAll;
        valid[slot] = runs;
        const int own = __shfl(entries, batch + (lane & 31) / 8);
        scales[slot] =
            (lane < 32 ? a.k_scales : a.v_scales)[reader.place(own, t * kKeys + (lane & 31)).scale];
        unsigned char *const k = codes_at(slot), *const v = k + kCodes;
#pragma unroll
        for (int u = 0; u < C::kLoads; ++u)
            reader.load(k + u * 1024, v + u * 1024, __shfl(entries, batch + reader.row_of(u) / 8), t,
                        u);
    };
    constexpr int kTileLoads = 2 * C::kLoads;
    if (count > 0) {
        entries = look(0);
        ahead = look(kBatch);
#pragma unroll
        for (int n = 0; n < kRing - 2; ++n) issue(n, n);
        if (!takes_new) issue(kRing - 2, kRing - 2);
    }
    w.load_q(a.p, it, head, lane);
    if (takes_new) {
        if (count > 0) wait_vmcnt<(kRing - 2) * kTileLoads>();
        else wait_vmcnt<0>();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        using T = Tile<HD>;
        int seen[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
            seen[rb] = (it.block * kFewRows + 16 * rb + i16) / a.p.group - 8 * g;
        w.tile([&](int kb, int kk) {
            const int row = i16 / 4 * 8 + kb * 4 + i16 % 4;
            return *reinterpret_cast<const f16x8*>(new_k + row * HD + ((4 * kk + g) ^ T::key(row)) * 8);
        }, [&](int db) {
            f16x8 v;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 8 * g + j, d = 16 * db + i16;
                v[j] = new_v[row * HD + ((d / 8) ^ T::key(row)) * 8 + d % 8];
            }
            return v;
        }, false, seen, a.p.c);
        asm volatile("" ::: "memory");
        if (count > 0) issue(kRing - 2, kRing - 2);
    }
    // Where this lane's operands lie in the first tile of codes, the others' being a
    // constant further on: 8 of row 8 (i / 4) + 4 kb + i % 4 of K; of V, for the transposing
    // read, 8 of the 16 columns of row 8g + i / 2.
    const unsigned base = unsigned(reinterpret_cast<uintptr_t>((lds_byte*)mine));
    unsigned k_at[2][R::KK], v_at[R::DB];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int kk = 0; kk < R::KK; ++kk) {
            const int row = i16 / 4 * 8 + kb * 4 + i16 % 4;
            k_at[kb][kk] =
                base + unsigned(row * HD + (((2 * kk + g / 2) ^ C::key(row)) * 16) + 8 * (g & 1));
            asm volatile("" : "+v"(k_at[kb][kk]));
        }
#pragma unroll
    for (int db = 0; db < R::DB; ++db) {
        const int row = 8 * g + i16 / 2;
        v_at[db] = base + unsigned(row * HD + ((db ^ C::key(row)) * 16) + 8 * (i16 & 1));
        asm volatile("" : "+v"(v_at[db]));
    }
    auto step = [&](int n, auto slot_c) __attribute__((always_inline)) {
        constexpr int slot = decltype(slot_c)::value, next = (slot + kRing - 1) % kRing;
        const int ahead_n = n + kRing - 1;
        if (ahead_n % kBatch == 0) {
            entries = ahead;
            ahead = look(ahead_n + kBatch);
        }
        // The slot's last reads were a step ago.
        asm volatile("" ::: "memory");
        issue(ahead_n, next);
        wait_vmcnt<(kRing - 1) * kTileLoads>();   // the newer tiles' loads, at least
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        const int t = tile_of(n);
        // The keys of the lane's group that are cached positions with a page: its first
        // `keys`. V's codes behind them become zeros.
        const int left = cached - t * kKeys;
        const bool whole = left >= kKeys && valid[slot] == kAll;
        const int keys = valid[slot] >> g & 1 ? min(max(left - 8 * g, 0), 8) : 0;
        const unsigned low = keys >= 4 ? ~0u : (1u << 8 * keys) - 1;
        const unsigned high = keys >= 8 ? ~0u : keys <= 4 ? 0u : (1u << 8 * (keys - 4)) - 1;
        // V's codes, four columns' operands at a time: all of them before the softmax,
        // where they have registers that long.
        constexpr bool kEarly = HD * RB <= 128;
        i32x2 raw[kEarly ? R::DB : 4];
        auto read_v = [&](int db, i32x2* to) __attribute__((always_inline)) {
            read_transposed<(2 * slot + 1) * kCodes>(v_at[db], v_at[db + 1], v_at[db + 2],
                                                     v_at[db + 3], to);
        };
        if constexpr (kEarly) {
#pragma unroll
            for (int db = 0; db < R::DB; db += 4) read_v(db, raw + db);
        }
        float k_scale[2], v_scale[FINE ? 8 : 1];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
            k_scale[kb] = scale_of(__shfl(scales[slot], i16 / 4 * 8 + kb * 4 + i16 % 4));
#pragma unroll
        for (int j = 0; j < (FINE ? 8 : 1); ++j)
            v_scale[j] = scale_of(__shfl(scales[slot], 32 + 8 * g + j));
        int seen[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) seen[rb] = keys - 1;
        w.tile([&](int kb, int kk) __attribute__((always_inline)) {
            const auto* at = (__attribute__((address_space(3))) const i32x2*)(
                uintptr_t(k_at[kb][kk] + unsigned(2 * slot * kCodes)));
            const i32x2 c = *at;
            return decode(c, k_scale[kb]);
        }, [&](int db) __attribute__((always_inline)) {
            if constexpr (!kEarly)
                if (db % 4 == 0) read_v(db, raw);
            const i32x2 r = raw[kEarly ? db : db % 4];
            const i32x2 c = {int(unsigned(r[0]) & low), int(unsigned(r[1]) & high)};
            if constexpr (!FINE) return decode(c, v_scale[0]);
            else return decode(c, v_scale);
        }, whole, seen, a.p.c);
    };
    for (int n = 0; n < count; n += kRing) {
        step(n, std::integral_constant<int, 0>{});
        if (n + 1 >= count) break;
        step(n + 1, std::integral_constant<int, 1>{});
        if (n + 2 >= count) break;
        step(n + 2, std::integral_constant<int, 2>{});
    }
    wait_vmcnt<0>();   // the loads past the last tile, before the LDS is used again
    asm volatile("" ::: "memory");
    auto* sums = reinterpret_cast<float2(*)[32]>(lds + kW * kWave);
    w.leave(reinterpret_cast<float*>(mine), sums[wave], lane);
    few_joined<HD, kWave / 2>(a.p, it, head, reinterpret_cast<const _Float16*>(lds), sums);
}

// Many rows. LDS: two buffers of tiles of halves for either group of waves, and each
// wave's share of the next tile's codes, a quarter of its rows.
template <int HD>
__global__ void __launch_bounds__(kThreads * kGroups, HD == 64 ? 4 : 2) paged8_many(Paged8Args a) {
    using P = Plan<HD, true>;
    constexpr int kKeys = P::kKeys, kTile = Tile<HD>::kHalves;
    using C = Cached<HD, kKeys>;
    constexpr int kEach = C::kLoads / 4;     // loads of a wave, of K and of V
    constexpr int kHalves = 2 * kGroups * 2 * kTile;
    constexpr unsigned kAll = (1u << C::kRuns) - 1;
    __shared__ __attribute__((aligned(16))) _Float16 lds[kHalves + 4 * kGroups * kEach * 1024];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int turn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int fr = lane & 31, h = lane >> 5;
    const int head = int(blockIdx.x % unsigned(a.p.kv_heads));
    Item it;
    if (!find_item<HD, true, true>(a.p, int(blockIdx.x / unsigned(a.p.kv_heads)), lane, &it)) return;
    store_splits(a.p, it, head);
    const int rows = it.seq.count * a.p.group, first_row = it.block * kManyRows + wave * 32;
    const Frags<HD> fo(lane);
    Rows<HD, kKeys> w;
    w.load_q(a.p, it, head, first_row + fr, rows, h);
    const int wave_place = (min(first_row + 32, rows) - 1) / a.p.group;
    const C reader(a, it, head, lane);
    int fresh, from, to;
    part_of8(a.p, it, kManyRows, kKeys, &fresh, &from, &to);
    auto buffer = [&](int i) { return lds + ((i & 1) * kGroups + turn) * 2 * kTile; };
    unsigned char* const codes = reinterpret_cast<unsigned char*>(lds + kHalves) +
                                 (turn * 4 + wave) * kEach * 2048;   // [load][K, V]
    unsigned char k_bytes[kEach], v_bytes[kEach];
    unsigned valid = kAll;
    // Tile t of the list on its way: new rows into buffer i, cached ones as codes.
    auto issue = [&](int t, int i, int entries) __attribute__((always_inline)) {
        if (t < fresh) {
            _Float16* kt = buffer(i);
            load_new<HD, kKeys>(a.p, it, head, t * kKeys, kt, kt + kTile, wave, 4, lane);
            return;
        }
        const int p0 = (t - fresh) * kKeys, run = p0 + lane % C::kRuns * 8;
        valid = unsigned(__ballot(lane < C::kRuns && (reader.held(entries) || run >= it.seq.cached)));
#pragma unroll
        for (int i4 = 0; i4 < kEach; ++i4) {
            const int u = wave + 4 * i4, row = reader.row_of(u);
            const int page = __shfl(entries, row / 8);
            const size_t scale = reader.place(page, p0 + row).scale;
            k_bytes[i4] = a.k_scales[scale];
            v_bytes[i4] = a.v_scales[scale];
            reader.load(codes + i4 * 2048, codes + i4 * 2048 + 1024, page, t - fresh, u);
        }
    };
    auto look = [&](int t) {
        return t >= fresh && t < to ? reader.entry((t - fresh) * kKeys + lane % C::kRuns * 8) : -1;
    };
    int t = from + turn, entries = look(t);
    if (t < to) {
        const int next = look(t + kGroups);
        issue(t, 0, entries);
        entries = next;
    }
    const int steps = (to - from + kGroups - 1) / kGroups;
    for (int i = 0; i < steps; ++i, t += kGroups) {
        _Float16 *const kt = buffer(i), *const vt = kt + kTile;
        const int limit = it.seq.cached - 1 - (t - fresh) * kKeys;
        const unsigned runs = valid;
        wait_vmcnt<0>();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        if (t < to && t >= fresh) {
            // This buffer's reads ended before the last step's barrier.
#pragma unroll
            for (int i4 = 0; i4 < kEach; ++i4) {
                const int u = wave + 4 * i4, row = reader.row_of(u);
                const bool ok = row <= limit && (runs >> (row / 8) & 1);
                reader.put(codes + i4 * 2048, kt, u, ok, scale_of(k_bytes[i4]));
                reader.put(codes + i4 * 2048 + 1024, vt, u, ok, scale_of(v_bytes[i4]));
            }
        }
        block_sync();
        if (t + kGroups < to) {
            const int next = look(t + 2 * kGroups);
            issue(t + kGroups, i + 1, entries);
            entries = next;
        }
        // No tile for this group, no row of this wave, or none that sees it.
        if (t >= to || first_row >= rows || (t < fresh && t * kKeys > wave_place)) continue;
        const int sees = t < fresh ? (first_row + fr) / a.p.group - t * kKeys : limit;
        tile(w, kt, vt, fo, t >= fresh && limit >= kKeys - 1 && runs == kAll, sees,
             t < fresh ? kAll : runs, a.p.c, h);
    }
    wait_vmcnt<0>();
    w.finish();
    many_result<HD>(a.p, it, head, w, lds, reinterpret_cast<float2(*)[32]>(codes - (turn * 4 + wave) * kEach * 2048),
                    wave, turn, fr, h);
}

// The least exponent e, -15 to 8, with `most` (finite, not negative) at most 448 2^e:
// 448 = 1.75 2^8.
__device__ __forceinline__ int exponent_of(float most) {
    const int bits = __builtin_bit_cast(int, most);
    const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
    return min(max(e, kLeastByte - 127), kMostByte - 127);
}

// Four values in e4m3 at 2^-e of their size (by = 2^-e), nearest even; what would pass
// e4m3's 448, or FP16's range at 2^8, goes to the largest that does not.
__device__ __forceinline__ int encode(const float (&x)[4], float by, int e) {
    const float most = e == kMostByte - 127 ? 240.0f : 448.0f;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = __builtin_isfinite(x[i]) ? fminf(fmaxf(x[i] * by, -most), most) : NAN;
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], low, true);
}

// The new rows of sequence s from `place` on to the end of that one's block, of K or V of
// a kv head: the block's scale, its older rows rounded again where that grows, the new ones.
// A wave takes every `step`-th of the kv heads' K and V; HD / 8 lanes a row.
template <int HD>
__device__ __forceinline__ void store_block(const Paged8Args& a, int s, const Sequence& q, int place,
                                            int unit, int step, int lane) {
    constexpr int kLanes = HD / 8, kRows = 64 / kLanes;
    const int p = q.cached + place, size = 1 << a.block_shift;
    const int column = column_of(a.p, p), in = p - column * a.p.page_size, before = in & (size - 1);
    if (column >= a.p.max_pages) return;
    const int page = a.p.table[size_t(s) * a.p.max_pages + column];
    if (page < 0 || page >= a.p.pages) return;
    const int fresh = min(size - before, q.count - place);
    const int lane_row = lane / kLanes, d = lane % kLanes * 8;
    for (; unit < 2 * a.p.kv_heads; unit += step) {
        const int head = unit >> 1, which = unit & 1;
        const size_t at = size_t(page) * a.p.kv_heads + head;
        const size_t block = (at * a.p.page_size + (in - before)) * HD + d;
        const size_t scale = at * a.blocks + (in >> a.block_shift);
        unsigned char* const pages = which ? a.v_pages : a.k_pages;
        unsigned char* const scales = which ? a.v_scales : a.k_scales;
        const _Float16* const x =
            (which ? a.p.v : a.p.k) + size_t(q.first + place) * a.p.kv_stride + size_t(head) * HD + d;
        const int was = before != 0 ? scale_byte(scales[scale]) - 127 : kLeastByte - 127;
        float most = 0.0f;
        for (int r = lane_row; r < fresh; r += kRows) {
            const f16x8 v = *reinterpret_cast<const f16x8*>(x + size_t(r) * a.p.kv_stride);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = __builtin_fabsf(float(v[i]));
                most = f < INFINITY ? fmaxf(most, f) : most;
            }
        }
#pragma unroll
        for (int i = 1; i < 64; i *= 2) most = fmaxf(most, __shfl_xor(most, i));
        const int e = max(exponent_of(most), was);
        const float by = __builtin_bit_cast(float, (127 - e) << 23);
        if (e > was) {
            const float up = scale_of(was + 127);
            for (int r = lane_row; r < before; r += kRows) {
                auto* row = reinterpret_cast<i32x2*>(pages + block + size_t(r) * HD);
                const f16x8 v = decode(*row, up);
                const float low[4] = {float(v[0]), float(v[1]), float(v[2]), float(v[3])};
                const float high[4] = {float(v[4]), float(v[5]), float(v[6]), float(v[7])};
                *row = i32x2{encode(low, by, e), encode(high, by, e)};
            }
        }
        for (int r = lane_row; r < fresh; r += kRows) {
            const f16x8 v = *reinterpret_cast<const f16x8*>(x + size_t(r) * a.p.kv_stride);
            const float low[4] = {float(v[0]), float(v[1]), float(v[2]), float(v[3])};
            const float high[4] = {float(v[4]), float(v[5]), float(v[6]), float(v[7])};
            *reinterpret_cast<i32x2*>(pages + block + size_t(before + r) * HD) =
                i32x2{encode(low, by, e), encode(high, by, e)};
        }
        if (lane == 0) scales[scale] = (unsigned char)(e + 127);
    }
}

// Joins the parts (the first `joins` workgroups) and stores the new rows, `waves` waves a
// block: `slots` blocks of each sequence, or, with slots 0, the block that each token leads
// (its sequence's first new one there).
struct Finish {
    unsigned joins, places, waves, slots;
};
template <int HD, bool FEW>
__global__ void __launch_bounds__(kThreads) paged8_finish(Paged8Args a, Finish f) {
    if (blockIdx.x < f.joins) {
        if constexpr (FEW) {
            const unsigned row = blockIdx.x / f.places;
            join_few<HD>(a.p, int(row / unsigned(a.p.heads)), int(row % unsigned(a.p.heads)),
                         int(blockIdx.x % f.places));
        } else {
            join_many<HD>(a.p, blockIdx.x);
        }
        return;
    }
    const int lane = threadIdx.x & 63;
    const unsigned id = (blockIdx.x - f.joins) * (kThreads / 64) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned block = id / f.waves, size = 1u << a.block_shift;
    int s, place;
    Sequence q;
    if (f.slots != 0) {
        s = int(block / f.slots);
        if (s >= a.p.sequences) return;
        q = sequence_of(a.p, s);
        place = max(0, int((unsigned(q.cached) / size + block % f.slots) * size) - q.cached);
        if (place >= q.count) return;
    } else {
        s = int(block) < a.p.tokens ? sequence_at(a.p, int(block), lane) : -1;
        if (s < 0) return;
        q = sequence_of(a.p, s);
        place = int(block) - q.first;
        if (place != 0 && (unsigned(q.cached + place) & (size - 1)) != 0) return;
    }
    store_block<HD>(a, s, q, place, int(id % f.waves), int(f.waves), lane);
}

}  // namespace

size_t paged8_workspace(const flint_paged_shape& s) { return space_of(s, sizes_of(s, true)).bytes; }

hipError_t launch_attention_paged8(void* o, void* k_pages, void* k_scales, void* v_pages,
                                   void* v_scales, const void* q, const void* k, const void* v,
                                   const void* offsets, const void* cached, const void* table,
                                   const flint_paged_shape& s, size_t block, float scale,
                                   void* workspace, hipStream_t stream) {
    const Sizes z = sizes_of(s, true);
    const Space w = space_of(s, z);
    int shift = 0;
    while ((size_t{1} << shift) < block) ++shift;
    const Paged8Args a{paged_args(o, q, k, v, offsets, cached, table, s, scale, z, w, workspace),
                       static_cast<unsigned char*>(k_pages), static_cast<unsigned char*>(v_pages),
                       static_cast<unsigned char*>(k_scales), static_cast<unsigned char*>(v_scales),
                       shift, int(s.page_size >> shift)};
    const dim3 grid(unsigned((z.blocks + z.most) * s.kv_heads));
    const bool many = many_rows(s), wide = s.head_width == 128;
    const size_t rows = std::min(s.max_new, s.tokens) * (s.heads / s.kv_heads);
    auto few_kernel = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        return rows <= 16 ? (block < 8 ? paged8_few<HD, 1, true> : paged8_few<HD, 1, false>)
                          : (block < 8 ? paged8_few<HD, 2, true> : paged8_few<HD, 2, false>);
    };
    auto* const kernel = many   ? (wide ? paged8_many<128> : paged8_many<64>)
                         : wide ? few_kernel(std::integral_constant<int, 128>{})
                                : few_kernel(std::integral_constant<int, 64>{});
    hipLaunchKernelGGL(kernel, grid, dim3(many ? kThreads * kGroups : kFewThreads), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    // As paged.hip joins them. A wave stores K or V of one kv head's block; where the
    // sequences' lengths leave more slots for blocks than there are tokens, the blocks are
    // looked for token by token, four waves a token (2,000 tokens of one sequence, 8 kv heads
    // of 128, blocks of 32: 11.5 us by sequence, 63 by token).
    const size_t sets = 256 / s.head_width, places = std::min(s.max_new, s.tokens);
    const size_t units = 2 * s.kv_heads, slots = (places + block - 2) / block + 1;
    const bool by_sequence =
        s.sequences * slots <= s.tokens && s.sequences * slots * units <= (size_t{1} << 22);
    const size_t waves = by_sequence ? units : std::min<size_t>(units, 4);
    const size_t stores = ((by_sequence ? s.sequences * slots : s.tokens) * waves + 3) / 4;
    const bool few = s.sequences * places * s.heads <= 4096;
    const size_t joins = z.slots == 0 ? 0
                         : few ? s.sequences * places * s.heads
                               : (s.tokens * ((s.heads + sets - 1) / sets) + 3) / 4;
    auto* const finish = few ? (wide ? paged8_finish<128, true> : paged8_finish<64, true>)
                             : (wide ? paged8_finish<128, false> : paged8_finish<64, false>);
    hipLaunchKernelGGL(finish, dim3(unsigned(joins + stores)), dim3(kThreads), 0, stream, a,
                       Finish{unsigned(joins), unsigned(places), unsigned(waves),
                              by_sequence ? unsigned(slots) : 0u});
    return hipGetLastError();
}

}  // namespace flint
