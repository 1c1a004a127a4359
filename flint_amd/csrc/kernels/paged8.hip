// Attention of new tokens over a paged cache of 8-bit values for gfx950, and their
// storing: paged.hip's work items and tiles, with the cached rows decoded on their way
// into LDS.
//
// A value of the cache is an e4m3 number times a power of two from 2^-15 to 2^8, which
// FP16 holds exactly: its subnormals reach 2^-24 = 2^-9 2^-15, and rows are stored with
// nothing past 240 at 2^8. So a decoded tile is the FP16 tile that packed.hip's and
// paged.hip's products read, and only the cache's own rounding is left.
//
// Reading the cache bounds few rows, at half of paged.hip's bytes. Codes go to LDS
// directly, two tiles ahead of their use: held in registers so long they spilled. K's
// are decoded as they become operands (a lane has one row, and its scale), V's into a
// tile of halves, for the transposing reads. Where rows are many, a tile's four waves
// decode a quarter of it each. The new rows, FP16 as they were given, lie in tiles of
// their own in front of the cached ones, so that no tile mixes the two.
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

// 16 codes of a row, and their values.
__device__ __forceinline__ void decode(const i32x4& codes, float scale, f16x8* low, f16x8* high) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale, false);
        const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], scale, true);
        f16x8& to = j < 2 ? *low : *high;
        to[4 * (j & 1)] = a[0];
        to[4 * (j & 1) + 1] = a[1];
        to[4 * (j & 1) + 2] = b[0];
        to[4 * (j & 1) + 3] = b[1];
    }
}

// Reads the cached rows of one sequence and kv head in tiles of KEYS positions. Codes
// lie in LDS as rows of HD bytes, 16-byte chunk c of row r at position c ^ key(r): 8 bytes
// of one chunk of 32 consecutive rows fall on each bank twice at most.
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
        return HD == 64 ? (row >> 2) & 3 : (row >> 1) & 7;
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
        f16x8 low, high;
        decode(c, scale, &low, &high);
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

// A tile's softmax and product with V (halves): products(s, zero) gives the scores, of
// which the keys up to `limit` (the lane's own) are seen, of the runs of 8 in `valid`; all
// of them where `whole` says so.
template <int HD, int KEYS, class Products>
__device__ __forceinline__ void take_tile(Rows<HD, KEYS>& w, const Products& products,
                                          const _Float16* vt, const Frags<HD>& fo, bool whole,
                                          int limit, unsigned valid, float c, int h) {
    constexpr int HB = KEYS / 32;
    auto scores = [&](f32x16 (&s)[HB], unsigned zero) __attribute__((always_inline)) {
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) s[hb] = f32x16{};
        products(s, zero);
        if (whole) return c;
        const int seen = limit - 4 * h + int(zero);
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[hb][r] = 32 * hb + result_row(r, 0) <= seen && (valid >> (4 * hb + (r >> 2)) & 1)
                               ? s[hb][r] * c
                               : -INFINITY;
        return 1.0f;
    };
    w.take(vt, fo, scores);
}

// The same with K a tile of halves.
template <int HD, int KEYS>
__device__ __forceinline__ void tile(Rows<HD, KEYS>& w, const _Float16* kt, const _Float16* vt,
                                     const Frags<HD>& fo, bool whole, int limit, unsigned valid,
                                     float c, int h) {
    using R = Rows<HD, KEYS>;
    take_tile(w, [&](f32x16 (&s)[R::HB], unsigned zero) __attribute__((always_inline)) {
#pragma unroll
        for (int kk = 0; kk < R::KK; ++kk)
#pragma unroll
            for (int hb = 0; hb < R::HB; ++hb)
                s[hb] = mfma(fo.row(kt + zero, hb, kk), w.q[kk], s[hb]);
    }, vt, fo, whole, limit, valid, c, h);
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

// Few rows. A wave's LDS: kRing tiles of codes (K and V each), and one tile of V's
// halves; the new rows' K goes through the last tile of codes.
template <int HD>
__global__ void __launch_bounds__(kFewThreads, HD == 64 ? 2 : 1) paged8_few(Paged8Args a) {
    using P = Plan<HD, false>;
    constexpr int kKeys = P::kKeys, kW = kFewWaves, kRing = 3;
    using C = Cached<HD, kKeys>;
    using R = Rows<HD, kKeys>;
    constexpr int kCodes = kKeys * HD;                      // bytes of a tile of K
    constexpr int kWave = (kRing + 1) * 2 * kCodes;         // bytes of a wave
    constexpr int kBatch = 64 / C::kRuns;                   // tiles of a load of the table
    constexpr unsigned kAll = (1u << C::kRuns) - 1;
    // One LDS object: with several the compiler waits for the loads under way.
    __shared__ __attribute__((aligned(16))) unsigned char lds[kW * kWave + kW * 32 * sizeof(float2)];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 31, h = lane >> 5;
    const int head = int(blockIdx.x % unsigned(a.p.kv_heads));
    Item it;
    if (!find_item<HD, false, true>(a.p, int(blockIdx.x / unsigned(a.p.kv_heads)), lane, &it))
        return;
    store_splits(a.p, it, head);
    const int rows = it.seq.count * a.p.group, first_row = it.block * kFewRows;
    const int cached = it.seq.cached;
    const Frags<HD> fo(lane);
    R w;
    const C reader(a, it, head, lane);
    int fresh, from, to;
    part_of8(a.p, it, kFewRows, kKeys, &fresh, &from, &to);
    unsigned char* const mine = lds + wave * kWave;
    auto codes_at = [&](int slot) { return mine + slot * 2 * kCodes; };
    _Float16* const vt = reinterpret_cast<_Float16*>(codes_at(kRing));
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
    if (takes_new) {
        _Float16* kt = reinterpret_cast<_Float16*>(codes_at(kRing - 1));
        load_new<HD, kKeys>(a.p, it, head, 0, kt, vt, 0, 1, lane);
    }
    int entries = 0, ahead = 0;        // of this batch of tiles, of the next
    int scales[kRing];                 // of a tile: lane l K's row l, or V's row l - 32
    unsigned valid[kRing];
    auto issue = [&](int n, int slot) __attribute__((always_inline)) {
        const int t = tile_of(n), batch = n % kBatch * C::kRuns;
        const int own = __shfl(entries, batch + fr / 8);
        const unsigned runs = unsigned(__ballot(reader.held(entries)) >> batch) & kAll;
        const int left = cached - t * kKeys;   // a run past the cache counts as there
        valid[slot] = runs | (left >= kKeys ? 0u : kAll << ((left + 7) / 8)) & kAll;
        scales[slot] = (h ? a.v_scales : a.k_scales)[reader.place(own, t * kKeys + fr).scale];
        unsigned char *const k = codes_at(slot), *const v = k + kCodes;
#pragma unroll
        for (int u = 0; u < C::kLoads; ++u)
            reader.load(k + u * 1024, v + u * 1024, __shfl(entries, batch + reader.row_of(u) / 8), t,
                        u);
    };
    if (count > 0) {
        entries = look(0);
        ahead = look(kBatch);
#pragma unroll
        for (int n = 0; n < kRing - 1; ++n) issue(n, n);
    }
    w.load_q(a.p, it, head, first_row + fr, rows, h);
    if (takes_new) {
        if (count > 0) wait_vmcnt<(kRing - 1) * 2 * C::kLoads>();
        else wait_vmcnt<0>();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        tile(w, reinterpret_cast<const _Float16*>(codes_at(kRing - 1)), vt, fo, false,
             (first_row + fr) / a.p.group, kAll, a.p.c, h);
        asm volatile("" ::: "memory");
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
        wait_vmcnt<(kRing - 1) * 2 * C::kLoads>();   // the newer tiles' loads, at least
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        const unsigned char* const k = codes_at(slot);
        const int t = tile_of(n), limit = cached - 1 - t * kKeys;
#pragma unroll
        for (int u = 0; u < C::kLoads; ++u) {
            const int row = reader.row_of(u);
            reader.put(k + kCodes + u * 1024, vt, u, row <= limit && (valid[slot] >> (row / 8) & 1),
                       scale_of(__shfl(scales[slot], 32 + row)));
        }
        const float k_scale = scale_of(__shfl(scales[slot], fr));
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        take_tile(w, [&](f32x16 (&s)[1], unsigned zero) __attribute__((always_inline)) {
            // 16 codes of a row are two k-steps' operands of either half of the wave:
            // lane half h has columns 16 kk + 8h ..
#pragma unroll
            for (int kk = 0; kk < R::KK; ++kk) {
                const i32x2 c = *reinterpret_cast<const i32x2*>(
                    k + zero + fr * HD + ((kk ^ C::key(fr)) * 16 + 8 * h));
                f16x8 f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[j], k_scale, false);
                    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[j], k_scale, true);
                    f[4 * j] = lo[0];
                    f[4 * j + 1] = lo[1];
                    f[4 * j + 2] = hi[0];
                    f[4 * j + 3] = hi[1];
                }
                s[0] = mfma(f, w.q[kk], s[0]);
            }
        }, vt, fo, limit >= kKeys - 1 && valid[slot] == kAll, limit, valid[slot], a.p.c, h);
    };
    for (int n = 0; n < count; n += kRing) {
        step(n, std::integral_constant<int, 0>{});
        if (n + 1 >= count) break;
        step(n + 1, std::integral_constant<int, 1>{});
        if (n + 2 >= count) break;
        step(n + 2, std::integral_constant<int, 2>{});
    }
    wait_vmcnt<0>();   // the loads past the last tile, before the LDS is used again
    w.finish();
    few_result<HD, kWave / 2>(a.p, it, head, w, reinterpret_cast<_Float16*>(lds),
                              reinterpret_cast<float2(*)[32]>(lds + kW * kWave), wave, fr, h);
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

// The new rows of one kv head in the block that token t leads (its sequence's first new
// token there), of K and then of V: the block's scale, its older rows rounded again where
// that grows, the new ones. A wave takes it; HD / 8 lanes a row.
template <int HD>
__device__ __forceinline__ void store_block(const Paged8Args& a, int t, int head, int lane) {
    constexpr int kLanes = HD / 8, kRows = 64 / kLanes;
    const int s = sequence_at(a.p, t, lane);
    if (s < 0) return;
    const Sequence q = sequence_of(a.p, s);
    const int place = t - q.first, p = q.cached + place, size = 1 << a.block_shift;
    const int column = column_of(a.p, p), in = p - column * a.p.page_size, before = in & (size - 1);
    if ((place != 0 && before != 0) || column >= a.p.max_pages) return;
    const int page = a.p.table[size_t(s) * a.p.max_pages + column];
    if (page < 0 || page >= a.p.pages) return;
    const int fresh = min(size - before, q.count - place);
    const int lane_row = lane / kLanes, d = lane % kLanes * 8;
    const size_t at = size_t(page) * a.p.kv_heads + head;
    const size_t block = (at * a.p.page_size + (in - before)) * HD + d;
    const size_t source = size_t(t) * a.p.kv_stride + size_t(head) * HD + d;
    const size_t scale = at * a.blocks + (in >> a.block_shift);
    for (int which = 0; which < 2; ++which) {
        unsigned char* const pages = which ? a.v_pages : a.k_pages;
        unsigned char* const scales = which ? a.v_scales : a.k_scales;
        const _Float16* const x = (which ? a.p.v : a.p.k) + source;
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
        int e = exponent_of(most);
        if (before != 0) {
            const int was = scale_byte(scales[scale]) - 127;
            if (e > was) {
                const float up = scale_of(was + 127);
                const float by = __builtin_bit_cast(float, (127 - e) << 23);
                for (int r = lane_row; r < before; r += kRows) {
                    auto* row = reinterpret_cast<i32x2*>(pages + block + size_t(r) * HD);
                    const i32x2 codes = *row;
                    i32x2 out;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const auto low =
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], up, false);
                        const auto high =
                            __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[j], up, true);
                        const float y[4] = {float(low[0]), float(low[1]), float(high[0]),
                                            float(high[1])};
                        out[j] = encode(y, by, e);
                    }
                    *row = out;
                }
            }
            e = max(e, was);
        }
        const float by = __builtin_bit_cast(float, (127 - e) << 23);
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

// Joins the parts (the first `joins` workgroups) and stores the new rows.
template <int HD, bool FEW>
__global__ void __launch_bounds__(kThreads) paged8_finish(Paged8Args a, unsigned joins,
                                                          unsigned places) {
    if (blockIdx.x < joins) {
        if constexpr (FEW) {
            const unsigned row = blockIdx.x / places;
            join_few<HD>(a.p, int(row / unsigned(a.p.heads)), int(row % unsigned(a.p.heads)),
                         int(blockIdx.x % places));
        } else {
            join_many<HD>(a.p, blockIdx.x);
        }
        return;
    }
    const unsigned id = (blockIdx.x - joins) * (kThreads / 64) +
                        __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = int(id / unsigned(a.p.kv_heads)), head = int(id % unsigned(a.p.kv_heads));
    if (t < a.p.tokens) store_block<HD>(a, t, head, threadIdx.x & 63);
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
    auto* const kernel = many ? (wide ? paged8_many<128> : paged8_many<64>)
                              : (wide ? paged8_few<128> : paged8_few<64>);
    hipLaunchKernelGGL(kernel, grid, dim3(many ? kThreads * kGroups : kFewThreads), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    // As paged.hip joins them. Below 2^24 workgroups: tokens x heads is at most 2^25.
    const size_t sets = 256 / s.head_width, places = std::min(s.max_new, s.tokens);
    const size_t stores = (s.tokens * s.kv_heads + 3) / 4;
    const bool few = s.sequences * places * s.heads <= 4096;
    const size_t joins = z.slots == 0 ? 0
                         : few ? s.sequences * places * s.heads
                               : (s.tokens * ((s.heads + sets - 1) / sets) + 3) / 4;
    auto* const finish = few ? (wide ? paged8_finish<128, true> : paged8_finish<64, true>)
                             : (wide ? paged8_finish<128, false> : paged8_finish<64, false>);
    hipLaunchKernelGGL(finish, dim3(unsigned(joins + stores)), dim3(kThreads), 0, stream, a,
                       unsigned(joins), unsigned(places));
    return hipGetLastError();
}

}  // namespace flint
