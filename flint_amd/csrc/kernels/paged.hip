// Attention of new tokens over a paged cache for gfx950: each new token sees the
// cached positions of its sequence and the sequence's new tokens up to itself;
// the new rows of k and v go into their pages in the same launch, and are read
// from k and v here, so no workgroup waits for another's store.
//
// The rows that share a head of K and V are taken together: row r of a sequence
// and kv head is new token r / group, query head r % group of the group. A work
// item is a block of such rows and a part of the sequence's 64- or 32-key tiles;
// the parts are joined by a second, small launch. Two kernels:
//  * few rows (up to 32: generation). Reading the cache bounds it: 2 values of
//    K and V a key and column against 4 FLOPs a row. Each wave streams tiles of
//    its own through two buffers in LDS, with no barrier until the results of the
//    workgroup's two waves are joined at the end. A tile's loads go out once the
//    pages of the one behind it are known, and that lookup is waited for with the
//    loads before it: other workgroups of the CU cover it, where there are any (long
//    caches 4.9 to 5.3 TB/s, 64 short ones 3.1). Until its first tile is there a
//    workgroup takes some 6 us (its item, the pages, the rows), so four small ones
//    share a CU (two at width 128): 64 sequences of 512 positions, 12 heads of 64,
//    take 29 us so, and 50 with one workgroup of four waves and tiles of 64 keys
//    (16 sequences of 4,096: 46 and 66).
//  * many rows (chunks of prompts). Each wave takes 32 of 128 rows, and the four
//    share the tiles, as in packed.hip. Here the lookup comes behind the next tile's
//    loads, so a tile's products wait for them.
#include <hip/hip_runtime.h>
#include <hip/hip_runtime.h>

#include "kernels/paged_parts.h"

namespace flint {
namespace {

// Where the rows of a tile's loads lie in the pages: lane u has load u's offset
// (halves) and the bytes there that hold cached positions with a page. One
// vector load of the table serves a whole tile, a tile ahead of its use (taken
// load by load, the table's latency bound the kernel). The offsets are formed at
// once, so the wave waits for the entries there, and for the loads before them.
struct Where {
    unsigned low, high, held;
};

// Reads the rows of K and V of one sequence and kv head, wherever they lie.
template <int HD, int KEYS>
struct Reader {
    using T = Tile<HD>;
    static constexpr int kLoads = KEYS / T::kLoadRows;   // of a tile
    const PagedArgs& a;
    const int* table;
    int kv, cached, total;
    const _Float16 *k, *v;   // the sequence's first new row of this head
    int row, lane;           // this lane's row of a load

    __device__ __forceinline__ Reader(const PagedArgs& args, const Item& it, int head, int lane_)
        : a(args), table(args.table + size_t(it.s) * args.max_pages), kv(head),
          cached(it.seq.cached), total(it.seq.cached + it.seq.count),
          k(args.k + size_t(it.seq.first) * args.kv_stride + size_t(head) * HD),
          v(args.v + size_t(it.seq.first) * args.kv_stride + size_t(head) * HD),
          row(lane_ / T::kChunks), lane(lane_) {}

    __device__ __forceinline__ Where find(int t) const {
        const int p0 = t * KEYS + (lane % kLoads) * T::kLoadRows;
        const int column = column_of(a, p0);
        const int page = p0 < cached ? table[column] : -1;   // cached ends inside the table
        const bool ok = page >= 0 && page < a.pages;
        const size_t from =
            ok ? (size_t(unsigned(page)) * unsigned(a.page_rows) +
                  unsigned(kv * a.page_size + p0 - column * a.page_size)) * HD
               : 0;
        return {unsigned(from), unsigned(from >> 32),
                ok ? unsigned(min(cached - p0, T::kLoadRows)) * HD * 2 : 0u};
    }

    // Bit u: load u's cached positions, if any, have a page.
    __device__ __forceinline__ unsigned valid(const Where& w, int t) const {
        const int p0 = t * KEYS + (lane % kLoads) * T::kLoadRows;
        return unsigned(__ballot(lane < kLoads && (w.held != 0 || p0 >= cached)));
    }

    static __device__ __forceinline__ void into(_Float16* lds, const _Float16* from, unsigned bytes,
                                                unsigned at) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc_of(from, bytes), (__attribute__((address_space(3))) void*)(lds_half*)lds, 16, at, 0,
            0, 0);
    }

    // Load u of tile t of K and of V: one load each at least. Rows of no
    // position, or of no page, are zeros.
    __device__ __forceinline__ void load(_Float16* kt, _Float16* vt, const Where& w, int t,
                                         int u) const {
        const int p0 = t * KEYS + u * T::kLoadRows;
        const int chunk = (lane % T::kChunks) ^ T::key(u * T::kLoadRows + row);
        const size_t from = size_t(unsigned(__builtin_amdgcn_readlane(int(w.high), u))) << 32 |
                            unsigned(__builtin_amdgcn_readlane(int(w.low), u));
        const unsigned held = unsigned(__builtin_amdgcn_readlane(int(w.held), u));
        const unsigned at = unsigned(row * HD + chunk * 8) * 2;
        if (p0 + T::kLoadRows <= cached || p0 >= total) {
            into(kt + u * 512, a.k_pages + from, held, at);
            into(vt + u * 512, a.v_pages + from, held, at);
        } else if (p0 + row < cached) {
            into(kt + u * 512, a.k_pages + from, held, at);
            into(vt + u * 512, a.v_pages + from, held, at);
        } else {
            const int skip = max(p0 - cached, 0);   // new rows before this load's
            const int rows = min(total - cached - skip, T::kLoadRows);
            const unsigned bytes = unsigned((rows - 1) * a.kv_stride + HD) * 2;
            const unsigned here = unsigned((p0 + row - cached - skip) * a.kv_stride + chunk * 8) * 2;
            into(kt + u * 512, k + size_t(skip) * a.kv_stride, bytes, here);
            into(vt + u * 512, v + size_t(skip) * a.kv_stride, bytes, here);
        }
    }
};

// The new rows of k and v that start in a block of query rows go to their
// pages; a block's part 0 does it.
template <int HD, int THREADS>
__device__ __forceinline__ void store_new(const PagedArgs& a, const Item& it, int head,
                                          int rows_of_block) {
    if (it.part != 0) return;
    const int from = (it.block * rows_of_block + a.group - 1) / a.group;
    const int to = min(((it.block + 1) * rows_of_block + a.group - 1) / a.group, it.seq.count);
    for (int i = threadIdx.x; i < (to - from) * (HD / 8); i += THREADS) {
        const int place = from + i / (HD / 8), d = i % (HD / 8) * 8;
        const int p = it.seq.cached + place, column = column_of(a, p);
        if (column >= a.max_pages) continue;
        const int page = a.table[size_t(it.s) * a.max_pages + column];
        if (page < 0 || page >= a.pages) continue;
        const size_t src = size_t(it.seq.first + place) * a.kv_stride + size_t(head) * HD + d;
        const size_t dst =
            ((size_t(page) * a.kv_heads + head) * a.page_size + (p - column * a.page_size)) * HD + d;
        *reinterpret_cast<f16x8*>(a.k_pages + dst) = *reinterpret_cast<const f16x8*>(a.k + src);
        *reinterpret_cast<f16x8*>(a.v_pages + dst) = *reinterpret_cast<const f16x8*>(a.v + src);
    }
}

template <int HD>
__global__ void __launch_bounds__(kFewThreads, HD == 64 ? 2 : 1) paged_few(PagedArgs a) {
    using P = Plan<HD, false>;
    using R = Reader<HD, P::kKeys>;
    constexpr int kTile = P::kKeys * HD, kW = kFewWaves;
    __shared__ __attribute__((aligned(16))) _Float16 lds[kW * 2 * 2 * kTile];   // [wave][buf][K, V]
    __shared__ float2 wave_sums[kW][32];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 31, h = lane >> 5;
    const int head = int(blockIdx.x % unsigned(a.kv_heads));
    Item it;
    if (!find_item<HD, false>(a, int(blockIdx.x / unsigned(a.kv_heads)), lane, &it)) return;
    store_splits(a, it, head);
    const int rows = it.seq.count * a.group, first_row = it.block * kFewRows;
    const Frags<HD> fo(lane);
    Rows<HD, P::kKeys> w;
    w.load_q(a, it, head, first_row + fr, rows, h);
    const int last = it.seq.cached + (first_row + fr) / a.group;
    const R reader(a, it, head, lane);
    int from, to;
    part_of(a, it, kFewRows, P::kKeys, &from, &to);
    _Float16* mine = lds + wave * 4 * kTile;
    auto issue = [&](const Where& at, int t, int buf) __attribute__((always_inline)) {
        _Float16* kt = mine + buf * 2 * kTile;
#pragma unroll
        for (int u = 0; u < R::kLoads; ++u) reader.load(kt, kt + kTile, at, t, u);
    };
    int t = from + wave;
    Where at = reader.find(t);
    unsigned valid = reader.valid(at, t);
    if (t < to) {
        issue(at, t, 0);
        at = reader.find(t + kW);
    }
    store_new<HD, kFewThreads>(a, it, head, kFewRows);   // waits for no more than the tile does
    for (int i = 0; t < to; ++i, t += kW) {
        unsigned next = 0;
        // The other buffer's reads ended with the last tile's products.
        asm volatile("" ::: "memory");
        if (t + kW < to) {
            next = reader.valid(at, t + kW);
            const Where ahead = reader.find(t + 2 * kW);
            issue(at, t + kW, (i + 1) & 1);
            at = ahead;
            wait_vmcnt<2 * R::kLoads>();   // the newer tile's loads of K and V, at least
        } else {
            wait_vmcnt<0>();
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        const _Float16* kt = mine + (i & 1) * 2 * kTile;
        w.tile(kt, kt + kTile, fo, t * P::kKeys, valid, it.seq.cached, last, a.c, h);
        valid = next;
    }
    w.finish();
    few_result<HD, 4 * kTile>(a, it, head, w, lds, wave_sums, wave, fr, h);
}

template <int HD>
__global__ void __launch_bounds__(kThreads * kGroups, HD == 64 ? 4 : 2) paged_many(PagedArgs a) {
    using P = Plan<HD, true>;
    constexpr int kTile = Tile<HD>::kHalves;
    constexpr int kEach = Tile<HD>::kLoads / 4;   // loads of a wave, of K and of V
    __shared__ __attribute__((aligned(16))) _Float16 lds[2 * kGroups * 2 * kTile];   // [buf][group][K, V]
    __shared__ float2 sums[4][32];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int turn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int fr = lane & 31, h = lane >> 5;
    const int head = int(blockIdx.x % unsigned(a.kv_heads));
    Item it;
    if (!find_item<HD, true>(a, int(blockIdx.x / unsigned(a.kv_heads)), lane, &it)) return;
    store_splits(a, it, head);
    const int rows = it.seq.count * a.group, first_row = it.block * kManyRows + wave * 32;
    const Frags<HD> fo(lane);
    Rows<HD, P::kKeys> w;
    w.load_q(a, it, head, first_row + fr, rows, h);
    const int last = it.seq.cached + (first_row + fr) / a.group;
    const int wave_last = it.seq.cached + (min(first_row + 32, rows) - 1) / a.group;
    const Reader<HD, P::kKeys> reader(a, it, head, lane);
    int from, to;
    part_of(a, it, kManyRows, P::kKeys, &from, &to);
    auto issue = [&](const Where& at, int t, int buf) __attribute__((always_inline)) {
        _Float16* kt = lds + (buf * kGroups + turn) * 2 * kTile;
#pragma unroll
        for (int i = 0; i < kEach; ++i) reader.load(kt, kt + kTile, at, t, wave + 4 * i);
    };
    int t = from + turn;
    Where at = reader.find(t);
    unsigned next = reader.valid(at, t);
    if (t < to) {
        issue(at, t, 0);
        at = reader.find(t + kGroups);
    }
    store_new<HD, kThreads * kGroups>(a, it, head, kManyRows);
    const int steps = (to - from + kGroups - 1) / kGroups;
    for (int i = 0; i < steps; ++i, t += kGroups) {
        const unsigned valid = next;
        wait_vmcnt<0>();
        block_sync();
        if (t + kGroups < to) {
            next = reader.valid(at, t + kGroups);
            issue(at, t + kGroups, (i + 1) & 1);
            at = reader.find(t + 2 * kGroups);
        }
        // No tile for this group, no row of this wave, or none that sees it.
        if (t >= to || first_row >= rows || t * P::kKeys > wave_last) continue;
        const _Float16* kt = lds + ((i & 1) * kGroups + turn) * 2 * kTile;
        w.tile(kt, kt + kTile, fo, t * P::kKeys, valid, it.seq.cached, last, a.c, h);
    }
    wait_vmcnt<0>();
    w.finish();
    many_result<HD>(a, it, head, w, lds, sums, wave, turn, fr, h);
}

template <int HD>
__global__ void __launch_bounds__(kThreads) paged_join_few(PagedArgs a) {
    join_few<HD>(a, int(blockIdx.x / unsigned(a.heads)), int(blockIdx.x % unsigned(a.heads)),
                 int(blockIdx.y));
}

template <int HD>
__global__ void __launch_bounds__(kThreads) paged_join_many(PagedArgs a) {
    join_many<HD>(a, blockIdx.x);
}

}  // namespace

size_t paged_workspace(const flint_paged_shape& s) { return space_of(s, sizes_of(s)).bytes; }

hipError_t launch_attention_paged(void* o, void* k_pages, void* v_pages, const void* q,
                                  const void* k, const void* v, const void* offsets,
                                  const void* cached, const void* table,
                                  const flint_paged_shape& s, float scale, void* workspace,
                                  hipStream_t stream) {
    const Sizes z = sizes_of(s);
    const Space w = space_of(s, z);
    PagedArgs a = paged_args(o, q, k, v, offsets, cached, table, s, scale, z, w, workspace);
    a.k_pages = static_cast<_Float16*>(k_pages);
    a.v_pages = static_cast<_Float16*>(v_pages);
    const dim3 grid(unsigned((z.blocks + z.most) * s.kv_heads));
    const bool many = many_rows(s), wide = s.head_width == 128;
    auto* const kernel = many ? (wide ? paged_many<128> : paged_many<64>)
                              : (wide ? paged_few<128> : paged_few<64>);
    hipLaunchKernelGGL(kernel, grid, dim3(many ? kThreads * kGroups : kFewThreads), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || z.slots == 0) return e;
    // Past some 4,096 rows there are waves enough without sharing a row out.
    const size_t sets = 256 / s.head_width, places = std::min(s.max_new, s.tokens);
    if (s.sequences * places * s.heads <= 4096) {
        auto* const join = wide ? paged_join_few<128> : paged_join_few<64>;
        hipLaunchKernelGGL(join, dim3(unsigned(s.sequences * s.heads), unsigned(places)),
                           dim3(kThreads), 0, stream, a);
    } else {
        auto* const join = wide ? paged_join_many<128> : paged_join_many<64>;
        const size_t waves = s.tokens * ((s.heads + sets - 1) / sets);
        hipLaunchKernelGGL(join, dim3(unsigned((waves + 3) / 4)), dim3(kThreads), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace flint
