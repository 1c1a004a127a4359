// Tiles of 64 rows of one head (64 or 128 halves a row) in LDS, and the MFMA
// fragments read from them, for the attention over packed sequences (packed.hip)
// and over a paged cache (paged.hip). The layouts are attention.hip's: scores
// transposed (a lane holds one query), probabilities used as the next product's
// operand straight from their registers.
#pragma once

#include <hip/hip_runtime.h>

#include "kernels/gemm_common.h"

namespace flint {
namespace {

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* base, unsigned bytes) {
    const uint64_t v = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
    void* p = reinterpret_cast<void*>((uint64_t(hi) << 32) | lo);
    return __builtin_amdgcn_make_buffer_rsrc(p, 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// lgkmcnt(0): the transposing reads are inline asm, invisible to the
// compiler's wait insertion.
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_sched_barrier(0);
}

// The value of lane ^ 32 (the other half of the wave holds the same query).
__device__ __forceinline__ float xor32(float v) { return __shfl_xor(v, 32); }

// Inclusive prefix sum over the wave by lane exchanges within the vector unit:
// 1, 2, 4 and 8 lanes up within 16, then the last lane of a row of 16, and of
// the first 32, to those above.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ int wave_sum(int v) {
    return __builtin_amdgcn_readlane(wave_scan(v), 63);
}

// A tile holds rows of HD halves back to back, 16-byte chunk c of row r at
// chunk position c ^ key(r). Two reads have to spread over the banks: the 16
// lanes of a row fragment take one chunk of 16 consecutive rows, those of a
// transposing read two neighbouring chunks of 4 consecutive rows. A row of 128
// halves covers all 64 banks, so its 16 rows need 16 keys; one of 64 covers
// half of them, so pairs of rows share 8 keys. Rotating the row bits left by
// one makes the keys of 4 neighbouring rows differ above bit 0, which keeps
// their chunk pairs apart.
template <int HD>
struct Tile {
    static_assert(HD == 64 || HD == 128, "head widths");
    static constexpr int kHalves = 64 * HD;
    static constexpr int kChunks = HD / 8;          // of a row
    static constexpr int kLoadRows = 64 / kChunks;  // rows of one load: 64 lanes, 16 bytes each
    static constexpr int kLoads = 64 / kLoadRows;   // loads of a tile

    static __device__ __forceinline__ int key(int row) {
        if constexpr (HD == 64) {
            const int r = (row >> 1) & 7;
            return ((r << 1) | (r >> 2)) & 7;
        } else {
            const int r = row & 15;
            return ((r << 1) | (r >> 3)) & 15;
        }
    }
};

// Rows 0 .. 63 at `from` (rows `stride` halves apart; those from `left` on read
// as zeros) into a tile by direct-to-LDS loads, shared out over WAVES waves.
template <int HD, int WAVES>
__device__ __forceinline__ void load_tile(_Float16* tile, const _Float16* from, int left, int stride,
                                          int wave, int lane) {
    using T = Tile<HD>;
    const int rows = min(left, 64);
    const auto rs = rsrc_of(from, rows <= 0 ? 0u : unsigned((rows - 1) * stride + HD) * 2u);
#pragma unroll
    for (int i = 0; i < T::kLoads / WAVES; ++i) {
        const int u = wave + WAVES * i;
        const int row = u * T::kLoadRows + lane / T::kChunks;
        const unsigned voff =
            unsigned(row * stride + (((lane % T::kChunks) ^ T::key(row)) * 8)) * 2u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, (__attribute__((address_space(3))) void*)(lds_half*)(tile + u * 512), 16, voff, 0, 0,
            0);
    }
}

// Per-lane byte offsets of the fragment reads, kept in registers (an empty asm
// makes them opaque, so they are not recomputed per read). Rows 16 and 32 apart
// have one key, so they are immediate offsets from these.
template <int HD>
struct Frags {
    unsigned rows[HD / 16];
    unsigned tr[HD / 32][2];

    __device__ __forceinline__ explicit Frags(int lane) {
        using T = Tile<HD>;
        const int fr = lane & 31, h = lane >> 5, j = lane & 15;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
            rows[kk] = unsigned((fr * HD + (((2 * kk + h) ^ T::key(fr)) * 8)) * 2);
            asm volatile("" : "+v"(rows[kk]));
        }
#pragma unroll
        for (int db = 0; db < HD / 32; ++db)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int row = 4 * h + (j >> 2) + 8 * t;
                const int col = 32 * db + 16 * ((lane >> 4) & 1) + 4 * (j & 3);
                tr[db][t] = unsigned((row * HD + (((col >> 3) ^ T::key(row)) * 8) + (col & 7)) * 2);
                asm volatile("" : "+v"(tr[db][t]));
            }
    }

    // An MFMA operand with tile rows as its rows and d as k: lane l gets row
    // 32 hb + l % 32, halves 16 kk + 8 (l / 32) .. + 8.
    __device__ __forceinline__ f16x8 row(const _Float16* tile, int hb, int kk) const {
        return *reinterpret_cast<const f16x8*>(reinterpret_cast<const char*>(tile) + rows[kk] +
                                               64 * HD * hb);
    }

    // An MFMA operand with d as its rows and tile rows as k, in the order the
    // probabilities' registers hold them: lane l (d = 32 db + l % 32, h = l /
    // 32) gets tile rows 16 cs + 4h .. + 3 (k 0..3) and 16 cs + 8 + 4h .. + 3
    // (k 4..7) of column d. wait_lds before the first use.
    template <int CS>
    __device__ __forceinline__ TrFrag transposed(const _Float16* tile, int db) const {
        const unsigned base = unsigned(reinterpret_cast<uintptr_t>((lds_half*)tile));
        TrFrag f;
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2"
                     : "=v"(f.lo) : "v"(base + tr[db][0]), "i"(32 * HD * CS));
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2"
                     : "=v"(f.hi) : "v"(base + tr[db][1]), "i"(32 * HD * CS));
        return f;
    }
    // For a slice known once the loops are unrolled.
    __device__ __forceinline__ TrFrag transposed(const _Float16* tile, int cs, int db) const {
        switch (cs) {
        case 0: return transposed<0>(tile, db);
        case 1: return transposed<1>(tile, db);
        case 2: return transposed<2>(tile, db);
        default: return transposed<3>(tile, db);
        }
    }
};

__device__ __forceinline__ f32x16 mfma(const f16x8& a, const f16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// The row (0..31) of an MFMA result that register r of a lane in half h holds.
__device__ __forceinline__ constexpr int result_row(int r, int h) {
    return 8 * (r >> 2) + 4 * h + (r & 3);
}

// A running maximum below every score: exp2(-inf - kFloor) is 0, and the first
// key that a query sees moves it.
constexpr float kFloor = -3e38f;
// What a lane's probabilities of a tile may add up to before the running
// maximum is moved: none of them is above it then, and FP16 holds 2^16.
constexpr float kSumLimit = 32768.0f;
// How far below a tile's maximum the reference lies, in log2 units: the largest
// probability is 2^5, so that those down to 2^-30 of it stay above 0 in FP16. (At
// 1 the keys under 2^-25 of a row's largest are in the sum l and 0 in the product
// with V: 0.3% of o where 130,000 are at 2^-25.5; at 2^5 so many lose 2^-13, a
// quarter of o's own rounding.) A lane's 32 add up to 2^10 at most. What it costs is
// moves where scores spread wide: 16,384 tokens, scores of deviation 1, 2, 4 and 8
// take 355, 355, 372 and 396 us; at 1 352, 355, 356 and 367, at 2^8 353, 361, 389
// and 418.
constexpr float kBelow = 5.0f, kBelowFactor = 0x1p-5f;

// P = 2^(ce s - m) as FP16, and the FP32 sum of this lane's (its half of the
// keys).
template <int HB>
__device__ __forceinline__ float exponentials(f16x8 (&p)[2 * HB], const f32x16 (&s)[HB], float ce,
                                              float m) {
    float sum = 0.0f;
#pragma unroll
    for (int hb = 0; hb < HB; ++hb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[hb][r], ce, -m));
            p[2 * hb + (r >> 3)][r & 7] = _Float16(e);
            sum += e;
        }
    return sum;
}

// A tile's probabilities and their sum. m, a query's reference in log2 units,
// need not be its maximum: O and l share it, and it only has to keep P inside
// FP16. So past the wave's first tile (started) the tile's maximum is not taken
// unless the sum passes kSumLimit, or overflows, for some query; then m moves to
// kBelow under the maximum, rescale(2^(m_old - m_new)) is called and the tile is
// taken again (scores() gives s and ce once more, so that no register holds s
// meanwhile).
// (scores uses an offset of 0 that the compiler cannot see through: otherwise it
// moves the products and the masks out of the loop and keeps them after all.)
template <int HB, class Scores, class Rescale>
__device__ __forceinline__ float probabilities(f16x8 (&p)[2 * HB], const Scores& scores, float* m,
                                               bool* started, const Rescale& rescale) {
    for (;;) {
        f32x16 s[HB];
        unsigned zero = 0;
        asm volatile("" : "+s"(zero));
        const float ce = scores(s, zero);
        const bool move = !*started;
        if (move) {
            *started = true;
            float mx = s[0][0];
#pragma unroll
            for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[hb][r]);
            mx *= ce;
            const float m_new = fmaxf(*m, fmaxf(mx, xor32(mx)) - kBelow);
            rescale(__builtin_amdgcn_exp2f(*m - m_new));
            *m = m_new;
        }
        const float sum = exponentials<HB>(p, s, ce, *m);
        if (move || !__any(sum > kSumLimit)) return sum;
        *started = false;
    }
}

// Four waves' results, transposed (a lane holds one row of its wave's 32), as
// FP16 rows in LDS: write_rows by the waves that hold them, a barrier, then
// copy_rows by all threads, 16 bytes each and whole rows side by side. Stored
// straight from the registers, 8 bytes of 32 rows at a time, they make a packed
// forward pass over 8 x 1,024 tokens of 8 heads of 128 take 37.5 us instead of
// 34.9. In LDS a row begins 16 bytes of banks after the one before.
template <int HD>
constexpr int kRowHalves = HD + 8;

template <int HD>
__device__ __forceinline__ void write_rows(_Float16* block, const f32x16* acc, float by, int row,
                                           int h) {
    _Float16* at = block + row * kRowHalves<HD>;
#pragma unroll
    for (int db = 0; db < HD / 32; ++db)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const f16x4 v = {_Float16(acc[db][4 * a] * by), _Float16(acc[db][4 * a + 1] * by),
                             _Float16(acc[db][4 * a + 2] * by), _Float16(acc[db][4 * a + 3] * by)};
            *reinterpret_cast<f16x4*>(at + 32 * db + 8 * a + 4 * h) = v;
        }
}

// to(row) is where row `row` (below `rows`) goes.
template <int HD, int THREADS, class To>
__device__ __forceinline__ void copy_rows(const _Float16* block, int rows, const To& to) {
#pragma unroll
    for (int i = threadIdx.x; i < 128 * (HD / 8); i += THREADS) {
        const int row = i / (HD / 8), d = i % (HD / 8) * 8;
        if (row < rows)
            *reinterpret_cast<f16x8*>(to(row) + d) =
                *reinterpret_cast<const f16x8*>(block + row * kRowHalves<HD> + d);
    }
}

}  // namespace
}  // namespace flint
