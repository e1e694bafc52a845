// Matrix-unit pieces of the attention kernels (td_attn_forward.hip, td_attn_backward.hip): 32 x 32 products of float32,
// float16 and bfloat16 operands, and the tiles of keys or rows that they read from LDS.
//
// Every product is 32 x 32 with a float32 accumulator: element e of lane l is row 8 (e / 4) + 4 (l / 32) + e % 4 of
// column l % 32. An operand is a fragment of 16 bytes a lane, l % 32 its row (or column) and l / 32 the half of a chunk
// of 32 bytes of the inner dimension: 16 elements in 16 bits, 8 in float32. The order of the inner dimension is free as
// long as both operands share it, which is what lets an accumulator be the next product's operand without leaving its
// registers: a score tile's elements 8 s .. 8 s + 7 are the 16 rows 16 s .. 16 s + 15 of its column, in the order
// (half, element) -> 16 s + 8 (element / 4) + 4 half + element % 4, and the other operand is read from LDS in that order.
#pragma once

#include <type_traits>

#include "td_attn.h"

namespace td {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mma;
template <>
struct Mma<f16> {
    __device__ __forceinline__ static f32x16 mul(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
};
template <>
struct Mma<bf16> {
    __device__ __forceinline__ static f32x16 mul(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};
template <>
struct Mma<float> {
    __device__ __forceinline__ static f32x16 mul(u32x4 a, u32x4 b, f32x16 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }
};

// Rows of DP elements in LDS, 16 bytes longer than their data: with that pitch the 32 rows of a fragment read, the
// transpose reads and the float32 column reads all go at the LDS's full rate (235 B/ns a CU, 118 and 109; without it
// 131, 71 or 37 for rows of 64, 128 or 256 bytes, by a probe of the reads alone).
template <typename T, int DP>
struct TileRows {
    static constexpr int kS = static_cast<int>(sizeof(T));
    static constexpr int kPitch = DP * kS + 16;      // bytes
    static constexpr int kChunks = DP * kS / 32;     // fragments of a row
    static constexpr int kPieces = DP * kS / 16;     // 16-byte pieces of a row

    // fragment `chunk` of rows row0 .. row0 + 31
    __device__ __forceinline__ static u32x4 rows(const unsigned char* tile, int row0, int chunk, int lane) {
        return *reinterpret_cast<const u32x4*>(tile + (row0 + (lane & 31)) * kPitch + chunk * 32 + (lane >> 5) * 16);
    }

    // acc += (columns d0 .. d0 + 31 of rows row0 .. row0 + 31)^T . w, with w a 32 x 32 tile over those rows in the
    // accumulator's layout (16-bit: its elements rounded to T by pack()).
    using Packed = std::conditional_t<sizeof(T) == 2, u32x4, f32x16>;
    static constexpr int kPacked = sizeof(T) == 2 ? 2 : 1;
    __device__ __forceinline__ static void pack(const f32x16& w, Packed (&o)[kPacked]) {
        if constexpr (kS == 4) {
            o[0] = w;
        } else {
            typedef T T8 __attribute__((ext_vector_type(8)));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                T8 v;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = static_cast<T>(w[8 * s + j]);
                o[s] = __builtin_bit_cast(u32x4, v);
            }
        }
    }
    __device__ __forceinline__ static f32x16 columns(const unsigned char* tile, int row0, int d0, int lane,
                                                     const Packed (&w)[kPacked], f32x16 acc) {
        if constexpr (kS == 4) {
            const unsigned char* at = tile + (row0 + 4 * (lane >> 5)) * kPitch + (d0 + (lane & 31)) * 4;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                acc = __builtin_amdgcn_mfma_f32_32x32x2f32(
                    *reinterpret_cast<const float*>(at + (8 * (e >> 2) + (e & 3)) * kPitch), w[0][e], acc, 0, 0, 0);
        } else {
            // transpose reads: of 16 lanes, lane i points at row i / 4, columns 4 (i % 4) .. of a 4 x 16 block and
            // receives its column i, the four rows
            using v4s = short __attribute__((ext_vector_type(4)));
            using lds_v4s = __attribute__((address_space(3))) v4s;
            const int i = lane & 15;
            const unsigned char* at = tile + (row0 + 4 * (lane >> 5) + (i >> 2)) * kPitch +
                                      (d0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3)) * 2;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 16 * s * kPitch));
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + (16 * s + 8) * kPitch));
                acc = Mma<T>::mul(__builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)),
                                  w[s], acc);
            }
        }
        return acc;
    }
};

// 16 bytes of row `row` at byte `at` (a multiple of 16): zeros past the head's D elements. VEC: D * sizeof(T), the base
// and every stride are multiples of 16 bytes, else element by element.
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 row_piece(const T* row, int at, int D) {
    constexpr int E = 16 / static_cast<int>(sizeof(T));
    const int d = at / static_cast<int>(sizeof(T));
    u32x4 r = {0u, 0u, 0u, 0u};
    if constexpr (VEC) {
        if (d < D) r = *reinterpret_cast<const u32x4*>(row + d);
    } else {
        typedef T TE __attribute__((ext_vector_type(E)));
        TE v = __builtin_bit_cast(TE, r);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (d + e < D) v[e] = row[d + e];
        r = __builtin_bit_cast(u32x4, v);
    }
    return r;
}

// NR rows of a tensor on their way to LDS through the registers of NT threads: rows whose bit in `gone` is set are
// zeros and are not read. VEC as in row_piece, and NR rows span less than 2^31 bytes.
template <typename T, int DP, int NR, int NT, bool VEC>
struct StagedRows {
    using R = TileRows<T, DP>;
    static constexpr int kN = NR * R::kPieces / NT;  // pieces a thread
    static_assert(NR <= 64 && NR * R::kPieces % NT == 0, "whole pieces for every thread");
    u32x4 r[kN];
    unsigned off[VEC ? kN : 1];  // bytes from the tile's first row

    __device__ __forceinline__ static int row_of(int u, int t) { return (t + u * NT) / R::kPieces; }
    __device__ __forceinline__ static int at_of(int u, int t) { return (t + u * NT) % R::kPieces * 16; }

    // f(i): elements from the tile's first row to its row i
    template <typename F>
    __device__ __forceinline__ void plan(F f, int D, int t) {
        if constexpr (VEC) {
#pragma unroll
            for (int u = 0; u < kN; ++u) {
                const int at = at_of(u, t);
                off[u] = static_cast<unsigned>(f(row_of(u, t)) * R::kS) + (at < D * R::kS ? at : 0);
            }
        }
    }
    // base: the tile's first row; f as in plan
    template <typename F>
    __device__ __forceinline__ void load(const T* base, F f, uint64_t gone, int D, int t) {
        if constexpr (VEC) {
            const unsigned char* const bytes = reinterpret_cast<const unsigned char*>(base);
            if (gone == 0) {
#pragma unroll
                for (int u = 0; u < kN; ++u) r[u] = *reinterpret_cast<const u32x4*>(bytes + off[u]);
            } else {
#pragma unroll
                for (int u = 0; u < kN; ++u) {
                    r[u] = u32x4{0u, 0u, 0u, 0u};
                    if (!((gone >> row_of(u, t)) & 1)) r[u] = *reinterpret_cast<const u32x4*>(bytes + off[u]);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < kN; ++u) {
                const int row = row_of(u, t);
                r[u] = u32x4{0u, 0u, 0u, 0u};
                if (!((gone >> row) & 1)) r[u] = row_piece<T, false>(base + f(row), at_of(u, t), D);
                __builtin_amdgcn_sched_barrier(0);  // one piece's loads at a time: all of them do not fit in registers
            }
        }
    }
    // The pieces past the row's end are cleared here and not in load(), where that would wait for the loads.
    __device__ __forceinline__ void store(unsigned char* tile, int D, int t) {
        if (VEC && D < DP) {
#pragma unroll
            for (int u = 0; u < kN; ++u)
                if (at_of(u, t) >= D * R::kS) r[u] = u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int u = 0; u < kN; ++u) *reinterpret_cast<u32x4*>(tile + row_of(u, t) * R::kPitch + at_of(u, t)) = r[u];
    }
};

// Workgroups. Shared: eight wavefronts of 32 rows (or keys) each share the tiles of the other side, the first four staging
// one of the two operands and the others the second. Staging and its barriers take a fifth of the time of four such
// wavefronts (they were left out to see: 8192 tokens x 8 heads of 32 273 -> 232 us, 4096 x 16 of 128 334 -> 272), and
// eight do it half as often for a row; rows of more than 256 bytes leave registers for four only. Private: four
// wavefronts have the same 32 rows (or keys) and every fourth tile each, staged by itself alone, for problems of few rows
// (keys).
constexpr int shared_waves(int row_bytes) { return row_bytes > 256 ? 4 : 8; }
template <typename T, int DP, bool PRIVATE>
constexpr int kWaves = PRIVATE ? 4 : shared_waves(DP * static_cast<int>(sizeof(T)));
template <typename T, int DP, bool PRIVATE>
constexpr int kTileRows = PRIVATE ? 32 : 32 * kWaves<T, DP, PRIVATE>;
inline int tile_rows(bool is_private, int row_bytes) { return is_private ? 32 : 32 * shared_waves(row_bytes); }

template <typename T, int DP, int NR, bool PRIVATE, bool VEC>
struct TwoTiles {
    static constexpr bool kBoth = kWaves<T, DP, PRIVATE> == 4;  // a thread stages both operands
    static constexpr int kThreads = PRIVATE ? 64 : 256;
    StagedRows<T, DP, NR, kThreads, VEC> a, b;  // not both: a alone, of the operand that the wavefront stages
    int t;
    bool second;
    __device__ __forceinline__ TwoTiles() : t(static_cast<int>(threadIdx.x) & (kThreads - 1)) {
        second = __builtin_amdgcn_readfirstlane(!kBoth && threadIdx.x >= 256);
    }
    template <typename F, typename G>
    __device__ __forceinline__ void plan(F f, G g, int D) {
        if constexpr (kBoth) {
            a.plan(f, D, t);
            b.plan(g, D, t);
        } else {
            a.plan([&](int x) { return second ? g(x) : f(x); }, D, t);
        }
    }
    template <typename F, typename G>
    __device__ __forceinline__ void load(const T* base_a, F f, const T* base_b, G g, uint64_t gone, int D) {
        if constexpr (kBoth) {
            a.load(base_a, f, gone, D, t);
            b.load(base_b, g, gone, D, t);
        } else {
            a.load(second ? base_b : base_a, [&](int x) { return second ? g(x) : f(x); }, gone, D, t);
        }
    }
    __device__ __forceinline__ void store(unsigned char* tile_a, unsigned char* tile_b, int D) {
        if constexpr (kBoth) {
            a.store(tile_a, D, t);
            b.store(tile_b, D, t);
        } else {
            a.store(second ? tile_b : tile_a, D, t);
        }
    }
};

// Orders a wavefront's LDS accesses before it against those after it. The LDS serves one wavefront's accesses in order,
// so this keeps the compiler from moving them and costs nothing.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Value of `v` in the lane 32 away
__device__ __forceinline__ float other_half(float v) { return xor_lane(v, 32); }

// The workgroup's place in the XCD-contiguous order: workgroup w runs on XCD w % 8, so that the `n` pieces of work in
// order are dealt in eight contiguous runs and neighbours (tiles of one head, which read the same keys) share an L2.
// Negative: no work.
__device__ __forceinline__ int xcd_order(int w, int n) {
    const int per = (n + kXcds - 1) / kXcds;
    const int i = (w % kXcds) * per + w / kXcds;
    return w / kXcds < per && i < n ? i : -1;
}
inline unsigned xcd_grid(int64_t n) { return static_cast<unsigned>((n + kXcds - 1) / kXcds * kXcds); }

// Work that is split: tiles (of rows or keys, numbered over the batch and key heads) before `whole` have a workgroup each,
// those from it on n, which write float32 parts [tile - whole][part][rows of a tile][D] that are joined afterwards.
struct TileSplit {
    int n, whole, total;
};
struct TileWork {
    int tile, part, parts;  // tile < 0: no work
};
__device__ __forceinline__ TileWork tile_work(const TileSplit& s) {
    const int block = static_cast<int>(blockIdx.x), first = (s.whole + kXcds - 1) / kXcds * kXcds;
    if (block < first) return TileWork{xcd_order(block, s.whole), 0, 1};
    const int i = xcd_order(block - first, (s.total - s.whole) * s.n);
    return i < 0 ? TileWork{-1, 0, 1} : TileWork{s.whole + i / s.n, i % s.n, s.n};
}
inline unsigned tile_grid(const TileSplit& s) {
    return xcd_grid(s.whole) + (s.n > 1 ? xcd_grid(static_cast<int64_t>(s.total - s.whole) * s.n) : 0);
}
// Every CU works at its own rate whether it holds four workgroups or one, so 4 1/8 tiles a CU take as long as 5. Where a
// few tiles are left over after an even share for every CU, those are split over all CUs (8400 tokens of 16 heads as 528
// tiles of 256 rows: forward 379 us with the 16 left over whole, 295 split; dQ 441 and 347; dK and dV 569 and 427).
inline TileSplit even_split(int total, int steps) {
    const int cus = cu_count(), rest = total % cus;
    TileSplit s{1, total, total};
    if (total < cus || total > 8 * cus || rest == 0 || rest > cus / 2) return s;
    int n = cus / rest;
    n = n < 8 ? n : 8;
    n = n < steps / 4 ? n : steps / 4;
    if (n < 2) return s;
    s.n = n;
    s.whole = total - rest;
    return s;
}

// Parts for shared tiles that leave CUs without work: the number that takes least, with `slots` workgroups at a time, a
// part's share of the loop and what it costs beside it (about four steps of 64 in 16 bits, one in float32, whose steps are
// longer), once more for the join. Measured (dQ): 8 heads x 1500 of 128, float16, 48 tiles on 256 slots: 58 us in 2 parts, 44
// in 5, 62 in 11; 5 x 8 x 1000 of 36, float32, 160 tiles: 203 whole, 156 in 3, 174 in 4; 96 heads x 400 of 32, float16, 192
// tiles on 512 slots: 20 whole, 29 in 3.
inline int parts_of(int total, int slots, int64_t loop, bool float32) {
    const double steps = loop / 64.0, fixed = float32 ? 1 : 4;
    const int64_t most = loop < 131072 ? (loop + 127) / 128 : 1024;
    int best = 1;
    double least = (total + slots - 1) / slots * (steps + fixed);
    for (int64_t rounds = 1; rounds <= 4; ++rounds) {
        int64_t n = slots * rounds / total;
        n = n < most ? n : most;
        if (n < 2) continue;
        const double cost = (total * n + slots - 1) / slots * (steps / n + fixed) + fixed;
        if (cost < least) {
            least = cost;
            best = static_cast<int>(n);
        }
    }
    return best;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kLowest = -3.4028234663852886e38f;

// An additive mask's entry in base 2. The lowest float32 (and a mask below 2^127.5) keeps finite, so that a row of it
// alone stays a uniform row, as in exact arithmetic with rounding to 24 bits; -inf stays -inf.
__device__ __forceinline__ float mask_log2(float m) {
    return m == kNegInf ? kNegInf : __builtin_fmaxf(m * kLog2e, kLowest);
}

// Scores past 2^16 (base 2) have steps of 2^-8 or more: fma(score, c, -m), which does not round the product, no longer
// cancels against a maximum m that was a rounded product, and what is added to m (log2 l, a factor's exponent) loses its
// bits. Rows of such a maximum take the products rounded and add the rest to the difference.
__device__ __forceinline__ bool big_score(float m) {
    return __builtin_fabsf(m) > 65536.f && __builtin_fabsf(m) < __builtin_inff();
}
__device__ __forceinline__ float rounded_product(float s, float c) {
#pragma clang fp contract(off)
    return s * c;
}

// Keys j0 .. j0 + 31 beyond `last`, the last key that a query sees, as bits
__device__ __forceinline__ uint32_t beyond(int j0, int last) {
    return last < j0 ? ~0u : last - j0 >= 31 ? 0u : ~0u << (last - j0 + 1);
}

// What the mask has for one row and 32 keys
struct MaskWord {
    uint32_t bits;
    int kind;
};
__device__ __forceinline__ MaskWord mask_word(const AttnParams& p, int b, int h, int i, int word) {
    if (word >= p.words) return MaskWord{~0u, kMaskAll};
    const int64_t row = b * p.bs[0] + h * p.bs[1] + i * p.bs[2];
    const int64_t tile = b * p.kinds_bs[0] + h * p.kinds_bs[1] + (p.bs[2] == 0 ? 0 : i >> 5);
    return MaskWord{p.bits[row * p.words + word], p.kinds[tile * p.words + word]};
}

// Elements x .. x + 3 of an accumulator, times `by`, to channels at .. at + 3 of a row of D. vec: whole groups of 4
template <typename T>
__device__ __forceinline__ void store4(T* row, int at, int D, bool vec, const f32x16& a, int x, float by) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(a[x + e] * by);
    if (vec) {
        if (at < D) *reinterpret_cast<T4*>(row + at) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (at + e < D) row[at + e] = v[e];
    }
}

// Scores of 32 keys (rows 8 i + 4 half + e) by 32 rows of the problem (columns), as the scores in base 2 with -inf where
// a pair is left out: s * c, plus the mask's values. `gone`: the lane's bits for its column's 32 keys. values: the mask's
// row at the first key of the tile, `left` keys inside it, or null.
template <typename T>
__device__ __forceinline__ void mask_scores(f32x16& s, float c, uint32_t gone, const T* values, int left, int half) {
    gone >>= 4 * half;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float add[4] = {0.f, 0.f, 0.f, 0.f};
        if (values != nullptr) {
            const int key = 8 * i + 4 * half;
            if (key + 4 <= left) {
                T four[4];  // no alignment is known, the hardware needs none
                __builtin_memcpy(four, values + key, sizeof(four));
#pragma unroll
                for (int e = 0; e < 4; ++e) add[e] = mask_log2(static_cast<float>(four[e]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key + e < left) add[e] = mask_log2(static_cast<float>(values[key + e]));
            }
            __builtin_amdgcn_sched_barrier(0);  // four loads at a time: registers
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float t = fmaf(s[4 * i + e], c, add[e]);
            s[4 * i + e] = (gone >> (8 * i + e)) & 1u ? kNegInf : t;
        }
    }
}

}  // namespace td
