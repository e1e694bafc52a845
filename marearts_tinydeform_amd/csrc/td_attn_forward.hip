// Attention among tokens, forward, on the matrix units (float32, float16, bfloat16).
//
// One pass over the keys with the running maximum m and sum l of the softmax (Milakov and Gimelshein, "Online normalizer
// calculation for softmax", 2018): S^T = K Q^T, P^T = 2^(S^T - m), O^T += V^T P^T, all three transposed, so that a
// lane's scores are of one row (its column), the row's statistics are one number a lane, and P^T is the second product's
// operand as it stands in the accumulator. P is rounded to the inputs' type for that product (half a step of each, not
// summed up: l adds the unrounded ones); everything else stays in float32.
//
// Bound by the vector units where heads are narrow: a score costs an exponential and five operations beside D / 32 of an
// MFMA's work (8400 tokens x 8 heads of 32, float16, batch 2: 243 to 264 us, 230 of them vector operations, MFMA busy 24%);
// by LDS reads and MFMAs together where they are wide (4096 tokens x 16 heads, bfloat16, batch 2: 64 wide 165 us, 830
// TFLOP/s, 128 wide 311 us, 883); by memory for single tokens (4 x 21760 keys, 4 key heads of 64: 18 us, 5 TB/s, and 6.7
// for the join).
#include "td_attn_mma.h"

// The build compiles this file once per type: TD_ATTN_TYPE 0 float32 (and the entry), 1 float16, 2 bfloat16.
#ifndef TD_ATTN_TYPE
#error "TD_ATTN_TYPE"
#endif

namespace td {
namespace {

// Rescaling O and l is put off until a row's maximum has grown by more than this (base 2): the sums then hold factors of
// up to 2^kSlack, and only tiles that move a maximum pay for the rescale.
constexpr float kSlack = 4.f;
// float16 holds P as 2^11 P (at most 2^(11 + kSlack) < 65504): small probabilities keep their bits down to 2^-25 and
// steps of 2^-35. The factor is in l as well and cancels.
template <typename T>
constexpr float kShift = std::is_same<T, f16>::value ? 11.f : 0.f;
// log2 of the factor that l holds: 11 as far as m has bits for it
template <typename T>
__device__ __forceinline__ float shift_of(float m) {
    return kShift<T> == 0.f ? 0.f : m - (m - kShift<T>);
}

struct Split {
    TileSplit t;
    int keys;   // keys of a part, a multiple of 128
    float* o;   // parts' unnormalised outputs [..][rows of a tile][D]
    float* ml;  // and maximum and sum [..][rows of a tile][2]
};

// Keys of a tile: 64 where the staged rows leave room for two workgroups on a CU
template <typename T, int DP, bool WK>
constexpr int key_tile() {
    return WK || DP * static_cast<int>(sizeof(T)) > 256 ? 32 : 64;
}

// Wavefronts a SIMD that the registers have to leave room for. A workgroup of eight takes two of each SIMD.
template <typename T, int DP, bool WK, bool SLOW>
constexpr int min_waves() {
    constexpr int bytes = DP * static_cast<int>(sizeof(T));
    if (WK) return bytes <= 64 ? 3 : bytes <= 128 ? 2 : SLOW ? 1 : 2;
    return bytes <= 64 || (bytes <= 128 && !SLOW) ? 4 : bytes <= 256 ? 2 : 1;
}

// WK: private key tiles (TwoTiles); the four wavefronts' partial results are joined in LDS.
// MASK: there is a mask tensor. VEC: operands are read 16 bytes at a time (StagedRows).
template <typename T, int DP, bool WK, bool MASK, bool VEC>
__global__ __launch_bounds__((kWaves<T, DP, WK> * kWave), (min_waves<T, DP, WK, MASK>())) void attn_forward_kernel(
    AttnParams p, Split sp, bool vec_out, int tiles) {
    using R = TileRows<T, DP>;
    constexpr int KT = key_tile<T, DP, WK>(), ND = DP / 32, BM = kTileRows<T, DP, WK>;
    constexpr int kTile = KT * R::kPitch;
    extern __shared__ __align__(16) unsigned char lds[];
    const TileWork work = tile_work(sp.t);
    if (work.tile < 0) return;
    const int tile = tiles - 1 - work.tile % tiles, bh = work.tile / tiles;  // causal: the long ones first
    const int b = bh / p.Hk, hk = bh % p.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int lane = threadIdx.x % kWave, half = lane >> 5;
    unsigned char* const kt_lds = lds + (WK ? wave * 2 * kTile : 0);
    unsigned char* const vt_lds = kt_lds + kTile;

    // the lane's row
    const int row0 = tile * BM, wrow0 = row0 + (WK ? 0 : wave * 32), r = wrow0 + (lane & 31);
    const bool live = r < p.rows;
    const int i = static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(live ? r : 0)));
    const int h = hk * p.G + (live ? r : 0) - i * p.G;
    u32x4 qf[R::kChunks];
    {
        const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
#pragma unroll
        for (int c = 0; c < R::kChunks; ++c)
            qf[c] = live ? row_piece<T, VEC>(q, c * 32 + half * 16, p.D) : u32x4{0u, 0u, 0u, 0u};
    }
    const T* const mrow = MASK ? static_cast<const T*>(p.mask) + b * p.ms[0] + h * p.ms[1] + i * p.ms[2] : nullptr;
    const int diag = static_cast<int>(p.diag);
    const int last = p.causal ? i + diag : 2147483647;

    // the workgroup's keys, and the wavefront's first and last row's
    int kend = p.K, k0 = 0;
    const int top_row = (row0 + BM < p.rows ? row0 + BM : p.rows) - 1;
    if (p.causal) {
        const int seen = static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(top_row))) + diag + 1;
        kend = seen < kend ? seen : kend;
    }
    if (work.parts > 1) {
        k0 = work.part * sp.keys;
        kend = k0 + static_cast<int64_t>(sp.keys) < kend ? k0 + sp.keys : kend;
    }
    const int wtop = wrow0 + 31 < p.rows ? wrow0 + 31 : p.rows - 1;
    const int wfirst = wrow0 < p.rows ? wrow0 : p.rows - 1;
    const int seen_all = p.causal ? static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(wfirst))) + diag : 2147483647;
    const int seen_any = p.causal ? static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(wtop))) + diag : 2147483647;

    const T* const kb = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* const vb = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
    const uint8_t* const pad = p.pad == nullptr ? nullptr : p.pad + static_cast<int64_t>(b) * p.K;
    // keys j0 + lane of a tile: whether nobody sees them
    auto pad_byte = [&](int64_t j0) {  // not looked at before the next tile: that would wait for the loads issued before it
        const int64_t j = j0 + lane;
        int v = 1;
        if (lane < KT && j < kend) v = pad != nullptr ? pad[j] : 0;
        return v;
    };

    TwoTiles<T, DP, KT, WK, VEC> staged;
    auto k_row = [&](int x) { return x * p.ks[1]; };
    auto v_row = [&](int x) { return x * p.vs[1]; };
    staged.plan(k_row, v_row, p.D);
    float m = kNegInf, l = 0.f;
    bool big = false;  // a row's maximum is
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x16{0.f};

    constexpr int step = WK ? 4 * KT : KT;
    constexpr uint64_t all = KT == 64 ? ~uint64_t{0} : (uint64_t{1} << (KT & 63)) - 1;
    int64_t j0 = k0 + (WK ? wave * KT : 0);
    uint64_t gone = __ballot(pad_byte(j0) != 0), gone_next;
    MaskWord mw[KT / 32] = {};
    auto fetch = [&](int64_t at, uint64_t g) {
        if constexpr (MASK)
#pragma unroll
            for (int x = 0; x < KT / 32; ++x) mw[x] = mask_word(p, b, h, i, static_cast<int>(at / 32) + x);
        staged.load(kb + at * p.ks[1], k_row, vb + at * p.vs[1], v_row, g & all, p.D);
    };
    if (j0 < kend) fetch(j0, gone);
    int next_pad = pad_byte(j0 + step);
    for (; j0 < kend; j0 += step) {
        if (!WK) __syncthreads();
        staged.store(kt_lds, vt_lds, p.D);
        if (WK)
            wave_sync();
        else
            __syncthreads();
        gone_next = __ballot(next_pad != 0);
        // what the tile's scores have to be masked by
        bool masked = (gone & all) != 0 || static_cast<int>(j0) + KT - 1 > seen_all, values = false, none = MASK;
        uint32_t bits[KT / 32];
#pragma unroll
        for (int x = 0; x < KT / 32; ++x) {
            bits[x] = mw[x].bits;
            if constexpr (MASK) {
                masked |= __any(mw[x].kind != kMaskNone);
                values |= __any(mw[x].kind == kMaskValues);
                none &= __all(mw[x].kind == kMaskAll);
            }
        }
        if (j0 + step < kend) {
            fetch(j0 + step, gone_next);
            next_pad = pad_byte(j0 + 2 * step);
        }
        const int j = static_cast<int>(j0);
        if ((gone & all) != all && j <= seen_any && !none) {
            f32x16 s[KT / 32];
#pragma unroll
            for (int x = 0; x < KT / 32; ++x) {
                s[x] = f32x16{0.f};
#pragma unroll
                for (int c = 0; c < R::kChunks; ++c)
                    s[x] = Mma<T>::mul(R::rows(kt_lds, 32 * x, c, lane), qf[c], s[x]);
            }
            float cc = p.c;
            if (masked) {
                cc = 1.f;
#pragma unroll
                for (int x = 0; x < KT / 32; ++x)
                    mask_scores<T>(s[x], p.c,
                                   bits[x] | static_cast<uint32_t>(gone >> (32 * x)) | beyond(j + 32 * x, last),
                                   values ? mrow + j + 32 * x : nullptr, p.K - j - 32 * x, half);
            }
            float mt = kNegInf;
#pragma unroll
            for (int x = 0; x < KT / 32; ++x)
#pragma unroll
                for (int e = 0; e < 16; ++e) mt = __builtin_fmaxf(mt, s[x][e]);
            mt = __builtin_fmaxf(mt, other_half(mt)) * cc;
            if (__any(mt > m + kSlack)) {
                const float to = __builtin_fmaxf(m, mt);
                const float shrink = to == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - to);
                m = to;
                big = __any(big_score(m));
                l *= shrink;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] *= shrink;
            }
            if (big) {
#pragma unroll
                for (int x = 0; x < KT / 32; ++x)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[x][e] = rounded_product(s[x][e], cc);
                cc = 1.f;
            }
            const float from = m == kNegInf ? 0.f : m - kShift<T>;
#pragma unroll
            for (int x = 0; x < KT / 32; ++x) {
                f32x16 pr;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    pr[e] = __builtin_amdgcn_exp2f(fmaf(s[x][e], cc, -from));
                    l += pr[e];
                }
                typename R::Packed w[R::kPacked];
                R::pack(pr, w);
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d] = R::columns(vt_lds, 32 * x, 32 * d, lane, w, o[d]);
            }
        }
        gone = gone_next;
        if (WK) wave_sync();
    }
    l += other_half(l);

    if constexpr (WK) {
        // join the four wavefronts' parts: maxima and sums first, then each scaled O, through LDS
        __syncthreads();
        float* const ml = reinterpret_cast<float*>(lds);  // [4][32][2]
        if (half == 0) {
            ml[(wave * 32 + lane) * 2] = m;
            ml[(wave * 32 + lane) * 2 + 1] = l;
        }
        __syncthreads();
        float to = kNegInf, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) to = __builtin_fmaxf(to, ml[(w * 32 + (lane & 31)) * 2]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = ml[(w * 32 + (lane & 31)) * 2], lw = ml[(w * 32 + (lane & 31)) * 2 + 1];
            sum += mw == kNegInf ? lw : lw * __builtin_amdgcn_exp2f(mw - to);
        }
        const float scale = m == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l = sum;
        // [4 waves][32 rows][DP] in two halves of the wavefronts: 2, 3 write and 0, 1 add, then 1 writes and 0 adds
        float* const part = ml + 256;
        const int at = (lane & 31) * (DP + 4) + 4 * half;
        constexpr int kPart = 32 * (DP + 4);
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= scale;
#pragma unroll
        for (int n = 2; n > 0; n >>= 1) {
            if (wave >= n && wave < 2 * n) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        *reinterpret_cast<f32x4*>(part + (wave - n) * kPart + at + 32 * d + 8 * x) =
                            f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
            }
            __syncthreads();
            if (wave < n) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(part + wave * kPart + at + 32 * d + 8 * x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[d][4 * x + e] += v[e];
                    }
            }
            __syncthreads();
        }
        if (wave != 0) return;
    }
    if (!live) return;

    const int64_t row = (static_cast<int64_t>(b) * p.H + h) * p.Q + i;
    if (work.parts > 1) {
        const int64_t part = (static_cast<int64_t>(work.tile - sp.t.whole) * work.parts + work.part) * BM + r - row0;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                store4<float>(sp.o + part * p.D, 32 * d + 8 * x + 4 * half, p.D, p.D % 4 == 0, o[d], 4 * x, 1.f);
        if (half == 0) {
            sp.ml[2 * part] = m;
            sp.ml[2 * part + 1] = l;
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t out_at = ((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        o[d] *= inv;
#pragma unroll
        for (int x = 0; x < 4; ++x)
            store4<T>(static_cast<T*>(p.out) + out_at, 32 * d + 8 * x + 4 * half, p.D, vec_out, o[d], 4 * x, 1.f);
        if (sizeof(T) == 2 && p.out_low != nullptr) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] -= static_cast<float>(static_cast<T>(o[d][e]));
#pragma unroll
            for (int x = 0; x < 4; ++x)
                store4<T>(static_cast<T*>(p.out_low) + out_at, 32 * d + 8 * x + 4 * half, p.D, vec_out, o[d], 4 * x, 1.f);
        }
    }
    if (p.stats != nullptr && half == 0) {
        float* const st = static_cast<float*>(p.stats) + 2 * row;
        st[0] = l == 0.f ? 0.f : m;
        st[1] = l == 0.f ? 0.f : __builtin_amdgcn_logf(l) - shift_of<T>(m);
    }
}

// Joins the parts of each row: out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s. A row has 256 / rows threads of the
// workgroup: with many parts all of them (a decoded token over a long cache has few rows and hundreds of parts), which
// each add every fourth or so part of a channel; with a few parts one for each channel.
constexpr int kJoinParts = 1024;  // most parts of a row (shape_of)
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnParams p, Split sp, int wide, int rows, int tile_rows,
                                                        int tiles) {
    __shared__ float factor[kJoinParts], part[256];
    const int t = threadIdx.x, each = 256 / rows, x = t % each, n = sp.t.n;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * rows + t / each;  // row of a tile that is split
    const int left = static_cast<int>(at / tile_rows), row = static_cast<int>(at % tile_rows);
    const int tile = sp.t.whole + left, bh = tile / tiles, r = (tiles - 1 - tile % tiles) * tile_rows + row;
    const bool live = r < p.rows;
    if (rows == 1 && !live) return;
    const int64_t part0 = (static_cast<int64_t>(left) * n) * tile_rows + row;  // part s: + s * tile_rows
    const int b = bh / p.Hk, i = static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(live ? r : 0)));
    const int h = bh % p.Hk * p.G + (live ? r : 0) - i * p.G;
    float m = kNegInf, l = 0.f, o = 0.f;
    const int d = x % wide, group = x / wide, groups = each / wide;
    if (rows == 1) {
        for (int s = t; s < n; s += 256) m = __builtin_fmaxf(m, sp.ml[2 * (part0 + static_cast<int64_t>(s) * tile_rows)]);
#pragma unroll
        for (int y = 32; y > 0; y >>= 1) m = __builtin_fmaxf(m, xor_lane(m, y));
        if (t % kWave == 0) part[t / kWave] = m;
        __syncthreads();
        m = __builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3]));
        for (int s = t; s < n; s += 256) {
            const float* ml = sp.ml + 2 * (part0 + static_cast<int64_t>(s) * tile_rows);
            const float f = ml[0] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m);
            factor[s] = f;
            l = fmaf(ml[1], f, l);
        }
        l = wave_sum(l);
        if (t % kWave == 0) part[4 + t / kWave] = l;
        __syncthreads();
        l = (part[4] + part[5]) + (part[6] + part[7]);
        if (d < p.D) {
#pragma unroll 4
            for (int s = group; s < n; s += groups) {
                const float f = factor[s];
                if (f != 0.f) o = fmaf(sp.o[(part0 + static_cast<int64_t>(s) * tile_rows) * p.D + d], f, o);
            }
        }
        __syncthreads();
        part[t] = o;
        __syncthreads();
        if (group == 0)
            for (int g = 1; g < groups; ++g) o += part[g * wide + d];
    } else if (live) {
        for (int s = 0; s < n; ++s) m = __builtin_fmaxf(m, sp.ml[2 * (part0 + static_cast<int64_t>(s) * tile_rows)]);
        for (int s = 0; s < n; ++s) {
            const int64_t q = part0 + static_cast<int64_t>(s) * tile_rows;
            const float f = sp.ml[2 * q] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(sp.ml[2 * q] - m);
            l = fmaf(sp.ml[2 * q + 1], f, l);
            if (f != 0.f && d < p.D) o = fmaf(sp.o[q * p.D + d], f, o);
        }
    }
    if (!live || group != 0) return;
    if (d < p.D) {
        const int64_t out_at = ((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D + d;
        o *= l == 0.f ? 0.f : 1.f / l;
        const T v = static_cast<T>(o);
        static_cast<T*>(p.out)[out_at] = v;
        if (sizeof(T) == 2 && p.out_low != nullptr)
            static_cast<T*>(p.out_low)[out_at] = static_cast<T>(o - static_cast<float>(v));
    }
    if (p.stats != nullptr && x == 0) {
        float* const st = static_cast<float*>(p.stats) + 2 * ((static_cast<int64_t>(b) * p.H + h) * p.Q + i);
        st[0] = l == 0.f ? 0.f : m;
        st[1] = l == 0.f ? 0.f : __builtin_amdgcn_logf(l) - shift_of<T>(m);
    }
}

// The launch shape. Workgroups of 256 rows that share key tiles, when they fill the GPU, with what is left over after an
// even share for every CU split (even_split); else workgroups of 32 rows with the keys over the wavefronts. Where either
// leaves CUs without work and the keys are many, the keys are split over workgroups too. Measured, both sides of each rule:
// private tiles below 512 x 128 rows (2 x 12 heads x 1500 of 64, bfloat16: 39 us, shared 53; 3 x 8 x 1100 of 32: 19, 34),
// but not for long loops of enough rows (2 x 8 x 1000 of 32 over 12000 keys: 87, shared in 8 parts 62; 8 heads x 100 over
// 8000: 21, shared 26). Parts below 256 workgroups (8 heads x 2000 as 504 private ones: 20 us whole, 28 in parts; 64 heads x
// 1100 as 320 shared ones: 38 whole, 62 in parts).
struct Shape {
    bool vec, wk;
    int tile_rows, tiles, keys;
    TileSplit t;
};

Shape shape_of(int dtype, const AttnParams& p) {
    const int elem = elem_size(dtype);
    auto ok = [&](const void* ptr, const int64_t (&s)[3]) {
        return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && s[0] * elem % 16 == 0 && s[1] * elem % 16 == 0 &&
               s[2] * elem % 16 == 0 && s[1] < (int64_t{1} << 31) / (64 * elem);
    };
    Shape s{};
    s.vec = p.D * elem % 16 == 0 && ok(p.q, p.qs) && ok(p.k, p.ks) && ok(p.v, p.vs);
    const int64_t heads = static_cast<int64_t>(p.B) * p.Hk;
    const bool can = s.vec && padded_width(p.D) * elem <= 256;  // wider rows' private tiles do not fit in registers
    const bool long_loop = p.K >= 8192 && p.rows >= 512;
    s.wk = can && !long_loop && heads * ((p.rows + 127) / 128) < 512;
    s.tile_rows = tile_rows(s.wk, padded_width(p.D) * elem);
    s.tiles = (p.rows + s.tile_rows - 1) / s.tile_rows;
    const int total = static_cast<int>(heads * s.tiles);
    s.t = TileSplit{1, total, total};
    if (s.wk && total < 256 && p.K > 1024) {
        int64_t n = (1024 + total - 1) / total;
        const int64_t most = (p.K + 511) / 512;
        n = n < most ? n : most;
        n = n < kJoinParts ? n : kJoinParts;
        s.t = TileSplit{static_cast<int>(n), 0, total};
    } else if (!s.wk && total < 256) {
        const int n = parts_of(total, padded_width(p.D) * elem <= 128 ? 512 : 256, p.K, dtype == kF32);
        s.t = TileSplit{n, n > 1 ? 0 : total, total};
    } else if (!s.wk && !p.causal) {  // causal tiles differ in length and even out by themselves
        s.t = even_split(total, (p.K + 63) / 64);
    }
    const int64_t keys = ((p.K + s.t.n - 1) / s.t.n + 127) / 128 * 128;
    s.keys = static_cast<int>(keys < 2147483520 ? keys : 2147483520);
    return s;
}

// Floats that the parts take: their outputs, maxima and sums
int64_t part_floats(const AttnParams& p, const Shape& s) {
    return static_cast<int64_t>(s.t.total - s.t.whole) * s.t.n * s.tile_rows * (p.D + 2);
}

template <typename T, int DP, bool WK, bool MASK, bool VEC>
int run(const AttnParams& p, const Shape& s, const Split& sp, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    constexpr int tile = 2 * key_tile<T, DP, WK>() * TileRows<T, DP>::kPitch;
    constexpr int join = (256 + 2 * 32 * (DP + 4)) * 4;
    constexpr int bytes = WK ? (4 * tile > join ? 4 * tile : join) : tile;
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
    auto* const fn = &attn_forward_kernel<T, DP, WK, MASK, VEC>;
    const hipError_t e =
        bytes > 64 * 1024 ? allow_dynamic_lds(reinterpret_cast<const void*>(fn), bytes, done) : hipSuccess;
    if (e != hipSuccess) return set_error(TD_E_LAUNCH, "attention: LDS size: %s", hipGetErrorString(e));
    const bool vec_out = p.D % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.out_low)) %
                                                 (4 * sizeof(T)) == 0;
    hipLaunchKernelGGL(fn, dim3(tile_grid(sp.t)), dim3(kWaves<T, DP, WK> * kWave), bytes, stream, p, sp, vec_out, s.tiles);
    if (sp.t.n > 1) {
        const int rows = sp.t.n <= 16 ? 256 / padded_width(p.D) : 1;  // of a workgroup; a tile's are a multiple of it
        const int64_t groups = static_cast<int64_t>(sp.t.total - sp.t.whole) * s.tile_rows / rows;
        hipLaunchKernelGGL((attn_join_kernel<T>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, stream, p, sp,
                           padded_width(p.D), rows, s.tile_rows, s.tiles);
    }
    const hipError_t le = hipGetLastError();
    return le == hipSuccess ? 0 : set_error(TD_E_LAUNCH, "attention launch failed: %s", hipGetErrorString(le));
}

template <typename T, int DP>
int run_dp(const AttnParams& p, const Shape& s, const Split& sp, hipStream_t stream) {
    const bool mask = p.mask_type != TD_MASK_NONE && p.K > 0;
    if (!s.vec)
        return mask ? run<T, DP, false, true, false>(p, s, sp, stream)
                    : run<T, DP, false, false, false>(p, s, sp, stream);
    if constexpr (DP * sizeof(T) <= 256)
        if (s.wk)
            return mask ? run<T, DP, true, true, true>(p, s, sp, stream)
                        : run<T, DP, true, false, true>(p, s, sp, stream);
    return mask ? run<T, DP, false, true, true>(p, s, sp, stream)
                : run<T, DP, false, false, true>(p, s, sp, stream);
}

}  // namespace

template <typename T>
int launch_attn_forward_t(int dtype, const AttnParams& p, hipStream_t stream) {
    const Shape s = shape_of(dtype, p);
    AttnParams q = p;
    float* const ws = reinterpret_cast<float*>(static_cast<unsigned char*>(p.ws) + plan_mask(q, p.ws));
    const Split sp{s.t, s.keys, ws, ws + part_floats(p, s) / (p.D + 2) * p.D};
    const int rc = launch_mask(dtype, q, stream);
    if (rc != 0) return rc;
    switch (padded_width(p.D)) {
        case 32: return run_dp<T, 32>(q, s, sp, stream);
        case 64: return run_dp<T, 64>(q, s, sp, stream);
        case 96: return run_dp<T, 96>(q, s, sp, stream);
        case 128: return run_dp<T, 128>(q, s, sp, stream);
        default: return run_dp<T, 256>(q, s, sp, stream);
    }
}

#if TD_ATTN_TYPE == 0
extern template int launch_attn_forward_t<f16>(int, const AttnParams&, hipStream_t);
extern template int launch_attn_forward_t<bf16>(int, const AttnParams&, hipStream_t);
template int launch_attn_forward_t<float>(int, const AttnParams&, hipStream_t);

int64_t attn_forward_workspace(int dtype, const AttnParams& p) {
    if (dtype == kF64) return 0;
    const Shape s = shape_of(dtype, p);
    AttnParams q = p;
    return plan_mask(q, nullptr) + part_floats(p, s) * 4;
}

int launch_attn_forward(int dtype, const AttnParams& p, hipStream_t stream) {
    switch (dtype) {
        case kF32: return launch_attn_forward_t<float>(dtype, p, stream);
        case kF16: return launch_attn_forward_t<f16>(dtype, p, stream);
        default: return launch_attn_forward_t<bf16>(dtype, p, stream);
    }
}
#elif TD_ATTN_TYPE == 1
template int launch_attn_forward_t<f16>(int, const AttnParams&, hipStream_t);
#else
template int launch_attn_forward_t<bf16>(int, const AttnParams&, hipStream_t);
#endif

}  // namespace td
