// Attention among tokens, backward, on the matrix units (float32, float16, bfloat16): the probabilities are computed again
// from the scores and the forward's statistics, P = 2^(t - m - log2 l), and with g = grad_out
//   dV = P^T g,  dP = g V^T,  dS = P (dP - delta),  delta = g . out,  dQ = scale dS K,  dK = scale dS^T Q.
// Three launches: delta (and the statistics in the order of the problem's rows); dQ, a workgroup's rows against every key,
// as the forward; dK and dV, a workgroup's keys against every row, so that no sum needs an atomic. That computes scores
// and dP twice, 7 products where 5 would do; the other way, dQ summed over key blocks in memory, moves 8 D bytes (read and
// written) for each row and block of 256 keys, and its order or its atomics change the result.
//
// P and dS are rounded to the inputs' type for their products: half a step of each, which leaves dQ and dK of 16-bit inputs
// with 1.4 to 1.5 times the error of one rounding at the end (a second, low part of dS would take that out for another
// product).
//
// Bound by the vector units where heads are narrow, by LDS reads beside the MFMAs where they are wide: 8400 tokens x 8
// heads of 32, float16, batch 2: dQ 320 us (680 TFLOP/s), dK and dV 410 (700); 4096 x 16 heads of 64, bfloat16: 240 (860)
// and 316 (870); of 128: 435 (950) and 688 (800).
#include "td_attn_mma.h"

#ifndef TD_ATTN_TYPE
#error "TD_ATTN_TYPE"
#endif

namespace td {
namespace {

// What the gradient kernels read of a row: m, log2 l, delta.
struct RowInfo {
    f32x4* rows;    // [B * Hk][rows]
    float* amax;    // float16: [B * Hk][blocks] largest |g| of 64 rows, then [B * Hk][key_blocks] largest |v| of 64 keys
    int blocks, key_blocks;
};

// float16 holds P as 2^15 P (normal numbers down to 2^-29) and dS as 2^15 P (dP - delta) 2^-e, e the exponent of
// 2 D max|g| max|v| >= |dP - delta|: it cannot overflow, and a product 2^8 under that bound with a P of 2^-13 still has
// all its bits. The other types have float32's exponents and need neither.
template <typename T>
constexpr bool kScaled = std::is_same<T, f16>::value;
template <typename T>
constexpr float kPShift = kScaled<T> ? 15.f : 0.f;

constexpr int kInfoRows = 64;

// 64 rows (or, in float16, the keys' values) a workgroup, four threads each
template <typename T>
__global__ __launch_bounds__(256) void attn_info_kernel(AttnParams p, RowInfo info, bool vec) {
    __shared__ float best[4];
    const int per = info.blocks + (kScaled<T> ? info.key_blocks : 0);
    const int bh = blockIdx.x / per, block = blockIdx.x % per, b = bh / p.Hk, hk = bh % p.Hk;
    const int t = threadIdx.x, part = t & 3;
    constexpr int E = 16 / static_cast<int>(sizeof(T));
    const bool is_row = block < info.blocks;
    const int n = (is_row ? block : block - info.blocks) * kInfoRows + (t >> 2);
    float top = 0.f;
    auto see = [&](float v) {
        const float a = __builtin_fabsf(v);
        top = a < __builtin_inff() && a > top ? a : top;  // what is not finite shows in the results by itself
    };
    if (is_row) {
        float delta = 0.f;
        if (n < p.rows) {
            const int i = static_cast<int>(fast_div(p.gdiv, n)), h = hk * p.G + n - i * p.G;
            const int64_t at = ((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D;
            const T *g = static_cast<const T*>(p.go) + at, *o = static_cast<const T*>(p.out) + at;
            const T* low = p.out_low == nullptr ? nullptr : static_cast<const T*>(p.out_low) + at;
            if (vec) {
                for (int d = part * E; d < p.D; d += 4 * E) {
                    float x[E], y[E];
                    VecIO<T, E>::unpack(VecIO<T, E>::load(g + d), x);
                    VecIO<T, E>::unpack(VecIO<T, E>::load(o + d), y);
                    if (low != nullptr) {
                        float z[E];
                        VecIO<T, E>::unpack(VecIO<T, E>::load(low + d), z);
#pragma unroll
                        for (int e = 0; e < E; ++e) y[e] += z[e];
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        delta = fmaf(x[e], y[e], delta);
                        see(x[e]);
                    }
                }
            } else {
                for (int d = part; d < p.D; d += 4) {
                    const float y = static_cast<float>(o[d]) + (low == nullptr ? 0.f : static_cast<float>(low[d]));
                    delta = fmaf(static_cast<float>(g[d]), y, delta);
                    see(static_cast<float>(g[d]));
                }
            }
            delta += xor_lane(delta, 1);
            delta += xor_lane(delta, 2);
            if (part == 0) {
                const float* st =
                    static_cast<const float*>(p.stats) + 2 * ((static_cast<int64_t>(b) * p.H + h) * p.Q + i);
                info.rows[static_cast<int64_t>(bh) * p.rows + n] = f32x4{st[0], st[1], delta, 0.f};
            }
        }
    } else if (n < p.K && (p.pad == nullptr || p.pad[static_cast<int64_t>(b) * p.K + n] == 0)) {
        const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + n * p.vs[1] + hk * p.vs[2];
        for (int d = part; d < p.D; d += 4) see(static_cast<float>(v[d]));
    }
    if constexpr (kScaled<T>) {
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) top = __builtin_fmaxf(top, xor_lane(top, x));
        if (t % kWave == 0) best[t / kWave] = top;
        __syncthreads();
        if (t == 0) {
            top = __builtin_fmaxf(__builtin_fmaxf(best[0], best[1]), __builtin_fmaxf(best[2], best[3]));
            const int64_t heads = static_cast<int64_t>(p.B) * p.Hk;
            if (is_row)
                info.amax[static_cast<int64_t>(bh) * info.blocks + block] = top;
            else
                info.amax[heads * info.blocks + static_cast<int64_t>(bh) * info.key_blocks + block - info.blocks] = top;
        }
    }
}

// The power of two that dP - delta is multiplied by (float16), a wavefront's lanes together
template <typename T>
__device__ __forceinline__ float ds_factor(const AttnParams& p, const RowInfo& info, int bh, int lane) {
    if constexpr (!kScaled<T>) return 1.f;
    const float* g = info.amax + static_cast<int64_t>(bh) * info.blocks;
    const float* v = info.amax + static_cast<int64_t>(p.B) * p.Hk * info.blocks +
                     static_cast<int64_t>(bh) * info.key_blocks;
    float a = 0.f, c = 0.f;
    for (int i = lane; i < info.blocks; i += kWave) a = __builtin_fmaxf(a, g[i]);
    for (int i = lane; i < info.key_blocks; i += kWave) c = __builtin_fmaxf(c, v[i]);
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) {
        a = __builtin_fmaxf(a, xor_lane(a, x));
        c = __builtin_fmaxf(c, xor_lane(c, x));
    }
    // 2 D max|g| max|v| < 2^42: an exponent from the float's bits, and none below 2^-100 (nothing but zeros)
    const unsigned u = __builtin_bit_cast(unsigned, __builtin_fmaxf(2.f * p.D * a * c, 0x1p-100f));
    const unsigned e = (u >> 23) + 1;                      // the bound is below 2^(e - 127)
    return __builtin_bit_cast(float, (254u - e) << 23);    // 2^(127 - e)
}

// Bytes of a row, as the tiles' heights go by them: 32 rows of 192 bytes are no whole number of pieces for 256 threads
template <typename T, int DP>
constexpr int staged_bytes() {
    return DP * static_cast<int>(sizeof(T)) == 192 ? 128 : DP * static_cast<int>(sizeof(T));
}

// dQ. The forward's shape, WK: private key tiles, the wavefronts' sums joined in LDS.
template <typename T, int DP, bool WK>
constexpr int dq_key_tile() {
    return WK || staged_bytes<T, DP>() > 128 ? 32 : 64;
}
// Wavefronts a SIMD that the registers leave room for with few spills or none. A workgroup of eight takes two of each SIMD.
// dK and dV under a mask (SLOW) stay at two: at four they spill 90 to 120 registers (1100 x 64 heads of 32, bfloat16: 87
// us, 182 with the spills).
template <typename T, int DP, bool WK, bool SLOW>
constexpr int dq_min_waves() {
    constexpr int bytes = DP * static_cast<int>(sizeof(T));
    if (WK) return bytes <= 64 && !SLOW ? 3 : bytes <= 128 ? 2 : 1;
    return bytes <= 64 || (bytes <= 128 && !SLOW) ? 4 : bytes <= 256 ? 2 : 1;
}
template <typename T, int DP, bool WK, bool SLOW>
constexpr int dkv_min_waves() {
    constexpr int bytes = DP * static_cast<int>(sizeof(T));
    if (WK) return bytes <= 64 && !SLOW ? 3 : bytes <= 128 ? 2 : 1;
    return bytes <= 64 && !SLOW ? 4 : bytes <= 256 ? 2 : 1;
}

// Sums over many keys (dQ) or rows (dK, dV) that are split over workgroups (TileSplit) leave float32 parts, which
// sum_parts_kernel adds in their order.
struct Parts {
    TileSplit t;
    float *a, *b;  // dQ, or dK and dV: [..][rows of a tile][D]
};

// Four channels of a row of a split tile a thread. keys: the rows are keys (dK, dV), else the problem's rows (dQ).
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(AttnParams p, TileSplit t, const float* __restrict__ part,
                                                        T* __restrict__ out, int quads, int tile_rows, int tiles,
                                                        bool keys, bool vec) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int d = static_cast<int>(id % quads) * 4;
    const int64_t at = id / quads;
    const int left = static_cast<int>(at / tile_rows), row = static_cast<int>(at % tile_rows);
    if (left >= t.total - t.whole || d >= p.D) return;
    const int tile = t.whole + left, bh = tile / tiles, b = bh / p.Hk, hk = bh % p.Hk;
    const int r = (keys ? tile % tiles : tiles - 1 - tile % tiles) * tile_rows + row;
    if (r >= (keys ? p.K : p.rows)) return;
    const float* at0 = part + (static_cast<int64_t>(left) * t.n * tile_rows + row) * p.D;
    const int64_t step = static_cast<int64_t>(tile_rows) * p.D;
    f32x16 s = f32x16{0.f};
#pragma unroll 4
    for (int k = 0; k < t.n; ++k) {
        const float* from = at0 + k * step + d;
        if (vec) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(from);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < p.D) s[e] += from[e];
        }
    }
    int64_t to;
    if (keys) {
        to = (static_cast<int64_t>(b) * p.K + r) * p.Hk + hk;
    } else {
        const int i = static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(r)));
        to = (static_cast<int64_t>(b) * p.Q + i) * p.H + hk * p.G + r - i * p.G;
    }
    store4<T>(out + to * p.D, d, p.D, vec && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(T)) == 0, s, 0, 1.f);
}

template <typename T>
void sum_parts(const AttnParams& p, const TileSplit& t, const float* part, void* out, int tile_rows, int tiles, bool keys,
               hipStream_t stream) {
    const int quads = (p.D + 3) / 4;
    const int64_t threads = static_cast<int64_t>(t.total - t.whole) * tile_rows * quads;
    hipLaunchKernelGGL((sum_parts_kernel<T>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, stream, p, t,
                       part, static_cast<T*>(out), quads, tile_rows, tiles, keys, p.D % 4 == 0);
}
template <typename T, int DP, bool WK, bool MASK, bool VEC>
__global__ __launch_bounds__((kWaves<T, DP, WK> * kWave), (dq_min_waves<T, DP, WK, MASK>())) void attn_dq_kernel(
    AttnParams p, RowInfo info, Parts parts, bool vec_out, int tiles) {
    using R = TileRows<T, DP>;
    constexpr int KT = dq_key_tile<T, DP, WK>(), ND = DP / 32, BM = kTileRows<T, DP, WK>;
    constexpr int kTile = KT * R::kPitch;
    extern __shared__ __align__(16) unsigned char lds[];
    const TileWork work = tile_work(parts.t);
    if (work.tile < 0) return;
    const int tile = tiles - 1 - work.tile % tiles, bh = work.tile / tiles;  // causal: the long ones first
    const int b = bh / p.Hk, hk = bh % p.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int lane = threadIdx.x % kWave, half = lane >> 5;
    unsigned char* const kt_lds = lds + (WK ? wave * 2 * kTile : 0);
    unsigned char* const vt_lds = kt_lds + kTile;

    const int row0 = tile * BM, wrow0 = row0 + (WK ? 0 : wave * 32), r = wrow0 + (lane & 31);
    const bool live = r < p.rows;
    const int i = static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(live ? r : 0)));
    const int h = hk * p.G + (live ? r : 0) - i * p.G;
    const int64_t out_at = ((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D;
    u32x4 qf[R::kChunks], gf[R::kChunks];
    {
        const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
        const T* g = static_cast<const T*>(p.go) + out_at;
#pragma unroll
        for (int c = 0; c < R::kChunks; ++c) {
            qf[c] = live ? row_piece<T, VEC>(q, c * 32 + half * 16, p.D) : u32x4{0u, 0u, 0u, 0u};
            gf[c] = live ? row_piece<T, VEC>(g, c * 32 + half * 16, p.D) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    const f32x4 ri = info.rows[static_cast<int64_t>(bh) * p.rows + (live ? r : 0)];
    const float ds_scale = ds_factor<T>(p, info, bh, lane);
    const float delta = ri[2] * ds_scale;
    const T* const mrow = MASK ? static_cast<const T*>(p.mask) + b * p.ms[0] + h * p.ms[1] + i * p.ms[2] : nullptr;
    // log2 l would be lost beside a large m (of large scores, or of an additive mask): it is subtracted after t - m then
    const bool apart = __any(live && big_score(ri[0])) || (MASK && p.mask_type == TD_MASK_FLOAT);
    const float from = (apart ? 0.f : ri[0]) + (ri[1] - kPShift<T>);
    const int diag = static_cast<int>(p.diag);
    const int last = p.causal ? i + diag : 2147483647;
    int kend = p.K;
    const int top_row = (row0 + BM < p.rows ? row0 + BM : p.rows) - 1;
    if (p.causal) {
        const int seen = static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(top_row))) + diag + 1;
        kend = seen < kend ? seen : kend;
    }
    const int wtop = wrow0 + 31 < p.rows ? wrow0 + 31 : p.rows - 1;
    const int wfirst = wrow0 < p.rows ? wrow0 : p.rows - 1;
    const int seen_all = p.causal ? static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(wfirst))) + diag : 2147483647;
    const int seen_any = p.causal ? static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(wtop))) + diag : 2147483647;

    const T* const kb = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* const vb = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
    const uint8_t* const pad = p.pad == nullptr ? nullptr : p.pad + static_cast<int64_t>(b) * p.K;
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
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[d] = f32x16{0.f};

    constexpr int step = WK ? 4 * KT : KT;
    constexpr uint64_t all = KT == 64 ? ~uint64_t{0} : (uint64_t{1} << (KT & 63)) - 1;
    int64_t j0 = WK ? wave * KT : 0;
    if (work.parts > 1) {
        const int64_t n = work.parts, each = ((kend > 0 ? kend : 0) + n * step - 1) / (n * step) * step;
        j0 += work.part * each;
        kend = (work.part + 1) * each < kend ? static_cast<int>((work.part + 1) * each) : kend;
    }
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
        uint32_t bits[KT / 32];
        bool masked[KT / 32], values[KT / 32], none[KT / 32];
#pragma unroll
        for (int x = 0; x < KT / 32; ++x) {
            const uint32_t pad_bits = static_cast<uint32_t>(gone >> (32 * x));
            const int jx = static_cast<int>(j0) + 32 * x;
            bits[x] = mw[x].bits;
            masked[x] = pad_bits != 0 || jx + 31 > seen_all;
            none[x] = pad_bits == ~0u || jx > seen_any;
            values[x] = false;
            if constexpr (MASK) {
                masked[x] |= __any(mw[x].kind != kMaskNone);
                values[x] = __any(mw[x].kind == kMaskValues);
                none[x] |= __all(mw[x].kind == kMaskAll);
            }
        }
        if (j0 + step < kend) {
            fetch(j0 + step, gone_next);
            next_pad = pad_byte(j0 + 2 * step);
        }
        const int j = static_cast<int>(j0);
        {
#pragma unroll
            for (int x = 0; x < KT / 32; ++x) {
                if (none[x]) continue;
                f32x16 s = f32x16{0.f}, dp = f32x16{0.f};
#pragma unroll
                for (int c = 0; c < R::kChunks; ++c) {
                    s = Mma<T>::mul(R::rows(kt_lds, 32 * x, c, lane), qf[c], s);
                    dp = Mma<T>::mul(R::rows(vt_lds, 32 * x, c, lane), gf[c], dp);
                }
                float cc = p.c;
                if (masked[x]) {
                    cc = 1.f;
                    mask_scores<T>(s, p.c,
                                   bits[x] | static_cast<uint32_t>(gone >> (32 * x)) | beyond(j + 32 * x, last),
                                   values[x] ? mrow + j + 32 * x : nullptr, p.K - j - 32 * x, half);
                }
                if (apart) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = rounded_product(s[e], cc) - ri[0];
                    cc = 1.f;
                }
                f32x16 ds;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    ds[e] = __builtin_amdgcn_exp2f(fmaf(s[e], cc, -from)) * fmaf(dp[e], ds_scale, -delta);
                typename R::Packed w[R::kPacked];
                R::pack(ds, w);
#pragma unroll
                for (int d = 0; d < ND; ++d) dq[d] = R::columns(kt_lds, 32 * x, 32 * d, lane, w, dq[d]);
            }
        }
        gone = gone_next;
        if (WK) wave_sync();
    }
    if constexpr (WK) {
        float* const part = reinterpret_cast<float*>(lds);
        const int at = (lane & 31) * (DP + 4) + 4 * half;
        constexpr int kPart = 32 * (DP + 4);
        __syncthreads();
#pragma unroll
        for (int n = 2; n > 0; n >>= 1) {
            if (wave >= n && wave < 2 * n) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        *reinterpret_cast<f32x4*>(part + (wave - n) * kPart + at + 32 * d + 8 * x) =
                            f32x4{dq[d][4 * x], dq[d][4 * x + 1], dq[d][4 * x + 2], dq[d][4 * x + 3]};
            }
            __syncthreads();
            if (wave < n) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(part + wave * kPart + at + 32 * d + 8 * x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dq[d][4 * x + e] += v[e];
                    }
            }
            __syncthreads();
        }
        if (wave != 0) return;
    }
    if (!live) return;
    const float back = static_cast<float>(p.scale) / ds_scale * (kScaled<T> ? 0x1p-15f : 1.f);
    const int64_t part_at = ((static_cast<int64_t>(work.tile - parts.t.whole) * work.parts + work.part) * BM + r -
                             row0) * p.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int at = 32 * d + 8 * x + 4 * half;
            if (work.parts > 1)
                store4<float>(parts.a + part_at, at, p.D, p.D % 4 == 0, dq[d], 4 * x, back);
            else
                store4<T>(static_cast<T*>(p.dq) + out_at, at, p.D, vec_out, dq[d], 4 * x, back);
        }
}

// dK and dV. WK: private row tiles. The scores stand untransposed here (a lane's column is its key), so that P and dS are
// operands of dV^T = g^T P and dK^T = Q^T dS as they stand. Rows past the end hold zeros and m = inf: P = 0.
template <typename T, int DP, bool WK>
constexpr int dkv_row_tile() {
    return WK || staged_bytes<T, DP>() > 128 ? 32 : 64;
}

// V of wide heads stays in LDS: its fragments would spill. With dK and dV the registers hold K's fragments only.
template <typename T, int DP, bool WK>
constexpr bool v_in_lds() {
    return !WK && DP * static_cast<int>(sizeof(T)) == 256;
}
// What LDS holds of a row beside its elements: m + log2 l (or log2 l, and m apart from it), delta, the mask words of the
// workgroup's keys, and with a mask its kind for each word and the row's offset in it
template <typename T, int DP, bool WK, bool MASK>
constexpr int dkv_row_bytes() {
    constexpr int words = kTileRows<T, DP, WK> / 8;  // bytes
    return 12 + words + (MASK ? 8 + words : 0) + (words == 4 ? 0 : 4);  // a multiple of 4 that leaves tiles 16-byte aligned
}

template <typename T, int DP, bool WK, bool MASK, bool VEC>
__global__ __launch_bounds__((kWaves<T, DP, WK> * kWave), (dkv_min_waves<T, DP, WK, MASK>())) void attn_dkv_kernel(
    AttnParams p, RowInfo info, Parts parts, bool vec_out, int tiles) {
    using R = TileRows<T, DP>;
    constexpr int RT = dkv_row_tile<T, DP, WK>(), ND = DP / 32, BM = kTileRows<T, DP, WK>;
    constexpr int kTile = RT * R::kPitch;
    constexpr int KW = BM / 32;  // words of 32 keys that the workgroup's keys have
    constexpr int kArea = 2 * kTile + RT * dkv_row_bytes<T, DP, WK, MASK>();
    extern __shared__ __align__(16) unsigned char lds[];
    const TileWork work = tile_work(parts.t);
    if (work.tile < 0) return;
    const int tile = work.tile % tiles, bh = work.tile / tiles;  // causal: the first keys are seen by the most rows
    const int b = bh / p.Hk, hk = bh % p.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int lane = threadIdx.x % kWave, half = lane >> 5;
    const int t = WK ? lane : static_cast<int>(threadIdx.x);
    unsigned char* const q_lds = lds + (WK ? wave * kArea : 0);
    unsigned char* const g_lds = q_lds + kTile;
    float* const m_lds = reinterpret_cast<float*>(g_lds + kTile);
    float* const a_lds = m_lds + RT;
    float* const d_lds = a_lds + RT;
    uint32_t* const w_lds = reinterpret_cast<uint32_t*>(d_lds + RT);   // [KW][RT]
    int* const k_lds = reinterpret_cast<int*>(w_lds + KW * RT);        // [KW][RT], with a mask
    int64_t* const o_lds = reinterpret_cast<int64_t*>(k_lds + KW * RT);

    // the lane's key
    const int key0 = tile * BM, wkey0 = key0 + (WK ? 0 : wave * 32), j = wkey0 + (lane & 31);
    const bool live = j < p.K && (p.pad == nullptr || p.pad[static_cast<int64_t>(b) * p.K + j] == 0);
    constexpr bool kVInLds = v_in_lds<T, DP, WK>();
    u32x4 kf[R::kChunks], vf[kVInLds ? 1 : R::kChunks];
    unsigned char* const v_own = lds + kArea;
    {
        const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + j * p.ks[1] + hk * p.ks[2];
        const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + j * p.vs[1] + hk * p.vs[2];
#pragma unroll
        for (int c = 0; c < R::kChunks; ++c) {
            kf[c] = live ? row_piece<T, VEC>(k, c * 32 + half * 16, p.D) : u32x4{0u, 0u, 0u, 0u};
            const u32x4 vc = live ? row_piece<T, VEC>(v, c * 32 + half * 16, p.D) : u32x4{0u, 0u, 0u, 0u};
            if constexpr (kVInLds)  // the wavefront's own rows: read back by this wavefront alone
                *reinterpret_cast<u32x4*>(v_own + (wave * 32 + (lane & 31)) * R::kPitch + c * 32 + half * 16) = vc;
            else
                vf[c] = vc;
        }
    }
    const float ds_scale = ds_factor<T>(p, info, bh, lane);
    const bool apart = MASK && p.mask_type == TD_MASK_FLOAT;
    const int diag = static_cast<int>(p.diag);
    const int mask_key = j < p.K ? j : p.K - 1;

    // rows that see any of the workgroup's keys (or the wavefront's): query >= key - diag
    int64_t r0 = 0;
    const int first_q = key0 - diag > 0 ? key0 - diag : 0, wfirst_q = wkey0 - diag > 0 ? wkey0 - diag : 0;
    if (p.causal) r0 = static_cast<int64_t>(first_q) * p.G / RT * RT;
    const int64_t wfirst_row = p.causal ? static_cast<int64_t>(wfirst_q) * p.G : 0;
    // from this row on every key of the wavefront is seen
    const int64_t whole_row = p.causal ? (static_cast<int64_t>(wkey0) + 31 - diag) * p.G : 0;
    const bool any = __any(live);

    const T* const qb = static_cast<const T*>(p.q) + b * p.qs[0] + hk * p.G * p.qs[2];
    const int64_t gs1 = static_cast<int64_t>(p.H) * p.D, gs2 = p.D;
    const T* const gb = static_cast<const T*>(p.go) + b * p.Q * gs1 + hk * p.G * gs2;
    const f32x4* const ib = info.rows + static_cast<int64_t>(bh) * p.rows;
    TwoTiles<T, DP, RT, WK, VEC> staged;
    // rows of a tile lie the same in every tile when the heads of a key head divide it
    const bool even = RT % p.G == 0;
    int64_t from_row = 0;
    auto split_row = [&](int x, int& i, int& g) {
        const uint32_t r = static_cast<uint32_t>(from_row + x);
        i = static_cast<int>(fast_div(p.gdiv, r));
        g = static_cast<int>(r) - i * p.G;
        i -= static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(from_row)));
    };
    auto q_row = [&](int x) {
        int i, g;
        split_row(x, i, g);
        return i * p.qs[1] + g * p.qs[2];
    };
    auto g_row = [&](int x) {
        int i, g;
        split_row(x, i, g);
        return i * gs1 + g * gs2;
    };
    if (even) staged.plan(q_row, g_row, p.D);
    f32x4 ri = f32x4{0.f, 0.f, 0.f, 0.f};
    int64_t mo = 0;
    MaskWord words[KW] = {};
    bool in_rows = false;
    int sees = 0;  // the last key that the row sees
    const bool bits = MASK || p.causal;
    auto fetch = [&](int64_t at) {
        from_row = at;
        const int64_t left = p.rows - at;
        const uint64_t gone = left >= RT ? 0 : ~uint64_t{0} << left;
        if (!even) staged.plan(q_row, g_row, p.D);
        const int64_t i0 = fast_div(p.gdiv, static_cast<uint32_t>(at));
        staged.load(qb + i0 * p.qs[1], q_row, gb + i0 * gs1, g_row, gone, p.D);
        if (t < RT) {
            const bool in = in_rows = t < left;
            ri = in ? ib[at + t] : f32x4{__builtin_inff(), 0.f, 0.f, 0.f};
            if (bits) {
                const int i = static_cast<int>(fast_div(p.gdiv, static_cast<uint32_t>(in ? at + t : 0)));
                const int h = hk * p.G + static_cast<int>(in ? at + t : 0) - i * p.G;
                if (MASK) mo = b * p.ms[0] + h * p.ms[1] + i * p.ms[2];
                sees = p.causal ? i + diag : 2147483647;
                if (MASK)
#pragma unroll
                    for (int w = 0; w < KW; ++w) words[w] = mask_word(p, b, h, i, key0 / 32 + w);
            }
        }
    };
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{0.f};

    constexpr int step = WK ? 4 * RT : RT;
    int64_t rend = p.rows;
    if (work.parts > 1) {
        const int64_t n = work.parts, each = (p.rows > r0 ? p.rows - r0 + n * step - 1 : 0) / (n * step) * step;
        r0 += work.part * each;
        rend = r0 + each < rend ? r0 + each : rend;
    }
    if (WK) r0 += wave * RT;
    if (r0 < rend) fetch(r0);
    for (; r0 < rend; r0 += step) {
        if (!WK) __syncthreads();
        staged.store(q_lds, g_lds, p.D);
        if (t < RT) {
            const bool two = ri[0] < __builtin_inff() && (apart || big_score(ri[0]));
            m_lds[t] = (two ? 0.f : ri[0]) + (ri[1] - kPShift<T>);
            a_lds[t] = two ? ri[0] : 0.f;
            d_lds[t] = ri[2] * ds_scale;
            if (MASK) o_lds[t] = mo;
            if (bits) {
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    w_lds[w * RT + t] = words[w].bits | beyond(key0 + 32 * w, sees);
                    if (MASK) k_lds[w * RT + t] = in_rows ? words[w].kind : kMaskAll;
                }
            }
        }
        if (WK)
            wave_sync();
        else
            __syncthreads();
        if (r0 + step < rend) fetch(r0 + step);
        if (any && r0 + RT > wfirst_row) {
            const uint32_t* const my_words = w_lds + (WK ? 0 : wave * RT);
#pragma unroll
            for (int x = 0; x < RT / 32; ++x) {
                bool masked = r0 + 32 * x < whole_row, values = false;
                if constexpr (MASK) {
                    const int kind = k_lds[(WK ? 0 : wave * RT) + 32 * x + (lane & 31)];
                    if (__all(kind == kMaskAll)) continue;
                    masked |= __any(kind != kMaskNone);
                    values = __any(kind == kMaskValues);
                }
                // the mask's values at the lane's key, on their way during the products where registers are left for them
                constexpr bool kEarly = MASK && DP * sizeof(T) <= 128;
                T entries[kEarly ? 16 : 1];
                if constexpr (kEarly)
                    if (values)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            entries[e] = static_cast<const T*>(
                                p.mask)[o_lds[32 * x + 8 * (e >> 2) + 4 * half + (e & 3)] + mask_key];
                f32x16 s = f32x16{0.f}, dp = f32x16{0.f};
#pragma unroll
                for (int c = 0; c < R::kChunks; ++c) {
                    s = Mma<T>::mul(R::rows(q_lds, 32 * x, c, lane), kf[c], s);
                    dp = Mma<T>::mul(R::rows(g_lds, 32 * x, c, lane),
                                     kVInLds ? R::rows(v_own, wave * 32, c, lane) : vf[kVInLds ? 0 : c], dp);
                }
                float cc = p.c;
                if (masked) {
                    cc = 1.f;
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int row = 32 * x + 8 * y + 4 * half;
                        const u32x4 w4 = *reinterpret_cast<const u32x4*>(my_words + row);
                        float add[4] = {0.f, 0.f, 0.f, 0.f};
                        if (kEarly && values) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                add[e] = mask_log2(static_cast<float>(entries[kEarly ? 4 * y + e : 0]));
                        } else if (MASK && values) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                add[e] = mask_log2(
                                    static_cast<float>(static_cast<const T*>(p.mask)[o_lds[row + e] + mask_key]));
                            __builtin_amdgcn_sched_barrier(0);  // four loads at a time: registers
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const unsigned w = w4[e];
                            const float t = fmaf(s[4 * y + e], p.c, add[e]);
                            s[4 * y + e] = (w >> (lane & 31)) & 1u ? kNegInf : t;
                        }
                    }
                }
                if (apart || __any(a_lds[32 * x + (lane & 31)] != 0.f)) {
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const f32x4 a4 = *reinterpret_cast<const f32x4*>(a_lds + 32 * x + 8 * y + 4 * half);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * y + e] = rounded_product(s[4 * y + e], cc) - a4[e];
                    }
                    cc = 1.f;
                }
                f32x16 ds;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int row = 32 * x + 8 * y + 4 * half;
                    const f32x4 m4 = *reinterpret_cast<const f32x4*>(m_lds + row);
                    const f32x4 d4 = *reinterpret_cast<const f32x4*>(d_lds + row);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float pr = __builtin_amdgcn_exp2f(fmaf(s[4 * y + e], cc, -m4[e]));
                        s[4 * y + e] = pr;
                        ds[4 * y + e] = pr * fmaf(dp[4 * y + e], ds_scale, -d4[e]);
                    }
                }
                typename R::Packed w[R::kPacked];
                R::pack(s, w);
#pragma unroll
                for (int d = 0; d < ND; ++d) dv[d] = R::columns(g_lds, 32 * x, 32 * d, lane, w, dv[d]);
                R::pack(ds, w);
#pragma unroll
                for (int d = 0; d < ND; ++d) dk[d] = R::columns(q_lds, 32 * x, 32 * d, lane, w, dk[d]);
            }
        }
        if (WK) wave_sync();
    }
    if constexpr (WK) {
        float* const part = reinterpret_cast<float*>(lds);
        const int at = (lane & 31) * (DP + 4) + 4 * half;
        constexpr int kPart = 32 * (DP + 4);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            f32x16(&sum)[ND] = which ? dv : dk;
            __syncthreads();
#pragma unroll
            for (int n = 2; n > 0; n >>= 1) {
                if (wave >= n && wave < 2 * n) {
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            *reinterpret_cast<f32x4*>(part + (wave - n) * kPart + at + 32 * d + 8 * x) =
                                f32x4{sum[d][4 * x], sum[d][4 * x + 1], sum[d][4 * x + 2], sum[d][4 * x + 3]};
                }
                __syncthreads();
                if (wave < n) {
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const f32x4 v = *reinterpret_cast<const f32x4*>(part + wave * kPart + at + 32 * d + 8 * x);
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum[d][4 * x + e] += v[e];
                        }
                }
                __syncthreads();
            }
        }
        if (wave != 0) return;
    }
    if (j >= p.K) return;
    const float pv = live ? (kScaled<T> ? 0x1p-15f : 1.f) : 0.f;
    const float back = static_cast<float>(p.scale) / ds_scale * (kScaled<T> ? 0x1p-15f : 1.f);
    const int64_t at = ((static_cast<int64_t>(b) * p.K + j) * p.Hk + hk) * p.D;
    const int64_t part_at = ((static_cast<int64_t>(work.tile - parts.t.whole) * work.parts + work.part) * BM + j -
                             key0) * p.D;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        if (!live) dk[d] = dv[d] = f32x16{0.f};  // a key that nobody sees: its column may hold anything
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int c = 32 * d + 8 * x + 4 * half;
            if (work.parts > 1) {
                store4<float>(parts.a + part_at, c, p.D, p.D % 4 == 0, dk[d], 4 * x, back);
                store4<float>(parts.b + part_at, c, p.D, p.D % 4 == 0, dv[d], 4 * x, pv);
            } else {
                store4<T>(static_cast<T*>(p.dk) + at, c, p.D, vec_out, dk[d], 4 * x, back);
                store4<T>(static_cast<T*>(p.dv) + at, c, p.D, vec_out, dv[d], 4 * x, pv);
            }
        }
    }
}

struct BackShape {
    bool vec;
    struct One {
        bool wk;
        int tile_rows, tiles;
        TileSplit t;
        int64_t part_floats(int D) const { return static_cast<int64_t>(t.total - t.whole) * t.n * tile_rows * D; }
    } q, k;
};

bool back_vec(int dtype, const AttnParams& p) {
    const int elem = elem_size(dtype);
    auto ok = [&](const void* ptr, const int64_t (&s)[3]) {
        return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && s[0] * elem % 16 == 0 && s[1] * elem % 16 == 0 &&
               s[2] * elem % 16 == 0 && s[1] < (int64_t{1} << 31) / (128 * elem) &&
               s[2] < (int64_t{1} << 31) / (int64_t{2} * p.G * elem);
    };
    return p.D * elem % 16 == 0 && ok(p.q, p.qs) && ok(p.k, p.ks) && ok(p.v, p.vs) &&
           reinterpret_cast<uintptr_t>(p.go) % 16 == 0 &&
           static_cast<int64_t>(p.H) * p.D < (int64_t{1} << 31) / (128 * elem);
}

// Workgroups of 256 rows (keys) that share tiles, when they fill the GPU; else of 32 rows (keys) with the others' tiles
// over the wavefronts, which needs no second launch, for heads whose private tiles fit in the registers. Where that
// still leaves CUs without work and the loops are long, parts; where many tiles leave a few over, parts of those
// (even_split). Measured, both sides: private below 384 x 128 rows (4 key heads x 16000 rows of 64, bfloat16, 500: dQ 170
// us, shared 143; 2 x 12 heads x 1500, 288: 53, shared 60, dK and dV 67, shared 86), but not for long loops (2 x 8 x 1000 of
// 32 over 12000 keys: dQ 87, shared 68); a part has 1024 steps or more of a private tile (3000 rows by 2 x 8 x 200 keys of 64:
// 33 us, with 512 39, with 256 45); parts below 256 shared workgroups (64 heads x 1100 as 320: dQ 45 us, in parts 52).
BackShape back_shape(int dtype, const AttnParams& p, bool vec) {
    BackShape s{};
    s.vec = vec;
    const int64_t heads = static_cast<int64_t>(p.B) * p.Hk;
    const bool can = vec && padded_width(p.D) * elem_size(dtype) <= 128;
    const int row_bytes = padded_width(p.D) * elem_size(dtype);
    // wide: the widest rows of which two workgroups fit on a CU
    auto shape = [&](int n, int over, int wide) {
        BackShape::One o{};
        const bool long_loop = over >= 8192 && n >= 512;
        o.wk = can && !long_loop && heads * ((n + 127) / 128) < 384;
        o.tile_rows = tile_rows(o.wk, padded_width(p.D) * elem_size(dtype));
        o.tiles = (n + o.tile_rows - 1) / o.tile_rows;
        const int total = static_cast<int>(heads * o.tiles);
        o.t = TileSplit{1, total, total};
        if (o.wk && total > 0 && total < 384) {
            const int want = (1024 + total - 1) / total, most = over / 1024, parts = want < most ? want : most;
            if (parts > 1) o.t = TileSplit{parts, 0, total};
        } else if (!o.wk && total > 0 && total < 256) {
            const int parts = parts_of(total, row_bytes <= wide ? 512 : 256, over, dtype == kF32);
            if (parts > 1) o.t = TileSplit{parts, 0, total};
        } else if (!o.wk && !p.causal) {
            o.t = even_split(total, (over + 63) / 64);
        }
        return o;
    };
    s.q = shape(p.rows, p.K, 128);
    s.k = shape(p.K, p.rows, 64);
    return s;
}

template <typename T, int DP, bool WK, bool MASK, bool VEC>
int run_dq(const AttnParams& p, const BackShape& s, const RowInfo& info, float* ws, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    constexpr int tile = 2 * dq_key_tile<T, DP, WK>() * TileRows<T, DP>::kPitch;
    constexpr int join = 2 * 32 * (DP + 4) * 4;
    constexpr int bytes = WK ? (4 * tile > join ? 4 * tile : join) : tile;
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
    auto* const fn = &attn_dq_kernel<T, DP, WK, MASK, VEC>;
    const hipError_t e =
        bytes > 64 * 1024 ? allow_dynamic_lds(reinterpret_cast<const void*>(fn), bytes, done) : hipSuccess;
    if (e != hipSuccess) return set_error(TD_E_LAUNCH, "attention backward: LDS size: %s", hipGetErrorString(e));
    const bool vec_out = p.D % 4 == 0 && reinterpret_cast<uintptr_t>(p.dq) % (4 * sizeof(T)) == 0;
    const Parts parts{s.q.t, ws, nullptr};
    hipLaunchKernelGGL(fn, dim3(tile_grid(s.q.t)), dim3(kWaves<T, DP, WK> * kWave), bytes, stream, p, info, parts, vec_out,
                       s.q.tiles);
    if (s.q.t.n > 1) sum_parts<T>(p, s.q.t, parts.a, p.dq, s.q.tile_rows, s.q.tiles, false, stream);
    return 0;
}

template <typename T, int DP, bool WK, bool MASK, bool VEC>
int run_dkv(const AttnParams& p, const BackShape& s, const RowInfo& info, float* ws, hipStream_t stream) {
    static std::atomic<uint64_t> done{0};
    constexpr int RT = dkv_row_tile<T, DP, WK>();
    constexpr int area = 2 * RT * TileRows<T, DP>::kPitch + RT * dkv_row_bytes<T, DP, WK, MASK>();
    constexpr int join = 2 * 32 * (DP + 4) * 4;
    constexpr int own = v_in_lds<T, DP, WK>() ? kTileRows<T, DP, WK> * TileRows<T, DP>::kPitch : 0;
    constexpr int bytes = WK ? (4 * area > join ? 4 * area : join) : area + own;
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
    auto* const fn = &attn_dkv_kernel<T, DP, WK, MASK, VEC>;
    const hipError_t e =
        bytes > 64 * 1024 ? allow_dynamic_lds(reinterpret_cast<const void*>(fn), bytes, done) : hipSuccess;
    if (e != hipSuccess) return set_error(TD_E_LAUNCH, "attention backward: LDS size: %s", hipGetErrorString(e));
    const bool vec_out = p.D % 4 == 0 && reinterpret_cast<uintptr_t>(p.dk) % (4 * sizeof(T)) == 0 &&
                         reinterpret_cast<uintptr_t>(p.dv) % (4 * sizeof(T)) == 0;
    const Parts parts{s.k.t, ws, ws + s.k.part_floats(p.D)};
    hipLaunchKernelGGL(fn, dim3(tile_grid(s.k.t)), dim3(kWaves<T, DP, WK> * kWave), bytes, stream, p, info, parts, vec_out,
                       s.k.tiles);
    if (s.k.t.n > 1) {
        sum_parts<T>(p, s.k.t, parts.a, p.dk, s.k.tile_rows, s.k.tiles, true, stream);
        sum_parts<T>(p, s.k.t, parts.b, p.dv, s.k.tile_rows, s.k.tiles, true, stream);
    }
    return 0;
}

template <typename T, int DP>
int run_dp(const AttnParams& p, const BackShape& s, const RowInfo& info, float* ws, hipStream_t stream) {
    const bool mask = p.mask_type != TD_MASK_NONE && p.K > 0;
    int rc = 0;
    if (p.dq != nullptr && p.rows > 0) {
        if (!s.vec)
            rc = mask ? run_dq<T, DP, false, true, false>(p, s, info, ws, stream)
                      : run_dq<T, DP, false, false, false>(p, s, info, ws, stream);
        else if (!s.q.wk)
            rc = mask ? run_dq<T, DP, false, true, true>(p, s, info, ws, stream)
                      : run_dq<T, DP, false, false, true>(p, s, info, ws, stream);
        else if constexpr (DP * sizeof(T) <= 128)
            rc = mask ? run_dq<T, DP, true, true, true>(p, s, info, ws, stream)
                      : run_dq<T, DP, true, false, true>(p, s, info, ws, stream);
    }
    if (rc == 0 && p.dk != nullptr && p.K > 0) {
        if (!s.vec)
            rc = mask ? run_dkv<T, DP, false, true, false>(p, s, info, ws, stream)
                      : run_dkv<T, DP, false, false, false>(p, s, info, ws, stream);
        else if (!s.k.wk)
            rc = mask ? run_dkv<T, DP, false, true, true>(p, s, info, ws, stream)
                      : run_dkv<T, DP, false, false, true>(p, s, info, ws, stream);
        else if constexpr (DP * sizeof(T) <= 128)
            rc = mask ? run_dkv<T, DP, true, true, true>(p, s, info, ws, stream)
                      : run_dkv<T, DP, true, false, true>(p, s, info, ws, stream);
    }
    return rc;
}

RowInfo info_of(const AttnParams& p, void* at) {
    RowInfo r{};
    r.rows = static_cast<f32x4*>(at);
    r.amax = reinterpret_cast<float*>(r.rows + static_cast<int64_t>(p.B) * p.Hk * p.rows);
    r.blocks = (p.rows + kInfoRows - 1) / kInfoRows;
    r.key_blocks = (p.K + kInfoRows - 1) / kInfoRows;
    return r;
}

// A multiple of 16
int64_t info_bytes(int dtype, const AttnParams& p) {
    const RowInfo r = info_of(p, nullptr);
    const int64_t heads = static_cast<int64_t>(p.B) * p.Hk;
    return heads * p.rows * 16 + (dtype == kF16 ? (heads * (r.blocks + r.key_blocks) * 4 + 15) / 16 * 16 : 0);
}

}  // namespace

template <typename T>
int launch_attn_backward_t(int dtype, const AttnParams& given, hipStream_t stream) {
    AttnParams p = given;
    const BackShape s = back_shape(dtype, p, back_vec(dtype, p));
    const RowInfo info = info_of(p, static_cast<unsigned char*>(p.ws) + plan_mask(p, p.ws));
    float* const ws = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(info.rows) + info_bytes(dtype, p));
    int rc = launch_mask(dtype, p, stream);
    if (rc != 0) return rc;
    const int64_t blocks =
        static_cast<int64_t>(p.B) * p.Hk * (info.blocks + (kScaled<T> ? info.key_blocks : 0));
    const bool vec = p.D * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(p.go) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.out_low)) % 16 == 0;
    if (blocks > 0)
        hipLaunchKernelGGL((attn_info_kernel<T>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p, info, vec);
    switch (padded_width(p.D)) {
        case 32: rc = run_dp<T, 32>(p, s, info, ws, stream); break;
        case 64: rc = run_dp<T, 64>(p, s, info, ws, stream); break;
        case 96: rc = run_dp<T, 96>(p, s, info, ws, stream); break;
        case 128: rc = run_dp<T, 128>(p, s, info, ws, stream); break;
        default: rc = run_dp<T, 256>(p, s, info, ws, stream);
    }
    if (rc != 0) return rc;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : set_error(TD_E_LAUNCH, "attention backward launch failed: %s", hipGetErrorString(e));
}

#if TD_ATTN_TYPE == 0
extern template int launch_attn_backward_t<f16>(int, const AttnParams&, hipStream_t);
extern template int launch_attn_backward_t<bf16>(int, const AttnParams&, hipStream_t);
template int launch_attn_backward_t<float>(int, const AttnParams&, hipStream_t);

int64_t attn_backward_workspace(int dtype, const AttnParams& p) {
    if (dtype == kF64) return static_cast<int64_t>(p.B) * p.H * p.Q * 8;
    int64_t parts = 0;  // dQ's and then dK's and dV's
    for (const bool vec : {false, true}) {  // the gradients' alignment is not known yet
        const BackShape s = back_shape(dtype, p, vec);
        const int64_t q = s.q.part_floats(p.D), k = 2 * s.k.part_floats(p.D);
        parts = parts > q ? parts : q;
        parts = parts > k ? parts : k;
    }
    AttnParams q = p;
    return plan_mask(q, nullptr) + info_bytes(dtype, p) + parts * 4;
}

int launch_attn_backward(int dtype, const AttnParams& p, hipStream_t stream) {
    switch (dtype) {
        case kF32: return launch_attn_backward_t<float>(dtype, p, stream);
        case kF16: return launch_attn_backward_t<f16>(dtype, p, stream);
        default: return launch_attn_backward_t<bf16>(dtype, p, stream);
    }
}
#elif TD_ATTN_TYPE == 1
template int launch_attn_backward_t<f16>(int, const AttnParams&, hipStream_t);
#else
template int launch_attn_backward_t<bf16>(int, const AttnParams&, hipStream_t);
#endif

}  // namespace td
