// Attention among tokens (include/tinydeform_dense.h): the argument checks of its C entries, float64's kernels, one
// wavefront a row on the vector units, and masks as bits.
#include <math.h>

#include "td_attn.h"

namespace td {
namespace {

__device__ __forceinline__ const double* at(const void* base, const int64_t (&s)[3], int b, int tok, int h) {
    return static_cast<const double*>(base) + b * s[0] + static_cast<int64_t>(tok) * s[1] + h * s[2];
}

constexpr double kLog2eD = 1.4426950408889634, kLowestD = -1.7976931348623157e308;

template <typename A>
constexpr A neg_inf() {
    return -static_cast<A>(__builtin_inf());
}

// Whether (query i, key j) is left out by causal, padding or the mask, and the additive mask's term in base 2 (its lowest
// value kept finite, so that a row of it alone is a uniform row). A -inf of a float mask leaves the pair out whatever
// its score is.
__device__ __forceinline__ bool pair_masked(const AttnParams& p, int b, int h, int i, int j, double& add) {
    add = 0;
    if (p.causal && j > i + p.diag) return true;
    if (p.pad != nullptr && p.pad[static_cast<int64_t>(b) * p.K + j]) return true;
    if (p.mask_type == TD_MASK_NONE) return false;
    const int64_t m = b * p.ms[0] + h * p.ms[1] + i * p.ms[2] + j;
    if (p.mask_type == TD_MASK_BYTES) return static_cast<const uint8_t*>(p.mask)[m] != 0;
    add = static_cast<const double*>(p.mask)[m];
    if (add == neg_inf<double>()) return true;
    add *= kLog2eD;
    if (add < kLowestD) add = kLowestD;
    return false;
}

// scores are in base 2: c = scale * log2(e)
__device__ __forceinline__ double score_factor(const AttnParams& p) {
    return p.scale * kLog2eD;
}

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const double o = xor_lane(v, m);
        v = o > v ? o : v;
    }
    return v;
}

constexpr int kMaxPerLane = TD_ATTN_MAX_HEAD_DIM / kWave;  // head channels per lane

// One wavefront per (b, h, i): keys 64 at a time, one per lane for the scores, then lanes over the head's channels.
// The running maximum m and sum l (Milakov and Gimelshein's one-pass softmax) are kept in float64. Bound by the
// latency of its row loads: float64 is here for checks, not for speed.
__global__ __launch_bounds__(64) void attn_forward_row_kernel(AttnParams p) {
    __shared__ double sp[kWave];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;  // (b * H + h) * Q + i
    const int i = static_cast<int>(row % p.Q), h = static_cast<int>((row / p.Q) % p.H);
    const int b = static_cast<int>(row / p.Q / p.H), hk = h / p.G;
    const double* q = at(p.q, p.qs, b, i, h);
    double m = neg_inf<double>(), l = 0, acc[kMaxPerLane] = {};
    for (int j0 = 0; j0 < p.K; j0 += kWave) {
        const int j = j0 + lane;
        double t = neg_inf<double>(), add;
        if (j < p.K && !pair_masked(p, b, h, i, j, add)) {
            const double* k = at(p.k, p.ks, b, j, hk);
            double s = 0;
            for (int d = 0; d < p.D; ++d) s += q[d] * k[d];
            t = s * score_factor(p) + add;
        }
        const double m_new = wave_max(m > t ? m : t == t ? t : m);
        const double from = m_new == neg_inf<double>() ? 0 : m_new;
        const double shrink = exp2(m - from), e = exp2(t - from);
        m = m_new;
        l = l * shrink + wave_sum(e);
        __syncthreads();
        sp[lane] = e;
        __syncthreads();
        const int n = p.K - j0 < kWave ? p.K - j0 : kWave;
#pragma unroll
        for (int u = 0; u < kMaxPerLane; ++u) {
            const int d = u * kWave + lane;
            if (d >= p.D) break;
            double o = acc[u] * shrink;
            for (int x = 0; x < n; ++x)
                if (sp[x] != 0) o += sp[x] * at(p.v, p.vs, b, j0 + x, hk)[d];
            acc[u] = o;
        }
    }
    double* out = static_cast<double*>(p.out) + ((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D;
#pragma unroll
    for (int u = 0; u < kMaxPerLane; ++u) {
        const int d = u * kWave + lane;
        if (d < p.D) out[d] = l == 0 ? 0 : acc[u] / l;
    }
    if (p.stats != nullptr && lane == 0) {
        double* st = static_cast<double*>(p.stats) + 2 * row;
        st[0] = l == 0 ? 0 : m;
        st[1] = l == 0 ? 0 : log2(l);
    }
}

// delta[row] = grad_out . out of each (b, h, i), one wavefront each
__global__ __launch_bounds__(64) void attn_delta_row_kernel(AttnParams p) {
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int i = static_cast<int>(row % p.Q), h = static_cast<int>((row / p.Q) % p.H);
    const int64_t at0 = (((row / p.Q / p.H) * p.Q + i) * p.H + h) * p.D;
    double s = 0;
    for (int d = lane; d < p.D; d += kWave)
        s += static_cast<const double*>(p.go)[at0 + d] * static_cast<const double*>(p.out)[at0 + d];
    s = wave_sum(s);
    if (lane == 0) static_cast<double*>(p.delta)[row] = s;
}

// The probability of a pair and the gradient of its score: P = 2^(t - m - log2 l), dS = P (grad_out . v - delta)
__device__ __forceinline__ void pair_grad(const AttnParams& p, int b, int h, int i, int j, double& prob, double& ds) {
    double add;
    prob = ds = 0;
    if (pair_masked(p, b, h, i, j, add)) return;
    const double* q = at(p.q, p.qs, b, i, h);
    const double* k = at(p.k, p.ks, b, j, h / p.G);
    const double* v = at(p.v, p.vs, b, j, h / p.G);
    const double* g = static_cast<const double*>(p.go) + ((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D;
    const int64_t row = (static_cast<int64_t>(b) * p.H + h) * p.Q + i;
    const double* st = static_cast<const double*>(p.stats) + 2 * row;
    double s = 0, dp = 0;
    for (int d = 0; d < p.D; ++d) {
        s += q[d] * k[d];
        dp += g[d] * v[d];
    }
    prob = exp2(s * score_factor(p) + add - st[0] - st[1]);
    ds = prob * (dp - static_cast<const double*>(p.delta)[row]);
}

__global__ __launch_bounds__(64) void attn_dq_row_kernel(AttnParams p) {
    __shared__ double sd[kWave];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int i = static_cast<int>(row % p.Q), h = static_cast<int>((row / p.Q) % p.H);
    const int b = static_cast<int>(row / p.Q / p.H), hk = h / p.G;
    double acc[kMaxPerLane] = {};
    for (int j0 = 0; j0 < p.K; j0 += kWave) {
        double prob = 0, ds = 0;
        if (j0 + lane < p.K) pair_grad(p, b, h, i, j0 + lane, prob, ds);
        __syncthreads();
        sd[lane] = ds;
        __syncthreads();
        const int n = p.K - j0 < kWave ? p.K - j0 : kWave;
#pragma unroll
        for (int u = 0; u < kMaxPerLane; ++u) {
            const int d = u * kWave + lane;
            if (d >= p.D) break;
            for (int x = 0; x < n; ++x)
                if (sd[x] != 0) acc[u] += sd[x] * at(p.k, p.ks, b, j0 + x, hk)[d];
        }
    }
    double* dq = static_cast<double*>(p.dq) + ((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D;
#pragma unroll
    for (int u = 0; u < kMaxPerLane; ++u)
        if (u * kWave + lane < p.D) dq[u * kWave + lane] = acc[u] * p.scale;
}

// One wavefront per (b, key head, j): the rows of every head that shares the key, 64 at a time
__global__ __launch_bounds__(64) void attn_dkv_row_kernel(AttnParams p) {
    __shared__ double sp[kWave], sd[kWave];
    const int lane = threadIdx.x;
    const int64_t id = blockIdx.x;  // (b * Hk + hk) * K + j
    const int j = static_cast<int>(id % p.K), hk = static_cast<int>((id / p.K) % p.Hk);
    const int b = static_cast<int>(id / p.K / p.Hk);
    double dk[kMaxPerLane] = {}, dv[kMaxPerLane] = {};
    for (int r0 = 0; r0 < p.rows; r0 += kWave) {
        double prob = 0, ds = 0;
        const int r = r0 + lane;
        if (r < p.rows) pair_grad(p, b, hk * p.G + r % p.G, r / p.G, j, prob, ds);
        __syncthreads();
        sp[lane] = prob;
        sd[lane] = ds;
        __syncthreads();
        const int n = p.rows - r0 < kWave ? p.rows - r0 : kWave;
#pragma unroll
        for (int u = 0; u < kMaxPerLane; ++u) {
            const int d = u * kWave + lane;
            if (d >= p.D) break;
            for (int x = 0; x < n; ++x) {
                const int i = (r0 + x) / p.G, h = hk * p.G + (r0 + x) % p.G;
                if (sp[x] != 0)
                    dv[u] += sp[x] * static_cast<const double*>(
                                         p.go)[((static_cast<int64_t>(b) * p.Q + i) * p.H + h) * p.D + d];
                if (sd[x] != 0) dk[u] += sd[x] * at(p.q, p.qs, b, i, h)[d];
            }
        }
    }
    const int64_t o = ((static_cast<int64_t>(b) * p.K + j) * p.Hk + hk) * p.D;
#pragma unroll
    for (int u = 0; u < kMaxPerLane; ++u) {
        const int d = u * kWave + lane;
        if (d >= p.D) break;
        static_cast<double*>(p.dk)[o + d] = dk[u] * p.scale;
        static_cast<double*>(p.dv)[o + d] = dv[u];
    }
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : set_error(TD_E_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace

int launch_attn_forward_f64(const AttnParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(attn_forward_row_kernel, dim3(static_cast<unsigned>(p.B) * p.H * p.Q), dim3(64), 0, stream, p);
    return launched("attention");
}

int launch_attn_backward_f64(const AttnParams& p, hipStream_t stream) {
    const unsigned rows = static_cast<unsigned>(p.B) * p.H * p.Q, keys = static_cast<unsigned>(p.B) * p.Hk * p.K;
    if (rows > 0) hipLaunchKernelGGL(attn_delta_row_kernel, dim3(rows), dim3(64), 0, stream, p);
    if (rows > 0 && p.dq != nullptr) hipLaunchKernelGGL(attn_dq_row_kernel, dim3(rows), dim3(64), 0, stream, p);
    if (keys > 0 && p.dk != nullptr) hipLaunchKernelGGL(attn_dkv_row_kernel, dim3(keys), dim3(64), 0, stream, p);
    return launched("attention backward");
}

namespace {

// The mask as bits, a wavefront for 32 rows by two words of 32 keys: each mask entry is read once here instead of once by
// every head that shares it, and a tile that the mask leaves as it is, or leaves nothing of, costs its readers nothing.
template <typename T>
__global__ __launch_bounds__(256) void attn_mask_kernel(AttnParams p, int64_t tiles, int tile_rows, int mask_rows,
                                                        int mask_heads) {
    const int lane = threadIdx.x % kWave, half = lane >> 5, pairs = (p.words + 1) / 2;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (id >= tiles * pairs) return;
    const int word = static_cast<int>(id % pairs) * 2 + half, j0 = word * 32;
    const int64_t tile = id / pairs, at = tile / tile_rows;  // at: batch and head of the mask
    const int row = static_cast<int>(tile % tile_rows) * 32 + (lane & 31);
    const int64_t b = at / mask_heads, h = at % mask_heads;
    uint32_t bits = ~0u;
    bool values = false;
    const bool in = row < mask_rows && word < p.words;
    if (in) {
        const int64_t m0 = b * p.ms[0] + h * p.ms[1] + row * p.ms[2] + j0;
        const int left = p.K - j0;
        if (p.mask_type == TD_MASK_BYTES) {
            const uint8_t* m = static_cast<const uint8_t*>(p.mask) + m0;
            if (left >= 32) {
                uint32_t v[8];
                __builtin_memcpy(v, m, 32);
                bits = 0;
#pragma unroll
                for (int k = 0; k < 32; ++k) bits |= ((v[k / 4] >> (8 * (k % 4))) & 0xffu ? 1u : 0u) << k;
            } else {
                for (int k = 0; k < left; ++k)
                    if (m[k] == 0) bits &= ~(1u << k);
            }
        } else {
            const T* m = static_cast<const T*>(p.mask) + m0;
            auto see = [&](T entry, int k) {
                const float v = static_cast<float>(entry);
                if (v != neg_inf<float>()) bits &= ~(1u << k);
                values |= v != 0.f && v != neg_inf<float>();
            };
            if (left >= 32) {
                T v[32];
                __builtin_memcpy(v, m, sizeof(v));
#pragma unroll
                for (int k = 0; k < 32; ++k) see(v[k], k);
            } else {
                for (int k = 0; k < left; ++k) see(m[k], k);
            }
        }
        p.bits[(at * mask_rows + row) * p.words + word] = bits;
    }
    // keys past the end are set in the bits; rows past the end say nothing
    const uint32_t past = p.K - j0 >= 32 || word >= p.words ? 0u : ~0u << (p.K - j0);
    const uint64_t mine = half ? ~uint64_t{0} << 32 : ~uint64_t{0} >> 32;
    const uint64_t any_values = __ballot(in && values) & mine, any_bits = __ballot(in && (bits & ~past)) & mine;
    const uint64_t any_left = __ballot(in && bits != ~0u) & mine;
    if ((lane & 31) == 0 && word < p.words)
        p.kinds[tile * p.words + word] = static_cast<uint8_t>(any_left == 0     ? kMaskAll
                                                              : any_values != 0 ? kMaskValues
                                                              : any_bits != 0 || past != 0 ? kMaskBits
                                                                                           : kMaskNone);
}

struct MaskShape {
    int batches, heads, rows, tile_rows;
};
MaskShape mask_shape(const AttnParams& p) {
    MaskShape m{p.ms[0] == 0 ? 1 : p.B, p.ms[1] == 0 ? 1 : p.H, p.ms[2] == 0 ? 1 : p.Q, 0};
    m.tile_rows = (m.rows + 31) / 32;
    return m;
}

}  // namespace

int64_t plan_mask(AttnParams& p, void* at) {
    if (p.mask_type == TD_MASK_NONE || p.K == 0 || p.Q == 0) return 0;
    const MaskShape m = mask_shape(p);
    p.words = (p.K + 31) / 32;
    const int64_t heads = static_cast<int64_t>(m.batches) * m.heads;
    const int64_t bits = (heads * m.rows * p.words * 4 + 15) / 16 * 16;
    const int64_t kinds = (heads * m.tile_rows * p.words + 15) / 16 * 16;
    p.bits = static_cast<uint32_t*>(at);
    p.kinds = static_cast<uint8_t*>(at) + bits;
    const int64_t per_batch = m.heads;
    p.bs[0] = m.batches == 1 ? 0 : per_batch * m.rows;
    p.bs[1] = m.heads == 1 ? 0 : m.rows;
    p.bs[2] = m.rows == 1 ? 0 : 1;
    p.kinds_bs[0] = m.batches == 1 ? 0 : per_batch * m.tile_rows;
    p.kinds_bs[1] = m.heads == 1 ? 0 : m.tile_rows;
    return bits + kinds;
}

int launch_mask(int dtype, const AttnParams& p, hipStream_t stream) {
    if (p.words == 0) return 0;
    const MaskShape m = mask_shape(p);
    const int64_t tiles = static_cast<int64_t>(m.batches) * m.heads * m.tile_rows;
    const int64_t groups = (tiles * ((p.words + 1) / 2) + 3) / 4;
    if (groups > 16777215) return set_error(TD_E_ARG, "attention: the mask has too many entries");
    const dim3 grid(static_cast<unsigned>(groups));
    if (dtype == kF32)
        hipLaunchKernelGGL((attn_mask_kernel<float>), grid, dim3(256), 0, stream, p, tiles, m.tile_rows, m.rows, m.heads);
    else if (dtype == kF16)
        hipLaunchKernelGGL((attn_mask_kernel<f16>), grid, dim3(256), 0, stream, p, tiles, m.tile_rows, m.rows, m.heads);
    else
        hipLaunchKernelGGL((attn_mask_kernel<bf16>), grid, dim3(256), 0, stream, p, tiles, m.tile_rows, m.rows, m.heads);
    return launched("attention mask");
}

AttnParams attn_params(const td_attn_args& a) {
    AttnParams p{};
    p.q = a.query;
    p.k = a.key;
    p.v = a.value;
    p.mask = a.mask;
    p.pad = a.key_padding;
    p.out = a.out;
    p.stats = a.stats;
    p.out_low = a.dtype == TD_F16 || a.dtype == TD_BF16 ? a.out_low : nullptr;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a.query_stride[i];
        p.ks[i] = a.key_stride[i];
        p.vs[i] = a.value_stride[i];
        p.ms[i] = a.mask_stride[i];
    }
    p.B = static_cast<int>(a.B);
    p.Q = static_cast<int>(a.Q);
    p.K = static_cast<int>(a.K);
    p.H = static_cast<int>(a.H);
    p.Hk = static_cast<int>(a.Hk);
    p.D = static_cast<int>(a.D);
    p.G = p.H / p.Hk;
    p.rows = p.Q * p.G;
    p.gdiv = make_fastdiv(static_cast<uint32_t>(p.G));
    p.mask_type = a.mask_type;
    p.causal = a.causal != 0;
    p.diag = a.K - a.Q;
    p.scale = a.scale;
    p.c = static_cast<float>(a.scale * 1.4426950408889634);
    return p;
}

namespace {

constexpr int64_t kIntMax = 2147483647;
constexpr int64_t kMaxRows = kIntMax - 1023;  // the numbers of a last tile's rows are 32-bit too

int check_args(const td_attn_args* a) {
    set_error(TD_OK, "");
    if (a == nullptr) return set_error(TD_E_ARG, "null pointer argument");
    if (a->dtype < TD_F32 || a->dtype > TD_F64) return set_error(TD_E_DTYPE, "unknown dtype code %d", a->dtype);
    if (a->B < 0 || a->Q < 0 || a->K < 0) return set_error(TD_E_ARG, "sizes must be non-negative");
    if (a->H <= 0 || a->Hk <= 0) return set_error(TD_E_ARG, "need at least one head");
    if (a->H > kIntMax || a->H % a->Hk != 0)
        return set_error(TD_E_ARG, "the heads of key and value must divide the heads of query");
    if (a->D < 1 || a->D > TD_ATTN_MAX_HEAD_DIM)
        return set_error(TD_E_ARG, "head dim must be from 1 to %d", TD_ATTN_MAX_HEAD_DIM);
    if (a->B > kIntMax || a->Q > kMaxRows || a->K > kMaxRows ||
        static_cast<__int128>(a->B) * a->Q * a->H > kMaxRows || static_cast<__int128>(a->B) * a->K * a->Hk > kMaxRows)
        return set_error(TD_E_ARG, "too many (batch, token, head) rows");
    for (int i = 0; i < 3; ++i)
        if (a->query_stride[i] < 0 || a->key_stride[i] < 0 || a->value_stride[i] < 0 || a->mask_stride[i] < 0)
            return set_error(TD_E_ARG, "strides must be non-negative");
    if (!(a->scale > 0) || !isfinite(a->scale)) return set_error(TD_E_ARG, "scale must be positive and finite");
    if (a->mask_type < TD_MASK_NONE || a->mask_type > TD_MASK_FLOAT)
        return set_error(TD_E_ARG, "unknown mask type %d", a->mask_type);
    return TD_OK;
}

bool has_queries(const td_attn_args* a) { return a->B * a->Q > 0; }
bool has_keys(const td_attn_args* a) { return a->B * a->K > 0; }

int check_pointers(const td_attn_args* a) {
    if (has_queries(a) && (a->query == nullptr || a->out == nullptr))
        return set_error(TD_E_ARG, "null pointer argument");
    if (has_keys(a) && (a->key == nullptr || a->value == nullptr)) return set_error(TD_E_ARG, "null pointer argument");
    if (has_queries(a) && has_keys(a) && a->mask_type != TD_MASK_NONE && a->mask == nullptr)
        return set_error(TD_E_ARG, "null pointer argument");
    return TD_OK;
}

}  // namespace
}  // namespace td

using namespace td;

extern "C" int64_t td_attn_forward_workspace(const td_attn_args* args) {
    const int rc = check_args(args);
    return rc != TD_OK ? rc : args->B * args->Q == 0 ? 0 : attn_forward_workspace(args->dtype, attn_params(*args));
}

extern "C" int td_attn_forward(const td_attn_args* args, void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_args(args);
    if (rc == TD_OK) rc = check_pointers(args);
    if (rc != TD_OK) return rc;
    if (!has_queries(args)) return TD_OK;
    AttnParams p = attn_params(*args);
    const int64_t need = attn_forward_workspace(args->dtype, p);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr))
        return set_error(TD_E_WORKSPACE, "attention: the workspace has %lld bytes, %lld are needed",
                         static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    p.ws = workspace;
    if (args->dtype == TD_F64) return launch_attn_forward_f64(p, static_cast<hipStream_t>(stream));
    return launch_attn_forward(args->dtype, p, static_cast<hipStream_t>(stream));
}

extern "C" int64_t td_attn_backward_workspace(const td_attn_args* args) {
    const int rc = check_args(args);
    return rc != TD_OK ? rc : attn_backward_workspace(args->dtype, attn_params(*args));
}

extern "C" int td_attn_backward(const td_attn_args* args, const void* grad_out, void* grad_query, void* grad_key,
                                void* grad_value, void* workspace, int64_t workspace_bytes, void* stream) {
    const int64_t need = td_attn_backward_workspace(args);
    if (need < 0) return static_cast<int>(need);
    const int rc = check_pointers(args);
    if (rc != TD_OK) return rc;
    if ((has_queries(args) && (grad_out == nullptr || args->stats == nullptr)) ||
        (grad_key == nullptr) != (grad_value == nullptr))
        return set_error(TD_E_ARG, "null pointer argument");
    if (workspace_bytes < need || (need > 0 && workspace == nullptr))
        return set_error(TD_E_WORKSPACE, "attention backward: the workspace has %lld bytes, %lld are needed",
                         static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    if (!has_queries(args) && !has_keys(args)) return TD_OK;
    AttnParams p = attn_params(*args);
    p.go = grad_out;
    p.dq = grad_query;
    p.dk = grad_key;
    p.dv = grad_value;
    p.ws = p.delta = workspace;
    if (args->dtype == TD_F64) return launch_attn_backward_f64(p, static_cast<hipStream_t>(stream));
    return launch_attn_backward(args->dtype, p, static_cast<hipStream_t>(stream));
}
