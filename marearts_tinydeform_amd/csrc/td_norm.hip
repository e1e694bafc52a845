// Layer norm with a residual, forward and backward (include/tinydeform_dense.h).
#include <math.h>

#include "../../include/tinydeform_dense.h"
#include "td_internal.h"

namespace td {
namespace {

// A row is held in the registers of a team of LANES threads, NV pieces of V elements each (piece u of lane l: elements
// (u * LANES + l) * V ..), so that x and the residual are read once and the mean, the deviations' square sum and the
// output come from registers. Bound by memory: the kernels stream (67200 x 256 with a residual, bfloat16: 17.6 us, 5.9
// TB/s; 44446 x 256, float32: forward 22.5 us, 6.1, backward 28.9, 6.3; 43520 x 1024, bfloat16: 31.0, 5.7, and 45.2, 5.9; a
// copy of such sizes reaches 5.4 to 7.8). V: 16 bytes where the row and every pointer allow, else one element.
template <typename T, int V>
struct Piece {
    typedef T type __attribute__((ext_vector_type(V)));
};

// Sums over a team, every lane receiving the total. Within 16 lanes by data-parallel moves (quads, then mirrored halves),
// then by swapping rows of 16 and halves of 32; 256 lanes by way of LDS.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
    v += dpp_move<0xb1>(v);   // quad_perm 1, 0, 3, 2
    v += dpp_move<0x4e>(v);   // quad_perm 2, 3, 0, 1
    v += dpp_move<0x141>(v);  // row_half_mirror
    v += dpp_move<0x140>(v);  // row_mirror
    const auto swapped = [](unsigned a, auto f) {
        const auto r = f(a);
        const unsigned low = r[0], high = r[1];
        return __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
    };
    if constexpr (LANES >= 32)
        v = swapped(__builtin_bit_cast(unsigned, v),
                    [](unsigned a) { return __builtin_amdgcn_permlane16_swap(a, a, false, false); });
    if constexpr (LANES >= 64)
        v = swapped(__builtin_bit_cast(unsigned, v),
                    [](unsigned a) { return __builtin_amdgcn_permlane32_swap(a, a, false, false); });
    return v;
}
template <int LANES>
__device__ __forceinline__ double lane_sum(double v) {
#pragma unroll
    for (int m = 1; m < (LANES < kWave ? LANES : kWave); m <<= 1) v += xor_lane(v, m);
    return v;
}
// N sums together; `lds` [4 * N] of the workgroup, for teams of 256
template <int LANES, int N, typename A>
__device__ __forceinline__ void team_sum(A (&v)[N], A* lds) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = lane_sum<LANES>(v[n]);
    if constexpr (LANES > kWave) {
        const int wave = threadIdx.x / kWave;
        __syncthreads();  // the previous sums have been read
        if (threadIdx.x % kWave == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) lds[wave * N + n] = v[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = (lds[n] + lds[N + n]) + (lds[2 * N + n] + lds[3 * N + n]);
    }
}

template <typename T, int V, int LANES, int NV>
struct RowLoad {
    using P = typename Piece<T, V>::type;
    P p[NV];
    __device__ __forceinline__ void load(const T* row, int C, int lane) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int at = (u * LANES + lane) * V;
            p[u] = P{};
            if (at < C) p[u] = *reinterpret_cast<const P*>(row + at);
        }
    }
    template <typename A>
    __device__ __forceinline__ A get(int u, int e) const {
        return static_cast<A>(p[u][e]);
    }
};

constexpr int kNormThreads = 256;

template <typename T, typename A, int V, int LANES, int NV>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                            const T* __restrict__ w, const T* __restrict__ b,
                                                            T* __restrict__ out, A* __restrict__ stats, int64_t rows,
                                                            int C, A eps) {
    constexpr int kTeams = kNormThreads / LANES;
    __shared__ A lds[8];
    const int lane = threadIdx.x % LANES;
    RowLoad<T, V, LANES, NV> rx, rr, rw, rb;
    if (w != nullptr) rw.load(w, C, lane);
    if (b != nullptr) rb.load(b, C, lane);
    const A inv = static_cast<A>(1) / C;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / LANES; row < rows;
         row += static_cast<int64_t>(gridDim.x) * kTeams) {
        rx.load(x + row * C, C, lane);
        if (res != nullptr) rr.load(res + row * C, C, lane);
        A h[NV][V], sum[1] = {0};
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[u][e] = rx.template get<A>(u, e);
                if (res != nullptr) h[u][e] += rr.template get<A>(u, e);
                sum[0] += h[u][e];
            }
        team_sum<LANES>(sum, lds);
        const A mean = sum[0] * inv;
        sum[0] = 0;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const bool in = (u * LANES + lane) * V < C;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[u][e] -= mean;
                if (in) sum[0] += h[u][e] * h[u][e];
            }
        }
        team_sum<LANES>(sum, lds);
        const A rstd = static_cast<A>(1) / sqrt(sum[0] * inv + eps);
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int at = (u * LANES + lane) * V;
            typename Piece<T, V>::type o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                A v = h[u][e] * rstd;
                if (w != nullptr) v *= rw.template get<A>(u, e);
                if (b != nullptr) v += rb.template get<A>(u, e);
                o[e] = static_cast<T>(v);
            }
            if (at < C) *reinterpret_cast<typename Piece<T, V>::type*>(out + row * C + at) = o;
        }
        if (stats != nullptr && lane == 0) {
            stats[2 * row] = mean;
            stats[2 * row + 1] = rstd;
        }
    }
}

// dx = rstd (w g - mean(w g) - xhat mean(w g xhat)) and, in registers over the team's rows, the column sums of g xhat and
// g. The teams of a workgroup are added in LDS and each workgroup writes one partial sum [2][C]; norm_sum_kernel adds
// those (4 to 5 us). The order depends on the sizes only.
template <typename T, typename A, int V, int LANES, int NV>
__global__ __launch_bounds__(kNormThreads) void norm_backward_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                                     const T* __restrict__ w,
                                                                     const A* __restrict__ stats,
                                                                     const T* __restrict__ g, T* __restrict__ dx,
                                                                     A* __restrict__ partial, int64_t rows, int C) {
    constexpr int kTeams = kNormThreads / LANES, kCols = LANES * NV * V;
    __shared__ A lds[8];
    __shared__ __align__(16) A cols[kTeams > 1 ? kTeams * kCols : 1];
    const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
    RowLoad<T, V, LANES, NV> rx, rr, rg, rw;
    if (w != nullptr) rw.load(w, C, lane);
    const A inv = static_cast<A>(1) / C;
    A dw[NV][V] = {}, db[NV][V] = {};
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + team; row < rows;
         row += static_cast<int64_t>(gridDim.x) * kTeams) {
        rx.load(x + row * C, C, lane);
        rg.load(g + row * C, C, lane);
        if (res != nullptr) rr.load(res + row * C, C, lane);
        const A mean = stats[2 * row], rstd = stats[2 * row + 1];
        A xh[NV][V], sum[2] = {0, 0};
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                A h = rx.template get<A>(u, e);
                if (res != nullptr) h += rr.template get<A>(u, e);
                xh[u][e] = (h - mean) * rstd;
                const A gv = rg.template get<A>(u, e);  // 0 past the row's end
                const A wg = w == nullptr ? gv : gv * rw.template get<A>(u, e);
                sum[0] += wg;
                sum[1] += wg * xh[u][e];
                dw[u][e] += gv * xh[u][e];
                db[u][e] += gv;
            }
        team_sum<LANES>(sum, lds);
        const A m1 = sum[0] * inv, m2 = sum[1] * inv;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int at = (u * LANES + lane) * V;
            typename Piece<T, V>::type o;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const A gv = rg.template get<A>(u, e);
                const A wg = w == nullptr ? gv : gv * rw.template get<A>(u, e);
                o[e] = static_cast<T>(rstd * (wg - m1 - xh[u][e] * m2));
            }
            if (at < C) *reinterpret_cast<typename Piece<T, V>::type*>(dx + row * C + at) = o;
        }
    }
    if (partial == nullptr) return;
    A* const to = partial + static_cast<int64_t>(blockIdx.x) * 2 * C;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (kTeams > 1) {
            __syncthreads();
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    cols[team * kCols + (u * LANES + lane) * V + e] = which ? db[u][e] : dw[u][e];
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += kNormThreads) {
                A s = 0;
#pragma unroll
                for (int k = 0; k < kTeams; ++k) s += cols[k * kCols + c];
                to[which * C + c] = s;
            }
        } else {
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int at = (u * LANES + lane) * V + e;
                    if (at < C) to[which * C + at] = which ? db[u][e] : dw[u][e];
                }
        }
    }
}

// Workgroups of the backward kernel: enough for every CU to hold four, fewer where the partial sums get wide
int64_t partials(int64_t rows, int64_t C) {
    const int64_t most = C <= 1024 ? 1024 : C >= 4096 ? 256 : (int64_t{1} << 20) / C;
    const int64_t n = (rows + 7) / 8;
    return n < most ? n : most;
}

// Sums of the n partial sums of each of 2 C columns: 16 columns a workgroup, 64 threads a column, eight loads in flight
template <typename T, typename A>
__global__ __launch_bounds__(1024) void norm_sum_kernel(const A* __restrict__ partial, int64_t n, T* dw, T* db, int C) {
    __shared__ A lds[1024];
    const int col = threadIdx.x % 16, k = threadIdx.x / 16;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 16 + col, width = 2 * static_cast<int64_t>(C);
    A s = 0;
    if (c < width) {
#pragma unroll 8
        for (int64_t i = k; i < n; i += 64) s += partial[i * width + c];
    }
    lds[threadIdx.x] = s;
    __syncthreads();
    if (k < 8) {  // thread k adds the sums 8 k .. 8 k + 7 into the place of the first
        s = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += lds[(8 * k + i) * 16 + col];
        lds[8 * k * 16 + col] = s;
    }
    __syncthreads();
    if (k != 0 || c >= width) return;
    s = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += lds[i * 128 + col];
    if (c < C) {
        if (dw != nullptr) dw[c] = static_cast<T>(s);
    } else if (db != nullptr) {
        db[c - C] = static_cast<T>(s);
    }
}

struct NormArgs {
    const void *x, *res, *w, *b, *go;
    void *out, *stats, *dx, *dw, *db, *ws;
    int64_t rows;
    int C;
    double eps;
};

template <typename T, typename A, int V, int LANES, int NV>
void launch(const NormArgs& n, bool back, hipStream_t stream) {
    const T *x = static_cast<const T*>(n.x), *res = static_cast<const T*>(n.res), *w = static_cast<const T*>(n.w);
    constexpr int kTeams = kNormThreads / LANES;
    if (back) {
        A* const partial = n.dw != nullptr || n.db != nullptr ? static_cast<A*>(n.ws) : nullptr;
        hipLaunchKernelGGL((norm_backward_kernel<T, A, V, LANES, NV>),
                           dim3(static_cast<unsigned>(partials(n.rows, n.C))), dim3(kNormThreads), 0, stream, x, res, w,
                           static_cast<const A*>(n.stats), static_cast<const T*>(n.go), static_cast<T*>(n.dx), partial,
                           n.rows, n.C);
    } else {
        const int64_t need = (n.rows + kTeams - 1) / kTeams;
        hipLaunchKernelGGL((norm_kernel<T, A, V, LANES, NV>), dim3(static_cast<unsigned>(need < 2048 ? need : 2048)),
                           dim3(kNormThreads), 0, stream, x, res, w, static_cast<const T*>(n.b),
                           static_cast<T*>(n.out), static_cast<A*>(n.stats), n.rows, n.C, static_cast<A>(n.eps));
    }
}

// The smallest team that holds a row
template <typename T, typename A, int V>
void launch_v(const NormArgs& n, bool back, hipStream_t stream) {
    const int pieces = (n.C + V - 1) / V;
    if (pieces <= 16) return launch<T, A, V, 16, 1>(n, back, stream);
    if (pieces <= 32) return launch<T, A, V, 32, 1>(n, back, stream);
    if (pieces <= 64) return launch<T, A, V, 64, 1>(n, back, stream);
    if (pieces <= 128) return launch<T, A, V, 64, 2>(n, back, stream);
    if (pieces <= 256) return launch<T, A, V, 64, 4>(n, back, stream);
    if (pieces <= 512) return launch<T, A, V, 256, 2>(n, back, stream);
    if (pieces <= 1024) return launch<T, A, V, 256, 4>(n, back, stream);
    if (pieces <= 2048) return launch<T, A, V, 256, 8>(n, back, stream);
    if constexpr (V < 8) {
        if (pieces <= 4096) return launch<T, A, V, 256, 16>(n, back, stream);
        if constexpr (V < 4) {
            if (pieces <= 8192) return launch<T, A, V, 256, 32>(n, back, stream);
            if constexpr (V < 2) launch<T, A, V, 256, 64>(n, back, stream);
        }
    }
}

template <typename T, typename A>
int run(const NormArgs& n, bool back, hipStream_t stream) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    uintptr_t bits = 0;
    for (const void* ptr : {n.x, n.res, n.w, n.b, n.go, static_cast<const void*>(n.out), static_cast<const void*>(n.dx)})
        bits |= reinterpret_cast<uintptr_t>(ptr);
    if (n.rows > 0) {
        if (n.C % V == 0 && bits % 16 == 0)
            launch_v<T, A, V>(n, back, stream);
        else
            launch_v<T, A, 1>(n, back, stream);
    }
    if (back && (n.dw != nullptr || n.db != nullptr))
        hipLaunchKernelGGL((norm_sum_kernel<T, A>), dim3((2 * n.C + 15) / 16), dim3(1024), 0, stream,
                           static_cast<const A*>(n.ws), partials(n.rows, n.C), static_cast<T*>(n.dw),
                           static_cast<T*>(n.db), n.C);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : set_error(TD_E_LAUNCH, "layer norm launch failed: %s", hipGetErrorString(e));
}

int run_type(int dtype, const NormArgs& n, bool back, hipStream_t stream) {
    switch (dtype) {
        case TD_F32: return run<float, float>(n, back, stream);
        case TD_F16: return run<f16, float>(n, back, stream);
        case TD_BF16: return run<bf16, float>(n, back, stream);
        default: return run<double, double>(n, back, stream);
    }
}

int check(int dtype, int64_t rows, int64_t C) {
    set_error(TD_OK, "");
    if (dtype < TD_F32 || dtype > TD_F64) return set_error(TD_E_DTYPE, "unknown dtype code %d", dtype);
    if (rows < 0 || C < 0) return set_error(TD_E_ARG, "sizes must be non-negative");
    if (rows > 2147483647) return set_error(TD_E_ARG, "too many rows");
    if (C < 1 || C > TD_NORM_MAX_CHANNELS)
        return set_error(TD_E_ARG, "channels must be from 1 to %d", TD_NORM_MAX_CHANNELS);
    return TD_OK;
}

}  // namespace
}  // namespace td

using namespace td;

extern "C" int td_layer_norm_forward(int dtype, const void* x, const void* residual, const void* weight,
                                     const void* bias, void* out, void* stats, int64_t rows, int64_t C, double eps,
                                     void* stream) {
    const int rc = check(dtype, rows, C);
    if (rc != TD_OK) return rc;
    if (!(eps >= 0) || !isfinite(eps)) return set_error(TD_E_ARG, "eps must be non-negative and finite");
    if (rows == 0) return TD_OK;
    if (x == nullptr || out == nullptr) return set_error(TD_E_ARG, "null pointer argument");
    NormArgs n{};
    n.x = x;
    n.res = residual;
    n.w = weight;
    n.b = bias;
    n.out = out;
    n.stats = stats;
    n.rows = rows;
    n.C = static_cast<int>(C);
    n.eps = eps;
    return run_type(dtype, n, false, static_cast<hipStream_t>(stream));
}

extern "C" int64_t td_layer_norm_backward_workspace(int dtype, int64_t rows, int64_t C) {
    const int rc = check(dtype, rows, C);
    return rc != TD_OK ? rc : partials(rows, C) * 2 * C * (dtype == TD_F64 ? 8 : 4);
}

extern "C" int td_layer_norm_backward(int dtype, const void* x, const void* residual, const void* weight,
                                      const void* stats, const void* grad_out, void* grad_x, void* grad_weight,
                                      void* grad_bias, int64_t rows, int64_t C, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    const int64_t need = td_layer_norm_backward_workspace(dtype, rows, C);
    if (need < 0) return static_cast<int>(need);
    if (rows > 0 && (x == nullptr || stats == nullptr || grad_out == nullptr || grad_x == nullptr))
        return set_error(TD_E_ARG, "null pointer argument");
    if ((grad_weight != nullptr || grad_bias != nullptr) &&
        (workspace_bytes < need || (need > 0 && workspace == nullptr)))
        return set_error(TD_E_WORKSPACE, "layer norm backward: the workspace has %lld bytes, %lld are needed",
                         static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    NormArgs n{};
    n.x = x;
    n.res = residual;
    n.w = weight;
    n.stats = const_cast<void*>(stats);
    n.go = grad_out;
    n.dx = grad_x;
    n.dw = grad_weight;
    n.db = grad_bias;
    n.ws = workspace;
    n.rows = rows;
    n.C = static_cast<int>(C);
    return run_type(dtype, n, true, static_cast<hipStream_t>(stream));
}
