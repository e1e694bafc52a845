// Layer norm with a residual, forward and backward (include/tinydeform_dense.h).
#include <math.h>

#include "../../include/tinydeform_dense.h"
#include "td_internal.h"

namespace td {
namespace {

template <typename T, typename A>
__device__ __forceinline__ A load_sum(const T* x, const T* r, int64_t i) {
    const A v = cvt<A>(x[i]);
    return r == nullptr ? v : v + cvt<A>(r[i]);
}

// One wavefront a row, three passes over it: the mean, the variance around it, the output.
template <typename T, typename A>
__global__ __launch_bounds__(64) void norm_row_kernel(const T* x, const T* res, const T* w, const T* b, T* out,
                                                      A* stats, int C, A eps) {
    const int64_t row = blockIdx.x, base = row * C;
    const int lane = threadIdx.x;
    A s = 0, v = 0;
    for (int i = lane; i < C; i += kWave) s += load_sum<T, A>(x, res, base + i);
    const A mean = wave_sum(s) / C;
    for (int i = lane; i < C; i += kWave) {
        const A d = load_sum<T, A>(x, res, base + i) - mean;
        v += d * d;
    }
    const A rstd = static_cast<A>(1) / sqrt(wave_sum(v) / C + eps);
    for (int i = lane; i < C; i += kWave) {
        A o = (load_sum<T, A>(x, res, base + i) - mean) * rstd;
        if (w != nullptr) o *= cvt<A>(w[i]);
        if (b != nullptr) o += cvt<A>(b[i]);
        out[base + i] = static_cast<T>(o);
    }
    if (stats != nullptr && lane == 0) {
        stats[2 * row] = mean;
        stats[2 * row + 1] = rstd;
    }
}

// dx = rstd (w g - mean(w g) - xhat mean(w g xhat)), one wavefront a row
template <typename T, typename A>
__global__ __launch_bounds__(64) void norm_dx_row_kernel(const T* x, const T* res, const T* w, const A* stats,
                                                         const T* g, T* dx, int C) {
    const int64_t row = blockIdx.x, base = row * C;
    const int lane = threadIdx.x;
    const A mean = stats[2 * row], rstd = stats[2 * row + 1];
    A s1 = 0, s2 = 0;
    for (int i = lane; i < C; i += kWave) {
        const A wg = cvt<A>(g[base + i]) * (w == nullptr ? static_cast<A>(1) : cvt<A>(w[i]));
        s1 += wg;
        s2 += wg * (load_sum<T, A>(x, res, base + i) - mean) * rstd;
    }
    s1 = wave_sum(s1) / C;
    s2 = wave_sum(s2) / C;
    for (int i = lane; i < C; i += kWave) {
        const A wg = cvt<A>(g[base + i]) * (w == nullptr ? static_cast<A>(1) : cvt<A>(w[i]));
        const A xh = (load_sum<T, A>(x, res, base + i) - mean) * rstd;
        dx[base + i] = static_cast<T>(rstd * (wg - s1 - xh * s2));
    }
}

constexpr int kRowBlock = 256;  // rows of one partial sum

// Partial column sums of g xhat and g over kRowBlock rows: partial[block][2][C]
template <typename T, typename A>
__global__ __launch_bounds__(64) void norm_dw_kernel(const T* x, const T* res, const A* stats, const T* g, A* partial,
                                                     int64_t rows, int C) {
    const int c = blockIdx.x * kWave + threadIdx.x;
    if (c >= C) return;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kRowBlock;
    const int64_t r1 = r0 + kRowBlock < rows ? r0 + kRowBlock : rows;
    A dw = 0, db = 0;
    for (int64_t r = r0; r < r1; ++r) {
        const A gv = cvt<A>(g[r * C + c]);
        dw += gv * (load_sum<T, A>(x, res, r * C + c) - stats[2 * r]) * stats[2 * r + 1];
        db += gv;
    }
    partial[(2 * static_cast<int64_t>(blockIdx.y)) * C + c] = dw;
    partial[(2 * static_cast<int64_t>(blockIdx.y) + 1) * C + c] = db;
}

template <typename T, typename A>
__global__ __launch_bounds__(64) void norm_dw_sum_kernel(const A* partial, int64_t blocks, T* dw, T* db, int C) {
    const int c = blockIdx.x * kWave + threadIdx.x;
    if (c >= C) return;
    A sw = 0, sb = 0;
    for (int64_t i = 0; i < blocks; ++i) {
        sw += partial[2 * i * C + c];
        sb += partial[(2 * i + 1) * C + c];
    }
    if (dw != nullptr) dw[c] = static_cast<T>(sw);
    if (db != nullptr) db[c] = static_cast<T>(sb);
}

struct NormArgs {
    const void *x, *res, *w, *b, *go;
    void *out, *stats, *dx, *dw, *db, *ws;
    int64_t rows;
    int C;
    double eps;
};

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : set_error(TD_E_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

template <typename T, typename A>
int forward(const NormArgs& n, hipStream_t stream) {
    hipLaunchKernelGGL((norm_row_kernel<T, A>), dim3(static_cast<unsigned>(n.rows)), dim3(64), 0, stream,
                       static_cast<const T*>(n.x), static_cast<const T*>(n.res), static_cast<const T*>(n.w),
                       static_cast<const T*>(n.b), static_cast<T*>(n.out), static_cast<A*>(n.stats), n.C,
                       static_cast<A>(n.eps));
    return launched("layer norm");
}

template <typename T, typename A>
int backward(const NormArgs& n, hipStream_t stream) {
    const T *x = static_cast<const T*>(n.x), *res = static_cast<const T*>(n.res), *g = static_cast<const T*>(n.go);
    const A* stats = static_cast<const A*>(n.stats);
    const int64_t blocks = (n.rows + kRowBlock - 1) / kRowBlock;
    const unsigned cols = static_cast<unsigned>((n.C + kWave - 1) / kWave);
    if (n.rows > 0)
        hipLaunchKernelGGL((norm_dx_row_kernel<T, A>), dim3(static_cast<unsigned>(n.rows)), dim3(64), 0, stream, x, res,
                           static_cast<const T*>(n.w), stats, g, static_cast<T*>(n.dx), n.C);
    if (n.dw != nullptr || n.db != nullptr) {
        A* partial = static_cast<A*>(n.ws);
        if (blocks > 0)
            hipLaunchKernelGGL((norm_dw_kernel<T, A>), dim3(cols, static_cast<unsigned>(blocks)), dim3(64), 0, stream, x,
                               res, stats, g, partial, n.rows, n.C);
        hipLaunchKernelGGL((norm_dw_sum_kernel<T, A>), dim3(cols), dim3(64), 0, stream, partial, blocks,
                           static_cast<T*>(n.dw), static_cast<T*>(n.db), n.C);
    }
    return launched("layer norm backward");
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case TD_F32: return forward<float, float>(n, s);
        case TD_F16: return forward<f16, float>(n, s);
        case TD_BF16: return forward<bf16, float>(n, s);
        default: return forward<double, double>(n, s);
    }
}

extern "C" int64_t td_layer_norm_backward_workspace(int dtype, int64_t rows, int64_t C) {
    const int rc = check(dtype, rows, C);
    return rc != TD_OK ? rc : (rows + kRowBlock - 1) / kRowBlock * 2 * C * (dtype == TD_F64 ? 8 : 4);
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case TD_F32: return backward<float, float>(n, s);
        case TD_F16: return backward<f16, float>(n, s);
        case TD_BF16: return backward<bf16, float>(n, s);
        default: return backward<double, double>(n, s);
    }
}
