// Layer norm over rows of features and its gradient (tcbnn_layernorm_forward / _backward).
//
//   mean = sum x / N,  var = sum (x - mean)^2 / N,  rstd = 1 / sqrt(var + eps),  y = (x - mean) rstd gamma + beta
//   xh = (x - mean) rstd,  g = dy gamma,  dx = rstd (g - mean(g) - xh mean(g xh)),
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
#include "head.h"

namespace tcbnn {
namespace {

using namespace head;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxFeatures = 65536;

__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += lds[w];
    return v;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layernorm_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, T* __restrict__ y,
                                                             float* __restrict__ mean_out, float* __restrict__ rstd_out, int n,
                                                             float eps, long long x_ld, long long y_ld) {
    __shared__ float lds[kWaves];
    const long long row = blockIdx.x;
    x += row * x_ld;
    y += row * y_ld;
    float s = 0.0f;
    for (int i = threadIdx.x; i < n; i += kThreads) s += (float)x[i];
    const float mean = block_sum(s, lds) / (float)n;
    s = 0.0f;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float d = (float)x[i] - mean;
        s = __builtin_fmaf(d, d, s);
    }
    const float rstd = 1.0f / sqrtf(block_sum(s, lds) / (float)n + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float xh = ((float)x[i] - mean) * rstd;
        y[i] = (T)__builtin_fmaf(xh, gamma ? gamma[i] : 1.0f, beta ? beta[i] : 0.0f);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layernorm_dx_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                                const float* __restrict__ mean_in,
                                                                const float* __restrict__ rstd_in, const T* dy, T* dx, int n,
                                                                long long x_ld, long long dy_ld, long long dx_ld) {
    __shared__ float lds[kWaves];
    const long long row = blockIdx.x;
    x += row * x_ld;
    dy += row * dy_ld;
    dx += row * dx_ld;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float sg = 0.0f, sgx = 0.0f;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float g = (float)dy[i] * (gamma ? gamma[i] : 1.0f);
        sg += g;
        sgx = __builtin_fmaf(g, ((float)x[i] - mean) * rstd, sgx);
    }
    sg = block_sum(sg, lds) / (float)n;
    sgx = block_sum(sgx, lds) / (float)n;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float g = (float)dy[i] * (gamma ? gamma[i] : 1.0f);
        const float xh = ((float)x[i] - mean) * rstd;
        dx[i] = (T)((g - sg - xh * sgx) * rstd);
    }
}

// a thread a feature, all rows in order
template <typename T>
__global__ __launch_bounds__(kThreads) void layernorm_params_kernel(const T* __restrict__ x, const float* __restrict__ mean,
                                                                    const float* __restrict__ rstd, const T* __restrict__ dy,
                                                                    float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                                    int rows, int n, long long x_ld, long long dy_ld) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    float sg = 0.0f, sb = 0.0f;
    for (long long r = 0; r < rows; ++r) {
        const float d = (float)dy[r * dy_ld + i];
        sb += d;
        sg = __builtin_fmaf(d, ((float)x[r * x_ld + i] - mean[r]) * rstd[r], sg);
    }
    if (dgamma) dgamma[i] = sg;
    if (dbeta) dbeta[i] = sb;
}

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

extern "C" int tcbnn_layernorm_forward(const tcbnn_layernorm_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    TCBNN_REQUIRE(dtype_known(d->dtype), "layernorm: unknown dtype");
    TCBNN_REQUIRE(d->rows >= 0 && d->features > 0, "layernorm: bad shape");
    TCBNN_REQUIRE(d->features <= kMaxFeatures, "layernorm: at most %d features", kMaxFeatures);
    TCBNN_REQUIRE(d->eps >= 0.0f, "layernorm: eps must be 0 or more");
    const long long x_ld = row_stride(d->input_ld, d->features), y_ld = row_stride(d->output_ld, d->features);
    TCBNN_REQUIRE(x_ld > 0 && y_ld > 0, "layernorm: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->input);
    TCBNN_NOTNULL(d->output);
    TCBNN_REQUIRE(d->output != d->input || d->rows == 1 || x_ld == y_ld, "layernorm: an output over its input has the input's stride");
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(layernorm_kernel<T>, dim3((unsigned)d->rows), dim3(kThreads), 0, (hipStream_t)stream, (const T*)d->input,
                           d->gamma, d->beta, (T*)d->output, d->mean, d->rstd, d->features, d->eps, x_ld, y_ld);
    });
    TCBNN_LAUNCH_CHECK("layernorm_kernel");
    return TCBNN_OK;
}

extern "C" size_t tcbnn_layernorm_grad_workspace_bytes(int rows, int features) { return 0; }

extern "C" int tcbnn_layernorm_backward(const tcbnn_layernorm_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    TCBNN_REQUIRE(dtype_known(d->dtype), "layernorm: unknown dtype");
    TCBNN_REQUIRE(d->rows >= 0 && d->features > 0, "layernorm: bad shape");
    TCBNN_REQUIRE(d->features <= kMaxFeatures, "layernorm: at most %d features", kMaxFeatures);
    const long long x_ld = row_stride(d->input_ld, d->features), dy_ld = row_stride(d->grad_output_ld, d->features),
                    dx_ld = row_stride(d->grad_input_ld, d->features);
    TCBNN_REQUIRE(x_ld > 0 && dy_ld > 0 && dx_ld > 0, "layernorm: rows overlap");
    if (d->rows > 0) {
        TCBNN_NOTNULL(d->input);
        TCBNN_NOTNULL(d->mean);
        TCBNN_NOTNULL(d->rstd);
        TCBNN_NOTNULL(d->grad_output);
    }
    TCBNN_REQUIRE(d->grad_input != d->grad_output || d->grad_input == nullptr || d->rows <= 1 || dx_ld == dy_ld,
                  "layernorm: a gradient over another has its stride");
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        if (d->grad_gamma || d->grad_beta)
            hipLaunchKernelGGL(layernorm_params_kernel<T>, dim3((unsigned)((d->features + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                               (hipStream_t)stream, (const T*)d->input, d->mean, d->rstd, (const T*)d->grad_output, d->grad_gamma,
                               d->grad_beta, d->rows, d->features, x_ld, dy_ld);
        if (d->grad_input && d->rows > 0)
            hipLaunchKernelGGL(layernorm_dx_kernel<T>, dim3((unsigned)d->rows), dim3(kThreads), 0, (hipStream_t)stream,
                               (const T*)d->input, d->gamma, d->mean, d->rstd, (const T*)d->grad_output, (T*)d->grad_input,
                               d->features, x_ld, dy_ld, dx_ld);
    });
    TCBNN_LAUNCH_CHECK("layernorm_dx_kernel");
    return TCBNN_OK;
}
