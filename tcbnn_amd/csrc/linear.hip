// Linear layers and their gradients (tcbnn_linear_forward / _backward):  z = x w^T + b,  y = act(z) + r;
// dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = column sums of dz.
#include "head.h"

namespace tcbnn {
namespace {

using namespace head;

constexpr int kTile = 64, kDepth = 16, kThreads = 256;
constexpr int kMaxIn = 1 << 20;

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == TCBNN_ACT_RELU) return z > 0.0f || z != z ? z : 0.0f;
    if constexpr (ACT == TCBNN_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    if constexpr (ACT == TCBNN_ACT_SILU) return z / (1.0f + expf(-z));
    return z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == TCBNN_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == TCBNN_ACT_GELU)
        return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    if constexpr (ACT == TCBNN_ACT_SILU) {
        const float p = 1.0f / (1.0f + expf(-z));
        return p * (1.0f + z * (1.0f - p));
    }
    return 1.0f;
}
template <typename F>
void by_activation(int act, F&& f) {
    if (act == TCBNN_ACT_RELU) return f(std::integral_constant<int, TCBNN_ACT_RELU>());
    if (act == TCBNN_ACT_GELU) return f(std::integral_constant<int, TCBNN_ACT_GELU>());
    if (act == TCBNN_ACT_SILU) return f(std::integral_constant<int, TCBNN_ACT_SILU>());
    return f(std::integral_constant<int, TCBNN_ACT_NONE>());
}

// c[i][j] = epilogue(sum over k of a(i, k) b(j, k)), operands anywhere: a(i, k) = a[i * a_i + k * a_k]
struct ProductParams {
    long long m, n, k, a_i, a_k, b_i, b_k;
    const float* bias;
    const void* residual;
    void* out;
    void* preact;
    long long residual_ld, out_ld, preact_ld;
};

template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void product_kernel(const T* __restrict__ a, const T* __restrict__ b, const ProductParams p) {
    __shared__ float la[kDepth][kTile + 1], lb[kDepth][kTile + 1];
    const int tid = threadIdx.x, ti = tid >> 4, tj = tid & 15;
    const long long i0 = (long long)blockIdx.y * kTile, j0 = (long long)blockIdx.x * kTile;
    float acc[4][4] = {};
    for (long long k0 = 0; k0 < p.k; k0 += kDepth) {
        __syncthreads();
        for (int e = tid; e < kTile * kDepth; e += kThreads) {
            const int ra = p.a_k == 1 ? e / kDepth : e % kTile, ka = p.a_k == 1 ? e % kDepth : e / kTile;
            la[ka][ra] = i0 + ra < p.m && k0 + ka < p.k ? (float)a[(i0 + ra) * p.a_i + (k0 + ka) * p.a_k] : 0.0f;
            const int rb = p.b_k == 1 ? e / kDepth : e % kTile, kb = p.b_k == 1 ? e % kDepth : e / kTile;
            lb[kb][rb] = j0 + rb < p.n && k0 + kb < p.k ? (float)b[(j0 + rb) * p.b_i + (k0 + kb) * p.b_k] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[u][v] = __builtin_fmaf(la[k][ti + 16 * u], lb[k][tj + 16 * v], acc[u][v]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const long long i = i0 + ti + 16 * u, j = j0 + tj + 16 * v;
            if (i >= p.m || j >= p.n) continue;
            const float z = acc[u][v] + (p.bias ? p.bias[j] : 0.0f);
            if (p.preact) ((T*)p.preact)[i * p.preact_ld + j] = (T)z;
            float y = activate<ACT>(z);
            if (p.residual) y += (float)((const T*)p.residual)[i * p.residual_ld + j];
            ((T*)p.out)[i * p.out_ld + j] = (T)y;
        }
}

// dz = dy act'(z) in the operands' type (nothing to write without an activation) and its column sums in fp32: a thread a
// column, all rows in order
template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void dz_kernel(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                      float* __restrict__ db, int rows, int n, long long dy_ld, long long z_ld) {
    const int j = blockIdx.x * kThreads + threadIdx.x;
    if (j >= n) return;
    float s = 0.0f;
    for (long long r = 0; r < rows; ++r) {
        float g = (float)dy[r * dy_ld + j];
        if constexpr (ACT != TCBNN_ACT_NONE) {
            g *= slope<ACT>((float)z[r * z_ld + j]);
            dz[r * n + j] = (T)g;
        }
        s += g;
    }
    if (db) db[j] = s;
}

template <typename T, int ACT>
void launch_product(const T* a, const T* b, const ProductParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)((p.n + kTile - 1) / kTile), (unsigned)((p.m + kTile - 1) / kTile));
    hipLaunchKernelGGL(HIP_KERNEL_NAME(product_kernel<T, ACT>), grid, dim3(kThreads), 0, stream, a, b, p);
}

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

static int check_linear(int rows, int in_features, int out_features, int dtype, int activation) {
    TCBNN_REQUIRE(dtype_known(dtype), "linear: unknown dtype");
    TCBNN_REQUIRE(activation >= TCBNN_ACT_NONE && activation <= TCBNN_ACT_SILU, "linear: unknown activation");
    TCBNN_REQUIRE(rows >= 0 && in_features > 0 && out_features > 0, "linear: bad shape");
    TCBNN_REQUIRE(in_features <= kMaxIn, "linear: at most %d inputs", kMaxIn);
    return TCBNN_OK;
}

extern "C" size_t tcbnn_linear_workspace_bytes(int rows, int in_features, int out_features, int dtype) { return 0; }

extern "C" int tcbnn_linear_forward(const tcbnn_linear_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_linear(d->rows, d->in_features, d->out_features, d->dtype, d->activation)) return rc;
    const long long x_ld = row_stride(d->input_ld, d->in_features), w_ld = row_stride(d->weight_ld, d->in_features),
                    r_ld = row_stride(d->residual_ld, d->out_features), y_ld = row_stride(d->output_ld, d->out_features),
                    z_ld = row_stride(d->preact_ld, d->out_features);
    TCBNN_REQUIRE(x_ld > 0 && w_ld > 0 && r_ld > 0 && y_ld > 0 && z_ld > 0, "linear: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->input);
    TCBNN_NOTNULL(d->weight);
    TCBNN_NOTNULL(d->output);
    TCBNN_REQUIRE(d->output != d->residual || d->rows == 1 || y_ld == r_ld, "linear: an output over its residual has the residual's stride");
    ProductParams p = {d->rows, d->out_features, d->in_features, x_ld, 1, w_ld, 1, d->bias, d->residual, d->output, d->preact, r_ld, y_ld, z_ld};
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        by_activation(d->activation, [&](auto act) {
            launch_product<T, act.value>((const T*)d->input, (const T*)d->weight, p, (hipStream_t)stream);
        });
    });
    TCBNN_LAUNCH_CHECK("product_kernel");
    return TCBNN_OK;
}

extern "C" size_t tcbnn_linear_grad_workspace_bytes(int rows, int in_features, int out_features, int dtype) {
    if (rows <= 0 || in_features <= 0 || out_features <= 0 || !dtype_known(dtype)) return 0;
    return (size_t)rows * out_features * dtype_bytes(dtype);
}

extern "C" int tcbnn_linear_backward(const tcbnn_linear_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_linear(d->rows, d->in_features, d->out_features, d->dtype, d->activation)) return rc;
    const long long x_ld = row_stride(d->input_ld, d->in_features), w_ld = row_stride(d->weight_ld, d->in_features),
                    z_ld = row_stride(d->preact_ld, d->out_features), dy_ld = row_stride(d->grad_output_ld, d->out_features),
                    dx_ld = row_stride(d->grad_input_ld, d->in_features), dw_ld = row_stride(d->grad_weight_ld, d->in_features);
    TCBNN_REQUIRE(x_ld > 0 && w_ld > 0 && z_ld > 0 && dy_ld > 0 && dx_ld > 0 && dw_ld > 0, "linear: rows overlap");
    const bool active = d->activation != TCBNN_ACT_NONE;
    if (d->rows > 0) {
        TCBNN_NOTNULL(d->grad_output);
        if (active) TCBNN_NOTNULL(d->preact);
        if (d->grad_weight) TCBNN_NOTNULL(d->input);
        if (d->grad_input) TCBNN_NOTNULL(d->weight);
        if (active && tcbnn_linear_grad_workspace_bytes(d->rows, d->in_features, d->out_features, d->dtype) > 0) {
            TCBNN_NOTNULL(d->workspace);
            TCBNN_REQUIRE(d->workspace_bytes >= tcbnn_linear_grad_workspace_bytes(d->rows, d->in_features, d->out_features, d->dtype),
                          "linear: workspace too small");
        }
    }
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        const T* dz = active ? (const T*)d->workspace : (const T*)d->grad_output;
        const long long dz_ld = active ? d->out_features : dy_ld;
        by_activation(d->activation, [&](auto act) {
            if (active || d->grad_bias)
                hipLaunchKernelGGL(HIP_KERNEL_NAME(dz_kernel<T, act.value>), dim3((unsigned)((d->out_features + kThreads - 1) / kThreads)),
                                   dim3(kThreads), 0, (hipStream_t)stream, (const T*)d->grad_output, (const T*)d->preact,
                                   (T*)d->workspace, d->grad_bias, d->rows, d->out_features, dy_ld, z_ld);
        });
        if (d->grad_input && d->rows > 0)
            launch_product<T, TCBNN_ACT_NONE>(dz, (const T*)d->weight,
                                              {d->rows, d->in_features, d->out_features, dz_ld, 1, 1, w_ld, nullptr, nullptr, d->grad_input,
                                               nullptr, 0, dx_ld, 0},
                                              (hipStream_t)stream);
        if (d->grad_weight)
            launch_product<T, TCBNN_ACT_NONE>(dz, (const T*)d->input,
                                              {d->out_features, d->in_features, d->rows, 1, dz_ld, 1, x_ld, nullptr, nullptr, d->grad_weight,
                                               nullptr, 0, dw_ld, 0},
                                              (hipStream_t)stream);
    });
    TCBNN_LAUNCH_CHECK("product_kernel");
    return TCBNN_OK;
}
