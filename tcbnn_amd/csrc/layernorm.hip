// Layer norm over rows of features and its gradient (tcbnn_layernorm_forward / _backward).
//
//   mean = sum x / N,  var = sum (x - mean)^2 / N,  rstd = 1 / sqrt(var + eps),  y = (x - mean) rstd gamma + beta
//   xh = (x - mean) rstd,  g = dy gamma,  dx = rstd (g - mean(g) - xh mean(g xh)),
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// Bound by memory: every value is read once and kept in registers as fp32 (the variance is summed about the mean, which one
// pass over the memory allows because the row is still there).  A row belongs to a team of W wavefronts whose lanes hold R
// vectors of 16 bytes each; teams go from row to row, so gamma, beta and the gradient's sums over rows stay in registers too.
// 16384 x 4096 bf16: 50 us forward (268 MB, 5.3 TB/s); 8192 x 4096: 46 us backward (201 MB and the sums, 4.4 TB/s).  A row
// alone (1 x 4096) takes 3.2 us: the launch, one latency of memory and two sums over a team.
#include "rows.h"

namespace tcbnn {
namespace {

using namespace head;

// All teams of a workgroup take the same number of steps; one without a row of its own computes on the last one
// and keeps nothing.
template <typename T, int W, int R>
__global__ __launch_bounds__(forward_threads(W)) void layernorm_kernel(const T* x, const float* __restrict__ gamma,
                                                                       const float* __restrict__ beta, T* y,
                                                                       float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                                       int rows, int n, float eps, long long x_ld, long long y_ld) {
    constexpr int kTeams = forward_threads(W) / (64 * W);
    using Slice = RowSlice<T, W, R>;
    constexpr int V = Slice::V;
    __shared__ float slots[2][kTeams][W];
    const int lane = threadIdx.x % (64 * W), wave = lane >> 6, team = threadIdx.x / (64 * W);
    Slice g, b, s;
    typename Slice::Raw raw;
    const long long stride = (long long)gridDim.x * kTeams;
    auto request = [&](long long first) { Slice::request(x + min(first + team, (long long)rows - 1) * x_ld, lane, n, raw); };
    request((long long)blockIdx.x * kTeams);
    g.load_param(gamma, lane, n, 1.0f);
    b.load_param(beta, lane, n, 0.0f);
    const float inv = 1.0f / (float)n;
    for (long long first = (long long)blockIdx.x * kTeams; first < rows; first += stride) {
        const bool mine = first + team < rows;
        const long long row = first + team;
        s.take(raw);
        if (first + stride < rows) request(first + stride);
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) sum += s.v[r][e];
        const float mean = team_sum<W>(sum, slots[0][team], wave) * inv;
        float sq = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                // what lies past the row (the last slices' lanes alone) has no share in the variance
                const bool in = (r + 1) * Slice::kStep <= n || r * Slice::kStep + lane * V + e < n;
                const float d = in ? s.v[r][e] - mean : 0.0f;
                s.v[r][e] = d;
                sq = __builtin_fmaf(d, d, sq);
            }
        const float rstd = 1.0f / sqrtf(__builtin_fmaf(team_sum<W>(sq, slots[1][team], wave), inv, eps));
        if (!mine) continue;
        if (lane == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) s.v[r][e] = __builtin_fmaf(s.v[r][e] * rstd, g.v[r][e], b.v[r][e]);
        s.store(y + row * y_ld, lane, n);
    }
}

// Rows that a workgroup's registers do not hold: a workgroup a row, which is read three times (twice from the cache).  Rows beyond
// the workgroups of a launch are taken by the same ones afterwards (with two workgroups a compute unit from the start 20000 x 8196 fp32 takes
// 520 us, 498 with one a row); between two sums into one slot lies the barrier of the other's.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void layernorm_long_kernel(const T* x, const float* __restrict__ gamma,
                                                                      const float* __restrict__ beta, T* y,
                                                                      float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                                      int rows, int n, float eps, long long x_ld, long long y_ld) {
    __shared__ float slots[2][kLongThreads / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* from = x + row * x_ld;
        T* to = y + row * y_ld;
        float s = 0.0f;
        for (int i = threadIdx.x; i < n; i += kLongThreads) s += (float)from[i];
        const float mean = long_sum(s, slots[0]) / (float)n;
        s = 0.0f;
        for (int i = threadIdx.x; i < n; i += kLongThreads) {
            const float d = (float)from[i] - mean;
            s = __builtin_fmaf(d, d, s);
        }
        const float rstd = 1.0f / sqrtf(long_sum(s, slots[1]) / (float)n + eps);
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
        for (int i = threadIdx.x; i < n; i += kLongThreads)
            to[i] = (T)__builtin_fmaf(((float)from[i] - mean) * rstd, gamma ? gamma[i] : 1.0f, beta ? beta[i] : 0.0f);
    }
}

// ---- gradient.  A workgroup of 16 wavefronts is 16 / W teams; all of them take the same number of steps (a team without a
// row of its own computes on the last one and keeps nothing).  PARAMS: sums over the workgroup's rows of dy xh and
// dy, one row of `partial` a workgroup: [2][n] each; a workgroup that has all rows writes the gradients themselves.
template <typename T, int W, int R, bool PARAMS>
__global__ __launch_bounds__(kGradThreads) void layernorm_grad_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                                      const float* __restrict__ mean_in,
                                                                      const float* __restrict__ rstd_in, const T* dy, T* dx,
                                                                      float* __restrict__ partial, float* __restrict__ dgamma,
                                                                      float* __restrict__ dbeta, int rows, int n, long long x_ld,
                                                                      long long dy_ld, long long dx_ld) {
    constexpr int kTeams = kGradThreads / (64 * W);
    using Slice = RowSlice<T, W, R>;
    constexpr int V = Slice::V;
    __shared__ float slots[2][kTeams][2][W];
    __shared__ float sums[PARAMS && kTeams > 1 ? kTeams * 64 * W * V : 1];
    const int lane = threadIdx.x % (64 * W), wave = lane >> 6, team = threadIdx.x / (64 * W);
    Slice g, s, d, dg, db;
    typename Slice::Raw raw_x, raw_dy;
    float next_mean, next_rstd;
    const long long stride = (long long)gridDim.x * kTeams;
    auto request = [&](long long first) {
        const long long row = min(first + team, (long long)rows - 1);
        next_mean = mean_in[row];
        next_rstd = rstd_in[row];
        Slice::request(x + row * x_ld, lane, n, raw_x);
        Slice::request(dy + row * dy_ld, lane, n, raw_dy);
    };
    request((long long)blockIdx.x * kTeams);
    g.load_param(gamma, lane, n, 1.0f);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) dg.v[r][e] = db.v[r][e] = 0.0f;
    const float inv = 1.0f / (float)n;
    int parity = 0;
    for (long long first = (long long)blockIdx.x * kTeams; first < rows; first += stride, parity ^= 1) {
        const bool mine = first + team < rows;
        const long long row = min(first + team, (long long)rows - 1);
        s.take(raw_x);
        d.take(raw_dy);
        const float mean = next_mean, rstd = next_rstd;
        if (first + stride < rows) request(first + stride);
        float sg = 0.0f, sgx = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (s.v[r][e] - mean) * rstd;  // (past the row dy is 0, and so is every product)
                s.v[r][e] = xh;
                if constexpr (PARAMS) {
                    const float dv = mine ? d.v[r][e] : 0.0f;
                    db.v[r][e] += dv;
                    dg.v[r][e] = __builtin_fmaf(dv, xh, dg.v[r][e]);
                }
                const float gv = d.v[r][e] * g.v[r][e];
                d.v[r][e] = gv;
                sg += gv;
                sgx = __builtin_fmaf(gv, xh, sgx);
            }
        if (dx) {
            sg = wave_sum(sg);
            sgx = wave_sum(sgx);
            if constexpr (W > 1) {
                slots[parity][team][0][wave] = sg;
                slots[parity][team][1][wave] = sgx;
                __syncthreads();
                sg = sgx = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    sg += slots[parity][team][0][w];
                    sgx += slots[parity][team][1][w];
                }
            }
            sg *= inv;
            sgx *= inv;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) d.v[r][e] = (d.v[r][e] - sg - s.v[r][e] * sgx) * rstd;
            if (mine) d.store(dx + row * dx_ld, lane, n);
        }
    }
    if constexpr (PARAMS) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float* out = gridDim.x > 1 ? partial + ((size_t)blockIdx.x * 2 + which) * n : (which == 0 ? dgamma : dbeta);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const Slice& a = which == 0 ? dg : db;
                if constexpr (kTeams == 1) {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (out && r * Slice::kStep + lane * V + e < n) out[r * Slice::kStep + lane * V + e] = a.v[r][e];
                } else {
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < V; ++e) sums[(team * V + e) * 64 * W + lane] = a.v[r][e];  // (lanes side by side: no bank twice)
                    __syncthreads();
                    for (int c = threadIdx.x; c < Slice::kStep; c += kGradThreads) {
                        const int e = c / (64 * W), l = c % (64 * W), i = r * Slice::kStep + l * V + e;
                        float t = 0.0f;
                        for (int k = 0; k < kTeams; ++k) t += sums[(k * V + e) * 64 * W + l];
                        if (out && i < n) out[i] = t;
                    }
                }
            }
        }
    }
}

// Rows that a workgroup's registers do not hold: the gradient of the input, a workgroup a row ...
template <typename T>
__global__ __launch_bounds__(kLongThreads) void layernorm_long_grad_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                                           const float* __restrict__ mean_in,
                                                                           const float* __restrict__ rstd_in, const T* dy, T* dx, int rows,
                                                                           int n, long long x_ld, long long dy_ld, long long dx_ld) {
    __shared__ float slots[2][kLongThreads / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *from = x + row * x_ld, *dy_row = dy + row * dy_ld;
        T* to = dx + row * dx_ld;
        const float mean = mean_in[row], rstd = rstd_in[row];
        float sg = 0.0f, sgx = 0.0f;
        for (int i = threadIdx.x; i < n; i += kLongThreads) {
            const float g = (float)dy_row[i] * (gamma ? gamma[i] : 1.0f);
            sg += g;
            sgx = __builtin_fmaf(g, ((float)from[i] - mean) * rstd, sgx);
        }
        sg = long_sum(sg, slots[0]) / (float)n;
        sgx = long_sum(sgx, slots[1]) / (float)n;
        for (int i = threadIdx.x; i < n; i += kLongThreads) {
            const float g = (float)dy_row[i] * (gamma ? gamma[i] : 1.0f);
            to[i] = (T)((g - sg - ((float)from[i] - mean) * rstd * sgx) * rstd);
        }
    }
}

// ... and the parameters' sums: 256 features a workgroup, every so manieth row, sums as above.
constexpr int kColumnThreads = 256;
template <typename T>
__global__ __launch_bounds__(kColumnThreads) void layernorm_columns_kernel(const T* __restrict__ x, const float* __restrict__ mean,
                                                                           const float* __restrict__ rstd, const T* __restrict__ dy,
                                                                           float* __restrict__ partial, int rows, int n,
                                                                           long long x_ld, long long dy_ld) {
    const int i = blockIdx.x * kColumnThreads + threadIdx.x;
    if (i >= n) return;
    float sg = 0.0f, sb = 0.0f;
    for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
        const float d = (float)dy[r * dy_ld + i];
        sb += d;
        sg = __builtin_fmaf(d, ((float)x[r * x_ld + i] - mean[r]) * rstd[r], sg);
    }
    partial[((size_t)blockIdx.y * 2) * n + i] = sg;
    partial[((size_t)blockIdx.y * 2 + 1) * n + i] = sb;
}

// The sums of all workgroups: 16 features a workgroup, 16 threads to a feature.
constexpr int kJoinThreads = 256, kJoinFeatures = 16;
__global__ __launch_bounds__(kJoinThreads) void layernorm_join_kernel(const float* __restrict__ partial, float* __restrict__ dgamma,
                                                                      float* __restrict__ dbeta, int parts, int n) {
    __shared__ float lds[kJoinThreads / kJoinFeatures][kJoinFeatures];
    const int c = threadIdx.x % kJoinFeatures, part = threadIdx.x / kJoinFeatures, i = blockIdx.x * kJoinFeatures + c;
    float* out = blockIdx.y == 0 ? dgamma : dbeta;
    if (out == nullptr) return;
    float s = 0.0f;
    if (i < n) {
        const float* p = partial + (size_t)blockIdx.y * n + i;
        constexpr int kStep = kJoinThreads / kJoinFeatures;
        for (int k = part; k < parts; k += 8 * kStep) {
            float v[8];  // (requests of their own, one wait)
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = k + u * kStep < parts ? p[(size_t)(k + u * kStep) * 2 * n] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
    }
    lds[part][c] = s;
    __syncthreads();
    if (part == 0 && i < n) {
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < kJoinThreads / kJoinFeatures; ++k) s += lds[k][c];
        out[i] = s;
    }
}

int check_norm(int rows, int features, int dtype) {
    TCBNN_REQUIRE(dtype_known(dtype), "layernorm: unknown dtype");
    TCBNN_REQUIRE(rows >= 0 && features > 0, "layernorm: bad shape");
    TCBNN_REQUIRE(features <= kMaxFeatures, "layernorm: at most %d features", kMaxFeatures);
    return TCBNN_OK;
}

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

extern "C" int tcbnn_layernorm_forward(const tcbnn_layernorm_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_norm(d->rows, d->features, d->dtype)) return rc;
    TCBNN_REQUIRE(d->eps >= 0.0f, "layernorm: eps must be 0 or more");
    const long long x_ld = row_stride(d->input_ld, d->features), y_ld = row_stride(d->output_ld, d->features);
    TCBNN_REQUIRE(x_ld > 0 && y_ld > 0, "layernorm: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->input);
    TCBNN_NOTNULL(d->output);
    TCBNN_REQUIRE(d->output != d->input || d->rows == 1 || x_ld == y_ld, "layernorm: an output over its input has the input's stride");
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        const int vectors = row_vectors(d->features, Elem<T>::kVec);
        if (vectors > kMaxVectors) {
            hipLaunchKernelGGL(layernorm_long_kernel<T>, dim3((unsigned)long_blocks(d->rows)), dim3(kLongThreads), 0, (hipStream_t)stream,
                               (const T*)d->input, d->gamma, d->beta, (T*)d->output, d->mean, d->rstd, d->rows, d->features, d->eps, x_ld, y_ld);
            return;
        }
        by_team(vectors, [&](auto w, auto r) {
            constexpr int W = w.value, R = r.value;
            const int teams = forward_threads(W) / (64 * W);
            // the registers of 2048 threads a compute unit, more where rows are left
            const int blocks = (int)std::min((d->rows + teams - 1LL) / teams, kComputeUnits * 2048LL / forward_threads(W));
            hipLaunchKernelGGL(HIP_KERNEL_NAME(layernorm_kernel<T, W, R>), dim3((unsigned)blocks), dim3(forward_threads(W)), 0,
                               (hipStream_t)stream, (const T*)d->input, d->gamma, d->beta, (T*)d->output, d->mean, d->rstd, d->rows,
                               d->features, d->eps, x_ld, y_ld);
        });
    });
    TCBNN_LAUNCH_CHECK("layernorm_kernel");
    return TCBNN_OK;
}

extern "C" size_t tcbnn_layernorm_grad_workspace_bytes(int rows, int features) {
    if (rows <= 0 || features <= 0 || features > kMaxFeatures) return 0;
    return (size_t)std::min(rows, kComputeUnits) * 2 * features * sizeof(float);
}

extern "C" int tcbnn_layernorm_backward(const tcbnn_layernorm_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_norm(d->rows, d->features, d->dtype)) return rc;
    const long long x_ld = row_stride(d->input_ld, d->features), dy_ld = row_stride(d->grad_output_ld, d->features),
                    dx_ld = row_stride(d->grad_input_ld, d->features);
    TCBNN_REQUIRE(x_ld > 0 && dy_ld > 0 && dx_ld > 0, "layernorm: rows overlap");
    const bool params = d->grad_gamma || d->grad_beta;
    if (d->rows > 0) {
        TCBNN_NOTNULL(d->input);
        TCBNN_NOTNULL(d->mean);
        TCBNN_NOTNULL(d->rstd);
        TCBNN_NOTNULL(d->grad_output);
        if (params) {
            TCBNN_NOTNULL(d->workspace);
            TCBNN_REQUIRE(d->workspace_bytes >= tcbnn_layernorm_grad_workspace_bytes(d->rows, d->features), "layernorm: workspace too small");
        }
    }
    TCBNN_REQUIRE(d->grad_input != d->grad_output || d->grad_input == nullptr || d->rows <= 1 || dx_ld == dy_ld,
                  "layernorm: a gradient over another has its stride");
    float* partial = (float*)d->workspace;
    int parts = 0;
    bool joined = false;
    if (d->rows > 0)
        by_dtype(d->dtype, [&](auto t) {
            using T = decltype(t);
            const int vectors = row_vectors(d->features, Elem<T>::kVec);
            if (vectors > kMaxVectors) {
                if (params) {
                    parts = std::min(d->rows, kComputeUnits);
                    hipLaunchKernelGGL(layernorm_columns_kernel<T>,
                                       dim3((unsigned)((d->features + kColumnThreads - 1) / kColumnThreads), (unsigned)parts),
                                       dim3(kColumnThreads), 0, (hipStream_t)stream, (const T*)d->input, d->mean, d->rstd,
                                       (const T*)d->grad_output, partial, d->rows, d->features, x_ld, dy_ld);
                }
                if (d->grad_input)
                    hipLaunchKernelGGL(layernorm_long_grad_kernel<T>, dim3((unsigned)long_blocks(d->rows)), dim3(kLongThreads), 0,
                                       (hipStream_t)stream, (const T*)d->input, d->gamma, d->mean, d->rstd, (const T*)d->grad_output,
                                       (T*)d->grad_input, d->rows, d->features, x_ld, dy_ld, dx_ld);
                return;
            }
            by_team(vectors, [&](auto w, auto r) {
                constexpr int W = w.value, R = r.value, kTeams = kGradThreads / (64 * W);
                parts = params ? grad_parts(d->rows, kTeams) : (int)std::min((d->rows + kTeams - 1LL) / kTeams, (long long)kComputeUnits);
                auto launch = [&](auto kernel) {
                    hipLaunchKernelGGL(kernel, dim3((unsigned)parts), dim3(kGradThreads), 0, (hipStream_t)stream, (const T*)d->input,
                                       d->gamma, d->mean, d->rstd, (const T*)d->grad_output, (T*)d->grad_input, partial, d->grad_gamma,
                                       d->grad_beta, d->rows, d->features, x_ld, dy_ld, dx_ld);
                };
                joined = params && parts == 1;
                if (params)
                    launch(layernorm_grad_kernel<T, W, R, true>);
                else if (d->grad_input)
                    launch(layernorm_grad_kernel<T, W, R, false>);
            });
        });
    if (params && !joined)
        hipLaunchKernelGGL(layernorm_join_kernel, dim3((unsigned)((d->features + kJoinFeatures - 1) / kJoinFeatures), 2), dim3(kJoinThreads),
                           0, (hipStream_t)stream, partial, d->grad_gamma, d->grad_beta, parts, d->features);
    TCBNN_LAUNCH_CHECK("layernorm_grad_kernel");
    return TCBNN_OK;
}
