// Log probabilities of given classes with entropy, rank and the best alternatives, and their gradient
// (tcbnn_logprobs_forward / _backward).
//
//   m = max x,  s = sum exp(x - m),  logsumexp = m + log s,  entropy = log s - (sum (x - m) exp(x - m)) / s
//   dx_j = g_logprob ([j = t] - p_j) - g_entropy p_j (log p_j + entropy)
#include "head.h"

namespace tcbnn {
namespace {

using namespace head;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;

// The order of classes as one number: larger logits first (NaN before all, -0 with +0), lower indices first among equals.
// Larger keys come first; 0 is below every class's key.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, int j) { return ((uint64_t)ordered(x) << 32) | (uint32_t)~j; }

__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)v, d);
        if (o > v) v = o;
    }
    return v;
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* lds, F f) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = f(v, lds[w]);
    return v;
}

struct LogProbsParams {
    const int32_t* targets;
    float *logprob, *entropy, *logsumexp, *top_logprob;
    int32_t *rank, *top_index;
    int classes, top;
    long long ld;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const T* __restrict__ x, const LogProbsParams p) {
    __shared__ float lds_f[kWaves];
    __shared__ uint64_t lds_k[kWaves];
    const long long row = blockIdx.x;
    x += row * p.ld;
    const int n = p.classes, tid = threadIdx.x;
    auto add = [](float a, float b) { return a + b; };
    // the largest key has the largest value (or NaN)
    uint64_t best = 0;
    for (int j = tid; j < n; j += kThreads) best = max(best, key_of((float)x[j], j));
    best = block_reduce(wave_max_key(best), lds_k, [](uint64_t a, uint64_t b) { return max(a, b); });
    const float m = (float)x[(int)~(uint32_t)best];
    const float shift = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, sx = 0.0f;
    for (int j = tid; j < n; j += kThreads) {
        const float d = (float)x[j] - shift;
        const float e = expf(d);
        s += e;
        if (e != 0.0f) sx = __builtin_fmaf(e, d, sx);
    }
    s = block_reduce(wave_sum(s), lds_f, add);
    sx = block_reduce(wave_sum(sx), lds_f, add);
    const float lse = m == -INFINITY ? m : m + logf(s);
    const int t = p.targets ? p.targets[row] : -1;
    const bool given = t >= 0 && t < n;
    const float xt = given ? (float)x[t] : 0.0f;
    int before = 0;
    if (p.rank && given) {
        const uint64_t kt = key_of(xt, t);
        for (int j = tid; j < n; j += kThreads) before += key_of((float)x[j], j) > kt;
        float c = wave_sum((float)before);
        before = (int)block_reduce(c, lds_f, add);
    }
    auto log_prob = [&](float v) { return m == -INFINITY ? m : v - lse; };
    if (tid == 0) {
        if (p.logprob) p.logprob[row] = given ? log_prob(xt) : (t < 0 ? 0.0f : NAN);
        if (p.entropy) p.entropy[row] = m == -INFINITY ? 0.0f : logf(s) - sx / s;
        if (p.logsumexp) p.logsumexp[row] = lse;
        if (p.rank) p.rank[row] = given ? before : -1;
    }
    for (int k = 0; k < p.top; ++k) {
        if (tid == 0) {
            const int j = (int)~(uint32_t)best;
            if (p.top_index) p.top_index[row * p.top + k] = j;
            if (p.top_logprob) p.top_logprob[row * p.top + k] = log_prob((float)x[j]);
        }
        uint64_t next = 0;
        for (int j = tid; j < n; j += kThreads) {
            const uint64_t key = key_of((float)x[j], j);
            if (key < best) next = max(next, key);
        }
        best = block_reduce(wave_max_key(next), lds_k, [](uint64_t a, uint64_t b) { return max(a, b); });
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_grad_kernel(const T* x, const int32_t* __restrict__ targets,
                                                                 const float* __restrict__ logsumexp,
                                                                 const float* __restrict__ entropy,
                                                                 const float* __restrict__ g_logprob,
                                                                 const float* __restrict__ g_entropy, T* dx, int n,
                                                                 long long x_ld, long long dx_ld) {
    const long long row = blockIdx.x;
    x += row * x_ld;
    dx += row * dx_ld;
    const float lse = logsumexp[row];
    const int t = g_logprob ? targets[row] : -1;
    const float g = t >= n ? NAN : (t >= 0 ? g_logprob[row] : 0.0f);
    const float ge = g_entropy ? g_entropy[row] : 0.0f, h = g_entropy ? entropy[row] : 0.0f;
    for (int j = threadIdx.x; j < n; j += kThreads) {
        float out = 0.0f;
        if (lse != -INFINITY) {
            const float lp = (float)x[j] - lse;
            const float p = expf(lp);
            out = g * ((j == t ? 1.0f : 0.0f) - p);
            if (p != 0.0f) out -= ge * p * (lp + h);
        } else if (g != g) {
            out = g;
        }
        dx[j] = (T)out;
    }
}

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

extern "C" size_t tcbnn_logprobs_workspace_bytes(int rows, int classes, int top, int dtype) { return 0; }

extern "C" int tcbnn_logprobs_forward(const tcbnn_logprobs_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    TCBNN_REQUIRE(dtype_known(d->dtype), "logprobs: unknown dtype");
    TCBNN_REQUIRE(d->rows >= 0 && d->classes > 0, "logprobs: bad shape");
    TCBNN_REQUIRE(d->top >= 0 && d->top <= kMaxTop && d->top <= d->classes, "logprobs: top is at most %d and the number of classes", kMaxTop);
    const long long ld = row_stride(d->logits_ld, d->classes);
    TCBNN_REQUIRE(ld > 0, "logprobs: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->logits);
    if (d->logprob || d->rank) TCBNN_NOTNULL(d->targets);
    const LogProbsParams p = {d->targets, d->logprob, d->entropy, d->logsumexp, d->top_logprob, d->rank, d->top_index, d->classes,
                              d->top_index || d->top_logprob ? d->top : 0, ld};
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(logprobs_kernel<T>, dim3((unsigned)d->rows), dim3(kThreads), 0, (hipStream_t)stream, (const T*)d->logits, p);
    });
    TCBNN_LAUNCH_CHECK("logprobs_kernel");
    return TCBNN_OK;
}

extern "C" int tcbnn_logprobs_backward(const tcbnn_logprobs_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    TCBNN_REQUIRE(dtype_known(d->dtype), "logprobs: unknown dtype");
    TCBNN_REQUIRE(d->rows >= 0 && d->classes > 0, "logprobs: bad shape");
    const long long x_ld = row_stride(d->logits_ld, d->classes), dx_ld = row_stride(d->grad_logits_ld, d->classes);
    TCBNN_REQUIRE(x_ld > 0 && dx_ld > 0, "logprobs: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->logits);
    TCBNN_NOTNULL(d->logsumexp);
    TCBNN_NOTNULL(d->grad_logits);
    if (d->grad_logprob) TCBNN_NOTNULL(d->targets);
    if (d->grad_entropy) TCBNN_NOTNULL(d->entropy);
    TCBNN_REQUIRE(d->grad_logits != d->logits || d->rows == 1 || x_ld == dx_ld, "logprobs: a gradient over the logits has their stride");
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(logprobs_grad_kernel<T>, dim3((unsigned)d->rows), dim3(kThreads), 0, (hipStream_t)stream,
                           (const T*)d->logits, d->targets, d->logsumexp, d->entropy, d->grad_logprob, d->grad_entropy,
                           (T*)d->grad_logits, d->classes, x_ld, dx_ld);
    });
    TCBNN_LAUNCH_CHECK("logprobs_grad_kernel");
    return TCBNN_OK;
}
