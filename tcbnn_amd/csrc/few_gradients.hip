// The gradients of products of very few rows (kFewGradientRows at most; gated.hip and linear_loss.hip call them):  dx = d w and dw = d^T x for d in fp32,
// kept with the rows of a column side by side ([columns][kFewGradientRows]).
//
// Bound by the weights' bytes and by those of their gradient: both go by once, in one launch.  A wavefront has a chunk of w's rows and 64
// vectors of its columns; a lane keeps its columns of x and its sums of dx in registers and goes down the chunk: a vector of w in, a vector of dw out,
// its values of d from the scalar cache.  fp32 multiply-adds do, 2 for each row and value moved, and d is not rounded, which the matrix instructions would
// ask for.  (With 16 rows they take longer than the matrix instructions: gradients of 16 x 512 -> 2 x 2000 bf16 37 us, 18 with tiles.)
#include "product.h"

namespace tcbnn {
namespace {

using namespace head;

constexpr int kFewThreads = 64, kFewAhead = 4, kFewJoinThreads = 256;

struct FewParams {
    Operand weight, input;
    void *dx, *dw;   // (each NULL where it is not wanted)
    long long dx_ld, dw_ld;
    float* partial;  // [chunks][rows][in], or NULL: one chunk
    int rows, in, outs, blocks, each;  // blocks of columns, rows of w a chunk
};

// M: rows that there are registers for; C: columns of a lane
template <typename T, int M, int C>
__global__ __launch_bounds__(kFewThreads) void few_gradients_kernel(const FewParams p, const float* __restrict__ all_d) {
    const int chunk = blockIdx.x / p.blocks, j = (blockIdx.x % p.blocks * kFewThreads + (int)threadIdx.x) * C, n = min(C, p.in - j);
    if (n <= 0) return;
    float x[M][C], s[M][C];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        Columns<T, C> v = {};
        if (p.dw && i < p.rows) v = get_columns<T, C>(p.input.p, p.input.ld, i, j, n);
#pragma unroll
        for (int c = 0; c < C; ++c) x[i][c] = (float)v[c], s[i][c] = 0.0f;
    }
    const int first = chunk * p.each, last = min(p.outs, first + p.each);
    // (FULL: the lane has all of its columns; rows past the chunk's last one are read as that one)
    auto go = [&](auto full) {
        auto get = [&](int r, Columns<T, C>* w) {
#pragma unroll
            for (int u = 0; u < kFewAhead; ++u) {
                const long long row = min(r + u, last - 1);
                if constexpr (full.value)
                    w[u] = *reinterpret_cast<const ColumnsAnywhere<T, C>*>((const T*)p.weight.p + row * p.weight.ld + j);
                else
                    w[u] = get_columns<T, C>(p.weight.p, p.weight.ld, row, j, n);
            }
        };
        Columns<T, C> w[kFewAhead] = {}, next[kFewAhead] = {};
        if (p.dx) get(first, next);
        for (int r = first; r < last; r += kFewAhead) {
#pragma unroll
            for (int u = 0; u < kFewAhead; ++u) w[u] = next[u];
            if (p.dx) get(r + kFewAhead, next);
#pragma unroll
            for (int u = 0; u < kFewAhead; ++u) {
                if (r + u >= last) break;
                const float* d = all_d + (long long)(r + u) * kFewGradientRows;  // [kFewGradientRows]
                float o[C];
#pragma unroll
                for (int c = 0; c < C; ++c) o[c] = 0.0f;
#pragma unroll
                for (int i = 0; i < M; ++i) {
                    const float f = d[i];
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        s[i][c] = __builtin_fmaf(f, (float)w[u][c], s[i][c]);
                        o[c] = __builtin_fmaf(f, x[i][c], o[c]);
                    }
                }
                if (p.dw) put_columns<T, C>(p.dw, p.dw_ld, r + u, j, full.value ? C : n, o);
            }
        }
    };
    if (n >= C)
        go(std::true_type());
    else
        go(std::false_type());
    if (!p.dx) return;
#pragma unroll
    for (int i = 0; i < M; ++i)
        if (i < p.rows) {
            if (p.partial)
                put_columns<float, C>(p.partial + (long long)chunk * p.rows * p.in, p.in, i, j, n, s[i]);
            else
                put_columns<T, C>(p.dx, p.dx_ld, i, j, n, s[i]);
        }
}

// dx of all chunks, always in the same order: 16 values a workgroup, 16 threads to a value
constexpr int kFewJoined = 16;
template <typename T>
__global__ __launch_bounds__(kFewJoinThreads) void few_join_kernel(const FewParams p, int chunks) {
    constexpr int kStep = kFewJoinThreads / kFewJoined;
    __shared__ float lds[kStep][kFewJoined];
    const int c = threadIdx.x % kFewJoined, part = threadIdx.x / kFewJoined;
    const long long n = (long long)p.rows * p.in, at = (long long)blockIdx.x * kFewJoined + c;
    float s = 0.0f;
    if (at < n)
        for (int k = part; k < chunks; k += 8 * kStep) {
            float v[8];  // (requests of their own, one wait)
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = k + u * kStep < chunks ? p.partial[(k + u * kStep) * n + at] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
    lds[part][c] = s;
    __syncthreads();
    if (part != 0 || at >= n) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < kStep; ++k) s += lds[k][c];
    const long long i = at / p.in;
    ((T*)p.dx)[i * p.dx_ld + (at - i * p.in)] = (T)s;
}

// Chunks of w's rows: 16 wavefronts a compute unit, as long as their sums of dx are no more bytes than w and dw.
inline int few_chunk(int rows, int in, int outs, int size) {
    const int width = kFewThreads * (16 / size), blocks = (in - 1) / width + 1;
    const int most = std::max(1, 16 * kComputeUnits / blocks), least = std::max(8, 4 * rows / size);
    return std::max((outs - 1) / most + 1, least);
}

}  // namespace

namespace head {

size_t few_gradients_bytes(int rows, int in_features, int outs, int dtype) {
    const int each = few_chunk(rows, in_features, outs, (int)dtype_bytes(dtype)), chunks = (outs - 1) / each + 1;
    return chunks > 1 ? (size_t)chunks * rows * in_features * sizeof(float) : 0;
}

int launch_few_gradients(int dtype, const float* d, int rows, int in_features, int outs, const Operand& weight, const Operand& input, void* dx, long long dx_ld,
                         void* dw, long long dw_ld, float* partial, hipStream_t stream) {
    if (!dx && !dw) return TCBNN_OK;
    by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        FewParams p = {weight, input, dx, dw, dx_ld, dw_ld, nullptr, rows, in_features, outs, 0, few_chunk(rows, in_features, outs, (int)sizeof(T))};
        const int chunks = (outs - 1) / p.each + 1;
        p.partial = dx && chunks > 1 ? partial : nullptr;
        p.blocks = (in_features - 1) / (kFewThreads * Elem<T>::kVec) + 1;
        auto go = [&](auto m) {
            constexpr int M = m.value, C = Elem<T>::kVec;
            hipLaunchKernelGGL(HIP_KERNEL_NAME(few_gradients_kernel<T, M, C>), dim3((unsigned)chunks * (unsigned)p.blocks), dim3(kFewThreads), 0, stream, p, d);
        };
        if (rows == 1)
            go(std::integral_constant<int, 1>());
        else
            go(std::integral_constant<int, kFewGradientRows>());
        if (p.partial)
            hipLaunchKernelGGL(few_join_kernel<T>, dim3((unsigned)(((long long)rows * in_features + kFewJoined - 1) / kFewJoined)), dim3(kFewJoinThreads), 0, stream, p, chunks);
    });
    TCBNN_LAUNCH_CHECK("few_gradients_kernel");
    return TCBNN_OK;
}

}  // namespace head
}  // namespace tcbnn
