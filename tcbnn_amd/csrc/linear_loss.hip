// The softmax cross entropy of a linear classifier without its logits (tcbnn_linear_loss_forward / _backward):  z = x w^T + b,
// logsumexp = log sum exp z_j,  loss = logsumexp - z_t;  d_j = dloss (exp(z_j - logsumexp) - [j = t]),  dx = d w,  dw = d^T x,  db = column sums of d.
//
// Forward, a tile of z stays in the registers that its sums end in: what leaves is the largest logit m of a row of the tile and the sum of
// exp(z - m), 8 bytes for a tile's width of logits, and z_t from the one lane that has it.  A second launch joins them.
// Backward, z is made again, a piece of the classes at a time, and becomes d where it lies; d goes to the workspace in the operands' type and from
// there through two products.  dx is summed over the pieces in fp32.  With pieces of kPieceBytes that are read back from the cache, four products
// (8 rows classes inputs operations a step) are nearly all of the time: 8192 x 1024 -> 131072 bf16 7.9 to 8.6 ms from card to card, in the former z 1.84 (1.20 PFLOP/s), d 2.35, dx 1.93, dw
// 1.86.  Single rows are bound by the weights' bytes, 1 x 4096 -> 131072 173 us (6.2 TB/s); small steps by their launches one after
// the other, 256 x 512 -> 1000 fp32 37 us; weights' gradients of few rows by what they write, 333 x 1000 -> 32003 f16 42 us of the step's 174 to 191.
#include "product.h"

namespace tcbnn {
namespace {

using namespace head;

struct LossParams {
    const int32_t* targets;
    float2* parts;          // [parts][rows_there] largest logit, sum of exponentials about it
    float* given;           // [rows] z_t
    long long rows_there;
    int first;              // the first class of the call
};
struct LossGradParams {
    const int32_t* targets;
    const float *lse, *dloss, *scale;  // (scale: of d in f16)
    const float *loss, *rest;          // [rows] each, or NULL (rest: what fp32 left of lse)
    float* sums;                       // [tiles of i][cols], or NULL
    int first, classes;                // the piece's first class
    long long low;                     // elements from d to what its rounding left of it, or 0
};

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// Up to it exponents of a row are taken about m log2 e, rounded: one fused multiply-add a logit, and what the rounding was (2^-8 at most) scales the
// sum back.  Beyond, that would be any number of powers of two, inf or 0 from 2^31 on, and nothing at all where m log2 e has no place in fp32 (a mask of the
// type's lowest value): there logits' differences to m are taken first, which are exact beside m.
constexpr float kNear = 65536.0f;
// exp(m - to) s: what a sum of exponentials about m is about `to`, m <= to
__device__ __forceinline__ float about(float m, float s, float to) { return m == to ? s : s * exp_fast(m - to); }
// f(v, v of the lane 32 away)
template <typename F>
__device__ __forceinline__ float across_halves(float v, F f) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float((uint32_t)a[0]), __uint_as_float((uint32_t)a[1]));
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }

// bias added to a wavefront's sums; what lies past the last column is -inf.  Register v of lane l is column 8 (v / 4) + 4 (l / 32) + v % 4 of a piece of 32.
template <int NI, int NJ>
__device__ __forceinline__ void add_bias(Acc (&acc)[NI][NJ], const ProductParams& p, long long j0, int lane) {
#pragma unroll
    for (int b = 0; b < NJ; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const long long j = j0 + 32 * b + 8 * q + 4 * (lane >> 5);
            if (p.bias) {
                const Columns<float, 4> c = get_columns<float, 4>(p.bias, 0, 0, (int)j, (int)min(4LL, p.cols - j));
#pragma unroll
                for (int a = 0; a < NI; ++a)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][b][4 * q + e] += c[e];
            }
            if (j0 + 32 * NJ > p.cols) {
#pragma unroll
                for (int a = 0; a < NI; ++a)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][b][4 * q + e] = j + e < p.cols ? acc[a][b][4 * q + e] : -INFINITY;
            }
        }
}

template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG>
__global__ __launch_bounds__(64 * WI * WJ * WS) __attribute__((amdgpu_waves_per_eu(short_waves(WI * WJ * WS, STAGES)))) void loss_product_kernel(const ProductParams p, const LossParams l) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass leaves a kernel's stub out where it instantiates a tile's requests twice)
    __shared__ __align__(1024) char lds[product_lds<BI, BJ, WI, WJ, WS, STAGES>()];
    constexpr int NI = BI / WI / 32, NJ = BJ / WJ / 32;
    Acc acc[NI][NJ];
    Spot spot;
    product_sums<T, BI, BJ, WI, WJ, WS, STAGES, ACCESS, HOLD, LONG, false, false>(p, blockIdx.x, lds, acc, spot);
    join_shares<WI, WJ, WS>(acc, lds, spot);
    float2* rows = reinterpret_cast<float2*>(lds);  // [WJ][BI]
    if (spot.share == 0) {
        const long long j0 = spot.j0 + spot.wj;
        add_bias(acc, p, j0, spot.lane);
#pragma unroll
        for (int a = 0; a < NI; ++a) {
            const int row = spot.wi + 32 * a + (spot.lane & 31);
            float m = -INFINITY, s = 0.0f;
#pragma unroll
            for (int b = 0; b < NJ; ++b)
#pragma unroll
                for (int v = 0; v < 16; ++v) m = fmaxf(m, acc[a][b][v]);
            m = across_halves(m, larger);
            const float base = m == -INFINITY ? 0.0f : m, c = base * kLog2e;
#pragma unroll
            for (int b = 0; b < NJ; ++b)
#pragma unroll
                for (int v = 0; v < 16; ++v) s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[a][b][v], kLog2e, -c));
            s = across_halves(s, add) * __builtin_amdgcn_exp2f(-__builtin_fmaf(base, kLog2e, -c));
            if (__any(fabsf(base) > kNear)) {
                float far = 0.0f;
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v) far += exp_fast(acc[a][b][v] - base);
                far = across_halves(far, add);
                s = fabsf(base) > kNear ? far : s;
            }
            if (spot.lane < 32) rows[spot.wj / (32 * NJ) * BI + row] = make_float2(m, s);
            const long long i = spot.i0 + row;
            const long long t = l.targets && i < p.rows ? (long long)l.targets[i] - l.first - j0 : -1;
            if (__any(t >= 0 && t < 32 * NJ && t + j0 < p.cols)) {
                const int at = (int)(t - 4 * (spot.lane >> 5));
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (t >= 0 && t + j0 < p.cols && at == 32 * b + 8 * (v / 4) + v % 4) l.given[i] = acc[a][b][v];
            }
        }
    }
    __syncthreads();
    for (int row = threadIdx.x; row < BI; row += 64 * WI * WJ * WS) {
        float2 r = rows[row];
#pragma unroll
        for (int w = 1; w < WJ; ++w) {
            const float2 o = rows[w * BI + row];
            const float m = fmaxf(r.x, o.x);
            r = make_float2(m, about(r.x, r.y, m) + about(o.x, o.y, m));
        }
        if (spot.i0 + row < p.rows) l.parts[spot.tile_j * l.rows_there + spot.i0 + row] = r;
    }
#endif
}

// few rows: a wavefront's 16 classes are a part
template <typename T, int SHARES>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(2, 4))) void loss_few_rows_kernel(const ProductParams p, const LossParams l) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = wave % SHARES;
    const long long part = p.first / kFewOutputs + (long long)blockIdx.x * (kFewWaves / SHARES) + wave / SHARES, j0 = part * kFewOutputs;
    // rows past the last one are read as the last one; nothing of them is kept
    const T* w = (const T*)p.j.p + min(j0 + (lane & 15), (long long)p.cols - 1) * p.j.ld;
    const T* x = (const T*)p.i.p + (long long)min(lane & 15, p.rows - 1) * p.i.ld;
    Acc4 acc = few_rows_sums<T, SHARES>(p, w, x);
    if (share != 0 || j0 >= p.cols) return;
    const int i = lane & 15;
    const long long j = j0 + 4 * (lane >> 4);
    const int t = l.targets && i < p.rows ? l.targets[i] : -1;
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        acc[e] = j + e < p.cols ? acc[e] + (p.bias ? p.bias[j + e] : 0.0f) : -INFINITY;
        if (j + e == t && j + e < p.cols) l.given[i] = acc[e];
        m = fmaxf(m, acc[e]);
    }
    m = __uint_as_float(across_rows(__float_as_uint(m), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
    const float c = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += exp_fast(acc[e] - c);
    s = __uint_as_float(across_rows(__float_as_uint(s), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
    if (lane < 16 && i < p.rows) l.parts[part * l.rows_there + i] = make_float2(m, s);
}

// a + b = (float)(a + b) + what this gives (Knuth's sum of two)
__device__ __forceinline__ float rest_of_sum(float a, float b) {
    const float sum = a + b, of_b = sum - a;
    return (a - (sum - of_b)) + (b - of_b);
}

// A row's parts joined, always in the same order: R rows a workgroup side by side, 1024 / R threads to a row.
constexpr int kLossJoinThreads = 1024;
template <int R>
__global__ __launch_bounds__(kLossJoinThreads) void loss_join_kernel(const LossParams l, float* __restrict__ loss, float* __restrict__ lse,
                                                                     float* __restrict__ rest, int rows, int classes, int parts) {
    constexpr int kStep = kLossJoinThreads / R, kWaves = kLossJoinThreads / 64;
    static_assert(R == 1 || R == 32, "");
    __shared__ float2 lds[kWaves][R];
    const int r = threadIdx.x % R, first = threadIdx.x / R;
    for (long long row0 = (long long)blockIdx.x * R; row0 < rows; row0 += (long long)gridDim.x * R) {
        const long long row = min(row0 + r, (long long)rows - 1);
        float m = -INFINITY, s = 0.0f;
        for (int k = first; k < parts; k += 4 * kStep) {
            float2 v[4];  // (requests of their own, one wait)
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = k + u * kStep < parts ? l.parts[(long long)(k + u * kStep) * l.rows_there + row] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float to = fmaxf(m, v[u].x);
                s = about(m, s, to) + about(v[u].x, v[u].y, to);
                m = to;
            }
        }
        const float to = R == 1 ? wave_max(m) : across_halves(m, larger);
        s = about(m, s, to);
        s = R == 1 ? wave_sum(s) : across_halves(s, add);
        if ((threadIdx.x & 63) < R) lds[threadIdx.x >> 6][r] = make_float2(to, s);
        __syncthreads();
        if (first == 0 && row0 + r < rows) {
            m = -INFINITY;
            s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds[w][r].x);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) s += about(lds[w][r].x, lds[w][r].y, m);
            const float log_s = logf(s);
            const bool none = m == -INFINITY && s == 0.0f;  // every class is forbidden
            if (lse) lse[row] = none ? -INFINITY : m + log_s;
            if (rest) {
                const float r = rest_of_sum(m, log_s);
                rest[row] = fabsf(r) < INFINITY ? r : 0.0f;
            }
            if (loss) {
                const int t = l.targets[row];
                loss[row] = t < 0 ? 0.0f : t >= classes ? NAN : none ? INFINITY : (m - l.given[row]) + log_s;
            }
        }
        __syncthreads();
    }
}

// ---- gradient
// A power of two that brings the largest |dloss| to 2^14 .. 2^15: d is no larger, and what is 2^-28 of it is still a normal number in f16.
// scale[0] is the factor, scale[1] its inverse.
constexpr int kScaleThreads = 1024;
__global__ __launch_bounds__(kScaleThreads) void loss_scale_kernel(const float* __restrict__ dloss, const int32_t* __restrict__ targets, float* __restrict__ scale, int rows) {
    __shared__ float lds[kScaleThreads / 64];
    float m = 0.0f;
    for (long long i = threadIdx.x; i < rows; i += kScaleThreads) {
        const float g = fabsf(dloss[i]);
        if (targets[i] >= 0 && g < INFINITY) m = fmaxf(m, g);
    }
    m = wave_max(m);
    lds[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kScaleThreads / 64; ++w) m = fmaxf(m, lds[w]);
        const int e = m > 0.0f ? min(14 - ilogbf(m), 120) : 0;
        scale[0] = ldexpf(1.0f, e);
        scale[1] = ldexpf(1.0f, -e);
    }
}

// exp(z - logsumexp) of a row's logits, logsumexp = lse + rest, as `factor` times near(z), or beyond(z) where lse is beyond kNear.  About c, lse log2 e as it is
// rounded, it is one fused multiply-add a logit; the factor is what that rounding and the rest make of it.
struct RowExp {
    float lse, rest, c, factor;
    bool far;
    __device__ __forceinline__ RowExp(float lse, float rest) : lse(lse), rest(rest), c(lse * kLog2e), far(fabsf(lse) > kNear) {
        factor = far ? 1.0f : __builtin_amdgcn_exp2f(-__builtin_fmaf(rest, kLog2e, __builtin_fmaf(lse, kLog2e, -c)));
    }
    __device__ __forceinline__ float near(float z) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, -c)); }
    // (no more than 1: the logit is made again, perhaps in another order, and so far from 0 one unit of it may be any number of powers of e; NaN stays)
    __device__ __forceinline__ float beyond(float z) const {
        const float d = (z - lse) - rest;
        return exp_fast(d > 0.0f ? 0.0f : d);
    }
};

// exp(-loss) - 1: what the given class' p - 1 is, good where p is near 1 too
__device__ __forceinline__ float given_d(float loss) {
    const float x = -loss;
    const float near = x * __builtin_fmaf(x, __builtin_fmaf(x, __builtin_fmaf(x, __builtin_fmaf(x, __builtin_fmaf(x, 1.0f / 720, 1.0f / 120), 1.0f / 24), 1.0f / 6), 0.5f), 1.0f);
    return x > -0.25f ? near : exp_fast(x) - 1.0f;
}

// the sum over the 32 lanes of a half, in the lanes whose number ends in 0
__device__ __forceinline__ float half_sum(float v) {
    v += __uint_as_float(dpp<kSwapPairs>(__float_as_uint(v)));
    v += __uint_as_float(dpp<kSwapTwos>(__float_as_uint(v)));
    v += __uint_as_float(dpp<kMirrorHalf>(__float_as_uint(v)));
    v += __uint_as_float(dpp<kMirrorRow>(__float_as_uint(v)));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((uint32_t)a[0]) + __uint_as_float((uint32_t)a[1]);
}

// d of a piece of the classes: p.out [rows][out_ld], the columns behind the last one of 16 bytes 0
template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG>
__global__ __launch_bounds__(64 * WI * WJ * WS) __attribute__((amdgpu_waves_per_eu(short_waves(WI * WJ * WS, STAGES)))) void loss_grad_product_kernel(const ProductParams p, const LossGradParams l) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass leaves a kernel's stub out where it instantiates a tile's requests twice)
    __shared__ __align__(1024) char lds[product_lds<BI, BJ, WI, WJ, WS, STAGES>()];
    constexpr int NI = BI / WI / 32, NJ = BJ / WJ / 32, V = Elem<T>::kVec, kThreads = 64 * WI * WJ * WS;
    constexpr int kOutRow = 32 * NJ * 4 + 16, kOutWave = 32 * kOutRow;
    Acc acc[NI][NJ];
    Spot spot;
    product_sums<T, BI, BJ, WI, WJ, WS, STAGES, ACCESS, HOLD, LONG, false, false>(p, blockIdx.x, lds, acc, spot);
    join_shares<WI, WJ, WS>(acc, lds, spot);
    const int lane = spot.lane;
    const long long j0 = spot.j0 + spot.wj;
    if (spot.share == 0) {
        add_bias(acc, p, j0, lane);
#pragma unroll
        for (int a = 0; a < NI; ++a) {
            const long long i = spot.i0 + spot.wi + 32 * a + (lane & 31), row = min(i, (long long)p.rows - 1);
            const int t = l.targets[row];
            const float lse = l.lse[row];
            const bool none = i >= p.rows || t < 0 || lse == -INFINITY;
            const float g = t < l.classes ? l.dloss[row] : NAN;
            const RowExp e(lse, l.rest ? l.rest[row] : 0.0f);
            const float gf = g * e.factor;
            if (__any(e.far)) {
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[a][b][v] = gf * (e.far ? e.beyond(acc[a][b][v]) : e.near(acc[a][b][v]));
            } else {
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[a][b][v] = gf * e.near(acc[a][b][v]);
            }
            if (__any(none)) {
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[a][b][v] = none ? 0.0f : acc[a][b][v];
            }
            const long long at = (long long)t - l.first - j0 - 4 * (lane >> 5);
            if (__any(!none && at >= 0 && at < 32 * NJ)) {
                const float given = l.loss ? g * given_d(l.loss[row]) : 0.0f;
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (!none && at == 32 * b + 8 * (v / 4) + v % 4) acc[a][b][v] = l.loss ? given : acc[a][b][v] - g;
            }
        }
    }
    if (l.sums) {
        float* columns = reinterpret_cast<float*>(lds);  // [WI][BJ]
        if (spot.share == 0) {
#pragma unroll
            for (int b = 0; b < NJ; ++b)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float s[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[e] = acc[0][b][4 * q + e];
#pragma unroll
                        for (int a = 1; a < NI; ++a) s[e] += acc[a][b][4 * q + e];
                        s[e] = half_sum(s[e]);
                    }
                    if ((lane & 31) == 0)
                        *reinterpret_cast<float4*>(columns + spot.wi / (32 * NI) * BJ + spot.wj + 32 * b + 8 * q + 4 * (lane >> 5)) = make_float4(s[0], s[1], s[2], s[3]);
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < BJ; c += kThreads) {
            float s = columns[c];
#pragma unroll
            for (int w = 1; w < WI; ++w) s += columns[w * BJ + c];
            if (spot.j0 + c < p.cols) l.sums[(long long)spot.tile_i * p.cols + spot.j0 + c] = s;
        }
        __syncthreads();
    }
    if (spot.share != 0) return;
    // ---- out: 32 rows of the wavefront at a time through LDS, so that a row leaves in whole runs of 64 bytes or more
    char* mine = lds + spot.wave * kOutWave;
    constexpr int kPerRow = 32 * NJ / V, kRowsAtOnce = 64 / kPerRow < 32 ? 64 / kPerRow : 32, kTimes = 32 / kRowsAtOnce;
    const int col = (lane % kPerRow) * V, row0 = lane / kPerRow % kRowsAtOnce;
    const long long j = j0 + col;
    const float scale = l.scale ? l.scale[0] : 1.0f;
    const bool there = j < p.cols && lane / kPerRow < kRowsAtOnce;
#pragma unroll 1
    for (int a = 0; a < NI; ++a) {
        const long long first = spot.i0 + spot.wi + 32 * a + row0;
#pragma unroll
        for (int k = 0; k < NI; ++k)  // (registers have no index: one of NI pieces of code)
            if (k == a) {
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<float4*>(mine + (lane & 31) * kOutRow + (32 * b + 8 * q + 4 * (lane >> 5)) * 4) =
                            make_float4(acc[k][b][4 * q], acc[k][b][4 * q + 1], acc[k][b][4 * q + 2], acc[k][b][4 * q + 3]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int r = 0; r < kTimes; ++r) {
            const long long i = first + r * kRowsAtOnce;
            const char* from = mine + (row0 + r * kRowsAtOnce) * kOutRow + col * 4;
            Vec<T> d;
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 q = *reinterpret_cast<const float4*>(from + e * 4);
                d[e] = (T)(q.x * scale), d[e + 1] = (T)(q.y * scale), d[e + 2] = (T)(q.z * scale), d[e + 3] = (T)(q.w * scale);
            }
            if (j + V > p.cols) {
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = j + e < p.cols ? d[e] : (T)0.0f;
            }
            if (there && i < p.rows) *reinterpret_cast<Vec<T>*>((T*)p.out + i * p.out_ld + j) = d;  // (rows of whole 16 bytes)
            if (l.low) {
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = j + e < p.cols ? (T)(*reinterpret_cast<const float*>(from + e * 4) * scale - (float)d[e]) : (T)0.0f;
                if (there && i < p.rows) *reinterpret_cast<Vec<T>*>((T*)p.out + l.low + i * p.out_ld + j) = d;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#endif
}

// few rows: a wavefront has 16 classes.  p.out: d in T as above, or (FLOAT) in fp32 as launch_few_gradients takes it
template <typename T, int SHARES, bool FLOAT>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(2, 4))) void loss_grad_few_rows_kernel(const ProductParams p, const LossGradParams l) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = wave % SHARES;
    const long long j0 = p.first + ((long long)blockIdx.x * (kFewWaves / SHARES) + wave / SHARES) * kFewOutputs;
    // rows past the last one are read as the last one; nothing of them is kept
    const T* w = (const T*)p.j.p + min(j0 + (lane & 15), (long long)p.cols - 1) * p.j.ld;
    const T* x = (const T*)p.i.p + (long long)min(lane & 15, p.rows - 1) * p.i.ld;
    const Acc4 acc = few_rows_sums<T, SHARES>(p, w, x);
    if (share != 0 || j0 >= p.cols) return;
    const int i = lane & 15, row = min(i, p.rows - 1), t = l.targets[row];
    const long long j = j0 + 4 * (lane >> 4);
    const float lse = l.lse[row], g = t < l.classes ? l.dloss[row] : NAN;
    const RowExp of(lse, l.rest ? l.rest[row] : 0.0f);
    const bool none = i >= p.rows || t < 0 || lse == -INFINITY;
    const float given = l.loss ? g * given_d(l.loss[row]) : 0.0f;
    float d[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool there = j + e < p.cols;
        const float z = acc[e] + (p.bias && there ? p.bias[j + e] : 0.0f);
        d[e] = g * of.factor * (of.far ? of.beyond(z) : of.near(z));
        d[e] = none || !there ? 0.0f : l.first + j + e == t ? (l.loss ? given : d[e] - g) : d[e];
        if (l.sums) {
            float s = d[e];
            s += __uint_as_float(dpp<kSwapPairs>(__float_as_uint(s)));
            s += __uint_as_float(dpp<kSwapTwos>(__float_as_uint(s)));
            s += __uint_as_float(dpp<kMirrorHalf>(__float_as_uint(s)));
            s += __uint_as_float(dpp<kMirrorRow>(__float_as_uint(s)));
            if (i == 0 && there) l.sums[j + e] = s;
        }
    }
    if constexpr (FLOAT) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i < kFewGradientRows && j + e < p.cols) ((float*)p.out)[(j + e) * kFewGradientRows + i] = d[e];
    } else {
        if (i >= p.rows || j >= p.out_ld) return;  // (rows end at whole 16 bytes: where they go on, four columns do)
        const float f = l.scale ? l.scale[0] : 1.0f;
        Columns<T, 4> v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(d[e] * f);
        T* to = (T*)p.out + i * p.out_ld + j;
        *reinterpret_cast<Columns<T, 4>*>(to) = v;
        if (l.low) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(d[e] * f - (float)v[e]);
            *reinterpret_cast<Columns<T, 4>*>(to + l.low) = v;
        }
    }
}
template <typename T, bool FLOAT>
void launch_grad_few_rows(const ProductParams& p, const LossGradParams& l, hipStream_t stream) {
    const int shares = few_shares(p.cols, p.sum, (int)sizeof(T));
    by_few_columns(p, shares, kFewOutputs * kFewWaves / shares, [&](auto s, dim3 grid, const ProductParams& q) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(loss_grad_few_rows_kernel<T, s.value, FLOAT>), grid, dim3(64 * kFewWaves), 0, stream, q, l);
    });
}

// ---- plans
// rows and columns of a tile (by_tile)
inline int cut_size(Access access, Cut cut, bool brief) { return brief ? 128 : access == ELEMENTS ? 32 : (access == WHOLE_PIECES ? kCuts16 : kCutsAnywhere)[cut].size; }
// The forward call's kernel: its tile, or the one for few rows; the number of parts that it leaves of a row.
struct LossPlan {
    Access access;
    Plan plan;
    bool few, brief;
    int parts;
    bool pack_x, pack_w;
};
inline LossPlan plan_loss(int rows, int classes, int sum, int size, Access access) {
    const bool vectors = access == WHOLE_PIECES;
    LossPlan l = {};
    l.access = access;
    l.plan = plan_product(rows, classes, sum, size, vectors, 0, CUT_256, true);
    l.few = rows <= kFewRows && (access == ELEMENTS || few_time(rows, classes, sum, size, vectors) < l.plan.time);
    l.brief = !l.few && short_sum(access, rows, classes, sum, size);
    const int width = l.few ? kFewOutputs : cut_size(access, l.plan.cut, l.brief);
    l.parts = (classes - 1) / width + 1;
    return l;
}
// ... with operands that lie anywhere copied where that and the product of the copies are estimated to take less time
inline LossPlan plan_loss(int rows, int classes, int sum, int size, Access access, bool x_anywhere, bool w_anywhere, bool copies_fit) {
    const LossPlan l = plan_loss(rows, classes, sum, size, access);
    if (l.few || access != ANYWHERE || !copies_fit) return l;
    LossPlan whole = plan_loss(rows, classes, sum, size, WHOLE_PIECES);
    const float copies = (x_anywhere ? pack_time(packed_bytes(rows, sum, size)) : 0.0f) + (w_anywhere ? pack_time(packed_bytes(classes, sum, size)) : 0.0f);
    if (whole.few || whole.plan.time + copies >= l.plan.time) return l;
    whole.pack_x = x_anywhere;
    whole.pack_w = w_anywhere;
    return whole;
}

// A piece of the classes whose d is in the workspace at a time: as many as kPieceBytes hold, pieces of about the same size (half and a quarter of it
// are slower, twice and four times no faster).
constexpr size_t kPieceBytes = (size_t)256 << 20;
constexpr int kPieceUnit = 256;
inline int piece_classes(int rows, int classes, int size) {
    const long long most = std::max<long long>(kPieceUnit, (long long)(kPieceBytes / ((size_t)rows * size)) / kPieceUnit * kPieceUnit);
    if (classes <= most) return classes;
    const long long pieces = (classes + most - 1) / most;
    return (int)(((classes + pieces - 1) / pieces + kPieceUnit - 1) / kPieceUnit * kPieceUnit);
}
// classes whose weights are copied at a time
inline int packed_classes(int classes, int in_features, int size) {
    const long long most = std::max<long long>(kPieceUnit, (long long)(kPieceBytes / (packed_ld(in_features, size) * size)) / kPieceUnit * kPieceUnit);
    return (int)std::min<long long>(classes, most);
}
// The splits of dx's sum over a whole piece, where there are several.  Where the weights lie is not known when a workspace is asked for: the splits are
// those of rows at whole 16 bytes, which are no fewer.
inline int carried_splits(int rows, int in_features, int piece, int size) {
    const int splits = plan_product(rows, in_features, piece, size, true, ~(size_t)0, CUT_256, true).splits;
    const int steps = (int)(((long long)piece * size + kStepBytes - 1) / kStepBytes), each = (steps + splits - 1) / splits;
    return (steps + each - 1) / each;  // (as cut_product cuts a whole piece: every part is written by the first)
}

// In 16 bits d is rounded before it is multiplied.  A row of d, and a column, is often little else than its given class' value, whose rounding then is that
// of all that it is multiplied with.  Over many rows these errors, like those of the sums' other terms, come to sqrt 2 of what rounding the results
// leaves (8192 rows bf16: 0.0024 of them, 0.0017 the rounding); few rows may be off by twice that.  Up to kTwoPlaneRows rows d is kept in
// two planes, its rounding and what that left, and both products sum over both.
constexpr int kTwoPlaneRows = 256;
inline bool two_planes(int rows, int dtype) { return dtype != TCBNN_F32 && rows <= kTwoPlaneRows; }
// where the second plane of a sum of n begins: whole steps
inline int plane_of(int n, int size) { return (n + kStepBytes / size - 1) / (kStepBytes / size) * (kStepBytes / size); }

// Which of a step's operands to copy (linear_loss_backward's three products a piece), where they lie anywhere.
struct LossPacking {
    bool x, w;
};
inline LossPacking loss_packing(int rows, int in_features, int piece, int classes, int size, bool planes, bool x_anywhere, bool w_anywhere) {
    if (in_features * size < 16) return {false, false};
    const int pieces = (classes - 1) / piece + 1;
    auto time = [&](int i, int j, int sum, bool whole) { return plan_product(i, j, sum, size, whole, 0).time; };
    LossPacking best = {false, false};
    float best_time = 0.0f;
    for (bool x : {false, true})
        for (bool w : {false, true}) {
            if ((x && !x_anywhere) || (w && !w_anywhere)) continue;
            const bool x_whole = x || !x_anywhere, w_whole = w || !w_anywhere;
            const float each = time(rows, piece, in_features, x_whole && w_whole) + time(rows, in_features, planes ? plane_of(piece, size) + piece : piece, w_whole) +
                               time(piece, in_features, planes ? plane_of(rows, size) + rows : rows, x_whole) +
                               (w ? pack_time(packed_bytes(piece, in_features, size)) : 0.0f);
            const float total = (float)pieces * each + (x ? pack_time(packed_bytes(rows, in_features, size)) : 0.0f);
            if (best_time == 0.0f || total < best_time) best = {x, w}, best_time = total;
        }
    return best;
}

struct LossWorkspace {
    size_t scale, x, w, d, sums, dx, split, total;  // offsets, in order
    int piece, splits;
};
inline LossWorkspace loss_workspace(int rows, int in_features, int classes, int dtype, bool anywhere) {
    const int size = (int)dtype_bytes(dtype), planes = two_planes(rows, dtype) ? 2 : 1;
    LossWorkspace w = {};
    if (rows <= kFewGradientRows) {
        w.piece = classes;
        w.split = whole_lines((size_t)classes * kFewGradientRows * sizeof(float));
        w.total = w.split + few_gradients_bytes(rows, in_features, classes, dtype);
        return w;
    }
    w.piece = piece_classes(rows * planes, classes, size);
    const bool carried = w.piece < classes;
    w.splits = carried ? carried_splits(rows, in_features, (planes - 1) * plane_of(w.piece, size) + w.piece, size) : 1;
    bool pack_x = false, pack_w = false;
    for (bool x : {false, anywhere})  // (which of the operands is not known here)
        for (bool v : {false, anywhere}) {
            const LossPacking packing = loss_packing(rows, in_features, w.piece, classes, size, planes > 1, x, v);
            pack_x |= packing.x;
            pack_w |= packing.w;
        }
    w.x = 256;
    w.w = w.x + (pack_x ? packed_bytes(rows, in_features, size) : 0);
    w.d = w.w + (pack_w ? packed_bytes(w.piece, in_features, size) : 0);
    w.sums = w.d + packed_bytes((long long)rows * planes, w.piece, size);
    w.dx = w.sums + whole_lines((size_t)((rows + 31) / 32) * w.piece * sizeof(float));
    w.split = w.dx + (carried ? whole_lines((size_t)w.splits * rows * in_features * sizeof(float)) : 0);
    w.total = w.split + std::max(gradient_product_bytes(rows, in_features, planes > 1 ? plane_of(w.piece, size) + w.piece : w.piece, dtype, true),
                                 gradient_product_bytes(planes > 1 ? plane_of(rows, size) + rows : rows, in_features, w.piece, dtype, true));
    return w;
}

int check_loss(int rows, int in_features, int classes, int dtype) {
    TCBNN_REQUIRE(dtype_known(dtype), "linear loss: unknown dtype");
    TCBNN_REQUIRE(rows >= 0 && in_features > 0 && classes > 0, "linear loss: bad shape");
    TCBNN_REQUIRE(rows <= kMaxRows, "linear loss: at most %d rows", kMaxRows);
    TCBNN_REQUIRE(in_features <= kMaxIn, "linear loss: at most %d inputs", kMaxIn);
    TCBNN_REQUIRE(classes <= kMaxOut, "linear loss: at most %d classes", kMaxOut);
    return TCBNN_OK;
}
// rows that are so far apart that 32 bits do not hold a tile
bool too_far(long long ld, int dtype) { return ld * 256 * (long long)dtype_bytes(dtype) > 0x7fffffffLL; }

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

// what a forward call needs, with room for copies or without
static size_t loss_forward_bytes(int rows, int in_features, int classes, int dtype, bool room) {
    const int size = (int)dtype_bytes(dtype);
    size_t parts = 0, copies = 0;
    for (bool x : {false, true})  // (which of the operands is not known here; parts are there for rows that lie anywhere in any case)
        for (bool w : {false, true}) {
            const LossPlan l = plan_loss(rows, classes, in_features, size, in_features * size < 16 ? ELEMENTS : x || w ? ANYWHERE : WHOLE_PIECES, x, w, room);
            parts = std::max(parts, (size_t)l.parts);
            copies = std::max(copies, (l.pack_x ? packed_bytes(rows, in_features, size) : 0) +
                                          (l.pack_w ? packed_bytes(packed_classes(classes, in_features, size), in_features, size) : 0));
        }
    return copies + whole_lines(parts * rows * sizeof(float2)) + whole_lines((size_t)rows * sizeof(float));
}
extern "C" size_t tcbnn_linear_loss_workspace_bytes(int rows, int in_features, int classes, int dtype, int anywhere) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || in_features > kMaxIn || classes <= 0 || classes > kMaxOut || !dtype_known(dtype)) return 0;
    // (no less with room for copies: these are multiplied in wider tiles, which leave fewer parts, and every call asks for the size without)
    const size_t without = loss_forward_bytes(rows, in_features, classes, dtype, false);
    return anywhere ? std::max(without, loss_forward_bytes(rows, in_features, classes, dtype, true)) : without;
}

extern "C" int tcbnn_linear_loss_forward(const tcbnn_linear_loss_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_loss(d->rows, d->in_features, d->classes, d->dtype)) return rc;
    ProductParams p = {};
    p.i = {d->input, row_stride(d->input_ld, d->in_features)};
    p.j = {d->weight, row_stride(d->weight_ld, d->in_features)};
    TCBNN_REQUIRE(p.i.ld > 0 && p.j.ld > 0, "linear loss: rows overlap");
    TCBNN_REQUIRE(!too_far(p.i.ld, d->dtype) && !too_far(p.j.ld, d->dtype), "linear loss: rows too far apart");
    if (d->rows == 0 || (!d->loss && !d->logsumexp && !d->logsumexp_rest)) return TCBNN_OK;
    TCBNN_NOTNULL(d->input);
    TCBNN_NOTNULL(d->weight);
    if (d->loss) TCBNN_NOTNULL(d->targets);
    TCBNN_NOTNULL(d->workspace);
    TCBNN_REQUIRE((uintptr_t)d->workspace % 16 == 0, "linear loss: the workspace is not aligned to 16 bytes");
    TCBNN_REQUIRE(d->workspace_bytes >= tcbnn_linear_loss_workspace_bytes(d->rows, d->in_features, d->classes, d->dtype, 0), "linear loss: workspace too small");
    const bool copies = d->workspace_bytes >= tcbnn_linear_loss_workspace_bytes(d->rows, d->in_features, d->classes, d->dtype, 1);
    p.rows = d->rows;
    p.cols = d->classes;
    p.sum = d->in_features;
    p.bias = d->bias;
    hipStream_t s = (hipStream_t)stream;
    return by_dtype(d->dtype, [&](auto type) -> int {
        using T = decltype(type);
        const LossPlan plan = plan_loss(p.rows, p.cols, p.sum, (int)sizeof(T), access_of<T, false, false>(p), lies_anywhere<T>(p.i, p.sum), lies_anywhere<T>(p.j, p.sum),
                                        copies);
        char* at = (char*)d->workspace;
        if (plan.pack_x) {
            p.i = launch_pack(d->dtype, p.i, p.rows, p.sum, at, s);
            p.padded_i = true;
            at += packed_bytes(p.rows, p.sum, (int)sizeof(T));
        }
        char* copy = at;
        const int piece = plan.pack_w ? packed_classes(p.cols, p.sum, (int)sizeof(T)) : p.cols;
        if (plan.pack_w) at += packed_bytes(piece, p.sum, (int)sizeof(T));
        LossParams l = {d->loss ? d->targets : nullptr, (float2*)at, (float*)(at + whole_lines((size_t)plan.parts * p.rows * sizeof(float2))), p.rows, 0};
        if (plan.few) {
            const int shares = few_shares(p.cols, p.sum, (int)sizeof(T));
            by_few_columns(p, shares, kFewOutputs * kFewWaves / shares, [&](auto n, dim3 grid, const ProductParams& q) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(loss_few_rows_kernel<T, n.value>), grid, dim3(64 * kFewWaves), 0, s, q, l);
            });
        } else {
            by_tile(plan.access, plan.plan.cut, plan.brief, [&](auto size, auto wi, auto wj, auto ws, auto stages, auto how, auto hold, auto keep) {
                constexpr int B = size.value, kThreads = 64 * wi.value * wj.value * ws.value;
                // rows beyond a launch's threads have one of their own
                const long long at_once = std::max(1LL, kMaxThreads / kThreads / plan.parts) * B;
                for (int c = 0; c < p.cols; c += piece) {
                    ProductParams r = p;
                    r.cols = std::min(piece, p.cols - c);
                    r.j.p = (const T*)p.j.p + c * p.j.ld;
                    r.bias = p.bias ? p.bias + c : nullptr;
                    if (plan.pack_w) r.j = launch_pack(d->dtype, r.j, r.cols, r.sum, copy, s);
                    r.padded_j = plan.pack_w;
                    for (long long first = 0; first < p.rows; first += at_once) {
                        ProductParams q = r;
                        LossParams part = l;
                        q.rows = (int)std::min(at_once, p.rows - first);
                        q.i.p = (const T*)p.i.p + first * p.i.ld;
                        part.targets = l.targets ? l.targets + first : nullptr;
                        part.parts += first + c / B * l.rows_there;  // (a piece is whole tiles)
                        part.given += first;
                        part.first = c;
                        cut_product(q, B, kStepBytes / (int)sizeof(T), 1, nullptr);
                        hipLaunchKernelGGL(HIP_KERNEL_NAME(loss_product_kernel<T, B, B, wi.value, wj.value, ws.value, stages.value, how.value, hold.value, keep.value>),
                                           dim3((unsigned)((long long)q.tiles_i * q.tiles_j)), dim3(kThreads), 0, s, q, part);
                    }
                }
            });
        }
        TCBNN_LAUNCH_CHECK("loss_product_kernel");
        if (p.rows <= kFewRows)
            hipLaunchKernelGGL(loss_join_kernel<1>, dim3((unsigned)p.rows), dim3(kLossJoinThreads), 0, s, l, d->loss, d->logsumexp, d->logsumexp_rest, p.rows, p.cols,
                               plan.parts);
        else
            hipLaunchKernelGGL(loss_join_kernel<32>, dim3((unsigned)std::min((p.rows + 31LL) / 32, kMaxThreads / kLossJoinThreads)), dim3(kLossJoinThreads), 0, s, l,
                               d->loss, d->logsumexp, d->logsumexp_rest, p.rows, p.cols, plan.parts);
        TCBNN_LAUNCH_CHECK("loss_join_kernel");
        return TCBNN_OK;
    });
}

extern "C" size_t tcbnn_linear_loss_grad_workspace_bytes(int rows, int in_features, int classes, int dtype, int anywhere) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || in_features > kMaxIn || classes <= 0 || classes > kMaxOut || !dtype_known(dtype)) return 0;
    return loss_workspace(rows, in_features, classes, dtype, anywhere != 0).total;
}

extern "C" int tcbnn_linear_loss_backward(const tcbnn_linear_loss_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_loss(d->rows, d->in_features, d->classes, d->dtype)) return rc;
    const long long x_ld = row_stride(d->input_ld, d->in_features), w_ld = row_stride(d->weight_ld, d->in_features),
                    dx_ld = row_stride(d->grad_input_ld, d->in_features), dw_ld = row_stride(d->grad_weight_ld, d->in_features);
    TCBNN_REQUIRE(x_ld > 0 && w_ld > 0 && dx_ld > 0 && dw_ld > 0, "linear loss: rows overlap");
    TCBNN_REQUIRE(!too_far(x_ld, d->dtype) && !too_far(w_ld, d->dtype), "linear loss: rows too far apart");
    if (!d->grad_input && !d->grad_weight && !d->grad_bias) return TCBNN_OK;
    hipStream_t s = (hipStream_t)stream;
    if (d->rows == 0) {  // the parameters' gradients are sums of nothing
        ProductParams dx = {}, dw = {};
        dw.rows = d->classes;
        dw.cols = d->in_features;
        dw.i.ld = d->classes;
        dw.j.ld = x_ld;
        dw.out = d->grad_weight;
        dw.out_ld = dw_ld;
        if (d->grad_bias) launch_column_join(nullptr, d->grad_bias, 0, d->classes, s);
        TCBNN_LAUNCH_CHECK("column_join_kernel");
        return launch_gradient_products(d->dtype, dx, dw, nullptr, 0, s);
    }
    TCBNN_NOTNULL(d->input);
    TCBNN_NOTNULL(d->weight);
    TCBNN_NOTNULL(d->targets);
    TCBNN_NOTNULL(d->logsumexp);
    TCBNN_NOTNULL(d->grad_loss);
    TCBNN_NOTNULL(d->workspace);
    TCBNN_REQUIRE((uintptr_t)d->workspace % 16 == 0, "linear loss: the workspace is not aligned to 16 bytes");
    TCBNN_REQUIRE(d->workspace_bytes >= loss_workspace(d->rows, d->in_features, d->classes, d->dtype, false).total, "linear loss: workspace too small");
    const bool copies = d->workspace_bytes >= loss_workspace(d->rows, d->in_features, d->classes, d->dtype, true).total;
    const LossWorkspace w = loss_workspace(d->rows, d->in_features, d->classes, d->dtype, copies);
    char* base = (char*)d->workspace;
    if (d->rows <= kFewGradientRows) {
        by_dtype(d->dtype, [&](auto type) {
            using T = decltype(type);
            ProductParams p = {};
            p.i = {d->input, x_ld};
            p.j = {d->weight, w_ld};
            p.rows = d->rows;
            p.cols = d->classes;
            p.sum = d->in_features;
            p.bias = d->bias;
            p.out = base;
            launch_grad_few_rows<T, true>(p, {d->targets, d->logsumexp, d->grad_loss, nullptr, d->loss, d->logsumexp_rest, d->grad_bias, 0, d->classes, 0}, s);
        });
        TCBNN_LAUNCH_CHECK("loss_grad_few_rows_kernel");
        return launch_few_gradients(d->dtype, (float*)base, d->rows, d->in_features, d->classes, {d->weight, w_ld}, {d->input, x_ld}, d->grad_input, dx_ld,
                                    d->grad_weight, dw_ld, (float*)(base + w.split), s);
    }
    float* scale = d->dtype == TCBNN_F16 ? (float*)base : nullptr;
    if (scale) hipLaunchKernelGGL(loss_scale_kernel, dim3(1), dim3(kScaleThreads), 0, s, d->grad_loss, d->targets, scale, d->rows);
    return by_dtype(d->dtype, [&](auto type) -> int {
        using T = decltype(type);
        ProductParams dx = {};
        Operand x = {d->input, x_ld};
        const bool planes = two_planes(d->rows, d->dtype);
        const LossPacking packing = loss_packing(d->rows, d->in_features, w.piece, d->classes, (int)sizeof(T), planes,
                                                 copies && lies_anywhere<T>(x, d->in_features), copies && lies_anywhere<T>({d->weight, w_ld}, d->in_features));
        if (packing.x) x = launch_pack(d->dtype, x, d->rows, d->in_features, base + w.x, s);
        const long long d_ld = packed_ld(w.piece, (int)sizeof(T)), low = planes ? d->rows * d_ld : 0;
        for (int first = 0; first < d->classes; first += w.piece) {
            const int classes = std::min(w.piece, d->classes - first);
            Operand weight = {(const T*)d->weight + first * w_ld, w_ld};
            if (packing.w) weight = launch_pack(d->dtype, weight, classes, d->in_features, base + w.w, s);
            ProductParams p = {};
            p.i = x;
            p.j = weight;
            p.padded_i = packing.x;
            p.padded_j = packing.w;
            p.rows = d->rows;
            p.cols = classes;
            p.sum = d->in_features;
            p.bias = d->bias ? d->bias + first : nullptr;
            p.out = base + w.d;
            p.out_ld = d_ld;
            LossGradParams l = {d->targets, d->logsumexp, d->grad_loss, scale, d->loss, d->logsumexp_rest, d->grad_bias ? (float*)(base + w.sums) : nullptr, first, d->classes, low};
            const Access access = access_of<T, false, false>(p);
            const Plan plan = plan_product(p.rows, p.cols, p.sum, (int)sizeof(T), access == WHOLE_PIECES, 0, CUT_256, true);
            const bool few = p.rows <= kFewRows && (access == ELEMENTS || few_time(p.rows, p.cols, p.sum, (int)sizeof(T), access == WHOLE_PIECES) < plan.time);
            const bool brief = !few && short_sum(access, p.rows, p.cols, p.sum, (int)sizeof(T));
            const int tiles_i = few ? 1 : (p.rows - 1) / cut_size(access, plan.cut, brief) + 1;
            if (l.sums && tiles_i == 1) l.sums = d->grad_bias + first;
            if (few) launch_grad_few_rows<T, false>(p, l, s);
            if (!few) by_tile(access, plan.cut, brief, [&](auto size, auto wi, auto wj, auto ws, auto stages, auto how, auto hold, auto keep) {
                constexpr int B = size.value, kThreads = 64 * wi.value * wj.value * ws.value;
                // rows beyond a launch's threads have one of their own
                const long long tiles_j = (p.cols - 1) / B + 1, at_once = std::max(1LL, kMaxThreads / kThreads / tiles_j) * B;
                for (long long row = 0; row < p.rows; row += at_once) {
                    ProductParams q = p;
                    LossGradParams part = l;
                    q.rows = (int)std::min(at_once, p.rows - row);
                    q.i.p = (const T*)p.i.p + row * p.i.ld;
                    q.out = (T*)p.out + row * p.out_ld;
                    part.targets += row;
                    part.lse += row;
                    part.dloss += row;
                    if (part.loss) part.loss += row;
                    if (part.rest) part.rest += row;
                    if (part.sums) part.sums += row / B * p.cols;
                    cut_product(q, B, kStepBytes / (int)sizeof(T), 1, nullptr);
                    hipLaunchKernelGGL(HIP_KERNEL_NAME(loss_grad_product_kernel<T, B, B, wi.value, wj.value, ws.value, stages.value, how.value, hold.value, keep.value>),
                                       dim3((unsigned)((long long)q.tiles_i * q.tiles_j)), dim3(kThreads), 0, s, q, part);
                }
            });
            if (d->grad_bias && tiles_i > 1) launch_column_join(l.sums, d->grad_bias + first, tiles_i, classes, s);
            TCBNN_LAUNCH_CHECK("loss_grad_product_kernel");
            ProductParams dw = {};
            dx.i = dw.i = {p.out, p.out_ld};
            dx.padded_i = dw.padded_i = classes >= Elem<T>::kVec;
            dx.factor = dw.factor = scale ? scale + 1 : nullptr;
            dx.j = weight;
            dx.padded_j = packing.w;
            dw.padded_j = packing.x;
            dx.i_low = dw.i_low = low;
            dx.plane = planes ? plane_of(classes, (int)sizeof(T)) : 0;
            dw.plane = planes ? plane_of(d->rows, (int)sizeof(T)) : 0;
            dx.rows = d->rows;
            dx.cols = d->in_features;
            dx.sum = classes;
            dx.out = d->grad_input;
            dx.out_ld = dx_ld;
            if (w.piece < d->classes) {
                dx.carry = first == 0 ? CARRY_FIRST : CARRY_ON;
                dx.splits = w.splits;
                dx.partial = (float*)(base + w.dx);
            }
            dw.j = x;
            dw.rows = classes;
            dw.cols = d->in_features;
            dw.sum = d->rows;
            dw.out = d->grad_weight ? (T*)d->grad_weight + first * dw_ld : nullptr;
            dw.out_ld = dw_ld;
            if (int rc = launch_gradient_products(d->dtype, dx, dw, (float*)(base + w.split), w.total - w.split, s, true)) return rc;
        }
        if (w.piece < d->classes && d->grad_input) {
            dx.partial_stride = (long long)d->rows * d->in_features;
            return launch_carried_sum(d->dtype, dx, s);
        }
        return TCBNN_OK;
    });
}
