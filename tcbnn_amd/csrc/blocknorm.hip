// The norms after and before a block, with its gate, its scale and the residual stream between them, and their gradient
// (tcbnn_blocknorm_forward / _backward).  Of every row, with P = scale gate after_gamma and Q = scale gate after_beta:
//
//   s = r + (b - mean1) rstd1 P + Q,   y = (s - mean2) rstd2 gamma + beta       (means of layer norms only)
//   g = dy gamma,  xh = (s - mean2) rstd2,  ds = ds' + rstd2 (g - mean(g) - xh mean(g xh))
//   yh = (b - mean1) rstd1,  h = ds P,  db = rstd1 (h - mean(h) - yh mean(h yh))
//
// and four sums over rows: A = sum ds yh, B = sum ds, C = sum dy xh, D = sum dy.  All parameters' gradients follow from them:
//   dgate = scale (after_gamma A + after_beta B),  dafter_gamma = scale gate A,  dafter_beta = scale gate B,  dgamma = C,  dbeta = D,
// so that a lane keeps two sums a feature for RMS norms and four for layer norms, not five.
//
// Bound by memory: every value is read once and kept in registers as fp32 through both norms.  Rows belong to teams of wavefronts as in
// the layer norm's kernels.
#include "rows.h"

namespace tcbnn {
namespace {

using namespace head;

constexpr int kSums = 4;
// Values of a lane whose parameters and sums stay in registers besides, with 16 wavefronts a workgroup (128 registers a thread).
constexpr int kHeld = 8;

struct NormsParams {
    const void *in, *block;  // (block: NULL without one)
    const float *gate, *after_gamma, *after_beta, *before_gamma, *before_beta;
    void *out, *y;
    float *after_mean, *after_rstd, *before_mean, *before_rstd;
    int rows, n, after, before;
    float scale, eps;
    long long in_ld, block_ld, out_ld, y_ld;
};

// P and Q of a feature
__device__ __forceinline__ float times(float x, const float* p, int i) { return p ? x * p[i] : x; }
template <typename P>
__device__ __forceinline__ float after_factor(const P& p, int i) { return times(times(p.scale, p.gate, i), p.after_gamma, i); }
template <typename P>
__device__ __forceinline__ float after_shift(const P& p, int i) { return p.after_beta ? times(p.scale, p.gate, i) * p.after_beta[i] : 0.0f; }

// a lane's P (of after_gamma) or Q (of after_beta), 0 past the row
template <typename P, typename Slice>
__device__ __forceinline__ void load_after(const P& p, const float* vector, Slice& s, int lane, int n) {
    Slice gate;
    s.load_param(vector, lane, n, 1.0f);
    gate.load_param(p.gate, lane, n, 1.0f);
#pragma unroll
    for (int r = 0; r < (int)(sizeof(s.v) / sizeof(s.v[0])); ++r)
#pragma unroll
        for (int e = 0; e < Slice::V; ++e) {
            const bool in = (r + 1) * Slice::kStep <= n || r * Slice::kStep + lane * Slice::V + e < n;
            s.v[r][e] = in ? p.scale * gate.v[r][e] * s.v[r][e] : 0.0f;
        }
}

// Rows of more bytes than the caches hold are requested and stored past them (PASSING): 16384 x 4096 bf16 100 us, 106 through them; gradients of 8192 x
// 4096 85 us and 91.
constexpr long long kPassingBytes = 256LL << 20;
template <typename F>
void by_passing(long long bytes, F&& f) {
    if (bytes > kPassingBytes) return f(std::true_type());
    f(std::false_type());
}

// Wavefronts a SIMD that the forward kernel's registers are to do for.  Two teams of 16 wavefronts a compute unit with RMS norms (3000 x 8000 bf16 46 us), one
// with layer norms, whose parameters take the registers (63 us; two that read their parameters anew for every row 103).  Of smaller teams
// three workgroups of 8 wavefronts with RMS norms and two with layer norms (8000 x 4000 67 us, three 79 with registers in memory).
constexpr int waves_wanted(int w, int values, bool layer) {
    if (values > kHeld) return 4;
    if (w == 16) return values <= (layer ? kHeld / 2 : kHeld) ? 8 : 4;
    return layer ? 5 : 6;
}
// LAYER: either norm may have means.  All teams of a workgroup take the same number of steps; one without a row of its own computes on the
// last one and keeps nothing.  Two sets of slots in turn: between two sums into one slot lies the barrier of a row in between.
template <typename T, int W, int R, bool LAYER, bool PASSING>
__global__ __launch_bounds__(forward_threads(W)) __attribute__((amdgpu_waves_per_eu(waves_wanted(W, R * Elem<T>::kVec, LAYER)))) void blocknorm_kernel(const NormsParams p) {
    constexpr int kTeams = forward_threads(W) / (64 * W);
    using Slice = RowSlice<T, W, R>;
    constexpr int V = Slice::V;
    constexpr bool kHold = R * V <= kHeld;
    __shared__ float slots[2][kTeams][4][W];
    const int lane = threadIdx.x % (64 * W), wave = lane >> 6, team = threadIdx.x / (64 * W), n = p.n;
    Slice P, Q, g, b, s, u;
    typename Slice::Raw raw_s, raw_u;
    const long long stride = (long long)gridDim.x * kTeams;
    auto request = [&](long long first) {
        const long long row = min(first + team, (long long)p.rows - 1);
        Slice::template request<PASSING>((const T*)p.in + row * p.in_ld, lane, n, raw_s);
        if (p.block) Slice::template request<PASSING>((const T*)p.block + row * p.block_ld, lane, n, raw_u);
    };
    request((long long)blockIdx.x * kTeams);
    auto parameters_after = [&] {
        load_after(p, p.after_gamma, P, lane, n);
        if constexpr (LAYER) {
            if (p.after_beta) {
                load_after(p, p.after_beta, Q, lane, n);
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < V; ++e) Q.v[r][e] = 0.0f;
            }
        }
    };
    auto parameters_before = [&] {
        g.load_param(p.before_gamma, lane, n, 1.0f);
        if constexpr (LAYER) b.load_param(p.before_beta, lane, n, 0.0f);
    };
    if constexpr (kHold) {
        if (p.block) parameters_after();
        if (p.before) parameters_before();
    }
    const float inv = 1.0f / (float)n;
    // the values' differences from their mean in place of them; 1 / deviation
    auto normalize = [&](Slice& x, int kind, float& mean, float* mean_slot, float* square_slot) {
        mean = 0.0f;
        if (LAYER && kind == TCBNN_NORM_LAYER) {
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) sum += x.v[r][e];
            mean = team_sum<W>(sum, mean_slot, wave) * inv;
        }
        float sq = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (LAYER) {
                    // what lies past the row (the last slices' lanes alone) has no share in the variance
                    const bool in = (r + 1) * Slice::kStep <= n || r * Slice::kStep + lane * V + e < n;
                    x.v[r][e] = in ? x.v[r][e] - mean : 0.0f;
                }
                sq = __builtin_fmaf(x.v[r][e], x.v[r][e], sq);
            }
        return 1.0f / sqrtf(__builtin_fmaf(team_sum<W>(sq, square_slot, wave), inv, p.eps));
    };
    int parity = 0;
    for (long long first = (long long)blockIdx.x * kTeams; first < p.rows; first += stride, parity ^= 1) {
        const bool mine = first + team < p.rows;
        const long long row = first + team;
        float (*slot)[W] = slots[parity][team];
        s.take(raw_s);
        if (p.block) u.take(raw_u);
        if (first + stride < p.rows) request(first + stride);
        float mean, rstd;
        if (p.block) {
            rstd = 1.0f;
            if (p.after) {
                rstd = normalize(u, p.after, mean, slot[0], slot[1]);
                if (mine && lane == 0) {
                    if (p.after_mean) p.after_mean[row] = mean;
                    if (p.after_rstd) p.after_rstd[row] = rstd;
                }
            }
            if constexpr (!kHold) parameters_after();
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if constexpr (LAYER) s.v[r][e] += Q.v[r][e];
                    s.v[r][e] = __builtin_fmaf(u.v[r][e] * rstd, P.v[r][e], s.v[r][e]);
                }
        }
        if (mine && p.out) s.template store<PASSING>((T*)p.out + row * p.out_ld, lane, n);
        if (!p.before) continue;
        rstd = normalize(s, p.before, mean, slot[2], slot[3]);
        if (!mine) continue;
        if (lane == 0) {
            if (p.before_mean) p.before_mean[row] = mean;
            if (p.before_rstd) p.before_rstd[row] = rstd;
        }
        if constexpr (!kHold) parameters_before();
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) s.v[r][e] = __builtin_fmaf(s.v[r][e] * rstd, g.v[r][e], LAYER ? b.v[r][e] : 0.0f);
        s.template store<PASSING>((T*)p.y + row * p.y_ld, lane, n);
    }
}

// Rows that a workgroup's registers do not hold: a workgroup a row, whose values are made anew in every pass from what lies in the cache.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void blocknorm_long_kernel(const NormsParams p) {
    __shared__ float slots[4][kLongThreads / 64];
    const float inv = 1.0f / (float)p.n;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* in = (const T*)p.in + row * p.in_ld;
        const T* block = (const T*)p.block + row * p.block_ld;
        auto sum = [&](float* slot, auto f) {
            float s = 0.0f;
            for (int i = threadIdx.x; i < p.n; i += kLongThreads) s += f(i);
            __syncthreads();  // (the last sum of the row before may be the only other one, into the same slot)
            return long_sum(s, slot);
        };
        auto statistics = [&](int kind, float* slot, float& mean, auto f) {
            mean = kind == TCBNN_NORM_LAYER ? sum(slot, f) * inv : 0.0f;
            return 1.0f / sqrtf(sum(slot + kLongThreads / 64, [&](int i) { const float d = f(i) - mean; return d * d; }) * inv + p.eps);
        };
        float mean1 = 0.0f, rstd1 = 1.0f, mean2, rstd2;
        if (p.after) {
            rstd1 = statistics(p.after, slots[0], mean1, [&](int i) { return (float)block[i]; });
            if (threadIdx.x == 0) {
                if (p.after_mean) p.after_mean[row] = mean1;
                if (p.after_rstd) p.after_rstd[row] = rstd1;
            }
        }
        auto stream = [&](int i) {
            const float s = (float)in[i];
            return p.block ? __builtin_fmaf(((float)block[i] - mean1) * rstd1, after_factor(p, i), s + after_shift(p, i)) : s;
        };
        if (p.before) {
            rstd2 = statistics(p.before, slots[2], mean2, stream);
            if (threadIdx.x == 0) {
                if (p.before_mean) p.before_mean[row] = mean2;
                if (p.before_rstd) p.before_rstd[row] = rstd2;
            }
        }
        for (int i = threadIdx.x; i < p.n; i += kLongThreads) {
            const float s = stream(i);
            if (p.out) ((T*)p.out)[row * p.out_ld + i] = (T)s;
            if (p.before)
                ((T*)p.y)[row * p.y_ld + i] =
                    (T)__builtin_fmaf((s - mean2) * rstd2, p.before_gamma ? p.before_gamma[i] : 1.0f, p.before_beta ? p.before_beta[i] : 0.0f);
        }
    }
}

// ---- gradient
struct NormsGradParams {
    const void *stream, *block;
    const float *gate, *after_gamma, *after_beta, *before_gamma;
    const float *after_mean, *after_rstd, *before_mean, *before_rstd;
    const void *dy, *ds;  // (each NULL where it is 0)
    void *dr, *db;
    float* grads[5];      // gate, after_gamma, after_beta, before_gamma, before_beta
    float* partial;       // [parts][kSums][n]
    float* row_sums;      // [rows][kSums]: long rows
    int rows, n, after, before;
    float scale;
    bool params;
    long long stream_ld, block_ld, dy_ld, ds_ld, dr_ld, db_ld;
};

// the parameters' gradients of a feature from its sums over all rows
__device__ __forceinline__ void put_parameters(const NormsGradParams& p, int i, const float (&t)[kSums]) {
    if (p.grads[0]) p.grads[0][i] = p.scale * (times(t[0], p.after_gamma, i) + (p.after_beta ? p.after_beta[i] * t[1] : 0.0f));
    if (p.grads[1]) p.grads[1][i] = times(p.scale, p.gate, i) * t[0];
    if (p.grads[2]) p.grads[2][i] = times(p.scale, p.gate, i) * t[1];
    if (p.grads[3]) p.grads[3][i] = t[2];
    if (p.grads[4]) p.grads[4][i] = t[3];
}

// A workgroup of 16 wavefronts is 16 / W teams, and keeps its rows' sums; a workgroup that has all rows writes the parameters' gradients themselves.
// LAYER: the sums B and D, and means.
template <typename T, int W, int R, bool LAYER, bool PASSING>
__global__ __launch_bounds__(kGradThreads) void blocknorm_grad_kernel(const NormsGradParams p) {
    constexpr int kTeams = kGradThreads / (64 * W);
    using Slice = RowSlice<T, W, R>;
    constexpr int V = Slice::V;
    __shared__ float slots[2][kTeams][4][W];
    __shared__ float sums[kTeams > 1 ? kTeams * 64 * W * V : 1];
    const int lane = threadIdx.x % (64 * W), wave = lane >> 6, team = threadIdx.x / (64 * W), n = p.n;
    Slice P, g, d, x, acc[kSums];
    typename Slice::Raw raw_s, raw_u, raw_dy, raw_ds;
    float next[4];
    const bool with_block = p.block != nullptr;
    const long long stride = (long long)gridDim.x * kTeams;
    // What a phase of a row reads is requested when the phase of the row before has taken its own: less lies in registers at a time.
    auto row_of = [&](long long first) { return min(first + team, (long long)p.rows - 1); };
    auto request_dy = [&](long long row) {
        if (p.dy) {
            next[2] = LAYER && p.before == TCBNN_NORM_LAYER ? p.before_mean[row] : 0.0f;
            next[3] = p.before_rstd[row];
            Slice::template request<PASSING>((const T*)p.dy + row * p.dy_ld, lane, n, raw_dy);
            Slice::template request<PASSING>((const T*)p.stream + row * p.stream_ld, lane, n, raw_s);
        }
    };
    auto request_ds = [&](long long row) {
        if (p.ds) Slice::template request<PASSING>((const T*)p.ds + row * p.ds_ld, lane, n, raw_ds);
    };
    auto request_block = [&](long long row) {
        if (with_block) {
            next[0] = LAYER && p.after == TCBNN_NORM_LAYER ? p.after_mean[row] : 0.0f;
            next[1] = p.after ? p.after_rstd[row] : 1.0f;
            Slice::template request<PASSING>((const T*)p.block + row * p.block_ld, lane, n, raw_u);
        }
    };
    {
        const long long row = row_of((long long)blockIdx.x * kTeams);
        request_dy(row);
        request_ds(row);
        request_block(row);
    }
    load_after(p, p.after_gamma, P, lane, n);
    g.load_param(p.before_gamma, lane, n, 1.0f);
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[k].v[r][e] = 0.0f;
    const float inv = 1.0f / (float)n;
    // the sums over the row of g and g x, of which the latter is in LDS slots' second half
    auto row_sums = [&](float (*slot)[W], int kind, float& sg, float& sgx) {
        const bool means = LAYER && kind == TCBNN_NORM_LAYER;
        sgx = wave_sum(sgx);
        if (means) sg = wave_sum(sg);
        if constexpr (W > 1) {
            slot[1][wave] = sgx;
            if (means) slot[0][wave] = sg;
            __syncthreads();
            sg = sgx = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                sgx += slot[1][w];
                if (means) sg += slot[0][w];
            }
        }
        sgx *= inv;
        sg = means ? sg * inv : 0.0f;
    };
    int parity = 0;
    for (long long first = (long long)blockIdx.x * kTeams; first < p.rows; first += stride, parity ^= 1) {
        const bool mine = first + team < p.rows;
        const long long row = row_of(first);
        float (*slot)[W] = slots[parity][team];
        const bool more = first + stride < p.rows;
        const long long next_row = row_of(first + stride);
        const float mean2 = next[2], rstd2 = next[3];
        Slice e_;  // dy
        if (p.dy) e_.take(raw_dy), x.take(raw_s);
        if (more) request_dy(next_row);
        float sg = 0.0f, sgx = 0.0f;
        if (p.dy) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (LAYER ? x.v[r][e] - mean2 : x.v[r][e]) * rstd2;  // (past the row dy is 0, and so is every product)
                    x.v[r][e] = xh;
                    const float dv = mine ? e_.v[r][e] : 0.0f;
                    acc[2].v[r][e] = __builtin_fmaf(dv, mine ? xh : 0.0f, acc[2].v[r][e]);
                    if constexpr (LAYER) acc[3].v[r][e] += dv;
                    const float gv = e_.v[r][e] * g.v[r][e];
                    e_.v[r][e] = gv;
                    if constexpr (LAYER) sg += gv;
                    sgx = __builtin_fmaf(gv, xh, sgx);
                }
            row_sums(slot, p.before, sg, sgx);
        }
        if (p.ds) {
            d.take(raw_ds);
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) d.v[r][e] = 0.0f;
        }
        if (more) request_ds(next_row);
        if (p.dy) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float v = __builtin_fmaf(-x.v[r][e], sgx, e_.v[r][e]);
                    if constexpr (LAYER) v -= sg;
                    d.v[r][e] = __builtin_fmaf(v, rstd2, d.v[r][e]);
                }
        }
        if (mine && p.dr) d.template store<PASSING>((T*)p.dr + row * p.dr_ld, lane, n);
        if (!with_block) continue;
        const float mean1 = next[0], rstd1 = next[1];
        Slice& y = x;  // the block's output
        y.take(raw_u);
        if (more) request_block(next_row);
        sg = sgx = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float yh = (LAYER ? y.v[r][e] - mean1 : y.v[r][e]) * rstd1;
                y.v[r][e] = yh;
                const float dv = mine ? d.v[r][e] : 0.0f;
                acc[0].v[r][e] = __builtin_fmaf(dv, mine ? yh : 0.0f, acc[0].v[r][e]);
                if constexpr (LAYER) acc[1].v[r][e] += dv;
                const float h = d.v[r][e] * P.v[r][e];
                d.v[r][e] = h;
                if constexpr (LAYER) sg += h;
                sgx = __builtin_fmaf(h, yh, sgx);
            }
        if (p.after && p.db) {
            row_sums(slot + 2, p.after, sg, sgx);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float v = __builtin_fmaf(-y.v[r][e], sgx, d.v[r][e]);
                    if constexpr (LAYER) v -= sg;
                    d.v[r][e] = v * rstd1;
                }
        }
        if (mine && p.db) d.template store<PASSING>((T*)p.db + row * p.db_ld, lane, n);
    }
    if (!p.params) return;
    const bool last = gridDim.x == 1;
    float* to = p.partial + (size_t)blockIdx.x * kSums * n;
    auto put = [&](int i, const float (&t)[kSums]) {
        if (i >= n) return;
        if (last) {
            put_parameters(p, i, t);
        } else {
#pragma unroll
            for (int k = 0; k < kSums; ++k)
                if (LAYER || k % 2 == 0) to[(size_t)k * n + i] = t[k];
        }
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if constexpr (kTeams == 1) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float t[kSums] = {acc[0].v[r][e], acc[1].v[r][e], acc[2].v[r][e], acc[3].v[r][e]};
                put(r * Slice::kStep + lane * V + e, t);
            }
        } else {
            constexpr int kEach = (Slice::kStep + kGradThreads - 1) / kGradThreads;
            float t[kEach][kSums] = {};
#pragma unroll
            for (int k = 0; k < kSums; ++k) {
                if (!LAYER && k % 2) continue;
                __syncthreads();
#pragma unroll
                for (int e = 0; e < V; ++e) sums[(team * V + e) * 64 * W + lane] = acc[k].v[r][e];  // (lanes side by side: no bank twice)
                __syncthreads();
#pragma unroll
                for (int q = 0; q < kEach; ++q) {
                    const int c = q * kGradThreads + (int)threadIdx.x;
                    t[q][k] = 0.0f;
                    if (c < Slice::kStep)
                        for (int w = 0; w < kTeams; ++w) t[q][k] += sums[(w * V + c / (64 * W)) * 64 * W + c % (64 * W)];
                }
            }
#pragma unroll
            for (int q = 0; q < kEach; ++q) {
                const int c = q * kGradThreads + (int)threadIdx.x;
                if (c < Slice::kStep) put(r * Slice::kStep + c % (64 * W) * V + c / (64 * W), t[q]);
            }
        }
    }
}

// Rows that a workgroup's registers do not hold: the means of g, g xh, h and h yh of every row first, ...
template <typename T>
struct LongRow {
    const T *stream, *block, *dy, *ds;
    float mean1, rstd1, mean2, rstd2;
    float m[kSums];
    __device__ __forceinline__ LongRow(const NormsGradParams& p, long long row)
        : stream((const T*)p.stream + row * p.stream_ld), block((const T*)p.block + row * p.block_ld), dy((const T*)p.dy + row * p.dy_ld),
          ds((const T*)p.ds + row * p.ds_ld), mean1(p.block && p.after == TCBNN_NORM_LAYER ? p.after_mean[row] : 0.0f),
          rstd1(p.block && p.after ? p.after_rstd[row] : 1.0f), mean2(p.dy && p.before == TCBNN_NORM_LAYER ? p.before_mean[row] : 0.0f),
          rstd2(p.dy ? p.before_rstd[row] : 1.0f), m{0.0f, 0.0f, 0.0f, 0.0f} {}
    __device__ __forceinline__ void sums_of(const NormsGradParams& p, long long row) {
#pragma unroll
        for (int k = 0; k < kSums; ++k) m[k] = p.row_sums[row * kSums + k];
    }
    __device__ __forceinline__ float xh(int i) const { return ((float)stream[i] - mean2) * rstd2; }
    __device__ __forceinline__ float yh(int i) const { return ((float)block[i] - mean1) * rstd1; }
    __device__ __forceinline__ float g(const NormsGradParams& p, int i) const { return times((float)dy[i], p.before_gamma, i); }
    // the gradient of the stream, once the first two means are there
    __device__ __forceinline__ float d(const NormsGradParams& p, int i) const {
        float v = p.ds ? (float)ds[i] : 0.0f;
        if (p.dy) v = __builtin_fmaf(__builtin_fmaf(-xh(i), m[1], g(p, i)) - m[0], rstd2, v);
        return v;
    }
    __device__ __forceinline__ float h(const NormsGradParams& p, int i) const { return d(p, i) * after_factor(p, i); }
};
template <typename T>
__global__ __launch_bounds__(kLongThreads) void blocknorm_long_sums_kernel(const NormsGradParams p) {
    __shared__ float slots[kSums][kLongThreads / 64];
    const float inv = 1.0f / (float)p.n;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        LongRow<T> l(p, row);
        auto sum = [&](float* slot, auto f) {
            float s = 0.0f;
            for (int i = threadIdx.x; i < p.n; i += kLongThreads) s += f(i);
            __syncthreads();  // (the last sum of the row before may be the only other one, into the same slot)
            return long_sum(s, slot) * inv;
        };
        if (p.dy) {
            if (p.before == TCBNN_NORM_LAYER) l.m[0] = sum(slots[0], [&](int i) { return l.g(p, i); });
            l.m[1] = sum(slots[1], [&](int i) { return l.g(p, i) * l.xh(i); });
        }
        if (p.block && p.after) {
            if (p.after == TCBNN_NORM_LAYER) l.m[2] = sum(slots[2], [&](int i) { return l.h(p, i); });
            l.m[3] = sum(slots[3], [&](int i) { return l.h(p, i) * l.yh(i); });
        }
        if (threadIdx.x == 0) {
#pragma unroll
            for (int k = 0; k < kSums; ++k) p.row_sums[row * kSums + k] = l.m[k];
        }
    }
}
// ... then the parameters' sums, 256 features a workgroup, every so manieth row, ...
constexpr int kColumnThreads = 256;
template <typename T>
__global__ __launch_bounds__(kColumnThreads) void blocknorm_long_columns_kernel(const NormsGradParams p) {
    const int i = blockIdx.x * kColumnThreads + threadIdx.x;
    if (i >= p.n) return;
    float t[kSums] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (long long row = blockIdx.y; row < p.rows; row += gridDim.y) {
        LongRow<T> l(p, row);
        l.sums_of(p, row);
        if (p.block) {
            const float d = l.d(p, i);
            t[0] = __builtin_fmaf(d, l.yh(i), t[0]);
            t[1] += d;
        }
        if (p.dy) {
            const float e = (float)l.dy[i];
            t[2] = __builtin_fmaf(e, l.xh(i), t[2]);
            t[3] += e;
        }
    }
#pragma unroll
    for (int k = 0; k < kSums; ++k) p.partial[((size_t)blockIdx.y * kSums + k) * p.n + i] = t[k];
}
// ... and last, because they may lie over what the others read, the gradients of the rows.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void blocknorm_long_grad_kernel(const NormsGradParams p) {
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        LongRow<T> l(p, row);
        l.sums_of(p, row);
        for (int i = threadIdx.x; i < p.n; i += kLongThreads) {
            const float d = l.d(p, i);
            float v = 0.0f;
            if (p.db) {
                v = d * after_factor(p, i);
                if (p.after) v = (__builtin_fmaf(-l.yh(i), l.m[3], v) - l.m[2]) * l.rstd1;
            }
            if (p.dr) ((T*)p.dr)[row * p.dr_ld + i] = (T)d;
            if (p.db) ((T*)p.db)[row * p.db_ld + i] = (T)v;
        }
    }
}

// The sums of all workgroups, always in the same order: 16 features a workgroup, 16 threads to a feature.
constexpr int kJoinThreads = 256, kJoinFeatures = 16;
__global__ __launch_bounds__(kJoinThreads) void blocknorm_join_kernel(const NormsGradParams p, int parts) {
    constexpr int kStep = kJoinThreads / kJoinFeatures;
    __shared__ float lds[kSums][kStep][kJoinFeatures];
    const bool all = p.after == TCBNN_NORM_LAYER || p.before == TCBNN_NORM_LAYER;  // (otherwise B and D are not there)
    const int c = threadIdx.x % kJoinFeatures, part = threadIdx.x / kJoinFeatures, i = blockIdx.x * kJoinFeatures + c;
    float t[kSums] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i < p.n)
        for (int k = part; k < parts; k += 4 * kStep) {
            float v[4][kSums];  // (requests of their own, one wait)
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int w = 0; w < kSums; ++w) v[u][w] = (all || w % 2 == 0) && k + u * kStep < parts ? p.partial[((size_t)(k + u * kStep) * kSums + w) * p.n + i] : 0.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int w = 0; w < kSums; ++w) t[w] += v[u][w];
        }
#pragma unroll
    for (int w = 0; w < kSums; ++w) lds[w][part][c] = t[w];
    __syncthreads();
    if (part == 0 && i < p.n) {
#pragma unroll
        for (int w = 0; w < kSums; ++w) {
            t[w] = 0.0f;
#pragma unroll
            for (int k = 0; k < kStep; ++k) t[w] += lds[w][k][c];
        }
        put_parameters(p, i, t);
    }
}

int check_norms(int rows, int features, int dtype, int after, int before, float scale) {
    TCBNN_REQUIRE(dtype_known(dtype), "blocknorm: unknown dtype");
    TCBNN_REQUIRE(after >= TCBNN_NORM_NONE && after <= TCBNN_NORM_LAYER && before >= TCBNN_NORM_NONE && before <= TCBNN_NORM_LAYER, "blocknorm: unknown norm");
    TCBNN_REQUIRE(rows >= 0 && features > 0, "blocknorm: bad shape");
    TCBNN_REQUIRE(features <= kMaxFeatures, "blocknorm: at most %d features", kMaxFeatures);
    TCBNN_REQUIRE(scale - scale == 0.0f, "blocknorm: the scale is not finite");
    return TCBNN_OK;
}
// an output over an input has its stride
bool over(const void* out, long long out_ld, const void* in, long long in_ld, int rows) { return out == nullptr || out != in || rows <= 1 || out_ld == in_ld; }

// 16-byte vectors of a row up to which the gradient's kernel keeps it, with its parameters and sums
inline int max_grad_vectors(int dtype) { return 1024 * kHeld / (int)(16 / dtype_bytes(dtype)); }
inline bool long_grad(int features, int dtype) { return row_vectors(features, (int)(16 / dtype_bytes(dtype))) > max_grad_vectors(dtype); }

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

extern "C" int tcbnn_blocknorm_forward(const tcbnn_blocknorm_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_norms(d->rows, d->features, d->dtype, d->after, d->before, d->scale)) return rc;
    TCBNN_REQUIRE(d->eps >= 0.0f, "blocknorm: eps must be 0 or more");
    const long long in_ld = row_stride(d->stream_in_ld, d->features), block_ld = row_stride(d->block_ld, d->features),
                    out_ld = row_stride(d->stream_out_ld, d->features), y_ld = row_stride(d->output_ld, d->features);
    TCBNN_REQUIRE(in_ld > 0 && block_ld > 0 && out_ld > 0 && y_ld > 0, "blocknorm: rows overlap");
    TCBNN_REQUIRE(!d->after_beta || d->after == TCBNN_NORM_LAYER, "blocknorm: after_beta without a layer norm");
    TCBNN_REQUIRE(!d->before_beta || d->before == TCBNN_NORM_LAYER, "blocknorm: before_beta without a layer norm");
    TCBNN_REQUIRE(!d->after_gamma || d->after != TCBNN_NORM_NONE, "blocknorm: after_gamma without a norm");
    TCBNN_REQUIRE(!d->before_gamma || d->before != TCBNN_NORM_NONE, "blocknorm: before_gamma without a norm");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->stream_in);
    TCBNN_REQUIRE(d->block || (d->after == TCBNN_NORM_NONE && !d->gate), "blocknorm: a norm or a gate without a block");
    TCBNN_REQUIRE(d->stream_out || d->output, "blocknorm: nothing to write");
    if (d->before != TCBNN_NORM_NONE) TCBNN_NOTNULL(d->output);
    TCBNN_REQUIRE(!d->output || d->before != TCBNN_NORM_NONE, "blocknorm: an output without a norm before");
    TCBNN_REQUIRE(d->stream_out != d->output, "blocknorm: one buffer for the stream and the output");
    TCBNN_REQUIRE(over(d->stream_out, out_ld, d->stream_in, in_ld, d->rows) && over(d->stream_out, out_ld, d->block, block_ld, d->rows) &&
                      over(d->output, y_ld, d->stream_in, in_ld, d->rows) && over(d->output, y_ld, d->block, block_ld, d->rows),
                  "blocknorm: an output over an input has its stride");
    const NormsParams p = {d->stream_in, d->block, d->gate, d->after_gamma, d->after_beta, d->before_gamma, d->before_beta, d->stream_out, d->output,
                           d->after == TCBNN_NORM_LAYER ? d->after_mean : nullptr, d->after_rstd, d->before == TCBNN_NORM_LAYER ? d->before_mean : nullptr,
                           d->before_rstd, d->rows, d->features, d->after, d->before, d->scale, d->eps, in_ld, block_ld, out_ld, y_ld};
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        const int vectors = row_vectors(p.n, Elem<T>::kVec);
        if (vectors > kMaxVectors) {
            hipLaunchKernelGGL(blocknorm_long_kernel<T>, dim3((unsigned)long_blocks(p.rows)), dim3(kLongThreads), 0, (hipStream_t)stream, p);
            return;
        }
        by_team(vectors, [&](auto w, auto r) {
            constexpr int W = w.value, R = r.value;
            const int teams = forward_threads(W) / (64 * W);
            const bool layer = p.after == TCBNN_NORM_LAYER || p.before == TCBNN_NORM_LAYER;
            // As many workgroups as a compute unit has registers for, more where rows are left: 16384 x 4096 bf16 with a fourth of 512 threads, which
            // begins when the others end, 132 us, three 106.
            const long long threads = 256 * waves_wanted(W, R * Elem<T>::kVec, layer);
            const dim3 blocks((unsigned)std::min((p.rows + teams - 1LL) / teams, kComputeUnits * (threads / forward_threads(W))));
            const long long bytes = (long long)p.rows * p.n * sizeof(T) * (1 + (p.block != nullptr) + (p.out != nullptr) + (p.y != nullptr));
            by_passing(bytes, [&](auto passing) {
                if (layer)
                    hipLaunchKernelGGL(HIP_KERNEL_NAME(blocknorm_kernel<T, W, R, true, passing.value>), blocks, dim3(forward_threads(W)), 0, (hipStream_t)stream, p);
                else
                    hipLaunchKernelGGL(HIP_KERNEL_NAME(blocknorm_kernel<T, W, R, false, passing.value>), blocks, dim3(forward_threads(W)), 0, (hipStream_t)stream, p);
            });
        });
    });
    TCBNN_LAUNCH_CHECK("blocknorm_kernel");
    return TCBNN_OK;
}

// The parts of the parameters' sums, then four means of every row where rows are long.
static size_t part_bytes(int rows, int features) { return (size_t)std::min(rows, kComputeUnits) * kSums * features * sizeof(float); }
extern "C" size_t tcbnn_blocknorm_grad_workspace_bytes(int rows, int features, int dtype) {
    if (rows <= 0 || features <= 0 || features > kMaxFeatures || !dtype_known(dtype)) return 0;
    return part_bytes(rows, features) + (long_grad(features, dtype) ? (size_t)rows * kSums * sizeof(float) : 0);
}

extern "C" int tcbnn_blocknorm_backward(const tcbnn_blocknorm_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_norms(d->rows, d->features, d->dtype, d->after, d->before, d->scale)) return rc;
    NormsGradParams p = {d->stream_out, d->block, d->gate, d->after_gamma, d->after_beta, d->before_gamma, d->after_mean, d->after_rstd,
                         d->before_mean, d->before_rstd, d->before == TCBNN_NORM_NONE ? nullptr : d->grad_output, d->grad_stream_out, d->grad_stream_in, d->grad_block,
                         {d->grad_gate, d->grad_after_gamma, d->grad_after_beta, d->grad_before_gamma, d->grad_before_beta},
                         (float*)d->workspace, nullptr, d->rows, d->features, d->after, d->before, d->scale, false,
                         row_stride(d->stream_out_ld, d->features), row_stride(d->block_ld, d->features), row_stride(d->grad_output_ld, d->features),
                         row_stride(d->grad_stream_out_ld, d->features), row_stride(d->grad_stream_in_ld, d->features),
                         row_stride(d->grad_block_ld, d->features)};
    TCBNN_REQUIRE(p.stream_ld > 0 && p.block_ld > 0 && p.dy_ld > 0 && p.ds_ld > 0 && p.dr_ld > 0 && p.db_ld > 0, "blocknorm: rows overlap");
    TCBNN_REQUIRE(!d->after_beta || d->after == TCBNN_NORM_LAYER, "blocknorm: after_beta without a layer norm");
    TCBNN_REQUIRE(!d->after_gamma || d->after != TCBNN_NORM_NONE, "blocknorm: after_gamma without a norm");
    TCBNN_REQUIRE(!d->before_gamma || d->before != TCBNN_NORM_NONE, "blocknorm: before_gamma without a norm");
    TCBNN_REQUIRE(!d->grad_output || d->before != TCBNN_NORM_NONE, "blocknorm: a gradient of an output without a norm before");
    TCBNN_REQUIRE(!d->grad_after_beta || d->after == TCBNN_NORM_LAYER, "blocknorm: grad_after_beta without a layer norm");
    TCBNN_REQUIRE(!d->grad_before_beta || d->before == TCBNN_NORM_LAYER, "blocknorm: grad_before_beta without a layer norm");
    TCBNN_REQUIRE(!d->grad_after_gamma || d->after != TCBNN_NORM_NONE, "blocknorm: grad_after_gamma without a norm");
    TCBNN_REQUIRE(!d->grad_before_gamma || d->before != TCBNN_NORM_NONE, "blocknorm: grad_before_gamma without a norm");
    const bool after_params = d->grad_gate || d->grad_after_gamma || d->grad_after_beta;
    p.params = after_params || d->grad_before_gamma || d->grad_before_beta;
    if (d->rows > 0) {
        if (p.dy) {
            TCBNN_NOTNULL(d->stream_out);
            TCBNN_NOTNULL(d->before_rstd);
            if (d->before == TCBNN_NORM_LAYER) TCBNN_NOTNULL(d->before_mean);
        }
        if (d->grad_block || after_params) {
            TCBNN_NOTNULL(d->block);
            if (d->after != TCBNN_NORM_NONE) TCBNN_NOTNULL(d->after_rstd);
            if (d->after == TCBNN_NORM_LAYER) TCBNN_NOTNULL(d->after_mean);
        }
        TCBNN_REQUIRE(!d->grad_stream_in || d->grad_stream_in != d->grad_block, "blocknorm: one buffer for both gradients");
        TCBNN_REQUIRE(over(p.dr, p.dr_ld, p.dy, p.dy_ld, p.rows) && over(p.dr, p.dr_ld, p.ds, p.ds_ld, p.rows) && over(p.db, p.db_ld, p.dy, p.dy_ld, p.rows) &&
                          over(p.db, p.db_ld, p.ds, p.ds_ld, p.rows) && over(p.db, p.db_ld, p.block, p.block_ld, p.rows),
                      "blocknorm: a gradient over another has its stride");
        const size_t need = tcbnn_blocknorm_grad_workspace_bytes(d->rows, d->features, d->dtype);
        TCBNN_NOTNULL(d->workspace);
        TCBNN_REQUIRE((uintptr_t)d->workspace % 4 == 0, "blocknorm: the workspace is not aligned to 4 bytes");
        TCBNN_REQUIRE(d->workspace_bytes >= need, "blocknorm: workspace too small");
    }
    // what nothing asked for depends on is not read
    if (!d->grad_block && !after_params) p.block = nullptr;
    if (!p.params && !p.dr && !p.db) return TCBNN_OK;
    int parts = 0;
    bool joined = false;
    if (d->rows > 0)
        by_dtype(d->dtype, [&](auto t) {
            using T = decltype(t);
            const int vectors = row_vectors(p.n, Elem<T>::kVec);
            if (long_grad(p.n, d->dtype)) {
                p.row_sums = (float*)((char*)d->workspace + part_bytes(p.rows, p.n));
                const dim3 blocks((unsigned)long_blocks(p.rows));
                hipLaunchKernelGGL(blocknorm_long_sums_kernel<T>, blocks, dim3(kLongThreads), 0, (hipStream_t)stream, p);
                if (p.params) {
                    parts = std::min(p.rows, kComputeUnits);
                    hipLaunchKernelGGL(blocknorm_long_columns_kernel<T>, dim3((unsigned)((p.n + kColumnThreads - 1) / kColumnThreads), (unsigned)parts),
                                       dim3(kColumnThreads), 0, (hipStream_t)stream, p);
                }
                if (p.dr || p.db) hipLaunchKernelGGL(blocknorm_long_grad_kernel<T>, blocks, dim3(kLongThreads), 0, (hipStream_t)stream, p);
                return;
            }
            by_team(vectors, [&](auto w, auto r) {
                constexpr int W = w.value, R = r.value, kTeams = kGradThreads / (64 * W);
                if constexpr (R * Elem<T>::kVec <= kHeld) {
                    parts = p.params ? grad_parts(p.rows, kTeams) : (int)std::min((p.rows + kTeams - 1LL) / kTeams, (long long)kComputeUnits);
                    joined = p.params && parts == 1;
                    const long long bytes = (long long)p.rows * p.n * sizeof(T) * ((p.block != nullptr) + 2 * (p.dy != nullptr) + (p.ds != nullptr) +
                                                                                  (p.dr != nullptr) + (p.db != nullptr));
                    by_passing(bytes, [&](auto passing) {
                        if (p.after == TCBNN_NORM_LAYER || p.before == TCBNN_NORM_LAYER)
                            hipLaunchKernelGGL(HIP_KERNEL_NAME(blocknorm_grad_kernel<T, W, R, true, passing.value>), dim3((unsigned)parts), dim3(kGradThreads), 0,
                                               (hipStream_t)stream, p);
                        else
                            hipLaunchKernelGGL(HIP_KERNEL_NAME(blocknorm_grad_kernel<T, W, R, false, passing.value>), dim3((unsigned)parts), dim3(kGradThreads), 0,
                                               (hipStream_t)stream, p);
                    });
                }
            });
        });
    if (p.params && !joined)
        hipLaunchKernelGGL(blocknorm_join_kernel, dim3((unsigned)((p.n + kJoinFeatures - 1) / kJoinFeatures)), dim3(kJoinThreads), 0, (hipStream_t)stream, p, parts);
    TCBNN_LAUNCH_CHECK("blocknorm_grad_kernel");
    return TCBNN_OK;
}
