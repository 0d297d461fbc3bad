// The gated feed-forward product and its gradients (tcbnn_gated_forward / _backward):  z = x w^T + b with 2 n columns, the gate's first;
// h = act(g) u of its halves g and u;  dg = dh u act'(g),  du = dh act(g),  dx = [dg du] w,  dw = [dg du]^T x,  db = column sums.
//
// Forward, both projections are one product: a tile's columns alternate between 16 rows of the gate's weights and the same 16 of the
// rest, so that g and u of a column are in one lane's registers when the sum is done, and z leaves only where it is asked for.
// Backward, [dg du] is one matrix of 2 n columns, as w is one of 2 n rows: a pass makes it, and two products of the linear layer's follow.
//
// Large products are bound by the matrix instructions, 8192 x 4096 -> 2 x 8192 bf16 with z kept 877 to 929 us from card to card (1.25 to 1.18 PFLOP/s), gradients of 8192 x
// 1024 -> 2 x 4096 289 to 311 us, of which the products take 225 to 250 (1.22 to 1.10 PFLOP/s) and the pass 58 (5.8 TB/s); single rows by the weights' bytes, 1 x 4096 -> 2 x 8192
// 26 us (5.1 TB/s, the launch included); 77 x 1023 -> 2 x 1537 f16 takes 8.5 us, steps of the sum one after the other.
#include "product.h"

namespace tcbnn {
namespace {

using namespace head;

constexpr int kMaxFeatures = kMaxOut / 2;

// their z -> the outputs: C neighbouring columns of a row, of which `n` exist
template <typename T, int C>
__device__ __forceinline__ void finish(const ProductParams& p, long long i, int j, int n, const float* bias_g, const float* bias_u, float* g, float* u) {
#pragma unroll
    for (int e = 0; e < C; ++e) g[e] += bias_g[e], u[e] += bias_u[e];
    if (p.preact) {
        put_columns<T, C>(p.preact, p.preact_ld, i, j, n, g);
        put_columns<T, C>((T*)p.preact + p.cols, p.preact_ld, i, j, n, u);
    }
    by_activation(p.activation, [&](auto act) {
#pragma unroll
        for (int e = 0; e < C; ++e) g[e] = activate<T, act.value>(g[e]) * u[e];
    });
    put_columns<T, C>(p.out, p.out_ld, i, j, n, g);
}

// `p.cols` is n; a workgroup's tile is BI rows by BJ / 2 columns of either half.
template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG>
__global__ __launch_bounds__(64 * WI * WJ * WS) __attribute__((amdgpu_waves_per_eu(short_waves(WI * WJ * WS, STAGES)))) void gated_product_kernel(const ProductParams p) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass leaves a kernel's stub out where it instantiates a tile's requests twice)
    __shared__ __align__(1024) char lds[product_lds<BI, BJ, WI, WJ, WS, STAGES>()];
    constexpr int NI = BI / WI / 32, NJ = BJ / WJ / 32, V = Elem<T>::kVec;
    constexpr int kOutRow = 32 * NJ * 4 + 16, kOutWave = 32 * kOutRow;
    Acc acc[NI][NJ];
    Spot spot;
    product_sums<T, BI, BJ, WI, WJ, WS, STAGES, ACCESS, HOLD, LONG, false, false, true>(p, blockIdx.x, lds, acc, spot);
    const int lane = spot.lane, share = spot.share;

    // ---- out: 32 rows of the wavefront at a time through LDS (16 columns of g, 16 of u and so on), shared among wavefronts that shared the sum
    char* mine = lds + spot.wave * kOutWave;
    const char* first_share = lds + spot.wave % (WI * WJ) * kOutWave;
    constexpr int kPerRow = 16 * NJ / V, kShareRows = 32 / WS;  // lanes to a row, rows of a wavefront
    constexpr int kRowsAtOnce = 64 / kPerRow < kShareRows ? 64 / kPerRow : kShareRows, kTimes = kShareRows / kRowsAtOnce;
    const int col = (lane % kPerRow) * V, j = (int)spot.j0 + spot.wj / 2 + col, n = lane / kPerRow < kRowsAtOnce ? min(V, p.cols - j) : 0;
    const int at = (col / kPairedRows * 2 * kPairedRows + col % kPairedRows) * 4;
    float bias_g[V], bias_u[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        bias_g[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
        bias_u[e] = p.bias && e < n ? p.bias[(long long)p.cols + j + e] : 0.0f;
    }
#pragma unroll 1
    for (int a = 0; a < NI; ++a) {
        const int row0 = share * kShareRows + lane / kPerRow % kRowsAtOnce;
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
        if constexpr (WS > 1)
            __syncthreads();
        else
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int r = 0; r < kTimes; ++r) {
            const long long i = first + r * kRowsAtOnce;
            const char* from = first_share + (row0 + r * kRowsAtOnce) * kOutRow + at;
            float z[2][V];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    float4 q = *reinterpret_cast<const float4*>(from + (half * kPairedRows + e) * 4);
#pragma unroll
                    for (int w = 1; w < WS; ++w) {
                        const float4 o = *reinterpret_cast<const float4*>(from + w * (WI * WJ * kOutWave) + (half * kPairedRows + e) * 4);
                        q.x += o.x, q.y += o.y, q.z += o.z, q.w += o.w;
                    }
                    z[half][e] = q.x, z[half][e + 1] = q.y, z[half][e + 2] = q.z, z[half][e + 3] = q.w;
                }
            if (i < p.rows && n > 0) finish<T, V>(p, i, j, n, bias_g, bias_u, z[0], z[1]);
        }
        if constexpr (WS > 1) {
            if (NI > 1) __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
#endif
}

// few rows: 8 rows of the gate's weights and the same 8 of the rest are a wavefront's 16
constexpr int kFewPairs = kFewOutputs / 2;
template <typename T, int SHARES>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(2, 4))) void gated_few_rows_kernel(const ProductParams p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = wave % SHARES;
    const long long j0 = p.first + ((long long)blockIdx.x * (kFewWaves / SHARES) + wave / SHARES) * kFewPairs;
    // rows past the last one are read as the last one; nothing of them is kept
    const T* w = (const T*)p.j.p + (min(j0 + lane % kFewPairs, (long long)p.cols - 1) + (lane & kFewPairs ? p.cols : 0)) * p.j.ld;
    const T* x = (const T*)p.i.p + (long long)min(lane & 15, p.rows - 1) * p.i.ld;
    const Acc4 acc = few_rows_sums<T, SHARES>(p, w, x);
    if (share != 0) return;
    float g[4], u[4], bias_g[4], bias_u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        g[e] = acc[e];
        u[e] = __shfl_xor(acc[e], 32);
    }
    const int i = lane & 15;
    const long long j = j0 + 4 * (lane >> 4);
    const int n = (int)min(4LL, p.cols - j);
    if (lane >= 32 || i >= p.rows || n <= 0) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bias_g[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
        bias_u[e] = p.bias && e < n ? p.bias[p.cols + j + e] : 0.0f;
    }
    finish<T, 4>(p, i, (int)j, n, bias_g, bias_u, g, u);
}

// ---- [dg du] in the operands' type, and its column sums in fp32, unrounded.  Bound by memory, and built as the linear layer's pass is: a thread has
// one vector of 16 bytes of columns, of both halves, and goes down its share of the rows.
// Rows that one thread takes: two at a time, so that the card is full early; what has no parts needs no join (bf16, 8 rows a thread at least
// as in the linear layer's pass / 2: 64 x 2000 6.6 us / 3.4, 1000 x 999 17 / 6.9, 200 x 500 f16 13 / 5.8).
constexpr int kGatedAtOnce = 2;
inline int gated_dz_rows(int rows, int vectors) {
    const long long threads = 1024LL * kComputeUnits;  // four workgroups a compute unit
    const int each = (int)(((long long)rows * vectors + threads - 1) / threads), deep = kDzThreads / dz_lanes(vectors);
    if (rows <= 2 * kGatedAtOnce * deep) return (rows + deep - 1) / deep;
    return (each + kGatedAtOnce - 1) / kGatedAtOnce * kGatedAtOnce;
}
inline int gated_dz_parts(int rows, int vectors) {
    const int deep = kDzThreads / dz_lanes(vectors) * gated_dz_rows(rows, vectors);
    return (rows + deep - 1) / deep;
}
template <typename T, int ACT>
__global__ __launch_bounds__(kDzThreads) void gated_dz_kernel(const T* __restrict__ dh, const T* __restrict__ z, T* __restrict__ dz,
                                                              float* __restrict__ sums, int rows, int n, int lanes, int each, long long dh_ld,
                                                              long long z_ld, long long dz_ld) {
    constexpr int V = Elem<T>::kVec, kAtOnce = kGatedAtOnce;
    __shared__ float lds[2][kDzThreads * V];
    const int deep = kDzThreads / lanes, lane = threadIdx.x % lanes, depth = threadIdx.x / lanes;
    const int j = (blockIdx.x * lanes + lane) * V, left = n - j;
    const long long first = (long long)blockIdx.y * deep * each;
    const long long last = min((long long)rows, first + (long long)deep * each);
    float s[2][V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[0][e] = s[1][e] = 0.0f;
    if (depth < deep && left > 0) {
        auto get = [&](const T* p) {
            if (left >= V) return load_vec(p);
            Vec<T> v;
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = e < left ? p[e] : (T)0.0f;
            return v;
        };
        auto put = [&](T* to, const float* d) {
            if (left >= V) {
                Vec<T> v;
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = (T)d[e];
                store_vec(to, v);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < left) to[e] = (T)d[e];
            }
        };
        for (long long r = first + depth; r < last; r += kAtOnce * deep) {
            Vec<T> d[kAtOnce], g[kAtOnce], u[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const long long at = min(r + k * deep, last - 1);  // (rows past the end are read once more and not used)
                d[k] = get(dh + at * dh_ld + j);
                g[k] = get(z + at * z_ld + j);
                u[k] = get(z + at * z_ld + n + j);
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (r + k * deep >= last) break;
                float dg[V], du[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float gate = (float)g[k][e], out = (float)d[k][e];
                    dg[e] = out * (float)u[k][e] * slope<T, ACT>(gate);
                    du[e] = out * activate<T, ACT>(gate);
                    s[0][e] += dg[e];
                    s[1][e] += du[e];
                }
                T* to = dz + (r + k * deep) * dz_ld + j;
                put(to, dg);
                put(to + n, du);
                if (left <= V) {  // (zeros to the row's whole 16 bytes)
                    for (long long e = 2LL * n; e < dz_ld; ++e) dz[(r + k * deep) * dz_ld + e] = (T)0.0f;
                }
            }
        }
    }
    if (sums == nullptr) return;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < V; ++e) lds[half][e * kDzThreads + threadIdx.x] = s[half][e];
    __syncthreads();
    for (int c = threadIdx.x; c < lanes * V; c += kDzThreads) {
        const int l = c / V, e = c % V, col = (blockIdx.x * lanes + l) * V + e;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float t = 0.0f;
            for (int d = 0; d < deep; ++d) t += lds[half][e * kDzThreads + d * lanes + l];
            if (col < n) sums[((size_t)blockIdx.y * 2 + half) * n + col] = t;
        }
    }
}

// few rows: [dg du] in fp32 as launch_few_gradients takes it, and its sums; a lane has a column
template <typename T, int ACT>
__global__ __launch_bounds__(kDzThreads) void gated_dz_few_rows_kernel(const T* __restrict__ dh, const T* __restrict__ z, float* __restrict__ dz,
                                                                       float* __restrict__ db, int rows, int n, long long dh_ld, long long z_ld) {
    const int j = blockIdx.x * kDzThreads + threadIdx.x;
    if (j >= n) return;
    float d[2][kFewGradientRows];
#pragma unroll
    for (int i = 0; i < kFewGradientRows; ++i) {
        const long long r = min(i, rows - 1);
        const float out = (float)dh[r * dh_ld + j], gate = (float)z[r * z_ld + j], up = (float)z[r * z_ld + n + j];
        d[0][i] = i < rows ? out * up * slope<T, ACT>(gate) : 0.0f;
        d[1][i] = i < rows ? out * activate<T, ACT>(gate) : 0.0f;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float* to = dz + ((long long)half * n + j) * kFewGradientRows;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kFewGradientRows; i += 4) {
            *reinterpret_cast<float4*>(to + i) = make_float4(d[half][i], d[half][i + 1], d[half][i + 2], d[half][i + 3]);
            s += d[half][i] + d[half][i + 1] + d[half][i + 2] + d[half][i + 3];
        }
        if (db) db[half * n + j] = s;
    }
}

// The tile is the one that the linear layer's estimates would take for a product of 2 n columns; sums are not split.  Operands that lie anywhere are
// copied where the product of the copies and the copying are estimated to take less time, and the workspace holds them.
// (Tiles for short sums: 8192 x 256 -> 2 x 4096 bf16 with z kept, 4 steps, 86 us, 101 in tiles of 256; 8192 x 384 -> 2 x 512, 6 steps, 15.2 and 16.0; 8192 x 512 -> 2 x 2048, 8
// steps, 60 and 58.)
constexpr int kGatedShortSteps = 6;
struct GatedPlan {
    Access access;
    Plan plan;
    bool few, brief, pack_i, pack_j;
};
inline GatedPlan plan_gated(int rows, int cols, int sum, int size, Access access, bool i_anywhere, bool j_anywhere, size_t workspace_bytes) {
    const bool vectors = access == WHOLE_PIECES;
    GatedPlan g = {access, plan_product(rows, 2 * cols, sum, size, vectors, 0, CUT_256, true), false, false, false, false};
    g.few = rows <= kFewRows && (access == ELEMENTS || few_time(rows, 2 * cols, sum, size, vectors) < g.plan.time);
    g.brief = !g.few && short_sum(access, rows, 2 * cols, sum, size, kGatedShortSteps);
    if (g.few || access != ANYWHERE) return g;
    const Plan whole = plan_product(rows, 2 * cols, sum, size, true, 0, CUT_256, true);
    const size_t i_bytes = i_anywhere ? packed_bytes(rows, sum, size) : 0, j_bytes = j_anywhere ? packed_bytes(2LL * cols, sum, size) : 0;
    if (i_bytes + j_bytes > workspace_bytes) return g;
    if (whole.time + (i_anywhere ? pack_time(i_bytes) : 0.0f) + (j_anywhere ? pack_time(j_bytes) : 0.0f) >= g.plan.time) return g;
    return {WHOLE_PIECES, whole, false, short_sum(WHOLE_PIECES, rows, 2 * cols, sum, size, kGatedShortSteps), i_anywhere, j_anywhere};
}
template <typename T>
GatedPlan plan_gated(const ProductParams& p, size_t workspace_bytes) {
    return plan_gated(p.rows, p.cols, p.sum, (int)sizeof(T), access_of<T, false, false>(p), lies_anywhere<T>(p.i, p.sum), lies_anywhere<T>(p.j, p.sum), workspace_bytes);
}

template <typename T>
int launch_gated(ProductParams p, int dtype, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const GatedPlan g = plan_gated<T>(p, workspace_bytes);
    if (g.pack_i) p.i = launch_pack(dtype, p.i, p.rows, p.sum, workspace, stream);
    if (g.pack_j) p.j = launch_pack(dtype, p.j, 2LL * p.cols, p.sum, (char*)workspace + (g.pack_i ? packed_bytes(p.rows, p.sum, (int)sizeof(T)) : 0), stream);
    p.padded_i = g.pack_i;
    p.padded_j = g.pack_j;
    if (g.few) {
        const int shares = few_shares(2 * p.cols, p.sum, (int)sizeof(T));
        by_few_columns(p, shares, kFewPairs * kFewWaves / shares, [&](auto s, dim3 grid, const ProductParams& q) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_few_rows_kernel<T, s.value>), grid, dim3(64 * kFewWaves), 0, stream, q);
        });
        TCBNN_LAUNCH_CHECK("gated_few_rows_kernel");
        return TCBNN_OK;
    }
    by_tile(g.access, g.plan.cut, g.brief, [&](auto size, auto wi, auto wj, auto ws, auto stages, auto how, auto hold, auto keep) {
        constexpr int B = size.value, WI = wi.value, WJ = wj.value, WS = ws.value, S = stages.value, H = hold.value;
        constexpr bool L = keep.value;
        constexpr int kThreads = 64 * WI * WJ * WS;
        // rows beyond a launch's threads have one of their own
        const long long tiles_j = (p.cols + B / 2 - 1) / (B / 2), at_once = std::max(1LL, kMaxThreads / kThreads / tiles_j) * B;
        for (long long first = 0; first < p.rows; first += at_once) {
            ProductParams q = p;
            q.rows = (int)std::min(at_once, p.rows - first);
            q.i.p = (const T*)p.i.p + first * p.i.ld;
            q.out = (T*)p.out + first * p.out_ld;
            q.preact = p.preact ? (T*)p.preact + first * p.preact_ld : nullptr;
            cut_product(q, B, kStepBytes / (int)sizeof(T), 1, nullptr);
            q.tiles_j = (int)tiles_j;
            hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_product_kernel<T, B, B, WI, WJ, WS, S, how.value, H, L>),
                               dim3((unsigned)((long long)q.tiles_i * q.tiles_j)), dim3(kThreads), 0, stream, q);
        }
    });
    TCBNN_LAUNCH_CHECK("gated_product_kernel");
    return TCBNN_OK;
}

// the kernel that launch_gated takes, as a profiler lists it
template <typename T>
void gated_name(const ProductParams& p, size_t workspace_bytes, char* buf, size_t len) {
    const char* type = std::is_same_v<T, float> ? "float" : (std::is_same_v<T, _Float16> ? "_Float16" : "__bf16");
    const GatedPlan g = plan_gated<T>(p, workspace_bytes);
    if (g.few) {
        snprintf(buf, len, "gated_few_rows_kernel<%s, %d>", type, few_shares(2 * p.cols, p.sum, (int)sizeof(T)));
        return;
    }
    static const char* const shape[3][CUTS] = {
        {"256, 256, 2, 4, 1, 2", "128, 128, 2, 2, 1, 2", "128, 128, 2, 2, 2, 4", "64, 64, 2, 2, 2, 4", "32, 32, 1, 1, 4, 8"},
        {"", "128, 128, 2, 2, 1, 2", "", "64, 64, 2, 2, 2, 2", "32, 32, 1, 1, 4, 2"},
        {"32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2"}};
    const int hold = g.access == ANYWHERE && g.plan.cut != CUT_128 ? 4 : 1;
    snprintf(buf, len, "gated_product_kernel<%s, %s, (Access)%d, %d, %s>", type, g.brief ? "128, 128, 2, 2, 1, 1" : shape[g.access][g.plan.cut], (int)g.access, hold,
             hold == 4 && g.plan.cut != CUT_64 ? "true" : "false");
}

int check_gated(int rows, int in_features, int features, int dtype, int activation) {
    TCBNN_REQUIRE(dtype_known(dtype), "gated: unknown dtype");
    TCBNN_REQUIRE(activation >= TCBNN_ACT_NONE && activation <= TCBNN_ACT_SILU, "gated: unknown activation");
    TCBNN_REQUIRE(rows >= 0 && in_features > 0 && features > 0, "gated: bad shape");
    TCBNN_REQUIRE(rows <= kMaxRows, "gated: at most %d rows", kMaxRows);
    TCBNN_REQUIRE(in_features <= kMaxIn, "gated: at most %d inputs", kMaxIn);
    TCBNN_REQUIRE(features <= kMaxFeatures, "gated: at most %d features", kMaxFeatures);
    return TCBNN_OK;
}

ProductParams gated_product(const tcbnn_gated_desc* d) {
    ProductParams p = {};
    p.i = {d->input, row_stride(d->input_ld, d->in_features)};
    p.j = {d->weight, row_stride(d->weight_ld, d->in_features)};
    p.rows = d->rows;
    p.cols = d->features;
    p.sum = d->in_features;
    p.activation = d->activation;
    p.bias = d->bias;
    p.out = d->output;
    p.preact = d->preact;
    p.out_ld = row_stride(d->output_ld, d->features);
    p.preact_ld = row_stride(d->preact_ld, 2LL * d->features);
    return p;
}

// What the gradients need of a workspace: dz in dtype, rows at whole 16 bytes, the parts of the column sums, copies of weights and input that lie
// anywhere where the products' estimates say so, and what split sums need.
struct GatedGradWorkspace {
    size_t sums, weight, input, split, total;
    bool pack_weight, pack_input;
};
GatedGradWorkspace grad_workspace(int rows, int in_features, int features, int dtype, bool anywhere) {
    const int size = (int)dtype_bytes(dtype), n = 2 * features;
    auto worth = [&](int i, int sum, size_t bytes) {
        return anywhere && in_features * size >= 16 &&
               plan_product(i, in_features, sum, size, true, 0).time + pack_time(bytes) < plan_product(i, in_features, sum, size, false, 0).time;
    };
    const size_t weight = packed_bytes(n, in_features, size), input = packed_bytes(rows, in_features, size);
    GatedGradWorkspace w = {};
    w.pack_weight = worth(rows, n, weight);
    w.pack_input = worth(n, rows, input);
    if (rows <= kFewGradientRows) {
        w.split = whole_lines((size_t)n * kFewGradientRows * sizeof(float));
        w.total = w.split + few_gradients_bytes(rows, in_features, n, dtype);
        w.pack_weight = w.pack_input = false;
        return w;
    }
    w.sums = packed_bytes(rows, n, size);
    w.weight = w.sums + whole_lines(sizeof(float) * gated_dz_parts(rows, out_vectors(features, dtype)) * n);
    w.input = w.weight + (w.pack_weight ? weight : 0);
    w.split = w.input + (w.pack_input ? input : 0);
    w.total = w.split + gradient_product_bytes(rows, in_features, n, dtype, true);
    return w;
}

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

extern "C" size_t tcbnn_gated_workspace_bytes(int rows, int in_features, int features, int dtype) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || in_features > kMaxIn || features <= 0 || features > tcbnn::kMaxFeatures || !dtype_known(dtype)) return 0;
    const int size = (int)dtype_bytes(dtype);
    if (in_features * size < 16) return 0;
    size_t need = 0;
    for (bool i : {false, true})  // (where the operands will lie is not known here)
        for (bool j : {false, true}) {
            const GatedPlan g = plan_gated(rows, features, in_features, size, ANYWHERE, i, j, ~(size_t)0);
            need = std::max(need, (g.pack_i ? packed_bytes(rows, in_features, size) : 0) + (g.pack_j ? packed_bytes(2LL * features, in_features, size) : 0));
        }
    return need;
}

extern "C" int tcbnn_gated_kernel_name(const tcbnn_gated_desc* d, char* buf, size_t len) {
    TCBNN_NOTNULL(d);
    TCBNN_NOTNULL(buf);
    if (int rc = check_gated(d->rows, d->in_features, d->features, d->dtype, d->activation)) return rc;
    by_dtype(d->dtype, [&](auto t) { gated_name<decltype(t)>(gated_product(d), d->workspace ? d->workspace_bytes : 0, buf, len); });
    return TCBNN_OK;
}

extern "C" int tcbnn_gated_forward(const tcbnn_gated_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_gated(d->rows, d->in_features, d->features, d->dtype, d->activation)) return rc;
    const ProductParams p = gated_product(d);
    TCBNN_REQUIRE(p.i.ld > 0 && p.j.ld > 0 && p.out_ld > 0 && p.preact_ld > 0, "gated: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->input);
    TCBNN_NOTNULL(d->weight);
    TCBNN_NOTNULL(d->output);
    TCBNN_REQUIRE((uintptr_t)d->workspace % 16 == 0, "gated: the workspace is not aligned to 16 bytes");
    return by_dtype(d->dtype, [&](auto t) {
        return launch_gated<decltype(t)>(p, d->dtype, d->workspace, d->workspace ? d->workspace_bytes : 0, (hipStream_t)stream);
    });
}

extern "C" size_t tcbnn_gated_grad_workspace_bytes(int rows, int in_features, int features, int dtype, int anywhere) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || in_features > kMaxIn || features <= 0 || features > tcbnn::kMaxFeatures || !dtype_known(dtype)) return 0;
    return grad_workspace(rows, in_features, features, dtype, anywhere != 0).total;
}

extern "C" int tcbnn_gated_backward(const tcbnn_gated_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_gated(d->rows, d->in_features, d->features, d->dtype, d->activation)) return rc;
    const long long x_ld = row_stride(d->input_ld, d->in_features), w_ld = row_stride(d->weight_ld, d->in_features),
                    z_ld = row_stride(d->preact_ld, 2LL * d->features), dh_ld = row_stride(d->grad_output_ld, d->features),
                    dx_ld = row_stride(d->grad_input_ld, d->in_features), dw_ld = row_stride(d->grad_weight_ld, d->in_features);
    TCBNN_REQUIRE(x_ld > 0 && w_ld > 0 && z_ld > 0 && dh_ld > 0 && dx_ld > 0 && dw_ld > 0, "gated: rows overlap");
    if (d->rows > 0) {
        TCBNN_NOTNULL(d->grad_output);
        TCBNN_NOTNULL(d->preact);
        if (d->grad_weight) TCBNN_NOTNULL(d->input);
        if (d->grad_input) TCBNN_NOTNULL(d->weight);
        TCBNN_NOTNULL(d->workspace);
        TCBNN_REQUIRE((uintptr_t)d->workspace % 16 == 0, "gated: the workspace is not aligned to 16 bytes");
        TCBNN_REQUIRE(d->workspace_bytes >= tcbnn_gated_grad_workspace_bytes(d->rows, d->in_features, d->features, d->dtype, 0), "gated: workspace too small");
    }
    if (!d->grad_input && !d->grad_weight && !d->grad_bias) return TCBNN_OK;
    if (d->rows > 0 && d->rows <= kFewGradientRows) {
        const int n = 2 * d->features;
        float* dz = (float*)d->workspace;
        by_dtype(d->dtype, [&](auto t) {
            using T = decltype(t);
            by_activation(d->activation, [&](auto act) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_dz_few_rows_kernel<T, act.value>), dim3((unsigned)((d->features - 1) / kDzThreads + 1)), dim3(kDzThreads), 0,
                                   (hipStream_t)stream, (const T*)d->grad_output, (const T*)d->preact, dz, d->grad_bias, d->rows, d->features, dh_ld, z_ld);
            });
        });
        TCBNN_LAUNCH_CHECK("gated_dz_few_rows_kernel");
        return launch_few_gradients(d->dtype, dz, d->rows, d->in_features, n, {d->weight, w_ld}, {d->input, x_ld}, d->grad_input, dx_ld, d->grad_weight, dw_ld,
                                    (float*)((char*)d->workspace + whole_lines((size_t)n * kFewGradientRows * sizeof(float))), (hipStream_t)stream);
    }
    const int vectors = out_vectors(d->features, d->dtype), lanes = dz_lanes(vectors), parts = d->rows > 0 ? gated_dz_parts(d->rows, vectors) : 0;
    const int n = 2 * d->features, size = (int)dtype_bytes(d->dtype);
    const bool copies = d->workspace_bytes >= tcbnn_gated_grad_workspace_bytes(d->rows, d->in_features, d->features, d->dtype, 1);
    const GatedGradWorkspace w = d->rows > 0 ? grad_workspace(d->rows, d->in_features, d->features, d->dtype, copies) : GatedGradWorkspace{};
    const long long dz_ld = packed_ld(n, size);
    char* base = (char*)d->workspace;
    float* sums = d->grad_bias ? (parts == 1 ? d->grad_bias : (float*)(base + w.sums)) : nullptr;
    if (d->rows > 0)
        by_dtype(d->dtype, [&](auto t) {
            using T = decltype(t);
            by_activation(d->activation, [&](auto act) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_dz_kernel<T, act.value>), dim3((unsigned)((vectors + lanes - 1) / lanes), (unsigned)parts), dim3(kDzThreads),
                                   0, (hipStream_t)stream, (const T*)d->grad_output, (const T*)d->preact, (T*)d->workspace, sums, d->rows, d->features, lanes,
                                   gated_dz_rows(d->rows, vectors), dh_ld, z_ld, dz_ld);
            });
        });
    if (d->grad_bias && sums != d->grad_bias) launch_column_join(sums, d->grad_bias, parts, n, (hipStream_t)stream);
    TCBNN_LAUNCH_CHECK("gated_dz_kernel");
    ProductParams dx = {}, dw = {};
    dx.i = dw.i = {d->workspace, dz_ld};
    dx.padded_i = dw.padded_i = n * size >= 16;
    dx.j = {d->weight, w_ld};
    dw.j = {d->input, x_ld};
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        if (d->grad_input && w.pack_weight && lies_anywhere<T>(dx.j, d->in_features)) {
            dx.j = launch_pack(d->dtype, dx.j, n, d->in_features, base + w.weight, (hipStream_t)stream);
            dx.padded_j = true;
        }
        if (d->grad_weight && w.pack_input && lies_anywhere<T>(dw.j, d->in_features)) {
            dw.j = launch_pack(d->dtype, dw.j, d->rows, d->in_features, base + w.input, (hipStream_t)stream);
            dw.padded_j = true;
        }
    });
    dx.rows = d->rows;
    dx.cols = d->in_features;
    dx.sum = n;
    dx.out = d->grad_input;
    dx.out_ld = dx_ld;
    dw.rows = n;
    dw.cols = d->in_features;
    dw.sum = d->rows;
    dw.out = d->grad_weight;
    dw.out_ld = dw_ld;
    return launch_gradient_products(d->dtype, dx, dw, d->rows > 0 ? (float*)(base + w.split) : nullptr, d->rows > 0 ? d->workspace_bytes - w.split : 0,
                                    (hipStream_t)stream, true);
}
