// Linear layers and their gradients (tcbnn_linear_forward / _backward):  z = x w^T + b,  y = act(z) + r;
// dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = column sums of dz.
//
// All three products are one kernel: c[i][j] = sum over s of I(i, s) J(j, s), where an operand lies in memory either along the
// sum (x and w of the forward product: rows of s) or across it (w of dx, dz and x of dw: a row for every s).
//
// Large products are bound by the matrix instructions, as far as power and the barriers between steps let them run: 8192 x 4096 x
// 4096 in bf16 takes 222 us (1.24 PFLOP/s), 254 with bias, GELU, residual and z kept, because 134 MB more of traffic and the
// activations follow the tiles' last steps; 8192^3 811 us (1.36 PFLOP/s); fp32 4096^3 949 us (145 TFLOP/s).  Of the gradients
// of 8192 x 4096 x 1024 dx takes 83 us and dw 86 (0.8 PFLOP/s): operands across the sum need twice the LDS requests.  Rows that lie
// anywhere go through registers, 348 us instead of 222.  Small products are bound by a launch and the latency of their steps,
// products of few rows by the weights' bytes.
#include "product.h"

namespace tcbnn {
namespace {

using namespace head;

template <typename T, int C>
__device__ __forceinline__ void finish(const ProductParams& p, long long i, int j, int n, const float* bias, Columns<T, C> residual, float* z) {
    if constexpr (std::is_same_v<T, _Float16>) {
        if (p.factor) {
            const float f = *p.factor;
#pragma unroll
            for (int e = 0; e < C; ++e) z[e] *= f;
        }
    }
#pragma unroll
    for (int e = 0; e < C; ++e) z[e] += bias[e];
    if (p.preact) put_columns<T, C>(p.preact, p.preact_ld, i, j, n, z);
    by_activation(p.activation, [&](auto act) {
#pragma unroll
        for (int e = 0; e < C; ++e) z[e] = activate<T, act.value>(z[e]);
    });
    if (p.residual) {
#pragma unroll
        for (int e = 0; e < C; ++e) z[e] += (float)residual[e];
    }
    put_columns<T, C>(p.out, p.out_ld, i, j, n, z);
}

// A tile of a linear layer's product or of its gradients'
template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG, bool ACROSS_I, bool ACROSS_J, bool PLANES>
__device__ __forceinline__ void product(const ProductParams& p, int block, char* lds) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass leaves a kernel's stub out where it instantiates a tile's requests twice)
    constexpr int NI = BI / WI / 32, NJ = BJ / WJ / 32, V = Elem<T>::kVec;
    // a wavefront's 32 rows of c on their way out, 16 bytes between rows
    constexpr int kOutRow = 32 * NJ * 4 + 16, kOutWave = 32 * kOutRow;
    Acc acc[NI][NJ];
    Spot spot;
    product_sums<T, BI, BJ, WI, WJ, WS, STAGES, ACCESS, HOLD, LONG, ACROSS_I, ACROSS_J, false, PLANES>(p, block, lds, acc, spot);
    const auto [split, tile_i, tile_j, share, wi, wj, wave, lane, i0, j0] = spot;

    // ---- out: 32 rows of the wavefront at a time through LDS, so that a row leaves in whole runs of 64 bytes or more.  Wavefronts
    // that shared the sum take a share of the rows each.
    char* mine = lds + wave * kOutWave;
    const char* first_share = lds + wave % (WI * WJ) * kOutWave;
    constexpr int kPerRow = 32 * NJ / V, kShareRows = 32 / WS;  // lanes to a row, rows of a wavefront
    constexpr int kRowsAtOnce = 64 / kPerRow < kShareRows ? 64 / kPerRow : kShareRows, kTimes = kShareRows / kRowsAtOnce;
    const int col = (lane % kPerRow) * V, j = (int)j0 + wj + col, n = lane / kPerRow < kRowsAtOnce ? min(V, p.cols - j) : 0;
    float bias[V];
#pragma unroll
    for (int e = 0; e < V; ++e) bias[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
#pragma unroll 1
    for (int a = 0; a < NI; ++a) {
        const int row0 = share * kShareRows + lane / kPerRow % kRowsAtOnce;
        const long long first = i0 + wi + 32 * a + row0;
        Vec<T> residual[kTimes];
        if (p.residual && p.splits == 1) {  // (a carried sum has none)
#pragma unroll
            for (int r = 0; r < kTimes; ++r)
                if (first + r * kRowsAtOnce < p.rows) residual[r] = get_columns<T, V>(p.residual, p.residual_ld, first + r * kRowsAtOnce, j, n);
        }
#pragma unroll
        for (int k = 0; k < NI; ++k)  // (registers have no index: one of NI pieces of code)
            if (k == a) {
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<float4*>(mine + (lane & 31) * kOutRow + (32 * b + 8 * g + 4 * (lane >> 5)) * 4) =
                            make_float4(acc[k][b][4 * g], acc[k][b][4 * g + 1], acc[k][b][4 * g + 2], acc[k][b][4 * g + 3]);
            }
        if constexpr (WS > 1)
            __syncthreads();
        else
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int r = 0; r < kTimes; ++r) {
            const long long i = first + r * kRowsAtOnce;
            const char* from = first_share + (row0 + r * kRowsAtOnce) * kOutRow + col * 4;
            float z[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                float4 q = *reinterpret_cast<const float4*>(from + e * 4);
#pragma unroll
                for (int w = 1; w < WS; ++w) {
                    const float4 o = *reinterpret_cast<const float4*>(from + w * (WI * WJ * kOutWave) + e * 4);
                    q.x += o.x, q.y += o.y, q.z += o.z, q.w += o.w;
                }
                z[e] = q.x, z[e + 1] = q.y, z[e + 2] = q.z, z[e + 3] = q.w;
            }
            if (i < p.rows && n > 0) {
                if (p.splits > 1 || p.carry) {
                    float* partial = p.partial + split * p.partial_stride;
#pragma unroll
                    for (int e = 0; e < V; e += 4) {
                        if (p.carry == CARRY_ON) {
                            const Columns<float, 4> before = get_columns<float, 4>(partial, p.cols, i, j + e, n - e);
#pragma unroll
                            for (int k = 0; k < 4; ++k) z[e + k] += before[k];
                        }
                        put_columns<float, 4>(partial, p.cols, i, j + e, n - e, z + e);
                    }
                } else {
                    finish<T, V>(p, i, j, n, bias, residual[r], z);
                }
            }
        }
        if constexpr (WS > 1) {
            if (NI > 1) __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
#endif
}
template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG, bool ACROSS_I, bool ACROSS_J, bool PLANES>
__global__ __launch_bounds__(64 * WI * WJ * WS) void product_kernel(const ProductParams p) {
    __shared__ __align__(1024) char lds[product_lds<BI, BJ, WI, WJ, WS, STAGES>()];
    product<T, BI, BJ, WI, WJ, WS, STAGES, ACCESS, HOLD, LONG, ACROSS_I, ACROSS_J, PLANES>(p, blockIdx.x, lds);
}

// The sums of a split product's parts, always in the same order, and what follows them: four columns of a row a thread, all parts requested
// before the first is added (one after the other, 3 x 408 in 8 parts took 8.8 us).
constexpr int kJoinVector = 4;
template <typename T>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductParams p) {
    constexpr int C = kJoinVector;
    const int per_row = (p.cols + C - 1) / C;
    const long long v = (long long)blockIdx.x * 256 + threadIdx.x, i = v / per_row;
    if (i >= p.rows) return;
    const int j = (int)(v - i * per_row) * C, n = min(C, p.cols - j);
    Columns<float, C> part[kMaxSplits];
#pragma unroll
    for (int k = 0; k < kMaxSplits; ++k)
        if (k < p.splits) part[k] = get_columns<float, C>(p.partial + k * p.partial_stride, p.cols, i, j, n);
    float z[C], bias[C];
#pragma unroll
    for (int e = 0; e < C; ++e) {
        z[e] = 0.0f;
        bias[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
    }
    Columns<T, C> residual = {};
    if (p.residual) residual = get_columns<T, C>(p.residual, p.residual_ld, i, j, n);
#pragma unroll
    for (int k = 0; k < kMaxSplits; ++k)
        if (k < p.splits) {
#pragma unroll
            for (int e = 0; e < C; ++e) z[e] += part[k][e];
        }
    finish<T, C>(p, i, j, n, bias, residual, z);
}

template <typename T, int SHARES>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(2, 4))) void few_rows_kernel(const ProductParams p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = wave % SHARES;
    const int j0 = p.first + (blockIdx.x * (kFewWaves / SHARES) + wave / SHARES) * kFewOutputs;
    // rows past the last one are read as the last one; nothing of them is kept
    const T* w = (const T*)p.j.p + (long long)min(j0 + (lane & 15), p.cols - 1) * p.j.ld;
    const T* x = (const T*)p.i.p + (long long)min(lane & 15, p.rows - 1) * p.i.ld;
    const Acc4 acc = few_rows_sums<T, SHARES>(p, w, x);
    if (share != 0) return;
    const int i = lane & 15, j = j0 + 4 * (lane >> 4), n = min(4, p.cols - j);
    if (i >= p.rows || n <= 0) return;
    float z[4], bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        z[e] = acc[e];
        bias[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
    }
    Columns<T, 4> residual = {};
    if (p.residual) residual = get_columns<T, 4>(p.residual, p.residual_ld, i, j, n);
    finish<T, 4>(p, i, j, n, bias, residual, z);
}

// ---- dz = dy act'(z) in the operands' type (nothing to write without an activation), and its column sums in fp32, unrounded.
// Bound by memory: a thread has one vector of 16 bytes of columns and goes down its share of the rows, four rows requested at
// a time; the workgroups' sums are joined afterwards, always in the same order.  8192 x 4096 bf16 with GELU: 42 us for 201 MB (4.8 TB/s)
// and 5 us for the join.  dz is rounded to the operands' type because that is what the matrix instructions of dx and dw take: each term
// of theirs then has two roundings of its own in place of one, which in 16 bits are sqrt 2 of the error that dw would have otherwise.
template <typename T, int ACT>
__global__ __launch_bounds__(kDzThreads) void dz_kernel(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                        float* __restrict__ sums, int rows, int n, int lanes, int each,
                                                        long long dy_ld, long long z_ld) {
    constexpr int V = Elem<T>::kVec, kAtOnce = 4;
    __shared__ float lds[kDzThreads * V];
    const int deep = kDzThreads / lanes, lane = threadIdx.x % lanes, depth = threadIdx.x / lanes;
    const int j = (blockIdx.x * lanes + lane) * V, left = n - j;
    const long long first = (long long)blockIdx.y * deep * each;
    const long long last = min((long long)rows, first + (long long)deep * each);
    float s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.0f;
    if (depth < deep && left > 0) {
        auto get = [&](const T* p) {
            if (left >= V) return load_vec(p);
            Vec<T> v;
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = e < left ? p[e] : (T)0.0f;
            return v;
        };
        for (long long r = first + depth; r < last; r += kAtOnce * deep) {
            Vec<T> g[kAtOnce], x[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const long long at = min(r + u * deep, last - 1);  // (rows past the end are read once more and not used)
                g[u] = get(dy + at * dy_ld + j);
                if constexpr (ACT != TCBNN_ACT_NONE) x[u] = get(z + at * z_ld + j);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (r + u * deep >= last) break;
                float d[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    d[e] = (float)g[u][e];
                    if constexpr (ACT != TCBNN_ACT_NONE) d[e] *= slope<T, ACT>((float)x[u][e]);
                    s[e] += d[e];
                }
                if constexpr (ACT != TCBNN_ACT_NONE) {
                    T* to = dz + (r + u * deep) * n + j;
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
                }
            }
        }
    }
    if (sums == nullptr) return;
#pragma unroll
    for (int e = 0; e < V; ++e) lds[e * kDzThreads + threadIdx.x] = s[e];
    __syncthreads();
    for (int c = threadIdx.x; c < lanes * V; c += kDzThreads) {
        const int l = c / V, e = c % V, col = (blockIdx.x * lanes + l) * V + e;
        float t = 0.0f;
        for (int d = 0; d < deep; ++d) t += lds[e * kDzThreads + d * lanes + l];
        if (col < n) sums[(size_t)blockIdx.y * n + col] = t;
    }
}

// the sums of all parts: 16 columns a workgroup (and 16 more where there are more than a launch has threads for), 16 threads to a column
constexpr int kJoinColumns = 16;
__global__ __launch_bounds__(kDzThreads) void column_join_kernel(const float* __restrict__ sums, float* __restrict__ db, int parts, int n) {
    constexpr int kStep = kDzThreads / kJoinColumns;
    __shared__ float lds[kStep][kJoinColumns];
    const int c = threadIdx.x % kJoinColumns, part = threadIdx.x / kJoinColumns;
    for (int j = blockIdx.x * kJoinColumns + c; j - c < n; j += gridDim.x * kJoinColumns) {
        float s = 0.0f;
        if (j < n)
            for (int k = part; k < parts; k += 8 * kStep) {
                float v[8];  // (requests of their own, one wait)
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = k + u * kStep < parts ? sums[(size_t)(k + u * kStep) * n + j] : 0.0f;
#pragma unroll
                for (int u = 0; u < 8; ++u) s += v[u];
            }
        lds[part][c] = s;
        __syncthreads();
        if (part == 0 && j < n) {
            s = 0.0f;
#pragma unroll
            for (int k = 0; k < kStep; ++k) s += lds[k][c];
            db[j] = s;
        }
        __syncthreads();
    }
}

// ---- both products of small gradients in one launch.  A launch more takes as long as these products do (102 x 24 -> 21 f16 with its dz:
// 13.0 us in three launches, 9.9 in two; 128 x 1024 -> 512 18.8 and 16.3).  The first `blocks` workgroups have the product with the longer sum:
// started last, they would run on alone (1024 x 1024 -> 10 bf16 15.1 us, 12.6 so).
template <typename T, Access ACCESS, int STAGES, int HOLD, bool PLANES>
__global__ __launch_bounds__(256) void small_gradients_kernel(const ProductParams dx, const ProductParams dw, int blocks, bool dw_first) {
    __shared__ __align__(1024) char lds[product_lds<32, 32, 1, 1, 4, STAGES>()];
    const int second = (int)blockIdx.x >= blocks, block = (int)blockIdx.x - (second ? blocks : 0);
    if (second == dw_first)
        product<T, 32, 32, 1, 1, 4, STAGES, ACCESS, HOLD, ACCESS == ANYWHERE, false, true, PLANES>(dx, block, lds);
    else
        product<T, 32, 32, 1, 1, 4, STAGES, ACCESS, HOLD, ACCESS == ANYWHERE, true, true, PLANES>(dw, block, lds);
}

// dx and dw in one launch, where in tiles of 32 x 32, four a compute unit at most, they are estimated to take less time together than
// apart in tiles and splits of their own; false: nothing is launched
template <typename T>
bool launch_small_gradients(ProductParams dx, ProductParams dw, size_t workspace_bytes, hipStream_t stream) {
    const Access access_dx = access_of<T, false, true>(dx), access_dw = access_of<T, true, true>(dw), access = std::max(access_dx, access_dw);
    float together = -kCuts16[CUT_32].start, apart = 0.0f;
    for (const ProductParams* p : {&dx, &dw}) {
        if ((long long)((p->rows + 31) / 32) * ((p->cols + 31) / 32) > 4 * kComputeUnits) return false;
        together += plan_product(p->rows, p->cols, p->plane + p->sum, (int)sizeof(T), access == WHOLE_PIECES, 0, CUT_32).time;
        apart += plan_product(p->rows, p->cols, p->plane + p->sum, (int)sizeof(T), (p == &dx ? access_dx : access_dw) == WHOLE_PIECES, workspace_bytes).time;
    }
    if (access == ELEMENTS || together >= apart) return false;
    cut_product(dx, 32, kStepBytes / (int)sizeof(T), 1, nullptr);
    cut_product(dw, 32, kStepBytes / (int)sizeof(T), 1, nullptr);
    const int blocks_dx = dx.tiles_i * dx.tiles_j, blocks_dw = dw.tiles_i * dw.tiles_j;
    const bool dw_first = dw.plane + dw.sum > dx.plane + dx.sum;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks_dx + blocks_dw)), dim3(256), 0, stream, dx, dw, dw_first ? blocks_dw : blocks_dx, dw_first);
    };
    if constexpr (sizeof(T) == 2) {
        if (dx.plane) {
            if (access == WHOLE_PIECES)
                go(small_gradients_kernel<T, WHOLE_PIECES, 8, 1, true>);
            else
                go(small_gradients_kernel<T, ANYWHERE, 2, 4, true>);
            return true;
        }
    }
    if (access == WHOLE_PIECES)
        go(small_gradients_kernel<T, WHOLE_PIECES, 8, 1, false>);
    else
        go(small_gradients_kernel<T, ANYWHERE, 2, 4, false>);
    return true;
}

// ---- both products of large gradients in one launch, where neither has a tile of 256 for every compute unit: the first `blocks` workgroups have the one with
// the longer sum.  (Gated product of 8192 x 1024 -> 2 x 4096 bf16 with its pass over dz: 303 us, 372 in launches of their own.)
template <typename T>
__global__ __launch_bounds__(512) void large_gradients_kernel(const ProductParams dx, const ProductParams dw, int blocks, bool dw_first) {
    __shared__ __align__(1024) char lds[product_lds<256, 256, 2, 4, 1, 2>()];
    const int second = (int)blockIdx.x >= blocks, block = (int)blockIdx.x - (second ? blocks : 0);
    if (second == dw_first)
        product<T, 256, 256, 2, 4, 1, 2, WHOLE_PIECES, 1, false, false, true, false>(dx, block, lds);
    else
        product<T, 256, 256, 2, 4, 1, 2, WHOLE_PIECES, 1, false, true, true, false>(dw, block, lds);
}
// A step of a tile of 256 across the sum, where every compute unit has one: 1.75 us measured in both (as long products alone have it, 1.6, and the plans).
template <typename T>
bool launch_large_gradients(ProductParams dx, ProductParams dw, size_t workspace_bytes, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (dx.plane || dx.carry || access_of<T, false, true>(dx) != WHOLE_PIECES || access_of<T, true, true>(dw) != WHOLE_PIECES) return false;
        constexpr float kStep = 1.75f;
        cut_product(dx, 256, kStepBytes / (int)sizeof(T), 1, nullptr);
        cut_product(dw, 256, kStepBytes / (int)sizeof(T), 1, nullptr);
        const long long blocks_dx = (long long)dx.tiles_i * dx.tiles_j, blocks_dw = (long long)dw.tiles_i * dw.tiles_j;
        if (blocks_dx + blocks_dw > 2 * kComputeUnits) return false;
        const float steps_dx = (float)(dx.split_sum / (kStepBytes / (int)sizeof(T))), steps_dw = (float)(dw.split_sum / (kStepBytes / (int)sizeof(T)));
        // in one round the longer sum; otherwise what is left over begins when the first are done
        const float longest = std::max(steps_dx, steps_dw), work = ((float)blocks_dx * steps_dx + (float)blocks_dw * steps_dw) / (float)kComputeUnits;
        const float together = kCuts16[CUT_256].start + kStep * (blocks_dx + blocks_dw <= kComputeUnits ? longest : longest + work);
        float apart = 0.0f;
        for (const ProductParams* p : {&dx, &dw}) apart += plan_product(p->rows, p->cols, p->sum, (int)sizeof(T), true, workspace_bytes, CUT_256, true).time;
        if (together >= apart) return false;
        const bool dw_first = steps_dw > steps_dx;
        hipLaunchKernelGGL(large_gradients_kernel<T>, dim3((unsigned)(blocks_dx + blocks_dw)), dim3(512), 0, stream, dx, dw, (int)(dw_first ? blocks_dw : blocks_dx),
                           dw_first);
        return true;
    }
    return false;
}

// Tiles of 64 whose rows lie anywhere: the loop for long sums takes registers that a third workgroup of a compute unit would have
// (bf16, with that loop / without: 1000 x 1001 x 999, one tile a compute unit, 9.8 us / 13.5; 2000 x 777 x 1111, three, 24.4 / 19.6).
template <typename T>
bool long_sums(const ProductParams& p, const Plan& plan) {
    const long long tiles = (long long)((p.rows + 63) / 64) * ((p.cols + 63) / 64) * plan.splits;
    return tiles <= 2 * kComputeUnits && ((long long)p.plane + p.sum) * sizeof(T) > (long long)kLongSteps * kStepBytes * plan.splits;
}

// (tiles of single elements are for memory where addresses do not fit; they are slower in any size)
template <typename T>
bool few_rows(const ProductParams& p, Access access, const Plan& plan) {
    return p.rows <= kFewRows && (access == ELEMENTS || few_time(p.rows, p.cols, p.sum, (int)sizeof(T), access == WHOLE_PIECES) < plan.time);
}

// the kernel that launch_product takes for a forward product, as a profiler lists it
template <typename T>
void product_name(const ProductParams& p, size_t workspace_bytes, char* buf, size_t len) {
    const char* type = std::is_same_v<T, float> ? "float" : (std::is_same_v<T, _Float16> ? "_Float16" : "__bf16");
    const Access access = access_of<T, false, false>(p);
    const Plan plan = plan_product(p.rows, p.cols, p.sum, (int)sizeof(T), access == WHOLE_PIECES, workspace_bytes);
    if (few_rows<T>(p, access, plan)) {
        snprintf(buf, len, "few_rows_kernel<%s, %d>", type, few_shares(p.cols, p.sum, (int)sizeof(T)));
        return;
    }
    static const char* const shape[3][CUTS] = {
        {"256, 256, 2, 4, 1, 2", "128, 128, 2, 2, 1, 2", "128, 128, 2, 2, 2, 4", "64, 64, 2, 2, 2, 4", "32, 32, 1, 1, 4, 8"},
        {"", "128, 128, 2, 2, 1, 2", "", "64, 64, 2, 2, 2, 2", "32, 32, 1, 1, 4, 2"},
        {"32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2"}};
    const int hold = access == ANYWHERE && plan.cut != CUT_128 ? 4 : 1;
    const bool keep = hold == 4 && (plan.cut != CUT_64 || long_sums<T>(p, plan));
    snprintf(buf, len, "product_kernel<%s, %s, (Access)%d, %d, %s, false, false, false>%s", type, shape[access][plan.cut], (int)access, hold, keep ? "true" : "false",
             plan.splits > 1 ? " + product_join_kernel" : "");
}

// (rows beyond a launch's threads in launches of their own)
template <typename T>
void launch_join(const ProductParams& p, hipStream_t stream) {
    const long long per_row = (p.cols + kJoinVector - 1) / kJoinVector, at_once = std::max(1LL, (kMaxThreads - 255) / per_row);
    for (long long first = 0; first < p.rows; first += at_once) {
        ProductParams q = p;
        q.rows = (int)std::min(at_once, p.rows - first);
        q.partial = p.partial + first * p.cols;
        q.residual = p.residual ? (const T*)p.residual + first * p.residual_ld : nullptr;
        q.out = (T*)p.out + first * p.out_ld;
        q.preact = p.preact ? (T*)p.preact + first * p.preact_ld : nullptr;
        hipLaunchKernelGGL(product_join_kernel<T>, dim3((unsigned)((q.rows * per_row + 255) / 256)), dim3(256), 0, stream, q);
    }
}

// ---- dx of few rows: tiles of 32, 64 or 128 rows by 256 columns, so that a row of the weights is read in runs of 512 bytes, and a sum that all compute
// units share (16 x 131072 classes -> 4096 bf16, both planes: 176 us, 6.1 TB/s of the weights, 467 in tiles of 32; the loss's step of 78 x 2488 -> 43155
// classes 298 us, 313 in tiles of 128; small products are faster in small tiles: the gradients of 64 x 512 -> 2000 classes 29 us, 32 with
// wide ones, which the estimates below tell apart).
template <typename T, int BI, int STAGES, bool PLANES>
__global__ __launch_bounds__(256) void wide_product_kernel(const ProductParams p) {
    __shared__ __align__(1024) char lds[product_lds<BI, 256, 1, 4, 1, STAGES>()];
    product<T, BI, 256, 1, 4, 1, STAGES, WHOLE_PIECES, 1, false, false, true, PLANES>(p, blockIdx.x, lds);
}
constexpr int kWideRows = 128, kWideSplits = 64;
// Its join: 16 vectors a workgroup, 16 threads to a vector, always in the same order (64 splits of 5 x 554 21 us with a thread to a vector).
constexpr int kWideJoined = 16, kWideJoinThreads = 256;
template <typename T>
__global__ __launch_bounds__(kWideJoinThreads) void wide_join_kernel(const ProductParams p) {
    constexpr int C = kJoinVector, kParts = kWideJoinThreads / kWideJoined, kAtOnce = 4;
    __shared__ Columns<float, C> lds[kParts][kWideJoined];
    const int per_row = (p.cols + C - 1) / C, lane = threadIdx.x % kWideJoined, part = threadIdx.x / kWideJoined;
    const long long v = (long long)blockIdx.x * kWideJoined + lane, i = v / per_row;
    const int j = (int)(v - i * per_row) * C, n = i < p.rows ? min(C, p.cols - j) : 0;
    Columns<float, C> z = {};
    if (n > 0)
        for (int k = part; k < p.splits; k += kAtOnce * kParts) {
            Columns<float, C> s[kAtOnce];  // (requests of their own, one wait)
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                s[u] = k + u * kParts < p.splits ? get_columns<float, C>(p.partial + (k + u * kParts) * p.partial_stride, p.cols, i, j, n) : Columns<float, C>{};
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) z += s[u];
        }
    lds[part][lane] = z;
    __syncthreads();
    if (part != 0 || n <= 0) return;
#pragma unroll
    for (int k = 1; k < kParts; ++k) z += lds[k][lane];
    float sum[C];
#pragma unroll
    for (int e = 0; e < C; ++e) sum[e] = z[e];
    const float bias[C] = {};
    finish<T, C>(p, i, j, n, bias, Columns<T, C>{}, sum);
}
struct WidePlan {
    int splits;
    float time;
};
inline WidePlan plan_wide(int rows, int cols, int sum, int size, bool planes) {
    const int tiles = (cols - 1) / 256 + 1, steps = (int)(((long long)sum * size + kStepBytes - 1) / kStepBytes);
    const int splits = std::max(1, std::min({kWideSplits, kComputeUnits / tiles, steps / 4})), each = (steps + splits - 1) / splits;
    const float read = (float)cols * (float)sum * (float)size / (planes ? 12.0e6f : 6.0e6f), rounds = std::ceil((float)(tiles * splits) / (float)kComputeUnits);
    const float partial = splits > 1 ? 2.3f + (float)splits * (float)rows * (float)cols * 8.0f / 4.0e6f : 0.0f;
    return {(steps + each - 1) / each, 3.0f + std::max(rounds * (float)each * (rows > 64 ? 0.9f : 0.35f), read) + partial};
}
inline size_t wide_bytes(int rows, int cols, int sum, int size) {
    const WidePlan w = plan_wide(rows, cols, sum, size, false);
    return size == 2 && rows <= kWideRows && w.splits > 1 ? (size_t)w.splits * rows * cols * sizeof(float) : 0;
}
template <typename T>
bool launch_wide(ProductParams dx, float* workspace, size_t workspace_bytes, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (dx.rows > kWideRows || dx.carry || access_of<T, false, true>(dx) != WHOLE_PIECES) return false;
        const int sum = dx.plane + dx.sum;
        const WidePlan w = plan_wide(dx.rows, dx.cols, sum, (int)sizeof(T), dx.plane != 0);
        if (wide_bytes(dx.rows, dx.cols, sum, (int)sizeof(T)) > workspace_bytes) return false;
        if (w.time >= plan_product(dx.rows, dx.cols, sum, (int)sizeof(T), true, workspace_bytes, CUT_256, true).time) return false;
        cut_product(dx, 256, kStepBytes / (int)sizeof(T), w.splits, workspace);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)(dx.tiles_j * dx.splits)), dim3(256), 0, stream, dx);
        };
        if (dx.rows > 64)
            dx.plane ? go(wide_product_kernel<T, 128, 3, true>) : go(wide_product_kernel<T, 128, 3, false>);
        else if (dx.rows <= 32)
            dx.plane ? go(wide_product_kernel<T, 32, 4, true>) : go(wide_product_kernel<T, 32, 4, false>);
        else
            dx.plane ? go(wide_product_kernel<T, 64, 3, true>) : go(wide_product_kernel<T, 64, 3, false>);
        if (dx.splits > kMaxSplits)
            hipLaunchKernelGGL(wide_join_kernel<T>, dim3((unsigned)((dx.rows * (long long)((dx.cols - 1) / kJoinVector + 1) - 1) / kWideJoined + 1)), dim3(kWideJoinThreads), 0, stream, dx);
        else if (dx.splits > 1)
            launch_join<T>(dx, stream);
        return true;
    }
    return false;
}

// ---- dw of few rows, a short sum (dw of 16 x 4096 -> 131072 classes bf16 290 us, 3.7 TB/s of what is written, 390 in tiles of 256; the whole step of a
// loss of 333 x 1000 -> 32003 f16, 6 steps, 160 us and 164, of 500 x 1024 -> 32000, 8 steps, 160 and 165, of 700, 11 steps, 240 and 238; of few tiles smaller ones are
// faster: 64 x 1024 -> 8000, 504 tiles, 47.5 us and 48.5 with the plan's, 200 x 512 -> 4000, 128 tiles, 41.7 and 39.8).
template <typename T, bool PLANES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void short_product_kernel(const ProductParams p) {
    __shared__ __align__(1024) char lds[product_lds<128, 128, 2, 2, 1, 1>()];
    product<T, 128, 128, 2, 2, 1, 1, WHOLE_PIECES, 1, false, true, true, PLANES>(p, blockIdx.x, lds);
}
template <typename T>
bool launch_short(ProductParams dw, hipStream_t stream) {
    if (access_of<T, true, true>(dw) != WHOLE_PIECES) return false;
    const long long tiles = ((dw.rows - 1) / 128 + 1LL) * ((dw.cols - 1) / 128 + 1);
    if (!short_sum(WHOLE_PIECES, dw.rows, dw.cols, dw.plane + dw.sum, (int)sizeof(T)) || tiles > kMaxThreads / 256) return false;
    cut_product(dw, 128, kStepBytes / (int)sizeof(T), 1, nullptr);
    const dim3 grid((unsigned)tiles);
    if constexpr (sizeof(T) == 2) {
        if (dw.plane) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(short_product_kernel<T, true>), grid, dim3(256), 0, stream, dw);
            return true;
        }
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(short_product_kernel<T, false>), grid, dim3(256), 0, stream, dw);
    return true;
}

// A carried sum has the splits that it began with.
template <typename T, bool ACROSS_I, bool ACROSS_J>
int launch_product(ProductParams p, float* workspace, size_t workspace_bytes, hipStream_t stream, bool fine = false) {
    const Access access = access_of<T, ACROSS_I, ACROSS_J>(p);
    Plan plan = plan_product(p.rows, p.cols, p.plane + p.sum, (int)sizeof(T), access == WHOLE_PIECES, workspace_bytes, CUT_256, fine);
    if (p.carry) plan.splits = p.splits;
    if constexpr (!ACROSS_I && !ACROSS_J) {
        if (few_rows<T>(p, access, plan)) {
            const int shares = few_shares(p.cols, p.sum, (int)sizeof(T));
            by_few_columns(p, shares, kFewOutputs * kFewWaves / shares, [&](auto s, dim3 grid, const ProductParams& q) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<T, s.value>), grid, dim3(64 * kFewWaves), 0, stream, q);
            });
            TCBNN_LAUNCH_CHECK("few_rows_kernel");
            return TCBNN_OK;
        }
    }
    auto go = [&](auto size, auto wi, auto wj, auto ws, auto stages, auto how, auto hold, auto keep) {
        constexpr int B = size.value, WI = wi.value, WJ = wj.value, WS = ws.value, S = stages.value, H = hold.value;
        constexpr bool L = keep.value;
        constexpr int kThreads = 64 * WI * WJ * WS;
        // rows beyond a launch's threads (2^29 rows, where they are too short for larger tiles than 32) have one of their own
        cut_product(p, B, kStepBytes / (int)sizeof(T), plan.splits, workspace);
        const long long at_once = kMaxThreads / kThreads / ((long long)p.tiles_j * p.splits) * B;
        for (long long first = 0; first < p.rows; first += at_once) {
            ProductParams q = p;
            q.rows = (int)std::min(at_once, p.rows - first);
            q.i.p = (const T*)p.i.p + (ACROSS_I ? first : first * p.i.ld);
            q.residual = p.residual ? (const T*)p.residual + first * p.residual_ld : nullptr;
            q.out = (T*)p.out + first * p.out_ld;
            q.preact = p.preact ? (T*)p.preact + first * p.preact_ld : nullptr;
            cut_product(q, B, kStepBytes / (int)sizeof(T), plan.splits, workspace);
            if (p.carry) {
                q.partial = workspace + first * p.cols;
                q.partial_stride = (long long)p.rows * p.cols;
            }
            const dim3 grid((unsigned)((long long)q.tiles_i * q.tiles_j * q.splits));
            if constexpr (sizeof(T) == 2 && ACROSS_J) {
                if (p.plane)
                    hipLaunchKernelGGL(HIP_KERNEL_NAME(product_kernel<T, B, B, WI, WJ, WS, S, how.value, H, L, ACROSS_I, ACROSS_J, true>), grid, dim3(kThreads), 0,
                                       stream, q);
            }
            if (!p.plane)
                hipLaunchKernelGGL(HIP_KERNEL_NAME(product_kernel<T, B, B, WI, WJ, WS, S, how.value, H, L, ACROSS_I, ACROSS_J, false>), grid, dim3(kThreads), 0,
                                   stream, q);
            if (q.splits > 1 && !q.carry) launch_join<T>(q, stream);
        }
    };
    constexpr std::integral_constant<int, 256> n256;
    constexpr std::integral_constant<int, 128> n128;
    constexpr std::integral_constant<int, 64> n64;
    constexpr std::integral_constant<int, 32> n32;
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 8> eight;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    constexpr std::integral_constant<Access, WHOLE_PIECES> pieces;
    constexpr std::integral_constant<Access, ANYWHERE> anywhere;
    constexpr std::integral_constant<Access, ELEMENTS> elements;
    if (access == WHOLE_PIECES) {
        switch (plan.cut) {
            case CUT_256: go(n256, two, four, one, two, pieces, one, no); break;
            case CUT_128: go(n128, two, two, one, two, pieces, one, no); break;
            case CUT_128_DEEP: go(n128, two, two, two, four, pieces, one, no); break;
            case CUT_64: go(n64, two, two, two, four, pieces, one, no); break;
            default: go(n32, one, one, four, eight, pieces, one, no); break;
        }
    } else if (access == ANYWHERE) {
        switch (plan.cut) {
            case CUT_128: go(n128, two, two, one, two, anywhere, one, no); break;
            case CUT_64:
                if (long_sums<T>(p, plan))
                    go(n64, two, two, two, two, anywhere, four, yes);
                else
                    go(n64, two, two, two, two, anywhere, four, no);
                break;
            default: go(n32, one, one, four, two, anywhere, four, yes); break;
        }
    } else {
        go(n32, one, one, four, two, elements, one, no);
    }
    TCBNN_LAUNCH_CHECK("product_kernel");
    return TCBNN_OK;
}

constexpr int kPackThreads = 256;
template <typename T>
__global__ __launch_bounds__(kPackThreads) void pack_rows_kernel(const T* __restrict__ x, T* __restrict__ to, long long rows, int n, long long x_ld, long long to_ld) {
    constexpr int V = Elem<T>::kVec;
    const int vectors = (n + V - 1) / V;
    for (long long at = (long long)blockIdx.x * kPackThreads + threadIdx.x; at < rows * vectors; at += (long long)gridDim.x * kPackThreads) {
        const long long row = at / vectors;
        const int i = (int)(at - row * vectors) * V;
        const T* from = x + row * x_ld + i;
        Vec<T> v;
        if (i + V <= n) {
            v = load_vec(from);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = i + e < n ? from[e] : (T)0.0f;
        }
        *reinterpret_cast<Vec<T>*>(to + row * to_ld + i) = v;
    }
}

// the partial sums of a split product
size_t split_bytes(int rows, int cols, int sum, int dtype, bool forward, bool fine = false) {
    const int size = (int)dtype_bytes(dtype);
    int splits = 1;
    for (bool vectors : {false, true}) {  // (where the operands will lie is not known here)
        const Plan plan = plan_product(rows, cols, sum, size, vectors, ~(size_t)0, CUT_256, fine);
        if (!forward || rows > kFewRows || few_time(rows, cols, sum, size, vectors) >= plan.time) splits = std::max(splits, plan.splits);
    }
    return splits > 1 ? (size_t)splits * rows * cols * sizeof(float) : 0;
}

}  // namespace

namespace head {

size_t gradient_product_bytes(int rows, int in_features, int out_features, int dtype, bool together) {
    const size_t wide = together ? wide_bytes(rows, in_features, out_features, (int)dtype_bytes(dtype)) : 0;
    return std::max(wide, std::max(split_bytes(rows, in_features, out_features, dtype, false, together),
                                   split_bytes(out_features, in_features, rows, dtype, false, together)));
}

int launch_gradient_products(int dtype, const ProductParams& dx, const ProductParams& dw, float* workspace, size_t workspace_bytes, hipStream_t stream,
                             bool together) {
    return by_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (dx.out && dw.out && dx.rows > 0 && !dx.carry && launch_small_gradients<T>(dx, dw, workspace_bytes, stream)) {
            TCBNN_LAUNCH_CHECK("small_gradients_kernel");
            return TCBNN_OK;
        }
        if (together && dx.out && dw.out && dx.rows > 0 && launch_large_gradients<T>(dx, dw, workspace_bytes, stream)) {
            TCBNN_LAUNCH_CHECK("large_gradients_kernel");
            return TCBNN_OK;
        }
        const bool wide = together && dx.out && dx.rows > 0 && launch_wide<T>(dx, workspace, workspace_bytes, stream);
        TCBNN_LAUNCH_CHECK("wide_product_kernel");
        if (dx.out && dx.rows > 0 && !wide)
            if (int rc = launch_product<T, false, true>(dx, dx.carry ? dx.partial : workspace, workspace_bytes, stream, together)) return rc;
        const bool brief = together && dw.out && launch_short<T>(dw, stream);
        TCBNN_LAUNCH_CHECK("short_product_kernel");
        if (dw.out && !brief)
            if (int rc = launch_product<T, true, true>(dw, workspace, workspace_bytes, stream, together)) return rc;
        return TCBNN_OK;
    });
}

int launch_carried_sum(int dtype, const ProductParams& dx, hipStream_t stream) {
    by_dtype(dtype, [&](auto t) { launch_join<decltype(t)>(dx, stream); });
    TCBNN_LAUNCH_CHECK("product_join_kernel");
    return TCBNN_OK;
}

Operand launch_pack(int dtype, const Operand& o, long long rows, int n, void* to, hipStream_t stream) {
    const long long ld = packed_ld(n, (int)dtype_bytes(dtype));
    by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const long long vectors = rows * (ld / Elem<T>::kVec);
        hipLaunchKernelGGL(pack_rows_kernel<T>, dim3((unsigned)std::min((vectors + kPackThreads - 1) / kPackThreads, 8LL * kComputeUnits)), dim3(kPackThreads), 0,
                           stream, (const T*)o.p, (T*)to, rows, n, o.ld, ld);
    });
    return {to, ld};
}

void launch_column_join(const float* sums, float* out, int parts, int n, hipStream_t stream) {
    hipLaunchKernelGGL(column_join_kernel, dim3((unsigned)std::min((n + kJoinColumns - 1LL) / kJoinColumns, kMaxThreads / kDzThreads)), dim3(kDzThreads), 0,
                       stream, sums, out, parts, n);
}

}  // namespace head
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

static int check_linear(int rows, int in_features, int out_features, int dtype, int activation) {
    TCBNN_REQUIRE(dtype_known(dtype), "linear: unknown dtype");
    TCBNN_REQUIRE(activation >= TCBNN_ACT_NONE && activation <= TCBNN_ACT_SILU, "linear: unknown activation");
    TCBNN_REQUIRE(rows >= 0 && in_features > 0 && out_features > 0, "linear: bad shape");
    TCBNN_REQUIRE(rows <= kMaxRows, "linear: at most %d rows", kMaxRows);
    TCBNN_REQUIRE(in_features <= kMaxIn, "linear: at most %d inputs", kMaxIn);
    TCBNN_REQUIRE(out_features <= kMaxOut, "linear: at most %d outputs", kMaxOut);
    return TCBNN_OK;
}

extern "C" size_t tcbnn_linear_workspace_bytes(int rows, int in_features, int out_features, int dtype) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || out_features <= 0 || !dtype_known(dtype)) return 0;
    return split_bytes(rows, out_features, in_features, dtype, true);
}

static ProductParams forward_product(const tcbnn_linear_desc* d) {
    ProductParams p = {};
    p.i = {d->input, row_stride(d->input_ld, d->in_features)};
    p.j = {d->weight, row_stride(d->weight_ld, d->in_features)};
    p.rows = d->rows;
    p.cols = d->out_features;
    p.sum = d->in_features;
    p.activation = d->activation;
    p.bias = d->bias;
    p.residual = d->residual;
    p.out = d->output;
    p.preact = d->preact;
    p.residual_ld = row_stride(d->residual_ld, d->out_features);
    p.out_ld = row_stride(d->output_ld, d->out_features);
    p.preact_ld = row_stride(d->preact_ld, d->out_features);
    return p;
}

extern "C" int tcbnn_linear_kernel_name(const tcbnn_linear_desc* d, char* buf, size_t len) {
    TCBNN_NOTNULL(d);
    TCBNN_NOTNULL(buf);
    if (int rc = check_linear(d->rows, d->in_features, d->out_features, d->dtype, d->activation)) return rc;
    by_dtype(d->dtype, [&](auto t) { product_name<decltype(t)>(forward_product(d), d->workspace ? d->workspace_bytes : 0, buf, len); });
    return TCBNN_OK;
}

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
    const ProductParams p = forward_product(d);
    return by_dtype(d->dtype, [&](auto t) { return launch_product<decltype(t), false, false>(p, (float*)d->workspace, d->workspace ? d->workspace_bytes : 0, (hipStream_t)stream); });
}

// What the gradients need of a workspace: dz in dtype, then the parts of the column sums (whole 256 bytes each).
static size_t dz_bytes(int rows, int out_features, int dtype) { return whole_lines((size_t)rows * out_features * dtype_bytes(dtype)); }

static size_t sum_bytes(int rows, int out_features, int dtype) {
    return rows == 0 ? 0 : whole_lines(sizeof(float) * dz_parts(rows, out_vectors(out_features, dtype), true) * (size_t)out_features);
}
extern "C" size_t tcbnn_linear_grad_workspace_bytes(int rows, int in_features, int out_features, int dtype) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || out_features <= 0 || !dtype_known(dtype)) return 0;
    return dz_bytes(rows, out_features, dtype) + sum_bytes(rows, out_features, dtype) + gradient_product_bytes(rows, in_features, out_features, dtype);
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
        TCBNN_NOTNULL(d->workspace);
        TCBNN_REQUIRE((uintptr_t)d->workspace % 16 == 0, "linear: the workspace is not aligned to 16 bytes");
        TCBNN_REQUIRE(d->workspace_bytes >= tcbnn_linear_grad_workspace_bytes(d->rows, d->in_features, d->out_features, d->dtype),
                      "linear: workspace too small");
    }
    return by_dtype(d->dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (active || d->grad_bias) {
            const int vectors = out_vectors(d->out_features, d->dtype), lanes = dz_lanes(vectors), parts = dz_parts(d->rows, vectors, active);
            float* sums = d->grad_bias ? (float*)((char*)d->workspace + dz_bytes(d->rows, d->out_features, d->dtype)) : nullptr;
            if (d->grad_bias && parts == 1 && d->rows > 0) sums = d->grad_bias;
            if (d->rows > 0)
                by_activation(d->activation, [&](auto act) {
                    hipLaunchKernelGGL(HIP_KERNEL_NAME(dz_kernel<T, act.value>), dim3((unsigned)((vectors + lanes - 1) / lanes), (unsigned)parts),
                                       dim3(kDzThreads), 0, (hipStream_t)stream, (const T*)d->grad_output, (const T*)d->preact,
                                       (T*)d->workspace, sums, d->rows, d->out_features, lanes, dz_rows(d->rows, vectors, active), dy_ld, z_ld);
                });
            if (d->grad_bias && sums != d->grad_bias) launch_column_join(sums, d->grad_bias, d->rows > 0 ? parts : 0, d->out_features, (hipStream_t)stream);
        }
        TCBNN_LAUNCH_CHECK("dz_kernel");
        const size_t before = dz_bytes(d->rows, d->out_features, d->dtype) + sum_bytes(d->rows, d->out_features, d->dtype);
        float* partials = d->rows > 0 ? (float*)((char*)d->workspace + before) : nullptr;
        const size_t partial_bytes = d->rows > 0 ? d->workspace_bytes - before : 0;
        const Operand dz = active ? Operand{d->workspace, d->out_features} : Operand{d->grad_output, dy_ld};
        ProductParams dx = {}, dw = {};
        dx.i = dw.i = dz;
        dx.j = {d->weight, w_ld};
        dx.rows = d->rows;
        dx.cols = d->in_features;
        dx.sum = d->out_features;
        dx.out = d->grad_input;
        dx.out_ld = dx_ld;
        dw.j = {d->input, x_ld};
        dw.rows = d->out_features;
        dw.cols = d->in_features;
        dw.sum = d->rows;
        dw.out = d->grad_weight;
        dw.out_ld = dw_ld;
        return launch_gradient_products(d->dtype, dx, dw, partials, partial_bytes, (hipStream_t)stream);
    });
}