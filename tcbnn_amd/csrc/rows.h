// What the norms' kernels (layernorm.hip, blocknorm.hip) share: a row in the registers of a team of wavefronts, sums over a team, and how many
// wavefronts a team has.
#pragma once

#include "head.h"

namespace tcbnn {
namespace head {

constexpr int kMaxFeatures = 65536;

// R vectors of a row, 64 W lanes side by side
template <typename T, int W, int R>
struct RowSlice {
    static constexpr int V = Elem<T>::kVec;
    static constexpr int kStep = 64 * W * V;  // elements that one vector of every lane covers
    float v[R][V];

    // A row's vectors are requested a step before they are taken up: what lies past the row is 0.  PASSING: nothing of the row stays in the caches.
    using Raw = Vec<T>[R];
    template <bool PASSING = false>
    static __device__ __forceinline__ void request(const T* __restrict__ row, int lane, int n, Raw& raw) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = r * kStep + lane * V;
            if ((r + 1) * kStep <= n || i + V <= n) {
                raw[r] = PASSING ? __builtin_nontemporal_load(reinterpret_cast<const VecAnywhere<T>*>(row + i)) : load_vec(row + i);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) raw[r][e] = i + e < n ? row[i + e] : (T)0.0f;
            }
        }
    }
    __device__ __forceinline__ void take(const Raw& raw) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) v[r][e] = (float)raw[r][e];
    }
    template <bool PASSING = false>
    __device__ __forceinline__ void store(T* __restrict__ row, int lane, int n) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = r * kStep + lane * V;
            if ((r + 1) * kStep <= n || i + V <= n) {
                Vec<T> x;
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = (T)v[r][e];
                if constexpr (PASSING)
                    __builtin_nontemporal_store(x, reinterpret_cast<VecAnywhere<T>*>(row + i));
                else
                    store_vec(row + i, x);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (i + e < n) row[i + e] = (T)v[r][e];
            }
        }
    }
    // the lane's part of a vector of parameters, or `fill` where there is none
    __device__ __forceinline__ void load_param(const float* __restrict__ p, int lane, int n, float fill) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = r * kStep + lane * V;
            if (p == nullptr) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[r][e] = fill;
            } else if ((r + 1) * kStep <= n || i + V <= n) {
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const Vec<float> x = load_vec(p + i + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[r][e + k] = x[k];
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) v[r][e] = i + e < n ? p[i + e] : 0.0f;
            }
        }
    }
};

// The sum over a team's wavefronts.  Two alternating slots: whoever writes a slot again has passed the barrier after its last
// reading, so one barrier a sum is enough.
template <int W>
__device__ __forceinline__ float team_sum(float v, float* slot, int wave) {
    v = wave_sum(v);
    if constexpr (W > 1) {
        slot[wave] = v;  // (all lanes of a wavefront write the same value)
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += slot[w];
    }
    return v;
}

constexpr int forward_threads(int w) { return w > 4 ? 64 * w : 256; }

// Rows that a workgroup's registers do not hold: a workgroup a row.
constexpr int kLongThreads = 1024;
inline int long_blocks(int rows) { return (int)std::min((long long)rows, kMaxThreads / kLongThreads); }
__device__ __forceinline__ float long_sum(float v, float* slot) { return team_sum<kLongThreads / 64>(v, slot, threadIdx.x >> 6); }

// The team of wavefronts that keeps a row of so many vectors of 16 bytes: one vector a lane, two in the longest (8192 x 4096 bf16 in
// teams of 8 wavefronts 26.2 us forward and 46 backward; 4, two vectors a lane, 28.0 and 71; 16, half of them idle, 34.0 and 61).
inline int row_vectors(int n, int per_vector) { return (n + per_vector - 1) / per_vector; }
constexpr int kMaxVectors = 2 * 16 * 64;
template <typename F>
void by_team(int vectors, F&& f) {
    using std::integral_constant;
    if (vectors <= 64) return f(integral_constant<int, 1>(), integral_constant<int, 1>());
    if (vectors <= 128) return f(integral_constant<int, 2>(), integral_constant<int, 1>());
    if (vectors <= 256) return f(integral_constant<int, 4>(), integral_constant<int, 1>());
    if (vectors <= 512) return f(integral_constant<int, 8>(), integral_constant<int, 1>());
    if (vectors <= 1024) return f(integral_constant<int, 16>(), integral_constant<int, 1>());
    return f(integral_constant<int, 16>(), integral_constant<int, 2>());
}

constexpr int kGradThreads = 1024;  // of a workgroup that sums over rows
// Workgroups whose sums over rows are joined afterwards.  Up to four rows a team they are one: the launch that joins them takes as
// long as those rows (bf16, us in one launch / two: 16 x 512 3.7 / 3.7, 32 x 512 4.7 / 6.3, 4 x 4096 7.8 / 9.0, 64 x 512 6.8 / 6.5).
inline int grad_parts(int rows, int teams) {
    const int steps = (int)((rows + teams - 1LL) / teams);
    return steps <= 4 ? 1 : std::min(steps, kComputeUnits);
}

}  // namespace head
}  // namespace tcbnn
