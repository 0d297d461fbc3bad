// What the float head's kernels (linear.hip, layernorm.hip, logprobs.hip) share: element types, vector loads and stores at
// any alignment, sums over wavefronts, the choice of a kernel by type, and the sizes of grids.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace tcbnn {
namespace head {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kVec = 4;  // elements of 16 bytes
};
template <>
struct Elem<__bf16> {
    static constexpr int kVec = 8;
};
template <>
struct Elem<_Float16> {
    static constexpr int kVec = 8;
};

// 16 bytes of elements.  The second type has the alignment of ONE element: rows of odd length start anywhere, and a wavefront's
// requests need no more (the hardware splits what crosses a line).
template <typename T>
using Vec = T __attribute__((ext_vector_type(Elem<T>::kVec)));
template <typename T>
using VecAnywhere = T __attribute__((ext_vector_type(Elem<T>::kVec), aligned(sizeof(T))));

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
    return *reinterpret_cast<const VecAnywhere<T>*>(p);
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, Vec<T> v) {
    *reinterpret_cast<VecAnywhere<T>*>(p) = v;
}

inline bool dtype_known(int dtype) { return dtype == TCBNN_F32 || dtype == TCBNN_BF16 || dtype == TCBNN_F16; }
inline size_t dtype_bytes(int dtype) { return dtype == TCBNN_F32 ? 4 : 2; }

// f(T()) for the element type that `dtype` names (known, as dtype_known says)
template <typename F>
auto by_dtype(int dtype, F&& f) {
    if (dtype == TCBNN_BF16) return f(__bf16());
    if (dtype == TCBNN_F16) return f(_Float16());
    return f(float());
}

// The distance between rows: 0 stands for rows without gaps.  A negative result is a row that overlaps the next.
inline long long row_stride(long long ld, long long length) { return ld == 0 ? length : (ld < length ? -1 : ld); }

// ---- sums and maxima over the 64 lanes, by DPP within 16 lanes and lane swaps beyond (a shuffle through LDS takes ten times
// as long).  Every lane gets the same bits, and the order is the same in every call.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kSwapPairs = 0xb1, kSwapTwos = 0x4e, kMirrorHalf = 0x141, kMirrorRow = 0x140;
// f(v, v of the lane 16 or 32 away)
template <typename F>
__device__ __forceinline__ uint32_t across_rows(uint32_t v, F f) {
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f((uint32_t)a[0], (uint32_t)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f((uint32_t)b[0], (uint32_t)b[1]);
}
template <typename F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, F f) {
    v = f(v, dpp<kSwapPairs>(v));
    v = f(v, dpp<kSwapTwos>(v));
    v = f(v, dpp<kMirrorHalf>(v));
    v = f(v, dpp<kMirrorRow>(v));
    return across_rows(v, f);
}
__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float(wave_reduce(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ float wave_max(float v) {
    return __uint_as_float(wave_reduce(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}

// What grids are sized for.  A constant, not the device's own count: how work is split decides the order of sums, and the size
// of a workspace is asked for before a device is chosen.
constexpr int kComputeUnits = 256;

// A launch's threads along one axis are counted in 32 bits, without an error: what would be more is cut into several launches, taken
// by fewer workgroups, or refused.
constexpr long long kMaxThreads = 0xffffffffLL;

}  // namespace head
}  // namespace tcbnn
