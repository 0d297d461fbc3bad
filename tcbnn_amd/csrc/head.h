// What the float head's kernels (linear.hip, layernorm.hip, logprobs.hip) share: element types, vector loads and stores at
// any alignment, sums over wavefronts and workgroups, activations, and the choice of a kernel by type.
#pragma once

#include <utility>

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

// ---- sums and maxima over the 64 lanes; every lane gets the result.  The order is the same in every call.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

}  // namespace head
}  // namespace tcbnn
