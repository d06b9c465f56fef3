// Element types of the tensor operators: loads to and one rounding from 32-bit floats.
#pragma once
#include <hip/hip_runtime.h>

namespace fvsrn {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// V adjacent elements of one lane
template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

template <class T>
__device__ __forceinline__ float toFloat(T v) { return float(v); }

// (round to nearest, ties to even: the one rounding of an output)
template <class T>
__device__ __forceinline__ T fromFloat(float v) { return T(v); }

}  // namespace fvsrn
