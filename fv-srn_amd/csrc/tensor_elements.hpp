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

// N adjacent elements at any address of an element, in pieces of 16, 8, 4 and 2 bytes: gfx950 loads and stores these at any alignment.  (Written with vectors: a
// copy of an array would come out as N loads.)
template <int BYTES, int ALIGN> struct Piece;
#define FVSRN_PIECE(BYTES, ALIGN, ...) \
    template <> struct Piece<BYTES, ALIGN> { typedef __VA_ARGS__ type __attribute__((aligned(ALIGN))); };
typedef unsigned uint2_piece __attribute__((ext_vector_type(2)));
typedef unsigned uint4_piece __attribute__((ext_vector_type(4)));
FVSRN_PIECE(16, 4, uint4_piece)
FVSRN_PIECE(8, 4, uint2_piece)
FVSRN_PIECE(4, 4, unsigned)
FVSRN_PIECE(16, 2, uint4_piece)
FVSRN_PIECE(8, 2, uint2_piece)
FVSRN_PIECE(4, 2, unsigned)
FVSRN_PIECE(2, 2, unsigned short)
FVSRN_PIECE(8, 1, uint2_piece)
#undef FVSRN_PIECE

constexpr int pieceOf(int bytes) { return bytes >= 16 ? 16 : bytes >= 8 ? 8 : bytes >= 4 ? 4 : 2; }

template <class T, int N>
__device__ __forceinline__ void loadWide(T* to, const T* from) {
    if constexpr (N > 0) {
        constexpr int B = pieceOf(N * sizeof(T));
        const auto piece = *reinterpret_cast<const typename Piece<B, alignof(T)>::type*>(from);
        __builtin_memcpy(to, &piece, B);
        loadWide<T, N - B / int(sizeof(T))>(to + B / sizeof(T), from + B / sizeof(T));
    }
}

template <class T, int N>
__device__ __forceinline__ void storeWide(T* to, const T* from) {
    if constexpr (N > 0) {
        constexpr int B = pieceOf(N * sizeof(T));
        typename Piece<B, alignof(T)>::type piece;
        __builtin_memcpy(&piece, from, B);
        *reinterpret_cast<typename Piece<B, alignof(T)>::type*>(to) = piece;
        storeWide<T, N - B / int(sizeof(T))>(to + B / sizeof(T), from + B / sizeof(T));
    }
}

template <class T>
__device__ __forceinline__ float toFloat(T v) { return float(v); }

// (round to nearest, ties to even: the one rounding of an output)
template <class T>
__device__ __forceinline__ T fromFloat(float v) { return T(v); }

}  // namespace fvsrn
