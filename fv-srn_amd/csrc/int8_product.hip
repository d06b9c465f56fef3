// Layers in 8-bit integers (include/fvsrn.h): codes and scales of matrix rows, and the matrix product of two such matrices with scales, bias and
// activation behind it.
#include "tensor_ops.hpp"

#include <algorithm>

#include "../../include/fvsrn.h"
#include "tensor_elements.hpp"

namespace fvsrn {
namespace {

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef int int16_t_ __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------------------------------------------------
// codes and scales
// ---------------------------------------------------------------------------------------------------------------------

// Bound by memory: every value is read once and a quarter or half of its bytes written.  `width` lanes share a row, 8 values of each in turn
// (rows longer than 8 width HELD are read a second time, from the caches).
constexpr int kHeld = 8;

template <class T, bool ALIGNED>
__device__ __forceinline__ void loadEight(const T* row, int k, int cols, float (&v)[8]) {
    if (ALIGNED && k + 8 <= cols) {
        const Pack<T, 8> x = *reinterpret_cast<const Pack<T, 8>*>(row + k);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = toFloat(x.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < cols ? toFloat(row[k + j]) : 0.f;
    }
}

template <bool ALIGNED>
__device__ __forceinline__ void storeEight(signed char* row, int k, int cols, const float (&v)[8], float scale, bool zero) {
    Pack<signed char, 8> q;
#pragma unroll
    for (int j = 0; j < 8; ++j) q.v[j] = zero ? 0 : (signed char)int(__builtin_rintf(__fdiv_rn(v[j], scale)));  // (the definition's quotient: rounded to 32 bits)
    if (ALIGNED && k + 8 <= cols) {
        *reinterpret_cast<Pack<signed char, 8>*>(row + k) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < cols) row[k + j] = q.v[j];
    }
}

// ALIGNED: row starts are multiples of 8 elements in x and of 8 bytes in the codes
template <class T, bool ALIGNED, int HELD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantizeParams p, const int width) {
    const int lane = threadIdx.x & 63, at = lane & (width - 1);
    const long long own = (blockIdx.x * 4LL + (threadIdx.x >> 6)) * (64 / width) + lane / width, row = min(own, p.rows - 1);
    const T* const x = static_cast<const T*>(p.x) + row * p.ldx;
    float v[HELD][8], most = 0.f, odd = 0.f;
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int k = (j * width + at) * 8;
        loadEight<T, ALIGNED>(x, min(k, p.cols), p.cols, v[j]);
    }
    auto look = [&](const float(&w)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            most = fmaxf(most, fabsf(w[e]));
            odd += w[e] * 0.f;  // (NaN once a value is no finite number)
        }
    };
#pragma unroll
    for (int j = 0; j < HELD; ++j) look(v[j]);
    for (int k = (HELD * width + at) * 8; k < p.cols; k += width * 8) {
        float w[8];
        loadEight<T, ALIGNED>(x, k, p.cols, w);
        look(w);
    }
    for (int o = 1; o < width; o <<= 1) {
        most = fmaxf(most, __shfl_xor(most, o, 64));
        odd += __shfl_xor(odd, o, 64);
    }
    if (own >= p.rows) return;
    const bool bad = odd != odd;
    const float scale = fmaxf(__fdiv_rn(most, 127.f), 0x1p-126f);
    if (at == 0) p.scales[row] = bad ? __builtin_nanf("") : scale;
    signed char* const q = p.codes + row * p.ldc;
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int k = (j * width + at) * 8;
        if (k < p.cols) storeEight<ALIGNED>(q, k, p.cols, v[j], scale, bad);
    }
    for (int k = (HELD * width + at) * 8; k < p.cols; k += width * 8) {
        float w[8];
        loadEight<T, ALIGNED>(x, k, p.cols, w);
        storeEight<ALIGNED>(q, k, p.cols, w, scale, bad);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------------------------------------------------

// The activations of the network kernels (renderer_activations.cuh) on 32-bit floats
__device__ __forceinline__ float activated(float y, int kind, float p) {
    switch (kind) {
        case FVSRN_ACT_RELU: return y < 0.f ? 0.f : y;  // (NaN stays NaN)
        case FVSRN_ACT_SINE: return sinf(p * y);
        case FVSRN_ACT_SNAKE: { const float s = sinf(p * y); return y + s * s / p; }
        case FVSRN_ACT_SNAKEALT: return (y + 1.f - cosf(2.f * p * y)) / (2.f * p);
        case FVSRN_ACT_SIGMOID: return 1.f / (1.f + expf(-y));
        default: return y;
    }
}

// 16 bytes of a row from column k, zeros behind its end
template <bool ALIGNED>
__device__ __forceinline__ int4_t loadCodes(const signed char* row, int k, int K) {
    if (ALIGNED && k + 16 <= K) return *reinterpret_cast<const int4_t*>(row + k);
    union { int4_t v; signed char c[16]; } u;
#pragma unroll
    for (int j = 0; j < 16; ++j) u.c[j] = k + j < K ? row[k + j] : 0;
    return u.v;
}

// v_mfma_i32_32x32x32_i8: lane l holds 16 consecutive k of row l % 32 of either operand (k half l / 32); register r of the result is row
// 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32.  One workgroup: 64 tokens x 64 channels, four waves of 32 x 32.
template <class T, bool ALIGNED>
__global__ __launch_bounds__(256) void matmul_int8_kernel(const Int8Params p, const int activation) {
    constexpr int S = 80;  // LDS row: 64 bytes of k and 16 of padding
    __shared__ __attribute__((aligned(16))) signed char as[64 * S], bs[64 * S];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long m0 = blockIdx.x * 64LL;
    const int n0 = blockIdx.y * 64;
    const int lr = tid >> 2, lk = (tid & 3) * 16;
    const signed char* const ar = p.a + min(m0 + lr, p.M - 1) * p.lda;
    const signed char* const br = p.b + (long long)min(n0 + lr, p.N - 1) * p.ldb;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32, col = lane & 31, half = lane >> 5;
    int16_t_ acc = {};
    for (int k0 = 0; k0 < p.K; k0 += 64) {
        const int4_t av = loadCodes<ALIGNED>(ar, k0 + lk, p.K), bv = loadCodes<ALIGNED>(br, k0 + lk, p.K);
        __syncthreads();
        *reinterpret_cast<int4_t*>(as + lr * S + lk) = av;
        *reinterpret_cast<int4_t*>(bs + lr * S + lk) = bv;
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 64; kk += 32) {
            const int4_t a = *reinterpret_cast<const int4_t*>(as + (wm + col) * S + kk + half * 16);
            const int4_t b = *reinterpret_cast<const int4_t*>(bs + (wn + col) * S + kk + half * 16);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, acc, 0, 0, 0);
        }
    }
    const int n = n0 + wn + col;
    if (n >= p.N) return;
    const float sb = p.scaleB[n], bias = p.bias ? p.bias[n] : 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const long long m = m0 + wm + 8 * (r >> 2) + 4 * half + (r & 3);
        if (m < p.M) static_cast<T*>(p.out)[m * p.ldo + n] = fromFloat<T>(activated(fmaf(float(acc[r]) * sb, p.scaleA[m], bias), activation, p.actParam));
    }
}

int powerOfTwoAtLeast(long long v) {
    int r = 1;
    while (r < v) r <<= 1;
    return r;
}

bool multipleOf(const void* ptr, size_t bytes) { return reinterpret_cast<size_t>(ptr) % bytes == 0; }

template <class F>
hipError_t withType(int dtype, F&& f) {
    if (dtype == FVSRN_TENSOR_F16) return f(f16_t{});
    if (dtype == FVSRN_TENSOR_BF16) return f(bf16_t{});
    return f(float{});
}

}  // namespace

hipError_t launch_quantize_rows(const QuantizeParams& p, int dtype, hipStream_t s) {
    return withType(dtype, [&](auto element) {
        typedef decltype(element) T;
        const bool aligned = multipleOf(p.x, 8 * sizeof(T)) && p.ldx % 8 == 0 && multipleOf(p.codes, 8) && p.ldc % 8 == 0;
        const int width = std::min(64, powerOfTwoAtLeast((p.cols + 7) / 8));
        const unsigned grid = unsigned((p.rows + 4 * (64 / width) - 1) / (4 * (64 / width)));
        auto launch = [&](auto held) {
            constexpr int H = decltype(held)::value;
            if (aligned) quantize_rows_kernel<T, true, H><<<grid, 256, 0, s>>>(p, width);
            else quantize_rows_kernel<T, false, H><<<grid, 256, 0, s>>>(p, width);
            return hipGetLastError();
        };
        if (p.cols <= 512) return launch(std::integral_constant<int, 1>{});
        if (p.cols <= 2048) return launch(std::integral_constant<int, 4>{});
        return launch(std::integral_constant<int, kHeld>{});
    });
}

hipError_t launch_matmul_int8(const Int8Params& p, int activation, int outDtype, hipStream_t s) {
    return withType(outDtype, [&](auto element) {
        typedef decltype(element) T;
        const bool aligned = multipleOf(p.a, 16) && multipleOf(p.b, 16) && p.lda % 16 == 0 && p.ldb % 16 == 0;
        const dim3 grid(unsigned((p.M + 63) / 64), unsigned((p.N + 63) / 64));
        if (aligned) matmul_int8_kernel<T, true><<<grid, 256, 0, s>>>(p, activation);
        else matmul_int8_kernel<T, false><<<grid, 256, 0, s>>>(p, activation);
        return hipGetLastError();
    });
}

}  // namespace fvsrn
