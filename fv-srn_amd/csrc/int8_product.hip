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
    const float scale = fmaxf(most * (1.f / 127.f), 0x1p-126f);
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

// sin(2 pi v) of v revolutions.  The whole turns go in 64 bits, so an argument of 2^24 still has all of a 32-bit result behind it; then the Taylor series up to
// t^13 on [-pi/2, pi/2] (the first term left out is 7e-10).  Short and without branches: it is expanded for every output of a tile.
__device__ __forceinline__ float sineOfTurns(double v) {
    float r = float(v - __builtin_rint(v));
    r = fabsf(r) > 0.25f ? copysignf(0.5f, r) - r : r;
    const float t = r * 6.28318531f, q = t * t;
    float s = fmaf(q, 1.f / 6227020800.f, -1.f / 39916800.f);
    s = fmaf(q, s, 1.f / 362880.f);
    s = fmaf(q, s, -1.f / 5040.f);
    s = fmaf(q, s, 1.f / 120.f);
    s = fmaf(q, s, -1.f / 6.f);
    return fmaf(q * t, s, t);
}

// The activations of the network kernels (renderer_activations.cuh) on 32-bit floats
__device__ __forceinline__ float activated(float y, int kind, float p) {
    constexpr double kTurn = 0.15915494309189535;  // 1 / (2 pi)
    switch (kind) {
        case FVSRN_ACT_RELU: return y < 0.f ? 0.f : y;  // (NaN stays NaN)
        case FVSRN_ACT_SINE: return sineOfTurns(double(p * y) * kTurn);
        case FVSRN_ACT_SNAKE: { const float s = sineOfTurns(double(p * y) * kTurn); return y + s * s / p; }
        case FVSRN_ACT_SNAKEALT: return (y + 1.f - sineOfTurns(double(2.f * p * y) * kTurn + 0.25)) / (2.f * p);
        case FVSRN_ACT_SIGMOID: return 1.f / (1.f + expf(-y));
        default: return y;
    }
}

// Sums of products are exact whatever their order, so k may be cut and joined anywhere.

// 16 bytes of a row from column k, zeros behind its end.  ALIGNED: k and the row start are multiples of 16 (and so is K: no chunk is cut); otherwise one unaligned
// load, which costs what the lines it touches cost, and single bytes at the row's end.
template <bool ALIGNED>
__device__ __forceinline__ int4_t loadCodes(const signed char* row, int k, int K) {
    if (k + 16 <= K) {
        if (ALIGNED) return *reinterpret_cast<const int4_t*>(row + k);
        int4_t v;
        __builtin_memcpy(&v, row + k, 16);
        return v;
    }
    int4_t v = {0, 0, 0, 0};
    if (ALIGNED) return v;
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (k + j < K) v[j >> 2] |= int(static_cast<unsigned char>(row[k + j])) << (8 * (j & 3));
    return v;
}

__device__ __forceinline__ float scaled(int acc, float sa, float sb, float bias, int activation, float param) {
    return activated(fmaf(float(acc) * sb, sa, bias), activation, param);
}

// Few tokens: bound by the weights' bytes, or by how long one wave takes through its part of k.  v_mfma_i32_16x16x64_i8 with the weights as its rows: lane l holds 16
// consecutive k (part l / 16) of channel l % 16 and of token l % 16; register r of the result is channel 4 (l / 16) + r, token l % 16.  A workgroup has 16 channels and 16 MT
// tokens; its eight waves take every eighth 256 bytes of k straight from memory into registers -- each weight is read once by the chip, nothing is
// worth a turn through LDS but the eight sums at the end.
template <class T, bool ALIGNED, int MT>
__global__ __launch_bounds__(512) void matmul_int8_few_kernel(const Int8Params p, const int activation) {
    constexpr int W = 8, U = 4;
    __shared__ int4_t sums[W][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, part = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const long long m0 = blockIdx.y * (16LL * MT);
    const signed char* const br = p.b + (long long)min(n0 + col, p.N - 1) * p.ldb;
    const signed char* ar[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) ar[t] = p.a + min(m0 + t * 16 + col, p.M - 1) * p.lda;
    int4_t acc[MT] = {};
    for (int k0 = wave * 64 * U; k0 < p.K; k0 += W * 64 * U) {
        int4_t b[U], a[MT][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * 64 + part * 16;
            b[u] = loadCodes<ALIGNED>(br, k, p.K);
#pragma unroll
            for (int t = 0; t < MT; ++t) a[t][u] = loadCodes<ALIGNED>(ar[t], k, p.K);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[u], a[t][u], acc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < MT; t += W) {
        int4_t s = sums[0][t][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) s += sums[w][t][lane];
        const long long m = m0 + t * 16 + col;
        if (m >= p.M) continue;
        const float sa = p.scaleA[m];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = n0 + part * 4 + r;
            if (n < p.N) static_cast<T*>(p.out)[m * p.ldo + n] = fromFloat<T>(scaled(s[r], sa, p.scaleB[n], p.bias ? p.bias[n] : 0.f, activation, p.actParam));
        }
    }
}

// Any alignment: v_mfma_i32_32x32x32_i8, lane l holds 16 consecutive k (half l / 32) of row l % 32 of either operand; register r of the result is row
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
        if (m < p.M) static_cast<T*>(p.out)[m * p.ldo + n] = fromFloat<T>(scaled(acc[r], p.scaleA[m], sb, bias, activation, p.actParam));
    }
}

// Aligned rows: a tile of TM tokens x TN channels for WM x WN waves of 32 x 32 pieces, 128 bytes of k at a time, which go from memory into LDS without passing
// a register (two buffers: the next 128 bytes travel while these are multiplied).  LDS holds rows of eight 16-byte chunks, chunk c of row r at place c ^ swizzle(r) so that
// the 32 rows a wave reads at one k spread over all banks; the loads write LDS in lane order, so it is their source that is permuted.
// A wave's channels are paired -- column l of its piece j is channel 2 l + j -- so that a lane stores two adjacent outputs.
template <class T, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void matmul_int8_tile_kernel(const Int8Params p, const int activation, const int tilesM, const int tilesN) {
    constexpr int BK = 128, WAVES = WM * WN, PM = TM / WM / 32, PN = TN / WN / 32;
    static_assert(PN == 2, "a wave's channels are paired");
    constexpr int LOADS = (TM + TN) * BK / (64 * 16) / WAVES;  // 1 KiB each: eight rows
    static_assert((TM + TN) / 8 % WAVES == 0 && TM / 8 % LOADS == 0, "a wave's loads are all tokens' or all channels'");
    __shared__ __attribute__((aligned(1024))) signed char lds[2][(TM + TN) * BK];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Tiles of an XCD (workgroup id % 8) are neighbours, in columns of up to eight tiles of tokens: what one reads the others find in its L2.
    const unsigned tiles = unsigned(tilesM) * tilesN, id = blockIdx.x, share = tiles / 8, more = tiles % 8, xcd = id % 8;
    const unsigned at = xcd * share + min(xcd, more) + id / 8;
    const unsigned band = at / (8u * tilesN), inBand = at % (8u * tilesN), bandRows = min(8u, unsigned(tilesM) - band * 8);
    const long long m0 = (long long)(band * 8 + inBand % bandRows) * TM;
    const int n0 = int(inBand / bandRows) * TN;

    const int lr = lane >> 3;
    const signed char* source[LOADS];
    int chunk[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int row = (wave * LOADS + j) * 8 + lr;  // of the tile: tokens, then channels
        if (row < TM) {
            chunk[j] = ((lane & 7) ^ (row & 7)) * 16;
            source[j] = p.a + min(m0 + row, p.M - 1) * p.lda;
        } else {
            chunk[j] = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
            source[j] = p.b + (long long)min(n0 + row - TM, p.N - 1) * p.ldb;
        }
    }
    auto load = [&](int k0, int buffer) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int k = k0 + chunk[j];
            // (a chunk behind the row's end is never multiplied: any address will do)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(source[j] + (k < p.K ? k : 0)),
                                             (__attribute__((address_space(3))) void*)(&lds[buffer][(wave * LOADS + j) * 1024]), 16, 0, 0);
        }
    };
    const int wm = (wave / WN) * (PM * 32), wn = (wave % WN) * (PN * 32), col = lane & 31, half = lane >> 5;
    int16_t_ acc[PM][PN] = {};
    auto multiply = [&](int buffer, int kk, bool cut) {
        int4_t a[PM], b[PN];
#pragma unroll
        for (int i = 0; i < PM; ++i) {
            const int row = wm + i * 32 + col;
            a[i] = *reinterpret_cast<const int4_t*>(&lds[buffer][row * BK + (((kk * 2 + half) ^ (row & 7)) * 16)]);
        }
#pragma unroll
        for (int j = 0; j < PN; ++j) {
            const int row = wn + 2 * col + j;
            b[j] = *reinterpret_cast<const int4_t*>(&lds[buffer][(TM + row) * BK + (((kk * 2 + half) ^ ((row >> 1) & 7)) * 16)]);
            if (cut && half) b[j] = int4_t{0, 0, 0, 0};  // K ends in the middle of this step
        }
#pragma unroll
        for (int i = 0; i < PM; ++i)
#pragma unroll
            for (int j = 0; j < PN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    };
    load(0, 0);
    int buffer = 0, k0 = 0;
    for (; k0 + BK <= p.K; k0 += BK, buffer ^= 1) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the tile is in LDS
        __syncthreads();                     // everybody's is, and nobody reads the other buffer any more
        if (k0 + BK < p.K) load(k0 + BK, buffer ^ 1);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) multiply(buffer, kk, false);
    }
    if (k0 < p.K) {
        __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
#pragma unroll 1
        for (int left = p.K - k0, kk = 0; kk * 32 < left; ++kk) multiply(buffer, kk, left - kk * 32 < 32);
    }
    const int n = n0 + wn + 2 * col;
    float sb[2], bias[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int c = min(n + j, p.N - 1);
        sb[j] = p.scaleB[c];
        bias[j] = p.bias ? p.bias[c] : 0.f;
    }
    const bool paired = n + 1 < p.N && p.ldo % 2 == 0 && reinterpret_cast<size_t>(p.out) % (2 * sizeof(T)) == 0;
#pragma unroll
    for (int i = 0; i < PM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const long long m = m0 + wm + i * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
            if (m >= p.M) continue;
            const float sa = p.scaleA[m];
            T* const out = static_cast<T*>(p.out) + m * p.ldo + n;
            Pack<T, 2> o;
#pragma unroll
            for (int j = 0; j < 2; ++j) o.v[j] = fromFloat<T>(scaled(acc[i][j][r], sa, sb[j], bias[j], activation, p.actParam));
            if (paired) *reinterpret_cast<Pack<T, 2>*>(out) = o;
            else {
                if (n < p.N) out[0] = o.v[0];
                if (n + 1 < p.N) out[1] = o.v[1];
            }
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
        const bool aligned = multipleOf(p.a, 16) && multipleOf(p.b, 16) && p.lda % 16 == 0 && p.ldb % 16 == 0 && p.K % 16 == 0;
        auto few = [&](auto isAligned, auto tokens) {
            constexpr int MT = decltype(tokens)::value;
            const dim3 grid(unsigned((p.N + 15) / 16), unsigned((p.M + 16 * MT - 1) / (16 * MT)));
            matmul_int8_few_kernel<T, decltype(isAligned)::value, MT><<<grid, 512, 0, s>>>(p, activation);
            return hipGetLastError();
        };
        auto fewOf = [&](auto isAligned) {
            if (p.M <= 16) return few(isAligned, std::integral_constant<int, 1>{});
            if (p.M <= 32) return few(isAligned, std::integral_constant<int, 2>{});
            return few(isAligned, std::integral_constant<int, 4>{});
        };
        if (p.M <= 256) return aligned ? fewOf(std::true_type{}) : fewOf(std::false_type{});
        const long long big = ((p.M + 255) / 256) * ((p.N + 255) / 256);
        if (aligned && p.N > 64) {
            if (big >= 256 && p.K >= 1024) {
                matmul_int8_tile_kernel<T, 256, 256, 2, 4><<<unsigned(big), 512, 0, s>>>(p, activation, int((p.M + 255) / 256), (p.N + 255) / 256);
                return hipGetLastError();
            }
            const long long tilesM = (p.M + 127) / 128, tilesN = (p.N + 127) / 128;
            if (tilesM * tilesN < (1LL << 24)) {
                matmul_int8_tile_kernel<T, 128, 128, 2, 2><<<unsigned(tilesM * tilesN), 256, 0, s>>>(p, activation, int(tilesM), int(tilesN));
                return hipGetLastError();
            }
        }
        const dim3 grid(unsigned((p.M + 63) / 64), unsigned((p.N + 63) / 64));
        if (aligned) matmul_int8_kernel<T, true><<<grid, 256, 0, s>>>(p, activation);
        else matmul_int8_kernel<T, false><<<grid, 256, 0, s>>>(p, activation);
        return hipGetLastError();
    });
}

}  // namespace fvsrn
