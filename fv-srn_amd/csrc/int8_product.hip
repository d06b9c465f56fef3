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

// Bound by memory: every value is read once and a quarter or half of its bytes written.  `width` lanes share a row, 8 values of each in turn, in registers
// from the maximum to the codes (of rows longer than 8 width HELD the rest is read a second time, from the caches).  Short rows go ROWS at a time: one
// 16-byte load a lane would leave the memory idle.  Any alignment: the loads and stores of 8 values are as fast as the lines they touch.  Measured, fp16: 262144 x 256
// 35 - 41 us (202 MB, 5.0 - 5.8 TB/s), 200000 x 1000 114 us (5.3 TB/s), 100003 x 250 17 us (76 MB, 4.5 TB/s).
// The piece that a row's end cuts begins 8 before it instead (what it shares with the piece before is written twice, with the same codes); only rows of less
// than 8 go value by value.
__device__ __forceinline__ int pieceAt(int k, int cols) { return min(k, max(cols - 8, 0)); }

template <class T>
__device__ __forceinline__ void loadEight(const T* row, int k, int cols, T (&v)[8]) {
    if (cols >= 8) {
        loadWide<T, 8>(v, row + pieceAt(k, cols));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < cols ? row[j] : T(0.f);
    }
}

// The largest magnitude of pairs of values, by their bits: without its sign a float is ordered like its bits, and what is no finite number is above all others.
template <class T>
struct Largest {
    typedef unsigned word;
    static constexpr unsigned kInfinity = 0x7f800000u;
    word most = 0;
    __device__ __forceinline__ void look(const T (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    __device__ __forceinline__ unsigned key() const { return most; }
    static __device__ __forceinline__ float value(unsigned key) { return __uint_as_float(key); }
};
template <class T>
struct Largest16 {
    typedef unsigned short word __attribute__((ext_vector_type(2)));
    word most = {0, 0};
    __device__ __forceinline__ void look(const T (&v)[8]) {
        const word sign = {0x7fff, 0x7fff};
        word w[4];
        __builtin_memcpy(w, v, 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) most = __builtin_elementwise_max(most, w[j] & sign);
    }
    __device__ __forceinline__ unsigned key() const { return max(most.x, most.y); }
    static __device__ __forceinline__ float value(unsigned key) { return toFloat(__builtin_bit_cast(T, (unsigned short)key)); }
};
template <>
struct Largest<f16_t> : Largest16<f16_t> { static constexpr unsigned kInfinity = 0x7c00u; };
template <>
struct Largest<bf16_t> : Largest16<bf16_t> { static constexpr unsigned kInfinity = 0x7f80u; };

// The codes are the quotients v / scale rounded to 32 bits, rounded to integers.  A division is ten instructions, and they would be what the kernel waits for: where it
// can be, the quotient is q = v y with y = 1 / scale rounded, corrected by its exact remainder, q + (v - q scale) y, which is the rounded quotient
// (Markstein's theorem: y correctly rounded, the divisor's significand not all ones, nothing subnormal: `exact` says so).  Adding 1.5 2^23 leaves the nearest integer
// (ties to even) in the low bits.
template <class T>
__device__ __forceinline__ void storeEight(signed char* row, int k, int cols, const T (&v)[8], float scale, float y, bool exact, bool zero) {
    unsigned w[8], word[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = toFloat(v[j]), q = x * y;
        const float quotient = exact ? fmaf(fmaf(-q, scale, x), y, q) : __fdiv_rn(x, scale);
        w[j] = __float_as_uint(quotient + 12582912.f);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // the low bytes of four words
        const unsigned lo = __builtin_amdgcn_perm(w[4 * j + 1], w[4 * j], 0x0c0c0400u), hi = __builtin_amdgcn_perm(w[4 * j + 3], w[4 * j + 2], 0x04000c0cu);
        word[j] = zero ? 0u : lo | hi;
    }
    if (cols >= 8) {
        storeWide<signed char, 8>(row + pieceAt(k, cols), reinterpret_cast<const signed char*>(word));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < cols) row[j] = (signed char)(word[j >> 2] >> (8 * (j & 3)));
    }
}

template <class T, int HELD, int ROWS>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantizeParams p, const int width) {
    const int lane = threadIdx.x & 63, at = lane & (width - 1), group = (threadIdx.x >> 6) * (64 / width) + lane / width, groups = 4 * (64 / width);
    const long long first = blockIdx.x * (long long)(groups * ROWS) + group;  // rows first, first + groups, ...
    T v[ROWS][HELD][8];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const T* const x = static_cast<const T*>(p.x) + min(first + r * groups, p.rows - 1) * p.ldx;
#pragma unroll
        for (int j = 0; j < HELD; ++j) loadEight(x, (j * width + at) * 8, p.cols, v[r][j]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const long long row = min(first + r * groups, p.rows - 1);
        const T* const x = static_cast<const T*>(p.x) + row * p.ldx;
        Largest<T> largest;
#pragma unroll
        for (int j = 0; j < HELD; ++j) largest.look(v[r][j]);
        for (int k = (HELD * width + at) * 8; k < p.cols; k += width * 8) {
            T w[8];
            loadEight(x, k, p.cols, w);
            largest.look(w);
        }
        unsigned key = largest.key();
        for (int o = 1; o < width; o <<= 1) key = max(key, __shfl_xor(key, o, 64));
        if (first + r * groups >= p.rows) return;
        const bool bad = key >= Largest<T>::kInfinity;
        signed char* const q = p.codes + row * p.ldc;
        const float scale = fmaxf(Largest<T>::value(key) * (1.f / 127.f), 0x1p-126f);
        if (at == 0) p.scales[row] = bad ? __builtin_nanf("") : scale;
        const float y = __fdiv_rn(1.f, scale);
        const bool exact = scale > 0x1p-90f && (__float_as_uint(scale) & 0x7fffffu) != 0x7fffffu;
        auto store = [&](const T(&w)[8], int k) {
            // (a branch per row and not a choice per value)
            if (exact) storeEight(q, k, p.cols, w, scale, y, true, bad);
            else storeEight(q, k, p.cols, w, scale, y, false, bad);
        };
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int k = (j * width + at) * 8;
            if (k < p.cols) store(v[r][j], k);
        }
        for (int k = (HELD * width + at) * 8; k < p.cols; k += width * 8) {
            T w[8];
            loadEight(x, k, p.cols, w);
            store(w, k);
        }
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
template <int KIND>
__device__ __forceinline__ float activated(float y, float p) {
    constexpr double kTurn = 0.15915494309189535;  // 1 / (2 pi)
    if constexpr (KIND == FVSRN_ACT_RELU) {
        return y < 0.f ? 0.f : y;  // (NaN stays NaN)
    } else if constexpr (KIND == FVSRN_ACT_SINE) {
        return sineOfTurns(double(p * y) * kTurn);
    } else if constexpr (KIND == FVSRN_ACT_SNAKE) {
        const float s = sineOfTurns(double(p * y) * kTurn);
        return y + s * s / p;
    } else if constexpr (KIND == FVSRN_ACT_SNAKEALT) {
        return (y + 1.f - sineOfTurns(double(2.f * p * y) * kTurn + 0.25)) / (2.f * p);
    } else if constexpr (KIND == FVSRN_ACT_SIGMOID) {
        return 1.f / (1.f + expf(-y));
    } else {
        return y;
    }
}

// f(activation as a constant): one wave-uniform branch in front of the outputs of a wave
template <class F>
__device__ __forceinline__ void withActivation(int kind, F&& f) {
    switch (kind) {
        case FVSRN_ACT_RELU: return f(std::integral_constant<int, FVSRN_ACT_RELU>{});
        case FVSRN_ACT_SINE: return f(std::integral_constant<int, FVSRN_ACT_SINE>{});
        case FVSRN_ACT_SNAKE: return f(std::integral_constant<int, FVSRN_ACT_SNAKE>{});
        case FVSRN_ACT_SNAKEALT: return f(std::integral_constant<int, FVSRN_ACT_SNAKEALT>{});
        case FVSRN_ACT_SIGMOID: return f(std::integral_constant<int, FVSRN_ACT_SIGMOID>{});
        default: return f(std::integral_constant<int, FVSRN_ACT_NONE>{});
    }
}

// Sums of products are exact whatever their order, so k may be cut and joined anywhere.

// 16 bytes of a row from column k, zeros behind the row's end, in two steps so that many loads are on their way before the first is looked at.
//   kAligned: k and the row start are multiples of 16, and so is K: no chunk is cut, and one behind the end (the row's start is read for it) is dropped.
//   Otherwise the row's last 16 bytes are read where the chunk reaches behind its end, and shifted down: in one load at whatever address (kBytes), or as the five
// aligned words that hold them (kWords).  An odd address makes a load several times as long, a fifth word a quarter: with few waves on the way through k the words win
// (64 x 4096 x 4095 20 against 39 us, 100003 x 4 x 250 10 against 13), in tiles, which wait for LDS and not for these, the single load (8192 x
// 4096 x 4095 160 against 204 us).  A word is read only if one of its bytes is the row's, and an aligned word never leaves a page, so nothing is touched that the
// row does not share with its neighbours.
enum CodeLoads { kAligned, kWords, kBytes };
template <CodeLoads HOW>
struct Codes {
    static constexpr bool ALIGNED = HOW == kAligned;
    int4_t v;
    unsigned w;

    static __device__ __forceinline__ const signed char* start(const signed char* row, int k, int K) { return row + min(k, max(K - 16, 0)); }

    __device__ __forceinline__ void load(const signed char* row, int k, int K) {
        if (ALIGNED) {
            v = *reinterpret_cast<const int4_t*>(row + (k < K ? k : 0));
        } else if (K >= 16 && HOW == kBytes) {
            __builtin_memcpy(&v, start(row, k, K), 16);
        } else if (K >= 16) {
            const size_t at = reinterpret_cast<size_t>(start(row, k, K));
            const unsigned* const words = reinterpret_cast<const unsigned*>(at & ~size_t(3));
            unsigned from[4];
            loadWide<unsigned, 4>(from, words);
            __builtin_memcpy(&v, from, 16);
            w = words[at & 3 ? 4 : 3];
        } else {
            v = int4_t{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 15; ++j)
                if (j < K) v[j >> 2] |= int(static_cast<unsigned char>(row[j])) << (8 * (j & 3));
        }
    }

    // cut: whether K may end in or before this chunk
    __device__ __forceinline__ int4_t get(const signed char* row, int k, int K, bool cut) const {
        if (ALIGNED || K < 16) return !cut || k < K ? v : int4_t{0, 0, 0, 0};
        typedef unsigned long long word_t;
        unsigned u[4];
        if (HOW == kWords) {
            const unsigned odd = unsigned(reinterpret_cast<size_t>(start(row, k, K))) & 3;
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = __builtin_amdgcn_alignbyte(j < 3 ? unsigned(v[j + 1]) : w, unsigned(v[j]), odd);
        } else {
            __builtin_memcpy(u, &v, 16);
        }
        if (cut) {
            const int bits = 8 * max(0, k + 16 - K);  // how far the load began before k: below 128 in a chunk that has bytes of the row
            const word_t lo = u[0] | word_t(u[1]) << 32, hi = u[2] | word_t(u[3]) << 32;
            const word_t low = bits >= 128 ? 0 : bits >= 64 ? hi >> (bits & 63) : bits > 0 ? lo >> bits | hi << (64 - bits) : lo;
            const word_t high = bits >= 64 ? 0 : hi >> bits;
            u[0] = unsigned(low);
            u[1] = unsigned(low >> 32);
            u[2] = unsigned(high);
            u[3] = unsigned(high >> 32);
        }
        return int4_t{int(u[0]), int(u[1]), int(u[2]), int(u[3])};
    }
};

template <int KIND>
__device__ __forceinline__ float scaled(int acc, float sa, float sb, float bias, float param) {
    return activated<KIND>(fmaf(float(acc) * sb, sa, bias), param);
}

// Few tokens: bound by the weights' bytes, or by how long one wave takes through its part of k.  v_mfma_i32_16x16x64_i8 with the weights as its rows: lane l holds 16
// consecutive k (part l / 16) of channel l % 16 and of token l % 16; register r of the result is channel 4 (l / 16) + r, token l % 16.  A workgroup has 16 channels and 16 MT
// tokens; its eight waves take every eighth 256 bytes of k straight from memory into registers -- each weight is read once by the chip, nothing is
// worth a turn through LDS but the eight sums at the end.  1 x 4096 x 4096: 5.6 us (17 MB, 3.0 TB/s: the launch and one way through the memory are most of it).
template <class T, CodeLoads HOW, int MT>
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
        Codes<HOW> b[U], a[MT][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * 64 + part * 16;
            b[u].load(br, k, p.K);
#pragma unroll
            for (int t = 0; t < MT; ++t) a[t][u].load(ar[t], k, p.K);
        }
        // (the same for all lanes; both operands are cut: what lies behind K in one is not 0 in the other)
        auto multiply = [&](bool cut) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * 64 + part * 16;
                const int4_t bu = b[u].get(br, k, p.K, cut);
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bu, a[t][u].get(ar[t], k, p.K, cut), acc[t], 0, 0, 0);
            }
        };
        if (k0 + 64 * U > p.K) multiply(true);
        else multiply(false);
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
        withActivation(activation, [&](auto kind) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + part * 4 + r;
                if (n < p.N)
                    static_cast<T*>(p.out)[m * p.ldo + n] = fromFloat<T>(scaled<decltype(kind)::value>(s[r], sa, p.scaleB[n], p.bias ? p.bias[n] : 0.f, p.actParam));
            }
        });
    }
}

// Few channels (the last layer of a network) for many tokens: bound by the tokens' bytes.  The same instruction with the same operands -- 16 channels as its rows, 16
// tokens as its columns, a lane's four results four channels of one token -- but a wave takes 64 tokens through all of k, and nothing is joined.  200000 x 16 x 1000:
// 60 us (206 MB, 3.4 TB/s), 100003 x 4 x 250 10 - 12 us.
template <class T, CodeLoads HOW>
__global__ __launch_bounds__(256) void matmul_int8_narrow_kernel(const Int8Params p, const int activation) {
    constexpr int GROUPS = 4;
    const int lane = threadIdx.x & 63, col = lane & 15, part = lane >> 4;
    const long long m0 = (blockIdx.x * 4LL + (threadIdx.x >> 6)) * (16 * GROUPS);
    if (m0 >= p.M) return;
    const signed char* const br = p.b + (long long)min(col, p.N - 1) * p.ldb;
    const signed char* ar[GROUPS];
#pragma unroll
    for (int t = 0; t < GROUPS; ++t) ar[t] = p.a + min(m0 + t * 16 + col, p.M - 1) * p.lda;
    int4_t acc[GROUPS] = {};
#pragma unroll 2
    for (int k = part * 16; k < p.K + part * 16; k += 64) {  // (as many steps for every lane)
        Codes<HOW> b, a[GROUPS];
        b.load(br, k, p.K);
#pragma unroll
        for (int t = 0; t < GROUPS; ++t) a[t].load(ar[t], k, p.K);
        const bool cut = k - part * 16 + 64 > p.K;
        const int4_t bk = b.get(br, k, p.K, cut);
#pragma unroll
        for (int t = 0; t < GROUPS; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bk, a[t].get(ar[t], k, p.K, cut), acc[t], 0, 0, 0);
    }
    const int n = part * 4;
    if (n >= p.N) return;
    float sb[4], bias[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int c = min(n + r, p.N - 1);
        sb[r] = p.scaleB[c];
        bias[r] = p.bias ? p.bias[c] : 0.f;
    }
    withActivation(activation, [&](auto kind) {
#pragma unroll
        for (int t = 0; t < GROUPS; ++t) {
            const long long m = m0 + t * 16 + col;
            if (m >= p.M) continue;
            const float sa = p.scaleA[m];
            T o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fromFloat<T>(scaled<decltype(kind)::value>(acc[t][r], sa, sb[r], bias[r], p.actParam));
            T* const out = static_cast<T*>(p.out) + m * p.ldo + n;
            if (n + 4 <= p.N) {
                storeWide<T, 4>(out, o);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < p.N) out[r] = o[r];
            }
        }
    });
}

// A tile of TM tokens x TN channels for WM x WN waves, each with PM x 2 pieces of 32 x 32, 64 bytes of k a stage.  v_mfma_i32_32x32x32_i8: lane l holds 16
// consecutive k (half l / 32) of row l % 32 of either operand; register r of the result is row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32.
//   Stages go from memory into LDS without passing a register, into a ring of RING: while one is multiplied the others travel (a stage of 256 x 256 is multiplied in
// 0.4 us, which is less than the way from memory).  The wait for the next stage and the barrier stand between the two halves of a stage's products, and the
// operands of a half are read while the half before is multiplied, so the matrix units have work queued at every wait.
//   Not DIRECT (rows that are not aligned to 16 bytes): a stage goes through registers, asked for a stage ahead of its way into a ring of two -- unaligned addresses
// are for registers only, and so is the masking of the chunk in which K ends.
//   LDS holds rows of four 16-byte chunks, chunk c of row r at place c ^ (r / 4) % 4, so that 16 rows read at one k lie in 64 different banks; the loads write LDS in
// lane order, so it is their source that is permuted.  A wave's channels are paired -- column l of its piece j is channel 2 l + j -- so that a lane stores two adjacent
// outputs and a wave whole 128-byte lines of 16-bit ones; they lie in LDS in the order in which they are read (every second row would meet every second
// bank twice: half of the LDS cycles).
//   Measured: 8192 x 4096 x 4096 127 - 138 us by card (2.0 - 2.16 POP/s; the matrix units have 64 of 100 cycles of the CUs, LDS reads and writes as many, at a clock that falls to
// 1.65 - 1.85 GHz under them; two workgroups of 256 x 128 a CU, which load half as much again: 147 - 153 us against 133), 262144 x 256 x 256 43 - 46 us
// (201 MB, 4.4 - 4.7 TB/s).
template <class T, int TM, int TN, int WM, int WN, int RING, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void matmul_int8_tile_kernel(const Int8Params p, const int activation, const int tilesM, const int tilesN) {
    constexpr int BK = 64, WAVES = WM * WN, PM = TM / WM / 32, STAGE = (TM + TN) * BK;
    static_assert(TN / WN == 64, "a wave's channels are paired");
    constexpr int LOADS = STAGE / 1024 / WAVES;  // of a wave, 1 KiB each: 16 rows
    static_assert(STAGE % (1024 * WAVES) == 0 && LOADS * (RING - 2) < 64, "the waits below count loads");
    static_assert(DIRECT || RING == 2, "through registers two buffers do");
    constexpr int FLOWING = LOADS * (RING - 2);  // loads that may still be on their way when the next stage is waited for
    __shared__ __attribute__((aligned(1024))) signed char lds[RING][STAGE];
    __shared__ __attribute__((aligned(16))) float scaleA[TM], scaleB[TN], bias[TN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Tiles of an XCD (workgroup id % 8) are neighbours, in columns of up to eight tiles of tokens: what one reads the others find in its L2.
    const unsigned tiles = unsigned(tilesM) * tilesN, id = blockIdx.x, share = tiles / 8, more = tiles % 8, xcd = id % 8;
    const unsigned at = xcd * share + min(xcd, more) + id / 8;
    const unsigned band = at / (8u * tilesN), inBand = at % (8u * tilesN), bandRows = min(8u, unsigned(tilesM) - band * 8);
    const long long m0 = (long long)(band * 8 + inBand % bandRows) * TM;
    const int n0 = int(inBand / bandRows) * TN;

    const signed char* source[LOADS];
    int chunk[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int row = (wave * LOADS + j) * 16 + (lane >> 2);  // of the tile: tokens, then channels, of each 64 the even ones before the odd ones
        const bool token = row < TM;
        const int channel = ((row - TM) & ~63) + 2 * (row & 31) + ((row >> 5) & 1);
        chunk[j] = ((lane & 3) ^ ((row >> 2) & 3)) * 16;
        source[j] = (token ? p.a + min(m0 + row, p.M - 1) * p.lda : p.b + (long long)min(n0 + channel, p.N - 1) * p.ldb) + (DIRECT ? chunk[j] : 0);
    }
    const int stages = (p.K + BK - 1) / BK;
    Codes<kBytes> staged[LOADS];
    auto fetch = [&](int stage) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) staged[j].load(source[j], stage * BK + chunk[j], p.K);
    };
    auto put = [&](int stage, bool cut) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            *reinterpret_cast<int4_t*>(&lds[stage % RING][(wave * LOADS + j) * 1024 + lane * 16]) = staged[j].get(source[j], stage * BK + chunk[j], p.K, cut);
    };
    auto load = [&](int stage) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int k = stage * BK;
            // (a chunk behind the row's end meets zeros in the other operand: any address of the row will do)
            const signed char* const from = source[j] + (k + chunk[j] < p.K ? k : -chunk[j]);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                             (__attribute__((address_space(3))) void*)(&lds[stage % RING][(wave * LOADS + j) * 1024]), 16, 0, 0);
        }
    };
    const int wm = (wave / WN) * (PM * 32), wn = (wave % WN) * 64, col = lane & 31, half = lane >> 5;
    struct Operands { int4_t a[PM], b[2]; };
    auto read = [&](Operands& o, int stage, int kk) {
        const signed char* const buffer = lds[stage % RING];
#pragma unroll
        for (int i = 0; i < PM; ++i) {
            const int row = wm + i * 32 + col;
            o.a[i] = *reinterpret_cast<const int4_t*>(buffer + row * BK + (((kk * 2 + half) ^ ((row >> 2) & 3)) * 16));
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = TM + wn + j * 32 + col;
            o.b[j] = *reinterpret_cast<const int4_t*>(buffer + row * BK + (((kk * 2 + half) ^ ((row >> 2) & 3)) * 16));
        }
    };
    int16_t_ acc[PM][2] = {};
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int i = 0; i < PM; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(o.a[i], o.b[j], acc[i][j], 0, 0, 0);
    };
    for (int e = threadIdx.x; e < TM; e += 64 * WAVES) scaleA[e] = p.scaleA[min(m0 + e, p.M - 1)];
    for (int e = threadIdx.x; e < TN; e += 64 * WAVES) {
        const int n = min(n0 + e, p.N - 1);
        scaleB[e] = p.scaleB[n];
        bias[e] = p.bias ? p.bias[n] : 0.f;
    }
    // The next stage is everybody's to read behind the barrier, and nobody reads the one before it any more.  RING - 2 stages may still be on their way (FLOWING
    // loads of this wave); at the end of k all have to be there.
    auto arrive = [&](bool flowing) {
        if (flowing) __builtin_amdgcn_s_waitcnt((FLOWING & 15) | (FLOWING >> 4) << 14 | 0x0070);  // vmcnt(FLOWING) lgkmcnt(0)
        else __builtin_amdgcn_s_waitcnt(0x0070);                                                  // vmcnt(0) lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
    };
    Operands even, odd;
    if constexpr (DIRECT) {
        for (int s = 0; s < min(RING - 1, stages); ++s) load(s);
        arrive(stages >= RING - 1);
        read(even, 0, 0);
#pragma unroll 1
        for (int s = 0; s < stages - 1; ++s) {
            if (s + RING - 1 < stages) load(s + RING - 1);
            read(odd, s, 1);
            multiply(even);
            arrive(s + RING - 1 < stages);
            read(even, s + 1, 0);
            multiply(odd);
        }
    } else {
        fetch(0);
        put(0, true);
        if (stages > 1) fetch(1);
        __syncthreads();
        read(even, 0, 0);
#pragma unroll 1
        for (int s = 0; s < stages - 1; ++s) {
            // (nobody reads stage s - 1 any more since the last barrier)
            if ((s + 2) * BK > p.K) put(s + 1, true);
            else put(s + 1, false);
            if (s + 2 < stages) fetch(s + 2);
            read(odd, s, 1);
            multiply(even);
            // (lgkmcnt(0) only: what was fetched stays on its way)
            __builtin_amdgcn_s_waitcnt(0xc07f);
            asm volatile("s_barrier" ::: "memory");
            read(even, s + 1, 0);
            multiply(odd);
        }
    }
    // the last stage: zeros in the place of what lies behind K
    read(odd, stages - 1, 1);
    const int left = p.K - (stages - 1) * BK;
    const int4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        even.b[j] = half * 16 < left ? even.b[j] : zero;
        odd.b[j] = 32 + half * 16 < left ? odd.b[j] : zero;
    }
    multiply(even);
    multiply(odd);
    const int cn = wn + 2 * col, n = n0 + cn;
    const float sb0 = scaleB[cn], sb1 = scaleB[cn + 1], bias0 = bias[cn], bias1 = bias[cn + 1];
    const bool paired = p.ldo % 2 == 0 && reinterpret_cast<size_t>(p.out) % (2 * sizeof(T)) == 0;
    T* const out = static_cast<T*>(p.out) + (m0 + wm + 4 * half) * p.ldo + n;
    const long long rows = p.M - (m0 + wm + 4 * half);
    auto store = [&](auto kind, auto isWhole) {
#pragma unroll
        for (int i = 0; i < PM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 sa = *reinterpret_cast<const float4*>(&scaleA[wm + i * 32 + 8 * q + 4 * half]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    constexpr int A = decltype(kind)::value;
                    const int row = i * 32 + 8 * q + r;
                    const float s = r == 0 ? sa.x : r == 1 ? sa.y : r == 2 ? sa.z : sa.w;
                    Pack<T, 2> o;
                    o.v[0] = fromFloat<T>(scaled<A>(acc[i][0][4 * q + r], s, sb0, bias0, p.actParam));
                    o.v[1] = fromFloat<T>(scaled<A>(acc[i][1][4 * q + r], s, sb1, bias1, p.actParam));
                    T* const to = out + row * p.ldo;
                    if (decltype(isWhole)::value) {
                        *reinterpret_cast<Pack<T, 2>*>(to) = o;
                    } else if (row < rows) {
                        if (n < p.N) to[0] = o.v[0];
                        if (n + 1 < p.N) to[1] = o.v[1];
                    }
                }
            }
    };
    withActivation(activation, [&](auto kind) {
        if (paired && m0 + TM <= p.M && n0 + TN <= p.N) store(kind, std::true_type{});
        else store(kind, std::false_type{});
    });
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

// 16 values of a lane in rows of up to 1024: what a row costs beside its values -- the maximum's way through the lanes, the reciprocal -- is spread over them
int quantizeWidth(int cols) { return std::min(64, powerOfTwoAtLeast(cols <= 1024 ? (cols + 15) / 16 : (cols + 7) / 8)); }

hipError_t launch_quantize_rows(const QuantizeParams& p, int dtype, hipStream_t s) {
    return withType(dtype, [&](auto element) {
        typedef decltype(element) T;
        const int width = quantizeWidth(p.cols);
        auto launch = [&](auto held, auto rows) {
            constexpr int H = decltype(held)::value, R = decltype(rows)::value;
            const long long rowsOfBlock = 4 * (64 / width) * R;
            quantize_rows_kernel<T, H, R><<<unsigned((p.rows + rowsOfBlock - 1) / rowsOfBlock), 256, 0, s>>>(p, width);
            return hipGetLastError();
        };
        // (rows at a time: only where there are enough of them for 8 waves on each CU all the same)
        if (p.cols <= 1024 && p.rows * width >= 4LL * 64 * 2048) return launch(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
        if (p.cols <= 1024) return launch(std::integral_constant<int, 2>{}, std::integral_constant<int, 1>{});
        if (p.cols <= 2048) return launch(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
        return launch(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    });
}

hipError_t launch_matmul_int8(const Int8Params& p, int activation, int outDtype, hipStream_t s) {
    return withType(outDtype, [&](auto element) {
        typedef decltype(element) T;
        const bool aligned = multipleOf(p.a, 16) && multipleOf(p.b, 16) && p.lda % 16 == 0 && p.ldb % 16 == 0 && p.K % 16 == 0;
        using std::integral_constant;
        auto few = [&](auto loads, auto tokens) {
            constexpr int MT = decltype(tokens)::value;
            const dim3 grid(unsigned((p.N + 15) / 16), unsigned((p.M + 16 * MT - 1) / (16 * MT)));
            matmul_int8_few_kernel<T, decltype(loads)::value, MT><<<grid, 512, 0, s>>>(p, activation);
            return hipGetLastError();
        };
        auto fewOf = [&](auto loads) {
            if (p.M <= 16) return few(loads, integral_constant<int, 1>{});
            if (p.M <= 32) return few(loads, integral_constant<int, 2>{});
            return few(loads, integral_constant<int, 4>{});
        };
        auto tiles = [&](int edge) { return ((p.M + edge - 1) / edge) * ((p.N + edge - 1) / edge); };
        // (up to 64 tokens, unless there are channels enough for tiles on every CU: 33 x 16384 x 2047 34 us this way, 20 in tiles; 64 x 4096 x 4096 13 and 17)
        if (p.M <= 16 || (p.M <= 64 && tiles(64) < 256)) return aligned ? fewOf(integral_constant<CodeLoads, kAligned>{}) : fewOf(integral_constant<CodeLoads, kWords>{});
        if (p.N <= 16) {
            const unsigned grid = unsigned((p.M + 255) / 256);
            if (aligned) matmul_int8_narrow_kernel<T, kAligned><<<grid, 256, 0, s>>>(p, activation);
            else matmul_int8_narrow_kernel<T, kWords><<<grid, 256, 0, s>>>(p, activation);
            return hipGetLastError();
        }
        // The largest tile that still gives every CU one (edges of 256 only with k long enough to hide their beginning and end: one fits a CU). 8192 x 4096 x 4096: 133
        // us with 256, 180 with 128, 300 with 64; 262144 x 256 x 256: 46, 43, 61 us; 2048 x 1024 x 1024: 16, 10, 9 us.  (256 in eight waves of 128 x 64, which read less LDS
        // than sixteen of 64 x 64: 133 against 137 us.)
        auto launch = [&](auto edge, auto wavesM, auto wavesN, auto ring) {
            constexpr int E = decltype(edge)::value, WM = decltype(wavesM)::value, WN = decltype(wavesN)::value, R = decltype(ring)::value;
            const int tilesM = int((p.M + E - 1) / E), tilesN = (p.N + E - 1) / E;
            if (aligned) matmul_int8_tile_kernel<T, E, E, WM, WN, R, true><<<unsigned(tiles(E)), 64 * WM * WN, 0, s>>>(p, activation, tilesM, tilesN);
            else matmul_int8_tile_kernel<T, E, E, WM, WN, 2, false><<<unsigned(tiles(E)), 64 * WM * WN, 0, s>>>(p, activation, tilesM, tilesN);
            return hipGetLastError();
        };
        if (tiles(256) >= 256 && p.K >= 1024) return launch(integral_constant<int, 256>{}, integral_constant<int, 2>{}, integral_constant<int, 4>{}, integral_constant<int, 4>{});
        if (tiles(128) >= 256) return launch(integral_constant<int, 128>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{}, integral_constant<int, 3>{});
        return launch(integral_constant<int, 64>{}, integral_constant<int, 2>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
    });
}

}  // namespace fvsrn
