// The gated linear recurrence h_t = a_t h_{t-1} + u_t and its gradients (include/fvsrn.h, fvsrn_gated_scan*).
//
// A span of steps acts on the state that enters it as h -> A h + U with A = prod a_t and U = the state it reaches from 0; two spans join as
// (A2 A1, A2 U1 + U2).  The gradient k that a span passes to the step before it acts the other way round, k -> A k + D, with the same A: with
// L_t = dout_t + k_{t+1}, k_t = a_t L_t.  So both passes are: fold spans, join them, walk each span again from its true entry state.
//
// Bound by memory: 2 - 3 elements move per step and channel against a handful of multiply-adds.  Two ways to lay a wave onto the data:
//   channels  lanes are channels, steps run in registers; waves of a workgroup take consecutive spans of a tile of steps and join through LDS
//   rows      lanes are consecutive steps of one gate with its (up to four) channels beside each other -- the layout of colours along a ray -- and
//             join by lane shuffles
#include "tensor_ops.hpp"

#include <algorithm>
#include <cmath>

#include "../../include/fvsrn.h"
#include "tensor_elements.hpp"

namespace fvsrn {
namespace {

// A gate a and 1 - a, both to about an ulp of their own: a gate next to 1 is raised to the length of the series, a sample of a thin medium is all of its
// 1 - a, and a dense one's a is all that is left of what lies behind it.  EXP: y = n ln 2 + r with |r| <= ln 2 / 2 (Cody and Waite's two-part ln 2) and the
// Taylor series of q = exp(r) - 1 (the first term left out is r^9 / 9!, 6e-10 of r): a = 2^n + 2^n q, 1 - a = -((2^n - 1) + 2^n q).
template <bool EXP>
__device__ __forceinline__ void gateOf(float g, float scale, float& a, float& rest) {
    if constexpr (EXP) {
        float y = scale * g;
        y = y < -110.f ? -110.f : y;  // (exp(-110) is 0 in 32 bits; NaN stays NaN)
        const float n = fminf(__builtin_rintf(y * 1.44269504f), 127.f);
        float r = fmaf(n, -0.693145752f, y);
        r = fmaf(n, -1.42860677e-6f, r);
        float q = fmaf(r, 1.f / 40320.f, 1.f / 5040.f);
        q = fmaf(r, q, 1.f / 720.f);
        q = fmaf(r, q, 1.f / 120.f);
        q = fmaf(r, q, 1.f / 24.f);
        q = fmaf(r, q, 1.f / 6.f);
        q = fmaf(r, q, 0.5f);
        q = fmaf(r * r, q, r);
        const float two = __builtin_amdgcn_ldexpf(1.f, int(n));
        a = fmaf(two, q, two);
        rest = -fmaf(two, q, two - 1.f);
    } else {
        a = g;
        rest = 1.f - g;
    }
}

// A barrier for what goes through LDS: __syncthreads would also wait for the stores of the last tile and the loads of the next one.
__device__ __forceinline__ void ldsBarrier() {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
}

__device__ __forceinline__ int lengthOf(const ScanParams& p, long long b) {
    return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}
// step i of a sequence of n steps is at position t; behind the sequence (outputs are zero there) i is the position itself
__device__ __forceinline__ int positionOf(int i, int n, int reverse) { return reverse && i < n ? n - 1 - i : i; }

// ---------------------------------------------------------------------------------------------------------------------
// lanes are channels
// ---------------------------------------------------------------------------------------------------------------------

constexpr int kScanWaves = 8;  // waves that share a tile
// steps of a wave that are held in registers, for V channels of a lane
// (twice as many cost more waves than they hide latency: series of 65536 x 1024 bf16 150 us against 132; backward, 16-bit pairs are better off with 8 steps and
// the four registers they spill at four waves a SIMD: 224 us against 259)
constexpr int forwardSteps(int V) { return V == 1 ? 16 : V == 2 ? 8 : 4; }
constexpr int backwardSteps(int V, int elementBytes) { return V == 1 || (V == 2 && elementBytes == 2) ? 8 : 4; }

// What a lane stands for: V adjacent channels, each with a gate of its own, or (SHARED) the V channels of one gate.  V == 1 and slots > 1 (backward, gates
// of many channels): `slots` lanes of a gate's channels -- padded to a power of two, so that their sum is a butterfly of shuffles -- and, for
// gates of more than 64 channels, `parts` waves.
struct ChannelLane {
    int c, g, part;
    bool live;
};
template <int V, bool SHARED>
__device__ __forceinline__ ChannelLane channelLane(const ScanParams& p, int block, int lane, int slots, int parts) {
    ChannelLane r;
    r.part = 0;
    if (V > 1 || slots == 1) {
        const long long own = block * 64LL + lane, last = p.C / V - 1;
        r.live = own <= last;
        r.c = int(min(own, last)) * V;
        r.g = SHARED ? r.c / V : V > 1 ? r.c : r.c / p.G;
    } else if (parts == 1) {
        const int j = lane & (slots - 1);
        const long long g = (long long)block * (64 / slots) + lane / slots;
        r.live = g < p.Cg && j < p.G;
        r.g = int(min(g, (long long)(p.Cg - 1)));
        r.c = r.g * p.G + min(j, p.G - 1);
    } else {
        r.g = block / parts;
        r.part = block % parts;
        const int j = r.part * 64 + lane;
        r.live = j < p.G;
        r.c = r.g * p.G + min(j, p.G - 1);
    }
    return r;
}
inline long long channelBlocks(const ScanParams& p, const ScanPlan& plan) {
    if (plan.slots == 1) return (p.C / plan.vec + 63LL) / 64;
    if (plan.parts == 1) return (p.Cg + 64 / plan.slots - 1) / (64 / plan.slots);
    return (long long)p.Cg * plan.parts;
}

// V channels of steps i .. i + L - 1, zeros from step `end` on
template <class T, int V, int L>
__device__ __forceinline__ void loadChannels(const T* p, long long step, int i, int n, int end, int reverse, T (&to)[L][V]) {
    if (i >= end) {  // (these conditions are the same for all lanes)
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) to[k][v] = T(0.f);
    } else if (i + L <= end) {
        const T* at = p + positionOf(i, n, reverse) * step;
        const long long next = reverse ? -step : step;
#pragma unroll
        for (int k = 0; k < L; ++k) loadWide<T, V>(to[k], at + k * next);
    } else {  // every load is made, the last step's again for those behind it: a branch for each would have them wait for each other
#pragma unroll
        for (int k = 0; k < L; ++k) loadWide<T, V>(to[k], p + positionOf(min(i + k, end - 1), n, reverse) * step);
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) to[k][v] = i + k < end ? to[k][v] : T(0.f);
    }
}

// The gates of steps i .. i + L - 1 (1 from step `end` on), and the factor of x: 1 - a of BLEND, 1 of ADD.  use(k, v, a, factor)
template <class T, int V, int L, class F>
__device__ __forceinline__ void withGates(const ScanParams& p, const T (&raw)[L][V], int i, int end, F&& use) {
    if (p.exp) {
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, rest;
                gateOf<true>(toFloat(raw[k][v]), p.scale, a, rest);
                use(k, v, a, p.blend ? rest : 1.f);
            }
    } else {
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, rest;
                gateOf<false>(toFloat(raw[k][v]), p.scale, a, rest);
                if (i + L > end && i + k >= end) a = 1.f;  // (read as 0; a gate of 0 in EXP is 1 already, and x is 0)
                use(k, v, a, p.blend ? rest : 1.f);
            }
    }
}

// The state behind spans 0 .. count - 1 of a call that is cut into them, from their (A, U) (of span 0 U is the state, whatever its A): the waves fold a part each and join.
// One after the other the folds of 127 spans took 20 us, which is most of what a span's steps take.
template <int NW, int V, int GV>
__device__ __forceinline__ void foldBefore(const float* wa, const float* wu, long long stride, int count, int w, int lane, float (&joined)[NW][GV + V][64], float (&h)[V]) {
    const int each = (count + NW - 1) / NW, last = min(count, (w + 1) * each);
    float A[GV], U[V];
#pragma unroll
    for (int v = 0; v < GV; ++v) A[v] = 1.f;
#pragma unroll
    for (int v = 0; v < V; ++v) U[v] = 0.f;
#pragma unroll 4
    for (int s = w * each; s < last; ++s) {
        float a[GV];
#pragma unroll
        for (int v = 0; v < GV; ++v) {
            a[v] = s == 0 ? 0.f : wa[s * stride + v];
            A[v] *= a[v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) U[v] = fmaf(a[GV == V ? v : 0], U[v], wu[s * stride + v]);
    }
#pragma unroll
    for (int v = 0; v < GV; ++v) joined[w][v][lane] = A[v];
#pragma unroll
    for (int v = 0; v < V; ++v) joined[w][GV + v][lane] = U[v];
    ldsBarrier();
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = 0.f;
#pragma unroll 2
    for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(joined[j][GV == V ? v : 0][lane], h[v], joined[j][GV + v][lane]);
}

// What spans first .. count - 1 pass back of the gradient k that enters them from behind, from their (A, D)
template <int NW, int V, int GV>
__device__ __forceinline__ void foldBehind(const float* wa, const float* wd, long long stride, int first, int count, int w, int lane, float (&joined)[NW][GV + V][64], float (&k)[V]) {
    const int each = (max(0, count - first) + NW - 1) / NW, from = min(count, first + w * each), last = min(count, from + each);
    float A[GV], D[V];
#pragma unroll
    for (int v = 0; v < GV; ++v) A[v] = 1.f;
#pragma unroll
    for (int v = 0; v < V; ++v) D[v] = 0.f;
#pragma unroll 4
    for (int s = from; s < last; ++s) {
#pragma unroll
        for (int v = 0; v < V; ++v) D[v] = fmaf(A[GV == V ? v : 0], wd[s * stride + v], D[v]);
#pragma unroll
        for (int v = 0; v < GV; ++v) A[v] *= wa[s * stride + v];
    }
#pragma unroll
    for (int v = 0; v < GV; ++v) joined[w][v][lane] = A[v];
#pragma unroll
    for (int v = 0; v < V; ++v) joined[w][GV + v][lane] = D[v];
    ldsBarrier();
#pragma unroll 2
    for (int j = NW - 1; j >= 0; --j)
#pragma unroll
        for (int v = 0; v < V; ++v) k[v] = fmaf(joined[j][GV == V ? v : 0][lane], k[v], joined[j][GV + v][lane]);
}

// Forward.  AGGREGATE: only (A, U) of this workgroup's span, span 0 with h0 folded in (its A slot then holds h0 for the second launch: d_last may be d_h0).  The second
// launch takes the spans from the last to the first: what the first launch read last is what the memory-side cache still holds.
// Measured: 65536 x 1024 bf16 61 us for the spans (268 MB, 4.4 TB/s) and 79 us for the walk (405 MB, 5.1 TB/s); 64 x 512 x 4096 bf16 in one launch 149 us (805 MB,
// 5.4 TB/s).
template <class T, int NW, int V, bool SHARED, bool AGGREGATE>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void scan_channels_kernel(const ScanParams p, const ScanPlan plan, const int blocks, const long long units) {
    constexpr int L = forwardSteps(V), GV = SHARED ? 1 : V;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (known to be the same for a wave: its addresses are scalars)
    const int w = NW == 1 ? 0 : wave;
    const long long unit = NW == 1 ? blockIdx.x * 4LL + wave : blockIdx.x;
    if (unit >= units) return;  // (NW == 1 only, and nothing is joined across its waves)
    const long long b = unit / blocks;
    const ChannelLane ch = channelLane<V, SHARED>(p, int(unit % blocks), lane, 1, 1);
    const int n = lengthOf(p, b), span = AGGREGATE ? blockIdx.y : gridDim.y - 1 - blockIdx.y;
    const int begin = span * plan.chunkSteps, end = min(p.out ? p.T : n, begin + plan.chunkSteps), inside = min(n, end);
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + ch.g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + ch.c * p.xs[2];
    T* const op = p.out ? static_cast<T*>(p.out) + b * p.os[0] + ch.c * p.os[2] : nullptr;
    const long long state = b * p.C + ch.c, stored = (b * plan.chunks) * p.C + ch.c, plane = p.B * plan.chunks * p.C;
    float h[V], A[GV];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = 0.f;
#pragma unroll
    for (int v = 0; v < GV; ++v) A[v] = 1.f;
    if (span == 0 && (AGGREGATE || plan.chunks == 1)) {
        if (p.h0)
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = p.h0[state + v];
        if constexpr (AGGREGATE) {
            if (w == 0 && ch.live)
#pragma unroll
                for (int v = 0; v < V; ++v) p.ws[stored + v] = h[v];
        }
    }
    __shared__ float joined[NW == 1 ? 1 : 2][NW][GV + V][NW == 1 ? 1 : 64];
    int buffer = 0;
    if constexpr (NW > 1 && !AGGREGATE) {
        if (plan.chunks > 1) {
            const float* const wa = p.ws + stored;
            if (span == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = wa[v];
            } else {
                foldBefore<NW, V, GV>(wa, wa + plane, p.C, span, w, lane, joined[0], h);
                buffer = 1;
            }
        }
    }
    T rawG[L][GV], rawX[L][V];
    auto load = [&](int i) {
        loadChannels<T, GV, L>(gp, p.gs[1], i, n, inside, p.reverse, rawG);
        loadChannels<T, V, L>(xp, p.xs[1], i, n, inside, p.reverse, rawX);
    };
    load(begin + w * L);
    // d_last may be d_h0, and wave 0 stores it when it has passed the last tile's barrier: by then every wave's h0 has to be here.  ldsBarrier does not wait for it, so
    // it is waited for in front of the first one.  (Without a tile there is no barrier, and what wave 0 stores is h0 itself.)
    if constexpr (NW > 1 && !AGGREGATE) {
#pragma unroll
        for (int v = 0; v < V; ++v) asm volatile("" : "+v"(h[v]));
    }
    for (int tile = begin; tile < end; tile += NW * L) {
        const int i0 = tile + w * L;
        float a[L][GV], u[L][V], a2[GV], u2[V];
#pragma unroll
        for (int v = 0; v < V; ++v) u2[v] = 0.f;
#pragma unroll
        for (int v = 0; v < GV; ++v) a2[v] = 1.f;
        withGates<T, GV, L>(p, rawG, i0, inside, [&](int k, int v, float gate, float factor) {
            a[k][v] = gate;
            a2[v] *= gate;
#pragma unroll
            for (int c = SHARED ? 0 : v; c < (SHARED ? V : v + 1); ++c) {
                u[k][c] = factor * toFloat(rawX[k][c]);
                u2[c] = fmaf(gate, u2[c], u[k][c]);
            }
        });
        if (tile + NW * L < end) load(i0 + NW * L);  // (on its way while this tile is joined and stored)
        float pre[V];
#pragma unroll
        for (int v = 0; v < V; ++v) pre[v] = h[v];
        if constexpr (NW > 1) {
#pragma unroll
            for (int v = 0; v < GV; ++v) joined[buffer][w][v][lane] = a2[v];
#pragma unroll
            for (int v = 0; v < V; ++v) joined[buffer][w][GV + v][lane] = u2[v];
            ldsBarrier();  // (one barrier a tile: the two buffers take turns, and a wave can only be one tile ahead)
#pragma unroll 2
            for (int j = 0; j < NW; ++j) {
                float aj[GV];
#pragma unroll
                for (int v = 0; v < GV; ++v) {
                    aj[v] = joined[buffer][j][v][lane];
                    if (AGGREGATE) A[v] *= aj[v];
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (j == w) pre[v] = h[v];
                    h[v] = fmaf(aj[SHARED ? 0 : v], h[v], joined[buffer][j][GV + v][lane]);
                }
            }
            buffer ^= 1;
        }
        if constexpr (!AGGREGATE) {
            const bool whole = i0 + L <= inside;
            const long long next = p.reverse ? -p.os[1] : p.os[1];
            T* const at = op && whole ? op + positionOf(i0, n, p.reverse) * p.os[1] : op;
#pragma unroll
            for (int k = 0; k < L; ++k) {
                T o[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    pre[v] = fmaf(a[k][SHARED ? 0 : v], pre[v], u[k][v]);
                    o[v] = fromFloat<T>(whole || i0 + k < n ? pre[v] : 0.f);
                }
                if (!op || !ch.live) continue;
                if (whole) storeWide<T, V>(at + k * next, o);
                else if (i0 + k < end) storeWide<T, V>(op + positionOf(i0 + k, n, p.reverse) * p.os[1], o);
            }
            if constexpr (NW == 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = pre[v];
            }
        }
    }
    if (w != 0 || !ch.live) return;
    if constexpr (AGGREGATE) {
        float* const wa = p.ws + stored + (long long)span * p.C;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (span > 0) wa[v] = A[SHARED ? 0 : v];
            wa[plane + v] = h[v];
        }
    } else if (p.last && span == plan.chunks - 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.last[state + v] = h[v];
    }
}

// Backward, scratch memory: for each span A, U (span 0 from h0) and D; then for each tile what its span's first steps up to it make of the state that enters the
// span, h -> A h + U (a call of one span: A is not there, U the state itself); then the parts of gate sums.
struct BackwardScratch {
    float *spans, *heads, *partial;
    long long plane, headPlane;
};
__host__ __device__ inline BackwardScratch backwardScratch(const ScanParams& p, const ScanPlan& plan) {
    BackwardScratch r;
    const int tilesOfSpan = plan.chunkSteps / plan.tile;
    r.plane = plan.chunks > 1 ? p.B * plan.chunks * (long long)p.C : 0;
    r.headPlane = tilesOfSpan > 1 ? p.B * plan.chunks * tilesOfSpan * (long long)p.C : 0;
    r.spans = p.ws;
    r.heads = p.ws + 3 * r.plane;
    r.partial = r.heads + (plan.chunks > 1 ? 2 : 1) * r.headPlane;
    return r;
}
inline size_t backwardFloats(const ScanParams& p, const ScanPlan& plan) {
    ScanParams q = p;
    q.ws = nullptr;
    const size_t partial = plan.parts > 1 ? size_t(p.B) * p.T * p.Cg * plan.parts : 0;
    const BackwardScratch s = backwardScratch(q, plan);
    return size_t(3 * s.plane + (plan.chunks > 1 ? 2 : 1) * s.headPlane) + partial;
}

// Backward, first launch of a call that is cut into spans.  8 x 4096 x 1024 f16: 46 us (207 MB, 4.5 TB/s).
template <class T, int NW, int V, bool SHARED>
__global__ __launch_bounds__(64 * NW) void scan_channels_spans_kernel(const ScanParams p, const ScanPlan plan, const int blocks) {
    constexpr int L = backwardSteps(V, sizeof(T)), GV = SHARED ? 1 : V;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long b = blockIdx.x / blocks;
    const ChannelLane ch = channelLane<V, SHARED>(p, int(blockIdx.x % blocks), lane, plan.slots, plan.parts);
    const int n = lengthOf(p, b), span = blockIdx.y;
    const int begin = span * plan.chunkSteps, end = min(n, begin + plan.chunkSteps), tilesOfSpan = plan.chunkSteps / plan.tile;
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + ch.g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + ch.c * p.xs[2];
    const T* const dp = p.dout ? static_cast<const T*>(p.dout) + b * p.ds[0] + ch.c * p.ds[2] : nullptr;
    const BackwardScratch ws = backwardScratch(p, plan);
    float* const heads = ws.heads + ((b * plan.chunks + span) * tilesOfSpan) * p.C + ch.c;
    float A[GV], U[V], D[V];
#pragma unroll
    for (int v = 0; v < GV; ++v) A[v] = 1.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        U[v] = span == 0 && p.h0 ? p.h0[b * p.C + ch.c + v] : 0.f;
        D[v] = 0.f;
    }
    __shared__ float joined[2][NW][GV + 2 * V][64];
    int buffer = 0;
    T rawG[L][GV], rawX[L][V], rawD[L][V];
    auto load = [&](int i) {
        loadChannels<T, GV, L>(gp, p.gs[1], i, n, end, p.reverse, rawG);
        loadChannels<T, V, L>(xp, p.xs[1], i, n, end, p.reverse, rawX);
        if (dp) loadChannels<T, V, L>(dp, p.ds[1], i, n, end, p.reverse, rawD);
    };
    load(begin + w * L);
    for (int tile = begin, j = 0; tile < end; tile += NW * L, ++j) {
        if (tilesOfSpan > 1 && w == 0 && ch.live) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                heads[(long long)j * p.C + v] = span == 0 ? 0.f : A[SHARED ? 0 : v];
                heads[ws.headPlane + (long long)j * p.C + v] = U[v];
            }
        }
        const int i0 = tile + w * L;
        float a2[GV], u2[V], d2[V];
#pragma unroll
        for (int v = 0; v < V; ++v) u2[v] = d2[v] = 0.f;
#pragma unroll
        for (int v = 0; v < GV; ++v) a2[v] = 1.f;
        withGates<T, GV, L>(p, rawG, i0, end, [&](int k, int v, float gate, float factor) {
            a2[v] *= gate;
#pragma unroll
            for (int c = SHARED ? 0 : v; c < (SHARED ? V : v + 1); ++c) {
                u2[c] = fmaf(gate, u2[c], factor * toFloat(rawX[k][c]));
                if (dp) d2[c] = fmaf(a2[v], toFloat(rawD[k][c]), d2[c]);
            }
        });
        if (tile + NW * L < end) load(i0 + NW * L);
#pragma unroll
        for (int v = 0; v < GV; ++v) joined[buffer][w][v][lane] = a2[v];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            joined[buffer][w][GV + v][lane] = u2[v];
            joined[buffer][w][GV + V + v][lane] = d2[v];
        }
        ldsBarrier();
#pragma unroll 2
        for (int s = 0; s < NW; ++s) {
            float as[GV];
#pragma unroll
            for (int v = 0; v < GV; ++v) as[v] = joined[buffer][s][v][lane];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                U[v] = fmaf(as[SHARED ? 0 : v], U[v], joined[buffer][s][GV + v][lane]);
                D[v] = fmaf(A[SHARED ? 0 : v], joined[buffer][s][GV + V + v][lane], D[v]);
            }
#pragma unroll
            for (int v = 0; v < GV; ++v) A[v] *= as[v];
        }
        buffer ^= 1;
    }
    if (w != 0 || !ch.live) return;
    const long long at = (b * plan.chunks + span) * p.C + ch.c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        ws.spans[at + v] = A[SHARED ? 0 : v];
        ws.spans[ws.plane + at + v] = U[v];
        ws.spans[2 * ws.plane + at + v] = D[v];
    }
}

// Backward: the states of a tile again on the way in, gradients on the way out.  A call of one span walks all tiles forwards first and keeps the state at the head of
// each.  8 x 4096 x 1024 f16 behind its spans 77 us (349 MB, 4.5 TB/s), 64 x 512 x 4096 bf16 in one launch 341 - 353 us (1.88 GB with what is read twice, 5.4 TB/s).
template <class T, int NW, int V, bool SHARED>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW, 4) void scan_channels_backward_kernel(const ScanParams p, const ScanPlan plan, const int blocks, const long long units) {
    constexpr int L = backwardSteps(V, sizeof(T)), GV = SHARED ? 1 : V;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (known to be the same for a wave: its addresses are scalars)
    const int w = NW == 1 ? 0 : wave;
    const long long unit = NW == 1 ? blockIdx.x * 4LL + wave : blockIdx.x;
    if (unit >= units) return;
    const long long b = unit / blocks;
    const ChannelLane ch = channelLane<V, SHARED>(p, int(unit % blocks), lane, plan.slots, plan.parts);
    const int n = lengthOf(p, b), span = gridDim.y - 1 - blockIdx.y;
    const int begin = span * plan.chunkSteps, end = min(p.T, begin + plan.chunkSteps), inside = min(n, end);
    const int tiles = (end - begin + plan.tile - 1) / plan.tile, tilesOfSpan = plan.chunkSteps / plan.tile;
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + ch.g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + ch.c * p.xs[2];
    const T* const dp = p.dout ? static_cast<const T*>(p.dout) + b * p.ds[0] + ch.c * p.ds[2] : nullptr;
    T* const dgp = p.dgate ? static_cast<T*>(p.dgate) + b * p.dgs[0] + ch.g * p.dgs[2] : nullptr;
    T* const dxp = p.dx ? static_cast<T*>(p.dx) + b * p.dxs[0] + ch.c * p.dxs[2] : nullptr;
    const BackwardScratch ws = backwardScratch(p, plan);
    const long long state = b * p.C + ch.c;
    const bool kept = tilesOfSpan > 1;
    float* const heads = ws.heads + ((b * plan.chunks + span) * tilesOfSpan) * p.C + ch.c;
    float* const partial = ws.partial + (b * p.T * (long long)p.Cg + ch.g) * plan.parts + ch.part;
    float h[V], k[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        h[v] = p.h0 ? p.h0[state + v] : 0.f;
        k[v] = p.dlast ? p.dlast[state + v] : 0.f;
    }
    __shared__ float joined[NW == 1 ? 1 : 2][NW][GV + 3 * V][NW == 1 ? 1 : 64];
    int buffer = 0;
    if constexpr (NW > 1) {
        if (plan.chunks > 1) {
            typedef float Fold[NW][GV + V][64];
            static_assert(sizeof(Fold) <= sizeof(joined[0]), "a fold borrows a buffer");
            const float* const wa = ws.spans + (b * plan.chunks) * p.C + ch.c;
            if (span > 0) foldBefore<NW, V, GV>(wa, wa + ws.plane, p.C, span, w, lane, reinterpret_cast<Fold&>(joined[0]), h);
            foldBehind<NW, V, GV>(wa, wa + 2 * ws.plane, p.C, span + 1, plan.chunks, w, lane, reinterpret_cast<Fold&>(joined[1]), k);
            ldsBarrier();  // (the walk below begins with the first buffer, and a wave may still be reading the second one)
        }
    }
    if (kept && plan.chunks == 1) {
        // one span: the states at the head of every tile, for the walk back
        float at[V];
#pragma unroll
        for (int v = 0; v < V; ++v) at[v] = h[v];
        for (int j = 0; j < tiles; ++j) {
            if (w == 0)  // (written and read again by this lane; a dead one's channel is a live one's, and so is its value)
#pragma unroll
                for (int v = 0; v < V; ++v) heads[(long long)j * p.C + v] = at[v];
            const int i0 = begin + j * plan.tile + w * L;
            T rawG[L][GV], rawX[L][V];
            loadChannels<T, GV, L>(gp, p.gs[1], i0, n, inside, p.reverse, rawG);
            loadChannels<T, V, L>(xp, p.xs[1], i0, n, inside, p.reverse, rawX);
            float a2[GV], u2[V];
#pragma unroll
            for (int v = 0; v < V; ++v) u2[v] = NW == 1 ? at[v] : 0.f;
#pragma unroll
            for (int v = 0; v < GV; ++v) a2[v] = 1.f;
            withGates<T, GV, L>(p, rawG, i0, inside, [&](int k, int v, float gate, float factor) {
                a2[v] *= gate;
#pragma unroll
                for (int c = SHARED ? 0 : v; c < (SHARED ? V : v + 1); ++c) u2[c] = fmaf(gate, u2[c], factor * toFloat(rawX[k][c]));
            });
            if constexpr (NW > 1) {
#pragma unroll
                for (int v = 0; v < GV; ++v) joined[buffer][w][v][lane] = a2[v];
#pragma unroll
                for (int v = 0; v < V; ++v) joined[buffer][w][GV + v][lane] = u2[v];
                ldsBarrier();
#pragma unroll 2
                for (int s = 0; s < NW; ++s)
#pragma unroll
                    for (int v = 0; v < V; ++v) at[v] = fmaf(joined[buffer][s][SHARED ? 0 : v][lane], at[v], joined[buffer][s][GV + v][lane]);
                buffer ^= 1;
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) at[v] = u2[v];
            }
        }
    }
    T rawG[L][GV], rawX[L][V], rawD[L][V];
    auto load = [&](int i) {
        loadChannels<T, GV, L>(gp, p.gs[1], i, n, inside, p.reverse, rawG);
        loadChannels<T, V, L>(xp, p.xs[1], i, n, inside, p.reverse, rawX);
        if (dp) loadChannels<T, V, L>(dp, p.ds[1], i, n, inside, p.reverse, rawD);
    };
    for (int j = tiles - 1; j >= 0; --j) {
        const int i0 = begin + j * plan.tile + w * L;
        load(i0);
        // the state at the head of the tile: of a wave on its own its own, of waves that share one what wave 0 says below
        float head[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            head[v] = h[v];
            if (kept && w == 0 && begin + j * plan.tile < n)
                head[v] = plan.chunks == 1 ? heads[(long long)j * p.C + v] : span == 0 ? heads[ws.headPlane + (long long)j * p.C + v]
                                                                                     : fmaf(heads[(long long)j * p.C + v], h[v], heads[ws.headPlane + (long long)j * p.C + v]);
        }
        float a[L][GV], rest[L][GV], x[L][V], d[L][V], a2[GV], u2[V], d2[V];
        withGates<T, GV, L>(p, rawG, i0, inside, [&](int k, int v, float gate, float factor) {
            a[k][v] = gate;
            rest[k][v] = factor;
        });
#pragma unroll
        for (int v = 0; v < V; ++v) u2[v] = d2[v] = 0.f;
#pragma unroll
        for (int v = 0; v < GV; ++v) a2[v] = 1.f;
#pragma unroll
        for (int q = 0; q < L; ++q) {
#pragma unroll
            for (int v = 0; v < GV; ++v) a2[v] *= a[q][v];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                x[q][v] = toFloat(rawX[q][v]);
                d[q][v] = dp ? toFloat(rawD[q][v]) : 0.f;
                if (NW > 1) {
                    u2[v] = fmaf(a[q][SHARED ? 0 : v], u2[v], rest[q][SHARED ? 0 : v] * x[q][v]);
                    d2[v] = fmaf(a2[SHARED ? 0 : v], d[q][v], d2[v]);
                }
            }
        }
        float hw[V], kw[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            hw[v] = head[v];
            kw[v] = k[v];
        }
        if constexpr (NW > 1) {
#pragma unroll
            for (int v = 0; v < GV; ++v) joined[buffer][w][v][lane] = a2[v];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                joined[buffer][w][GV + v][lane] = u2[v];
                joined[buffer][w][GV + V + v][lane] = d2[v];
                if (w == 0) joined[buffer][0][GV + 2 * V + v][lane] = head[v];
            }
            ldsBarrier();
#pragma unroll
            for (int v = 0; v < V; ++v) hw[v] = joined[buffer][0][GV + 2 * V + v][lane];
#pragma unroll 2
            for (int s = 0; s < w; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) hw[v] = fmaf(joined[buffer][s][SHARED ? 0 : v][lane], hw[v], joined[buffer][s][GV + v][lane]);
#pragma unroll 2
            for (int s = NW - 1; s >= 0; --s)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (s == w) kw[v] = k[v];
                    k[v] = fmaf(joined[buffer][s][SHARED ? 0 : v][lane], k[v], joined[buffer][s][GV + V + v][lane]);
                }
            buffer ^= 1;
        }
        float entry[L][V];
#pragma unroll
        for (int q = 0; q < L; ++q)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                entry[q][v] = hw[v];
                hw[v] = fmaf(a[q][SHARED ? 0 : v], hw[v], rest[q][SHARED ? 0 : v] * x[q][v]);
            }
        // (what is needed of x and the states on the way in: the gate's gradient takes l times it)
#pragma unroll
        for (int q = 0; q < L; ++q)
#pragma unroll
            for (int v = 0; v < V; ++v) entry[q][v] = p.blend ? entry[q][v] - x[q][v] : entry[q][v];
        float sum[L][GV];
#pragma unroll
        for (int q = L - 1; q >= 0; --q) {
#pragma unroll
            for (int v = 0; v < GV; ++v) sum[q][v] = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int g = SHARED ? 0 : v;
                const float l = d[q][v] + kw[v];
                x[q][v] = rest[q][g] * l;  // the gradient of x
                sum[q][g] = SHARED ? fmaf(l, entry[q][v], sum[q][g]) : l * entry[q][v];
                kw[v] = a[q][g] * l;
            }
#pragma unroll
            for (int v = 0; v < GV; ++v) sum[q][v] = p.exp ? sum[q][v] * (p.scale * a[q][v]) : sum[q][v];
        }
        const bool first = V > 1 || plan.slots == 1 || (lane & (plan.slots - 1)) == 0;
        if (V == 1 && plan.slots > 1) {
#pragma unroll
            for (int q = 0; q < L; ++q) sum[q][0] = ch.live ? sum[q][0] : 0.f;
            for (int o = 1; o < plan.slots; o <<= 1)
#pragma unroll
                for (int q = 0; q < L; ++q) sum[q][0] += __shfl_xor(sum[q][0], o, 64);
        }
        if (ch.live) {
#pragma unroll
            for (int q = 0; q < L; ++q) {
                const int i = i0 + q;
                if (i >= end) break;
                const bool in = i < inside;
                const long long t = positionOf(i, n, p.reverse);
                T dx[V], dg[GV];
#pragma unroll
                for (int v = 0; v < V; ++v) dx[v] = fromFloat<T>(in ? x[q][v] : 0.f);
#pragma unroll
                for (int v = 0; v < GV; ++v) dg[v] = fromFloat<T>(in ? sum[q][v] : 0.f);
                if (dxp) storeWide<T, V>(dxp + t * p.dxs[1], dx);
                if (dgp && first) {
                    if (V == 1 && plan.parts > 1) partial[t * (long long)p.Cg * plan.parts] = in ? sum[q][0] : 0.f;
                    else storeWide<T, GV>(dgp + t * p.dgs[1], dg);
                }
            }
        }
        if constexpr (NW == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) k[v] = kw[v];
        }
    }
    if (p.dh0 && span == 0 && w == 0 && ch.live)
#pragma unroll
        for (int v = 0; v < V; ++v) p.dh0[state + v] = k[v];
}

// Sums of the parts of gates with more than 64 channels, in their order (16 x 1000 steps of three parts: 4 us).
template <class T>
__global__ __launch_bounds__(256) void scan_gate_sum_kernel(const ScanParams p, const float* partial, const int parts) {
    const long long count = p.B * p.T * (long long)p.Cg;
    for (long long e = blockIdx.x * 256LL + threadIdx.x; e < count; e += gridDim.x * 256LL) {
        float s = 0.f;
        for (int q = 0; q < parts; ++q) s += partial[e * parts + q];
        const long long g = e % p.Cg, t = (e / p.Cg) % p.T, b = e / p.Cg / p.T;
        static_cast<T*>(p.dgate)[b * p.dgs[0] + t * p.dgs[1] + g * p.dgs[2]] = fromFloat<T>(s);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// lanes are steps
// ---------------------------------------------------------------------------------------------------------------------

// Steps of a lane: 8, and backward 4 for rows of up to 256 steps, which are one tile either way (65536 rays x 256 with gradients: 102 us with 4 steps, whose
// registers leave room for more waves, against 130 with 8; 262144 x 512, two tiles against one: 1018 against 899).
constexpr int kRowSteps = 8, kRowStepsShort = 4;
constexpr int rowSteps(int T, bool backward) { return backward && T <= 64 * kRowStepsShort ? kRowStepsShort : kRowSteps; }

// (A, U) of this lane's span joined with its row's lanes before it (FORWARD) or behind it, over the `width` lanes of a row: an inclusive scan.
template <int G, bool FORWARD>
__device__ __forceinline__ void joinLanes(float& A, float (&U)[G], int width, int lane) {
    const int at = lane & (width - 1);
    for (int o = 1; o < width; o <<= 1) {
        const float a = FORWARD ? __shfl_up(A, o, width) : __shfl_down(A, o, width);
        float u[G];
#pragma unroll
        for (int c = 0; c < G; ++c) u[c] = FORWARD ? __shfl_up(U[c], o, width) : __shfl_down(U[c], o, width);
        if (FORWARD ? at >= o : at + o < width) {
#pragma unroll
            for (int c = 0; c < G; ++c) U[c] = fmaf(A, u[c], U[c]);
            A *= a;
        }
    }
}

// K steps of G channels of one lane, steps i .. i + K - 1 of a sequence of n, with as wide accesses as the strides allow: all of it in one piece, a step in one
// piece, or element by element.  A lane's steps are 128 bytes of colours with absorption apart from the next lane's: reading them element by element
// would touch 64 lines with each instruction.
template <class T, int G, int K>
struct StepBlock {
    T v[K * G];  // in the order of memory
    __device__ __forceinline__ void load(const T* base, long long step, long long channel) {
        if (channel == 1 && step == G) {
            loadWide<T, K * G>(v, base);
        } else if (channel == 1) {
#pragma unroll
            for (int q = 0; q < K; ++q) loadWide<T, G>(v + q * G, base + q * step);
        } else {
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) v[q * G + c] = base[q * step + c * channel];
        }
    }
    __device__ __forceinline__ void store(T* base, long long step, long long channel) const {
        if (channel == 1 && step == G) {
            storeWide<T, K * G>(base, v);
        } else if (channel == 1) {
#pragma unroll
            for (int q = 0; q < K; ++q) storeWide<T, G>(base + q * step, v + q * G);
        } else {
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) base[q * step + c * channel] = v[q * G + c];
        }
    }
};

// to[q][c] = channel c of step i + q, 0 behind the sequence
template <class T, int G, int K>
__device__ __forceinline__ void loadSteps(const T* p, long long step, long long channel, int i, int n, int reverse, float (&to)[K][G]) {
    if (i + K <= n) {
        StepBlock<T, G, K> block;
        if (reverse) {
            block.load(p + (long long)(n - K - i) * step, step, channel);
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) to[q][c] = toFloat(block.v[(K - 1 - q) * G + c]);
        } else {
            block.load(p + (long long)i * step, step, channel);
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) to[q][c] = toFloat(block.v[q * G + c]);
        }
    } else {
#pragma unroll
        for (int q = 0; q < K; ++q)
#pragma unroll
            for (int c = 0; c < G; ++c) to[q][c] = i + q < n ? toFloat(p[positionOf(i + q, n, reverse) * step + c * channel]) : 0.f;
    }
}

// zeros behind the sequence, nothing behind T
template <class T, int G, int K>
__device__ __forceinline__ void storeSteps(T* p, long long step, long long channel, int i, int n, int T_, int reverse, const float (&from)[K][G]) {
    if (i + K <= n) {
        StepBlock<T, G, K> block;
        if (reverse) {
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) block.v[(K - 1 - q) * G + c] = fromFloat<T>(from[q][c]);
            block.store(p + (long long)(n - K - i) * step, step, channel);
        } else {
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) block.v[q * G + c] = fromFloat<T>(from[q][c]);
            block.store(p + (long long)i * step, step, channel);
        }
    } else {
#pragma unroll
        for (int q = 0; q < K; ++q)
#pragma unroll
            for (int c = 0; c < G; ++c)
                if (i + q < T_) p[positionOf(i + q, n, reverse) * step + c * channel] = fromFloat<T>(i + q < n ? from[q][c] : 0.f);
    }
}

// A gate's row with its G channels; `beside`: the gate is the element behind its channels (the colours and absorptions of a transfer function), read with them
template <class T, int G, int K>
__device__ __forceinline__ void loadRow(const ScanParams& p, const T* gp, const T* xp, bool beside, int i, int n, float (&g)[K], float (&x)[K][G]) {
    if (beside) {
        float both[K][G + 1];
        loadSteps<T, G + 1, K>(xp, p.xs[1], 1, i, n, p.reverse, both);
#pragma unroll
        for (int q = 0; q < K; ++q) {
            g[q] = both[q][G];
#pragma unroll
            for (int c = 0; c < G; ++c) x[q][c] = both[q][c];
        }
    } else {
        float one[K][1];
        loadSteps<T, 1, K>(gp, p.gs[1], 1, i, n, p.reverse, one);
#pragma unroll
        for (int q = 0; q < K; ++q) g[q] = one[q][0];
        loadSteps<T, G, K>(xp, p.xs[1], G == 1 ? 1 : p.xs[2], i, n, p.reverse, x);
    }
}

// a and the factor of x (1 - a of BLEND, 1 of ADD) of a lane's steps; behind the sequence x was read as 0, and the gate is 1
template <int K>
__device__ __forceinline__ void rowGates(const ScanParams& p, int i, int n, float (&m)[K], float (&rest)[K]) {
    if (p.exp) {
#pragma unroll
        for (int q = 0; q < K; ++q) gateOf<true>(m[q], p.scale, m[q], rest[q]);
    } else {
#pragma unroll
        for (int q = 0; q < K; ++q) {
            gateOf<false>(m[q], p.scale, m[q], rest[q]);
            m[q] = i + q < n ? m[q] : 1.f;
        }
    }
    if (!p.blend)
#pragma unroll
        for (int q = 0; q < K; ++q) rest[q] = 1.f;
}

// Scratch memory of rows that are cut into spans: for each span A (0 for span 0, whose U starts from h0), U and, backward, D of the G channels; each row's h0;
// backward, the state at the head of each tile.
struct RowScratch {
    float *spans, *h0, *heads;
};
__host__ __device__ inline RowScratch rowScratch(const ScanParams& p, const ScanPlan& plan, bool backward) {
    RowScratch r;
    const long long rows = plan.chunks > 1 ? p.B * p.Cg : 0;
    r.spans = p.ws;
    r.h0 = r.spans + rows * plan.chunks * (1 + (backward ? 2 : 1) * p.G);
    r.heads = r.h0 + rows * p.G;
    return r;
}

// What spans from .. to - 1 of a row make of what enters them: (A, U) in all lanes, U from h before them, or (A, D), D from k behind them.  64 lanes take a part each.
template <int G, bool FORWARD>
__device__ __forceinline__ void foldSpans(const float* spans, int entry, int from, int to, int lane, float& A, float (&U)[G]) {
    const int each = (to - from + 63) / 64;
    const int first = min(to, from + lane * each), last = min(to, first + each);
    A = 1.f;
#pragma unroll
    for (int c = 0; c < G; ++c) U[c] = 0.f;
    for (int s = first; s < last; ++s) {
        const float* const e = spans + (long long)s * entry;
        const float a = e[0];
#pragma unroll
        for (int c = 0; c < G; ++c) U[c] = FORWARD ? fmaf(a, U[c], e[1 + c]) : fmaf(A, e[1 + G + c], U[c]);
        A *= a;
    }
    joinLanes<G, FORWARD>(A, U, 64, lane);
    A = __shfl(A, FORWARD ? 63 : 0, 64);
#pragma unroll
    for (int c = 0; c < G; ++c) U[c] = __shfl(U[c], FORWARD ? 63 : 0, 64);
}

// First launch of a call whose rows are cut into spans (few rows with many steps): a wave per row and span.  Both launches of 100 x 20000 x 4 fp32: 30 us, where a wave
// that walks its row alone takes 131, and 49 against 402 backward.
template <class T, int G, bool BACKWARD>
__global__ __launch_bounds__(256) void scan_rows_spans_kernel(const ScanParams p, const ScanPlan plan, const bool beside) {
    constexpr int K = kRowSteps, ENTRY = 1 + (BACKWARD ? 2 : 1) * G;
    const int lane = threadIdx.x & 63, span = blockIdx.y;
    const long long rows = p.B * p.Cg, row = blockIdx.x * 4LL + (threadIdx.x >> 6);
    if (row >= rows) return;
    const long long b = row / p.Cg, g = row % p.Cg;
    const int n = lengthOf(p, b), begin = span * plan.chunkSteps, end = min(n, begin + plan.chunkSteps);
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + g * G * p.xs[2];
    const T* const dp = BACKWARD && p.dout ? static_cast<const T*>(p.dout) + b * p.ds[0] + g * G * p.ds[2] : nullptr;
    const RowScratch ws = rowScratch(p, plan, BACKWARD);
    float At = 1.f, Ut[G], Dt[G];
#pragma unroll
    for (int c = 0; c < G; ++c) {
        Ut[c] = span == 0 && p.h0 ? p.h0[b * p.C + g * G + c] : 0.f;
        Dt[c] = 0.f;
        if (span == 0 && lane == 0) ws.h0[row * G + c] = Ut[c];
    }
    for (int tile = begin; tile < end; tile += 64 * K) {
        const int i0 = tile + lane * K;
        float m[K], rest[K], x[K][G], d[K][G];
        loadRow<T, G, K>(p, gp, xp, beside, i0, n, m, x);
        if (dp) loadSteps<T, G, K>(dp, p.ds[1], G == 1 ? 1 : p.ds[2], i0, n, p.reverse, d);
        rowGates<K>(p, i0, n, m, rest);
        float A = 1.f, U[G], D[G];
#pragma unroll
        for (int c = 0; c < G; ++c) U[c] = D[c] = 0.f;
#pragma unroll
        for (int q = 0; q < K; ++q) {
            A *= m[q];
#pragma unroll
            for (int c = 0; c < G; ++c) {
                U[c] = fmaf(m[q], U[c], rest[q] * x[q][c]);
                if (dp) D[c] = fmaf(A, d[q][c], D[c]);
            }
        }
        float A2 = A;
        joinLanes<G, true>(A, U, 64, lane);
        A = __shfl(A, 63, 64);
        if (dp) joinLanes<G, false>(A2, D, 64, lane);
#pragma unroll
        for (int c = 0; c < G; ++c) {
            Ut[c] = fmaf(A, Ut[c], __shfl(U[c], 63, 64));
            if (dp) Dt[c] = fmaf(At, __shfl(D[c], 0, 64), Dt[c]);
        }
        At *= A;
    }
    if (lane != 0) return;
    float* const e = ws.spans + (row * plan.chunks + span) * ENTRY;
    e[0] = span == 0 ? 0.f : At;
#pragma unroll
    for (int c = 0; c < G; ++c) {
        e[1 + c] = Ut[c];
        if (BACKWARD) e[1 + G + c] = Dt[c];
    }
}

// Forward: bound by memory where 16-byte pieces come in (262144 rays x 512 with three channels fp32: 435 us, 2.15 GB, 4.95 TB/s), by the work on each sample -- its gate,
// its conversions -- in 16 bits (370 - 425 us for half the bytes; lanes joined by cross-lane moves take 2 % off).
template <class T, int G>
__global__ __launch_bounds__(256) void scan_rows_kernel(const ScanParams p, const ScanPlan plan, const bool beside) {
    constexpr int K = kRowSteps;
    const int width = plan.width, lane = threadIdx.x & 63, at = lane & (width - 1), span = blockIdx.y;
    const long long rows = p.B * p.Cg, own = (blockIdx.x * 4LL + (threadIdx.x >> 6)) * (64 / width) + lane / width;
    const bool live = own < rows;
    const long long row = live ? own : rows - 1, b = row / p.Cg, g = row % p.Cg;
    // (a row with more than one tile has a wave for itself: only then the loop below ends at its own length)
    const int n = lengthOf(p, b), begin = span * plan.chunkSteps, end = min(p.out || width < 64 ? p.T : n, begin + plan.chunkSteps);
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + g * G * p.xs[2];
    T* const op = p.out ? static_cast<T*>(p.out) + b * p.os[0] + g * G * p.os[2] : nullptr;
    const long long state = b * p.C + g * G;
    float h[G];
    if (plan.chunks > 1) {
        const RowScratch ws = rowScratch(p, plan, false);
        float A;
        if (span > 0) foldSpans<G, true>(ws.spans + row * plan.chunks * (1 + G), 1 + G, 0, span, lane, A, h);
        else
#pragma unroll
            for (int c = 0; c < G; ++c) h[c] = ws.h0[row * G + c];  // (a copy: d_last may be d_h0)
    } else {
#pragma unroll
        for (int c = 0; c < G; ++c) h[c] = p.h0 ? p.h0[state + c] : 0.f;
    }
    for (int tile = begin; tile < end; tile += width * K) {
        const int i0 = tile + at * K;
        float m[K], rest[K], u[K][G];
        loadRow<T, G, K>(p, gp, xp, beside, i0, n, m, u);
        rowGates<K>(p, i0, n, m, rest);
        float A = 1.f, U[G];
#pragma unroll
        for (int c = 0; c < G; ++c) U[c] = 0.f;
#pragma unroll
        for (int q = 0; q < K; ++q) {
#pragma unroll
            for (int c = 0; c < G; ++c) {
                u[q][c] *= rest[q];
                U[c] = fmaf(m[q], U[c], u[q][c]);
            }
            A *= m[q];
        }
        joinLanes<G, true>(A, U, width, lane);
        // the state that enters this lane's span: the row's, taken through the lanes before
        const float before = __shfl_up(A, 1, width);
        float pre[G];
#pragma unroll
        for (int c = 0; c < G; ++c) {
            const float u1 = __shfl_up(U[c], 1, width);
            pre[c] = at ? fmaf(before, h[c], u1) : h[c];
            h[c] = __shfl(fmaf(A, h[c], U[c]), width - 1, width);
        }
        if (op) {
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) u[q][c] = pre[c] = fmaf(m[q], pre[c], u[q][c]);
            if (live) storeSteps<T, G, K>(op, p.os[1], G == 1 ? 1 : p.os[2], i0, n, p.T, p.reverse, u);
        }
    }
    if (p.last && live && at == 0 && span == plan.chunks - 1)
#pragma unroll
        for (int c = 0; c < G; ++c) p.last[state + c] = h[c];
}

// Backward: 16384 rays x 512 with three channels fp32 57 us (269 MB, 4.7 TB/s).
template <class T, int G, int K>
__global__ __launch_bounds__(256) void scan_rows_backward_kernel(const ScanParams p, const ScanPlan plan, const bool beside, const bool outBeside) {
    const int width = plan.width, lane = threadIdx.x & 63, at = lane & (width - 1), span = blockIdx.y;
    const long long rows = p.B * p.Cg, own = (blockIdx.x * 4LL + (threadIdx.x >> 6)) * (64 / width) + lane / width;
    const bool live = own < rows;
    const long long row = live ? own : rows - 1, b = row / p.Cg, g = row % p.Cg;
    const int n = lengthOf(p, b);
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + g * G * p.xs[2];
    const T* const dp = p.dout ? static_cast<const T*>(p.dout) + b * p.ds[0] + g * G * p.ds[2] : nullptr;
    T* const dgp = p.dgate ? static_cast<T*>(p.dgate) + b * p.dgs[0] + g * p.dgs[2] : nullptr;
    T* const dxp = p.dx ? static_cast<T*>(p.dx) + b * p.dxs[0] + g * G * p.dxs[2] : nullptr;
    const long long state = b * p.C + g * G;
    const int tile = width * K, tilesOfSpan = (plan.chunkSteps + tile - 1) / tile;
    const int firstTile = span * tilesOfSpan, tiles = min(tilesOfSpan, (p.T + tile - 1) / tile - firstTile);
    const RowScratch ws = rowScratch(p, plan, true);
    float* const heads = ws.heads + (row * plan.chunks + span) * tilesOfSpan * G;  // the row's state at the head of each tile of the span, if there is more than one
    float h[G], k[G];
#pragma unroll
    for (int c = 0; c < G; ++c) {
        h[c] = p.h0 ? p.h0[state + c] : 0.f;
        k[c] = p.dlast ? p.dlast[state + c] : 0.f;
    }
    if (plan.chunks > 1) {
        const float* const spans = ws.spans + row * plan.chunks * (1 + 2 * G);
        float A, D[G];
        if (span > 0) foldSpans<G, true>(spans, 1 + 2 * G, 0, span, lane, A, h);
        foldSpans<G, false>(spans, 1 + 2 * G, span + 1, plan.chunks, lane, A, D);
#pragma unroll
        for (int c = 0; c < G; ++c) k[c] = fmaf(A, k[c], D[c]);
    }
    for (int pass = tiles > 1 ? 0 : 1; pass < 2; ++pass) {
        for (int step = 0; step < tiles; ++step) {
            const int j = pass ? tiles - 1 - step : step;
            const int i0 = (firstTile + j) * tile + at * K;
            if (tiles > 1) {
                if (pass == 0) {
                    if (at == 0 && live)
#pragma unroll
                        for (int c = 0; c < G; ++c) heads[(long long)j * G + c] = h[c];
                } else {
#pragma unroll
                    for (int c = 0; c < G; ++c) {
                        float v = 0.f;
                        if (at == 0 && live) v = heads[(long long)j * G + c];  // (its own store of the first pass)
                        h[c] = __shfl(v, 0, width);
                    }
                }
            }
            float m[K], rest[K], x[K][G], d[K][G];
            loadRow<T, G, K>(p, gp, xp, beside, i0, n, m, x);
            if (dp && pass) {
                loadSteps<T, G, K>(dp, p.ds[1], G == 1 ? 1 : p.ds[2], i0, n, p.reverse, d);
            } else {
#pragma unroll
                for (int q = 0; q < K; ++q)
#pragma unroll
                    for (int c = 0; c < G; ++c) d[q][c] = 0.f;
            }
            float A = 1.f, U[G], D[G];
#pragma unroll
            for (int c = 0; c < G; ++c) U[c] = D[c] = 0.f;
            rowGates<K>(p, i0, n, m, rest);
#pragma unroll
            for (int q = 0; q < K; ++q) {
                A *= m[q];
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    U[c] = fmaf(m[q], U[c], rest[q] * x[q][c]);
                    D[c] = fmaf(A, d[q][c], D[c]);
                }
            }
            float A2 = A;
            joinLanes<G, true>(A, U, width, lane);
            const float before = __shfl_up(A, 1, width);
            float pre[G];
#pragma unroll
            for (int c = 0; c < G; ++c) {
                const float u1 = __shfl_up(U[c], 1, width);
                pre[c] = at ? fmaf(before, h[c], u1) : h[c];
            }
            if (pass == 0) {
#pragma unroll
                for (int c = 0; c < G; ++c) h[c] = __shfl(fmaf(A, h[c], U[c]), width - 1, width);
                continue;
            }
            float kw[G], dg[K][1], entry[K][G];
            if (dp) {
                joinLanes<G, false>(A2, D, width, lane);
                const float behind = __shfl_down(A2, 1, width);
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    const float d1 = __shfl_down(D[c], 1, width);
                    kw[c] = at + 1 < width ? fmaf(behind, k[c], d1) : k[c];
                    k[c] = __shfl(fmaf(A2, k[c], D[c]), 0, width);
                }
            } else {  // only the last state's gradient comes in: one product of gates for all channels
                float none[1] = {0.f};
                joinLanes<1, false>(A2, none, width, lane);
                const float behind = __shfl_down(A2, 1, width), all = __shfl(A2, 0, width);
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    kw[c] = at + 1 < width ? behind * k[c] : k[c];
                    k[c] *= all;
                }
            }
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    entry[q][c] = pre[c];
                    pre[c] = fmaf(m[q], pre[c], rest[q] * x[q][c]);
                }
#pragma unroll
            for (int q = K - 1; q >= 0; --q) {
                float s = 0.f;
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    const float l = d[q][c] + kw[c];
                    s = fmaf(l, p.blend ? entry[q][c] - x[q][c] : entry[q][c], s);
                    x[q][c] = rest[q] * l;
                    kw[c] = m[q] * l;
                }
                dg[q][0] = p.exp ? s * (p.scale * m[q]) : s;
            }
            if (!live) continue;
            if (outBeside) {
                float both[K][G + 1];
#pragma unroll
                for (int q = 0; q < K; ++q) {
                    both[q][G] = dg[q][0];
#pragma unroll
                    for (int c = 0; c < G; ++c) both[q][c] = x[q][c];
                }
                storeSteps<T, G + 1, K>(dxp, p.dxs[1], 1, i0, n, p.T, p.reverse, both);
            } else {
                if (dgp) storeSteps<T, 1, K>(dgp, p.dgs[1], 1, i0, n, p.T, p.reverse, dg);
                if (dxp) storeSteps<T, G, K>(dxp, p.dxs[1], G == 1 ? 1 : p.dxs[2], i0, n, p.T, p.reverse, x);
            }
        }
    }
    if (p.dh0 && live && at == 0 && span == 0)
#pragma unroll
        for (int c = 0; c < G; ++c) p.dh0[state + c] = k[c];
}

// The gate is the element behind its row's channels: one tensor of colours and absorptions, or its gradient
bool gateBeside(const void* x, const long long* xs, const void* gate, const long long* gs, const ScanParams& p, size_t e) {
    return p.Cg == 1 && (p.G == 1 || xs[2] == 1) && xs[1] == gs[1] && (xs[0] == gs[0] || p.B == 1) && (p.T == 1 || xs[1] > p.G) &&
           static_cast<const char*>(gate) == static_cast<const char*>(x) + p.G * e;
}

// ---------------------------------------------------------------------------------------------------------------------
// dispatch
// ---------------------------------------------------------------------------------------------------------------------

int powerOfTwoAtLeast(long long v) {
    int r = 1;
    while (r < v) r <<= 1;
    return r;
}

template <class F>
hipError_t withType(int dtype, F&& f) {
    if (dtype == FVSRN_TENSOR_F16) return f(f16_t{});
    if (dtype == FVSRN_TENSOR_BF16) return f(bf16_t{});
    return f(float{});
}

template <class F>
hipError_t withGroup(int G, F&& f) {
    switch (G) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        default: return f(std::integral_constant<int, 4>{});
    }
}

// channels of a lane with gates of their own: 8 bytes, and half of it backwards, where a step has twice the registers
constexpr int widestLane(int elementBytes, bool backward) { return elementBytes == 2 && !backward ? 4 : 2; }

// f(channels of a lane, whether they share a gate)
template <class T, bool BACKWARD, class F>
hipError_t withLane(const ScanPlan& plan, F&& f) {
    if (plan.shared) {
        if (plan.vec == 2) return f(std::integral_constant<int, 2>{}, std::true_type{});
        if (plan.vec == 3) return f(std::integral_constant<int, 3>{}, std::true_type{});
        return f(std::integral_constant<int, 4>{}, std::true_type{});
    }
    if constexpr (widestLane(sizeof(T), BACKWARD) == 4)
        if (plan.vec == 4) return f(std::integral_constant<int, 4>{}, std::false_type{});
    if (plan.vec == 2) return f(std::integral_constant<int, 2>{}, std::false_type{});
    return f(std::integral_constant<int, 1>{}, std::false_type{});
}

}  // namespace

ScanPlan planScan(const ScanParams& p, int dtype, bool backward) {
    ScanPlan plan{};
    plan.slots = plan.parts = plan.vec = plan.chunks = plan.waves = 1;
    // How far a step and the next gate's channels are away, of x -- or, where x stands still along the steps (broadcast), of what is written, or of the gate: an operand
    // that stands still costs nothing either way.  (8 x 4096 steps of 1024 channels fp32 with such an x: 70 us, backward 161, as the others lie, 529 and 1625 by x.)
    double step = 0, next = 0;  // (any 64-bit strides)
    const long long* const moves[3] = {p.xs, backward ? p.dxs : p.os, p.gs};
    for (int i = 0; i < 3 && step == 0; ++i) {
        step = std::fabs(double(moves[i][1]));
        next = std::fabs(double(moves[i][2])) * (i < 2 ? p.G : 1);
    }
    // Lanes along the steps where steps lie closer together than gates (colours along a ray: step 4, next ray's far away), or where there are too few
    // gates beside each other: 64 x 4096 steps of 6 channels take 31 us with lanes along the steps and 27 along the channels, backward 54 and 55; 4 channels
    // 19 and 27, 28 and 53; 12 channels 56 and 28, 115 and 58.
    plan.rows = p.G <= 4 && (p.Cg < 10 || step < next);
    if (plan.rows) {
        const int K = rowSteps(p.T, backward);
        plan.width = std::min(64, powerOfTwoAtLeast((p.T + K - 1) / K));
        plan.tile = plan.width * K;
        const int tiles = std::max(1, int((p.T + (long long)plan.tile - 1) / plan.tile));
        // Spans while there are fewer than 8 waves of rows for each CU (a row of several tiles is a wave)
        const long long rows = p.B * p.Cg, want = tiles > 1 ? (2048 + rows - 1) / rows : 1;
        const int tilesOfSpan = int((tiles + std::min(want, (long long)tiles) - 1) / std::min(want, (long long)tiles));
        plan.chunks = (tiles + tilesOfSpan - 1) / tilesOfSpan;
        plan.chunkSteps = tilesOfSpan * plan.tile;
        ScanParams q = p;
        q.ws = nullptr;
        plan.wsFloats = plan.chunks > 1 ? size_t(rowScratch(q, plan, backward).heads - q.ws) : 0;
        if (backward && tilesOfSpan > 1) plan.wsFloats += size_t(rows) * plan.chunks * tilesOfSpan * p.G;
        return plan;
    }
    // Channels of a lane.  A gate's two to four, if they are adjacent: its factor is worked out once and its gradient summed in the lane.  Otherwise
    // adjacent channels with adjacent gates, for 8 bytes a load where that leaves every lane something to do.
    // (The strides of operands that are not there count too: the scratch memory is asked for before the pointers are known.)
    const bool adjacent = p.xs[2] == 1 && (backward ? p.ds[2] == 1 && p.dxs[2] == 1 : p.os[2] == 1);
    if (adjacent && p.G >= 2 && p.G <= 4) {
        plan.vec = p.G;
        plan.shared = 1;
    } else if (adjacent && p.G == 1 && p.gs[2] == 1 && (!backward || p.dgs[2] == 1)) {
        const int most = widestLane(dtype == FVSRN_TENSOR_F32 ? 4 : 2, backward);
        for (int v = most; v > 1 && plan.vec == 1; v >>= 1)
            if (p.C % v == 0 && p.C >= 64 * v) plan.vec = v;
    }
    const int L = backward ? backwardSteps(plan.vec, dtype == FVSRN_TENSOR_F32 ? 4 : 2) : forwardSteps(plan.vec);
    if (backward && p.G > 1 && !plan.shared) {
        plan.slots = std::min(64, powerOfTwoAtLeast(p.G));
        plan.parts = (p.G + 63) / 64;
    }
    const long long units = p.B * channelBlocks(p, plan);
    // Waves share a tile of steps while there are fewer than 16 waves of channels for each of the 256 CUs.
    plan.waves = units >= 4096 || p.T <= 2 * L ? 1 : kScanWaves;
    plan.tile = plan.waves * L;
    const int tiles = int((p.T + (long long)plan.tile - 1) / plan.tile);
    // Spans: two workgroups for each CU (384 for the chip: 164 us where 512 take 138, 768 152, 2048 238), and at least two tiles a span.
    const long long want = plan.waves == 1 ? 1 : (512 + units - 1) / units;
    const int spans = int(std::max(1LL, std::min(want, (long long)tiles / 2)));
    const int tilesOfSpan = std::max(1, (tiles + spans - 1) / spans);
    plan.chunks = std::max(1, (tiles + tilesOfSpan - 1) / tilesOfSpan);
    plan.chunkSteps = tilesOfSpan * plan.tile;
    // A few tiles of twice the waves in one launch are better than spans in two: 16 x 500 x 1024 23 us against 29, 100 x 1001 x 64 22 against 27, 1 x 256 x 256 10
    // against 13; with few workgroups only up to two tiles (1 x 500 x 256: 18 us against 13).
    const int wide = 2 * kScanWaves * L, wideTiles = int((p.T + (long long)wide - 1) / wide);
    if (!backward && plan.chunks > 1 && wideTiles <= (units >= 96 ? 4 : 2)) {
        plan.waves = 2 * kScanWaves;
        plan.tile = wide;
        plan.chunks = 1;
        plan.chunkSteps = wideTiles * wide;
    }
    plan.wsFloats = backward ? backwardFloats(p, plan) : plan.chunks > 1 ? 2 * size_t(p.B) * p.C * plan.chunks : 0;
    return plan;
}

hipError_t launch_gated_scan(const ScanParams& p, const ScanPlan& plan, int dtype, hipStream_t s) {
    return withType(dtype, [&](auto element) {
        typedef decltype(element) T;
        if (plan.rows) {
            const dim3 grid(unsigned((p.B * p.Cg * plan.width + 255) / 256), unsigned(plan.chunks));
            const bool beside = gateBeside(p.x, p.xs, p.gate, p.gs, p, sizeof(T));
            return withGroup(p.G, [&](auto g) {
                if (plan.chunks > 1) {
                    scan_rows_spans_kernel<T, decltype(g)::value, false><<<grid, 256, 0, s>>>(p, plan, beside);
                    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
                }
                scan_rows_kernel<T, decltype(g)::value><<<grid, 256, 0, s>>>(p, plan, beside);
                return hipGetLastError();
            });
        }
        const int blocks = int(channelBlocks(p, plan));
        const long long units = p.B * blocks;
        return withLane<T, false>(plan, [&](auto vec, auto shared) {
            constexpr int V = decltype(vec)::value;
            constexpr bool SHARED = decltype(shared)::value;
            if (plan.waves == 1) {
                scan_channels_kernel<T, 1, V, SHARED, false><<<unsigned((units + 3) / 4), 256, 0, s>>>(p, plan, blocks, units);
                return hipGetLastError();
            }
            const dim3 grid(unsigned(units), unsigned(plan.chunks));
            if (plan.waves > kScanWaves) {
                scan_channels_kernel<T, 2 * kScanWaves, V, SHARED, false><<<grid, 128 * kScanWaves, 0, s>>>(p, plan, blocks, units);
                return hipGetLastError();
            }
            if (plan.chunks > 1) {
                scan_channels_kernel<T, kScanWaves, V, SHARED, true><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks, units);
                if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            }
            scan_channels_kernel<T, kScanWaves, V, SHARED, false><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks, units);
            return hipGetLastError();
        });
    });
}

hipError_t launch_gated_scan_backward(const ScanParams& p, const ScanPlan& plan, int dtype, hipStream_t s) {
    return withType(dtype, [&](auto element) {
        typedef decltype(element) T;
        if (plan.rows) {
            const dim3 grid(unsigned((p.B * p.Cg * plan.width + 255) / 256), unsigned(plan.chunks));
            const bool beside = gateBeside(p.x, p.xs, p.gate, p.gs, p, sizeof(T));
            const bool outBeside = p.dx && p.dgate && gateBeside(p.dx, p.dxs, p.dgate, p.dgs, p, sizeof(T));
            return withGroup(p.G, [&](auto g) {
                if (plan.chunks > 1) {
                    scan_rows_spans_kernel<T, decltype(g)::value, true><<<grid, 256, 0, s>>>(p, plan, beside);
                    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
                }
                if (rowSteps(p.T, true) == kRowStepsShort) scan_rows_backward_kernel<T, decltype(g)::value, kRowStepsShort><<<grid, 256, 0, s>>>(p, plan, beside, outBeside);
                else scan_rows_backward_kernel<T, decltype(g)::value, kRowSteps><<<grid, 256, 0, s>>>(p, plan, beside, outBeside);
                return hipGetLastError();
            });
        }
        const int blocks = int(channelBlocks(p, plan));
        const long long units = p.B * blocks;
        const hipError_t e = withLane<T, true>(plan, [&](auto vec, auto shared) {
            constexpr int V = decltype(vec)::value;
            constexpr bool SHARED = decltype(shared)::value;
            if (plan.waves == 1) {
                scan_channels_backward_kernel<T, 1, V, SHARED><<<unsigned((units + 3) / 4), 256, 0, s>>>(p, plan, blocks, units);
                return hipGetLastError();
            }
            const dim3 grid(unsigned(units), unsigned(plan.chunks));
            if (plan.chunks > 1) {
                scan_channels_spans_kernel<T, kScanWaves, V, SHARED><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks);
                if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            }
            scan_channels_backward_kernel<T, kScanWaves, V, SHARED><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks, units);
            return hipGetLastError();
        });
        if (e != hipSuccess || plan.parts == 1 || !p.dgate) return e;
        const long long count = p.B * p.T * (long long)p.Cg;
        scan_gate_sum_kernel<T><<<unsigned(std::min(4096LL, (count + 255) / 256)), 256, 0, s>>>(p, backwardScratch(p, plan).partial, plan.parts);
        return hipGetLastError();
    });
}

}  // namespace fvsrn
