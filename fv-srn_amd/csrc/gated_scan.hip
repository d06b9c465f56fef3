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

__device__ __forceinline__ int lengthOf(const ScanParams& p, long long b) {
    return p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
}
// step i of a sequence of n steps is at position t; behind the sequence (outputs are zero there) i is the position itself
__device__ __forceinline__ int positionOf(int i, int n, int reverse) { return reverse && i < n ? n - 1 - i : i; }

constexpr int kScanWaves = 8;    // channels: waves that share a tile
constexpr int kForwardSteps = 16; // channels: steps of a wave held in registers
constexpr int kBackwardSteps = 8;

// ---------------------------------------------------------------------------------------------------------------------
// lanes are channels
// ---------------------------------------------------------------------------------------------------------------------

// What a wave's lanes stand for.  slots == 1: 64 V adjacent channels.  Otherwise (backward) `slots` lanes of a gate's channels -- padded to a power of two, so
// that their sum is a butterfly of shuffles -- and, for gates of more than 64 channels, `parts` waves.
struct ChannelLane {
    int c, g, part;
    bool live;
};
template <int V>
__device__ __forceinline__ ChannelLane channelLane(const ScanParams& p, int block, int lane, int slots, int parts) {
    ChannelLane r;
    r.part = 0;
    if (slots == 1) {
        const long long c = (long long)(block * 64LL + lane) * V;
        r.live = c < p.C;
        r.c = int(min(c, (long long)(p.C - V)));
        r.g = r.c / p.G;
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
inline long long channelBlocks(const ScanParams& p, int vec, int slots, int parts) {
    if (slots == 1) return (p.C + 64LL * vec - 1) / (64LL * vec);
    if (parts == 1) return (p.Cg + 64 / slots - 1) / (64 / slots);
    return (long long)p.Cg * parts;
}

// Forward.  AGGREGATE: only (A, U) of this workgroup's span, span 0 with h0 folded in (its A slot then holds h0 for the second launch: d_last may be d_h0).
template <class T, bool EXP, bool BLEND, int NW, int V, bool AGGREGATE>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void scan_channels_kernel(const ScanParams p, const ScanPlan plan, const int blocks, const long long units) {
    constexpr int L = kForwardSteps;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int w = NW == 1 ? 0 : wave;
    const long long unit = NW == 1 ? blockIdx.x * 4LL + wave : blockIdx.x;
    if (unit >= units) return;  // (NW == 1 only, and nothing is joined across its waves)
    const long long b = unit / blocks;
    const ChannelLane ch = channelLane<V>(p, int(unit % blocks), lane, 1, 1);
    const int n = lengthOf(p, b), span = blockIdx.y;
    const int begin = span * plan.chunkSteps, end = min(p.out ? p.T : n, begin + plan.chunkSteps);
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + ch.g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + ch.c * p.xs[2];
    T* const op = p.out ? static_cast<T*>(p.out) + b * p.os[0] + ch.c * p.os[2] : nullptr;
    const long long state = b * p.C + ch.c, stored = (b * plan.chunks) * p.C + ch.c, plane = p.B * plan.chunks * p.C;
    float h[V], A[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A[v] = 1.f;
        h[v] = 0.f;
    }
    if (span == 0 || plan.chunks == 1) {
        if (p.h0)
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = p.h0[state + v];
        if constexpr (AGGREGATE) {
            if (w == 0 && ch.live)
#pragma unroll
                for (int v = 0; v < V; ++v) p.ws[stored + v] = h[v];
        }
    }
    if (!AGGREGATE && plan.chunks > 1) {
        const float* const wa = p.ws + stored;
        const float* const wu = wa + plane;
        if (span == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = wa[v];
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = wu[v];
            for (int s = 1; s < span; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = fmaf(wa[(long long)s * p.C + v], h[v], wu[(long long)s * p.C + v]);
        }
    }
    __shared__ float2 joined[NW == 1 ? 1 : 2][NW][NW == 1 ? 1 : 64 * V];
    int buffer = 0;
    for (int tile = begin; tile < end; tile += NW * L) {
        const int i0 = tile + w * L;
        float m[L][V], u[L][V];
#pragma unroll
        for (int k = 0; k < L; ++k) {
            const int i = i0 + k;
            if (i < n && i < end) {
                const long long t = positionOf(i, n, p.reverse);
                const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(xp + t * p.xs[1]);
                const Pack<T, V> g = *reinterpret_cast<const Pack<T, V>*>(gp + t * p.gs[1]);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    m[k][v] = toFloat(g.v[v]);
                    u[k][v] = toFloat(x.v[v]);
                }
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) m[k][v] = EXP ? 0.f : 1.f, u[k][v] = 0.f;
            }
        }
        float a2[V], u2[V];
#pragma unroll
        for (int v = 0; v < V; ++v) a2[v] = 1.f, u2[v] = 0.f;
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float rest;
                gateOf<EXP>(m[k][v], p.scale, m[k][v], rest);
                if (BLEND) u[k][v] *= rest;
                if (NW > 1 || AGGREGATE) {
                    u2[v] = fmaf(m[k][v], u2[v], u[k][v]);
                    a2[v] *= m[k][v];
                }
            }
        float pre[V];
#pragma unroll
        for (int v = 0; v < V; ++v) pre[v] = h[v];
        if constexpr (NW > 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) joined[buffer][w][lane * V + v] = make_float2(a2[v], u2[v]);
            __syncthreads();  // (one barrier a tile: the two buffers take turns, and a wave can only be one tile ahead)
#pragma unroll
            for (int j = 0; j < NW; ++j)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (j == w) pre[v] = h[v];
                    const float2 s = joined[buffer][j][lane * V + v];
                    h[v] = fmaf(s.x, h[v], s.y);
                    if (AGGREGATE) A[v] *= s.x;
                }
            buffer ^= 1;
        } else if constexpr (AGGREGATE) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = fmaf(a2[v], h[v], u2[v]);
                A[v] *= a2[v];
            }
        }
        if constexpr (!AGGREGATE) {
#pragma unroll
            for (int k = 0; k < L; ++k) {
                const int i = i0 + k;
#pragma unroll
                for (int v = 0; v < V; ++v) pre[v] = fmaf(m[k][v], pre[v], u[k][v]);
                if (op && i < end && ch.live) {
                    Pack<T, V> o;
#pragma unroll
                    for (int v = 0; v < V; ++v) o.v[v] = fromFloat<T>(i < n ? pre[v] : 0.f);
                    *reinterpret_cast<Pack<T, V>*>(op + (long long)positionOf(i, n, p.reverse) * p.os[1]) = o;
                }
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
            if (span > 0) wa[v] = A[v];
            wa[plane + v] = h[v];
        }
    } else if (p.last && span == plan.chunks - 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) p.last[state + v] = h[v];
    }
}

// Backward, first launch of a call that is cut into spans: A, U (span 0 from h0) and D of every span.
template <class T, bool EXP, bool BLEND, int NW>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void scan_channels_spans_kernel(const ScanParams p, const ScanPlan plan, const int blocks, const long long units) {
    constexpr int L = kBackwardSteps;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int w = NW == 1 ? 0 : wave;
    const long long unit = NW == 1 ? blockIdx.x * 4LL + wave : blockIdx.x;
    if (unit >= units) return;
    const long long b = unit / blocks;
    const ChannelLane ch = channelLane<1>(p, int(unit % blocks), lane, plan.slots, plan.parts);
    const int n = lengthOf(p, b), span = blockIdx.y;
    const int begin = span * plan.chunkSteps, end = min(n, begin + plan.chunkSteps);
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + ch.g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + ch.c * p.xs[2];
    const T* const dp = p.dout ? static_cast<const T*>(p.dout) + b * p.ds[0] + ch.c * p.ds[2] : nullptr;
    float A = 1.f, U = 0.f, D = 0.f;
    if (span == 0 && p.h0) U = p.h0[b * p.C + ch.c];
    __shared__ float4 joined[NW == 1 ? 1 : 2][NW][NW == 1 ? 1 : 64];
    int buffer = 0;
    for (int tile = begin; tile < end; tile += NW * L) {
        float a2 = 1.f, u2 = 0.f, d2 = 0.f;
#pragma unroll
        for (int k = 0; k < L; ++k) {
            const int i = tile + w * L + k;
            if (i < end) {
                const long long t = positionOf(i, n, p.reverse);
                float a, rest;
                gateOf<EXP>(toFloat(gp[t * p.gs[1]]), p.scale, a, rest);
                const float x = toFloat(xp[t * p.xs[1]]);
                u2 = fmaf(a, u2, BLEND ? rest * x : x);
                a2 *= a;
                if (dp) d2 = fmaf(a2, toFloat(dp[t * p.ds[1]]), d2);
            }
        }
        if constexpr (NW > 1) {
            joined[buffer][w][lane] = make_float4(a2, u2, d2, 0.f);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                const float4 s = joined[buffer][j][lane];
                U = fmaf(s.x, U, s.y);
                D = fmaf(A, s.z, D);
                A *= s.x;
            }
            buffer ^= 1;
        } else {
            U = fmaf(a2, U, u2);
            D = fmaf(A, d2, D);
            A *= a2;
        }
    }
    if (w != 0 || !ch.live) return;
    const long long plane = p.B * plan.chunks * p.C, at = (b * plan.chunks + span) * p.C + ch.c;
    p.ws[at] = A;
    p.ws[plane + at] = U;
    p.ws[2 * plane + at] = D;
}

template <class T, bool EXP, bool BLEND, int NW>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void scan_channels_backward_kernel(const ScanParams p, const ScanPlan plan, const int blocks, const long long units) {
    constexpr int L = kBackwardSteps;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int w = NW == 1 ? 0 : wave;
    const long long unit = NW == 1 ? blockIdx.x * 4LL + wave : blockIdx.x;
    if (unit >= units) return;
    const long long b = unit / blocks;
    const ChannelLane ch = channelLane<1>(p, int(unit % blocks), lane, plan.slots, plan.parts);
    const int n = lengthOf(p, b), span = blockIdx.y;
    const int begin = span * plan.chunkSteps, end = min(p.T, begin + plan.chunkSteps);
    const int tiles = (end - begin + plan.tile - 1) / plan.tile;
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + ch.g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + ch.c * p.xs[2];
    const T* const dp = p.dout ? static_cast<const T*>(p.dout) + b * p.ds[0] + ch.c * p.ds[2] : nullptr;
    T* const dgp = p.dgate ? static_cast<T*>(p.dgate) + b * p.dgs[0] + ch.g * p.dgs[2] : nullptr;
    T* const dxp = p.dx ? static_cast<T*>(p.dx) + b * p.dxs[0] + ch.c * p.dxs[2] : nullptr;
    const long long plane = plan.chunks > 1 ? p.B * plan.chunks * p.C : 0;
    const long long state = b * p.C + ch.c;
    const int tilesOfSpan = plan.chunkSteps / plan.tile;
    // the states at the head of every tile, if a span has more than one
    const bool kept = tilesOfSpan > 1;
    float* const heads = p.ws + 3 * plane + ((b * plan.chunks + span) * tilesOfSpan) * p.C + ch.c;
    float* const partial = p.ws + 3 * plane + (kept ? p.B * plan.chunks * tilesOfSpan * p.C : 0) + b * p.T * (long long)p.Cg * plan.parts + (long long)ch.g * plan.parts + ch.part;
    float h = 0.f, k = p.dlast ? p.dlast[state] : 0.f;
    if (p.h0) h = p.h0[state];
    if (plan.chunks > 1) {
        const float* const wa = p.ws + (b * plan.chunks) * p.C + ch.c;
        if (span > 0) {
            h = wa[plane];
            for (int s = 1; s < span; ++s) h = fmaf(wa[(long long)s * p.C], h, wa[plane + (long long)s * p.C]);
        }
        for (int s = plan.chunks - 1; s > span; --s) k = fmaf(wa[(long long)s * p.C], k, wa[2 * plane + (long long)s * p.C]);
    }
    __shared__ float4 joined[NW == 1 ? 1 : 2][NW][NW == 1 ? 1 : 64];
    int buffer = 0;
    if (kept) {
        for (int j = 0; j < tiles; ++j) {
            if (w == 0) heads[(long long)j * p.C] = h;  // (written and read again by this lane; dead lanes: the copy of a live one's channel)
            float a2 = 1.f, u2 = 0.f;
#pragma unroll
            for (int q = 0; q < L; ++q) {
                const int i = begin + j * plan.tile + w * L + q;
                if (i < n && i < end) {
                    const long long t = positionOf(i, n, p.reverse);
                    float a, rest;
                    gateOf<EXP>(toFloat(gp[t * p.gs[1]]), p.scale, a, rest);
                    const float x = toFloat(xp[t * p.xs[1]]);
                    u2 = fmaf(a, u2, BLEND ? rest * x : x);
                    a2 *= a;
                }
            }
            if constexpr (NW > 1) {
                joined[buffer][w][lane] = make_float4(a2, u2, 0.f, 0.f);
                __syncthreads();
#pragma unroll
                for (int s = 0; s < NW; ++s) h = fmaf(joined[buffer][s][lane].x, h, joined[buffer][s][lane].y);
                buffer ^= 1;
            } else {
                h = fmaf(a2, h, u2);
            }
        }
    }
    for (int j = tiles - 1; j >= 0; --j) {
        const int i0 = begin + j * plan.tile + w * L;
        float m[L], rest[L], x[L], d[L], before[L];
#pragma unroll
        for (int q = 0; q < L; ++q) {
            const int i = i0 + q;
            m[q] = EXP ? 0.f : 1.f;
            x[q] = d[q] = 0.f;
            if (i < n && i < end) {
                const long long t = positionOf(i, n, p.reverse);
                m[q] = toFloat(gp[t * p.gs[1]]);
                x[q] = toFloat(xp[t * p.xs[1]]);
                if (dp) d[q] = toFloat(dp[t * p.ds[1]]);
            }
        }
        // (the head of the tile: every wave of it needs the state that wave 0 kept)
        if (kept && NW == 1) h = heads[(long long)j * p.C];
        float a2 = 1.f, u2 = 0.f, d2 = 0.f;
#pragma unroll
        for (int q = 0; q < L; ++q) {
            gateOf<EXP>(m[q], p.scale, m[q], rest[q]);
            u2 = fmaf(m[q], u2, BLEND ? rest[q] * x[q] : x[q]);
            a2 *= m[q];
            d2 = fmaf(a2, d[q], d2);
        }
        float hw = h, kw = k;
        if constexpr (NW > 1) {
            float4 mine = make_float4(a2, u2, d2, 0.f);
            if (w == 0) mine.w = kept ? heads[(long long)j * p.C] : h;
            joined[buffer][w][lane] = mine;
            __syncthreads();
            hw = joined[buffer][0][lane].w;
#pragma unroll
            for (int s = 0; s < NW - 1; ++s)
                if (s < w) hw = fmaf(joined[buffer][s][lane].x, hw, joined[buffer][s][lane].y);
#pragma unroll
            for (int s = NW - 1; s >= 0; --s) {
                if (s == w) kw = k;
                k = fmaf(joined[buffer][s][lane].x, k, joined[buffer][s][lane].z);
            }
            buffer ^= 1;
        }
#pragma unroll
        for (int q = 0; q < L; ++q) {
            before[q] = hw;
            hw = fmaf(m[q], hw, BLEND ? rest[q] * x[q] : x[q]);
        }
#pragma unroll
        for (int q = L - 1; q >= 0; --q) {
            const int i = i0 + q;
            const float a = m[q], l = d[q] + kw;
            const bool in = i < n && i < end;
            const long long t = positionOf(i, n, p.reverse);
            if (dxp && i < end && ch.live) dxp[t * p.dxs[1]] = fromFloat<T>(in ? (BLEND ? rest[q] * l : l) : 0.f);
            if (p.dgate) {
                float s = l * (BLEND ? before[q] - x[q] : before[q]);
                if (EXP) s *= p.scale * a;
                if (plan.slots > 1) {
                    s = ch.live ? s : 0.f;
                    for (int o = 1; o < plan.slots; o <<= 1) s += __shfl_xor(s, o, 64);
                }
                const bool first = plan.slots == 1 || (lane & (plan.slots - 1)) == 0;
                if (i < end && ch.live && first) {
                    if (plan.parts > 1) partial[t * (long long)p.Cg * plan.parts] = in ? s : 0.f;
                    else dgp[t * p.dgs[1]] = fromFloat<T>(in ? s : 0.f);
                }
            }
            kw = a * l;
        }
        if constexpr (NW == 1) k = kw;
    }
    if (p.dh0 && span == 0 && w == 0 && ch.live) p.dh0[state] = k;
}

// Sums of the parts of gates with more than 64 channels, in their order.
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

constexpr int kRowSteps = 8;          // steps of a lane, forward
constexpr int kRowStepsBackward = 4;  // and backward

// Inclusive scan over the `width` lanes of a row: (A, U) of every span from the row's first lane to this one (FORWARD), or (A, U) = (A, D) from this lane to
// the row's last.
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

template <class T, bool EXP, bool BLEND, int G>
__global__ __launch_bounds__(256) void scan_rows_kernel(const ScanParams p, const int width) {
    constexpr int K = kRowSteps;
    const int lane = threadIdx.x & 63, at = lane & (width - 1);
    const long long rows = p.B * p.Cg, own = (blockIdx.x * 4LL + (threadIdx.x >> 6)) * (64 / width) + lane / width;
    const bool live = own < rows;
    const long long row = live ? own : rows - 1, b = row / p.Cg, g = row % p.Cg;
    const int n = lengthOf(p, b);
    const T* const gp = static_cast<const T*>(p.gate) + b * p.gs[0] + g * p.gs[2];
    const T* const xp = static_cast<const T*>(p.x) + b * p.xs[0] + g * G * p.xs[2];
    T* const op = p.out ? static_cast<T*>(p.out) + b * p.os[0] + g * G * p.os[2] : nullptr;
    const long long state = b * p.C + g * G;
    float h[G];
#pragma unroll
    for (int c = 0; c < G; ++c) h[c] = p.h0 ? p.h0[state + c] : 0.f;
    for (int tile = 0; tile < p.T; tile += width * K) {
        const int i0 = tile + at * K;
        float m[K], u[K][G];
#pragma unroll
        for (int q = 0; q < K; ++q) {
            const int i = i0 + q;
            m[q] = EXP ? 0.f : 1.f;
#pragma unroll
            for (int c = 0; c < G; ++c) u[q][c] = 0.f;
            if (i < n) {
                const long long t = positionOf(i, n, p.reverse);
                m[q] = toFloat(gp[t * p.gs[1]]);
#pragma unroll
                for (int c = 0; c < G; ++c) u[q][c] = toFloat(xp[t * p.xs[1] + c * p.xs[2]]);
            }
        }
        float A = 1.f, U[G];
#pragma unroll
        for (int c = 0; c < G; ++c) U[c] = 0.f;
#pragma unroll
        for (int q = 0; q < K; ++q) {
            float rest;
            gateOf<EXP>(m[q], p.scale, m[q], rest);
#pragma unroll
            for (int c = 0; c < G; ++c) {
                if (BLEND) u[q][c] *= rest;
                U[c] = fmaf(m[q], U[c], u[q][c]);
            }
            A *= m[q];
        }
        joinLanes<G, true>(A, U, width, lane);
        // the state that enters this lane's span: the row's, taken through the lanes before
        float before = __shfl_up(A, 1, width), pre[G];
#pragma unroll
        for (int c = 0; c < G; ++c) {
            const float u1 = __shfl_up(U[c], 1, width);
            pre[c] = at ? fmaf(before, h[c], u1) : h[c];
            h[c] = __shfl(fmaf(A, h[c], U[c]), width - 1, width);
        }
        if (op) {
#pragma unroll
            for (int q = 0; q < K; ++q) {
                const int i = i0 + q;
                const long long t = positionOf(i, n, p.reverse);
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    pre[c] = fmaf(m[q], pre[c], u[q][c]);
                    if (i < p.T && live) op[t * p.os[1] + c * p.os[2]] = fromFloat<T>(i < n ? pre[c] : 0.f);
                }
            }
        }
    }
    if (p.last && live && at == 0)
#pragma unroll
        for (int c = 0; c < G; ++c) p.last[state + c] = h[c];
}

template <class T, bool EXP, bool BLEND, int G>
__global__ __launch_bounds__(256) void scan_rows_backward_kernel(const ScanParams p, const int width) {
    constexpr int K = kRowStepsBackward;
    const int lane = threadIdx.x & 63, at = lane & (width - 1);
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
    const int tile = width * K, tiles = (p.T + tile - 1) / tile;
    float* const heads = p.ws + row * tiles * G;  // the row's state at the head of each tile, if there is more than one
    float h[G], k[G];
#pragma unroll
    for (int c = 0; c < G; ++c) {
        h[c] = p.h0 ? p.h0[state + c] : 0.f;
        k[c] = p.dlast ? p.dlast[state + c] : 0.f;
    }
    for (int pass = tiles > 1 ? 0 : 1; pass < 2; ++pass) {
        for (int step = 0; step < tiles; ++step) {
            const int j = pass ? tiles - 1 - step : step;
            const int i0 = j * tile + at * K;
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
#pragma unroll
            for (int q = 0; q < K; ++q) {
                const int i = i0 + q;
                m[q] = EXP ? 0.f : 1.f;
#pragma unroll
                for (int c = 0; c < G; ++c) x[q][c] = d[q][c] = 0.f;
                if (i < n) {
                    const long long t = positionOf(i, n, p.reverse);
                    m[q] = toFloat(gp[t * p.gs[1]]);
#pragma unroll
                    for (int c = 0; c < G; ++c) x[q][c] = toFloat(xp[t * p.xs[1] + c * p.xs[2]]);
                    if (dp && pass)
#pragma unroll
                        for (int c = 0; c < G; ++c) d[q][c] = toFloat(dp[t * p.ds[1] + c * p.ds[2]]);
                }
            }
            float A = 1.f, U[G], D[G];
#pragma unroll
            for (int c = 0; c < G; ++c) U[c] = D[c] = 0.f;
#pragma unroll
            for (int q = 0; q < K; ++q) {
                gateOf<EXP>(m[q], p.scale, m[q], rest[q]);
                A *= m[q];
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    U[c] = fmaf(m[q], U[c], BLEND ? rest[q] * x[q][c] : x[q][c]);
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
            joinLanes<G, false>(A2, D, width, lane);
            const float behind = __shfl_down(A2, 1, width);
            float kw[G], state1[K][G];
#pragma unroll
            for (int c = 0; c < G; ++c) {
                const float d1 = __shfl_down(D[c], 1, width);
                kw[c] = at + 1 < width ? fmaf(behind, k[c], d1) : k[c];
                k[c] = __shfl(fmaf(A2, k[c], D[c]), 0, width);
            }
#pragma unroll
            for (int q = 0; q < K; ++q)
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    state1[q][c] = pre[c];
                    pre[c] = fmaf(m[q], pre[c], BLEND ? rest[q] * x[q][c] : x[q][c]);
                }
#pragma unroll
            for (int q = K - 1; q >= 0; --q) {
                const int i = i0 + q;
                const long long t = positionOf(i, n, p.reverse);
                const float a = m[q];
                float s = 0.f;
#pragma unroll
                for (int c = 0; c < G; ++c) {
                    const float l = d[q][c] + kw[c];
                    s = fmaf(l, BLEND ? state1[q][c] - x[q][c] : state1[q][c], s);
                    if (dxp && i < p.T && live) dxp[t * p.dxs[1] + c * p.dxs[2]] = fromFloat<T>(i < n ? (BLEND ? rest[q] * l : l) : 0.f);
                    kw[c] = a * l;
                }
                if (EXP) s *= p.scale * a;
                if (dgp && i < p.T && live) dgp[t * p.dgs[1]] = fromFloat<T>(i < n ? s : 0.f);
            }
        }
    }
    if (p.dh0 && live && at == 0)
#pragma unroll
        for (int c = 0; c < G; ++c) p.dh0[state + c] = k[c];
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
hipError_t withTypes(int dtype, int gateMode, int inputMode, F&& f) {
    auto modes = [&](auto element) {
        if (gateMode == FVSRN_GATE_EXP) return inputMode == FVSRN_INPUT_BLEND ? f(element, std::true_type{}, std::true_type{}) : f(element, std::true_type{}, std::false_type{});
        return inputMode == FVSRN_INPUT_BLEND ? f(element, std::false_type{}, std::true_type{}) : f(element, std::false_type{}, std::false_type{});
    };
    if (dtype == FVSRN_TENSOR_F16) return modes(f16_t{});
    if (dtype == FVSRN_TENSOR_BF16) return modes(bf16_t{});
    return modes(float{});
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

}  // namespace

ScanPlan planScan(const ScanParams& p, int dtype, bool backward) {
    ScanPlan plan{};
    plan.slots = plan.parts = plan.vec = plan.chunks = plan.waves = 1;
    const long long step = std::llabs(p.xs[1]), next = std::llabs(p.xs[2]) * p.G;
    // Lanes along the steps where steps lie closer together than gates (colours along a ray: step 4, next ray's far away), or where there are too few
    // gates beside each other to fill half a wave.
    plan.rows = p.G <= 4 && (p.Cg < 32 || step < next);
    if (plan.rows) {
        const int K = backward ? kRowStepsBackward : kRowSteps;
        plan.width = std::min(64, powerOfTwoAtLeast((p.T + K - 1) / std::max(K, 1)));
        plan.tile = plan.width * K;
        const long long tiles = (p.T + (long long)plan.tile - 1) / plan.tile;
        plan.chunkSteps = p.T;
        plan.wsFloats = backward && tiles > 1 ? size_t(p.B) * p.C * tiles : 0;
        return plan;
    }
    const int L = backward ? kBackwardSteps : kForwardSteps;
    if (backward && p.G > 1) {
        plan.slots = std::min(64, powerOfTwoAtLeast(p.G));
        plan.parts = (p.G + 63) / 64;
    }
    const long long units = p.B * channelBlocks(p, plan.vec, plan.slots, plan.parts);
    // Waves share a tile of steps while there are fewer than 16 waves of channels for each of the 256 CUs.
    plan.waves = units >= 4096 || p.T <= 2 * L ? 1 : kScanWaves;
    plan.tile = plan.waves * L;
    const int tiles = int((p.T + (long long)plan.tile - 1) / plan.tile);
    // Spans: two workgroups for each CU, and at least two tiles a span.
    const long long want = plan.waves == 1 ? 1 : (512 + units - 1) / units;
    const int spans = int(std::max(1LL, std::min(want, (long long)tiles / 2)));
    const int tilesOfSpan = (tiles + spans - 1) / std::max(1, spans);
    plan.chunks = std::max(1, (tiles + tilesOfSpan - 1) / std::max(1, tilesOfSpan));
    plan.chunkSteps = std::max(1, tilesOfSpan) * plan.tile;
    const size_t state = size_t(p.B) * p.C;
    if (!backward) {
        plan.wsFloats = plan.chunks > 1 ? 2 * state * plan.chunks : 0;
    } else {
        plan.wsFloats = plan.chunks > 1 ? 3 * state * plan.chunks : 0;
        if (tilesOfSpan > 1) plan.wsFloats += state * plan.chunks * tilesOfSpan;
        if (plan.parts > 1) plan.wsFloats += size_t(p.B) * p.T * p.Cg * plan.parts;
    }
    return plan;
}

hipError_t launch_gated_scan(const ScanParams& p, const ScanPlan& plan, int dtype, int gateMode, int inputMode, hipStream_t s) {
    return withTypes(dtype, gateMode, inputMode, [&](auto element, auto isExp, auto isBlend) {
        typedef decltype(element) T;
        constexpr bool EXP = decltype(isExp)::value, BLEND = decltype(isBlend)::value;
        if (plan.rows) {
            const unsigned grid = unsigned((p.B * p.Cg * plan.width + 255) / 256);
            return withGroup(p.G, [&](auto g) {
                scan_rows_kernel<T, EXP, BLEND, decltype(g)::value><<<grid, 256, 0, s>>>(p, plan.width);
                return hipGetLastError();
            });
        }
        const int blocks = int(channelBlocks(p, plan.vec, 1, 1));
        const long long units = p.B * blocks;
        if (plan.waves == 1) {
            scan_channels_kernel<T, EXP, BLEND, 1, 1, false><<<unsigned((units + 3) / 4), 256, 0, s>>>(p, plan, blocks, units);
            return hipGetLastError();
        }
        const dim3 grid(unsigned(units), unsigned(plan.chunks));
        if (plan.chunks > 1) {
            scan_channels_kernel<T, EXP, BLEND, kScanWaves, 1, true><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks, units);
            if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
        scan_channels_kernel<T, EXP, BLEND, kScanWaves, 1, false><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks, units);
        return hipGetLastError();
    });
}

hipError_t launch_gated_scan_backward(const ScanParams& p, const ScanPlan& plan, int dtype, int gateMode, int inputMode, hipStream_t s) {
    return withTypes(dtype, gateMode, inputMode, [&](auto element, auto isExp, auto isBlend) {
        typedef decltype(element) T;
        constexpr bool EXP = decltype(isExp)::value, BLEND = decltype(isBlend)::value;
        if (plan.rows) {
            const unsigned grid = unsigned((p.B * p.Cg * plan.width + 255) / 256);
            return withGroup(p.G, [&](auto g) {
                scan_rows_backward_kernel<T, EXP, BLEND, decltype(g)::value><<<grid, 256, 0, s>>>(p, plan.width);
                return hipGetLastError();
            });
        }
        const int blocks = int(channelBlocks(p, 1, plan.slots, plan.parts));
        const long long units = p.B * blocks;
        if (plan.waves == 1) {
            scan_channels_backward_kernel<T, EXP, BLEND, 1><<<unsigned((units + 3) / 4), 256, 0, s>>>(p, plan, blocks, units);
        } else {
            const dim3 grid(unsigned(units), unsigned(plan.chunks));
            if (plan.chunks > 1) {
                scan_channels_spans_kernel<T, EXP, BLEND, kScanWaves><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks, units);
                if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            }
            scan_channels_backward_kernel<T, EXP, BLEND, kScanWaves><<<grid, 64 * kScanWaves, 0, s>>>(p, plan, blocks, units);
        }
        if (const hipError_t e = hipGetLastError(); e != hipSuccess || plan.parts == 1 || !p.dgate) return e;
        const long long count = p.B * p.T * (long long)p.Cg;
        const float* const partial = p.ws + plan.wsFloats - size_t(count) * plan.parts;
        scan_gate_sum_kernel<T><<<unsigned(std::min(4096LL, (count + 255) / 256)), 256, 0, s>>>(p, partial, plan.parts);
        return hipGetLastError();
    });
}

}  // namespace fvsrn
