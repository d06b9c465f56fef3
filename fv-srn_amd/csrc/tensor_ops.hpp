// Launch interface of the tensor operators (gated_scan.hip, int8_product.hip); the checks of arguments are in tensor_ops.cpp.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>

namespace fvsrn {

struct ScanParams {
    const void *gate, *x, *dout;
    const float *h0, *dlast;
    const int* lengths;
    void *out, *dgate, *dx;
    float *last, *dh0;
    float* ws;
    long long gs[3], xs[3], os[3], ds[3], dgs[3], dxs[3];  // strides of gate, x, out, dout, dgate, dx: batch, step, channel
    long long B;
    int T, C, Cg, G;  // steps, channels, gate channels, channels of a gate
    float scale;
    int reverse, exp, blend;  // exp: FVSRN_GATE_EXP; blend: FVSRN_INPUT_BLEND
};

// How a call is cut (planScan): `rows` lays the lanes along the steps of one gate (few channels beside each other), otherwise lanes are channels.
struct ScanPlan {
    int rows;
    int width;       // rows: lanes of a wave that share a row
    int waves;       // channels: waves that share a tile of steps (1 or kScanWaves)
    int vec;         // channels: adjacent channels of a lane
    int shared;      // channels: those of a lane have one gate
    int tile;        // steps of a tile
    int chunks;      // spans of steps that run side by side
    int chunkSteps;  // steps of a span, a multiple of the tile
    int slots;       // backward, channels: lanes of a gate's channels (a power of two; 1: every channel has its own gate)
    int parts;       // backward, channels: lane groups that share one gate's sum
    size_t wsFloats; // scratch memory
};
ScanPlan planScan(const ScanParams& p, int dtype, bool backward);
hipError_t launch_gated_scan(const ScanParams& p, const ScanPlan& plan, int dtype, hipStream_t s);
hipError_t launch_gated_scan_backward(const ScanParams& p, const ScanPlan& plan, int dtype, hipStream_t s);

struct QuantizeParams {
    const void* x;
    signed char* codes;
    float* scales;
    long long rows, ldx, ldc;
    int cols;
};
int quantizeWidth(int cols);  // lanes of a row
hipError_t launch_quantize_rows(const QuantizeParams& p, int dtype, hipStream_t s);

struct Int8Params {
    const signed char *a, *b;
    const float *scaleA, *scaleB, *bias;
    void* out;
    long long lda, ldb, ldo, M;
    int N, K;
    float actParam;
};
hipError_t launch_matmul_int8(const Int8Params& p, int activation, int outDtype, hipStream_t s);

}  // namespace fvsrn
