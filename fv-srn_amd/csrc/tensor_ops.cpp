// C ABI of the tensor operators (include/fvsrn.h: fvsrn_quantize_rows, fvsrn_matmul_int8, fvsrn_gated_scan*): every argument is checked here, on the host,
// before anything is enqueued; the kernels are in gated_scan.hip and int8_product.hip.
#include "api_internal.hpp"
#include "tensor_ops.hpp"

namespace {

bool knownDtype(int d) { return d == FVSRN_TENSOR_F32 || d == FVSRN_TENSOR_F16 || d == FVSRN_TENSOR_BF16; }
size_t elementSize(int d) { return d == FVSRN_TENSOR_F32 ? 4 : 2; }

int noDevice() { return fail(FVSRN_ERR_NO_DEVICE, "no HIP device available: the MI355X kernels cannot run (there is no CPU fallback)"); }

// Addresses an operand reaches, [first, last); empty ones overlap nothing
struct Range {
    const char* name = "";
    unsigned long long first = 0, last = 0;
    bool operator&&(const Range& o) const { return first < o.last && o.first < last; }
};

// false: the operand's addresses leave 64 bits, or it does not begin at a multiple of its element
bool rangeOf(const char* name, const void* ptr, size_t element, int dims, const long long* size, const long long* stride, Range& r) {
    r.name = name;
    if (!ptr) return true;
    __int128 lo = 0, hi = 0;
    for (int d = 0; d < dims; ++d) {
        if (size[d] == 0) return true;
        const __int128 reach = __int128(size[d] - 1) * stride[d];
        (reach < 0 ? lo : hi) += reach;
    }
    const __int128 base = reinterpret_cast<unsigned long long>(ptr);
    const __int128 first = base + lo * __int128(element), last = base + (hi + 1) * __int128(element);
    if (first < 0 || last > (__int128(1) << 63) || base % __int128(element) != 0) return false;
    r.first = (unsigned long long)first;
    r.last = (unsigned long long)last;
    return true;
}

unsigned long long magnitude(long long v) { return v < 0 ? 0ull - (unsigned long long)v : (unsigned long long)v; }

// Two elements (of `extent` strides' units each) of an output share an address: sorted by stride, some dimension does not step over all of the smaller ones
bool overlapsItself(const long long* size, const long long* stride, int dims, __int128 extent = 1) {
    for (int d = 0; d < dims; ++d)
        if (size[d] == 0) return false;
    int order[3] = {0, 1, 2};
    std::sort(order, order + dims, [&](int a, int b) { return magnitude(stride[a]) < magnitude(stride[b]); });
    __int128 reach = extent - 1;
    for (int j = 0; j < dims; ++j) {
        const int d = order[j];
        if (size[d] <= 1) continue;
        const __int128 s = stride[d] < 0 ? -__int128(stride[d]) : __int128(stride[d]);
        if (s <= reach) return true;
        reach += s * (size[d] - 1);
    }
    return false;
}

// Whether dgate and dx sit beside each other in one tensor, as the gate and x of colours with their absorption do: the same batch and step strides, and the
// channels of a step apart from each other and from every other step's
bool besideEachOther(const ScanParams& p, const void* dgate, const void* dx, long long e) {
    const long long outer[2] = {p.B, p.T}, stride[2] = {p.dxs[0], p.dxs[1]};
    for (int i = 0; i < 2; ++i)
        if (outer[i] > 1 && p.dgs[i] != p.dxs[i]) return false;
    if (p.dgs[2] < 0 || p.dxs[2] < 0) return false;
    const __int128 g0 = reinterpret_cast<unsigned long long>(dgate), x0 = reinterpret_cast<unsigned long long>(dx);
    const __int128 g1 = g0 + (__int128(p.Cg - 1) * p.dgs[2] + 1) * e, x1 = x0 + (__int128(p.C - 1) * p.dxs[2] + 1) * e;
    if (!(g1 <= x0 || x1 <= g0)) return false;
    const __int128 hull = std::max(g1, x1) - std::min(g0, x0);
    return !overlapsItself(outer, stride, 2, (hull + e - 1) / e);
}

std::string overlapping(const std::vector<Range>& outputs, const std::vector<Range>& inputs) {
    for (size_t i = 0; i < outputs.size(); ++i) {
        for (const Range& in : inputs)
            if (outputs[i] && in) return std::string(outputs[i].name) + " overlaps " + in.name;
    }
    return "";
}

// A launch has less than 2^32 threads in a dimension, whole workgroups of up to 256 (of 512: counted in them)
constexpr long long kMaxThreads = (1LL << 32) - 256;

struct ScanCall {
    const char* what;
    const fvsrn_scan_desc* d;
    ScanParams p{};
    ScanPlan plan{};
};

int scanShape(ScanCall& c, bool backward) {
    const fvsrn_scan_desc& d = *c.d;
    if (!knownDtype(d.dtype)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "unknown dtype");
    if (d.gate_mode != FVSRN_GATE_VALUE && d.gate_mode != FVSRN_GATE_EXP) return fail(FVSRN_ERR_INVALID_ARGUMENT, "unknown gate mode");
    if (d.input_mode != FVSRN_INPUT_ADD && d.input_mode != FVSRN_INPUT_BLEND) return fail(FVSRN_ERR_INVALID_ARGUMENT, "unknown input mode");
    if (d.gate_mode == FVSRN_GATE_EXP && !std::isfinite(d.gate_scale)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "gate_scale must be finite");
    if (d.length < 0 || d.batch < 0 || d.channels < 0 || d.gate_channels < 0) return fail(FVSRN_ERR_INVALID_ARGUMENT, "negative size");
    if (d.channels > 0 && (d.gate_channels == 0 || d.channels % d.gate_channels != 0)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "gate_channels must divide channels");
    // (what the kernels hold in 32 bits; more elements than this do not fit the memory either)
    if (d.channels > (1LL << 30) || d.length > (1 << 30)) return fail(FVSRN_ERR_UNSUPPORTED, "more than 2^30 channels or steps");
    if (d.batch > (1LL << 31) || __int128(d.batch) * std::max(1LL, d.channels) > (__int128(1) << 36) ||
        __int128(d.batch) * std::max(1LL, d.channels) * std::max(1, d.length) > (__int128(1) << 40))
        return fail(FVSRN_ERR_UNSUPPORTED, "too many elements for one call");
    ScanParams& p = c.p;
    p.B = d.batch; p.T = d.length; p.C = int(d.channels); p.Cg = int(d.gate_channels);
    p.G = p.Cg ? p.C / p.Cg : 1;
    p.scale = d.gate_scale;
    p.reverse = d.reverse != 0;
    p.exp = d.gate_mode == FVSRN_GATE_EXP;
    p.blend = d.input_mode == FVSRN_INPUT_BLEND;
    for (int i = 0; i < 3; ++i) {
        p.gs[i] = d.gate_stride[i]; p.xs[i] = d.x_stride[i]; p.os[i] = d.out_stride[i];
        p.ds[i] = d.dout_stride[i]; p.dgs[i] = d.dgate_stride[i]; p.dxs[i] = d.dx_stride[i];
    }
    if (p.B && p.C) c.plan = planScan(p, d.dtype, backward);
    return FVSRN_OK;
}

int scanLaunchable(const ScanCall& c) {
    const ScanParams& p = c.p;
    const __int128 lanes = c.plan.rows ? __int128(p.B) * p.Cg * c.plan.width
                                       : __int128(p.B) * (__int128(p.C) * (c.plan.slots > 1 ? 2 : 1) + 64) * c.plan.waves;
    if (lanes > kMaxThreads) return fail(FVSRN_ERR_UNSUPPORTED, std::string(c.what) + ": too many sequences for one launch, split the batch");
    return FVSRN_OK;
}

}  // namespace

extern "C" {

size_t fvsrn_scan_desc_size(void) { return sizeof(fvsrn_scan_desc); }

int fvsrn_gated_scan_workspace(const fvsrn_scan_desc* desc, int backward, size_t* bytes) {
    if (!desc || !bytes) return fail(FVSRN_ERR_INVALID_ARGUMENT, "null pointer");
    return guarded([&]() -> int {
        ScanCall c{"gated_scan", desc};
        if (const int rc = scanShape(c, backward != 0)) return rc;
        *bytes = c.plan.wsFloats * sizeof(float);
        return FVSRN_OK;
    });
}

int fvsrn_gated_scan(const fvsrn_scan_desc* desc, const void* d_gate, const void* d_x, const float* d_h0, const int* d_lengths, void* d_out, float* d_last,
                     void* d_workspace, size_t workspace_bytes, void* stream) {
    if (!desc) return fail(FVSRN_ERR_INVALID_ARGUMENT, "null pointer");
    return guarded([&]() -> int {
        ScanCall c{"gated_scan", desc};
        if (const int rc = scanShape(c, false)) return rc;
        ScanParams& p = c.p;
        if (p.B == 0 || p.C == 0) return FVSRN_OK;
        if (p.T > 0 && (!d_gate || !d_x)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "null pointer");
        if (p.T == 0 && !d_last) return FVSRN_OK;  // (no states to write; an empty tensor's address may be NULL)
        if (!d_out && !d_last) return fail(FVSRN_ERR_INVALID_ARGUMENT, "neither states nor last states are asked for");
        const size_t e = elementSize(desc->dtype);
        const long long gates[3] = {p.B, p.T, p.Cg}, full[3] = {p.B, p.T, p.C}, ends[2] = {p.B, p.C}, endStride[2] = {p.C, 1}, one[1] = {1};
        if (d_out && overlapsItself(full, p.os, 3)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "out_stride makes elements share an address");
        const size_t need = c.plan.wsFloats * sizeof(float);
        if (need > workspace_bytes || (need && !d_workspace))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "workspace too small: " + std::to_string(need) + " bytes are needed (fvsrn_gated_scan_workspace)");
        const long long wsSize[1] = {(long long)c.plan.wsFloats};
        Range gate, x, h0, len, out, last, ws;
        if (!rangeOf("gate", d_gate, e, 3, gates, p.gs, gate) || !rangeOf("x", d_x, e, 3, full, p.xs, x) || !rangeOf("h0", d_h0, 4, 2, ends, endStride, h0) ||
            !rangeOf("lengths", d_lengths, 4, 1, ends, one, len) || !rangeOf("out", d_out, e, 3, full, p.os, out) ||
            !rangeOf("last", d_last, 4, 2, ends, endStride, last) || !rangeOf("the workspace", need ? d_workspace : nullptr, 4, 1, wsSize, one, ws))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "an operand is not aligned to its elements or reaches beyond the address space");
        std::string clash = overlapping({out, last, ws}, {gate, x, len});
        if (clash.empty()) clash = overlapping({out, ws}, {h0, last});
        if (clash.empty()) clash = overlapping({out}, {ws});
        if (clash.empty() && d_last != d_h0) clash = overlapping({last}, {h0});
        if (!clash.empty()) return fail(FVSRN_ERR_INVALID_ARGUMENT, clash);
        if (const int rc = scanLaunchable(c)) return rc;
        if (fvsrn_device_count() == 0) return noDevice();
        p.gate = d_gate; p.x = d_x; p.h0 = d_h0; p.lengths = d_lengths; p.out = d_out; p.last = d_last;
        p.ws = static_cast<float*>(d_workspace);
        const hipError_t err = launch_gated_scan(p, c.plan, desc->dtype, static_cast<hipStream_t>(stream));
        if (err != hipSuccess) return fail(FVSRN_ERR_DEVICE, std::string("gated_scan failed: ") + hipGetErrorString(err));
        return FVSRN_OK;
    });
}

int fvsrn_gated_scan_backward(const fvsrn_scan_desc* desc, const void* d_gate, const void* d_x, const float* d_h0, const int* d_lengths, const void* d_dout,
                              const float* d_dlast, void* d_dgate, void* d_dx, float* d_dh0, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (!desc) return fail(FVSRN_ERR_INVALID_ARGUMENT, "null pointer");
    return guarded([&]() -> int {
        ScanCall c{"gated_scan_backward", desc};
        if (const int rc = scanShape(c, true)) return rc;
        ScanParams& p = c.p;
        if (p.B == 0 || p.C == 0) return FVSRN_OK;
        if (p.T > 0 && (!d_gate || !d_x)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "null pointer");
        if (p.T == 0 && !d_dh0) return FVSRN_OK;  // (an empty tensor's address may be NULL)
        if (!d_dgate && !d_dx && !d_dh0) return fail(FVSRN_ERR_INVALID_ARGUMENT, "no gradient is asked for");
        const size_t e = elementSize(desc->dtype);
        const long long gates[3] = {p.B, p.T, p.Cg}, full[3] = {p.B, p.T, p.C}, ends[2] = {p.B, p.C}, endStride[2] = {p.C, 1}, one[1] = {1};
        if (d_dgate && overlapsItself(gates, p.dgs, 3)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "dgate_stride makes elements share an address");
        if (d_dx && overlapsItself(full, p.dxs, 3)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "dx_stride makes elements share an address");
        const size_t need = c.plan.wsFloats * sizeof(float);
        if (need > workspace_bytes || (need && !d_workspace))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "workspace too small: " + std::to_string(need) + " bytes are needed (fvsrn_gated_scan_workspace)");
        const long long wsSize[1] = {(long long)c.plan.wsFloats};
        Range gate, x, h0, len, dout, dlast, dgate, dx, dh0, ws;
        if (!rangeOf("gate", d_gate, e, 3, gates, p.gs, gate) || !rangeOf("x", d_x, e, 3, full, p.xs, x) || !rangeOf("h0", d_h0, 4, 2, ends, endStride, h0) ||
            !rangeOf("lengths", d_lengths, 4, 1, ends, one, len) || !rangeOf("dout", d_dout, e, 3, full, p.ds, dout) ||
            !rangeOf("dlast", d_dlast, 4, 2, ends, endStride, dlast) || !rangeOf("dgate", d_dgate, e, 3, gates, p.dgs, dgate) ||
            !rangeOf("dx", d_dx, e, 3, full, p.dxs, dx) || !rangeOf("dh0", d_dh0, 4, 2, ends, endStride, dh0) ||
            !rangeOf("the workspace", need ? d_workspace : nullptr, 4, 1, wsSize, one, ws))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "an operand is not aligned to its elements or reaches beyond the address space");
        std::string clash = overlapping({dgate, dx, dh0, ws}, {gate, x, h0, len, dout, dlast});
        if (clash.empty()) clash = overlapping({dgate, dx, ws}, {dh0});
        if (clash.empty()) clash = overlapping({dgate, dx}, {ws});
        // gradients of colours and absorptions may sit beside each other in one tensor like the inputs
        if (clash.empty() && (dgate && dx) && !besideEachOther(p, d_dgate, d_dx, (long long)e)) clash = "dgate overlaps dx";
        if (!clash.empty()) return fail(FVSRN_ERR_INVALID_ARGUMENT, clash);
        if (const int rc = scanLaunchable(c)) return rc;
        if (fvsrn_device_count() == 0) return noDevice();
        p.gate = d_gate; p.x = d_x; p.h0 = d_h0; p.lengths = d_lengths; p.dout = d_dout; p.dlast = d_dlast;
        p.dgate = d_dgate; p.dx = d_dx; p.dh0 = d_dh0;
        p.ws = static_cast<float*>(d_workspace);
        const hipError_t err = launch_gated_scan_backward(p, c.plan, desc->dtype, static_cast<hipStream_t>(stream));
        if (err != hipSuccess) return fail(FVSRN_ERR_DEVICE, std::string("gated_scan_backward failed: ") + hipGetErrorString(err));
        return FVSRN_OK;
    });
}

int fvsrn_quantize_rows(const void* d_x, int dtype, long long rows, int cols, long long ldx, signed char* d_codes, long long ldc, float* d_scales, void* stream) {
    return guarded([&]() -> int {
        if (!knownDtype(dtype)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "unknown dtype");
        if (rows < 0 || cols <= 0) return fail(FVSRN_ERR_INVALID_ARGUMENT, "bad matrix size");
        if (rows == 0) return FVSRN_OK;
        if (!d_x || !d_codes || !d_scales) return fail(FVSRN_ERR_INVALID_ARGUMENT, "null pointer");
        if ((ldx < cols && !(ldx == 0 || rows == 1)) || (ldc < cols && rows > 1)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "a row stride is smaller than a row");
        if (cols > (1 << 30)) return fail(FVSRN_ERR_UNSUPPORTED, "more than 2^30 columns");
        if (__int128(rows) * quantizeWidth(cols) > kMaxThreads) return fail(FVSRN_ERR_UNSUPPORTED, "too many rows for one launch, split the matrix");
        const long long size[2] = {rows, cols}, sx[2] = {ldx, 1}, sc[2] = {ldc, 1}, one[1] = {1};
        Range x, codes, scales;
        if (!rangeOf("x", d_x, elementSize(dtype), 2, size, sx, x) || !rangeOf("the codes", d_codes, 1, 2, size, sc, codes) || !rangeOf("the scales", d_scales, 4, 1, size, one, scales))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "an operand is not aligned to its elements or reaches beyond the address space");
        std::string clash = overlapping({codes, scales}, {x});
        if (clash.empty()) clash = overlapping({codes}, {scales});
        if (!clash.empty()) return fail(FVSRN_ERR_INVALID_ARGUMENT, clash);
        if (fvsrn_device_count() == 0) return noDevice();
        QuantizeParams p{d_x, d_codes, d_scales, rows, ldx, ldc, cols};
        const hipError_t err = launch_quantize_rows(p, dtype, static_cast<hipStream_t>(stream));
        if (err != hipSuccess) return fail(FVSRN_ERR_DEVICE, std::string("quantize_rows failed: ") + hipGetErrorString(err));
        return FVSRN_OK;
    });
}

int fvsrn_matmul_int8(const signed char* d_a, long long lda, const float* d_scale_a, const signed char* d_b, long long ldb, const float* d_scale_b,
                      const float* d_bias, long long M, int N, int K, int activation, float act_param, void* d_out, int out_dtype, long long ldo, void* stream) {
    return guarded([&]() -> int {
        if (!knownDtype(out_dtype)) return fail(FVSRN_ERR_INVALID_ARGUMENT, "unknown dtype");
        if (activation < FVSRN_ACT_RELU || activation > FVSRN_ACT_NONE) return fail(FVSRN_ERR_INVALID_ARGUMENT, "unknown activation");
        if ((activation == FVSRN_ACT_SINE || activation == FVSRN_ACT_SNAKE || activation == FVSRN_ACT_SNAKEALT) && (!std::isfinite(act_param) || act_param == 0))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "the activation's parameter must be finite and not 0");
        if (M < 0 || N < 0 || K <= 0) return fail(FVSRN_ERR_INVALID_ARGUMENT, "bad matrix size");
        if (K > 131071) return fail(FVSRN_ERR_UNSUPPORTED, "K is over 131071: the sums of products of codes would not fit 32 bits");
        if (M == 0 || N == 0) return FVSRN_OK;
        if (!d_a || !d_b || !d_scale_a || !d_scale_b || !d_out) return fail(FVSRN_ERR_INVALID_ARGUMENT, "null pointer");
        if ((lda < K && !(lda == 0 || M == 1)) || (ldb < K && !(ldb == 0 || N == 1)) || (ldo < N && M > 1))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "a row stride is smaller than a row");
        if (N > (1 << 26)) return fail(FVSRN_ERR_UNSUPPORTED, "too many channels for one launch, split the weights");
        const auto tiles = [&](int edge) { return __int128((M + edge - 1) / edge) * ((N + edge - 1) / edge); };
        if (M > (1LL << 31) || (M > 64 && N > 16 && (tiles(128) * 256 > kMaxThreads || tiles(256) * 512 > kMaxThreads))) return fail(FVSRN_ERR_UNSUPPORTED, "too many rows for one launch, split the matrix");
        const long long as[2] = {M, K}, bs[2] = {N, K}, os[2] = {M, N}, sa[2] = {lda, 1}, sb[2] = {ldb, 1}, so[2] = {ldo, 1}, one[1] = {1};
        Range a, b, out, scaleA, scaleB, bias;
        if (!rangeOf("a", d_a, 1, 2, as, sa, a) || !rangeOf("b", d_b, 1, 2, bs, sb, b) || !rangeOf("out", d_out, elementSize(out_dtype), 2, os, so, out) ||
            !rangeOf("scale_a", d_scale_a, 4, 1, as, one, scaleA) || !rangeOf("scale_b", d_scale_b, 4, 1, bs, one, scaleB) || !rangeOf("bias", d_bias, 4, 1, bs, one, bias))
            return fail(FVSRN_ERR_INVALID_ARGUMENT, "an operand is not aligned to its elements or reaches beyond the address space");
        const std::string clash = overlapping({out}, {a, b, scaleA, scaleB, bias});
        if (!clash.empty()) return fail(FVSRN_ERR_INVALID_ARGUMENT, clash);
        if (fvsrn_device_count() == 0) return noDevice();
        Int8Params p{d_a, d_b, d_scale_a, d_scale_b, d_bias, d_out, lda, ldb, ldo, M, N, K, act_param};
        const hipError_t err = launch_matmul_int8(p, activation, out_dtype, static_cast<hipStream_t>(stream));
        if (err != hipSuccess) return fail(FVSRN_ERR_DEVICE, std::string("matmul_int8 failed: ") + hipGetErrorString(err));
        return FVSRN_OK;
    });
}

}  // extern "C"
