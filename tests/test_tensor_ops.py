"""
The tensor operators of a ray march: gated_scan and its gradients, quantize_rows, matmul_int8 (include/fvsrn.h) against plain statements in 64 bits.

Tolerances.  eps = 2^-24 is half a step of a 32-bit float.  A recurrence step in 32 bits adds at most STEP + |scale gate| half steps of what it
multiplies: the gate (the rounding of scale * gate shifts its logarithm by |scale gate| eps; exp - 1 itself two), the input factor 1 - a (two),
the product and the sum (two), and the joins of spans, which form the same products in another order (two more).  `bounds` carries these
errors through the recurrence in 64 bits, with absolute values: what is left at a step is the bound there.  An output of 16 bits is rounded once, by half a
step of its type.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import util  # noqa: F401
from fvsrn_amd import capi

EPS = 2.0 ** -24
STEP = 10.0
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -140, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # (half a step of the smallest values)
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------------------------------------------------
# the recurrence in 64 bits, with what 32-bit steps may add
# ---------------------------------------------------------------------------------------------------------------------

def plain_scan(gate, x, dout=None, dlast=None, *, gate_mode, gate_scale, input_mode, reverse, h0=None, lengths=None):
    """{name: (value, bound)} of the states, the last states and the gradients: one step after the other, numpy float64."""
    g, x = gate.detach().double().cpu().numpy(), x.detach().double().cpu().numpy()
    B, T, Ch = x.shape
    G = Ch // g.shape[2]
    n = np.full(B, T) if lengths is None else np.clip(lengths.cpu().numpy(), 0, T)
    h = np.zeros((B, Ch)) if h0 is None else h0.double().cpu().numpy().copy()
    e = np.zeros((B, Ch))
    out, out_e = np.zeros((B, T, Ch)), np.zeros((B, T, Ch))
    before, before_e = np.zeros((B, T, Ch)), np.zeros((B, T, Ch))
    rows = np.arange(B)

    def factors(t):
        y = np.repeat(g[rows, t], G, 1)
        if gate_mode == capi.GATE_EXP:
            y = gate_scale * y
            return np.exp(y), -np.expm1(y), (STEP + np.abs(y)) * EPS
        return y, 1.0 - y, np.full_like(y, STEP * EPS)

    steps = []
    for i in range(T):
        live = (i < n)[:, None]
        t = np.where(i < n, n - 1 - i if reverse else i, 0)
        steps.append((t, live))
        a, rest, c = factors(t)
        xt = x[rows, t]
        u = rest * xt if input_mode == capi.INPUT_BLEND else xt
        new = a * h + u
        new_e = np.abs(a) * (e + c * np.abs(h)) + c * np.abs(u) + EPS * np.abs(new)
        keep = live[:, 0]
        before[rows[keep], t[keep]], before_e[rows[keep], t[keep]] = h[keep], e[keep]
        h, e = np.where(live, new, h), np.where(live, new_e, e)
        out[rows[keep], t[keep]], out_e[rows[keep], t[keep]] = h[keep], e[keep]
    result = {"out": (out, out_e), "last": (h, e)}
    if dout is None and dlast is None:
        return result
    d = np.zeros_like(x) if dout is None else dout.double().cpu().numpy()
    k = np.zeros((B, Ch)) if dlast is None else dlast.double().cpu().numpy().copy()
    ke = np.zeros((B, Ch))
    dx, dx_e, da, da_e = (np.zeros_like(x) for _ in range(4))
    for t, live in reversed(steps):
        a, rest, c = factors(t)
        keep = live[:, 0]
        lam = d[rows, t] + k
        lam_e = ke + c * (np.abs(d[rows, t]) + np.abs(k))
        gain = rest if input_mode == capi.INPUT_BLEND else np.ones_like(rest)
        dx[rows[keep], t[keep]], dx_e[rows[keep], t[keep]] = (gain * lam)[keep], (np.abs(gain) * (lam_e + c * np.abs(lam)))[keep]
        xt = x[rows, t] if input_mode == capi.INPUT_BLEND else 0.0
        w, w_e = before[rows, t] - xt, before_e[rows, t] + EPS * (np.abs(before[rows, t]) + np.abs(xt))
        factor = gate_scale * a if gate_mode == capi.GATE_EXP else 1.0
        da[rows[keep], t[keep]] = (factor * lam * w)[keep]
        da_e[rows[keep], t[keep]] = (np.abs(factor) * (np.abs(lam) * (w_e + c * np.abs(w)) + lam_e * np.abs(w)))[keep]
        k, ke = np.where(live, a * lam, k), np.where(live, np.abs(a) * (lam_e + c * np.abs(lam)), ke)
    da, da_abs, da_e = (v.reshape(B, T, -1, G).sum(3) for v in (da, np.abs(da), da_e))
    result |= {"dgate": (da, da_e + (G + 2) * EPS * da_abs), "dx": (dx, dx_e), "dh0": (k, ke)}
    return result


def assert_within(got, want, name):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    v = got.detach().double().cpu().numpy()
    assert np.isfinite(v).all(), name
    tolerance = bound + HALF_STEP[got.dtype] * (np.abs(value) + bound) + TINY[got.dtype]
    off = np.abs(v - value) - tolerance
    if off.size:
        at = np.unravel_index(np.argmax(off), off.shape)
        assert off[at] <= 0, "%s at %s: %g, not %g (tolerance %g)" % (name, at, v[at], value[at], tolerance[at])


def scan_inputs(B, T, Ch, Cg, dtype, gate_mode, seed, *, h0=True, lengths=False, device="cuda"):
    r = np.random.RandomState(seed)
    gate = r.exponential(3.0, (B, T, Cg)) * (r.rand(B, T, Cg) < 0.7) if gate_mode == capi.GATE_EXP else 1.0 - 0.3 * r.rand(B, T, Cg)
    t = lambda a, ty: torch.from_numpy(np.ascontiguousarray(a)).to(ty).to(device)  # noqa: E731
    n = None
    if lengths:
        n = r.randint(0, T + 1, B)
        n[0] = 0
        if B > 1:
            n[1] = T + 5  # (clamped to T)
        n = t(n, torch.int32)
    return dict(gate=t(gate, dtype), x=t(r.randn(B, T, Ch), dtype), h0=t(r.randn(B, Ch), F32) if h0 else None, lengths=n,
                dout=t(r.randn(B, T, Ch), dtype), dlast=t(r.randn(B, Ch), F32))


def check_scan(case, how, *, states=True, dout=True, dlast=True, names=("out", "last", "dgate", "dx", "dh0")):
    how = dict(how, h0=case["h0"], lengths=case["lengths"])
    d, dl = case["dout"] if dout else None, case["dlast"] if dlast else None
    want = plain_scan(case["gate"], case["x"], d, dl, **how)
    out, last = capi.gated_scan(case["gate"], case["x"], states=states, **how)
    dgate, dx, dh0 = capi.gated_scan_backward(case["gate"], case["x"], d, dl, **how)
    got = dict(out=out, last=last, dgate=dgate, dx=dx, dh0=dh0)
    assert (out is None) == (not states)
    for name in names:
        if got[name] is not None:
            assert_within(got[name], want[name], name)
    return got


def modes(i):
    """The i-th of the eight combinations of gate, input and direction."""
    return dict(gate_mode=capi.GATE_EXP if i & 1 else capi.GATE_VALUE, input_mode=capi.INPUT_BLEND if i & 2 else capi.INPUT_ADD, reverse=bool(i & 4),
                gate_scale=-0.05 if i & 1 else 1.0)


# (batch, steps, channels, gate channels): one step; colours along rays within and beyond a wave's tile; channels of one wave, of a part of it, of many;
# tiles shared by waves, cut into spans; gates of 2, 8, 100 and 130 channels
SHAPES = [(1, 1, 1, 1), (3, 1, 12, 4), (1, 1, 300, 100), (2, 2, 5, 5), (5, 37, 3, 1), (2, 512, 3, 1), (3, 513, 4, 1), (2, 2049, 2, 1), (300, 9, 1, 1), (1, 1000, 4, 2),
          (2, 16, 64, 64), (2, 33, 40, 40), (2, 130, 65, 65), (1, 300, 100, 100), (1, 3000, 70, 70), (2, 1500, 96, 12), (3, 257, 200, 2), (1, 600, 130, 1), (2, 100, 66, 33),
          (1, 5000, 1, 1), (1, 20, 270000, 270000), (1, 40, 90000, 30000), (1, 129, 5, 1), (300, 4500, 1, 1),
          (3, 9000, 4, 4), (1, 20000, 2, 1), (1, 700, 128, 128), (2, 700, 512, 512), (1, 300, 300, 150)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_scan_and_gradients_against_64_bits(shape, dtype):
    k = SHAPES.index(shape) * 3 + [F32, F16, BF16].index(dtype)
    for i in ((k, k + 3) if shape[0] * shape[1] * shape[2] > 100000 else (k, k + 3, k + 5)):
        how = modes(i % 8)
        case = scan_inputs(*shape, dtype, how["gate_mode"], 100 + k, h0=bool(i % 3), lengths=i % 2 == 0)
        check_scan(case, how, states=i % 4 != 1)


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(8))
def test_scan_every_mode_in_both_lane_layouts(i):
    how = modes(i)
    for shape in ((4, 70, 3, 1), (2, 70, 64, 64), (2, 300, 80, 20)):
        case = scan_inputs(*shape, F32, how["gate_mode"], 7 + i, lengths=True)
        check_scan(case, how)
        check_scan(case, how, states=False, dout=False)
        check_scan(case, how, dlast=False)


@pytest.mark.gpu
def test_scan_strides_views_and_broadcasts():
    how = modes(7)
    r = torch.Generator().manual_seed(3)
    # colours and absorption of a sample beside each other, gradients too
    for B, T, Ch in ((9, 50, 3), (4, 600, 2)):
        both = torch.rand(B, T, Ch + 1, generator=r).cuda()
        grads = torch.full((B, T, Ch + 1), 7.0, device="cuda")
        case = dict(gate=both[..., Ch:], x=both[..., :Ch], dlast=torch.randn(B, Ch, generator=r).cuda())
        want = plain_scan(case["gate"], case["x"], None, case["dlast"], **how)
        capi.gated_scan_backward(case["gate"], case["x"], None, case["dlast"], dgate=grads[..., Ch:], dx=grads[..., :Ch], **how)
        assert_within(grads[..., Ch:], want["dgate"], "dgate")
        assert_within(grads[..., :Ch], want["dx"], "dx")
    # steps innermost, every second element, a batch of strided planes; the last two with outputs laid out like that too
    for x, gate in ((torch.randn(3, 40, 90, generator=r).cuda().transpose(1, 2), torch.rand(3, 40, 90, generator=r).cuda().transpose(1, 2)),
                    (torch.randn(2, 33, 160, generator=r).cuda()[:, :, ::2], torch.rand(2, 33, 80, generator=r).cuda()),
                    (torch.randn(50, 4, 100, generator=r).cuda().transpose(0, 1), torch.rand(50, 4, 100, generator=r).cuda().transpose(0, 1))):
        dout = torch.randn(x.shape, generator=r).cuda()
        want = plain_scan(gate, x, dout, None, **how)
        out, last = capi.gated_scan(gate, x, out=torch.empty_strided(x.shape, x.stride(), device="cuda"), **how)
        dgate, dx, _ = capi.gated_scan_backward(gate, x, dout, dx=torch.empty_strided(x.shape, x.stride(), device="cuda"), **how)
        for name, got in (("out", out), ("last", last), ("dgate", dgate), ("dx", dx)):
            assert_within(got, want[name], name)
    # gates shared by the batch, one input for every step: their gradients come per element
    gate = torch.rand(1, 70, 1, generator=r).cuda().expand(5, 70, 96)
    x = torch.randn(5, 1, 96, generator=r).cuda().expand(5, 70, 96)
    dout = torch.randn(5, 70, 96, generator=r).cuda()
    want = plain_scan(gate, x, dout, None, **how)
    dgate, dx, _ = capi.gated_scan_backward(gate, x, dout, dgate=torch.empty(5, 70, 96, device="cuda"), dx=torch.empty(5, 70, 96, device="cuda"), **how)
    assert_within(dgate, want["dgate"], "dgate")
    assert_within(dx, want["dx"], "dx")
    # addresses that are odd multiples of the element
    base = torch.randn(2 * 60 * 128 + 1, generator=r).to(F16).cuda()
    x = base[1:].view(2, 60, 128)
    gate = torch.rand(2 * 60 * 128 + 1, generator=r).to(F16).cuda()[1:].view(2, 60, 128)
    out, last = capi.gated_scan(gate, x, **how)
    want = plain_scan(gate, x, **how)
    assert_within(out, want["out"], "out")
    assert_within(last, want["last"], "last")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 70, 3, 1), (3, 300, 64, 64), (2, 2000, 70, 70), (3, 200, 16, 2)], ids=lambda s: "x".join(map(str, s)))
def test_scan_never_reads_behind_a_sequence(shape):
    """Infinities, NaN and the type's lowest value behind the lengths change nothing, and outputs are zero there."""
    for i in (3, 7):
        how = modes(i)
        case = scan_inputs(*shape, F32, how["gate_mode"], 5, lengths=True)
        clean = check_scan(case, how)
        n = case["lengths"].clamp(max=shape[1]).tolist()
        for name in ("gate", "x", "dout"):
            for b, m in enumerate(n):
                bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(F32).min], device="cuda")
                v = case[name][b, m:]
                v.copy_(bad[torch.arange(v.numel(), device="cuda") % 4].view(v.shape))
        kw = dict(how, h0=case["h0"], lengths=case["lengths"])
        out, last = capi.gated_scan(case["gate"], case["x"], **kw)
        dgate, dx, dh0 = capi.gated_scan_backward(case["gate"], case["x"], case["dout"], case["dlast"], **kw)
        for name, got in dict(out=out, last=last, dgate=dgate, dx=dx, dh0=dh0).items():
            assert torch.equal(got, clean[name]), name
        for b, m in enumerate(n):
            for t in (out, dgate, dx):
                assert not t[b, m:].any()
        assert torch.equal(last[0], case["h0"][0]) and torch.equal(dh0[0], case["dlast"][0])  # (the empty sequence passes both through)


@pytest.mark.gpu
def test_scan_of_no_steps_and_of_nothing():
    h0 = torch.randn(3, 8, device="cuda")
    gate, x = torch.empty(3, 0, 8, device="cuda"), torch.empty(3, 0, 8, device="cuda")
    out, last = capi.gated_scan(gate, x, h0=h0)
    assert out.shape == (3, 0, 8) and torch.equal(last, h0)
    assert not capi.gated_scan(gate, x)[1].any()
    d = torch.randn(3, 8, device="cuda")
    assert torch.equal(capi.gated_scan_backward(gate, x, None, d, h0=h0)[2], d)
    none = torch.empty(0, 5, 8, device="cuda")
    assert capi.gated_scan(none, none)[1].shape == (0, 8)


@pytest.mark.gpu
def test_scan_non_finite_values_stay_in_their_sequence_and_behind_their_step():
    for shape in ((3, 90, 3, 1), (3, 90, 64, 64), (3, 3000, 64, 64)):
        gate = torch.rand(shape[0], shape[1], shape[3], device="cuda") * 0.5 + 0.25
        x = torch.randn(shape[:3], device="cuda")
        clean = capi.gated_scan(gate, x)[0]
        x[1, 40, 1] = math.nan
        out = capi.gated_scan(gate, x)[0]
        assert out[1, 40:, 1].isnan().all()
        out[1, 40:, 1] = clean[1, 40:, 1]
        assert torch.equal(out, clean)
        # a gate of zero forgets everything before it
        x[1, 40, 1] = 0.0
        gate[:, 50] = 0.0
        assert torch.equal(capi.gated_scan(gate, x)[0][:, 50], x[:, 50])


@pytest.mark.gpu
def test_scan_thin_media_keep_their_precision():
    """1 - exp(-y) of samples with y = 1e-6: 32 bits of 1 - a, not of 1."""
    gate = torch.full((5, 300, 1), 1e-3, device="cuda")
    x = torch.rand(5, 300, 3, device="cuda")
    how = dict(gate_mode=capi.GATE_EXP, gate_scale=-1e-3, input_mode=capi.INPUT_BLEND, reverse=True)
    _, last = capi.gated_scan(gate, x, states=False, **how)
    want = plain_scan(gate, x, **how)["last"][0]
    assert np.abs(last.double().cpu().numpy() / want - 1).max() < 300 * 4 * EPS
    # and a dense one ends at the first sample it meets, with nothing lost on the way there
    gate = torch.tensor([0.0, 1e30, math.inf], device="cuda").view(1, 3, 1)
    out, _ = capi.gated_scan(gate, torch.ones(1, 3, 3, device="cuda"), gate_mode=capi.GATE_EXP, gate_scale=-1.0, input_mode=capi.INPUT_BLEND)
    assert out[0, :, 0].tolist() == [0.0, 1.0, 1.0]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 20, 3, 1), (1, 40, 64, 64), (2, 24, 16, 2)], ids=lambda s: "x".join(map(str, s)))
def test_scan_gradients_against_differences(shape):
    """d(sum of dout out + dlast last) along a random direction, by a central difference of the 64-bit statement."""
    how = modes(3)
    case = scan_inputs(*shape, F32, how["gate_mode"], 11)
    grads = dict(zip(("gate", "x", "h0"), capi.gated_scan_backward(case["gate"], case["x"], case["dout"], case["dlast"], h0=case["h0"], **how)))
    d, dl = case["dout"].double().cpu().numpy(), case["dlast"].double().cpu().numpy()

    def value(**moved):
        c = {k: (moved.get(k, case[k])) for k in ("gate", "x", "h0")}
        r = plain_scan(c["gate"], c["x"], h0=c["h0"], **how)
        return (d * r["out"][0]).sum() + (dl * r["last"][0]).sum()

    step = 1e-5
    for name in ("gate", "x", "h0"):
        v = torch.randn(case[name].shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64).cuda()
        slope = (value(**{name: case[name].double() + step * v}) - value(**{name: case[name].double() - step * v})) / (2 * step)
        got = float((grads[name].double() * v).sum())
        size = float((grads[name].double().abs() * v.abs()).sum())
        assert abs(got - slope) <= 1e-5 * size, name  # (the difference's own error: step^2 and 2^-53 / step of the value)


@pytest.mark.gpu
def test_scan_in_place_steps_equal_the_whole():
    """A march of single steps, the state in place, on a stream of its own -- and the same as one call."""
    T, R = 17, 500
    gate, x = torch.rand(1, T, R, device="cuda") * 20, torch.rand(1, T, 3 * R, device="cuda")
    how = dict(gate_mode=capi.GATE_EXP, gate_scale=-0.01, input_mode=capi.INPUT_BLEND)
    whole = capi.gated_scan(gate, x, states=False, **how)[1]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        h = torch.zeros(1, 3 * R, device="cuda")
        for t in range(T):
            assert capi.gated_scan(gate[:, t:t + 1], x[:, t:t + 1], states=False, h0=h, last=h, **how)[1] is h
    torch.cuda.current_stream().wait_stream(stream)
    assert (h - whole).abs().max() <= 2 * T * STEP * EPS * whole.abs().max()
    # long sequences cut into spans: the state in place too
    gate, x, h0 = torch.rand(1, 4000, 64, device="cuda"), torch.randn(1, 4000, 64, device="cuda"), torch.randn(1, 64, device="cuda")
    want = capi.gated_scan(gate, x, h0=h0)
    h = h0.clone()
    out, _ = capi.gated_scan(gate, x, h0=h, last=h)
    assert torch.equal(out, want[0]) and torch.equal(h, want[1])
    # raw stream handles: the call runs there
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = capi.gated_scan(gate, x, h0=h0, stream=other.cuda_stream)
    other.synchronize()
    assert torch.equal(got[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 300, 3, 1), (2, 3000, 64, 64), (2, 200, 260, 2)], ids=lambda s: "x".join(map(str, s)))
def test_scan_captured_and_replayed(shape):
    """Two graphs that hold the same calls, replayed in turn with new inputs between, equal the eager calls bit for bit (sums have a fixed order)."""
    how = modes(3)
    cases = [scan_inputs(*shape, F32, how["gate_mode"], s) for s in (1, 2, 3, 4)]
    inputs = [{k: v.clone() for k, v in cases[0].items() if v is not None} for _ in range(2)]

    def both(c):
        out, last = capi.gated_scan(c["gate"], c["x"], h0=c["h0"], **how)
        return (out, last) + capi.gated_scan_backward(c["gate"], c["x"], c["dout"], c["dlast"], h0=c["h0"], **how)

    for c in inputs:
        both(c)
    torch.cuda.synchronize()
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g, c in zip(graphs, inputs):
        with torch.cuda.graph(g):
            results.append(both(c))
    for turn in range(4):
        for g, c, r, new in zip(graphs, inputs, results, (cases[turn], cases[(turn + 1) % 4])):
            for k in c:
                c[k].copy_(new[k])
            g.replay()
            if turn % 2:
                torch.cuda.synchronize()
            for got, want in zip(r, both(new)):
                assert torch.equal(got, want)


# ---------------------------------------------------------------------------------------------------------------------
# codes and scales
# ---------------------------------------------------------------------------------------------------------------------

def plain_codes(x):
    """The definition, in numpy float32 (its divisions are rounded to 32 bits there too)."""
    v = x.float().cpu().numpy()
    bad = ~np.isfinite(v).all(1)
    scale = np.maximum(np.abs(np.where(np.isfinite(v), v, 0)).max(1) * (np.float32(1) / np.float32(127)), np.float32(2.0 ** -126))
    q = np.where(bad[:, None], 0, np.rint(np.where(bad[:, None], 0, v) / scale[:, None]))
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def assert_codes(x, codes, scales):
    q, s = plain_codes(x)
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
    assert np.array_equal(codes.cpu().numpy(), q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 7), (3, 8), (700, 9), (33, 63), (2, 64), (129, 250), (64, 256), (3, 511), (7, 513), (9, 2049), (5, 4096), (2, 5003), (1, 20000), (20003, 250), (70001, 40)])
def test_codes_and_scales(rows, cols, dtype):
    x = (torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows * cols)) * 3).to(dtype).cuda()
    assert_codes(x, *capi.quantize_rows(x))
    wide = torch.randn(rows, cols + 5, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    codes = torch.full((rows, cols + 3), 99, dtype=torch.int8, device="cuda")
    capi.quantize_rows(wide[:, 2:cols + 2], codes=codes[:, 1:cols + 1])
    assert_codes(wide[:, 2:cols + 2], codes[:, 1:cols + 1], capi.quantize_rows(wide[:, 2:cols + 2])[1])
    assert (codes[:, 0] == 99).all() and (codes[:, cols + 1:] == 99).all()  # (what is beside the codes stays as it was)


@pytest.mark.gpu
def test_codes_of_special_rows():
    x = torch.randn(12, 40, generator=torch.Generator().manual_seed(2))
    x[0] = 0.0
    x[1] = 1e-44
    x[2] = torch.finfo(F32).max
    x[3, 5] = math.nan
    x[4, 39] = -math.inf
    x[5, 0] = math.inf
    x[6] = torch.arange(40) + 0.5  # ties once scaled
    x[6, 0] = 127.0
    x[7] = 2.0 ** -126
    x[8] = -0.0
    x[9, 1:] = 0.0
    x = x.cuda()
    codes, scales = capi.quantize_rows(x)
    assert_codes(x, codes, scales)
    assert scales[3:6].isnan().all() and not codes[3:6].any() and not codes[0].any() and float(scales[0]) == 2.0 ** -126
    # every product with a row that was no number is none, whatever the activation
    w, sw = capi.quantize_rows(torch.randn(6, 40, device="cuda"))
    for activation in capi.ACTIVATIONS:
        y = capi.matmul_int8(codes, scales, w, sw, torch.ones(6, device="cuda"), activation)
        assert y[3:6].isnan().all() and y[:2].isfinite().all() and y[6:].isfinite().all(), activation
    # row 2 is 40 times the largest number: its products are that times the sum of a channel's codes and scale, beyond 32 bits where that is over 1, and nowhere else
    y = capi.matmul_int8(codes, scales, w, sw, torch.ones(6, device="cuda"))
    z = (codes[2].double() * w.double()).sum(1) * scales[2].double() * sw.double()
    assert torch.equal(y[2].isinf(), z.abs() > torch.finfo(F32).max) and torch.equal(y[2][y[2].isfinite()].sign(), z[y[2].isfinite()].sign())
    assert capi.quantize_rows(torch.empty(0, 4, device="cuda"))[0].shape == (0, 4)
    one = torch.randn(1, 40, device="cuda")
    assert_codes(one.expand(3, 40), *capi.quantize_rows(one.expand(3, 40)))


# ---------------------------------------------------------------------------------------------------------------------
# product
# ---------------------------------------------------------------------------------------------------------------------

def plain_product(a, sa, b, sb, bias, activation, param, dtype):
    """(values, bound).  acc -> acc sb -> fma with sa and the bias: three roundings of 32 bits; behind them the activation's slope (at most 2 for the snakes: 1 +
    sin; their 1 / p terms have a slope bounded by it) times that error, the argument's rounding in sine and cosine and four half steps of the terms it sums."""
    acc = a.long().cpu().numpy().astype(np.float64) @ b.long().cpu().numpy().astype(np.float64).T
    z = acc * sa.double().cpu().numpy()[:, None] * sb.double().cpu().numpy()
    err = 3 * EPS * np.abs(z)
    if bias is not None:
        z = z + bias.double().cpu().numpy()
        err = err + EPS * np.abs(z)
    p = param
    if activation == "ReLU":
        y = np.maximum(z, 0)
    elif activation == "Sine":
        y, err = np.sin(p * z), abs(p) * (err + EPS * np.abs(z)) + 4 * EPS
    elif activation == "Snake":
        y, err = z + np.sin(p * z) ** 2 / p, 2 * (err + EPS * np.abs(z)) + 4 * EPS * (np.abs(z) + 2 / abs(p))
    elif activation == "SnakeAlt":
        y, err = (z + 1 - np.cos(2 * p * z)) / (2 * p), (1 + 1 / abs(2 * p)) * (err + EPS * np.abs(z)) + 4 * EPS * (np.abs(z) + 3) / abs(2 * p)
    elif activation == "Sigmoid":
        y = 1 / (1 + np.exp(-z))
        err = y * (1 - y) * (err + 2 * EPS) * 2 + 4 * EPS * y
    else:
        y = z
    return y, err + HALF_STEP[dtype] * np.abs(y) + TINY[dtype]


PRODUCTS = [(1, 1, 1), (1, 17, 5), (3, 64, 64), (65, 63, 130), (130, 257, 100), (64, 64, 16), (257, 129, 1000), (1, 100, 4096), (16, 300, 777), (17, 48, 1024), (33, 33, 33),
            (128, 256, 128), (300, 300, 320), (1000, 4, 250), (513, 520, 512), (5, 1, 131071), (600, 1, 64), (1, 3001, 70), (260, 256, 256), (2048, 192, 96),
            (300, 40, 7), (100, 16, 15), (300, 300, 1), (70, 100, 31), (300, 20, 17), (5000, 16, 250), (40, 20000, 33), (20, 20000, 64), (300, 70, 48), (3000, 2900, 80),
            (4200, 4100, 1040), (4200, 4100, 1031)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product_is_exact_in_integers(M, N, K):
    """Every code from -128 to 127; sums below 2^24 come out as they are, larger ones rounded once."""
    g = torch.Generator().manual_seed(M + N + K)
    a, b = (torch.randint(-128, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((M, K), (N, K)))
    one_m, one_n = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    want = (a.cpu().long().numpy().astype(np.float64) @ b.cpu().long().numpy().astype(np.float64).T).astype(np.float32)
    assert np.array_equal(capi.matmul_int8(a, one_m, b, one_n).cpu().numpy(), want)
    a.fill_(-128), b.fill_(-128)  # the largest sum there is
    assert (capi.matmul_int8(a, one_m, b, one_n) == float(np.float32(16384 * K))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("activation,param", [("None", 1.0), ("ReLU", 1.0), ("Sine", 3.0), ("Snake", 0.7), ("SnakeAlt", 1.5), ("Sigmoid", 1.0)])
@pytest.mark.parametrize("M,N,K", [(1, 40, 256), (20, 33, 100), (300, 260, 256), (70, 4, 250)])
def test_product_scales_bias_activation(M, N, K, activation, param, dtype):
    g = torch.Generator().manual_seed(M)
    a, sa = capi.quantize_rows(torch.randn(M, K, generator=g).cuda())
    b, sb = capi.quantize_rows((torch.randn(N, K, generator=g) / math.sqrt(K)).cuda())
    for bias in (None, torch.randn(N, generator=g).cuda()):
        y, bound = plain_product(a, sa, b, sb, bias, activation, param, dtype)
        got = capi.matmul_int8(a, sa, b, sb, bias, activation, param, dtype=dtype).double().cpu().numpy()
        off = np.abs(got - y) - bound
        assert off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.gpu
def test_product_strides_and_neighbours():
    g = torch.Generator().manual_seed(4)
    for M, N, K, pad in ((40, 70, 100, 3), (300, 130, 128, 16), (2, 50, 64, 1), (200, 200, 256, 5)):
        wide_a, wide_b = (torch.randint(-128, 128, (r, K + pad), generator=g, dtype=torch.int8).cuda() for r in (M, N))
        a, b = wide_a[:, pad:], wide_b[:, :K]
        out = torch.full((M + 1, N + 7), 5.0, device="cuda")
        one = torch.ones(max(M, N), device="cuda")
        capi.matmul_int8(a, one[:M], b, one[:N], out=out[:M, 3:N + 3])
        want = (a.cpu().long() @ b.cpu().long().t()).float()
        assert torch.equal(out[:M, 3:N + 3].cpu(), want)
        assert (out[:, :3] == 5).all() and (out[:, N + 3:] == 5).all() and (out[M] == 5).all()
        one_row = a[:1].expand(M, K)
        assert torch.equal(capi.matmul_int8(one_row, one[:M], b, one[:N]).cpu(), want[:1].expand(M, N))
    e = torch.empty(0, 64, dtype=torch.int8, device="cuda")
    assert capi.matmul_int8(e, torch.empty(0, device="cuda"), b[:, :64], one[:b.shape[0]]).shape == (0, b.shape[0])


@pytest.mark.gpu
def test_operands_beyond_32_bits_of_offset():
    """Rows and sequences more than 2^31 elements apart, and more than 2^32 bytes."""
    far = 2 ** 31 + 2 ** 20
    g = torch.Generator().manual_seed(8)
    a = torch.empty(2 * far + 64, dtype=torch.int8, device="cuda").as_strided((3, 64), (far, 1))
    a.copy_(torch.randint(-128, 128, (3, 64), generator=g, dtype=torch.int8))
    b = torch.randint(-128, 128, (100, 64), generator=g, dtype=torch.int8).cuda()
    one = torch.ones(100, device="cuda")
    out = torch.empty(2 * far + 100, dtype=F16, device="cuda").as_strided((3, 100), (far, 1))
    want = (a.cpu().long() @ b.cpu().long().t()).float()
    assert torch.equal(capi.matmul_int8(a, one[:3], b, one).cpu(), want)
    capi.matmul_int8(a, one[:3] / 1024, b, one, out=out)
    assert torch.equal(out.cpu(), (want / 1024).to(F16))
    many = a[:1].expand(300, 64)
    assert torch.equal(capi.matmul_int8(a[2:].expand(300, 64), one[:1].expand(300).contiguous(), b, one).cpu(), want[2:].expand(300, 100)) and many.stride(0) == 0
    x = torch.empty(2 * far + 5000, dtype=F16, device="cuda").as_strided((3, 64), (far, 1))
    x.copy_(torch.randn(3, 64, generator=g))
    assert_codes(x, *capi.quantize_rows(x, codes=torch.empty(2 * far + 64, dtype=torch.int8, device="cuda").as_strided((3, 64), (far, 1))))
    how = modes(7)
    for shape in ((2, 6, 3, 1), (2, 300, 64, 64)):
        B, T, Ch, Cg = shape
        x = torch.empty(far + T * Ch, dtype=F16, device="cuda").as_strided((B, T, Ch), (far, Ch, 1))
        x.copy_(torch.randn(B, T, Ch, generator=g))
        gate, d = torch.rand(B, T, Cg, generator=g).to(F16).cuda(), torch.randn(B, T, Ch, generator=g).to(F16).cuda()
        want = plain_scan(gate, x, d, None, **how)
        out, last = capi.gated_scan(gate, x, out=torch.empty(far + T * Ch, dtype=F16, device="cuda").as_strided((B, T, Ch), (far, Ch, 1)), **how)
        dgate, dx, _ = capi.gated_scan_backward(gate, x, d, dx=torch.empty(far + T * Ch, dtype=F16, device="cuda").as_strided((B, T, Ch), (far, Ch, 1)), **how)
        for name, got in (("out", out), ("last", last), ("dgate", dgate), ("dx", dx)):
            assert_within(got, want[name], name)
    # steps that far apart
    x = torch.empty(4 * far + 64, dtype=F16, device="cuda").as_strided((1, 5, 64), (1, far, 1))
    x.copy_(torch.randn(1, 5, 64, generator=g))
    gate = torch.rand(1, 5, 64, generator=g).to(F16).cuda()
    assert_within(capi.gated_scan(gate, x, **how)[0], plain_scan(gate, x, **how)["out"], "out")


@pytest.mark.gpu
def test_scan_negative_strides():
    """The C ABI takes strides that run backwards (an array seen from its end): the same as the turned tensor."""
    for B, T, Ch, Cg in ((3, 40, 3, 1), (2, 700, 64, 64), (2, 50, 96, 12)):
        how = modes(3)
        case = scan_inputs(B, T, Ch, Cg, F32, how["gate_mode"], 3)
        turned = {k: case[k].flip(1) for k in ("gate", "x", "dout")}
        want = plain_scan(turned["gate"], turned["x"], turned["dout"], case["dlast"], h0=case["h0"], **how)
        d = desc(B, T, Ch, Cg, gate_mode=how["gate_mode"], input_mode=how["input_mode"], gate_scale=how["gate_scale"], x_stride=(T * Ch, -Ch, 1), gate_stride=(T * Cg, -Cg, 1),
                 dout_stride=(T * Ch, -Ch, 1), out_stride=(T * Ch, -Ch, 1), dx_stride=(T * Ch, -Ch, 1), dgate_stride=(T * Cg, -Cg, 1))
        n = [C.c_size_t(0), C.c_size_t(0)]
        for backward in (0, 1):
            assert capi.lib().fvsrn_gated_scan_workspace(C.byref(d), backward, C.byref(n[backward])) == 0
        ws = torch.empty(max(n[0].value, n[1].value, 4), dtype=torch.uint8, device="cuda")
        out, last = torch.empty(B, T, Ch, device="cuda"), torch.empty(B, Ch, device="cuda")
        dgate, dx, dh0 = torch.empty(B, T, Cg, device="cuda"), torch.empty(B, T, Ch, device="cuda"), torch.empty(B, Ch, device="cuda")
        end = lambda t: t[:, -1:].data_ptr()  # noqa: E731
        s = torch.cuda.current_stream().cuda_stream
        assert capi.lib().fvsrn_gated_scan(C.byref(d), end(case["gate"]), end(case["x"]), case["h0"].data_ptr(), None, end(out), last.data_ptr(), ws.data_ptr(), n[0], s) == 0
        assert capi.lib().fvsrn_gated_scan_backward(C.byref(d), end(case["gate"]), end(case["x"]), case["h0"].data_ptr(), None, end(case["dout"]), case["dlast"].data_ptr(), end(dgate),
                                                    end(dx), dh0.data_ptr(), ws.data_ptr(), n[1], s) == 0
        for name, got in (("out", out.flip(1)), ("last", last), ("dgate", dgate.flip(1)), ("dx", dx.flip(1)), ("dh0", dh0)):
            assert_within(got, want[name], name)


@pytest.mark.gpu
def test_layer_captured_and_replayed():
    w, sw = capi.quantize_rows(torch.randn(256, 256, device="cuda") / 16)
    bias, x = torch.randn(256, device="cuda"), torch.randn(700, 256, device="cuda").half()

    def layer(x):
        q, s = capi.quantize_rows(x)
        return capi.matmul_int8(q, s, w, sw, bias, "ReLU", dtype=F16)

    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    for seed in range(3):
        x.copy_(torch.randn(700, 256, generator=torch.Generator().manual_seed(seed)).half())
        graph.replay()
        assert torch.equal(y, layer(x))


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_march_of_a_network_wider_than_the_fused_kernels():
    """rays -> 8-bit layers of 192 channels -> transfer function -> blend -> image and gradients: every stage against the 64-bit statement of what it was given."""
    W, H, T, step = 24, 16, 40, 0.05
    eye, right, up = capi.camera_on_a_sphere("Ym", (0, 0, 0), 0.4, 0.7, 1.6)
    fov = float(np.deg2rad(45.0))
    start, direction = capi.generate_rays(eye, right, up, fov, W, H)
    t = 0.6 + step * torch.arange(T, device="cuda")
    p = (start.view(-1, 1, 3) + t[:, None] * direction.view(-1, 1, 3)).view(-1, 3)
    g = torch.Generator().manual_seed(9)
    freq = (torch.randn(3, 64, generator=g) * 4).cuda()
    x = torch.cat((torch.sin(p @ freq), torch.cos(p @ freq), p), 1)
    sizes = [131, 192, 192, 1]
    for i, (K, N) in enumerate(zip(sizes, sizes[1:])):
        weight, bias = (torch.randn(N, K, generator=g) * math.sqrt(2 / K)).cuda(), (torch.randn(N, generator=g) * 0.1).cuda()
        activation, dtype = ("ReLU", F16) if i < 2 else ("Sigmoid", F32)
        w, sw = capi.quantize_rows(weight)
        q, s = capi.quantize_rows(x)
        assert_codes(x, q, s)
        y = capi.matmul_int8(q, s, w, sw, bias, activation, dtype=dtype)
        want, bound = plain_product(q, s, w, sw, bias, activation, 1.0, dtype)
        assert (np.abs(y.double().cpu().numpy() - want) <= bound).all(), i
        # the layer stands for the product in full: half a code of each factor
        full = x.double() @ weight.double().t() + bias.double()
        full = full.clamp(min=0) if activation == "ReLU" else torch.sigmoid(full)
        room = 0.5 * (s.double()[:, None] * weight.double().abs().sum(1) + sw.double() * x.double().abs().sum(1, keepdim=True)) + 0.25 * K * s.double()[:, None] * sw.double()
        assert ((y.double() - full).abs() <= room * 1.01 + 2.0 ** -10 * full.abs() + 1e-6).all(), i
        x = y
    scene = capi.Scene(eye=eye, right=right, up=up, fov_y_radians=fov, stepsize=step, tf_kind=capi.TF_IDENTITY, tf_scale_absorption=20.0, tf_scale_emission=1.0)
    colors = scene.evaluate_tf(x, 0.0, 1.0).view(W * H, T, 4)
    how = dict(gate_mode=capi.GATE_EXP, gate_scale=-step, input_mode=capi.INPUT_BLEND, reverse=True)
    rgb, absorption = colors[..., :3], colors[..., 3:]
    dpixel = torch.randn(W * H, 3, generator=g).cuda()
    want = plain_scan(absorption, rgb, None, dpixel, **how)
    _, pixel = capi.gated_scan(absorption, rgb, states=False, **how)
    dcolors = torch.empty_like(colors)
    capi.gated_scan_backward(absorption, rgb, None, dpixel, dgate=dcolors[..., 3:], dx=dcolors[..., :3], **how)
    assert_within(pixel, want["last"], "pixels")
    assert_within(dcolors[..., 3:], want["dgate"], "gradients of the absorption")
    assert_within(dcolors[..., :3], want["dx"], "gradients of the colours")


# ---------------------------------------------------------------------------------------------------------------------
# refusals (no GPU: nothing is enqueued before the arguments are checked)
# ---------------------------------------------------------------------------------------------------------------------

no_gpu = pytest.mark.skipif(capi.device_count() > 0, reason="made-up addresses: only where nothing can run")
OK = -6  # a call that passes every check ends at the missing device
GIB = 1 << 30


def desc(B=2, T=5, Ch=6, Cg=3, **kw):
    d = capi.ScanDesc(batch=B, length=T, channels=Ch, gate_channels=Cg, gate_scale=1.0)
    for name in ("gate_stride", "dgate_stride"):
        getattr(d, name)[:] = (T * Cg, Cg, 1)
    for name in ("x_stride", "out_stride", "dout_stride", "dx_stride"):
        getattr(d, name)[:] = (T * Ch, Ch, 1)
    for k, v in kw.items():
        if k.endswith("_stride"):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return d


def scan_call(d, gate=1 * GIB, x=2 * GIB, h0=3 * GIB, lengths=None, out=4 * GIB, last=5 * GIB, ws=6 * GIB, ws_bytes=GIB):
    return capi.lib().fvsrn_gated_scan(C.byref(d) if d is not None else None, gate, x, h0, lengths, out, last, ws, ws_bytes, None)


def backward_call(d, gate=1 * GIB, x=2 * GIB, h0=3 * GIB, lengths=None, dout=4 * GIB, dlast=5 * GIB, dgate=6 * GIB, dx=7 * GIB, dh0=8 * GIB, ws=9 * GIB, ws_bytes=GIB):
    return capi.lib().fvsrn_gated_scan_backward(C.byref(d), gate, x, h0, lengths, dout, dlast, dgate, dx, dh0, ws, ws_bytes, None)


@no_gpu
def test_scan_refusals():
    assert scan_call(desc()) == OK and backward_call(desc()) == OK
    assert scan_call(None) == -1
    for bad in (dict(dtype=3), dict(dtype=-1), dict(gate_mode=2), dict(input_mode=-1), dict(length=-1), dict(batch=-1), dict(gate_channels=4), dict(gate_channels=0),
                dict(gate_channels=-3), dict(gate_mode=1, gate_scale=math.nan), dict(gate_mode=1, gate_scale=math.inf), dict(out_stride=(30, 6, 0)), dict(out_stride=(6, 6, 1)),
                dict(out_stride=(0, 6, 1))):
        assert scan_call(desc(**bad)) == -1, bad
        assert capi.lib().fvsrn_last_error()
    for bad in (dict(dx_stride=(30, 5, 1)), dict(dgate_stride=(15, 3, 0)), dict(dtype=7)):
        assert backward_call(desc(**bad)) == -1, bad
    assert scan_call(desc(gate_scale=math.nan)) == OK  # (not read by this gate mode)
    for missing in ("gate", "x"):
        assert scan_call(desc(), **{missing: None}) == -1 and backward_call(desc(), **{missing: None}) == -1
    assert scan_call(desc(), out=None) == OK and scan_call(desc(), last=None) == OK and scan_call(desc(), out=None, last=None) == -1
    assert scan_call(desc(), h0=None) == OK and scan_call(desc(), h0=5 * GIB) == OK  # (the state in place)
    assert backward_call(desc(), dgate=None, dx=None, dh0=None) == -1 and backward_call(desc(), dgate=None, dx=None) == OK
    # sizes of zero need no pointers, and do nothing
    assert capi.lib().fvsrn_gated_scan(C.byref(desc(B=0)), None, None, None, None, None, None, None, 0, None) == 0
    assert scan_call(desc(T=0), gate=None, x=None) == OK
    # inputs may stand still, run backwards or share an address
    assert scan_call(desc(x_stride=(0, 0, 0), gate_stride=(0, 0, 0))) == OK
    assert scan_call(desc(x_stride=(30, -6, 1))) == OK
    assert scan_call(desc(x_stride=(1 << 62, 6, 1))) == -1
    # operands begin at an element
    for name in ("gate", "x", "h0", "out", "last"):
        assert scan_call(desc(), **{name: 10 * GIB + 2}) == -1, name
    assert scan_call(desc(dtype=1), x=10 * GIB + 2) == OK and scan_call(desc(dtype=1), x=10 * GIB + 1) == -1 and scan_call(desc(), lengths=10 * GIB + 2) == -1
    assert scan_call(desc(B=1 << 20, T=1 << 20, Ch=1024, Cg=1024)) == -4


@no_gpu
def test_scan_refuses_overlaps():
    for name in ("gate", "x", "h0"):
        for at in (0, 4, -4):
            kw = {name: 4 * GIB + at}
            assert scan_call(desc(), **kw) == -1, kw
    assert scan_call(desc(), last=4 * GIB + 8) == -1
    assert scan_call(desc(), last=3 * GIB + 4) == -1  # (beside h0, neither apart from it nor it)
    assert scan_call(desc(), lengths=4 * GIB) == -1
    for out in ("dgate", "dx", "dh0"):
        for name in ("gate", "x", "h0", "dout", "dlast"):
            assert backward_call(desc(), **{out: GIB, name: GIB}) == -1, (out, name)
    assert backward_call(desc(), dgate=7 * GIB) == -1 and backward_call(desc(), dh0=7 * GIB) == -1
    # colours and absorption beside each other, and what is not quite that
    ok = dict(Ch=3, Cg=1, dx_stride=(20, 4, 1), dgate_stride=(20, 4, 1))
    assert backward_call(desc(**ok), dgate=7 * GIB + 12) == OK and backward_call(desc(**ok), dgate=7 * GIB - 4) == OK
    assert backward_call(desc(**ok), dgate=7 * GIB + 8) == -1 and backward_call(desc(**ok), dgate=7 * GIB + 16) == -1
    assert backward_call(desc(**dict(ok, dgate_stride=(20, 8, 1))), dgate=7 * GIB + 12) == -1
    assert backward_call(desc(**dict(ok, dx_stride=(20, 3, 1), dgate_stride=(20, 3, 1))), dgate=7 * GIB + 12) == -1


@no_gpu
def test_scan_workspace_is_asked_for_and_checked():
    n = C.c_size_t(0)
    assert capi.lib().fvsrn_gated_scan_workspace(None, 0, C.byref(n)) == -1 and capi.lib().fvsrn_gated_scan_workspace(C.byref(desc()), 0, None) == -1
    assert capi.lib().fvsrn_gated_scan_workspace(C.byref(desc(dtype=9)), 0, C.byref(n)) == -1
    d = desc(B=1, T=60000, Ch=64, Cg=64)
    for backward, call in ((0, scan_call), (1, backward_call)):
        assert capi.lib().fvsrn_gated_scan_workspace(C.byref(d), backward, C.byref(n)) == 0 and n.value > 0
        assert call(d, ws_bytes=n.value) == OK and call(d, ws_bytes=n.value - 1) == -1 and call(d, ws=None, ws_bytes=n.value) == -1
        assert b"bytes" in capi.lib().fvsrn_last_error()
        assert call(d, ws=2 * GIB, ws_bytes=n.value) == -1  # (x)
    assert capi.lib().fvsrn_gated_scan_workspace(C.byref(desc(B=0)), 1, C.byref(n)) == 0 and n.value == 0


@no_gpu
def test_product_and_codes_refusals():
    def product(a=GIB, lda=64, sa=2 * GIB, b=3 * GIB, ldb=64, sb=4 * GIB, bias=5 * GIB, M=8, N=16, K=64, act=5, p=1.0, out=6 * GIB, dtype=0, ldo=16):
        return capi.lib().fvsrn_matmul_int8(a, lda, sa, b, ldb, sb, bias, M, N, K, act, p, out, dtype, ldo, None)

    assert product() == OK and product(bias=None) == OK and product(a=GIB + 1, lda=67) == OK
    for bad in (dict(dtype=3), dict(act=6), dict(act=-1), dict(act=1, p=0.0), dict(act=2, p=math.inf), dict(act=3, p=math.nan), dict(M=-1), dict(N=-1), dict(K=0), dict(lda=63), dict(ldb=63),
                dict(ldo=15), dict(a=None), dict(b=None), dict(sa=None), dict(sb=None), dict(out=None), dict(out=GIB + 63), dict(out=3 * GIB), dict(out=2 * GIB), dict(out=5 * GIB),
                dict(sa=2 * GIB + 2), dict(sb=4 * GIB + 1), dict(bias=5 * GIB + 3), dict(out=6 * GIB + 2)):
        assert product(**bad) == -1, bad
    assert product(K=131072, lda=131072, ldb=131072) == -4 and product(K=131071, lda=131071, ldb=131071) == OK
    assert product(N=(1 << 26) + 1, ldo=1 << 27) == -4 and product(M=(1 << 31) + 1) == -4
    assert product(M=0, a=None, out=None) == 0 and product(N=0) == 0
    assert product(act=0, p=math.nan) == OK  # (ReLU has no parameter)
    assert product(lda=0) == OK and product(M=1, ldo=1, lda=1) == OK

    def codes(x=GIB, dtype=1, rows=8, cols=64, ldx=64, q=2 * GIB, ldc=64, s=3 * GIB):
        return capi.lib().fvsrn_quantize_rows(x, dtype, rows, cols, ldx, q, ldc, s, None)

    assert codes() == OK and codes(ldx=0) == OK and codes(rows=0, x=None) == 0
    for bad in (dict(dtype=4), dict(rows=-1), dict(cols=0), dict(ldx=63), dict(ldc=63), dict(ldc=0), dict(x=None), dict(q=None), dict(s=None), dict(q=GIB + 100), dict(s=GIB), dict(s=2 * GIB)):
        assert codes(**bad) == -1, bad


def test_tensors_that_are_not_the_devices_are_refused():
    x = torch.zeros(2, 3, 4)
    for call in (lambda: capi.gated_scan(x, x), lambda: capi.gated_scan_backward(x, x, x), lambda: capi.quantize_rows(x[0]),
                 lambda: capi.matmul_int8(x[0].to(torch.int8), x[0, 0], x[0].to(torch.int8), x[0, 0])):
        with pytest.raises(capi.FvsrnError):
            call()


@pytest.mark.gpu
def test_tensor_refusals():
    f = lambda *s, dtype=F32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    x, g = f(2, 5, 6), f(2, 5, 3)
    for call in (lambda: capi.gated_scan(f(2, 5, 4), x), lambda: capi.gated_scan(g.half(), x), lambda: capi.gated_scan(g.double(), x.double()), lambda: capi.gated_scan(f(2, 4, 3), x),
                 lambda: capi.gated_scan(g, x, h0=f(2, 5)), lambda: capi.gated_scan(g, x, h0=f(2, 6, dtype=F16)), lambda: capi.gated_scan(g, x, lengths=f(2)),
                 lambda: capi.gated_scan(g, x, out=x), lambda: capi.gated_scan(g, x, out=f(2, 5, 1).expand(2, 5, 6)), lambda: capi.gated_scan(g, x, last=f(6, 2).t()),
                 lambda: capi.gated_scan_backward(g, x, f(2, 5, 5)), lambda: capi.gated_scan_backward(g, x, x.half()), lambda: capi.gated_scan_backward(g, x, x, dgate=g),
                 lambda: capi.gated_scan_backward(g, x, None, f(2, 6).half()), lambda: capi.quantize_rows(f(4, 6).t()), lambda: capi.quantize_rows(f(4)),
                 lambda: capi.quantize_rows(f(4, 6).double()), lambda: capi.quantize_rows(f(4, 6), scales=f(5)), lambda: capi.quantize_rows(f(4, 6), codes=f(4, 6)),
                 lambda: capi.matmul_int8(f(2, 8), f(2), f(3, 8), f(3)), lambda: capi.matmul_int8(f(2, 8, dtype=torch.int8), f(2), f(3, 9, dtype=torch.int8), f(3)),
                 lambda: capi.matmul_int8(f(2, 8, dtype=torch.int8), f(3), f(3, 8, dtype=torch.int8), f(3)),
                 lambda: capi.matmul_int8(f(2, 8, dtype=torch.int8), f(2), f(3, 8, dtype=torch.int8), f(3), f(2)),
                 lambda: capi.matmul_int8(f(2, 8, dtype=torch.int8), f(2), f(3, 8, dtype=torch.int8), f(3), activation="GELU"),
                 lambda: capi.matmul_int8(f(2, 8, dtype=torch.int8), f(2), f(3, 8, dtype=torch.int8), f(3), dtype=torch.float64)):
        with pytest.raises(capi.FvsrnError):
            call()


@no_gpu
def test_calls_of_more_threads_than_a_launch_has():
    # (less than 2^32 threads, in whole workgroups; sizes on both sides of the limit)
    def product(M, N, K=64):
        return capi.lib().fvsrn_matmul_int8(1 << 20, K, 1 << 50, 1 << 51, K, 1 << 52, None, M, N, K, 5, 1.0, 1 << 53, 1, N, None)

    assert product(1 << 31, 16) == OK  # (256 tokens a workgroup of 256)
    assert product((1 << 31) - 256, 128) == OK and product((1 << 31) - 255, 128) == -4  # (tiles of 256 tokens and 512 threads)
    assert product((1 << 31) - 256, 128, 1024) == OK and product((1 << 31) - 255, 17, 1024) == -4
    assert product((1 << 30) - 128, 129) == OK and product((1 << 30) - 127, 129) == -4  # (tiles of 128 and 256 threads)

    def codes(rows, cols):
        return capi.lib().fvsrn_quantize_rows(1 << 20, 1, rows, cols, cols, 1 << 50, cols, 1 << 52, None)

    assert codes((1 << 26) - 4, 1024) == OK and codes((1 << 26) - 3, 1024) == -4  # (a wave each)
    assert codes((1 << 28) - 16, 250) == OK and codes((1 << 28) - 15, 250) == -4  # (16 lanes each)
    # rows of one step and one gate, a lane each
    assert scan_call(desc(B=(1 << 31), T=1, Ch=1, Cg=1, gate_stride=(0, 0, 0), x_stride=(0, 0, 0), out_stride=(1, 1, 1)), out=1 << 50, last=1 << 52, h0=None) == OK
    for B, want in (((1 << 31) - 128, OK), ((1 << 31) - 127, -4)):
        assert scan_call(desc(B=B, T=1, Ch=2, Cg=2, gate_stride=(0, 0, 0), x_stride=(0, 0, 0), out_stride=(2, 2, 1)), out=1 << 50, last=1 << 52, h0=None) == want


@no_gpu
def test_strides_of_dimensions_of_one_may_be_anything():
    for s in (-(1 << 63), (1 << 63) - 1):
        assert scan_call(desc(B=1, T=1, Ch=1, Cg=1, x_stride=(s, s, s), gate_stride=(s, s, s), out_stride=(s, s, s))) == OK
        assert scan_call(desc(B=1, x_stride=(s, 6, 1), out_stride=(s, 6, 1))) == OK
        assert scan_call(desc(B=2, out_stride=(s, 6, 1))) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(5, 700, 3, 1), (2, 9000, 4, 1), (3, 300, 64, 64), (2, 3000, 70, 70), (2, 300, 260, 2)], ids=lambda s: "x".join(map(str, s)))
def test_scan_opaque_and_empty_samples(shape, dtype):
    """Gates of exactly 0 and 1: absorptions of infinity, of the type's largest value and of 0.  The same products and sums as by value, so the same bits."""
    B, T, Ch, Cg = shape
    r = np.random.RandomState(5)
    kind = torch.from_numpy(r.randint(0, 12, (B, T, Cg))).cuda()
    absorption = torch.zeros(B, T, Cg, device="cuda", dtype=dtype)
    absorption[kind == 0], absorption[kind == 1] = math.inf, torch.finfo(dtype).max
    value = (kind > 1).to(dtype)
    case = scan_inputs(B, T, Ch, Cg, dtype, capi.GATE_VALUE, 6)
    case["gate"] = value
    for blend in (capi.INPUT_ADD, capi.INPUT_BLEND):
        for reverse in (False, True):
            how = dict(input_mode=blend, reverse=reverse)
            want = check_scan(case, dict(how, gate_mode=capi.GATE_VALUE, gate_scale=1.0))
            how |= dict(gate_mode=capi.GATE_EXP, gate_scale=-2.0, h0=case["h0"])
            out, last = capi.gated_scan(absorption, case["x"], **how)
            dgate, dx, dh0 = capi.gated_scan_backward(absorption, case["x"], case["dout"], case["dlast"], **how)
            for name, got in (("out", out), ("last", last), ("dx", dx), ("dh0", dh0)):
                assert torch.equal(got, want[name]), name
            assert torch.equal(dgate[value == 0], torch.zeros_like(dgate[value == 0]))
            # -2 v is exact, but not what is left of a subnormal v: with s the step there (2^-24 of fp16) the rounding of v is off by s / 2, doubled s, and that of
            # -2 v by s / 2 again, 1.5 s together; both are multiples of s, so they are at most s apart
            f = torch.finfo(dtype)
            off = (dgate.double() + 2 * want["dgate"].double()).abs()[value == 1]
            assert (off <= torch.where(want["dgate"][value == 1].abs() < f.tiny, f.tiny * f.eps, 0.0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 300, 2, 2), (2, 9000, 1, 1), (2, 3000, 64, 64), (2, 5000, 70, 70)], ids=lambda s: "x".join(map(str, s)))
def test_scan_calls_at_once_on_two_streams_and_of_one_tensor(shape):
    """gate and x may be one tensor; two calls may run beside each other, each with scratch memory of its own."""
    how = modes(3)
    cases = [scan_inputs(*shape, F32, how["gate_mode"], s) for s in (1, 2)]

    def both(c):
        out, last = capi.gated_scan(c["gate"], c["gate"], h0=c["h0"], **how)
        return (out, last) + capi.gated_scan_backward(c["gate"], c["gate"], c["dout"], c["dlast"], h0=c["h0"], **how)

    want = [both(c) for c in cases]
    for c, w in zip(cases, want):
        plain = plain_scan(c["gate"], c["gate"], c["dout"], c["dlast"], h0=c["h0"], **how)
        for name, got in zip(("out", "last", "dgate", "dx", "dh0"), w):
            assert_within(got, plain[name], name)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for turn in range(4):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(both(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for a, b in zip(g, want[i % 2]):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 300, 3, 1), (2, 9000, 3, 1), (2, 3000, 64, 64), (2, 200, 260, 2), (9, 40, 100, 50)], ids=lambda s: "x".join(map(str, s)))
def test_scan_gradients_one_at_a_time(shape):
    """The entry without some of its outputs gives the same bits for the others."""
    how = modes(5)
    c = scan_inputs(*shape, F32, how["gate_mode"], 9, lengths=True)
    want = capi.gated_scan_backward(c["gate"], c["x"], c["dout"], c["dlast"], h0=c["h0"], lengths=c["lengths"], **how)
    d = desc(*shape, gate_mode=how["gate_mode"], input_mode=how["input_mode"], reverse=int(how["reverse"]), gate_scale=how["gate_scale"])
    n = C.c_size_t(0)
    assert capi.lib().fvsrn_gated_scan_workspace(C.byref(d), 1, C.byref(n)) == 0
    ws = torch.empty(max(n.value, 4), dtype=torch.uint8, device="cuda")
    for asked in range(1, 8):
        got = [torch.full_like(w, math.nan) if asked >> i & 1 else None for i, w in enumerate(want)]
        ptr = [None if g is None else g.data_ptr() for g in got]
        assert backward_call(d, *(c[k].data_ptr() for k in ("gate", "x", "h0", "lengths", "dout", "dlast")), *ptr, ws=ws.data_ptr(), ws_bytes=n.value) == 0
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert g is None or torch.equal(g, w), asked


# ---------------------------------------------------------------------------------------------------------------------
# what a program keeps and changes between its calls
# ---------------------------------------------------------------------------------------------------------------------

def described(T=5, gate_mode=capi.GATE_EXP, gate_scale=-1.0, input_mode=capi.INPUT_ADD, reverse=False, B=2, Ch=6, Cg=3):
    dense = lambda c: (T * c, c, 1)  # noqa: E731
    return capi._scan_plan(0, gate_mode, gate_scale, input_mode, reverse, (B, T, Cg), (B, T, Ch), dense(Cg), dense(Ch), dense(Ch), None, None, None)[0]


@pytest.mark.parametrize("name,field,first,second", [("gate_scale", "gate_scale", -0.5, -2.0), ("reverse", "reverse", False, True), ("gate_mode", "gate_mode", 1, 0), ("input_mode", "input_mode", 0, 1)])
def test_scan_takes_its_description_by_value(name, field, first, second):
    """A tensor that holds the scale, a mode or the direction and is changed in place: the next call goes by what it holds then."""
    v = torch.tensor(first)
    assert getattr(described(**{name: v}), field) == first
    v.fill_(second)
    assert getattr(described(**{name: v}), field) == second
    assert getattr(described(**{name: first}), field) == first


@pytest.mark.gpu
def test_scan_with_a_scale_that_is_trained():
    gate, x = torch.rand(4, 50, 1, device="cuda") * 5, torch.rand(4, 50, 3, device="cuda")
    step = torch.nn.Parameter(torch.tensor(-0.5))
    for value in (-0.5, -2.0):
        with torch.no_grad():
            step.fill_(value)
            how = dict(gate_mode=capi.GATE_EXP, input_mode=capi.INPUT_BLEND)
            got, want = (capi.gated_scan(gate, x, gate_scale=s, **how) for s in (step, value))
            back, back_want = (capi.gated_scan_backward(gate, x, x, gate_scale=s, **how) for s in (step, value))
        for a, b in zip(got + back[:2], want + back_want[:2]):
            assert torch.equal(a, b)


def negated(t, device="cpu"):
    """t as the imaginary part of a conjugate: a float32 view of memory that holds -t."""
    v = torch.complex(torch.zeros_like(t), -t).to(device).conj().imag
    assert v.is_neg() and torch.equal(v.cpu(), t)
    return v


def test_lazily_negated_views_are_refused():
    v = negated(torch.randn(2, 5, 3))
    with pytest.raises(capi.FvsrnError, match="resolve_neg"):
        capi._operand(v, "x", -1, F32)
    assert capi._operand(v.resolve_neg(), "x", -1, F32) and capi._operand(v.detach().clone(), "x", -1, F32)


@pytest.mark.gpu
def test_no_operand_may_be_a_lazily_negated_view():
    t = lambda *s: torch.rand(*s, device="cuda")  # noqa: E731
    gate, x, h0 = t(2, 5, 3), t(2, 5, 3), t(2, 3)
    n = lambda v: negated(v.cpu(), "cuda")  # noqa: E731
    flat = negated(torch.rand(4, 1), "cuda")  # (a matrix of one column has contiguous rows whatever its strides)
    codes, scales = capi.quantize_rows(flat.resolve_neg())
    for call in (lambda: capi.gated_scan(n(gate), x), lambda: capi.gated_scan(gate, n(x)), lambda: capi.gated_scan(gate, x, out=n(x)),
                 lambda: capi.gated_scan(n(gate[:1, :, :1]), x[:1, :, :1], h0=n(h0[:1, :1])), lambda: capi.gated_scan_backward(gate, x, n(x)),
                 lambda: capi.gated_scan_backward(gate, x, x, dx=n(x)), lambda: capi.gated_scan_backward(gate, x, x, dgate=n(gate)), lambda: capi.quantize_rows(flat),
                 lambda: capi.matmul_int8(codes, scales, codes, scales, out=n(t(4, 4)))):
        with pytest.raises(capi.FvsrnError, match="resolve_neg"):
            call()
    assert torch.equal(capi.gated_scan(gate, n(x).resolve_neg())[0], capi.gated_scan(gate, x)[0])


def test_sizes_beyond_an_int_are_refused(monkeypatch):
    """2^32 + n columns, channels or steps are not n of them: tensors without memory (they end at a null pointer where the size passes)."""
    monkeypatch.setattr(capi, "_launch_state", lambda t, what, stream: (-1, 0, None))
    meta = lambda *s, dtype=torch.int8: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    for n in ((1 << 31), (1 << 32) + 64, (1 << 33) + 5):
        for call in (lambda: capi.quantize_rows(meta(2, n, dtype=F16)), lambda: capi.matmul_int8(meta(1, n), meta(1, dtype=F32), meta(3, n), meta(3, dtype=F32)),
                     lambda: capi.matmul_int8(meta(1, 64), meta(1, dtype=F32), meta(n, 64), meta(n, dtype=F32)), lambda: described(T=n),
                     lambda: capi.gated_scan(meta(1, n, 1, dtype=F16), meta(1, n, 1, dtype=F16)), lambda: capi.gated_scan_backward(*[meta(1, n, 1, dtype=F16)] * 3)):
            with pytest.raises(capi.FvsrnError) as e:
                call()
            assert e.value.code == -4, e.value
    for mode in (dict(gate_mode=1 << 32), dict(input_mode=1 << 32), dict(gate_mode=2), dict(input_mode=-1)):
        with pytest.raises(capi.FvsrnError):
            described(**mode)


@pytest.mark.gpu
def test_rows_beyond_an_int_are_refused():
    """The same with memory behind them: rows of 2^32 + 64 codes, of which 64 would be read."""
    a = torch.empty(1, (1 << 32) + 64, dtype=torch.int8, device="cuda")
    one = torch.ones(1, device="cuda")
    out = torch.full((1, 1), 7.0, device="cuda")
    with pytest.raises(capi.FvsrnError):
        capi.matmul_int8(a, one, a, one, out=out)
    with pytest.raises(capi.FvsrnError):
        capi.quantize_rows(torch.empty(1, (1 << 32) + 64, dtype=F16, device="cuda"))
    assert float(out) == 7.0


def test_scan_does_not_drop_a_gradient(monkeypatch):
    """Tensors without memory: a call that passes ends at a null pointer."""
    monkeypatch.setattr(capi, "_launch_state", lambda t, what, stream: (-1, 0, None))
    meta = lambda *s, grad=False: torch.empty(*s, device="meta").requires_grad_(grad)  # noqa: E731
    for trained in range(3):
        gate, x, h0 = (meta(*s, grad=i == trained) for i, s in enumerate(((2, 5, 3), (2, 5, 6), (2, 6))))
        with pytest.raises(capi.FvsrnError, match="gated_scan_backward"):
            capi.gated_scan(gate, x, h0=h0)
        for call in (lambda: capi.gated_scan(gate.detach(), x.detach(), h0=h0.detach()), torch.no_grad()(lambda: capi.gated_scan(gate, x, h0=h0)),
                     lambda: capi.gated_scan_backward(gate, x, meta(2, 5, 6), h0=h0)):
            with pytest.raises(capi.FvsrnError, match="null pointer"):
                call()


@pytest.mark.gpu
def test_scan_in_an_autograd_function():
    how = modes(7)

    class Blend(torch.autograd.Function):
        @staticmethod
        def forward(ctx, gate, x, h0):
            ctx.save_for_backward(gate, x, h0)
            return capi.gated_scan(gate, x, h0=h0, **how)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dout, dlast):
            gate, x, h0 = ctx.saved_tensors
            return capi.gated_scan_backward(gate, x, dout, dlast, h0=h0, **how)

    for shape in ((5, 60, 3, 1), (2, 300, 64, 64)):
        c = scan_inputs(*shape, F32, how["gate_mode"], 21)
        leaves = [c[k].clone().requires_grad_() for k in ("gate", "x", "h0")]
        out, last = Blend.apply(*leaves)
        ((out * c["dout"]).sum() + (last * c["dlast"]).sum()).backward()
        want = plain_scan(c["gate"], c["x"], c["dout"], c["dlast"], h0=c["h0"], **how)
        for leaf, name in zip(leaves, ("dgate", "dx", "dh0")):
            assert_within(leaf.grad, want[name], name)
        with pytest.raises(capi.FvsrnError):
            capi.gated_scan(*leaves[:2], **how)


@no_gpu
def test_scans_of_no_steps_that_write_nothing():
    """Empty tensors have no address: nothing is asked for, and nothing is to be done."""
    empty = dict(gate=None, x=None, h0=None)
    assert backward_call(desc(T=0), dout=None, dgate=None, dx=None, dh0=None, **empty) == 0
    assert scan_call(desc(T=0), out=None, last=None, **empty) == 0
    assert backward_call(desc(T=0), dout=None, dgate=None, dx=None, **empty) == OK and scan_call(desc(T=0), out=None, **empty) == OK  # (there is something to write)
    assert backward_call(desc(T=0, dtype=3), dgate=None, dx=None, dh0=None, **empty) == -1


@pytest.mark.gpu
def test_scan_gradients_of_no_steps_without_a_state():
    for shape in ((3, 0, 8), (2, 0, 3)):
        gate, x = torch.empty(shape[0], 0, 1, device="cuda"), torch.empty(shape, device="cuda")
        dgate, dx, dh0 = capi.gated_scan_backward(gate, x, torch.empty(shape, device="cuda"), torch.randn(shape[0], shape[2], device="cuda"))
        assert dgate.shape == gate.shape and dx.shape == x.shape and dh0 is None


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 100, 64, 64), (1, 256, 256, 256), (3, 37, 70, 70), (1, 300, 300, 100), (1, 20000, 2, 1), (40, 300, 3, 1), (2, 500, 128, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_scan_state_in_place_equals_a_state_apart(shape, dtype):
    """last = h0 in every layout: eight or sixteen waves on a tile in one launch, spans, rows; sequences that end early, and empty ones."""
    for i in (3, 6):
        how = modes(i)
        c = scan_inputs(*shape, dtype, how["gate_mode"], 31, lengths=True)
        for lengths in (c["lengths"], None):
            for states in (True, False):
                want = capi.gated_scan(c["gate"], c["x"], h0=c["h0"], lengths=lengths, states=states, **how)
                for _ in range(3):
                    h = c["h0"].clone()
                    out, last = capi.gated_scan(c["gate"], c["x"], h0=h, last=h, lengths=lengths, states=states, **how)
                    assert last is h and torch.equal(h, want[1]) and (not states or torch.equal(out, want[0]))


@no_gpu
def test_scan_of_an_input_that_stands_still_is_laid_out_like_a_dense_one():
    """x broadcast along the steps says nothing of how the others lie: the scratch memory (and with it the layout) is that of a dense x."""
    def scratch(B, T, Ch, Cg, backward, **kw):
        n = C.c_size_t(0)
        assert capi.lib().fvsrn_gated_scan_workspace(C.byref(desc(B, T, Ch, Cg, **kw)), backward, C.byref(n)) == 0
        return n.value

    for B, T, Ch, Cg in ((8, 4096, 1024, 1024), (1, 9000, 30, 10), (3, 5000, 64, 32)):
        for backward in (0, 1):
            dense = scratch(B, T, Ch, Cg, backward)
            assert dense > 0 and dense == scratch(B, T, Ch, Cg, backward, x_stride=(Ch, 0, 1)) == scratch(B, T, Ch, Cg, backward, x_stride=(0, 0, 1))
    # steps innermost: the lanes go along them, whichever operand says so
    B, T, C_ = 2, 9000, 12
    turned = (T * C_, 1, T)
    rows = scratch(B, T, C_, C_, 0, x_stride=turned, out_stride=turned, gate_stride=turned)
    assert rows == scratch(B, T, C_, C_, 0, x_stride=(C_, 0, 1), out_stride=turned, gate_stride=turned) == scratch(B, T, C_, C_, 0, x_stride=(C_, 0, 1), out_stride=(0, 0, 1), gate_stride=turned)
    assert rows != scratch(B, T, C_, C_, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 70, 12, 12), (2, 700, 64, 64), (2, 3000, 70, 70), (2, 300, 60, 20), (3, 600, 30, 30), (2, 9, 10, 10), (4, 300, 3, 1)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
def test_scan_of_an_input_that_stands_still(shape, dtype):
    B, T, Ch, Cg = shape
    for i in (2, 7):
        how = modes(i)
        c = scan_inputs(B, T, Ch, Cg, dtype, how["gate_mode"], 17, lengths=True)
        c["x"] = c["x"][:, :1].expand(B, T, Ch)
        assert c["x"].stride(1) == 0
        check_scan(c, how)
        c["x"], c["gate"] = c["x"][:1, :, :1].expand(B, T, Ch), c["gate"][:, :1].expand(B, T, Cg)  # (nothing that is read moves)
        check_scan(c, how, states=False)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 90, 3, 1), (3, 90, 64, 64), (3, 3000, 64, 64), (2, 9000, 2, 2), (2, 9000, 3, 1), (3, 400, 16, 2), (3, 400, 66, 22), (2, 1200, 70, 1)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_infinite_states_and_gradients_stay_not_finite(shape, reverse):
    """An infinity at one step of one channel: infinite there, not finite from there on (the products of gates behind it fall below the smallest 32-bit number), and
    everything else keeps its bits.  Gradients the same way, towards the sequence's beginning."""
    B, T, Ch, Cg = shape
    r = torch.Generator().manual_seed(13)
    gate, x, dout = (torch.rand(B, T, Cg, generator=r) * 0.5 + 0.25).cuda(), torch.randn(B, T, Ch, generator=r).cuda(), torch.randn(B, T, Ch, generator=r).cuda()
    h0, dlast = torch.randn(B, Ch, generator=r).cuda(), torch.randn(B, Ch, generator=r).cuda()
    how = dict(reverse=reverse, h0=h0)
    clean, back = capi.gated_scan(gate, x, **how), capi.gated_scan_backward(gate, x, dout, dlast, **how)
    b, c, g = 1, 1, 1 // (Ch // Cg)
    for at in (0, 40, T - 1):
        for value in (math.inf, -math.inf):
            bad = x.clone()
            bad[b, at, c] = value
            out, last = capi.gated_scan(gate, bad, **how)
            later = slice(None, at + 1) if reverse else slice(at, None)
            assert out[b, at, c] == value and not out[b, later, c].isfinite().any() and not last[b, c].isfinite()
            assert not (out[b, later, c] == -value).any()  # (gates are positive)
            for got, want, where in ((out, clean[0], (b, later, c)), (last, clean[1], (b, c))):
                got[where] = want[where]
                assert torch.equal(got, want)
            bad = dout.clone()
            bad[b, at, c] = value
            dgate, dx, dh0 = capi.gated_scan_backward(gate, x, bad, dlast, **how)
            earlier = slice(at, None) if reverse else slice(None, at + 1)
            assert dx[b, at, c] == value and not dx[b, earlier, c].isfinite().any() and not dgate[b, earlier, g].isfinite().any() and not dh0[b, c].isfinite()
            for got, want, where in ((dx, back[1], (b, earlier, c)), (dgate, back[0], (b, earlier, g)), (dh0, back[2], (b, c))):
                got[where] = want[where]
                assert torch.equal(got, want)
