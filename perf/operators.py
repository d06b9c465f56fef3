"""The tensor operators of a ray march -- the gated scan with its gradients and the 8-bit layer -- at the sizes their callers use.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes a case's inputs on the GPU and ``run`` is one pass:
through the framework's calls where ``own`` is true, in elementary torch operations in 32 bits where it is not.  ``exact`` is the same result from
the definitions in 64 bits.  A case's ``op`` is one of

  scan        the recurrence h_t = a_t h_{t-1} + u_t along a ray or a series (a_t = gate or exp(scale gate), u_t = x_t or (1 - a_t) x_t)
  scan_grad   the same and its gradients, as one training step
  product     8-bit matrix product of quantized tokens with quantized weights, bias and activation included
  layer       a whole layer: quantization of the tokens, then the product
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------

def _scan(name, op, B, T, C, Cg, dtype="f32", gate="exp", input="blend", layout="separate", reverse=False, states=False, h0=False, ragged=False):
    return dict(name=name, op=op, B=B, T=T, C=C, Cg=Cg, dtype=dtype, gate=gate, input=input, layout=layout, reverse=reverse, states=states, h0=h0, ragged=ragged)


def _product(name, op, M, N, K, x="f16", y="f16", activation="ReLU"):
    return dict(name=name, op=op, M=M, N=N, K=K, x=x, y=y, activation=activation)


def listed():
    return [
        # one step of a march that carries its colours along, a 64 x 64 tile of rays: the smallest call, its launch is what it costs
        _scan("march step, 64x64 rays", "scan", 1, 1, 3 * 4096, 4096, h0=True),
        # a preview image: colours and absorptions as the transfer function leaves them, (rays, samples, rgb + absorption), blended back to front
        _scan("blend, 256x256 rays x 256", "scan", 65536, 256, 3, 1, layout="interleaved", reverse=True),
        # a frame's worth of samples in one call, the largest
        _scan("blend, 512x512 rays x 512", "scan", 262144, 512, 3, 1, layout="interleaved", reverse=True),
        # one long series of latent channels with every state kept
        _scan("series, 65536 x 1024", "scan", 1, 65536, 1024, 1024, "bf16", "value", "add", states=True, h0=True),
        # a training batch of rays: pixels, then gradients of every colour and absorption
        _scan("blend + gradients, 16384 rays x 512", "scan_grad", 16384, 512, 3, 1, layout="interleaved", reverse=True),
        # a training batch of series in half precision
        _scan("series + gradients, 8 x 4096 x 1024", "scan_grad", 8, 4096, 1024, 1024, "f16", "exp", "add", states=True, h0=True),
        # a padded batch of series of different lengths (one of them empty), gates shared by eight channels, odd sizes
        _scan("ragged + gradients, 37 x 1001 x 96", "scan_grad", 37, 1001, 96, 12, "f32", "value", "blend", reverse=True, states=True, h0=True, ragged=True),
        # one token through a wide layer: the weights' bytes are what it costs
        _product("product, 1 x 4096 x 4096", "product", 1, 4096, 4096, y="bf16", activation="None"),
        # a handful of points through a layer of odd width
        _product("layer, 48 x 1000 x 1000", "layer", 48, 1000, 1000, x="f32", activation="SnakeAlt"),
        # a tile of samples through a hidden layer twice as wide as the fused kernels hold
        _product("layer, 262144 x 256 x 256", "layer", 262144, 256, 256),
        # the last layer: four outputs, odd depth, colours in 32 bits
        _product("layer, 100003 x 4 x 250", "layer", 100003, 4, 250, y="f32", activation="Sigmoid"),
        # the largest product: the matrix units are what it costs
        _product("product, 8192 x 4096 x 4096", "product", 8192, 4096, 4096, x="bf16", y="bf16", activation="None"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rays", "planes", "series", "product", "layer"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    if kind in ("product", "layer"):
        N, K = _log(rng, 1, 4096), _log(rng, 16, 4096)
        most = min(262144, 8192 * 4096 * 4096 // (N * K), 262144 * 512 // (N + K))
        return dict(op=kind, M=_log(rng, 1, most), N=N, K=K, x=dtype, y=rng.choice(("f32", "f16", "bf16")),
                    activation=rng.choice(("None", "ReLU", "Sine", "Snake", "SnakeAlt", "Sigmoid")))
    case = dict(op=rng.choice(("scan", "scan_grad")), dtype=dtype, gate=rng.choice(("value", "exp")), input=rng.choice(("add", "blend")),
                reverse=rng.random() < 0.5, states=rng.random() < 0.5, h0=rng.random() < 0.5, ragged=rng.random() < 0.3, layout="separate")
    if kind == "rays":
        T, C = _log(rng, 1, 1024), rng.randint(1, 4)
        case |= dict(layout="interleaved", T=T, C=C, Cg=1, B=_log(rng, 1, min(262144, 24_000_000 // (T * (C + 1)))))
    elif kind == "planes":
        T, G = _log(rng, 1, 512), rng.randint(1, 4)
        Cg = _log(rng, 64, min(1 << 20, 67_000_000 // (T * G)))
        case |= dict(B=1, T=T, C=G * Cg, Cg=Cg)
    else:
        B, T = _log(rng, 1, 64), _log(rng, 1, 65536)
        G = rng.choice((1, 1, 2, 8, 64))
        Cg = _log(rng, 1, max(1, min(4096, 33_000_000 // (B * T)) // G))
        case |= dict(B=B, T=T, C=G * Cg, Cg=Cg)
        if B * T * G > 33_000_000:
            case["T"] = 33_000_000 // (B * G)
    return case


def work(case):
    if case["op"] in ("product", "layer"):
        M, N, K = case["M"], case["N"], case["K"]
        token = DTYPES[case["x"]].itemsize if case["op"] == "layer" else 1
        read = M * K * token + N * K + 8 * N + (4 * M if case["op"] == "product" else 0)
        return {"bytes": read + M * N * DTYPES[case["y"]].itemsize, "flops": 2 * M * N * K}
    e, rows = DTYPES[case["dtype"]].itemsize, case["B"] * case["C"]
    n, ng = rows * case["T"], case["B"] * case["T"] * case["Cg"]
    moved = e * (n + ng) + 4 * rows * (1 + case["h0"]) + e * n * case["states"]
    if case["op"] == "scan":
        return {"bytes": moved, "flops": 3 * n + 4 * ng}
    return {"bytes": moved + e * (n * case["states"] + n + ng) + 4 * rows * (1 + case["h0"]), "flops": 10 * n + 8 * ng}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def _quantized(x):
    """Codes and scales of the rows of x: scale = max |x| / 127 in 32 bits, code = x / scale in 32 bits, rounded to the nearest (ties to even)."""
    x = x.float()
    scale = torch.clamp(x.abs().amax(1) / 127.0, min=2.0 ** -126)
    return torch.round(x / scale[:, None]).to(torch.int8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    if case["op"] in ("product", "layer"):
        M, N, K = case["M"], case["N"], case["K"]
        w, scale_w = _quantized(normal(N, K) / math.sqrt(K))
        state = dict(case=case, w=w, scale_w=scale_w, bias=0.1 * normal(N))
        x = normal(M, K).to(DTYPES[case["x"]])
        if case["op"] == "product":
            state["q"], state["scale"] = _quantized(x)
        else:
            state["x"] = x
        return state
    B, T, C, Cg, dtype = (case[k] for k in ("B", "T", "C", "Cg", "dtype"))
    dtype = DTYPES[dtype]
    state = dict(case=case, scale=1.0)
    if case["gate"] == "exp":
        # absorptions behind a transfer function: empty space in half of the samples, and the step of a march through the unit box
        gate = torch.clamp(8.0 * normal(B, T, Cg), min=0.0)
        state["scale"] = -1.0 / max(T, 64)
    else:
        gate = 1.0 - 0.1 * uniform(B, T, Cg)
    x = uniform(B, T, C) if case["input"] == "blend" else normal(B, T, C)
    if case["layout"] == "interleaved":
        both = torch.cat((x, gate), 2).to(dtype)
        state["x"], state["gate"] = both[:, :, :C], both[:, :, C:]
    else:
        state["x"], state["gate"] = x.to(dtype), gate.to(dtype)
    state["h0"] = normal(B, C) if case["h0"] else None
    state["lengths"] = None
    if case["ragged"]:
        lengths = (uniform(B) * (T + 1)).floor().clamp(max=T)
        lengths[B // 2] = 0 if B > 1 else T
        state["lengths"] = lengths.to(torch.int32)
    if case["op"] == "scan_grad":
        state["dout"] = normal(B, T, C).to(dtype) if case["states"] else None
        state["dlast"] = normal(B, C)
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return _plain_product(state) if state["case"]["op"] in ("product", "layer") else _plain_scan(state)


def _run_own(state):
    from fvsrn_amd import capi
    case = state["case"]
    if case["op"] in ("product", "layer"):
        q, scale = capi.quantize_rows(state["x"]) if case["op"] == "layer" else (state["q"], state["scale"])
        return capi.matmul_int8(q, scale, state["w"], state["scale_w"], state["bias"], activation=case["activation"], dtype=DTYPES[case["y"]])
    how = dict(gate_mode=capi.GATE_EXP if case["gate"] == "exp" else capi.GATE_VALUE, gate_scale=state["scale"],
               input_mode=capi.INPUT_BLEND if case["input"] == "blend" else capi.INPUT_ADD, reverse=case["reverse"], h0=state["h0"], lengths=state["lengths"])
    out, last = capi.gated_scan(state["gate"], state["x"], states=case["states"], **how)
    if case["op"] == "scan":
        return {"out": out, "last": last}
    dgate, dx, dh0 = capi.gated_scan_backward(state["gate"], state["x"], state["dout"], state["dlast"], **how)
    return {"out": out, "last": last, "dgate": dgate, "dx": dx, "dh0": dh0}


def _activated(y, kind):
    if kind == "ReLU":
        return torch.clamp(y, min=0.0)
    if kind == "Sine":
        return torch.sin(y)
    if kind == "Snake":
        return y + torch.sin(y) ** 2
    if kind == "SnakeAlt":
        return (y + 1.0 - torch.cos(2.0 * y)) / 2.0
    if kind == "Sigmoid":
        return 1.0 / (1.0 + torch.exp(-y))
    return y


def _plain_product(state):
    case = state["case"]
    q, scale = _quantized(state["x"]) if case["op"] == "layer" else (state["q"], state["scale"])
    y = torch.matmul(q.float(), state["w"].float().t())
    y = y * scale[:, None] * state["scale_w"] + state["bias"]
    return _activated(y, case["activation"]).to(DTYPES[case["y"]])


def _recurrence(a, u):
    """h_t = a_t h_{t-1} + u_t along dimension 1 from h = 0, and the products of the gates up to t: spans of 1, 2, 4, ... steps joined."""
    d, T = 1, u.shape[1]
    while d < T:
        u = torch.cat((u[:, :d], u[:, d:] + a[:, d:] * u[:, :-d]), 1)
        a = torch.cat((a[:, :d], a[:, d:] * a[:, :-d]), 1)
        d *= 2
    return u, a


def _order(state, device):
    """Step i of sequence b is at t = order[b, i] (its own inverse), and whether the sequence has such a step."""
    case = state["case"]
    i = torch.arange(case["T"], device=device)[None, :]
    n = torch.full((case["B"], 1), case["T"], device=device) if state["lengths"] is None else state["lengths"][:, None].long()
    return torch.where(i < n, n - 1 - i if case["reverse"] else i.expand(case["B"], -1), i), i < n


def _plain_scan(state):
    case = state["case"]
    B, T, C, Cg, dtype = case["B"], case["T"], case["C"], case["Cg"], DTYPES[case["dtype"]]
    G = C // Cg
    gate, x = state["gate"].float(), state["x"].float().reshape(B, T, Cg, G)
    order = inside = None
    if state["lengths"] is not None:
        order, inside = _order(state, gate.device)
        inside = inside[:, :, None, None]

    def turned(v):
        if order is not None:
            return torch.gather(v, 1, order[:, :, None, None].expand(-1, -1, v.shape[2], v.shape[3]))
        return torch.flip(v, (1,)) if case["reverse"] else v

    gate, x = turned(gate[:, :, :, None]), turned(x)
    if case["gate"] == "exp":
        a, rest = torch.exp(state["scale"] * gate), -torch.expm1(state["scale"] * gate)
    else:
        a, rest = gate, 1.0 - gate
    u = rest * x if case["input"] == "blend" else x
    if inside is not None:
        a, u = torch.where(inside, a, 1.0), torch.where(inside, u, 0.0)
    h0 = torch.zeros(B, Cg, G, device=gate.device) if state["h0"] is None else state["h0"].reshape(B, Cg, G)
    h, through = _recurrence(a, u)
    h = h + through * h0[:, None]
    kept = h if inside is None else torch.where(inside, h, 0.0)
    result = {"out": turned(kept).reshape(B, T, C).to(dtype) if case["states"] else None, "last": h[:, -1].reshape(B, C)}
    if case["op"] == "scan":
        return result
    # the gradient of h_t: its own and what h_{t+1} passes on, the same recurrence run backwards with the gates one step later
    d = torch.zeros(B, T, Cg, G, device=gate.device) if state["dout"] is None else turned(state["dout"].float().reshape(B, T, Cg, G))
    if inside is not None:
        d = torch.where(inside, d, 0.0)
    d = torch.cat((d[:, :-1], d[:, -1:] + state["dlast"].reshape(B, 1, Cg, G)), 1)
    later = torch.cat((torch.ones_like(a[:, :1]), torch.flip(a, (1,))[:, :-1]), 1)
    d = torch.flip(_recurrence(later, torch.flip(d, (1,)))[0], (1,))
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    if case["input"] == "blend":
        dx, da = rest * d, d * (before - x)
    else:
        dx, da = d, d * before
    da = da.sum(3, keepdim=True)
    dgate = state["scale"] * a * da if case["gate"] == "exp" else da
    if inside is not None:
        dx, dgate = torch.where(inside, dx, 0.0), torch.where(inside, dgate, 0.0)
    result["dgate"], result["dx"] = turned(dgate).reshape(B, T, Cg).to(dtype), turned(dx).reshape(B, T, C).to(dtype)
    result["dh0"] = (a[:, 0] * d[:, 0]).reshape(B, C) if case["h0"] else None
    return result


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "scan_grad" and case["T"] > 20000:
        return None  # one step after the other, there and back: too long to wait for
    state = prepare(case, seed)
    return _exact_product(state) if case["op"] in ("product", "layer") else _exact_scan(state)


def _exact_product(state):
    case = state["case"]
    if case["op"] == "layer":  # the codes are defined by 32-bit divisions: what is exact is what follows from them
        x = state["x"].float()
        scale = torch.maximum(x.abs().max(dim=1).values / 127.0, torch.tensor(2.0 ** -126, device=x.device))
        q = torch.round(torch.div(x, scale.unsqueeze(1)))
    else:
        q, scale = state["q"], state["scale"]
    w, scale_w, bias = state["w"].double(), state["scale_w"].double(), state["bias"].double()
    y = torch.addmm(bias, q.double() * scale.double().unsqueeze(1), (w * scale_w.unsqueeze(1)).t().contiguous())
    kind = case["activation"]
    if kind == "ReLU":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif kind == "Sine":
        y = y.sin()
    elif kind == "Snake":
        y = y + (1.0 - (2.0 * y).cos()) / 2.0
    elif kind == "SnakeAlt":
        y = 0.5 * y + y.sin() ** 2
    elif kind == "Sigmoid":
        y = torch.sigmoid(y)
    return y


def _exact_scan(state):
    case = state["case"]
    B, T, C, Cg = case["B"], case["T"], case["C"], case["Cg"]
    dev = state["x"].device
    n = torch.full((B,), T, device=dev) if state["lengths"] is None else state["lengths"].long()
    rows = torch.arange(B, device=dev)

    def factors(t):
        g = state["gate"][rows, t].double().repeat_interleave(C // Cg, 1) if B > 1 else state["gate"][:, int(t)].double().repeat_interleave(C // Cg, 1)
        if case["gate"] == "exp":
            return torch.exp(state["scale"] * g), -torch.expm1(state["scale"] * g)
        return g, 1.0 - g

    def at(v, t):
        return v[rows, t].double() if B > 1 else v[:, int(t)].double()

    if B == 1:
        n = int(n[0])
        steps = [(n - 1 - i if case["reverse"] else i) for i in range(n)]
        live = [None] * n
    else:
        steps, live = [], []
        for i in range(T):
            t = n - 1 - i if case["reverse"] else torch.full_like(n, i)
            steps.append(t.clamp(0, max(T - 1, 0)))
            live.append((n > i)[:, None])
    h = torch.zeros(B, C, device=dev, dtype=torch.float64) if state["h0"] is None else state["h0"].double()
    grads = case["op"] == "scan_grad"
    out = torch.zeros(B, T, C, device=dev, dtype=torch.float64) if case["states"] else None
    passed = []
    for t, ok in zip(steps, live):
        a, rest = factors(t)
        x = at(state["x"], t)
        new = a * h + (rest * x if case["input"] == "blend" else x)
        if grads:
            passed.append(h)
        if ok is None:
            h = new
            if out is not None:
                out[0, t] = h[0]
        else:
            h = torch.where(ok, new, h)
            if out is not None:
                out[rows, t] = torch.where(ok, h, out[rows, t])
    result = {"out": out, "last": h}
    if not grads:
        return result
    dx, dg = torch.zeros(B, T, C, device=dev, dtype=torch.float64), torch.zeros(B, T, Cg, device=dev, dtype=torch.float64)
    carry = state["dlast"].double()
    for k in range(len(steps) - 1, -1, -1):
        t, ok = steps[k], live[k]
        a, rest = factors(t)
        d = carry + at(state["dout"], t) if state["dout"] is not None else carry
        da = d * (passed[k] - at(state["x"], t)) if case["input"] == "blend" else d * passed[k]
        if case["gate"] == "exp":
            da = state["scale"] * a * da
        da = da.reshape(B, Cg, C // Cg).sum(2)
        own_dx = rest * d if case["input"] == "blend" else d
        if ok is None:
            dx[0, t], dg[0, t], carry = own_dx[0], da[0], a * d
        else:
            dx[rows, t] = torch.where(ok, own_dx, dx[rows, t])
            dg[rows, t] = torch.where(ok, da, dg[rows, t])
            carry = torch.where(ok, a * d, carry)
    result |= {"dgate": dg, "dx": dx, "dh0": carry if case["h0"] else None}
    return result
