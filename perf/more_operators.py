"""The operators that train and serve a dense teacher, as cases that can be timed: root-mean-square norm with the residual's addition (forward, backward, and
into the 8-bit frames of the int8 product), the dense product with bias, activation and residual in its epilogue and its gradients, the gated feed-forward
block and the gradient of its gate, and the optimizer step whose gradients are clipped by their global norm.  All but the last work on frame buffers:
[nodes, frame_stride], frames contiguous, fp32 or bf16.

listed() names twelve cases, draw() gives further ones of the same ranges, prepare() makes what a program has in hand before the call, run() is one
pass (elementary torch operations in 32 bits, or with `own` the framework's operators), exact() the same in 64 bits, work() what a pass cannot do without.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
LR, BETA1, BETA2, MAX_NORM = 0.001, 0.9, 0.999, 1.0
# the operator's arguments are numbers of 32 bits, and so are these
RATE1, RATE2 = float(np.float32(1) - np.float32(BETA1)), float(np.float32(1) - np.float32(BETA2))


def listed():
    return [
        # one request's frame: the residual is added, normalised and quantised, and goes through an int8 layer
        {"name": "rms_int8_4096x1_bf16", "kind": "rms_int8", "nodes": 4096, "frames": 1, "n_out": 1024, "bf16": True, "residual": True},
        # hidden activations on a batch that divides nothing
        {"name": "rms_3000x5001", "kind": "rms_forward", "nodes": 3000, "frames": 5001, "bf16": False, "residual": True},
        # a wide layer on one GPU's share of a batch
        {"name": "rms_8192x16384_bf16", "kind": "rms_forward", "nodes": 8192, "frames": 16384, "bf16": True, "residual": True},
        # the gradient of the same in training, where a second path's gradient arrives as well
        {"name": "rms_grad_4096x16384_bf16", "kind": "rms_backward", "nodes": 4096, "frames": 16384, "bf16": True, "residual": True},
        # a dense layer for a single frame: the weights are what is read
        {"name": "dense_4096x4096x1", "kind": "dense", "n_in": 4096, "n_out": 4096, "frames": 1, "fp32": False, "bias": True, "activation": "gelu", "residual": True},
        # class scores of a small batch, odd sizes
        {"name": "dense_1020x1000x200", "kind": "dense", "n_in": 1020, "n_out": 1000, "frames": 200, "fp32": True, "bias": True, "activation": "none",
         "residual": False},
        # both gradients of a dense layer on a full batch
        {"name": "dense_grad_4096x4096x8192", "kind": "dense_backward", "n_in": 4096, "n_out": 4096, "frames": 8192},
        # the gated block for a few frames at a time
        {"name": "gated_4096x8192x16", "kind": "gated", "n_in": 4096, "hidden": 8192, "frames": 16, "activation": "silu", "keep": False},
        # the gated block of a training step: what its gradient needs is kept
        {"name": "gated_4096x8192x4096", "kind": "gated", "n_in": 4096, "hidden": 8192, "frames": 4096, "activation": "silu", "keep": True},
        # the gradient that goes back through the second product and the gate, odd sizes
        {"name": "gated_grad_2000x5500x3001", "kind": "gated_backward", "n_out": 2000, "hidden": 5500, "frames": 3001, "activation": "gelu"},
        # the step of a small MLP: two LUT layers and a normalised head
        {"name": "clip_step_mlp", "kind": "clip_step", "sizes": "26880 4480 70 70"},
        # the step of the regression network's six layers of 65536 tables
        {"name": "clip_step_6x65536x64", "kind": "clip_step", "sizes": " ".join(["4194304"] * 6)},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm; half of the time rounded to a multiple of eight."""
    n = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))
    return max(lo, n // 8 * 8) if n >= 64 and rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(("rms_int8", "rms_forward", "rms_forward", "rms_backward", "dense", "dense", "dense_backward", "gated", "gated", "gated_backward", "clip_step"))
    if kind.startswith("rms"):
        nodes = _log(rng, 16, 65536)
        case = {"kind": kind, "nodes": nodes, "frames": _log(rng, 1, max(1, min(65536, 4096 * 16384 // nodes))), "bf16": rng.random() < 0.5,
                "residual": rng.random() < 0.75}
        if kind == "rms_int8":
            case["n_out"] = _log(rng, 16, max(16, min(8192, (1 << 36) // (nodes * case["frames"]))))
        return case
    if kind == "clip_step":
        return {"kind": kind, "sizes": " ".join(str(_log(rng, 1, 1 << 20)) for _ in range(_log(rng, 1, 16)))}
    n_in, n_out = _log(rng, 64, 16384), _log(rng, 16, 16384)
    frames = _log(rng, 1, max(1, min(16384, (1 << 37) // (n_in * n_out), (1 << 26) // max(n_in, n_out))))
    activation = rng.choice(("silu", "gelu", "relu"))
    if kind == "dense":
        return {"kind": kind, "n_in": n_in, "n_out": n_out, "frames": frames, "fp32": rng.random() < 0.25, "bias": rng.random() < 0.5,
                "activation": rng.choice(("none", activation)), "residual": rng.random() < 0.5}
    if kind == "dense_backward":
        return {"kind": kind, "n_in": n_in, "n_out": n_out, "frames": frames}
    if kind == "gated":
        return {"kind": kind, "n_in": n_in, "hidden": n_out, "frames": frames, "activation": activation, "keep": rng.random() < 0.5}
    return {"kind": kind, "n_out": n_in, "hidden": n_out, "frames": frames, "activation": activation}


# ------------------------------------------------------------------------------------------------------------------------------ inputs
def _stride(frames, dtype):
    """Rows of a frame buffer are padded to 32 bytes."""
    per = 8 if dtype == torch.float32 else 16
    return (frames + per - 1) // per * per


def _frame_buffer(values, dtype):
    rows, frames = values.shape
    buf = torch.zeros((rows, _stride(frames, dtype)), dtype=dtype, device=values.device)
    buf[:, :frames] = values.to(dtype)
    return buf


def _weights(values):
    """Rows of bf16 weights on 16-byte boundaries, laid out once when the network is loaded."""
    rows, n = values.shape
    buf = torch.zeros((rows, (n + 7) // 8 * 8), dtype=torch.bfloat16, device=values.device)
    buf[:, :n] = values.to(torch.bfloat16)
    return buf[:, :n]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]

    def normal(*size):
        return torch.randn(size, device="cuda", generator=g)

    def uniform(*size):
        return torch.rand(size, device="cuda", generator=g)

    s = {"case": case, "kind": kind}
    if kind == "clip_step":
        sizes = [int(n) for n in case["sizes"].split()]
        s["params"] = [0.5 + 0.25 * normal(n) for n in sizes]
        s["grads"] = [0.02 * normal(n) * uniform(n) for n in sizes]
        s["m"], s["v"] = [torch.zeros_like(p) for p in s["params"]], [torch.zeros_like(p) for p in s["params"]]
        s["b1"], s["b2"], s["adam"] = BETA1, BETA2, None
        return s
    frames = s["frames"] = case["frames"]
    bf16 = torch.bfloat16
    if kind.startswith("rms"):
        nodes = case["nodes"]
        s["dtype"] = dtype = bf16 if case["bf16"] else torch.float32
        # a residual stream with a spread of each frame's own, and what a layer adds to it
        s["x"] = _frame_buffer(normal(nodes, frames) * (0.5 + 2.0 * uniform(1, frames)), dtype)
        s["r"] = _frame_buffer(normal(nodes, frames) * 0.5, dtype) if case["residual"] else None
        s["gamma"] = 1.0 + 0.2 * normal(nodes)
        if kind == "rms_backward":
            xf = s["x"][:, :frames].double()
            s["rstd"] = (1.0 / torch.sqrt(xf.square().mean(0) + EPS)).float()
            s["dy"] = _frame_buffer(normal(nodes, frames) / frames, dtype)
            s["r"] = _frame_buffer(normal(nodes, frames) / frames, dtype) if case["residual"] else None      # the gradient that arrives by the other path
        if kind == "rms_int8":
            w = normal(case["n_out"], nodes) / math.sqrt(nodes)
            s["w_scale"] = w.abs().amax(1) / 127.0
            s["w"] = torch.zeros((case["n_out"], (nodes + 15) // 16 * 16), dtype=torch.int8, device="cuda")
            s["w"][:, :nodes] = torch.clamp(torch.round(w / s["w_scale"][:, None]), -127, 127).to(torch.int8)
        return s
    if kind == "dense":
        n_in, n_out = case["n_in"], case["n_out"]
        s["dtype"] = dtype = torch.float32 if case["fp32"] else bf16
        s["x"] = _frame_buffer(normal(n_in, frames), bf16)
        s["w"] = _weights(normal(n_out, n_in) / math.sqrt(n_in))
        s["bias"] = 0.1 * normal(n_out) if case["bias"] else None
        s["r"] = _frame_buffer(normal(n_out, frames), dtype) if case["residual"] else None
    elif kind == "dense_backward":
        n_in, n_out = case["n_in"], case["n_out"]
        s["x"] = _frame_buffer(normal(n_in, frames), bf16)
        s["w"] = _weights(normal(n_out, n_in) / math.sqrt(n_in))
        s["dy"] = _frame_buffer(normal(n_out, frames) / frames, bf16)
    elif kind == "gated":
        n_in, hidden = case["n_in"], case["hidden"]
        s["x"] = _frame_buffer(normal(n_in, frames), bf16)
        s["w"] = _weights(normal(2 * hidden, n_in) * (1.5 / math.sqrt(n_in)))       # the gate's rows, then those that it multiplies
    else:
        n_out, hidden = case["n_out"], case["hidden"]
        s["dy"] = _frame_buffer(normal(n_out, frames) / frames, bf16)
        s["w"] = _weights(normal(n_out, hidden) / math.sqrt(hidden))
        s["z"] = _frame_buffer(1.5 * normal(2 * hidden, frames), bf16)
    return s


# ------------------------------------------------------------------------------------------------------------------------------ one pass
def _act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_rms(x, r, gamma, dtype):
    s = x.float() if r is None else (x.float() + r.float()).to(dtype).float()        # what is normalised is what is kept
    rstd = 1.0 / torch.sqrt((s * s).mean(0) + EPS)
    return s, rstd, (s * rstd) * gamma[:, None]


def _plain_rms_int8_dense(x, r, gamma, w, w_scale, dtype):
    s = x.float() if r is None else (x.float() + r.float()).to(dtype).float()
    rstd = 1.0 / torch.sqrt((s * s).mean(0) + EPS)
    t = s * gamma[:, None]
    top = t.abs().amax(0)
    unit = top / torch.full_like(top, 127.0)                 # (a division by a number would be a product with its reciprocal)
    q = torch.where(unit > 0, torch.clamp(torch.round(t / unit), -127, 127), torch.zeros_like(t))
    scale = unit * rstd
    return s, scale, torch.matmul(w.float(), q) * (w_scale[:, None] * scale)


def _plain_rms_backward(s, dy, rstd, gamma, dres):
    xh, g = s * rstd, dy * gamma[:, None]
    ds = rstd * (g - xh * (g * xh).mean(0))
    return (ds if dres is None else ds + dres), (dy * xh).sum(1)


def _plain_step(s):
    norm = torch.sqrt(sum(g.double().square().sum() for g in s["grads"])).float()
    factor = torch.where(norm > MAX_NORM, MAX_NORM / norm, torch.ones_like(norm))
    rate = LR * math.sqrt(1.0 - s["b2"]) / (1.0 - s["b1"])
    s["b1"], s["b2"] = s["b1"] * BETA1, s["b2"] * BETA2
    for p, g, m, v in zip(s["params"], s["grads"], s["m"], s["v"]):
        c = g * factor
        m.add_(RATE1 * (c - m))
        v.add_(RATE2 * (c * c - v))
        p.sub_(rate * m / (torch.sqrt(v) + 1e-7))
    return {"norm": norm, "params": s["params"], "m": s["m"], "v": s["v"]}


def run(state):
    s, case, kind = state, state["case"], state["kind"]
    if kind == "clip_step":
        if own:
            from binarybrain_b200 import ops
            if s["adam"] is None:                            # made once, when training starts
                s["adam"] = ops.Adam(s["params"], s["grads"], lr=LR, beta1=BETA1, beta2=BETA2, max_norm=MAX_NORM)
            norm = s["adam"].step()
            return {"norm": norm, "params": s["params"], "m": s["adam"].m, "v": s["adam"].v}
        return _plain_step(s)
    frames = s["frames"]
    if own:
        from binarybrain_b200 import ops
        if kind == "rms_forward":
            y, kept, rstd = ops.rms_norm_forward(s["x"], frames, gamma=s["gamma"], eps=EPS, residual=s["r"])
            return {"y": y[:, :frames], "s": kept[:, :frames], "rstd": rstd}
        if kind == "rms_int8":
            q, scale, kept = ops.rms_norm_int8(s["x"], frames, gamma=s["gamma"], eps=EPS, residual=s["r"])
            y = ops.int8_dense_forward(q, scale, s["w"], s["w_scale"], n_in=case["nodes"])
            return {"y": y[:, :frames], "s": kept[:, :frames], "scale": scale}
        if kind == "rms_backward":
            ds, dgamma = ops.rms_norm_backward(s["x"], s["dy"], s["rstd"], frames, gamma=s["gamma"], dresidual=s["r"])
            return {"ds": ds[:, :frames], "dgamma": dgamma}
        if kind == "dense":
            y = ops.dense_forward(s["x"], s["w"], frames, bias=s["bias"], activation=case["activation"], residual=s["r"], dtype=s["dtype"])
            return {"y": y[:, :frames]}
        if kind == "dense_backward":
            dx = ops.dense_backward_input(s["dy"], s["w"], frames)
            dW, dbias = ops.dense_backward_weights(s["x"], s["dy"], frames)
            return {"dx": dx[:, :frames], "dW": dW, "dbias": dbias}
        if kind == "gated":
            if case["keep"]:
                h, z = ops.gated_dense_forward(s["x"], s["w"], frames, activation=case["activation"], keep=True)
                return {"h": h[:, :frames], "z": z[:, :frames]}
            return {"h": ops.gated_dense_forward(s["x"], s["w"], frames, activation=case["activation"])[:, :frames]}
        return {"dz": ops.dense_backward_input(s["dy"], s["w"], frames, z=s["z"], activation=case["activation"], gated=True)[:, :frames]}
    bf16 = torch.bfloat16

    def seen(name):
        return None if s[name] is None else s[name][:, :frames]

    if kind == "rms_forward":
        kept, rstd, y = _plain_rms(seen("x"), seen("r"), s["gamma"], s["dtype"])
        return {"y": y.to(s["dtype"]), "s": kept.to(s["dtype"]), "rstd": rstd}
    if kind == "rms_int8":
        kept, scale, y = _plain_rms_int8_dense(seen("x"), seen("r"), s["gamma"], s["w"][:, :case["nodes"]], s["w_scale"], s["dtype"])
        return {"y": y, "s": kept.to(s["dtype"]), "scale": scale}
    if kind == "rms_backward":
        ds, dgamma = _plain_rms_backward(seen("x").float(), seen("dy").float(), s["rstd"], s["gamma"], None if s["r"] is None else seen("r").float())
        return {"ds": ds.to(s["dtype"]), "dgamma": dgamma}
    w = s["w"].float()
    if kind == "dense":
        z = torch.matmul(w, seen("x").float())
        y = _act(z + s["bias"][:, None] if s["bias"] is not None else z, case["activation"])
        return {"y": (y + seen("r").float() if s["r"] is not None else y).to(s["dtype"])}
    if kind == "dense_backward":
        dy = seen("dy").float()
        return {"dx": torch.matmul(w.t(), dy).to(bf16), "dW": torch.matmul(dy, seen("x").float().t()), "dbias": dy.sum(1)}
    if kind == "gated":
        z = torch.matmul(w, seen("x").float())
        h = (_act(z[:case["hidden"]], case["activation"]) * z[case["hidden"]:]).to(bf16)
        return {"h": h, "z": z.to(bf16)} if case["keep"] else {"h": h}
    dh, z, hidden = torch.matmul(w.t(), seen("dy").float()), seen("z").float(), case["hidden"]
    return {"dz": torch.cat([dh * z[hidden:] * _act_grad(z[:hidden], case["activation"]), dh * _act(z[:hidden], case["activation"])]).to(bf16)}


# ------------------------------------------------------------------------------------------------------------------------------ 64 bits
def _curve(z, name):
    """An activation and its slope."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    cdf = torch.special.ndtr(z)
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def exact(case, seed):
    """What run() returns, from the operators' definitions in 64 bits."""
    s, kind = prepare(case, seed), case["kind"]
    if kind == "clip_step":
        norm = sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]) ** 0.5
        factor = min(1.0, MAX_NORM / norm)
        rate = LR * (1 - BETA2) ** 0.5 / (1 - BETA1)
        m = [RATE1 * factor * g.double() for g in s["grads"]]
        v = [RATE2 * (factor * g.double()) ** 2 for g in s["grads"]]
        return {"norm": torch.tensor(norm, dtype=torch.float64), "params": [p.double() - rate * a / (b.sqrt() + 1e-7) for p, a, b in zip(s["params"], m, v)], "m": m, "v": v}
    frames = case["frames"]

    def wide(name):
        return s[name][:, :frames].to(torch.float64)

    if kind in ("rms_forward", "rms_int8"):
        # the sum is a number of 32 bits, kept in the frames' type
        kept = (wide("x") + wide("r")).float().to(s["dtype"]).double() if case["residual"] else wide("x")
        n = kept.shape[0]
        rstd = (torch.einsum("nf,nf->f", kept, kept) / n + EPS).rsqrt()
        if kind == "rms_forward":
            return {"y": kept * (s["gamma"].double()[:, None] * rstd), "s": kept, "rstd": rstd}
        # the weighted numbers, the unit and the quotient are numbers of 32 bits by definition
        t = (kept * s["gamma"].double()[:, None]).float().double()
        unit = (t.abs().amax(0) / 127.0).float().double()
        q = (t / unit).float().double().round().clamp(-127, 127)
        q[:, unit == 0] = 0.0
        return {"y": (s["w"][:, :n].double() @ q) * s["w_scale"].double()[:, None] * (unit * rstd), "s": kept, "scale": unit * rstd}
    if kind == "rms_backward":
        kept, dy, rstd = wide("x"), wide("dy"), s["rstd"].double()
        xh = kept * rstd
        gd = dy * s["gamma"].double()[:, None]
        ds = torch.addcmul(gd, xh, torch.einsum("nf,nf->f", gd, xh) / -kept.shape[0]) * rstd
        return {"ds": ds + wide("r") if case["residual"] else ds, "dgamma": torch.einsum("nf,nf->n", dy, xh)}
    w = s["w"].double()
    if kind == "dense":
        z = w @ wide("x")
        if case["bias"]:
            z += s["bias"].double()[:, None]
        y = _curve(z, case["activation"])[0]
        return {"y": y + wide("r") if case["residual"] else y}
    if kind == "dense_backward":
        return {"dx": torch.einsum("oi,of->if", w, wide("dy")), "dW": torch.einsum("of,if->oi", wide("dy"), wide("x")), "dbias": torch.einsum("of->o", wide("dy"))}
    hidden = case["hidden"]
    if kind == "gated":
        gate, up = w[:hidden] @ wide("x"), w[hidden:] @ wide("x")
        h = _curve(gate, case["activation"])[0] * up
        return {"h": h, "z": torch.cat([gate, up])} if case["keep"] else {"h": h}
    dh = torch.einsum("oh,of->hf", w, wide("dy"))
    value, slope = _curve(wide("z")[:hidden], case["activation"])
    return {"dz": torch.cat([dh * slope * wide("z")[hidden:], dh * value])}


def work(case):
    kind = case["kind"]
    if kind == "clip_step":
        n = sum(int(k) for k in case["sizes"].split())
        return {"bytes": 28 * n, "flops": 16 * n}
    f = case["frames"]
    if kind.startswith("rms"):
        n, e, r = case["nodes"], 2 if case["bf16"] else 4, int(case["residual"])
        if kind == "rms_forward":
            return {"bytes": (2 + 2 * r) * e * n * f + 4 * (n + f), "flops": 5 * n * f}
        if kind == "rms_backward":
            return {"bytes": (3 + r) * e * n * f + 8 * n + 4 * f, "flops": 10 * n * f}
        o = case["n_out"]
        return {"bytes": (1 + 2 * r) * e * n * f + 4 * n + n * o + 4 * o + 4 * o * f + 4 * f, "flops": 2 * n * o * f + 8 * n * f}
    if kind == "dense":
        i, o, e = case["n_in"], case["n_out"], 4 if case["fp32"] else 2
        return {"bytes": 2 * i * f + 2 * i * o + (4 * o if case["bias"] else 0) + (2 if case["residual"] else 1) * e * o * f, "flops": 2 * i * o * f}
    if kind == "dense_backward":
        i, o = case["n_in"], case["n_out"]
        return {"bytes": 4 * i * f + 2 * o * f + 2 * i * o + 4 * i * o + 4 * o, "flops": 4 * i * o * f}
    h = case["hidden"]
    if kind == "gated":
        i = case["n_in"]
        return {"bytes": 2 * i * f + 4 * i * h + (6 if case["keep"] else 2) * h * f, "flops": 4 * i * h * f}
    o = case["n_out"]
    return {"bytes": 2 * o * f + 2 * o * h + 8 * h * f, "flops": 2 * o * h * f}
