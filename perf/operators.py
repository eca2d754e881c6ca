"""The operators that put a dense teacher beside a LUT network, as cases that can be timed: layer norm over the nodes of a frame (forward and
backward), the int8 dense product with a scale per frame and per output node, and the distillation loss on a teacher's top logits with its gradient.
All work on frame buffers: [nodes, frame_stride], frames contiguous, fp32 or bf16.

listed() names twelve cases, draw() gives further ones of the same ranges, prepare() makes what a program has in hand before the call, run() is one
pass (elementary torch operations in 32 bits, or with `own` the framework's operators), exact() the same in 64 bits, work() what a pass cannot do without.
"""
import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # normalising one frame of hidden activations, as a server does for a single request
        {"name": "norm_1024x1_bf16", "kind": "norm_forward", "nodes": 1024, "frames": 1, "bf16": True, "affine": True},
        # the outputs of a 3000-node layer on a batch that divides nothing, without a learned scale
        {"name": "norm_3000x5001", "kind": "norm_forward", "nodes": 3000, "frames": 5001, "bf16": False, "affine": False},
        # a wide layer on one GPU's share of a batch
        {"name": "norm_8192x16384", "kind": "norm_forward", "nodes": 8192, "frames": 16384, "bf16": False, "affine": True},
        # the gradient in the training step of a small MLP on a batch of 512
        {"name": "norm_grad_420x512", "kind": "norm_backward", "nodes": 420, "frames": 512, "bf16": False, "affine": True},
        # the widest layers of the regression network
        {"name": "norm_grad_65536x1024", "kind": "norm_backward", "nodes": 65536, "frames": 1024, "bf16": False, "affine": True},
        # a dense layer's activations kept in bf16
        {"name": "norm_grad_4096x16384_bf16", "kind": "norm_backward", "nodes": 4096, "frames": 16384, "bf16": True, "affine": True},
        # a dense layer for a single frame: the weights are what is read
        {"name": "int8_4096x4096x1_bf16", "kind": "int8_dense", "n_in": 4096, "n_out": 4096, "frames": 1, "bf16": True, "bias": True},
        # class scores of a small batch, odd sizes
        {"name": "int8_1020x1000x200", "kind": "int8_dense", "n_in": 1020, "n_out": 1000, "frames": 200, "bf16": False, "bias": True},
        # a large dense layer on a full batch: the tensor cores are what counts
        {"name": "int8_8192x8192x8192_bf16", "kind": "int8_dense", "n_in": 8192, "n_out": 8192, "frames": 8192, "bf16": True, "bias": False},
        # ten classes, all of them known from the teacher, a small batch
        {"name": "distill_10x10x512", "kind": "distill", "classes": 10, "top": 10, "frames": 512, "bf16": False, "temperature": 4.0, "lse": False,
         "weights": False},
        # a thousand classes with 32 kept, odd number of frames, some of them padding
        {"name": "distill_1000x32x10001", "kind": "distill", "classes": 1000, "top": 32, "frames": 10001, "bf16": False, "temperature": 2.0, "lse": True,
         "weights": True},
        # a large vocabulary with 64 kept
        {"name": "distill_32768x64x4096_bf16", "kind": "distill", "classes": 32768, "top": 64, "frames": 4096, "bf16": True, "temperature": 1.0, "lse": False,
         "weights": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm; half of the time rounded to a multiple of eight."""
    n = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return max(lo, n // 8 * 8) if n >= 64 and rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(("norm_forward", "norm_backward", "int8_dense", "distill"))
    bf16 = rng.random() < 0.5
    if kind in ("norm_forward", "norm_backward"):
        nodes = _log(rng, 16, 65536)
        most = 8192 * 16384 if kind == "norm_forward" else 65536 * 1024
        return {"kind": kind, "nodes": nodes, "frames": _log(rng, 1, max(1, min(65536, most // nodes))), "bf16": bf16, "affine": rng.random() < 0.75}
    if kind == "int8_dense":
        n_in, n_out = _log(rng, 64, 16384), _log(rng, 16, 16384)
        frames = _log(rng, 1, min(16384, 8192 ** 3 // (n_in * n_out), 8192 * 8192 // max(n_in, n_out)))
        return {"kind": kind, "n_in": n_in, "n_out": n_out, "frames": frames, "bf16": bf16, "bias": rng.random() < 0.5}
    classes = _log(rng, 2, 65536)
    top = _log(rng, 1, min(128, classes))
    frames = _log(rng, 1, min(65536, 32768 * 4096 // (classes * (1 if bf16 else 2))))
    return {"kind": kind, "classes": classes, "top": top, "frames": frames, "bf16": bf16, "temperature": rng.choice((1.0, 2.0, 4.0)),
            "lse": rng.random() < 0.5, "weights": rng.random() < 0.5}


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


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, frames = case["kind"], case["frames"]
    dtype = torch.bfloat16 if case["bf16"] else torch.float32

    def normal(*size):
        return torch.randn(size, device="cuda", generator=g)

    def uniform(*size):
        return torch.rand(size, device="cuda", generator=g)

    s = {"case": case, "kind": kind, "frames": frames, "dtype": dtype}
    if kind in ("norm_forward", "norm_backward"):
        nodes = case["nodes"]
        # activations with a level and a spread of each frame's own
        x = normal(nodes, frames) * (0.25 + uniform(1, frames)) + 0.5 * normal(1, frames)
        s["x"] = _frame_buffer(x, dtype)
        s["gamma"] = 1.0 + 0.2 * normal(nodes) if case["affine"] else None
        s["beta"] = 0.2 * normal(nodes) if case["affine"] else None
        if kind == "norm_backward":
            xf = s["x"][:, :frames].double()
            s["mean"] = xf.mean(0).float()
            s["rstd"] = (1.0 / torch.sqrt(xf.var(0, unbiased=False) + EPS)).float()
            s["dy"] = _frame_buffer(normal(nodes, frames) / frames, dtype)
    elif kind == "int8_dense":
        n_in, n_out = case["n_in"], case["n_out"]
        s["x"] = _frame_buffer(normal(n_in, frames) * (0.5 + uniform(1, frames)), dtype)
        # weights laid out once, when the network is loaded: a scale per output node, rows padded to 16 bytes
        w = normal(n_out, n_in) / math.sqrt(n_in)
        s["w_scale"] = w.abs().amax(1) / 127.0
        s["w"] = torch.zeros((n_out, (n_in + 15) // 16 * 16), dtype=torch.int8, device="cuda")
        s["w"][:, :n_in] = torch.clamp(torch.round(w / s["w_scale"][:, None]), -127, 127).to(torch.int8)
        s["bias"] = 0.1 * normal(n_out) if case["bias"] else None
        s["n_in"] = n_in
    else:
        classes, top, temperature = case["classes"], case["top"], case["temperature"]
        teacher = 2.5 * normal(classes, frames)
        s["z"] = _frame_buffer(0.6 * teacher + 1.5 * normal(classes, frames), dtype)         # a student part of the way there
        teacher = teacher.to(dtype).float()
        values, index = torch.topk(teacher, top, dim=0)
        s["t"] = _frame_buffer(values, dtype)
        s["index"] = torch.full((top, _stride(frames, torch.float32)), -1, dtype=torch.int32, device="cuda")
        s["index"][:, :frames] = index.to(torch.int32)
        s["t_lse"] = torch.logsumexp(teacher / temperature, 0) if case["lse"] else None
        s["weight"] = (uniform(frames) > 0.0625).float() if case["weights"] else None        # one frame in sixteen is padding
        s["temperature"] = temperature
    return s


# ------------------------------------------------------------------------------------------------------------------------------ one pass
def _plain_norm_forward(x, gamma, beta):
    mean = x.mean(0)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(0) + EPS)
    y = d * rstd
    if gamma is not None:
        y = y * gamma[:, None] + beta[:, None]
    return y, mean, rstd


def _plain_norm_backward(x, dy, mean, rstd, gamma):
    xh = (x - mean) * rstd
    g = dy * gamma[:, None] if gamma is not None else dy
    dx = rstd * (g - g.mean(0) - xh * (g * xh).mean(0))
    return dx, (dy * xh).sum(1), dy.sum(1)


def _plain_int8_dense(x, w, w_scale, bias):
    top = x.abs().amax(0)
    scale = top / torch.full_like(top, 127.0)               # (a division by a number would be a product with its reciprocal)
    q = torch.where(scale > 0, torch.clamp(torch.round(x / scale), -127, 127), torch.zeros_like(x))
    y = torch.matmul(w.float(), q) * (w_scale[:, None] * scale)
    return (y + bias[:, None] if bias is not None else y), scale


def _plain_distill(z, t, index, temperature, t_lse, weight):
    frames = z.shape[1]
    zt = z / temperature
    top = zt.amax(0)
    e = torch.exp(zt - top)
    total = e.sum(0)
    tt = t / temperature
    if t_lse is None:
        t_top = tt.amax(0)
        t_lse = t_top + torch.log(torch.exp(tt - t_top).sum(0))
    log_p = tt - t_lse
    p = torch.exp(log_p)
    log_q = (torch.gather(zt, 0, index) - top) - torch.log(total)
    loss = temperature * temperature * (p * (log_p - log_q)).sum(0)
    dz = (e * (p.sum(0) / total)).scatter_add(0, index, -p) * (temperature / frames)
    if weight is not None:
        loss, dz = loss * weight, dz * weight
    return dz, loss.mean(), loss


def run(state):
    kind, frames, dtype = state["kind"], state["frames"], state["dtype"]
    if own:
        from binarybrain_b200 import ops
        if kind == "norm_forward":
            y, mean, rstd = ops.layer_norm_forward(state["x"], frames, gamma=state["gamma"], beta=state["beta"], eps=EPS)
            return {"y": y[:, :frames], "mean": mean, "rstd": rstd}
        if kind == "norm_backward":
            dx, dgamma, dbeta = ops.layer_norm_backward(state["x"], state["dy"], state["mean"], state["rstd"], frames, gamma=state["gamma"])
            return {"dx": dx[:, :frames], "dgamma": dgamma, "dbeta": dbeta}
        if kind == "int8_dense":
            q, scale = ops.quantize_int8(state["x"], frames)
            y = ops.int8_dense_forward(q, scale, state["w"], state["w_scale"], n_in=state["n_in"], bias=state["bias"], dtype=dtype)
            return {"y": y[:, :frames], "scale": scale}
        dz, loss, loss_buf = ops.distillation_loss(state["z"], state["t"], state["index"], frames, temperature=state["temperature"], t_lse=state["t_lse"],
                                                   weight=state["weight"])
        return {"dz": dz[:, :frames], "loss": loss, "loss_buf": loss_buf}
    if kind == "norm_forward":
        y, mean, rstd = _plain_norm_forward(state["x"][:, :frames].float(), state["gamma"], state["beta"])
        return {"y": y.to(dtype), "mean": mean, "rstd": rstd}
    if kind == "norm_backward":
        dx, dgamma, dbeta = _plain_norm_backward(state["x"][:, :frames].float(), state["dy"][:, :frames].float(), state["mean"], state["rstd"], state["gamma"])
        return {"dx": dx.to(dtype), "dgamma": dgamma, "dbeta": dbeta}
    if kind == "int8_dense":
        y, scale = _plain_int8_dense(state["x"][:, :frames].float(), state["w"][:, :state["n_in"]], state["w_scale"], state["bias"])
        return {"y": y.to(dtype), "scale": scale}
    dz, loss, loss_buf = _plain_distill(state["z"][:, :frames].float(), state["t"][:, :frames].float(), state["index"][:, :frames].long(), state["temperature"],
                                        state["t_lse"], state["weight"])
    return {"dz": dz.to(dtype), "loss": loss, "loss_buf": loss_buf}


# ------------------------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """What run() returns, from the operators' definitions in 64 bits."""
    s, frames = prepare(case, seed), case["frames"]

    def wide(name):
        return s[name][:, :frames].to(torch.float64)

    if case["kind"] == "norm_forward":
        x = wide("x")
        n = x.shape[0]
        mean = x.sum(0) / n
        rstd = ((x - mean).square().sum(0) / n + EPS).rsqrt()
        y = (x - mean) * rstd
        if case["affine"]:
            y = torch.addcmul(s["beta"].double()[:, None], y, s["gamma"].double()[:, None])
        return {"y": y, "mean": mean, "rstd": rstd}
    if case["kind"] == "norm_backward":
        x, dy, mean, rstd = wide("x"), wide("dy"), s["mean"].double(), s["rstd"].double()
        n = x.shape[0]
        x = (x - mean) * rstd
        dgamma, dbeta = torch.einsum("nf,nf->n", dy, x), torch.einsum("nf->n", dy)
        if case["affine"]:
            dy = dy * s["gamma"].double()[:, None]
        c1, c2 = dy.sum(0) / n, torch.einsum("nf,nf->f", dy, x) / n
        return {"dx": (dy - c1 - x * c2) * rstd, "dgamma": dgamma, "dbeta": dbeta}
    if case["kind"] == "int8_dense":
        x, n_in = wide("x"), case["n_in"]
        # the scale and the quotient are numbers of 32 bits by definition
        scale = (x.abs().amax(0) / 127.0).float().double()
        q = (x / scale).float().double().round().clamp(-127, 127)
        q[:, scale == 0] = 0.0
        y = (s["w"][:, :n_in].double() @ q) * s["w_scale"].double()[:, None] * scale
        if case["bias"]:
            y = y + s["bias"].double()[:, None]
        return {"y": y, "scale": scale}
    temperature, index = case["temperature"], s["index"][:, :frames].long()
    log_q = torch.log_softmax(wide("z") / temperature, 0)
    t = wide("t") / temperature
    log_p = t - s["t_lse"].double() if case["lse"] else torch.log_softmax(t, 0)
    p = log_p.exp()
    w = s["weight"].double() if case["weights"] else torch.ones(frames, dtype=torch.float64, device=t.device)
    loss = w * temperature ** 2 * torch.einsum("kf,kf->f", p, log_p - log_q.gather(0, index))
    target = torch.zeros_like(log_q).scatter_add_(0, index, p)
    dz = log_q.exp_().mul_(p.sum(0)).sub_(target).mul_(w * (temperature / frames))
    return {"dz": dz, "loss": loss.sum() / frames, "loss_buf": loss}


def work(case):
    e, frames = 2 if case["bf16"] else 4, case["frames"]
    if case["kind"] == "norm_forward":
        n = case["nodes"]
        return {"bytes": 2 * e * n * frames + (8 * n if case["affine"] else 0) + 8 * frames, "flops": 8 * n * frames}
    if case["kind"] == "norm_backward":
        n = case["nodes"]
        return {"bytes": 3 * e * n * frames + (12 if case["affine"] else 8) * n + 8 * frames, "flops": 16 * n * frames}
    if case["kind"] == "int8_dense":
        i, o = case["n_in"], case["n_out"]
        return {"bytes": e * i * frames + i * o + (8 if case["bias"] else 4) * o + e * o * frames + 4 * frames, "flops": 2 * i * o * frames}
    c, k = case["classes"], case["top"]
    return {"bytes": 2 * e * c * frames + (e + 4) * k * frames + 4 * frames * (1 + case["lse"] + case["weights"]), "flops": 8 * c * frames + 12 * k * frames}
