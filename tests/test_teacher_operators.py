"""Layer norm, the int8 dense product with its quantisers and the distillation loss against plain implementations in 64 bits.

Tolerances are bounds on the rounding of a computation in 32 bits, written out beside each check: U is half a unit in the last place of 1.0, and the
factors in front of it count the roundings on the way to a value, with room for the order of the sums.  A bf16 result may be off by half of ITS last
place on top of that, 2**-8 of the value.
"""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
BF = 2.0 ** -8
TYPES = [torch.float32, torch.bfloat16]
IDS = ["fp32", "bf16"]


def buffer(values, dtype, layout="rows"):
    """A CUDA frame buffer around `values` [rows, frames] with NaN in its padding.  layout: "rows" padded to 32 bytes, "odd": a stride and a first element
    that no vector access fits."""
    rows, frames = values.shape
    per = 32 // torch.tensor([], dtype=dtype).element_size()
    if layout == "rows":
        t = torch.full((rows, max(per, (frames + per - 1) // per * per)), float("nan"), dtype=dtype)
        t[:, :frames] = values.to(dtype)
        return t.cuda()
    t = torch.full((rows, frames + 5 + frames % 2), float("nan"), dtype=dtype)
    t[:, 1:1 + frames] = values.to(dtype)
    return t.cuda()[:, 1:]


def seen(t, frames):
    return t[:, :frames].double().cpu()


def normal(seed, *size):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(size))


# ------------------------------------------------------------------------------------------------------------------------ layer norm
def norm_case(nodes, frames, dtype, level, seed=0):
    x = (normal(seed, nodes, frames) * (0.25 + normal(seed + 1, 1, frames).abs()) + level * (1 + 0.1 * normal(seed + 2, 1, frames))).to(dtype)
    return x, (1 + 0.2 * normal(seed + 3, nodes)).float(), (0.3 * normal(seed + 4, nodes)).float()


def norm_forward_64(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(0)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(0) + eps)
    xh = (x - mean) * rstd
    g = torch.ones(x.shape[0], dtype=torch.float64) if gamma is None else gamma.double()
    b = torch.zeros(x.shape[0], dtype=torch.float64) if beta is None else beta.double()
    y = xh * g[:, None] + b[:, None]
    # the mean is off by 8 U of the mean magnitude, rstd relatively by twice what that is of a deviation, and the rest are four roundings
    level = x.abs().mean(0)
    off = 8 * U * level
    rel = 16 * U + 2 * (off * rstd) ** 2
    tol = g.abs()[:, None] * (off * rstd + xh.abs() * (rel + 2 * off * rstd)) + 4 * U * (y.abs() + b.abs()[:, None])
    return y, mean, rstd, tol, off, rel


NORM_SIZES = [(1, 1), (1, 37), (2, 8), (3, 1), (7, 5), (31, 33), (64, 9), (70, 100), (129, 257), (420, 512), (1000, 31), (1024, 1), (1025, 130), (3000, 401), (4097, 65),
              (5000, 1), (8192, 70), (9001, 16), (17000, 40), (40000, 3), (65536, 9), (70001, 33), (16, 20000), (100, 9001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("nodes,frames", NORM_SIZES)
def test_layer_norm_forward(nodes, frames, layout, dtype):
    from binarybrain_b200 import ops
    for affine, level in ((True, 0.5), (False, 30.0)):
        x, gamma, beta = norm_case(nodes, frames, dtype, level)
        gamma, beta = (gamma, beta) if affine else (None, None)
        want, mean_w, rstd_w, tol, off, rel = norm_forward_64(x, gamma, beta, 1e-5)
        y = buffer(torch.full((nodes, frames), 7.0), dtype, layout)
        guard = torch.isnan(y).clone()
        got, mean, rstd = ops.layer_norm_forward(buffer(x, dtype, layout), frames, gamma=None if gamma is None else gamma.cuda(),
                                                 beta=None if beta is None else beta.cuda(), y=y)
        assert got is y and torch.equal(torch.isnan(y), guard)                       # the padding is left alone
        if dtype == torch.bfloat16:
            tol = tol + BF * (want.abs() + tol)
        assert (seen(y, frames) - want).abs().sub(tol).max() <= 0
        assert (mean.cpu().double() - mean_w).abs().sub(off + U * mean_w.abs()).max() <= 0
        assert ((rstd.cpu().double() - rstd_w).abs() / rstd_w).sub(rel).max() <= 0


def norm_backward_64(x, dy, mean, rstd, gamma):
    x, dy, m, r = x.double(), dy.double(), mean.double(), rstd.double()
    g = torch.ones(x.shape[0], dtype=torch.float64) if gamma is None else gamma.double()
    xh, gd = (x - m) * r, dy * g[:, None]
    dx = r * (gd - gd.mean(0) - xh * (gd * xh).mean(0))
    # x - m is off by U of it, xh by two roundings more; the sums by 16 U (over the nodes) and 64 U (over the frames) of the sum of magnitudes
    a1, a2 = gd.abs().mean(0), (gd * xh).abs().mean(0)
    tol = r * (4 * U * gd.abs() + 16 * U * a1 + 24 * U * xh.abs() * a2) + 4 * U * dx.abs()
    return (dx, (dy * xh).sum(1), dy.sum(1)), (tol, 64 * U * (dy * xh).abs().sum(1), 64 * U * dy.abs().sum(1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("nodes,frames", NORM_SIZES)
def test_layer_norm_backward(nodes, frames, layout, dtype):
    from binarybrain_b200 import ops
    for affine, level in ((True, 0.5), (False, 5.0)):
        x, gamma, _ = norm_case(nodes, frames, dtype, level)
        gamma = gamma if affine else None
        dy = normal(9, nodes, frames).to(dtype)
        _, mean, rstd, *_ = norm_forward_64(x, None, None, 1e-5)
        mean, rstd = mean.float(), rstd.float()
        want, tol = norm_backward_64(x, dy, mean, rstd, gamma)
        start = [normal(10, nodes).float(), normal(11, nodes).float()]
        dx = buffer(torch.full((nodes, frames), 7.0), dtype, layout)
        guard = torch.isnan(dx).clone()
        args = (buffer(x, dtype, layout), buffer(dy, dtype, layout), mean.cuda(), rstd.cuda(), frames)
        kw = dict(gamma=None if gamma is None else gamma.cuda())
        got = ops.layer_norm_backward(*args, dx=dx, **kw)
        assert torch.equal(torch.isnan(dx), guard)
        again = [s.cuda() for s in start]
        ops.layer_norm_backward(*args, dgamma=again[0], dbeta=again[1], **kw)
        limit = tol[0] + (BF * (want[0].abs() + tol[0]) if dtype == torch.bfloat16 else 0)
        assert (seen(dx, frames) - want[0]).abs().sub(limit).max() <= 0
        for k in (0, 1):
            assert (got[k + 1].cpu().double() - want[k + 1]).abs().sub(tol[k + 1]).max() <= 0
            total = start[k].double() + want[k + 1]
            assert (again[k].cpu().double() - total).abs().sub(tol[k + 1] + U * (total.abs() + tol[k + 1])).max() <= 0


@pytest.mark.gpu
def test_layer_norm_gradient_against_differences():
    """<dx, direction> and <dgamma, direction> against central differences of sum(w * y) in 64 bits."""
    from binarybrain_b200 import ops
    nodes, frames, h = 37, 19, 1e-5
    x, gamma, beta = norm_case(nodes, frames, torch.float32, 0.5)
    w = normal(20, nodes, frames).float()
    y, mean, rstd = ops.layer_norm_forward(buffer(x, torch.float32), frames, gamma=gamma.cuda(), beta=beta.cuda())
    dx, dgamma, dbeta = ops.layer_norm_backward(buffer(x, torch.float32), buffer(w, torch.float32), mean, rstd, frames, gamma=gamma.cuda())
    f = lambda x, g, b: float((w.double() * norm_forward_64(x, g, b, 1e-5)[0]).sum())  # noqa: E731
    for got, arg in ((seen(dx, frames), 0), (dgamma.cpu().double(), 1), (dbeta.cpu().double(), 2)):
        d = normal(21 + arg, *got.shape)
        at = [x.double(), gamma.double(), beta.double()]
        up, down = list(at), list(at)
        up[arg], down[arg] = at[arg] + h * d, at[arg] - h * d
        slope = (f(*up) - f(*down)) / (2 * h)
        # truncation h^2 (third derivatives of order 10), 64 U of the sum of magnitudes for the kernel's own rounding
        assert abs(float((got * d).sum()) - slope) <= 1e-7 + 64 * U * float((got * d).abs().sum()) + 1e-9 * abs(slope)


@pytest.mark.gpu
def test_layer_norm_of_constant_and_of_broken_frames():
    """A frame of one value has no deviation: y = beta.  A NaN or an infinity stays in its own frame."""
    from binarybrain_b200 import ops
    nodes, frames = 300, 12
    x = normal(0, nodes, frames).float()
    x[:, 3] = 2.5
    x[7, 5] = float("nan")
    x[8, 6] = float("inf")
    beta = normal(1, nodes).float()
    y, mean, rstd = ops.layer_norm_forward(buffer(x, torch.float32), frames, beta=beta.cuda())
    y = seen(y, frames)
    assert torch.equal(y[:, 3], beta.double()) and float(mean[3]) == 2.5
    assert torch.isnan(y[:, 5]).all() and torch.isnan(y[:, 6]).all()
    assert torch.isfinite(y[:, [0, 1, 2, 3, 4, 7, 8, 9, 10, 11]]).all()


# ------------------------------------------------------------------------------------------------------------------------ int8
def quantize_32(x):
    """The quantiser's definition in numpy: IEEE divisions in 32 bits, ties to even.  x [nodes, frames] fp32 -> (q [frames, nodes], scale)."""
    top = np.abs(x).max(0)
    finite = np.isfinite(x).all(0)
    with np.errstate(all="ignore"):
        scale = np.where(finite, top / np.float32(127), np.float32(np.nan)).astype(np.float32)
        q = np.rint((x / np.where(scale > 0, scale, np.float32(1))).astype(np.float32))
    q = np.where(scale > 0, np.clip(np.nan_to_num(q), -127, 127), 0)
    return np.ascontiguousarray(q.T).astype(np.int8), scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("nodes,frames", [(1, 1), (1, 40), (5, 3), (16, 8), (17, 31), (127, 1), (128, 33), (130, 64), (1000, 100), (1020, 200), (4096, 1), (5000, 70),
                                          (10000, 17), (33000, 5), (70000, 9), (64, 9001)])
def test_quantize_frames(nodes, frames, layout, dtype):
    from binarybrain_b200 import ops
    x = (normal(0, nodes, frames) * torch.exp(2 * normal(1, 1, frames))).to(dtype)
    if frames > 4:
        x[:, 1] = 0.0
        x[nodes // 2, 2] = float("nan")
        x[nodes - 1, 3] = float("-inf")
        x[:, 4] = torch.round(x[:, 4].float() * 4).to(dtype) / 4                     # ties
        x[0, 4] = 127 * 0.5
    want, scale_w = quantize_32(x.float().numpy())
    q, scale = ops.quantize_int8(buffer(x, dtype, layout), frames)
    assert q.shape == (frames, (nodes + 15) // 16 * 16)
    assert np.array_equal(scale.cpu().numpy(), scale_w, equal_nan=True)
    assert np.array_equal(q[:, :nodes].cpu().numpy(), want) and not q[:, nodes:].any()


@pytest.mark.gpu
def test_quantize_smallest_numbers():
    """Frames whose scale is subnormal or rounds to 0."""
    from binarybrain_b200 import ops
    x = normal(0, 200, 6).float().numpy()
    x *= (np.float32(2.0) ** np.array([-110, -126, -140, -145, -149, -149], dtype=np.float32))
    want, scale_w = quantize_32(x)
    q, scale = ops.quantize_int8(buffer(torch.from_numpy(x), torch.float32), 6)
    assert np.array_equal(scale.cpu().numpy(), scale_w) and np.array_equal(q[:, :200].cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,nodes", [(1, 1), (3, 16), (10, 100), (7, 1000), (1, 131071), (300, 33)])
def test_quantize_channels(rows, nodes):
    from binarybrain_b200 import ops
    W = normal(0, rows, nodes).float()
    W[rows // 2] *= 1e-3
    if rows > 2:
        W[1] = 0.0
    q, scale = ops.quantize_int8_channels(W.cuda())
    want, scale_w = quantize_32(np.ascontiguousarray(W.numpy().T))
    assert np.array_equal(scale.cpu().numpy(), scale_w) and np.array_equal(q[:, :nodes].cpu().numpy(), want) and not q[:, nodes:].any()


def int8_case(n_in, n_out, frames, seed=0, rough=True):
    """Operands with whatever in their padding: the full range of 8 bits, -128 among them, so that sums reach their largest."""
    r = np.random.default_rng(seed)
    pad = (n_in + 15) // 16 * 16
    q, W = r.integers(-128, 128, (frames, pad)).astype(np.int8), r.integers(-128, 128, (n_out, pad)).astype(np.int8)
    if rough:
        W[n_out // 2], q[frames // 2] = -128, -128
    return (torch.from_numpy(q), torch.from_numpy(r.uniform(0.001, 0.1, frames).astype(np.float32)), torch.from_numpy(W),
            torch.from_numpy(r.uniform(0.001, 0.1, n_out).astype(np.float32)), torch.from_numpy(r.standard_normal(n_out).astype(np.float32)))


INT8_SIZES = [(1, 1, 1), (16, 8, 1), (33, 5, 2), (64, 16, 3), (1000, 10, 1), (4096, 257, 1), (1020, 1000, 4), (129, 130, 5), (512, 77, 8), (300, 129, 9), (1024, 128, 16),
              (777, 300, 17), (128, 128, 32), (100, 33, 33), (1020, 1000, 200), (2048, 64, 64), (255, 513, 100), (4099, 130, 65), (64, 1024, 129), (500, 1, 300), (16384, 40, 24),
              (131071, 3, 2), (131071, 20, 40), (640, 700, 513), (272, 2000, 777), (1, 300, 300), (2000, 129, 1025), (130, 5000, 3000), (1000, 4999, 2113), (33, 9001, 1500)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n_in,n_out,frames", INT8_SIZES)
def test_int8_dense(n_in, n_out, frames, dtype):
    from binarybrain_b200 import ops
    q, scale, W, w_scale, bias = int8_case(n_in, n_out, frames)
    acc = (W[:, :n_in].double() @ q[:, :n_in].double().T)                            # exact: below 2**31
    for layout, b in (("rows", bias), ("odd", None)):
        y = buffer(torch.full((n_out, frames), 7.0), dtype, layout)
        guard = torch.isnan(y).clone()
        ops.int8_dense_forward(q.cuda(), scale.cuda(), W.cuda(), w_scale.cuda(), n_in=n_in, bias=None if b is None else b.cuda(), y=y)
        product = acc * w_scale.double()[:, None] * scale.double()
        want = product if b is None else product + b.double()[:, None]
        tol = 3 * U * product.abs() + 2 * U * want.abs()                             # the sum to 32 bits, the two scales, their product with it, the bias
        if dtype == torch.bfloat16:
            tol = tol + BF * (want.abs() + tol)
        assert torch.equal(torch.isnan(y), guard)
        assert (seen(y, frames) - want).abs().sub(tol).max() <= 0


@pytest.mark.gpu
def test_int8_dense_takes_a_frame_without_a_scale():
    """A frame that was not finite is NaN in every node, one of zeros is the bias; the others are as they would be without them."""
    from binarybrain_b200 import ops
    for frames in (6, 150):
        x = normal(0, 200, frames).float()
        x[3, 1], x[:, 2] = float("inf"), 0.0
        W, w_scale = ops.quantize_int8_channels(normal(1, 50, 200).float().cuda())
        bias = normal(2, 50).float()
        y = seen(ops.int8_dense_forward(*ops.quantize_int8(buffer(x, torch.float32), frames), W, w_scale, n_in=200, bias=bias.cuda()), frames)
        assert torch.isnan(y[:, 1]).all() and torch.equal(y[:, 2], bias.double()) and torch.isfinite(y[:, [0, *range(3, frames)]]).all()


# ------------------------------------------------------------------------------------------------------------------------ distillation
def distill_64(z, t, index, temperature, t_lse, weight, batch):
    """Loss per frame, gradient and bounds on their rounding, frame by frame from the definition."""
    C, F = z.shape
    z, t = z.double().numpy(), t.double().numpy()
    dz, tol_dz, loss, tol_loss = np.zeros((C, F)), np.zeros((C, F)), np.zeros(F), np.zeros(F)
    for f in range(F):
        w = 1.0 if weight is None else float(weight[f])
        slots = [k for k in range(t.shape[0]) if 0 <= int(index[k, f]) < C and t[k, f] != -np.inf]
        if w == 0.0 or not slots:
            continue
        zt, tt = z[:, f] / temperature, t[slots, f] / temperature
        cls = index[slots, f].numpy()
        with np.errstate(all="ignore"):
            top = zt.max()
            a = np.where(np.isneginf(zt), 0.0, top - zt)                            # distance from the largest
            e = np.where(np.isneginf(zt), 0.0, np.exp(-a))
            lse = float(t_lse[f]) if t_lse is not None else tt.max() + np.log(np.exp(tt - tt.max()).sum())
            log_p = tt - lse
            p = np.exp(log_p)
            q = np.where(e > 0, e / e.sum(), 0.0)
            log_q = np.where(np.isneginf(zt[cls]), -np.inf, zt[cls] - top - np.log(e.sum()))
            term = np.where(p > 0, p * (log_p - log_q), 0.0)
        target = np.zeros(C)
        np.add.at(target, cls, p)
        g = w / batch * temperature
        dz[:, f] = g * (p.sum() * q - target)
        loss[f] = w * temperature ** 2 * term.sum()
        # exponents are off by a few U of their parts, sums by 32 U of the sum of magnitudes
        rp = (8 + 2 * (np.abs(tt) + abs(lse))) * U
        off = np.zeros(C)
        np.add.at(off, cls, p * rp)
        tol_dz[:, f] = g * (q * (p.sum() * (40 + 4 * a) * U + (p * rp).sum()) + off) + 8 * U * np.abs(dz[:, f])
        with np.errstate(invalid="ignore"):
            far = np.abs(log_p - log_q)
            tol_loss[f] = w * temperature ** 2 * np.where(p > 0, p * (far * (rp + 32 * U) + (np.abs(zt[cls]) + abs(top) + np.log(C) + np.abs(tt) + abs(lse) + 1) * 32 * U), 0.0).sum()
    return dz, loss, tol_dz, tol_loss


def distill_case(C, K, F, dtype, seed=0):
    z = (2 * normal(seed, C, F)).to(dtype)
    teacher = (2.5 * normal(seed + 1, C, F)).to(dtype).float()
    t, index = torch.topk(teacher, K, dim=0)
    weight = torch.from_numpy(np.random.default_rng(seed + 2).uniform(0.25, 2, F).astype(np.float32))
    weight[F // 3] = 0.0
    return z, t.to(dtype), index.to(torch.int32), weight, teacher


def check_distill(z, t, index, F, dtype, temperature, t_lse=None, weight=None, batch=None, layout="rows"):
    from binarybrain_b200 import ops
    C, K = z.shape[0], t.shape[0]
    n = F if batch is None else batch
    dz_w, loss_w, tol_dz, tol_loss = distill_64(z, t, index, temperature, t_lse, weight, n)
    dz = buffer(torch.full((C, F), 7.0), dtype, layout)
    guard = torch.isnan(dz).clone()
    ind = torch.full((K, (F + 7) // 8 * 8 + (layout == "odd")), 1 << 30, dtype=torch.int32)
    ind[:, :F] = index
    got, loss, loss_buf = ops.distillation_loss(buffer(z, dtype, layout), buffer(t, dtype, layout), ind.cuda(), F, temperature=temperature,
                                                t_lse=None if t_lse is None else t_lse.cuda(), weight=None if weight is None else weight.cuda(), batch_size=batch, dz=dz)
    assert torch.equal(torch.isnan(dz), guard)
    dz_g, buf = seen(dz, F).numpy(), loss_buf.cpu().double().numpy()
    loss_w[np.abs(loss_w) > 3.4028235e38] = np.inf                                   # beyond 32 bits
    if dtype == torch.bfloat16:
        tol_dz = tol_dz + BF * (np.abs(dz_w) + tol_dz) + 2.0 ** -134                 # (half of the smallest subnormal)
    tol_dz = tol_dz + 2.0 ** -149
    assert (np.abs(dz_g - dz_w) <= tol_dz).all()
    fin = np.isfinite(loss_w)
    assert np.array_equal(buf[~fin], loss_w[~fin]) and (np.abs(buf - loss_w)[fin] <= tol_loss[fin] + 4 * U * np.abs(loss_w[fin])).all()
    if fin.all():
        assert abs(float(loss) - loss_w.sum() / n) <= (tol_loss.sum() + 8 * U * np.abs(loss_w).sum()) / n
    return dz_g, float(loss), buf


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("classes,top,frames", [(1, 1, 1), (2, 1, 5), (2, 2, 33), (10, 10, 512), (10, 3, 1), (17, 16, 70), (100, 8, 129), (1000, 32, 65), (1000, 1, 8), (1023, 100, 40),
                                                (4097, 64, 33), (10007, 20, 17), (32768, 64, 9), (70000, 7, 3), (3, 2, 9001), (300, 300, 10)])
def test_distillation(classes, top, frames, dtype):
    z, t, index, weight, teacher = distill_case(classes, top, frames, dtype)
    check_distill(z, t, index, frames, dtype, 1.0)
    check_distill(z, t, index, frames, dtype, 3.0, weight=weight, layout="odd")
    check_distill(z, t, index, frames, dtype, 2.0, t_lse=torch.logsumexp(teacher.double() / 2.0, 0).float(), weight=weight, batch=frames * 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("classes,frames", [(40, 24), (5000, 24), (40000, 24)])
def test_distillation_where_a_mask_leaves_little_or_nothing(classes, frames, dtype):
    inf, lowest, K = float("inf"), float(torch.finfo(dtype).min), 6
    z, t, index, weight, _ = distill_case(classes, K, frames, dtype)
    index[2:, 0] = -1                                        # some slots
    index[:, 1] = -1                                         # no slot
    t[:, 2] = -inf                                           # no slot by its logits
    t[1:, 3] = -inf                                          # one slot
    index[3, 4] = classes                                    # the first class that is none
    index[:, 5] = 1 << 30
    index[1:4, 6] = index[0, 6]                              # a class four times
    index[:, 7] = 7                                          # the same everywhere
    z[::2, 8] = -inf                                         # classes taken out, some of them the teacher's
    z[index[:, 9].long(), 9] = -inf                          # all of the teacher's: an infinite loss
    z[:, 10] = -inf                                          # no class left
    z[:, 11] = lowest                                        # all of them as low as the type goes: even
    z[1:, 12] = lowest
    t[1:, 13] = lowest
    z[:, 14], weight[14] = float("nan"), 0.0                 # masked frames may hold anything
    z[0, 15], t[0, 15], weight[15] = inf, float("nan"), 0.0
    z[3, 16], index[:, 16] = float("nan"), -1                # ... and frames without a slot
    dz, loss, buf = check_distill(z, t, index, frames, dtype, 2.0, weight=weight)
    for f in (1, 2, 5, 14, 15, 16):
        assert not dz[:, f].any() and buf[f] == 0.0
    assert np.isposinf(buf[9]) and np.isposinf(buf[10])


@pytest.mark.gpu
def test_distillation_gradient_against_differences():
    """<dz, direction> against central differences of the definition's loss in 64 bits."""
    from binarybrain_b200 import ops
    C, K, F, T, h = 50, 8, 21, 2.0, 1e-4
    z, t, index, weight, _ = distill_case(C, K, F, torch.float32)
    dz, loss, _ = ops.distillation_loss(buffer(z, torch.float32), buffer(t, torch.float32), index.cuda().contiguous(), F, temperature=T, weight=weight.cuda())
    d = normal(5, C, F)
    up, down = (distill_64(z.double() + s * h * d, t, index, T, None, weight, F)[1].sum() / F for s in (1, -1))
    got = seen(dz, F)
    assert abs(float((got * d).sum()) - (up - down) / (2 * h)) <= 1e-7 + 64 * U * float((got * d).abs().sum())


@pytest.mark.gpu
def test_distillation_of_no_frames_and_of_no_slots():
    from binarybrain_b200 import ops
    z = torch.ones((5, 8), device="cuda")
    none = torch.zeros((0, 8), device="cuda"), torch.zeros((0, 8), dtype=torch.int32, device="cuda")
    dz, loss, buf = ops.distillation_loss(z, *none, 7)
    assert not dz[:, :7].any() and float(loss) == 0.0 and not buf.any()
    dz, loss, buf = ops.distillation_loss(z, torch.ones((2, 8), device="cuda"), torch.zeros((2, 8), dtype=torch.int32, device="cuda"), 0)
    assert float(loss) == 0.0 and buf.numel() == 0


# ------------------------------------------------------------------------------------------------------------------------ all of them
def everything(sizes=((64, 40, 30, 8), (700, 300, 333, 20), (3000, 1000, 9, 3), (20000, 200, 50, 16))):
    """One call of every operator and type at some sizes, as a function that makes the calls and returns all that they give."""
    from binarybrain_b200 import ops
    cases = []
    for n, o, F, K in sizes:
        for dtype in TYPES:
            x, gamma, beta = norm_case(n, F, dtype, 0.5, seed=n)
            z, t, index, weight, _ = distill_case(n, K, F, dtype, seed=n)
            W = ops.quantize_int8_channels(normal(n, o, n).float().cuda())
            cases.append((n, F, dtype, *(buffer(v, dtype) for v in (x, normal(n + 1, n, F), z, t)), gamma.cuda(), beta.cuda(), index.cuda(), weight.cuda(), W))

    def run():
        out = []
        for n, F, dtype, x, dy, z, t, gamma, beta, index, weight, W in cases:
            y, mean, rstd = ops.layer_norm_forward(x, F, gamma=gamma, beta=beta)
            dx, dgamma, dbeta = ops.layer_norm_backward(x, dy, mean, rstd, F, gamma=gamma)
            q, scale = ops.quantize_int8(y, F)
            s = ops.int8_dense_forward(q, scale, *W, n_in=n, dtype=dtype)
            dz, loss, buf = ops.distillation_loss(z, t, index, F, temperature=2.0, weight=weight)
            out += [y[:, :F], mean, rstd, dx[:, :F], dgamma, dbeta, q, scale, s[:, :F], dz[:, :F], loss, buf]
        return out
    return run


@pytest.mark.gpu
def test_the_same_bits_every_time_on_every_stream_and_in_a_graph():
    run = everything()
    want = [t.clone() for t in run()]
    for t, w in zip(run(), want):
        assert torch.equal(t, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()                                                      # also makes the stream's scratch
        again = run()
    side.synchronize()
    for t, u, w in zip(got, again, want):
        assert torch.equal(t, w) and torch.equal(u, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = run()
    for _ in range(2):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip(held, want):
            assert torch.equal(t, w)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows 2**30 elements apart: the last of them start beyond 2**31."""
    from binarybrain_b200 import ops
    rows, F = 4, 20
    try:
        big = torch.empty((rows, 1 << 30), dtype=torch.bfloat16, device="cuda")
        out = torch.empty((rows, 1 << 30), dtype=torch.bfloat16, device="cuda")
    except torch.OutOfMemoryError:
        pytest.skip("device memory")
    x = normal(0, rows, F).to(torch.bfloat16).cuda()
    dy = normal(1, rows, F).to(torch.bfloat16).cuda()
    big[:, :F] = x
    want, mean, rstd = ops.layer_norm_forward(x, F)
    ops.layer_norm_forward(big, F, y=out)
    assert torch.equal(out[:, :F], want[:, :F])
    want = ops.layer_norm_backward(x, dy, mean, rstd, F)
    out2 = big.clone()
    got = ops.layer_norm_backward(big, dy, mean, rstd, F, dx=out2)
    assert torch.equal(out2[:, :F], want[0][:, :F]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    del out2
    t, index = torch.ones((2, F), dtype=torch.bfloat16, device="cuda"), torch.arange(2, dtype=torch.int32, device="cuda")[:, None].repeat(1, F) + 2
    want = ops.distillation_loss(x, t, index, F)
    got = ops.distillation_loss(big, t, index, F, dz=out)
    assert torch.equal(out[:, :F], want[0][:, :F]) and torch.equal(got[1], want[1])
    q, scale = ops.quantize_int8(big, F)
    q_w, scale_w = ops.quantize_int8(x, F)
    assert torch.equal(q, q_w) and torch.equal(scale, scale_w)
    W, w_scale = ops.quantize_int8_channels(normal(2, rows, rows).float().cuda())
    want = ops.int8_dense_forward(q, scale, W, w_scale, n_in=rows, dtype=torch.bfloat16)
    ops.int8_dense_forward(q, scale, W, w_scale, n_in=rows, y=out)
    assert torch.equal(out[:, :F], want[:, :F])
    # weights of more than 2**31 bytes, with a frame and with a batch
    del big, out
    n_in, n_out = 65536, 33000
    W = torch.zeros((n_out, n_in), dtype=torch.int8, device="cuda")
    W[:, 5] = (torch.arange(n_out, device="cuda") % 101).to(torch.int8)
    for frames in (1, 40):
        q = torch.zeros((frames, n_in), dtype=torch.int8, device="cuda")
        q[:, 5] = 3
        one = torch.ones(max(n_out, frames), device="cuda")
        y = ops.int8_dense_forward(q, one, W, one, n_in=n_in)
        assert torch.equal(y[:, :frames], (3 * W[:, 5].float())[:, None].expand(n_out, frames))


@pytest.fixture(scope="module")
def native():
    import os
    from binarybrain_b200 import abi
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("library not built")
    from binarybrain_b200 import _native
    return _native


def test_refusals_of_the_library(native):
    """Sizes, strides and pointers that the entry points turn down before anything runs."""
    from binarybrain_b200 import abi
    v = torch.zeros(1024)
    i8 = torch.zeros(1024, dtype=torch.int8)
    a = i8.data_ptr() + (-i8.data_ptr()) % 16
    idx = torch.zeros(64, dtype=torch.int32)
    size, stride, null, large = -2, -3, -1, -6

    def refused(status, name, *args):
        with pytest.raises(abi.BbcuError) as e:
            getattr(native, name)(*args, 0)
        assert e.value.status == status, (name, args)
    for kind in ("fp32", "bf16"):
        norm, grad, quant, loss = (f"bbcu_{kind}_{n}" for n in ("LayerNormalization_Forward", "LayerNormalization_Backward", "QuantizeInt8_Frames", "LossDistillation"))
        dense = f"bbcu_int8_{kind}_DenseAffine_Forward"
        refused(size, norm, v, v, None, None, v, v, 1e-5, 0, 8, 8, 8)
        refused(size, norm, v, v, None, None, v, v, 1e-5, 4, -1, 8, 8)
        refused(size, norm, v, v, None, None, v, v, -1.0, 4, 8, 8, 8)
        refused(size, norm, v, v, None, None, v, v, float("nan"), 4, 8, 8, 8)
        refused(stride, norm, v, v, None, None, v, v, 1e-5, 4, 8, 7, 8)
        refused(stride, norm, v, v, None, None, v, v, 1e-5, 4, 8, 8, 7)
        refused(null, norm, None, v, None, None, v, v, 1e-5, 4, 8, 8, 8)
        refused(null, norm, v, v, None, None, v, None, 1e-5, 4, 8, 8, 8)
        refused(large, norm, v, v, None, None, v, v, 1e-5, 1 << 25, 8, 8, 8)
        refused(size, grad, v, v, v, None, v, v, v, v, 0, -4, 8, 8, 8, 8)
        refused(stride, grad, v, v, v, None, v, v, v, v, 0, 4, 8, 8, 8, 7)
        refused(null, grad, v, None, v, None, v, v, v, v, 0, 4, 8, 8, 8, 8)
        refused(size, quant, v, a, v, 0, 8, 8, 16)
        refused(stride, quant, v, a, v, 20, 8, 8, 16)
        refused(stride, quant, v, a, v, 16, 8, 8, 24)
        refused(stride, quant, v, a + 4, v, 16, 8, 8, 16)
        refused(null, quant, v, a, None, 16, 8, 8, 16)
        refused(size, dense, a, v, a, v, None, v, 0, 4, 8, 16, 16, 8)
        refused(large, dense, a, v, a, v, None, v, 131072, 4, 8, 131072, 131072, 8)
        refused(stride, dense, a, v, a, v, None, v, 17, 4, 8, 16, 32, 8)
        refused(stride, dense, a, v, a + 8, v, None, v, 16, 4, 8, 16, 16, 8)
        refused(stride, dense, a, v, a, v, None, v, 16, 4, 8, 16, 16, 7)
        refused(null, dense, a, None, a, v, None, v, 16, 4, 8, 16, 16, 8)
        refused(size, loss, v, v, v, idx, None, None, v, v, 0.0, 1.0, 1.0, 4, 2, 8, 8, 8, 8, 8)
        refused(size, loss, v, v, v, idx, None, None, v, v, float("nan"), 1.0, 1.0, 4, 2, 8, 8, 8, 8, 8)
        refused(size, loss, v, v, v, idx, None, None, v, v, float("inf"), 1.0, 1.0, 4, 2, 8, 8, 8, 8, 8)
        refused(size, loss, v, v, v, idx, None, None, v, v, 1.0, 1.0, 1.0, 0, 2, 8, 8, 8, 8, 8)
        refused(size, loss, v, v, v, idx, None, None, v, v, 1.0, 1.0, 1.0, 4, -1, 8, 8, 8, 8, 8)
        refused(stride, loss, v, v, v, idx, None, None, v, v, 1.0, 1.0, 1.0, 4, 2, 8, 8, 8, 8, 7)
        refused(null, loss, v, v, v, None, None, None, v, v, 1.0, 1.0, 1.0, 4, 2, 8, 8, 8, 8, 8)
        refused(null, loss, v, v, v, idx, None, None, v, None, 1.0, 1.0, 1.0, 4, 2, 8, 8, 8, 8, 8)
        # no frames, or no outputs: nothing to do, whatever the pointers are
        getattr(native, norm)(None, None, None, None, None, None, 1e-5, 4, 0, 0, 0, 0)
        getattr(native, quant)(None, 0, None, 4, 0, 0, 16, 0)
        getattr(native, dense)(0, None, 0, None, None, None, 4, 0, 8, 16, 16, 8, 0)
        getattr(native, dense)(0, None, 0, None, None, None, 4, 8, 0, 16, 16, 8, 0)
    refused(stride, "bbcu_fp32_QuantizeInt8_Channels", v, a, v, 17, 4, 17, 16)
    refused(size, "bbcu_fp32_QuantizeInt8_Channels", v, a, v, 0, 4, 17, 16)
    refused(null, "bbcu_fp32_QuantizeInt8_Channels", v, None, v, 16, 4, 16, 16)


def test_refusals_of_the_tensor_calls(native):
    """What the calls on tensors turn down: the host's memory first of all (there is no CPU path)."""
    from binarybrain_b200 import ops
    x = torch.zeros((4, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm_forward(x, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm_backward(x, x, x[0], x[0], 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_int8(x, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_int8_channels(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_dense_forward(x.to(torch.int8), x[0], x.to(torch.int8), x[0])
    with pytest.raises(ValueError, match="CUDA"):
        ops.distillation_loss(x, x, x.int(), 8)


@pytest.mark.gpu
def test_refusals_of_the_tensor_calls_on_the_device():
    from binarybrain_b200 import abi, ops
    x, v = torch.zeros((4, 8), device="cuda"), torch.zeros(8, device="cuda")
    q, idx = torch.zeros((8, 16), dtype=torch.int8, device="cuda"), torch.zeros((2, 8), dtype=torch.int32, device="cuda")
    for call in (lambda: ops.layer_norm_forward(x.half(), 8), lambda: ops.layer_norm_forward(x, 9), lambda: ops.layer_norm_forward(x.T, 4), lambda: ops.layer_norm_forward(x[0], 8),
                 lambda: ops.layer_norm_forward(x, 8, gamma=v[:3]), lambda: ops.layer_norm_forward(x, 8, beta=v.double()), lambda: ops.layer_norm_forward(x, 8, y=x[:3]),
                 lambda: ops.layer_norm_forward(x, 8, y=x.bfloat16()), lambda: ops.layer_norm_forward(x, 8, mean=v[:4]),
                 lambda: ops.layer_norm_backward(x, x.bfloat16(), v, v, 8), lambda: ops.layer_norm_backward(x, x[:2], v, v, 8), lambda: ops.layer_norm_backward(x, x, v[:2], v, 8),
                 lambda: ops.layer_norm_backward(x, x, v, v, 8, dgamma=v), lambda: ops.layer_norm_backward(x, x, v, v, 8, dgamma=v[::2], dbeta=v),
                 lambda: ops.quantize_int8(x.int(), 8), lambda: ops.int8_dense_forward(q.float(), v, q, v), lambda: ops.int8_dense_forward(q, v[:3], q, v),
                 lambda: ops.int8_dense_forward(q, v, q, v, y=x), lambda: ops.int8_dense_forward(q[:, ::2], v, q, v),
                 lambda: ops.distillation_loss(x, x[:2].bfloat16(), idx, 8), lambda: ops.distillation_loss(x, x[:2], idx.long(), 8), lambda: ops.distillation_loss(x, x[:3], idx, 8),
                 lambda: ops.distillation_loss(x, x[:2], idx, 8, weight=v[:2]), lambda: ops.distillation_loss(x, x[:2], idx, 8, dz=x[:1])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.distillation_loss(x, x[:2], idx, 8, temperature=0.0), lambda: ops.layer_norm_forward(x, 8, eps=-1.0), lambda: ops.int8_dense_forward(q, v, q, v, n_in=17)):
        with pytest.raises(abi.BbcuError):
            call()


@pytest.mark.gpu
def test_a_lut_network_learns_from_an_int8_teacher():
    """The example: all operators together.  A loss of 100 steps on is well below the first one, the mean divergence from the teacher of a student that knows
    nothing; and every step leaves the numbers that the next one needs finite."""
    import importlib.util
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("distill_int8_teacher", os.path.join(root, "examples", "distill_int8_teacher.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(steps=101, frames=333)
    assert all(math.isfinite(v) for v in losses) and losses[-1] < 0.7 * losses[0]


@pytest.mark.gpu
def test_the_teachers_layers_are_their_operators():
    from binarybrain_b200 import ops
    from binarybrain_b200.teacher import Int8Dense, LayerNormalization, top_logits
    x, dy = (buffer(normal(s, 90, 21), torch.float32) for s in (0, 1))
    norm = LayerNormalization(90, gamma=1.5, beta=0.25)
    y = norm.forward(x, 21)
    want, mean, rstd = ops.layer_norm_forward(x, 21, gamma=norm.gamma, beta=norm.beta)
    assert torch.equal(y[:, :21], want[:, :21])
    for turn in (1, 2):                                                  # the gradients of the weights add up
        if turn == 2:
            norm.forward(x, 21)
        dx = norm.backward(dy)
        dx_w, dgamma, dbeta = ops.layer_norm_backward(x, dy, mean, rstd, 21, gamma=norm.gamma)
        assert torch.equal(dx[:, :21], dx_w[:, :21]) and torch.equal(norm.dgamma, turn * dgamma) and torch.equal(norm.dbeta, turn * dbeta)
    W = normal(2, 30, 90).float().cuda()
    z = Int8Dense(W).forward(y, 21)
    assert torch.equal(z[:, :21], ops.int8_dense_forward(*ops.quantize_int8(y, 21), *ops.quantize_int8_channels(W), n_in=90)[:, :21])
    t, index = top_logits(z, 21, 4)
    assert torch.equal(t[:, :21], torch.gather(z, 0, index[:, :21].long())) and (t[:-1, :21] >= t[1:, :21]).all()
