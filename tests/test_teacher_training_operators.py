"""RMS norm with a residual, the dense product with its epilogue and gradients, the gated block and the clipped step against plain implementations in 64 bits.

Tolerances are bounds on rounding, written out beside each check: U is half a unit in the last place of 1.0 in 32 bits, BF in bf16.  Sums of products on the
tensor cores: a step adds 16 products to the running sum and may cut what does not fit, counted here as four half-units of the sum of all magnitudes a step.
"""
import math

import numpy as np
import pytest
import torch

from test_teacher_operators import BF, IDS, TYPES, U, buffer, normal, seen

BF16 = torch.bfloat16
ACTIVATIONS = ["none", "relu", "gelu", "silu"]


def weights(values, pad=0):
    """bf16 weights in rows on 16-byte boundaries, NaN between them."""
    rows, n = values.shape
    t = torch.full((rows, (n + 7) // 8 * 8 + 8 * pad), float("nan"), dtype=BF16)
    t[:, :n] = values.to(BF16)
    return t.cuda()[:, :n]


def close(got, want, tol, what=""):
    """|got - want| <= tol where want is a number; where it is not, the same non-number."""
    got, want = got.double().cpu(), want.double().cpu()
    tol = tol.cpu() if isinstance(tol, torch.Tensor) else tol
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), what
    assert torch.equal(torch.nan_to_num(got[~finite], nan=12345.0), torch.nan_to_num(want[~finite], nan=12345.0)), what
    excess = ((got - want).abs() - tol)[finite]
    assert excess.numel() == 0 or float(excess.max()) <= 0, (what, float(excess.max()))


# ------------------------------------------------------------------------------------------------------------------------ the dense product
def act64(z, name):
    """Activation, slope, and bounds on what 32 bits make of them: a few roundings, and in exp and erfc those of an argument up to z^2 / 2."""
    if name == "none":
        return z, torch.ones_like(z), 0 * z, 0 * z
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), 0 * z, 0 * z
    if name == "silu":
        p = torch.sigmoid(z)
        y, slope = z * p, p + z * p * (1 - p)
        return y, slope, 16 * U * y.abs(), 32 * U * (p + (z * p * (1 - p)).abs())
    # (through erfc: torch.special.ndtr loses its digits where it is small, 6.66e-16 instead of 6.22e-16 at -8)
    cdf, pdf = 0.5 * torch.special.erfc(z * -math.sqrt(0.5)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    y = z * cdf
    return y, cdf + z * pdf, (16 + 2 * z * z) * U * y.abs(), (16 + 2 * z * z) * U * (cdf + (z * pdf).abs())


def product64(A, B, promoted=False):
    """A B and a bound on its error in 32 bits on the tensor cores; promoted: sums are taken out every 768 of k, 48 steps."""
    A, B = A.double().cuda(), B.double().cuda()
    k = A.shape[1]
    steps = 48 + k / 768 if promoted else k / 16
    return (A @ B).cpu(), ((8 + 4 * steps) * U * (A.abs() @ B.abs())).cpu()


DENSE_SIZES = [(1, 1, 1), (7, 5, 3), (8, 16, 2), (33, 20, 17), (64, 128, 64), (63, 127, 65), (100, 30, 33), (129, 257, 255), (1020, 1000, 200), (2048, 512, 16), (4096, 16, 100),
               (16, 3000, 9), (700, 300, 4097), (5000, 64, 40), (256, 2050, 1030), (1000, 2304, 2047), (16390, 24, 1), (4096, 4096, 1), (300, 40000, 1), (20001, 130, 5)]


def dense_case(K, O, F, seed=0, rows=1):
    x = normal(seed, K, F).to(BF16)
    W = (normal(seed + 1, rows * O, K) / math.sqrt(K)).to(BF16)
    return x, W, (0.5 * normal(seed + 2, rows * O)).float()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("K,O,F", DENSE_SIZES)
def test_dense_forward(K, O, F, layout):
    from binarybrain_b200 import ops
    x, W, bias = dense_case(K, O, F)
    xd, Wd = buffer(x, BF16), weights(W, pad=1)
    for turn, dtype in enumerate((BF16, torch.float32)):
        z, tol = product64(W, x, promoted=dtype == torch.float32)
        for activation, has_bias, has_residual, keep in (("none", False, False, False), ("relu", True, False, True), ("gelu", True, True, False), ("silu", False, True, True)):
            r = normal(5 + turn, O, F).to(dtype)
            y, kept = buffer(torch.full((O, F), 7.0), dtype, layout), buffer(torch.full((O, F), 7.0), BF16, layout)
            guards = torch.isnan(y).clone(), torch.isnan(kept).clone()
            zb, tz = (z + bias.double()[:, None], tol + 2 * U * (z.abs() + bias.abs()[:, None])) if has_bias else (z, tol)
            want, slope, ta, _ = act64(zb, activation)
            ty = 1.2 * tz + ta                                            # no slope is above 1.13
            if has_residual:
                want, ty = want + r.double(), ty + U * (want.abs() + ty + r.double().abs())
            if dtype == BF16:
                ty = ty + BF * (want.abs() + ty)
            got = ops.dense_forward(xd, Wd, F, bias=bias.cuda() if has_bias else None, activation=activation, residual=buffer(r, dtype, layout) if has_residual else None,
                                    y=y, keep=kept if keep else False)
            if keep:
                got, z_got = got
                assert z_got is kept and torch.equal(torch.isnan(kept), guards[1])
                close(seen(kept, F), zb, tz + BF * (zb.abs() + tz), "z")
            assert got is y and torch.equal(torch.isnan(y), guards[0])    # the padding is left alone
            close(seen(y, F), want, ty, (activation, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("K,O,F", DENSE_SIZES)
def test_gated_dense_forward(K, O, F, layout):
    from binarybrain_b200 import ops
    x, W, bias = dense_case(K, O, F, seed=20, rows=2)
    z, tol = product64(W, x)
    for activation, has_bias, keep in (("silu", False, True), ("gelu", True, False), ("none", True, True)):
        y, kept = buffer(torch.full((O, F), 7.0), BF16, layout), buffer(torch.full((2 * O, F), 7.0), BF16, layout)
        guards = torch.isnan(y).clone(), torch.isnan(kept).clone()
        zb, tz = (z + bias.double()[:, None], tol + 2 * U * (z.abs() + bias.abs()[:, None])) if has_bias else (z, tol)
        a, _, ta, _ = act64(zb[:O], activation)
        ta = ta + 1.2 * tz[:O]
        want, ty = a * zb[O:], ta * (zb[O:].abs() + tz[O:]) + a.abs() * tz[O:] + 2 * U * (a * zb[O:]).abs()
        got = ops.gated_dense_forward(buffer(x, BF16), weights(W), F, bias=bias.cuda() if has_bias else None, activation=activation, y=y, keep=kept if keep else False)
        if keep:
            assert got[1] is kept and torch.equal(torch.isnan(kept), guards[1])
            close(seen(kept, F), zb, tz + BF * (zb.abs() + tz), "z")
        assert (got[0] if keep else got) is y and torch.equal(torch.isnan(y), guards[0])
        close(seen(y, F), want, ty + BF * (want.abs() + ty), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("K,O,F", DENSE_SIZES)
def test_dense_backward_input(K, O, F, layout):
    """W [O, K]: dx has K rows and sums over O."""
    from binarybrain_b200 import ops
    _, W, _ = dense_case(K, O, F, seed=30)
    dy, z = normal(33, O, F).to(BF16), (1.5 * normal(34, 2 * K, F)).to(BF16)
    d, tol = product64(W.t(), dy)
    zg, zu = z[:K].double(), z[K:].double()
    for activation, mode in (("none", "plain"), ("relu", "slope"), ("gelu", "slope"), ("silu", "gated"), ("gelu", "gated")):
        rows = 2 * K if mode == "gated" else K
        value, slope, ta, ts = act64(zg, activation)
        if mode == "plain":
            want, tw = d, tol
        elif mode == "slope":
            want, tw = d * slope, 1.2 * tol + (d.abs() + tol) * ts + 2 * U * d.abs()
        else:
            g, tg = d * slope * zu, (1.2 * tol + (d.abs() + tol) * ts + 4 * U * d.abs()) * zu.abs()
            u, tu = d * value, tol * value.abs() + (d.abs() + tol) * ta + 2 * U * (d * value).abs()
            want, tw = torch.cat([g, u]), torch.cat([tg, tu])
        dx = buffer(torch.full((rows, F), 7.0), BF16, layout)
        guard = torch.isnan(dx).clone()
        got = ops.dense_backward_input(buffer(dy, BF16), weights(W), F, z=None if mode == "plain" else buffer(z[:rows], BF16, layout), activation=activation,
                                       gated=mode == "gated", dx=dx)
        assert got is dx and torch.equal(torch.isnan(dx), guard)
        close(seen(dx, F), want, tw + BF * (want.abs() + tw), (activation, mode))


@pytest.mark.gpu
@pytest.mark.parametrize("K,O,F", DENSE_SIZES)
def test_dense_backward_weights(K, O, F):
    from binarybrain_b200 import ops
    x, dy = normal(40, K, F).to(BF16), normal(41, O, F).to(BF16)
    want, tol = product64(dy, x.t(), promoted=True)
    bias, tb = dy.double().sum(1), (8 * math.ceil(F / 2048) + 16) * U * dy.double().abs().sum(1)
    xd, dyd = buffer(x, BF16), buffer(dy, BF16)
    dW, db = ops.dense_backward_weights(xd, dyd, F)
    close(dW, want, tol)
    close(db, bias, tb)
    start = normal(42, O, K).float(), normal(43, O).float()
    for with_bias in (True, False):
        dW, db = start[0].cuda(), start[1].cuda()
        got = ops.dense_backward_weights(xd, dyd, F, dW=dW, dbias=db if with_bias else None)
        assert got[0] is dW and got[1] is (db if with_bias else None)
        close(dW, want + start[0].double(), tol + U * (want.abs() + start[0].double().abs() + tol))
        close(db, bias + start[1].double() if with_bias else start[1], tb + U * (bias.abs() + start[1].abs() + tb) if with_bias else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("K,O,F", [(70, 40, 33), (600, 300, 300), (4096, 256, 1)])
def test_what_is_not_a_number_stays_in_its_frame(K, O, F):
    """Infinities and NaN of one frame reach that frame's outputs and no others, forward and back; those of dy reach the weights' rows they belong to."""
    from binarybrain_b200 import ops
    x, W, _ = dense_case(K, O, F, seed=50)
    bad = F // 2
    x[K // 3, bad], x[K // 2, bad] = float("inf"), float("nan")
    for y in (ops.dense_forward(buffer(x, BF16), weights(W), F), ops.dense_forward(buffer(x, BF16), weights(W), F, dtype=torch.float32),
              ops.gated_dense_forward(buffer(x, BF16), weights(torch.cat([W, W])), F)):
        y = seen(y, F)
        assert torch.isnan(y[:, bad]).all() and torch.isfinite(y[:, torch.arange(F) != bad]).all()
    dy = normal(51, O, F).to(BF16)
    dy[O // 2, bad] = float("nan")
    dx = seen(ops.dense_backward_input(buffer(dy, BF16), weights(W), F), F)
    assert torch.isnan(dx[:, bad]).all() and torch.isfinite(dx[:, torch.arange(F) != bad]).all()
    dW, db = ops.dense_backward_weights(buffer(normal(52, K, F), BF16), buffer(dy, BF16), F)
    assert torch.isnan(dW[O // 2]).all() and torch.isnan(db[O // 2])
    rest = torch.arange(O) != O // 2
    assert torch.isfinite(dW.cpu()[rest]).all() and torch.isfinite(db.cpu()[rest]).all()


@pytest.mark.gpu
def test_activations_at_their_ends():
    """Pre-activations from -200 to 200 through a product with one weight of 1: values, slopes and no NaN."""
    from binarybrain_b200 import ops
    z = torch.cat([torch.linspace(-200, 200, 801), torch.linspace(-12, 12, 801), torch.tensor([0.0, -0.0, 1e-30, -1e-30])]).to(BF16)[None]
    F = z.shape[1]
    one = weights(torch.ones(1, 1))
    for activation in ACTIVATIONS:
        want, slope, ta, ts = act64(z.double(), activation)
        tiny = 2.0 ** -126
        close(seen(ops.dense_forward(buffer(z, BF16), one, F, activation=activation, dtype=torch.float32), F), want, ta + 2 * U * want.abs() + tiny, activation)
        got = seen(ops.dense_backward_input(buffer(torch.ones(1, F), BF16), one, F, z=buffer(z, BF16), activation=activation), F)
        close(got, slope, ts + BF * (slope.abs() + ts) + tiny, activation)


@pytest.mark.gpu
def test_dense_calls_without_frames():
    from binarybrain_b200 import ops
    x, dy, W = torch.zeros((24, 16), dtype=BF16, device="cuda"), torch.zeros((8, 16), dtype=BF16, device="cuda"), weights(torch.ones(8, 24))
    assert ops.dense_forward(x, W, 0).shape == (8, 0) and ops.gated_dense_forward(x, W, 0).shape == (4, 0) and ops.dense_backward_input(dy, W, 0).shape == (24, 0)
    dW, db = ops.dense_backward_weights(x, dy, 0)
    assert not dW.any() and not db.any() and dW.shape == (8, 24)
    dW, db = torch.ones_like(dW), torch.ones_like(db)
    ops.dense_backward_weights(x, dy, 0, dW=dW, dbias=db)
    assert (dW == 1).all() and (db == 1).all()


# frames of odd rows, few frames, one CTA's tiles, tiles whose k is split, pairs; the values of a call with outputs of its own, bit by bit
@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("K,O,F", [(70, 33, 5), (520, 300, 1), (300, 130, 65), (1020, 250, 200), (4096, 100, 40), (640, 700, 3001), (512, 1100, 4100)])
def test_dense_outputs_in_the_place_of_what_they_are_made_of(K, O, F, layout):
    from binarybrain_b200 import ops
    x, W, z = buffer(normal(90, K, F).to(BF16), BF16), ops.dense_weights(normal(91, O, K).cuda() / K ** 0.5), normal(92, 2 * K, F).to(BF16)
    for dtype in (BF16, torch.float32):
        r = normal(93, O, F).to(dtype)
        want = ops.dense_forward(x, W, F, activation="silu", residual=buffer(r, dtype, layout), dtype=dtype, y=buffer(r, dtype, layout))
        y = buffer(r, dtype, layout)
        assert torch.equal(ops.dense_forward(x, W, F, activation="silu", residual=y, dtype=dtype, y=y)[:, :F], want[:, :F])
    dy = buffer(normal(94, O, F).to(BF16), BF16)
    for gated in (False, True):
        zs = z if gated else z[:K]
        want = ops.dense_backward_input(dy, W, F, z=buffer(zs, BF16, layout), activation="gelu", gated=gated, dx=buffer(zs, BF16, layout))
        dz = buffer(zs, BF16, layout)
        assert torch.equal(ops.dense_backward_input(dy, W, F, z=dz, activation="gelu", gated=gated, dx=dz)[:, :F], want[:, :F])


@pytest.mark.gpu
def test_outputs_in_the_place_of_what_is_still_read_are_refused():
    from binarybrain_b200 import ops
    x, W, W2 = torch.zeros((64, 48), dtype=BF16, device="cuda"), ops.dense_weights(torch.zeros(64, 64, device="cuda")), ops.dense_weights(torch.zeros(128, 64, device="cuda"))
    other, z = torch.zeros_like(x), torch.zeros((128, 48), dtype=BF16, device="cuda")
    calls = [lambda: ops.dense_forward(x, W, 48, y=x), lambda: ops.dense_forward(x, W, 48, keep=x), lambda: ops.dense_forward(x, W, 48, y=other, keep=other),
             lambda: ops.dense_forward(x, W, 48, residual=other, keep=other), lambda: ops.gated_dense_forward(x, W2, 48, y=x), lambda: ops.gated_dense_forward(x, W2, 48, y=z[:64], keep=z),
             lambda: ops.dense_backward_input(x, W, 48, dx=x), lambda: ops.rms_norm_forward(x, 48, residual=x, y=other, s=other)]
    for call in calls:
        with pytest.raises(ValueError, match="memory of its own"):
            call()


# ------------------------------------------------------------------------------------------------------------------------ RMS norm
RMS_SIZES = [(1, 1), (1, 37), (2, 8), (3, 1), (7, 5), (31, 33), (64, 9), (70, 100), (129, 257), (420, 512), (1000, 31), (1024, 1), (1025, 130), (3000, 401), (4096, 1), (4097, 65),
             (5000, 1), (8192, 70), (9001, 16), (17000, 40), (40000, 3), (65536, 9), (70001, 33), (16, 20000), (100, 9001), (2500, 4800)]


def rms_case(N, F, dtype, seed=0):
    x = (normal(seed, N, F) * (0.25 + normal(seed + 1, 1, F).abs())).to(dtype)
    return x, normal(seed + 2, N, F).to(dtype), (1 + 0.2 * normal(seed + 3, N)).float()


def rms_64(s, eps):
    s = s.double()
    # squares and their sums: a thread's rows, then joins
    return 1 / torch.sqrt((s * s).mean(0) + eps), (s.shape[0] / 512 + 24) * U


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("N,F", RMS_SIZES)
def test_rms_norm_forward(N, F, layout, dtype):
    from binarybrain_b200 import ops
    x, r, gamma = rms_case(N, F, dtype)
    for has_residual, has_gamma in ((True, True), (False, True), (True, False)):
        s_w = (x.float() + r.float()).to(dtype) if has_residual else x
        rstd_w, rel = rms_64(s_w, 1e-5)
        want = s_w.double() * rstd_w * (gamma.double()[:, None] if has_gamma else 1)
        tol = (rel + 4 * U) * want.abs()
        y, s = buffer(torch.full((N, F), 7.0), dtype, layout), buffer(torch.full((N, F), 7.0), dtype, layout)
        guards = torch.isnan(y).clone(), torch.isnan(s).clone()
        xd = buffer(x, dtype, layout)
        got, kept, rstd = ops.rms_norm_forward(xd, F, gamma=gamma.cuda() if has_gamma else None, residual=buffer(r, dtype, layout) if has_residual else None, y=y,
                                               s=s if has_residual else None)
        assert got is y and torch.equal(torch.isnan(y), guards[0]) and kept is (s if has_residual else xd)
        if has_residual:
            assert torch.equal(torch.isnan(s), guards[1]) and torch.equal(s[:, :F].cpu(), s_w)
        close(rstd, rstd_w, rel * rstd_w)
        close(seen(y, F), want, tol + BF * (want.abs() + tol) if dtype == BF16 else tol)


def int8_of(s, gamma):
    """q and its unit by the definition, in 32 bits, each operation rounded as IEEE says."""
    t = s.float().numpy() * gamma.numpy()[:, None]
    unit = np.abs(t).max(0) / np.float32(127)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(unit > 0, np.clip(np.rint(t / unit), -127, 127), 0)
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(unit)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("N,F", RMS_SIZES)
def test_rms_norm_int8(N, F, layout, dtype):
    from binarybrain_b200 import ops
    x, r, gamma = rms_case(N, F, dtype, seed=4)
    x[:, F // 2] = r[:, F // 2] = 0                                        # a frame of zeros
    for has_residual in (True, False):
        s_w = (x.float() + r.float()).to(dtype) if has_residual else x
        rstd_w, rel = rms_64(s_w, 1e-5)
        q_w, unit = int8_of(s_w, gamma)
        q, scale, s = ops.rms_norm_int8(buffer(x, dtype, layout), F, gamma=gamma.cuda(), residual=buffer(r, dtype, layout) if has_residual else None)
        assert torch.equal(q[:, :N].t().cpu(), q_w) and not q[:, N:].any()
        close(scale, unit.double() * rstd_w, (rel + 2 * U) * unit.double() * rstd_w)
        if has_residual:
            assert torch.equal(s[:, :F].cpu(), s_w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("N,F", RMS_SIZES)
def test_rms_norm_backward(N, F, layout, dtype):
    from binarybrain_b200 import ops
    s, dr, gamma = rms_case(N, F, dtype, seed=8)
    dy = normal(12, N, F).to(dtype)
    rstd = rms_64(s, 1e-5)[0].float()
    r64, xh = rstd.double(), s.double() * rstd.double()
    for has_dr, has_gamma in ((True, True), (False, False)):
        g = dy.double() * gamma.double()[:, None] if has_gamma else dy.double()
        c, ca = (g * xh).mean(0), (g * xh).abs().mean(0)
        want = r64 * (g - xh * c) + (dr.double() if has_dr else 0)
        # the sum over the nodes by its magnitudes, and some roundings of each term
        tol = r64 * (6 * U * g.abs() + xh.abs() * ca * (N / 512 + 32) * U) + 2 * U * want.abs()
        dg, tg = (dy.double() * xh).sum(1), (F / 64 + 32) * U * (dy.double() * xh).abs().sum(1)
        ds = buffer(torch.full((N, F), 7.0), dtype, layout)
        guard = torch.isnan(ds).clone()
        args = (buffer(s, dtype, layout), buffer(dy, dtype, layout), rstd.cuda(), F)
        kw = dict(gamma=gamma.cuda() if has_gamma else None, dresidual=buffer(dr, dtype, layout) if has_dr else None)
        got, dgamma = ops.rms_norm_backward(*args, ds=ds, **kw)
        assert got is ds and torch.equal(torch.isnan(ds), guard)
        close(seen(ds, F), want, tol + BF * (want.abs() + tol) if dtype == BF16 else tol)
        close(dgamma, dg, tg)
        start = normal(13, N).float()
        again = start.cuda()
        ops.rms_norm_backward(*args, dgamma=again, **kw)
        close(again, dg + start.double(), tg + U * (dg.abs() + start.double().abs() + tg))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,F", [(70, 33), (4096, 5), (9001, 300)])
def test_rms_sum_may_take_the_place_of_either_term(N, F, dtype):
    from binarybrain_b200 import ops
    x, r, gamma = rms_case(N, F, dtype, seed=16)
    xd, rd = buffer(x, dtype), buffer(r, dtype)
    y, s, rstd = ops.rms_norm_forward(xd, F, gamma=gamma.cuda(), residual=rd)
    q, scale, _ = ops.rms_norm_int8(xd, F, gamma=gamma.cuda(), residual=rd)
    for where in (0, 1):
        xs, rs = xd.clone(), rd.clone()
        got = ops.rms_norm_forward(xs, F, gamma=gamma.cuda(), residual=rs, s=(xs, rs)[where])
        assert all(torch.equal(a[..., :F], b[..., :F]) for a, b in zip(got, (y, s, rstd)))
        xs, rs = xd.clone(), rd.clone()
        got = ops.rms_norm_int8(xs, F, gamma=gamma.cuda(), residual=rs, s=(xs, rs)[where])
        assert torch.equal(got[0], q) and torch.equal(got[1], scale) and torch.equal(got[2][:, :F], s[:, :F])


@pytest.mark.gpu
def test_rms_frames_that_are_not_numbers_and_frames_beyond_the_range():
    """A NaN or an infinity makes its frame's outputs NaN (an 8-bit frame: zeros with scale NaN) and no others; where squares are beyond the largest number rstd is 0."""
    from binarybrain_b200 import ops
    x = normal(60, 300, 20)
    x[5, 3], x[7, 9], x[:, 12] = float("nan"), float("inf"), 1e30
    xd = buffer(x, torch.float32)
    y, _, rstd = ops.rms_norm_forward(xd, 20)
    y = seen(y, 20)
    q, scale, _ = ops.rms_norm_int8(xd, 20)
    others = [f for f in range(20) if f not in (3, 9, 12)]
    assert torch.isnan(y[:, 3]).all() and torch.isnan(y[7, 9]) and (y[[i for i in range(300) if i != 7], 9] == 0).all() and (y[:, 12] == 0).all()
    assert torch.isfinite(y[:, others]).all() and rstd[12] == 0 and rstd[9] == 0
    assert torch.isnan(scale[[3, 9]]).all() and not q[[3, 9]].any() and torch.isfinite(scale[others]).all() and scale[12] == 0


# frames that are fewer than 16 bytes of a row, or as many: at the numbers of rows where a lane's rounds and the cluster end
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("N,F", [(4, 8), (17, 3), (1025, 2), (4095, 6), (4096, 4), (8193, 1), (16384, 8), (16385, 7), (20000, 5), (32768, 4), (32769, 3), (70003, 2), (131072, 1), (131089, 1)])
def test_rms_norm_of_few_frames(N, F, layout, dtype):
    test_rms_norm_forward(N, F, layout, dtype)
    test_rms_norm_int8(N, F, layout, dtype)
    test_rms_norm_backward(N, F, layout, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [5, 300, 5000])
def test_rms_few_frames_that_are_not_numbers(N, dtype):
    from binarybrain_b200 import ops
    x = normal(61, N, 4).to(dtype)
    x[N - 1, 0], x[N // 2, 2] = float("nan"), float("inf")
    xd = buffer(x, dtype)
    y, _, rstd = ops.rms_norm_forward(xd, 4)
    q, scale, _ = ops.rms_norm_int8(xd, 4)
    y, alone = seen(y, 4), seen(ops.rms_norm_forward(buffer(x[:, 1:2], dtype), 1)[0], 1)
    assert torch.isnan(y[:, 0]).all() and torch.isnan(y[N // 2, 2]) and (y[[n for n in range(N) if n != N // 2], 2] == 0).all() and rstd[2] == 0
    assert torch.isfinite(y[:, [1, 3]]).all() and torch.isnan(scale[[0, 2]]).all() and not q[[0, 2]].any() and torch.isfinite(scale[[1, 3]]).all()
    close(y[:, 1], alone[:, 0].double(), 64 * U * alone[:, 0].double().abs() + (2 * BF * alone[:, 0].double().abs() if dtype == BF16 else 0))


@pytest.mark.gpu
def test_rms_calls_without_frames():
    from binarybrain_b200 import ops
    x = torch.zeros((24, 16), device="cuda")
    assert ops.rms_norm_forward(x, 0, residual=x)[0].shape == (24, 0) and ops.rms_norm_int8(x, 0)[0].shape == (0, 32)
    ds, dgamma = ops.rms_norm_backward(x, x, x[0], 0)
    assert ds.shape == (24, 0) and not dgamma.any()
    dgamma = torch.ones(24, device="cuda")
    ops.rms_norm_backward(x, x, x[0], 0, dgamma=dgamma)
    assert (dgamma == 1).all()


# ------------------------------------------------------------------------------------------------------------------------ clipping
SIZES = [[1], [3, 5, 7], [26880, 4480, 70, 70], [1000003, 17, 65536], list(range(1, 200)), [5, 1 << 20, 0, 9]]


def tensors(sizes, seed, scale=1.0, odd=False):
    """odd: off 16-byte boundaries."""
    return [(scale * normal(seed + i, n + 1)).float().cuda()[1 if odd else 0:][:n] for i, n in enumerate(sizes)]


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("sizes", SIZES, ids=[str(len(s)) + "_" + str(max(s)) for s in SIZES])
def test_gradient_norm_and_clipping(sizes, odd):
    from binarybrain_b200 import ops
    for scale in (1.0, 1e-30, 1e30):
        g = tensors(sizes, 70, scale, odd)
        want = math.sqrt(sum(float(t.double().square().sum()) for t in g))
        clip = ops.GradientNorm(g)
        assert abs(float(clip.norm()) - want) <= 2 * U * want
        before = [t.clone() for t in g]
        assert abs(float(clip.clip_(2 * want)) - want) <= 2 * U * want and all(torch.equal(a, b) for a, b in zip(g, before))
        assert abs(float(clip.clip_(0.25 * want)) - want) <= 2 * U * want
        for a, b in zip(g, before):                                       # the limit and the factor are rounded to 32 bits, then the product
            close(a, 0.25 * b.double(), 4 * U * 0.25 * b.double().abs().cpu() + 2.0 ** -149)


@pytest.mark.gpu
def test_norms_that_are_not_numbers():
    from binarybrain_b200 import ops
    g = tensors([100, 300], 80)
    g[0][7] = float("nan")
    before = [t.clone() for t in g]
    assert math.isnan(float(ops.GradientNorm(g).clip_(0.5))) and torch.equal(g[1], before[1])
    g[0][7] = float("inf")
    assert math.isinf(float(ops.GradientNorm(g).clip_(0.5))) and not g[1].any() and torch.isnan(g[0][7])
    g = tensors([100], 81)
    ops.GradientNorm(g).clip_(0.0)
    assert not g[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("sizes", SIZES, ids=[str(len(s)) + "_" + str(max(s)) for s in SIZES])
def test_clipped_adam(sizes, max_norm, odd):
    """Three steps: the third one's operands have the size that training gives them."""
    from binarybrain_b200 import ops
    p = tensors(sizes, 90, odd=odd)
    g = tensors(sizes, 95, 0.1, odd)
    adam = ops.Adam(p, g, lr=0.01, max_norm=max_norm)
    c1, c2 = float(np.float32(1) - np.float32(0.9)), float(np.float32(1) - np.float32(0.999))
    for step in range(3):
        old = [[t.double().clone() for t in ts] for ts in (p, g, adam.m, adam.v)]
        want = math.sqrt(sum(float(t.square().sum()) for t in old[1]))
        factor = max_norm / want if want > max_norm else 1.0
        lr = 0.01 * math.sqrt(1 - 0.999 ** (step + 1)) / (1 - 0.9 ** (step + 1))
        norm = adam.step() if step < 2 else adam.update()
        assert norm.shape == () and abs(float(norm) - want) <= 2 * U * want
        for i in range(len(p)):
            p0, g0, m0, v0 = (ts[i] for ts in old)
            c = factor * g0
            m, v = m0 + c1 * (c - m0), v0 + c2 * (c * c - v0)
            tm, tv = 6 * U * (m0.abs() + c1 * c.abs()), 10 * U * (v0 + c2 * c * c)
            close(adam.m[i], m, tm.cpu())
            close(adam.v[i], v, tv.cpu())
            root = v.sqrt() + 1e-7
            move = lr * m / root
            # (the root's relative error is half of v's)
            tp = lr * tm / root + move.abs() * (0.5 * tv / v.clamp(min=1e-300) + 8 * U) + U * (p0.abs() + move.abs())
            close(p[i], p0 - move, tp.cpu())
            assert torch.equal(g[i].double(), g0) if step < 2 else not g[i].any()


# tensors as many as a warp, as a quarter of the CTAs and as a table of the kernels' has, and one more; empty ones among them, one larger than a piece
@pytest.mark.gpu
@pytest.mark.parametrize("count", [31, 32, 33, 74, 75, 511, 512, 513, 1300])
def test_clipping_and_the_clipped_step_of_many_tensors(count):
    sizes = [0 if i % 7 == 3 else 1 + 37 * i % 301 for i in range(count)]
    sizes[count // 2] = 20011
    test_gradient_norm_and_clipping(sizes, False)
    test_clipped_adam(sizes, 0.5, False)


@pytest.mark.gpu
def test_a_limit_that_is_not_reached_leaves_the_plain_step():
    from binarybrain_b200 import ops
    sizes = [26880, 4481, 70]
    runs = []
    for limit in (None, 1e30):
        p, g = tensors(sizes, 100), tensors(sizes, 105)
        adam = ops.Adam(p, g, max_norm=limit)
        for _ in range(2):
            norm = adam.step()
        adam.update()
        assert (norm is None) == (limit is None)
        runs.append(p + g + adam.m + adam.v)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


# ------------------------------------------------------------------------------------------------------------------------ all together
def feed_forward_64(x, r, gamma, Wgu, Wd, frames_loss):
    """The block in 64 bits on torch's own gradients: (y, s) of leaves that ask for gradients."""
    s = x + r
    n = s / torch.sqrt((s * s).mean(0) + 1e-5) * gamma[:, None]
    z = Wgu @ n
    h = torch.nn.functional.silu(z[:Wgu.shape[0] // 2]) * z[Wgu.shape[0] // 2:]
    return Wd @ h, s


@pytest.mark.gpu
@pytest.mark.parametrize("N,H,F", [(64, 100, 33), (512, 700, 260)])
def test_a_block_and_its_gradients(N, H, F):
    """Norm, gated block and dense layer with both residual paths, forward and back, against torch's gradients of the same in 64 bits.  What lies between the
    operators is bf16: each of the up to six stored intermediates adds a relative error of 2^-8 / sqrt(3) at most in the 2-norm where errors are independent."""
    from binarybrain_b200.teacher import FeedForward
    block = FeedForward(N, H, generator=torch.Generator(device="cuda").manual_seed(1))
    x, r, dy, ds = (buffer(normal(110 + i, N, F), BF16) for i in range(4))
    y, s = block.forward(x, F, residual=r)
    dx = block.backward(dy, ds)
    leaves = [t[:, :F].double().requires_grad_() for t in (x, r)] + [t.double().requires_grad_() for t in (block.norm.gamma, block.gated.W16, block.dense.W16)]
    y64, s64 = feed_forward_64(*leaves, F)
    (y64 * dy[:, :F].double()).sum().add((s64 * ds[:, :F].double()).sum()).backward()
    bound = 6 * 2.0 ** -8 / math.sqrt(3)
    for got, want in ((y[:, :F], y64), (s[:, :F], s64), (dx[:, :F], leaves[0].grad), (dx[:, :F], leaves[1].grad), (block.norm.dgamma, leaves[2].grad),
                      (block.gated.dW, leaves[3].grad), (block.dense.dW, leaves[4].grad)):
        assert float((got.double() - want.detach()).norm() / want.detach().norm()) <= bound


@pytest.mark.gpu
def test_the_gradient_by_differences():
    """The directional derivative of sum(dy y) along W, from the kernels' fp32 outputs of W + e D and W - e D, is sum(dW D).  W, D and e D are chosen so that
    W +- e D are bf16 numbers: the product is linear in W, and only the sums' rounding is left."""
    from binarybrain_b200 import ops
    K, O, F = 200, 130, 90
    W = torch.randint(-64, 65, (O, K), generator=torch.Generator().manual_seed(0)).double() / 64
    D = torch.randint(-1, 2, (O, K), generator=torch.Generator().manual_seed(1)).double()
    e = 0.25
    x, dy = normal(121, K, F).to(BF16), normal(122, O, F).to(BF16)
    up, down = (ops.dense_forward(buffer(x, BF16), weights(W + sign * e * D), F, dtype=torch.float32)[:, :F].double().cpu() for sign in (1, -1))
    dW, _ = ops.dense_backward_weights(buffer(x, BF16), buffer(dy, BF16), F)
    slope = float((dy.double() * (up - down)).sum() / (2 * e))
    along = float((dW.double().cpu() * D).sum())
    magnitude = float((dy.double().abs() * ((W.abs() + e) @ x.double().abs())).sum()) / e
    assert abs(slope - along) <= 200 * U * magnitude


@pytest.mark.gpu
def test_serving_through_8_bits_is_its_operators():
    from binarybrain_b200 import ops
    from binarybrain_b200.teacher import Int8Dense, RmsNormalization
    norm, dense = RmsNormalization(90, gamma=1.5), Int8Dense(normal(2, 30, 90).float().cuda())
    for F in (1, 21):
        x, r = (buffer(normal(s, 90, F), torch.float32) for s in (0, 1))
        q, scale, s = norm.forward_int8(x, F, residual=r)
        got = dense.forward_int8(q, scale)
        y, s_w = norm.forward(x, F, residual=r)
        assert torch.equal(s[:, :F], s_w[:, :F])
        want = dense.forward(y, F)
        # the two ways quantise the same numbers, up to the roundings of y: some fall on the other side of a half
        assert float((got - want)[:, :F].abs().max()) <= 3 * float((dense.w_scale * 127).max()) * float(scale.max())


@pytest.mark.gpu
def test_a_teacher_is_trained():
    """Two blocks, a dense head and clipped steps: all operators together.  Every step leaves finite numbers, and the gradients are cleared."""
    from binarybrain_b200 import ops
    from binarybrain_b200.teacher import DenseAffine, FeedForward, RmsNormalization, clipped_adam
    N, F, g = 96, 130, torch.Generator(device="cuda").manual_seed(2)
    blocks = [FeedForward(N, 160, generator=g) for _ in range(2)]
    norm, head = RmsNormalization(N), DenseAffine(torch.randn((10, N), device="cuda", generator=g) / 10, bias=torch.zeros(10, device="cuda"), dtype=torch.float32)
    layers = blocks + [norm, head]
    adam = clipped_adam(layers, 1.0, lr=1e-2)
    x, t = buffer(normal(130, N, F), BF16), normal(131, 10, F).float().cuda()
    losses = []
    for _ in range(5):
        y, s = blocks[0].forward(x, F)
        y, s = blocks[1].forward(y, F, residual=s)
        n, s = norm.forward(y, F, residual=s)
        out = head.forward(n, F)
        diff = out[:, :F] - t
        losses.append(float(diff.square().mean()))
        dy = torch.zeros((10, ops.frame_stride(F, BF16)), dtype=BF16, device="cuda")
        dy[:, :F] = diff * (2 / diff.numel())
        ds = norm.backward(head.backward(dy))
        ds = blocks[1].backward(ds, ds)
        blocks[0].backward(ds, ds)
        norm_before = float(adam.update())
        assert math.isfinite(norm_before) and norm_before > 0
        assert not any(grad.any() for layer in layers for _, grad in layer.parameters())
        for layer in blocks + [head]:
            layer.refresh()
    assert all(math.isfinite(v) for v in losses) and losses[-1] < losses[0]


# ------------------------------------------------------------------------------------------------------------------------ streams, graphs, refusals
@pytest.mark.gpu
def test_calls_on_another_stream_and_in_a_graph():
    """A chain of all operators on a side stream, then captured and replayed with other inputs in the same buffers: the bits of the eager calls."""
    from binarybrain_b200 import ops
    K, H, F = 260, 300, 70
    x, r, W, Wd, gamma = buffer(normal(140, K, F), BF16), buffer(normal(141, K, F), BF16), weights(normal(142, 2 * H, K) / 16), weights(normal(143, K, H) / 16), normal(144, K).float().cuda()
    p, g = tensors([1000, 333], 145), tensors([1000, 333], 147)
    clip, adam = ops.GradientNorm(g), ops.Adam(p, g, max_norm=0.5)       # (their tables are made outside of a capture)

    def chain():
        y, s, rstd = ops.rms_norm_forward(x, F, gamma=gamma, residual=r)
        h, z = ops.gated_dense_forward(y, W, F, keep=True)
        out = ops.dense_forward(h, Wd, F, residual=s)
        dz = ops.dense_backward_input(out, Wd, F, z=z, activation="silu", gated=True)
        dW, db = ops.dense_backward_weights(y, dz, F)
        ds, dgamma = ops.rms_norm_backward(s, ops.dense_backward_input(dz, W, F), rstd, F, gamma=gamma, dresidual=out)
        q, scale, _ = ops.rms_norm_int8(x, F, gamma=gamma, residual=r)
        return [t[:, :F] for t in (y, s, h, z, out, dz, ds)] + [rstd, dW, db, dgamma, q, scale, clip.norm()]
    want = [t.clone() for t in chain()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for turn in range(2):
        if turn == 1:
            x.copy_(buffer(normal(150, K, F), BF16))
            want = [t.clone() for t in chain()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    before = [t.clone() for t in p]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = adam.step()
    graph.replay()
    torch.cuda.synchronize()
    assert math.isfinite(float(norm)) and not any(torch.equal(a, b) for a, b in zip(p, before))


@pytest.fixture(scope="module")
def native():
    import os
    from binarybrain_b200 import abi
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("library not built")
    from binarybrain_b200 import _native
    return _native


def test_refusals_of_the_operators(native):
    """Sizes, strides, alignments and null pointers are turned down before anything runs (the addresses below are never read)."""
    from binarybrain_b200 import abi
    a, odd = 1 << 20, (1 << 20) + 2
    size, stride, null, large = -2, -3, -1, -6

    def refused(status, name, *args):
        with pytest.raises(abi.BbcuError) as e:
            getattr(native, name)(*args, 0)
        assert e.value.status == status, (name, args)
    for fwd in ("bbcu_bf16_DenseAffine_Forward", "bbcu_bf16_fp32_DenseAffine_Forward"):
        refused(size, fwd, a, a, None, None, a, None, 0, 0, 8, 8, 8, 8, 0, 8, 0)
        refused(size, fwd, a, a, None, None, a, None, 0, 8, -1, 8, 8, 8, 0, 8, 0)
        refused(size, fwd, a, a, None, None, a, None, 4, 8, 8, 8, 8, 8, 0, 8, 0)
        refused(size, fwd, a, a, None, None, a, None, -1, 8, 8, 8, 8, 8, 0, 8, 0)
        refused(large, fwd, a, a, None, None, a, None, 0, (1 << 27) + 8, 8, 8, (1 << 27) + 8, 8, 0, 8, 0)
        for ws, xs, rs, ys, zs in ((12, 8, 8, 8, 8), (0, 8, 8, 8, 8), (8, 12, 8, 8, 8), (8, 0, 8, 8, 8), (8, 8, 7, 8, 8), (8, 8, 8, 7, 8), (8, 8, 8, 8, 7)):
            refused(stride, fwd, a, a, None, a, a, a, 0, 8, 8, 8, ws, xs, rs, ys, zs)
        refused(stride, fwd, odd, a, None, None, a, None, 0, 8, 8, 8, 8, 8, 0, 8, 0)
        refused(stride, fwd, a, odd, None, None, a, None, 0, 8, 8, 8, 8, 8, 0, 8, 0)
        refused(null, fwd, None, a, None, None, a, None, 0, 8, 8, 8, 8, 8, 0, 8, 0)
        refused(null, fwd, a, a, None, None, None, None, 0, 8, 8, 8, 8, 8, 0, 8, 0)
        getattr(native, fwd)(None, None, None, None, None, None, 0, 8, 8, 0, 8, 8, 0, 8, 0, 0)
    gated, dx, dw = "bbcu_bf16_GatedDense_Forward", "bbcu_bf16_DenseAffine_BackwardInput", "bbcu_bf16_DenseAffine_BackwardWeights"
    refused(size, gated, a, a, None, a, None, 3, 0, 8, 8, 8, 8, 8, 0)
    refused(stride, gated, a, a, None, a, a, 3, 8, 8, 8, 8, 8, 8, 7)
    refused(null, gated, a, None, None, a, a, 3, 8, 8, 8, 8, 8, 8, 8)
    refused(size, dx, a, a, None, a, 0, 0, 8, 0, 8, 8, 8, 0, 8)
    refused(null, dx, a, a, None, a, 3, 1, 8, 8, 8, 8, 8, 8, 8)
    refused(stride, dx, a, a, a, a, 3, 1, 8, 8, 8, 8, 8, 7, 8)
    refused(stride, dx, odd, a, None, a, 0, 0, 8, 8, 8, 8, 8, 0, 8)
    refused(size, dw, a, a, a, a, 0, 0, 8, 8, 8, 8, 8)
    refused(stride, dw, a, odd, a, a, 0, 8, 8, 8, 8, 8, 8)
    refused(stride, dw, a, a, a, a, 0, 8, 8, 8, 8, 8, 7)
    refused(null, dw, a, None, a, a, 0, 8, 8, 8, 8, 8, 8)
    for t in ("fp32", "bf16"):
        fwd, int8, bwd = (f"bbcu_{t}_RmsNormalization_{n}" for n in ("Forward", "QuantizeInt8", "Backward"))
        refused(size, fwd, a, None, None, a, None, a, 1e-5, 0, 8, 8, 0, 0, 8)
        refused(size, fwd, a, None, None, a, None, a, -1.0, 8, 8, 8, 0, 0, 8)
        refused(large, fwd, a, None, None, a, None, a, 1e-5, (1 << 20) + 1, 8, 8, 0, 0, 8)
        refused(stride, fwd, a, None, None, a, None, a, 1e-5, 8, 8, 7, 0, 0, 8)
        refused(stride, fwd, a, a, a, a, None, a, 1e-5, 8, 8, 8, 7, 8, 8)
        refused(stride, fwd, a, a, a, a, None, a, 1e-5, 8, 8, 8, 8, 7, 8)
        refused(null, fwd, a, a, None, a, None, a, 1e-5, 8, 8, 8, 8, 8, 8)
        refused(null, fwd, a, None, None, a, None, None, 1e-5, 8, 8, 8, 0, 0, 8)
        refused(stride, int8, a, None, None, a, a, None, None, 1e-5, 17, 8, 8, 0, 0, 16)
        refused(stride, int8, a, None, None, odd, a, None, None, 1e-5, 16, 8, 8, 0, 0, 16)
        refused(null, int8, a, None, None, a, None, None, None, 1e-5, 16, 8, 8, 0, 0, 16)
        refused(size, bwd, a, a, None, a, None, a, a, 0, 0, 8, 8, 8, 0, 8)
        refused(stride, bwd, a, a, a, a, None, a, a, 0, 8, 8, 8, 8, 7, 8)
        refused(null, bwd, a, a, None, a, None, None, a, 0, 8, 8, 8, 8, 0, 8)
        getattr(native, fwd)(None, None, None, None, None, None, 1e-5, 8, 0, 0, 0, 0, 0, 0)
    refused(size, "bbcu_fp32_GradientNorm", -1, a, a, a)
    refused(null, "bbcu_fp32_GradientNorm", 1, a, a, None)
    refused(null, "bbcu_fp32_GradientNorm", 1, None, a, a)
    refused(size, "bbcu_fp32_GradientClip", 1, a, a, -1.0, a)
    refused(size, "bbcu_fp32_GradientClip", 1, a, a, float("nan"), a)
    refused(null, "bbcu_fp32_GradientClip", 1, a, None, 1.0, a)
    refused(size, "bbcu_fp32_OptimizerAdamClipped", 1, a, a, a, a, a, 0.1, 0.9, 0.99, float("nan"), a, 0)
    refused(null, "bbcu_fp32_OptimizerAdamClipped", 1, a, a, a, a, None, 0.1, 0.9, 0.99, 1.0, a, 0)


def test_refusals_of_the_tensor_calls(native):
    """The host's memory first of all (there is no CPU path)."""
    from binarybrain_b200 import ops
    x, w = torch.zeros((8, 16), dtype=BF16), torch.zeros((8, 8), dtype=BF16)
    for call in (lambda: ops.dense_forward(x, w, 8), lambda: ops.gated_dense_forward(x, w, 8), lambda: ops.dense_backward_input(x, w, 8),
                 lambda: ops.dense_backward_weights(x, x, 8), lambda: ops.rms_norm_forward(x, 8), lambda: ops.rms_norm_int8(x, 8),
                 lambda: ops.rms_norm_backward(x, x, x[0].float(), 8), lambda: ops.GradientNorm([x.float()]), lambda: ops.Adam([x.float()], [x.float()], max_norm=1.0)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for name in ("tanh", 3, []):
        with pytest.raises(ValueError, match="activation"):
            ops.dense_forward(x, w, 8, activation=name)
    with pytest.raises(ValueError, match="at least one"):
        ops.GradientNorm([])
    with pytest.raises(ValueError, match="max_norm"):
        ops.Adam([x.float()], [x.float()], max_norm=-1.0)


@pytest.mark.gpu
def test_refusals_of_the_tensor_calls_on_the_device():
    from binarybrain_b200 import abi, ops
    x, w, v = torch.zeros((8, 16), dtype=BF16, device="cuda"), torch.zeros((8, 8), dtype=BF16, device="cuda"), torch.zeros(16, device="cuda")
    odd = torch.zeros((8, 17), dtype=BF16, device="cuda")
    xf = x.float()
    for call in (lambda: ops.dense_forward(xf, w, 8), lambda: ops.dense_forward(x, w.float(), 8), lambda: ops.dense_forward(x, w, 17), lambda: ops.dense_forward(x[:4], w, 8),
                 lambda: ops.dense_forward(odd[:, 1:], w, 8), lambda: ops.dense_forward(odd, w, 8), lambda: ops.dense_forward(x, odd[:, :8], 8), lambda: ops.dense_forward(x, w.T, 8),
                 lambda: ops.dense_forward(x, w, 8, bias=v[:4]), lambda: ops.dense_forward(x, w, 8, bias=v.double()), lambda: ops.dense_forward(x, w, 8, residual=xf),
                 lambda: ops.dense_forward(x, w, 8, residual=x[:4]), lambda: ops.dense_forward(x, w, 8, y=x[:4]), lambda: ops.dense_forward(x, w, 8, keep=xf),
                 lambda: ops.dense_forward(x, w, 8, dtype=torch.half), lambda: ops.gated_dense_forward(x, w[:7], 8), lambda: ops.gated_dense_forward(x, w, 8, y=x),
                 lambda: ops.gated_dense_forward(x, w, 8, bias=v[:4]), lambda: ops.dense_backward_input(x, w, 8, gated=True),
                 lambda: ops.dense_backward_input(x, w, 8, z=x, activation="silu", gated=True), lambda: ops.dense_backward_input(x, w, 8, z=xf, activation="silu"),
                 lambda: ops.dense_backward_input(x, w, 8, dx=x[:4]), lambda: ops.dense_backward_weights(x, xf, 8), lambda: ops.dense_backward_weights(x, x, 8, dW=v),
                 lambda: ops.dense_backward_weights(x, x, 8, dW=torch.zeros(64, device="cuda")), lambda: ops.dense_backward_weights(x, x, 8, dbias=v),
                 lambda: ops.rms_norm_forward(x.half(), 8), lambda: ops.rms_norm_forward(x, 8, residual=xf), lambda: ops.rms_norm_forward(x, 8, s=x),
                 lambda: ops.rms_norm_forward(x, 8, gamma=v[:4]), lambda: ops.rms_norm_forward(x, 8, y=x[:4]), lambda: ops.rms_norm_int8(x, 8, s=x),
                 lambda: ops.rms_norm_int8(x.int(), 8), lambda: ops.rms_norm_backward(x, xf, v, 8), lambda: ops.rms_norm_backward(x, x, v[:4], 8),
                 lambda: ops.rms_norm_backward(x, x, v, 8, dresidual=x[:4]), lambda: ops.rms_norm_backward(x, x, v, 8, dgamma=v[:4]),
                 lambda: ops.GradientNorm([x]), lambda: ops.GradientNorm([xf.T]), lambda: ops.Adam([xf], [xf[:4]], max_norm=1.0), lambda: ops.Adam([xf], [x], max_norm=1.0),
                 lambda: ops.Adam([xf, xf], [xf], max_norm=1.0), lambda: ops.Adam([xf], [xf], max_norm=1.0), lambda: ops.GradientNorm([v, v]),
                 lambda: ops.GradientNorm([v[:9], v[8:]]), lambda: ops.Adam([v[:8], v[8:]], [xf[0, :8], xf[0, 7:15]], max_norm=1.0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.rms_norm_forward(x, 8, eps=-1.0), lambda: ops.GradientNorm([xf]).clip_(-1.0)):
        with pytest.raises(abi.BbcuError):
            call()


# ------------------------------------------------------------------------------------------------------------------------ scratch, large buffers
@pytest.mark.gpu
def test_host_threads_on_one_stream_with_scratch():
    """Chains of kernels with scratch between them from four host threads on one stream, forty times each: the bits of the same calls by themselves."""
    import threading
    from binarybrain_b200 import ops
    runs = []
    for k, (N, F, dtype) in enumerate([(300, 40, torch.float32), (2500, 1800, BF16), (4096, 1500, torch.float32), (9001, 100, BF16)]):
        s, dr, gamma = rms_case(N, F, dtype, seed=200 + k)
        dy, rstd = normal(210 + k, N, F).to(dtype), rms_64(s, 1e-5)[0].float().cuda()
        s, dr, dy, gamma, clip = buffer(s, dtype), buffer(dr, dtype), buffer(dy, dtype), gamma.cuda(), ops.GradientNorm(tensors([N, 7 * F, 3], 220 + k))

        def run(s=s, dr=dr, dy=dy, gamma=gamma, rstd=rstd, clip=clip, F=F):
            ds, dgamma = ops.rms_norm_backward(s, dy, rstd, F, gamma=gamma, dresidual=dr)
            y, _, r = ops.rms_norm_forward(s, F, gamma=gamma, residual=dr)
            q, scale, _ = ops.rms_norm_int8(s, F, gamma=gamma, residual=dr)
            return ds[:, :F], dgamma, y[:, :F], r, q, scale, clip.norm()
        runs.append(run)
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    stream, failed, start = torch.cuda.current_stream(), [], threading.Barrier(len(runs))

    def work(k):
        try:
            with torch.cuda.stream(stream):
                start.wait(60)
                got = [runs[k]() for _ in range(40)]
            stream.synchronize()
            failed.extend((k, i) for i, g in enumerate(got) if not all(torch.equal(a, b) for a, b in zip(g, want[k])))
        except Exception as e:  # noqa: BLE001 (a thread's exception is the test's)
            failed.append((k, repr(e)))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(runs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.gpu
def test_a_graph_keeps_its_scratch_beside_larger_calls():
    from binarybrain_b200 import ops
    s, dr, gamma = rms_case(2500, 1800, BF16, seed=230)
    dy, rstd = buffer(normal(231, 2500, 1800), BF16), rms_64(s, 1e-5)[0].float().cuda()
    s, dr, gamma, clip = buffer(s, BF16), buffer(dr, BF16), gamma.cuda(), ops.GradientNorm(tensors([5000, 3], 232))
    run = lambda: [*ops.rms_norm_backward(s, dy, rstd, 1800, gamma=gamma, dresidual=dr), *ops.rms_norm_forward(s, 1800, gamma=gamma, residual=dr), clip.norm()]  # noqa: E731
    want = [t.clone() for t in run()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    big = [buffer(normal(240 + i, 9001, 900), BF16) for i in range(3)]
    for _ in range(5):
        graph.replay()
        ops.rms_norm_backward(big[0], big[1], rstd[:900].contiguous(), 900, dresidual=big[2])
        ops.rms_norm_int8(big[0], 900, residual=big[1])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        n = min(1800, a.shape[-1]) if a.dim() == 2 else None
        assert torch.equal(a[:, :n], b[:, :n]) if n else torch.equal(a, b)


@pytest.mark.gpu
def test_buffers_of_more_than_2_31_elements():
    """The last rows and columns, whose offsets do not fit 32 bits, against the same in 64 bits.  (Some 20 GB at a time.)"""
    from binarybrain_b200 import ops
    F = 60000
    g = torch.Generator(device="cuda").manual_seed(3)

    def frames(rows):
        t = torch.empty((rows, F), dtype=BF16, device="cuda")
        for at in range(0, rows, 4096):
            t[at:at + 4096] = torch.randn((min(4096, rows - at), F), device="cuda", generator=g)
        return t
    R, C = slice(-70, None), slice(-300, None)                            # the corner that is looked at
    bound = 2.0 ** -7                                                     # two roundings to bf16 and the sums of 64 products, of values of order 1 (relative and absolute)

    def near(got, want):
        assert float(((got.double() - want).abs() - bound * (1 + want.abs())).max()) <= 0
    K, O = 64, 40000
    x, W, r = frames(K), weights(torch.randn(O, K, generator=torch.Generator().manual_seed(4)) / 8), frames(O)
    y, z = ops.dense_forward(x, W, F, activation="gelu", residual=r, keep=True)
    zw = W[R].double() @ x[:, C].double()
    near(z[R, C], zw)
    near(y[R, C], act64(zw, "gelu")[0] + r[R, C].double())
    dx = ops.dense_backward_input(r, W, F)
    near(dx[:, C] / 64, (W.double().t() @ r[:, C].double()) / 64)
    dW, db = ops.dense_backward_weights(x, r, F)
    close(dW[R], r[R].double() @ x.double().t(), 200 * U * (r[R].double().abs() @ x.double().abs().t()).cpu())
    close(db[R], r[R].double().sum(1), 300 * U * r[R].double().abs().sum(1).cpu())
    del y, z, dx
    kept, rstd = ops.rms_norm_forward(r, F, residual=r)[1:]
    s = 2 * r[:, C].double()
    rw = 1 / torch.sqrt((s * s).mean(0) + 1e-5)
    close(rstd[C], rw, (O / 512 + 24) * U * rw.cpu())
    assert torch.equal(kept[R, C], 2 * r[R, C])
    ds, _ = ops.rms_norm_backward(kept, r, rstd, F)
    xh, dy = kept[:, C].double() * rstd[C].double(), r[:, C].double()
    near(ds[R, C], (rstd[C].double() * (dy - xh * (dy * xh).mean(0)))[R])
    del ds
    q, scale, _ = ops.rms_norm_int8(kept, F)
    unit = (kept[:, C].float().abs().amax(0) / torch.full((300,), 127.0, device="cuda"))
    assert torch.equal(q[C, R], torch.round(kept[R, C].float() / unit).clamp(-127, 127).to(torch.int8).t())
    del q, kept, r
    H = 20000
    W = weights(torch.randn(2 * H, K, generator=torch.Generator().manual_seed(5)) / 8)
    h, z = ops.gated_dense_forward(x, W, F, keep=True)
    g64, u64 = W[H - 70:H].double() @ x[:, C].double(), W[R].double() @ x[:, C].double()
    near(z[H - 70:H, C], g64)
    near(z[R, C], u64)
    near(h[R, C] / 4, act64(g64, "silu")[0] * u64 / 4)
    dy, Wd = frames(K), weights(torch.randn(K, H, generator=torch.Generator().manual_seed(6)) / 8)
    dz = ops.dense_backward_input(dy, Wd, F, z=z, activation="silu", gated=True)
    d = Wd[:, R].double().t() @ dy[:, C].double()
    zg, zu = z[H - 70:H, C].double(), z[R, C].double()
    value, slope, _, _ = act64(zg, "silu")
    near(dz[H - 70:H, C] / 8, d * slope * zu / 8)
    near(dz[R, C] / 8, d * value / 8)


FIRST_CALLS = """
import torch
from binarybrain_b200 import ops
K, O = 512, 384
for F in (1, 300, 5000):
    def frames(rows):
        return torch.randn(rows, ops.frame_stride(F, torch.bfloat16), device="cuda").to(torch.bfloat16)
    x, dy, z, rstd, W = frames(K), frames(O), frames(2 * K), torch.rand(F, device="cuda"), ops.dense_weights(torch.randn(O, K, device="cuda"))
    norm = ops.GradientNorm([torch.randn(1000, device="cuda"), torch.randn(33, device="cuda")])
    calls = [lambda: ops.dense_forward(x, W, F, activation="gelu"), lambda: ops.gated_dense_forward(x, W, F), lambda: ops.dense_backward_weights(x, dy, F),
             lambda: ops.dense_backward_input(dy, W, F, z=z, activation="silu", gated=True), lambda: ops.rms_norm_forward(x, F, residual=x), lambda: ops.rms_norm_int8(x, F),
             lambda: ops.rms_norm_backward(x, x, rstd, F), norm.norm]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [call() for call in calls]
    graph.replay()
    for a, b in zip(captured, [call() for call in calls]):
        for s, t in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
            # (what lies in a frame buffer's padding is not written; rows of integers and weights have none)
            framed = s is not None and s.dim() == 2 and s.dtype == torch.bfloat16
            assert s is None or torch.equal(s[:, :F] if framed else s, t[:, :F] if framed else t)
print("same")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_may_be_captured():
    """Nothing that a first call sets up stands in the way of a capture, and a replay has the numbers of a call."""
    import subprocess
    import sys
    from pathlib import Path
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("same"), done.stderr[-2000:]
