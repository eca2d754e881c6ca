"""The teacher's operators where their arithmetic is strained: nodes far from all others, levels, spreads near the ends of 32 bits, frames of one value.  As
in test_teacher_operators.py, U is half a unit in the last place of 1.0 and the factors in front of it count roundings."""
import numpy as np
import pytest
import torch

from test_teacher_operators import BF, IDS, TYPES, U, buffer, normal


def far_nodes(nodes, frames, dtype):
    """Frames of N(0, 1) in which single nodes, the first ones among them, lie far from all others; a frame of each kind in turn."""
    x = normal(nodes, nodes, frames)
    for f in range(frames):
        kind = f % 8
        if kind < 3:
            x[0, f] = (100.0, 1000.0, 30000.0)[kind]
        elif kind == 3:
            x[-1, f] = 30000.0
        elif kind == 4:
            x[nodes // 2, f] = -1000.0
        elif kind == 5:
            x[:16, f] = 1000.0
        elif kind == 6:
            x[::97, f] = 1e4
        else:
            x[:, f] += torch.arange(nodes) * 0.1
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("nodes,frames,layout", [(300, 19, "odd"), (300, 19, "rows"), (4096, 24, "rows"), (5000, 40, "rows"), (5000, 9600, "rows"), (8192, 70, "odd"), (16384, 200, "rows"),
                                                 (65536, 9, "rows"), (65536, 9, "odd"), (1 << 20, 8, "rows")])
def test_layer_norm_of_frames_with_far_nodes(nodes, frames, layout, dtype):
    from binarybrain_b200 import ops
    x = far_nodes(nodes, min(frames, 200), dtype)
    x = x[:, torch.arange(frames) % x.shape[1]]
    y, mean, rstd = ops.layer_norm_forward(buffer(x, dtype, layout), frames, eps=1e-5)
    x = x.cuda().double()
    mean_w = x.mean(0)
    rstd_w = 1 / torch.sqrt((x - mean_w).square().mean(0) + 1e-5)
    # A value may be in 16 partial sums of about its own size.  A thread adds up to 128 squares one after the other, then 8 such sums, and they are joined in
    # 16 steps; half of that is left of it in a square root.  The mean's error counts by its square.
    off = 16 * U * x.abs().mean(0)
    rel = 80 * U + 2 * (off * rstd_w) ** 2
    assert ((mean.double() - mean_w).abs() - off - U * mean_w.abs()).max() <= 0
    assert ((rstd.double() - rstd_w).abs() / rstd_w - rel).max() <= 0
    want = (x - mean_w) * rstd_w
    tol = off * rstd_w + want.abs() * (rel + 2 * off * rstd_w) + 4 * U * want.abs()
    if dtype == torch.bfloat16:
        tol = tol + BF * (want.abs() + tol)
    assert ((y[:, :frames].double() - want).abs() - tol).max() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,layout", [(300, "odd"), (9001, "rows"), (9001, "odd")])
def test_layer_norm_of_broken_frames_beside_others(nodes, layout):
    """A NaN or an infinity stays in its own frame, wherever it is, also where the rows are read twice."""
    from binarybrain_b200 import ops
    frames = 24
    x = normal(1, nodes, frames).float()
    for f, (n, v) in enumerate(((0, "nan"), (nodes - 1, "nan"), (0, "inf"), (7, "-inf"), (nodes - 1, "inf"), (nodes // 2, "-inf"))):
        x[n, 2 * f] = float(v)
    y, mean, rstd = ops.layer_norm_forward(buffer(x, torch.float32, layout), frames)
    assert torch.isnan(y[:, 0:12:2]).all() and torch.isnan(rstd[0:12:2]).all()
    keep = [1, 3, 5, 7, 9, *range(11, frames)]
    want = x[:, keep].double()
    want = (want - want.mean(0)) / torch.sqrt(want.var(0, unbiased=False) + 1e-5)
    assert (y[:, keep].double().cpu() - want).abs().max() <= 64 * U * want.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("nodes,frames,layout", [(7, 5, "rows"), (300, 19, "rows"), (1000, 31, "rows"), (3000, 40, "rows"), (4096, 24, "rows"), (300, 19, "odd"), (9001, 16, "rows")])
def test_layer_norm_of_small_and_of_large_spreads(nodes, frames, layout, dtype):
    """Spreads at which rstd^3, and rstd^2 of the widest, is outside of 32 bits: the same digits as at 1, forward without eps and backward."""
    from binarybrain_b200 import ops
    from test_teacher_operators import norm_backward_64, norm_case, norm_forward_64
    for scale in (2.0 ** -58, 2.0 ** -45, 2.0 ** 45, 2.0 ** 55):
        x, gamma, beta = norm_case(nodes, frames, dtype, 0.5)
        x = (x.double() * scale).to(dtype)
        want, mean_w, rstd_w, tol, off, rel = norm_forward_64(x, gamma, beta, 0.0)
        y, mean, rstd = ops.layer_norm_forward(buffer(x, dtype, layout), frames, gamma=gamma.cuda(), beta=beta.cuda(), eps=0.0)
        if dtype == torch.bfloat16:
            tol = tol + BF * (want.abs() + tol)
        assert ((y[:, :frames].double().cpu() - want).abs() - tol).max() <= 0
        assert ((mean.cpu().double() - mean_w).abs() - off - U * mean_w.abs()).max() <= 0
        assert ((rstd.cpu().double() - rstd_w).abs() / rstd_w - rel).max() <= 0
        dy = normal(9, nodes, frames).to(dtype)
        mean, rstd = mean_w.float(), rstd_w.float()
        (dx_w, dgamma_w, dbeta_w), tol = norm_backward_64(x, dy, mean, rstd, gamma)
        dx, dgamma, dbeta = ops.layer_norm_backward(buffer(x, dtype, layout), buffer(dy, dtype, layout), mean.cuda(), rstd.cuda(), frames, gamma=gamma.cuda())
        limit = tol[0] + (BF * (dx_w.abs() + tol[0]) if dtype == torch.bfloat16 else 0)
        assert ((dx[:, :frames].double().cpu() - dx_w).abs() - limit).max() <= 0
        assert ((dgamma.cpu().double() - dgamma_w).abs() - tol[1]).max() <= 0
        assert ((dbeta.cpu().double() - dbeta_w).abs() - tol[2]).max() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("nodes", [1, 2, 3, 5, 15, 30, 60, 61, 100, 255, 300, 333, 500, 777, 1001, 1500, 2047, 2999, 3333, 4000, 4096, 4097, 5001, 9001, 20011, 70001])
def test_layer_norm_of_frames_of_one_value(nodes, layout, dtype):
    """No deviation, at any level and size: mean = the value, rstd = 1 / sqrt(eps), y = beta, each in every bit."""
    from binarybrain_b200 import ops
    levels = torch.tensor([2.5, 0.1, 1000.1, -7.7, 1e-30, -3e38, 12345.678, 0.0, 1 / 3, 6e4, -1e-3]).to(dtype)
    x = levels.expand(nodes, -1).clone()
    beta = normal(1, nodes).float().to(dtype).float()
    for eps in (1e-5, 1e-12):
        y, mean, rstd = ops.layer_norm_forward(buffer(x, dtype, layout), len(levels), beta=beta.cuda(), eps=eps)
        assert torch.equal(mean.cpu(), levels.float())
        assert (rstd.cpu().numpy() == np.float32(1) / np.sqrt(np.float32(eps))).all()
        assert torch.equal(y[:, :len(levels)].float().cpu(), beta[:, None].expand(-1, len(levels)))


@pytest.mark.gpu
def test_many_slots():
    """As many slots as a call takes, read once and by passes."""
    from test_teacher_operators import check_distill, distill_case
    for classes, frames in ((600, 9), (1500, 5), (9000, 6)):
        for dtype in (torch.float32, torch.bfloat16):
            z, t, index, weight, _ = distill_case(classes, 512, frames, dtype)
            index[1::7, 2] = index[0, 2]
            check_distill(z, t, index, frames, dtype, 2.0, weight=weight)


@pytest.mark.gpu
def test_layer_norm_backward_without_frames():
    from binarybrain_b200 import ops
    x, v = torch.ones((300, 8), device="cuda"), torch.zeros(0, device="cuda")
    dx, dgamma, dbeta = ops.layer_norm_backward(x, x, v, v, 0)
    assert not dgamma.any() and not dbeta.any()
    dgamma, dbeta = torch.full((300,), 2.0, device="cuda"), torch.full((300,), 3.0, device="cuda")
    ops.layer_norm_backward(x, x, v, v, 0, dgamma=dgamma, dbeta=dbeta)
    assert (dgamma == 2.0).all() and (dbeta == 3.0).all()


class Elsewhere(torch.Tensor):
    """A tensor of no memory that says it is on a CUDA device, for checks that end before any memory is asked for."""

    @staticmethod
    def __new__(cls, size, dtype, device):
        return torch.Tensor._make_wrapper_subclass(cls, size, dtype=dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError


def on_device(index):
    """x [4, 8], v [8], rows of 8-bit integers and indices"""
    device = torch.device("cuda", index)
    return (Elsewhere((4, 8), torch.float32, device), Elsewhere((8,), torch.float32, device), Elsewhere((8, 16), torch.int8, device), Elsewhere((4, 8), torch.int32, device))


def test_tensors_of_two_devices_are_refused():
    pytest.importorskip("binarybrain_b200._native")
    from binarybrain_b200 import ops
    (x, v, q, i), (x1, v1, q1, i1) = on_device(0), on_device(1)
    for call in (lambda: ops.layer_norm_forward(x, 8, gamma=v1), lambda: ops.layer_norm_forward(x, 8, beta=v1), lambda: ops.layer_norm_backward(x, x1, v, v, 8),
                 lambda: ops.layer_norm_backward(x, x, v, v, 8, gamma=v1), lambda: ops.layer_norm_backward(x, x, v1, v, 8), lambda: ops.int8_dense_forward(q, v, q1, v),
                 lambda: ops.int8_dense_forward(q, v1, q, v), lambda: ops.distillation_loss(x, x1, i, 8), lambda: ops.distillation_loss(x, x, i1, 8),
                 lambda: ops.distillation_loss(x, x, i, 8, weight=v1), lambda: ops.distillation_loss(x1, x1, i1, 8, t_lse=v)):
        with pytest.raises(ValueError, match="cuda:[01], as the others of the call"):
            call()


@pytest.mark.gpu
def test_tensors_of_another_than_the_current_device_are_refused():
    from binarybrain_b200 import ops
    x, v, q, i = on_device(torch.cuda.current_device() + 1)
    for call in (lambda: ops.layer_norm_forward(x, 8), lambda: ops.quantize_int8(x, 8), lambda: ops.distillation_loss(x, x, i, 8), lambda: ops.quantize_int8_channels(x)):
        with pytest.raises(ValueError, match="the current device is cuda:"):
            call()


def test_the_int8_product_refuses_more_than_it_counts():
    """Output nodes and frames within a tile of 2^31 would be no tiles at all; nothing is run or asked for (the pointers are made up)."""
    native = pytest.importorskip("binarybrain_b200._native")
    from binarybrain_b200 import abi
    at, most = 1 << 20, 1 << 30
    for kind in ("fp32", "bf16"):
        for nodes, frames in ((4, most + 1), (4, 2 ** 31 - 1), (most + 1, 8), (2 ** 31 - 1, 1), (2 ** 31 - 100, 2)):
            with pytest.raises(abi.BbcuError) as e:
                getattr(native, f"bbcu_int8_{kind}_DenseAffine_Forward")(at, at, at, at, None, at, 16, nodes, frames, 16, 16, frames, 0)
            assert e.value.status == -6, (nodes, frames)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,level", [(torch.float32, 2.0 ** 13), (torch.float32, -2.0 ** 16), (torch.bfloat16, 2.0 ** 7)], ids=["fp32+", "fp32-", "bf16"])
@pytest.mark.parametrize("classes,top,frames", [(10, 10, 40), (3000, 32, 33), (9000, 64, 20)])
def test_the_level_of_a_teachers_logits_does_not_count(classes, top, frames, dtype, level):
    """Without a sum over all of its classes a teacher's probabilities are those of its slots: the same in every bit whatever is added to all of a frame's
    logits, as long as the logits take it exactly."""
    from binarybrain_b200 import ops
    step = 1.0 if dtype == torch.bfloat16 else 2.0 ** -6
    t = torch.from_numpy(np.random.default_rng(classes).integers(0, int(8 / step), (top, frames)) * step)
    index = torch.argsort(normal(1, classes, frames), 0)[:top].to(torch.int32).cuda()
    z = buffer(normal(2, classes, frames), dtype)
    assert torch.equal((t + level).to(dtype).double() - level, t)
    for temperature in (1.0, 3.0):
        want = ops.distillation_loss(z, buffer(t, dtype), index, frames, temperature=temperature)
        got = ops.distillation_loss(z, buffer(t + level, dtype), index, frames, temperature=temperature)
        assert torch.equal(got[0][:, :frames], want[0][:, :frames]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n_in,n_out,frames", [(1000, 300, 1), (1000, 130, 5), (16384, 40, 24), (1024, 700, 333), (1024, 2048, 2048)])
def test_int8_product_of_scales_whose_product_is_no_number_of_32_bits(n_in, n_out, frames, dtype):
    from binarybrain_b200 import ops
    from test_teacher_operators import int8_case
    q, scale, W, w_scale, bias = int8_case(n_in, n_out, frames)
    W[0] = 0                                                                         # sums of 0 stay 0 where the scales' product is beyond the largest number
    acc = W[:, :n_in].cuda().double() @ q[:, :n_in].cuda().double().T                # exact: below 2**31
    for by_w, by_q in ((-85, -45), (-45, -85), (70, 45)):
        ws, s = (w_scale * 2.0 ** by_w).cuda(), (scale * 2.0 ** by_q).cuda()
        b = (bias.double() * 2.0 ** max(-126, by_w + by_q + 20)).float().cuda() if by_w + by_q < 0 else bias.cuda()
        y = ops.int8_dense_forward(q.cuda(), s, W.cuda(), ws, n_in=n_in, bias=b, dtype=dtype)[:, :frames].double()
        product = acc * ws.double()[:, None] * s.double()
        want = product + b.double()[:, None]
        tol = 3 * U * product.abs() + 2 * U * want.abs() + 2.0 ** -149
        if dtype == torch.bfloat16:
            tol = tol + BF * (want.abs() + tol) + 2.0 ** -134                        # (half of the smallest subnormal)
        inside = want.abs() < 2.0 ** 127
        assert ((y - want).abs() - tol)[inside].max() <= 0 and torch.equal(y[0], b[0].to(dtype).double().expand(frames))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("nodes,layout", [(40, "rows"), (300, "rows"), (300, "odd"), (3000, "rows"), (9001, "rows"), (9001, "odd"), (70001, "rows")])
def test_layer_norm_of_squares_beyond_the_largest_number(nodes, layout, dtype):
    """Deviations of finite values whose squares are infinite: rstd is 0, the mean a number, y = beta, and the gradient 0."""
    from binarybrain_b200 import ops
    frames, lowest = 12, float(torch.finfo(dtype).min)
    x = normal(nodes, nodes, frames)
    x[0, 0] = x[-1, 1] = x[nodes // 2, 2] = x[nodes // 3, 3] = lowest
    x[0, 4] = x[-1, 5] = -lowest
    x[7, 6] = 1e30
    x[:, 7] *= 1e25
    x[::2, 8] *= 1e22
    x = x.to(dtype)
    beta = normal(1, nodes).float().to(dtype).float()
    y, mean, rstd = ops.layer_norm_forward(buffer(x, dtype, layout), frames, beta=beta.cuda())
    assert not rstd[:9].any() and (rstd[9:] > 0.5).all()
    want = x.double().mean(0)
    assert ((mean.cpu().double() - want).abs() - 16 * U * x.double().abs().mean(0) - U * want.abs()).max() <= 0
    assert torch.equal(y[:, :9].float().cpu(), beta[:, None].expand(-1, 9))
    dx, dgamma, dbeta = ops.layer_norm_backward(buffer(x, dtype, layout), buffer(normal(2, nodes, frames), dtype, layout), mean, rstd, frames)
    assert not dx[:, :9].any() and torch.isfinite(dx[:, 9:frames]).all() and torch.isfinite(dgamma).all()
