"""Layers of the bf16 teacher as a network strings them together: which gradient a layer takes and returns, what it keeps, and what it refuses.

The refusals come before any operator, so that they are tested without a GPU too, on operators that only give buffers of the right shape.
"""
import math
import types

import pytest
import torch

from test_teacher_operators import buffer, normal

BF16 = torch.bfloat16
TYPES = [torch.float32, BF16]


@pytest.fixture
def shapes_only(monkeypatch):
    """The operators of `teacher` replaced by ones that return zeros of the shapes that the real ones return, and note their calls."""
    from binarybrain_b200 import ops, teacher
    calls = []

    def frames(rows, x):
        return torch.zeros((rows, x.shape[1]), dtype=BF16)

    def dense_forward(x, W, n, activation=None, keep=False, **kw):
        calls.append("dense_forward")
        y = frames(W.shape[0], x)
        return (y, frames(W.shape[0], x)) if keep else y

    def gated_dense_forward(x, W, n, keep=False, **kw):
        calls.append("gated_dense_forward")
        y = frames(W.shape[0] // 2, x)
        return (y, frames(W.shape[0], x)) if keep else y

    def dense_backward_input(dy, W, n, z=None, activation=None, gated=False, dx=None):
        calls.append(("dense_backward_input", None if z is None else tuple(z.shape), activation, gated))
        return frames(W.shape[1] * (2 if gated else 1), dy)

    def dense_backward_weights(x, dy, n, dW=None, dbias=None):
        calls.append("dense_backward_weights")
        return dW, dbias

    def rms_norm_forward(x, n, gamma=None, eps=1e-5, residual=None, y=None, s=None, rstd=None):
        return frames(x.shape[0], x), x if residual is None else frames(x.shape[0], x), torch.ones(n)

    def rms_norm_backward(s, dy, rstd, n, gamma=None, dresidual=None, ds=None, dgamma=None):
        return frames(s.shape[0], s), dgamma
    plain = types.SimpleNamespace(dense_weights=ops.dense_weights, dense_forward=dense_forward, gated_dense_forward=gated_dense_forward, dense_backward_input=dense_backward_input,
                                  dense_backward_weights=dense_backward_weights, rms_norm_forward=rms_norm_forward, rms_norm_backward=rms_norm_backward)
    monkeypatch.setattr(teacher, "ops", plain)
    return calls


def test_a_gradient_of_y_is_refused_where_that_of_z_is_needed(shapes_only):
    from binarybrain_b200.teacher import DenseAffine, GatedDense
    x, dy = torch.zeros((8, 16), dtype=BF16), torch.zeros((12, 16), dtype=BF16)
    for activation in ("relu", "gelu", "silu"):
        lower, upper = DenseAffine(torch.zeros(12, 8), activation=activation), DenseAffine(torch.zeros(8, 12))
        h = lower.forward(x, 16)
        upper.forward(h, 16)
        del shapes_only[:]
        with pytest.raises(ValueError, match="gradient of y"):
            lower.backward(dy)
        g = upper.backward(x)                                             # without `below`: the gradient of y
        with pytest.raises(ValueError, match="gradient of y"):
            lower.backward(g)
        assert "dense_backward_weights" in shapes_only and shapes_only.count("dense_backward_weights") == 1       # nothing was added to the refused layer's gradients
        upper.forward(lower.forward(x, 16), 16)
        assert lower.backward(upper.backward(x, below=lower)).shape == (8, 16)
        assert ("dense_backward_input", (12, 16), activation, False) in shapes_only
        lower.forward(x, 16)                                              # a new pass: the layer above has not been asked yet
        with pytest.raises(ValueError, match="gradient of y"):
            lower.backward(dy)
        lower.backward(dy, of_z=True)
    for plain in (DenseAffine(torch.zeros(12, 8)), DenseAffine(torch.zeros(12, 8), activation="none")):
        plain.forward(x, 16, residual=dy)
        plain.backward(dy)
    gate = GatedDense(torch.zeros(24, 8))
    gate.forward(x, 16)
    gate.backward(torch.zeros((24, 16), dtype=BF16))


def test_a_refused_backward_pass_of_the_layer_above_gives_nothing(shapes_only, monkeypatch):
    from binarybrain_b200 import teacher
    lower, upper = teacher.DenseAffine(torch.zeros(12, 8), activation="relu"), teacher.DenseAffine(torch.zeros(8, 12))
    x, dy = torch.zeros((8, 16), dtype=BF16), torch.zeros((12, 16), dtype=BF16)
    upper.forward(lower.forward(x, 16), 16)

    def refuses(*args, **kw):
        raise ValueError("dx: expected another shape")
    with monkeypatch.context() as m:
        m.setattr(teacher.ops, "dense_backward_input", refuses)
        with pytest.raises(ValueError, match="another shape"):
            upper.backward(x, below=lower)
    with pytest.raises(ValueError, match="gradient of y"):
        lower.backward(dy)
    lower.backward(upper.backward(x, below=lower))


def test_a_residual_beside_an_activation_is_for_serving(shapes_only):
    from binarybrain_b200.teacher import DenseAffine
    x, r = torch.zeros((8, 16), dtype=BF16), torch.zeros((12, 16), dtype=BF16)
    lower, upper = DenseAffine(torch.zeros(12, 8), activation="relu"), DenseAffine(torch.zeros(8, 12))
    upper.forward(lower.forward(x, 16, residual=r), 16)
    with pytest.raises(ValueError, match="residual"):
        upper.backward(x, below=lower)
    upper.forward(lower.forward(x, 16), 16)
    lower.backward(upper.backward(x, below=lower))


def test_a_pass_that_is_not_for_training_keeps_nothing(shapes_only):
    from binarybrain_b200.teacher import DenseAffine, FeedForward, GatedDense, RmsNormalization
    x = torch.zeros((8, 16), dtype=BF16)
    norm, block = RmsNormalization(8, device="cpu"), FeedForward(8, 12, device="cpu")
    for layer, passes in ((norm, lambda train: norm.forward(x, 16, train=train)), (block, lambda train: block.forward(x, 16, residual=x, train=train))):
        with pytest.raises(RuntimeError, match="nothing is kept"):
            layer.backward(x)
        passes(True)
        assert layer.backward(x, x).shape == (8, 16)
        with pytest.raises(RuntimeError, match="nothing is kept"):        # it has been used up
            layer.backward(x)
        passes(True)
        passes(False)                                                     # an evaluation between a training pass and its backward pass
        del shapes_only[:]
        with pytest.raises(RuntimeError, match="nothing is kept"):
            layer.backward(x)
        assert not shapes_only
    assert all(layer._saved is None for layer in (norm, block.norm, block.gated, block.dense))
    lower, gate, upper = DenseAffine(torch.zeros(12, 8), activation="relu"), GatedDense(torch.zeros(24, 8)), DenseAffine(torch.zeros(8, 12))
    for below in (lower, gate):
        upper.forward(below.forward(x, 16, train=False), 16)
        del shapes_only[:]
        with pytest.raises(RuntimeError, match="nothing is kept"):
            upper.backward(x, below=below)
        assert not shapes_only                                            # no gradient has been added to


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("K,H,O,F", [(64, 100, 40, 33), (300, 513, 260, 500)])
def test_two_dense_layers_and_their_gradients(K, H, O, F, activation):
    """activation(W1 x + b1), W2 of it + b2 + residual, against torch's gradients of the same in 64 bits.  Three stored intermediates (z, h and dz) lie between, each with a
    relative error of 2^-8 / sqrt(3) in the 2-norm where errors are independent, and the output is rounded once more.  (A rounded z keeps its sign, so that relu's
    slope is the same.)"""
    from binarybrain_b200.teacher import DenseAffine
    lower = DenseAffine((normal(1, H, K) / math.sqrt(K)).float().cuda(), bias=(0.5 * normal(2, H)).float().cuda(), activation=activation)
    upper = DenseAffine((normal(3, O, H) / math.sqrt(H)).float().cuda(), bias=(0.5 * normal(4, O)).float().cuda())
    x, r, dy = buffer(normal(5, K, F), BF16), buffer(normal(6, O, F), BF16), buffer(normal(7, O, F), BF16)
    y = upper.forward(lower.forward(x, F), F, residual=r)
    dx = lower.backward(upper.backward(dy, below=lower))
    leaves = [t.double().requires_grad_() for t in (x[:, :F], lower.W16, lower.bias, upper.W16, upper.bias)]
    z = leaves[1] @ leaves[0] + leaves[2][:, None]
    h = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": lambda t: 0.5 * t * torch.special.erfc(-t * math.sqrt(0.5))}[activation](z)
    y64 = leaves[3] @ h + leaves[4][:, None] + r[:, :F].double()
    (y64 * dy[:, :F].double()).sum().backward()
    bound = 4 * 2.0 ** -8 / math.sqrt(3)
    for got, want in ((y[:, :F], y64), (dx[:, :F], leaves[0].grad), (lower.dW, leaves[1].grad), (lower.dbias, leaves[2].grad), (upper.dW, leaves[3].grad), (upper.dbias, leaves[4].grad)):
        assert float((got.double() - want.detach()).norm() / want.detach().norm()) <= bound


@pytest.mark.gpu
def test_the_norm_does_not_overwrite_what_it_returns_as_s():
    """Without a residual s is x, which the backward pass reads: y in its place is refused, and x is left as it was."""
    from binarybrain_b200 import ops
    from binarybrain_b200.teacher import RmsNormalization
    for N, F, dtype in ((70, 33, BF16), (300, 5, torch.float32)):
        x = buffer(normal(20, N, F), dtype)
        before = x.clone()
        for call in (lambda: ops.rms_norm_forward(x, F, y=x), lambda: RmsNormalization(N).forward(x, F, y=x)):
            with pytest.raises(ValueError, match="memory of its own"):
                call()
        assert torch.equal(x[:, :F], before[:, :F])
        assert ops.rms_norm_forward(x, F, y=torch.empty_like(x))[1] is x


@pytest.mark.gpu
def test_outputs_that_reach_into_other_buffers_are_refused():
    """Wherever they begin: a row further on, a column further on, or the same memory in rows of another length."""
    from binarybrain_b200 import ops
    flat = torch.zeros(4096 * 64, dtype=BF16, device="cuda")
    rows = lambda first, n, stride=48, column=0: flat[first * 48 + column:].as_strided((n, 48 - column if stride == 48 else 48), (stride, 1))  # noqa: E731
    W, W2 = ops.dense_weights(torch.zeros(64, 64, device="cuda")), ops.dense_weights(torch.zeros(128, 64, device="cuda"))
    x, r, far, rstd = rows(0, 64), rows(100, 64), rows(500, 64), torch.ones(48, device="cuda")
    f = 48
    calls = [lambda: ops.dense_forward(x, W, f, y=rows(1, 64)), lambda: ops.dense_forward(x, W, f, y=rows(63, 64)), lambda: ops.dense_forward(x, W, 40, y=rows(0, 64, column=8)),
             lambda: ops.dense_forward(x, W, f, residual=r, y=rows(101, 64)), lambda: ops.dense_forward(x, W, f, residual=r, y=rows(100, 64, stride=64)),
             lambda: ops.dense_forward(x, W, f, residual=r, y=far, keep=rows(470, 64)), lambda: ops.dense_forward(x, W, f, y=far, keep=rows(37, 64)),
             lambda: ops.dense_forward(x, flat[4800:].as_strided((64, 64), (64, 1)), f, y=rows(150, 64)),
             lambda: ops.gated_dense_forward(x, W2, f, y=rows(564, 64), keep=rows(500, 128)), lambda: ops.gated_dense_forward(x, W2, f, y=far, keep=rows(20, 128)),
             lambda: ops.dense_backward_input(x, W, f, dx=rows(2, 64)), lambda: ops.dense_backward_input(x, W, f, z=r, activation="relu", dx=rows(99, 64)),
             lambda: ops.dense_backward_input(x, W, f, z=rows(100, 128), activation="relu", gated=True, dx=rows(164, 128)),
             lambda: ops.dense_backward_input(x, W, f, z=r, activation="relu", dx=rows(100, 64, stride=64)),
             lambda: ops.rms_norm_forward(x, f, y=rows(60, 64)), lambda: ops.rms_norm_forward(x, f, residual=r, s=rows(1, 64)), lambda: ops.rms_norm_forward(x, f, residual=r, y=rows(101, 64)),
             lambda: ops.rms_norm_forward(x, f, residual=r, y=far, s=rows(501, 64)), lambda: ops.rms_norm_forward(x, f, residual=r, y=x, s=x),
             lambda: ops.rms_norm_int8(x, f, residual=r, s=rows(120, 64)), lambda: ops.rms_norm_backward(x, r, rstd, f, ds=rows(1, 64)),
             lambda: ops.rms_norm_backward(x, r, rstd, f, ds=rows(80, 64)), lambda: ops.rms_norm_backward(x, r, rstd, f, dresidual=far, ds=rows(500, 64, stride=64))]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError, match="memory of its own"):
            call()
            pytest.fail(f"call {k}")


@pytest.mark.gpu
def test_sums_and_numbers_that_lie_in_other_buffers_are_refused():
    from binarybrain_b200 import ops
    flat = torch.zeros(8192, device="cuda")                               # 64 rows of 48 of bf16 are 1536 of these
    x, y, dy, dr = (flat[1536 * i:1536 * (i + 1)].view(BF16).view(64, 48) for i in range(4))
    numbers = lambda first, n=64: flat[first:first + n]  # noqa: E731
    W, W2, rest, f = ops.dense_weights(torch.zeros(64, 64, device="cuda")), ops.dense_weights(torch.zeros(128, 64, device="cuda")), 1536 * 4, 48
    weights = flat[:4096].view(64, 64)
    far = torch.zeros((64, 48), dtype=BF16, device="cuda"), torch.zeros((64, 48), dtype=BF16, device="cuda")
    calls = [lambda: ops.rms_norm_forward(x, f, y=y, rstd=numbers(1500)), lambda: ops.rms_norm_forward(x, f, y=y, rstd=numbers(1536)), lambda: ops.rms_norm_forward(x, f, y=y, gamma=numbers(3000)),
             lambda: ops.rms_norm_forward(x, f, residual=y, s=dy, gamma=numbers(3100)), lambda: ops.rms_norm_forward(x, f, gamma=numbers(rest), rstd=numbers(rest + 63)),
             lambda: ops.rms_norm_int8(x, f, residual=y, s=dy, gamma=numbers(3100)), lambda: ops.rms_norm_backward(x, dy, numbers(1536), f, ds=y),
             lambda: ops.rms_norm_backward(x, dy, numbers(rest), f, gamma=numbers(1600), ds=y), lambda: ops.rms_norm_backward(x, dy, numbers(rest), f, dgamma=numbers(40)),
             lambda: ops.rms_norm_backward(x, dy, numbers(rest), f, dresidual=dr, dgamma=numbers(5000)), lambda: ops.rms_norm_backward(x, dy, numbers(rest), f, dgamma=numbers(rest + 40)),
             lambda: ops.rms_norm_backward(x, dy, numbers(rest), f, gamma=numbers(rest + 100), dgamma=numbers(rest + 100)),
             lambda: ops.dense_forward(x, W, f, bias=numbers(1600), y=y), lambda: ops.dense_forward(x, W, f, bias=numbers(1600), y=dy, keep=y),
             lambda: ops.gated_dense_forward(x, W2, f, bias=numbers(1600, 128), y=y), lambda: ops.dense_backward_weights(x, far[0], f, dW=weights),
             lambda: ops.dense_backward_weights(far[0], dy, f, dW=weights), lambda: ops.dense_backward_weights(far[0], far[1], f, dW=weights, dbias=numbers(4095)),
             lambda: ops.dense_backward_weights(dr, far[0], f, dW=weights[:, :0].new_zeros(64, 64), dbias=numbers(4608))]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError, match="memory of its own"):
            call()
            pytest.fail(f"call {k}")
    ops.dense_backward_weights(far[0], far[1], f, dW=weights, dbias=numbers(4096))
    ops.rms_norm_backward(x, dy, numbers(rest), f, gamma=numbers(rest + 64), dgamma=numbers(rest + 128))


@pytest.mark.gpu
def test_buffers_side_by_side_in_the_same_rows_are_apart():
    from binarybrain_b200 import ops
    K, O, F = 96, 96, 40
    wide = torch.full((K, 3 * 48), float("nan"), dtype=BF16, device="cuda")
    x, y, z = wide[:, :48], wide[:, 48:96], wide[:, 96:]
    x[:, :F] = normal(30, K, F).to(BF16).cuda()
    W = ops.dense_weights((normal(31, O, K) / math.sqrt(K)).cuda())
    want, kept = ops.dense_forward(x.clone(), W, F, activation="silu", keep=True)
    ops.dense_forward(x, W, F, activation="silu", y=y, keep=z)
    assert torch.equal(y[:, :F], want[:, :F]) and torch.equal(z[:, :F], kept[:, :F])
    want = ops.rms_norm_forward(x.clone(), F)[0]
    ops.rms_norm_forward(x, F, y=y)
    assert torch.equal(y[:, :F], want[:, :F])


# sizes: few frames by lanes, one launch held in registers and read twice, two passes along the rows
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["rows", "odd"])
@pytest.mark.parametrize("N,F", [(70, 3), (4096, 4), (70, 33), (1025, 130), (16000, 60), (70001, 33), (2500, 4800)])
def test_norms_in_the_place_of_what_they_are_made_of(N, F, layout, dtype):
    from binarybrain_b200 import _native, ops
    x, r, dr = (normal(40 + i, N, F).to(dtype) for i in range(3))
    gamma = (1 + 0.2 * normal(43, N)).float().cuda()
    b = lambda t: buffer(t, dtype, layout)  # noqa: E731
    y, s, rstd = ops.rms_norm_forward(b(x), F, gamma=gamma, residual=b(r), y=b(x), s=b(x))
    for over_y, over_s in (("x", None), ("r", None), ("x", "r"), ("r", "x")):
        xs, rs = b(x), b(r)
        at = {"x": xs, "r": rs, None: b(x)}
        got = ops.rms_norm_forward(xs, F, gamma=gamma, residual=rs, y=at[over_y], s=at[over_s])
        assert got[0] is at[over_y] and got[1] is at[over_s]
        assert torch.equal(got[0][:, :F], y[:, :F]) and torch.equal(got[1][:, :F], s[:, :F]) and torch.equal(got[2], rstd), (over_y, over_s)
    want, _, alone = ops.rms_norm_forward(b(x), F, gamma=gamma, y=b(r))
    xs, got = b(x), torch.empty_like(alone)                               # x as y, of which the operator itself keeps nothing
    forward = _native.bbcu_fp32_RmsNormalization_Forward if dtype == torch.float32 else _native.bbcu_bf16_RmsNormalization_Forward
    forward(xs.data_ptr(), None, None, xs.data_ptr(), gamma, got, 1e-5, N, F, xs.stride(0), 0, 0, xs.stride(0))
    assert torch.equal(xs[:, :F], want[:, :F]) and torch.equal(got, alone)
    ds, dgamma = ops.rms_norm_backward(b(x), b(r), rstd, F, gamma=gamma, dresidual=b(dr), ds=b(x))
    for over in range(3):
        given = [b(x), b(r), b(dr)]
        got = ops.rms_norm_backward(given[0], given[1], rstd, F, gamma=gamma, dresidual=given[2], ds=given[over])
        assert got[0] is given[over] and torch.equal(got[0][:, :F], ds[:, :F]) and torch.equal(got[1], dgamma), over


def test_sums_that_are_too_long_for_16_bits_are_refused():
    """More than 2^20 terms of a bf16 output, before anything runs (the addresses are never read); fp32 outputs and gradients, whose sums are taken out, have no such limit."""
    import os
    from binarybrain_b200 import abi
    if not os.path.exists(abi.LIB_PATH):
        pytest.skip("library not built")
    from binarybrain_b200 import _native as native
    a, most = 1 << 20, 1 << 20
    n = most + 8

    def status(name, *args):
        with pytest.raises(abi.BbcuError) as e:
            getattr(native, name)(*args, 0)
        return e.value.status
    large, null = -6, -1
    for k, want in ((most, null), (n, large)):                            # (without y: what is not too large goes as far as that)
        assert status("bbcu_bf16_DenseAffine_Forward", a, a, None, None, None, None, 0, k, 8, 8, k, 8, 0, 8, 0) == want
        assert status("bbcu_bf16_GatedDense_Forward", a, a, None, None, None, 3, k, 8, 8, k, 8, 8, 0) == want
        assert status("bbcu_bf16_DenseAffine_BackwardInput", a, a, None, None, 0, 0, 8, k, 8, 8, 8, 0, 8) == want
    assert status("bbcu_bf16_fp32_DenseAffine_Forward", a, a, None, None, None, None, 0, n, 8, 8, n, 8, 0, 8, 0) == null
    assert status("bbcu_bf16_DenseAffine_BackwardWeights", None, None, a, a, 0, 8, 8, n, n, n, 8) == null


# ------------------------------------------------------------------------------------------------------------------------ sums of 32 bits
U = 2.0 ** -24


def error_of_product(K, O, F):
    """The error of the 2-norm of an fp32 product of K terms, and what that of a sum of 32 bits, term after term, is: the partial sums are sqrt(k / K) of the
    last one, each addition rounds by up to U / 2 to U of one, 0.43 U with errors evenly spread, independently: 0.43 U sqrt(sum k / K) = 0.3 U sqrt(K).  (One more
    rounding for the output.)"""
    from binarybrain_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(K + F)
    x = torch.randn((K, (F + 15) // 16 * 16), device="cuda", generator=g).to(BF16)
    W = ops.dense_weights(torch.randn((O, K), device="cuda", generator=g))
    got, want = ops.dense_forward(x, W, F, dtype=torch.float32)[:, :F].double(), W.double() @ x[:, :F].double()
    return float((got - want).norm() / want.norm()), (0.3 * math.sqrt(K) + 1) * U


@pytest.mark.gpu
@pytest.mark.parametrize("K,O,F", [(20000, 16, 8), (400000, 16, 8), (400000, 300, 4), (1 << 20, 150, 1)])
def test_sums_of_few_frames_keep_their_digits(K, O, F):
    error, in_order = error_of_product(K, O, F)
    assert error <= in_order


@pytest.mark.gpu
@pytest.mark.parametrize("K,O,F", [(64, 512, 512), (200, 300, 1000), (512, 512, 512), (700, 2048, 2000), (768, 2048, 2048), (768, 4000, 16), (1020, 1000, 200), (1500, 2500, 2500), (8192, 512, 2048)])
def test_sums_of_frames_keep_their_digits(K, O, F):
    from binarybrain_b200 import ops
    error, in_order = error_of_product(K, O, F)
    assert error <= in_order
    frames = (K + 15) // 16 * 16                                          # the weights' gradient: a sum over K frames
    g = torch.Generator(device="cuda").manual_seed(K)
    dy, x = (torch.randn((rows, frames), device="cuda", generator=g).to(BF16) for rows in (O, F))
    dW, _ = ops.dense_backward_weights(x, dy, K)
    want = dy[:, :K].double() @ x[:, :K].double().t()
    assert float((dW.double() - want).norm() / want.norm()) <= in_order


@pytest.mark.gpu
@pytest.mark.parametrize("F", [128, 8])
def test_the_longest_sum_of_a_16_bit_output(F):
    """2^20 terms that are all positive: what is cut is less than a tenth of the rounding to bf16, so that its error is that rounding, up to 2^-8 of the value, and a tenth."""
    from binarybrain_b200 import ops
    K, O = 1 << 20, 128
    g = torch.Generator(device="cuda").manual_seed(9)
    x, W = (torch.rand(shape, device="cuda", generator=g).to(BF16) for shape in ((K, 128), (O, K)))
    y = ops.dense_forward(x, W, F)[:, :F].double()
    want = W.double() @ x[:, :F].double()
    assert float(((y - want).abs() / want).max()) <= 1.1 * 2.0 ** -8


# ------------------------------------------------------------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.gpu
def test_norms_of_more_than_2_31_elements():
    """The last rows and columns of every output against 64 bits, of numbers that depend on their place: s and dy have nothing to do with one another, so that rows read
    from a wrong place show.  (Six buffers of 4.8 GB.)  Bounds: two roundings to bf16 of values of order 1, 2^-7 relative and absolute; dgamma a sum of 60000
    products in 32 bits in some 500 partial sums, 300 half-units of their magnitudes."""
    from binarybrain_b200 import ops
    N, F, eps = 40000, 60000, 1e-5
    g = torch.Generator(device="cuda").manual_seed(11)

    def frames():
        t = torch.empty((N, F), dtype=BF16, device="cuda")
        for at in range(0, N, 4096):
            t[at:at + 4096] = torch.randn((min(4096, N - at), F), device="cuda", generator=g)
        return t
    R, C = slice(-70, None), slice(-300, None)

    def near(got, want):
        assert float(((got.double() - want).abs() - 2.0 ** -7 * (1 + want.abs())).max()) <= 0
    x, r, gamma = frames(), frames(), 1 + 0.2 * torch.randn(N, device="cuda", generator=g)
    nowhere = lambda: torch.full((N, F), 77.0, dtype=BF16, device="cuda")  # noqa: E731
    y, s, rstd = ops.rms_norm_forward(x, F, gamma=gamma, residual=r, y=nowhere())
    s64 = (x[:, C] + r[:, C]).double()                                    # rounded once, as it is kept
    assert torch.equal(s[:, C].double(), s64)
    want = 1 / torch.sqrt((s64 * s64).mean(0) + eps)
    assert float(((rstd[C].double() - want).abs() / want).max()) <= (N / 512 + 24) * U
    near(y[R, C], s64[R] * want * gamma[R, None].double())
    del y
    q, scale, kept = ops.rms_norm_int8(x, F, gamma=gamma, residual=r)
    t = s[:, C].float() * gamma[:, None]
    unit = t.abs().amax(0) / torch.full((300,), 127.0, device="cuda")
    assert torch.equal(kept[R, C], s[R, C]) and torch.equal(q[C, R], torch.round(t[R] / unit).clamp(-127, 127).to(torch.int8).t())
    del q, kept, x, t
    dy = frames()
    ds, dgamma = ops.rms_norm_backward(s, dy, rstd, F, gamma=gamma, dresidual=r, ds=nowhere())
    xh, gd = s64 * rstd[C].double(), dy[:, C].double() * gamma[:, None].double()
    near(ds[R, C], (rstd[C].double() * (gd - xh * (gd * xh).mean(0)))[R] + r[R, C].double())
    terms = dy[R].double() * s[R].double() * rstd.double()
    assert float(((dgamma[R].double() - terms.sum(1)).abs() - 300 * U * terms.abs().sum(1)).max()) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("F", [4, 7, 200])
def test_rows_far_apart(F):
    """Rows of one buffer of 2^31 elements and more, 480000 elements apart, side by side in it: the bits of the same calls on buffers of their own.  (What takes one launch, or a few
    frames, has no such offsets otherwise.)"""
    from binarybrain_b200 import ops
    N, O, step, width = 4800, 4800, 480000, 208
    wide = torch.empty((N, step), dtype=BF16, device="cuda")
    column = iter(range(step - 12 * width, step, width))
    far = lambda t=None: (lambda v: v if t is None else v.copy_(t))(wide[:, (c := next(column)):c + width])  # noqa: E731
    x, r, dy, dr = (torch.zeros((N, width), dtype=BF16, device="cuda") for _ in range(4))
    for i, t in enumerate((x, r, dy, dr)):
        t[:, :F] = normal(60 + i, N, F).to(BF16).cuda()
    gamma = (1 + 0.2 * normal(64, N)).float().cuda()
    new = lambda: torch.empty((N, width), dtype=BF16, device="cuda")  # noqa: E731
    y, s, rstd = ops.rms_norm_forward(x, F, gamma=gamma, residual=r, y=new(), s=new())
    ds, dgamma = ops.rms_norm_backward(s, dy, rstd, F, gamma=gamma, dresidual=dr, ds=new())
    xf, sf = far(x), far()
    got = ops.rms_norm_forward(xf, F, gamma=gamma, residual=far(r), y=far(), s=sf)
    assert torch.equal(got[0][:, :F], y[:, :F]) and torch.equal(got[1][:, :F], s[:, :F]) and torch.equal(got[2], rstd)
    q, scale, _ = ops.rms_norm_int8(x, F, gamma=gamma, residual=r)
    got = ops.rms_norm_int8(xf, F, gamma=gamma, residual=far(r))
    assert torch.equal(got[0], q) and torch.equal(got[1], scale)
    dyf = far(dy)
    got = ops.rms_norm_backward(sf, dyf, rstd, F, gamma=gamma, dresidual=far(dr), ds=far())
    assert torch.equal(got[0][:, :F], ds[:, :F]) and torch.equal(got[1], dgamma)
    W = ops.dense_weights((normal(65, O, N) / math.sqrt(N)).cuda())
    yd, z = ops.dense_forward(x, W, F, activation="gelu", residual=r, y=new(), keep=new())
    got = ops.dense_forward(xf, W, F, activation="gelu", residual=far(r), y=far(), keep=far())
    assert torch.equal(got[0][:, :F], yd[:, :F]) and torch.equal(got[1][:, :F], z[:, :F])
    dx = ops.dense_backward_input(dy, W, F, z=r, activation="gelu", dx=new())
    rf = far(r)
    assert torch.equal(ops.dense_backward_input(dyf, W, F, z=rf, activation="gelu", dx=rf)[:, :F], dx[:, :F])
    assert all(torch.equal(a, b) for a, b in zip(ops.dense_backward_weights(xf, dyf, F), ops.dense_backward_weights(x, dy, F)))


# ------------------------------------------------------------------------------------------------------------------------ clipping
def test_pieces_of_the_largest_tensors_are_counted_without_overflow():
    """The count of a tensor's pieces is checked when the source is compiled, where an overflow is an error: for 2^31 - 1 elements, and by the kernels' own function."""
    import re
    from pathlib import Path
    source = (Path(__file__).parent.parent / "binarybrain_b200" / "csrc" / "gradient_norm.cu").read_text()
    assert re.search(r"static_assert\(pieces_of\(0x7fffffff, kPieceSize\)", source)
    assert not re.search(r"size \+ k(PieceSize|SmallPiece)", source)


@pytest.mark.gpu
def test_clipping_of_the_largest_tensor():
    """2^31 - 1 elements, 8 GB, in which ones lie in the first and the last pieces: the norm, the factor at both ends, and nothing else."""
    from binarybrain_b200 import ops
    n = (1 << 31) - 1
    big, small = torch.zeros(n, device="cuda"), torch.full((5,), 2.0, device="cuda")
    ones = [0, 8191, 8192, n - 8192, n - 8191, n - 2, n - 1]
    big[torch.tensor(ones, device="cuda")] = 1.0
    clip = ops.GradientNorm([small, big])
    want = math.sqrt(len(ones) + 20)
    assert abs(float(clip.norm()) - want) <= 2 * U * want
    clip.clip_(1.0)
    at = torch.nonzero(big).flatten().tolist()
    assert at == ones and all(abs(float(big[i]) - 1 / want) <= 4 * U / want for i in ones) and float((small - 2 / want).abs().max()) <= 8 * U / want
    assert abs(float(clip.norm()) - 1) <= 8 * U
