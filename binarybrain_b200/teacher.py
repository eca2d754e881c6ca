"""Layers of the dense teacher beside a LUT network, to train it and to serve it, and the normalised head of a student that learns from it.

No counterpart in the reference.  Like the other layers here they have ``forward(x, frames, total_frames)`` on CUDA frame buffers [nodes, stride], fp32
or bf16; the arithmetic is that of the bbcu_* operators (``ops``), there is no CPU path behind it.
"""
import torch

from . import ops


def _kept(layer):
    """What the last forward pass of a layer left for its backward pass."""
    if layer._saved is None:
        raise RuntimeError(f"{type(layer).__name__}: nothing is kept, the last pass was not one for training or has had its backward pass")
    return layer._saved


class LayerNormalization:
    """Layer norm over the nodes of a frame with a learned scale and offset a node; a batch that is sharded over frames needs no exchange but that of
    dgamma and dbeta, which backward() adds to."""

    def __init__(self, nodes, eps=1e-5, gamma=1.0, beta=0.0, device="cuda"):
        self.n_out, self.eps = nodes, eps
        self.gamma = torch.full((nodes,), float(gamma), device=device)
        self.beta = torch.full((nodes,), float(beta), device=device)
        self.dgamma, self.dbeta = torch.zeros_like(self.gamma), torch.zeros_like(self.beta)
        self._saved = None

    def forward(self, x, frames, total_frames=None, y=None):
        y, mean, rstd = ops.layer_norm_forward(x, frames, gamma=self.gamma, beta=self.beta, eps=self.eps, y=y)
        self._saved = x, mean, rstd, frames
        return y

    def backward(self, dy, dx=None):
        x, mean, rstd, frames = self._saved
        self._saved = None
        return ops.layer_norm_backward(x, dy, mean, rstd, frames, gamma=self.gamma, dx=dx, dgamma=self.dgamma, dbeta=self.dbeta)[0]


class Int8Dense:
    """A dense layer whose weights [out, in] are laid out once as 8-bit integers with a scale a row; frames are quantised as they come.  Inference only."""

    def __init__(self, W, bias=None, dtype=torch.float32):
        self.n_in, self.n_out, self.dtype = W.shape[1], W.shape[0], dtype
        self.W, self.w_scale = ops.quantize_int8_channels(W)
        self.bias = bias

    def forward(self, x, frames, total_frames=None, y=None):
        return self.forward_int8(*ops.quantize_int8(x, frames), y=y)

    def forward_int8(self, q, scale, y=None):
        """On frames that come as 8-bit integers already."""
        return ops.int8_dense_forward(q, scale, self.W, self.w_scale, n_in=self.n_in, bias=self.bias, y=y, dtype=self.dtype)


class RmsNormalization:
    """Root-mean-square norm over the nodes of a frame with a learned scale a node, and the residual's addition before it.  forward() returns (y, s): s = x +
    residual is what the next residual goes on from; backward() takes the gradients of both."""

    def __init__(self, nodes, eps=1e-5, gamma=1.0, device="cuda"):
        self.n_out, self.eps = nodes, eps
        self.gamma = torch.full((nodes,), float(gamma), device=device)
        self.dgamma = torch.zeros_like(self.gamma)
        self._saved = None

    def parameters(self):
        return [(self.gamma, self.dgamma)]

    def forward(self, x, frames, total_frames=None, residual=None, y=None, train=True):
        y, s, rstd = ops.rms_norm_forward(x, frames, gamma=self.gamma, eps=self.eps, residual=residual, y=y)
        self._saved = (s, rstd, frames) if train else None
        return y, s

    def forward_int8(self, x, frames, residual=None):
        """For serving: returns (q, scale, s), q and scale as Int8Dense.forward_int8 takes them."""
        return ops.rms_norm_int8(x, frames, gamma=self.gamma, eps=self.eps, residual=residual)

    def backward(self, dy, ds=None, out=None):
        s, rstd, frames = _kept(self)
        self._saved = None
        return ops.rms_norm_backward(s, dy, rstd, frames, gamma=self.gamma, dresidual=ds, ds=out, dgamma=self.dgamma)[0]


class DenseAffine:
    """A dense layer in bf16: y = activation(z) + residual, z = W x + bias.  The weights that are trained are fp32 (a contiguous fp32 W is taken as it is, and so is
    the bias, not copied); refresh() lays them out in bf16 as the product reads them, after they have changed.

    backward() returns the gradient of x and adds to dW and dbias.  Without an activation it takes the gradient of y, which is the residual's as well.  With one it
    takes that of z, as the layer above returns it when this one is its `below`: what is made of y by anything else, a norm or a loss, has no way back through an
    activation here, and neither has the residual beside one.  Gradients of frames are bf16, also where y is fp32."""

    gated = False                                        # a gated block's z has twice the rows of its y, which tells the gradients apart

    def __init__(self, W, bias=None, activation=None, dtype=torch.bfloat16):
        self.n_in, self.n_out, self.activation, self.dtype = W.shape[1], W.shape[0], activation, dtype
        self.W, self.bias = W.float().contiguous(), bias
        self.dW, self.dbias = torch.zeros_like(self.W), None if bias is None else torch.zeros_like(bias)
        self.W16 = ops.dense_weights(self.W)
        self._saved, self._z_given, self._beside = None, False, False

    def parameters(self):
        return [(self.W, self.dW)] + ([] if self.bias is None else [(self.bias, self.dbias)])

    def refresh(self):
        self.W16.copy_(self.W)

    def forward(self, x, frames, total_frames=None, residual=None, y=None, train=True):
        keep = train and self.activation not in (None, "none")
        y = ops.dense_forward(x, self.W16, frames, bias=self.bias, activation=self.activation, residual=residual, y=y, dtype=self.dtype, keep=keep)
        y, z = y if keep else (y, None)
        self._saved, self._z_given, self._beside = (x, z, frames) if train else None, False, keep and residual is not None
        return y

    def backward(self, dy, dx=None, below=None, of_z=False):
        """dy: the gradient of y, or, for a layer with an activation, of z: what the layer above returns when this one is its `below`, or, with of_z=True, the caller's
        own.  below: the layer whose output x is; where that has an activation or is gated, the gradient of its z is returned."""
        x, _, frames = _kept(self)
        if self.activation not in (None, "none") and not (self.gated or self._z_given or of_z):
            raise ValueError("dy: the gradient of y, where a layer with an activation takes that of z (give this layer to the one above as its `below`)")
        z, activation, gated = below.kept() if below is not None else (None, None, False)
        ops.dense_backward_weights(x, dy, frames, dW=self.dW, dbias=self.dbias)
        dx = ops.dense_backward_input(dy, self.W16, frames, z=z, activation=activation, gated=gated, dx=dx)
        self._saved = None
        if below is not None:
            below._z_given = True
        return dx

    def kept(self):
        """For the layer above, which makes the gradient of z."""
        if self._beside:
            raise ValueError("below: a layer with a residual beside its activation, whose gradient would be lost")
        return _kept(self)[1], self.activation, self.gated


class GatedDense(DenseAffine):
    """The gated block: activation(g) * u, g and u the upper and the lower half of W x + bias.  backward() takes the gradient of both, as the layer above
    returns it when this one is its `below`."""

    gated = True

    def __init__(self, W, bias=None, activation="silu"):
        super().__init__(W, bias, activation)
        self.n_out //= 2

    def forward(self, x, frames, total_frames=None, y=None, train=True):
        y = ops.gated_dense_forward(x, self.W16, frames, bias=self.bias, activation=self.activation, y=y, keep=train)
        y, z = y if train else (y, None)
        self._saved = (x, z, frames) if train else None
        return y


class FeedForward:
    """Norm, gated block and dense layer of a residual stream: forward(x, frames, residual) returns (y, s), s = x + residual and y what is to be added to it by
    the next norm; backward(dy, ds) returns the gradient of s, which is that of x and of the residual."""

    def __init__(self, nodes, hidden, generator=None, activation="silu", device="cuda"):
        def weights(rows, inputs):
            return torch.randn((rows, inputs), device=device, generator=generator) / inputs ** 0.5
        self.norm = RmsNormalization(nodes, device=device)
        self.gated = GatedDense(weights(2 * hidden, nodes), activation=activation)
        self.dense = DenseAffine(weights(nodes, hidden))

    def parameters(self):
        return self.norm.parameters() + self.gated.parameters() + self.dense.parameters()

    def refresh(self):
        self.gated.refresh()
        self.dense.refresh()

    def forward(self, x, frames, residual=None, train=True):
        n, s = self.norm.forward(x, frames, residual=residual, train=train)
        return self.dense.forward(self.gated.forward(n, frames, train=train), frames, train=train), s

    def backward(self, dy, ds=None):
        return self.norm.backward(self.gated.backward(self.dense.backward(dy, below=self.gated)), ds)


def clipped_adam(layers, max_norm, **kw):
    """Adam over all parameters of `layers`, clipped by the global norm of their gradients; call refresh() of the layers after its update()."""
    pairs = [pair for layer in layers for pair in layer.parameters()]
    return ops.Adam([p for p, _ in pairs], [g for _, g in pairs], max_norm=max_norm, **kw)


def top_logits(logits, frames, top, stride=None):
    """The `top` largest logits of every frame and their classes, as frame buffers that distillation_loss takes."""
    values, index = torch.topk(logits[:, :frames], top, dim=0)
    stride = ops.frame_stride(frames, logits.dtype) if stride is None else stride
    t = torch.empty((top, stride), dtype=logits.dtype, device=logits.device)
    i = torch.empty((top, stride), dtype=torch.int32, device=logits.device)
    t[:, :frames], i[:, :frames] = values, index
    return t, i
