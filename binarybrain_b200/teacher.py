"""Layers of the dense teacher beside a LUT network, and the normalised head of a student that learns from it.

No counterpart in the reference.  Like the other layers here they have ``forward(x, frames, total_frames)`` on CUDA frame buffers [nodes, stride], fp32
or bf16; the arithmetic is that of the bbcu_* operators (``ops``), there is no CPU path behind it.
"""
import torch

from . import ops


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
        q, scale = ops.quantize_int8(x, frames)
        return ops.int8_dense_forward(q, scale, self.W, self.w_scale, n_in=self.n_in, bias=self.bias, y=y, dtype=self.dtype)


def top_logits(logits, frames, top, stride=None):
    """The `top` largest logits of every frame and their classes, as frame buffers that distillation_loss takes."""
    values, index = torch.topk(logits[:, :frames], top, dim=0)
    stride = ops.frame_stride(frames, logits.dtype) if stride is None else stride
    t = torch.empty((top, stride), dtype=logits.dtype, device=logits.device)
    i = torch.empty((top, stride), dtype=torch.int32, device=logits.device)
    t[:, :frames], i[:, :frames] = values, index
    return t, i
