"""A LUT network learns from a dense teacher that is served in 8-bit integers.

    python examples/distill_int8_teacher.py [steps]

Teacher (random weights, bf16 frames): layer norm -> int8 dense -> ReLU -> layer norm -> int8 dense, of whose classes the top logits are kept.
Student (fp32 frames): three DifferentiableLut6 layers -> mean of every class's nodes -> layer norm with a learned scale -> logits.
Every step runs the distillation loss, the student's backward pass and Adam.  Prints the loss as it falls.
"""
import os
import sys

import numpy as np
import torch

if __package__ in (None, ""):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from binarybrain_b200 import ops
from binarybrain_b200.dist import ShardedDifferentiableLut6
from binarybrain_b200.teacher import Int8Dense, LayerNormalization, top_logits

INPUTS, HIDDEN, WIDTHS, CLASSES, TOP, TEMPERATURE = 256, 512, (1024, 600, 200), 20, 8, 2.0


class Teacher:
    def __init__(self, rng):
        dense = lambda o, i: Int8Dense(torch.from_numpy((rng.standard_normal((o, i)) / np.sqrt(i)).astype(np.float32)).cuda(), dtype=torch.bfloat16)  # noqa: E731
        self.norms = LayerNormalization(INPUTS), LayerNormalization(HIDDEN, gamma=3.0)
        self.dense = dense(HIDDEN, INPUTS), dense(CLASSES, HIDDEN)

    def logits(self, x, frames):
        h = self.dense[0].forward(self.norms[0].forward(x.to(torch.bfloat16), frames), frames)
        return self.dense[1].forward(self.norms[1].forward(torch.relu_(h), frames), frames)


class Student:
    def __init__(self, rng):
        self.layers = []
        for n_in, n_out in zip((INPUTS,) + WIDTHS, WIDTHS):
            idx = np.stack([rng.permutation(n_in)[:6] for _ in range(n_out)]).astype(np.int32)
            W = np.clip(rng.normal(0.5, 0.25, (n_out, 64)), 0, 1).astype(np.float32)
            self.layers.append(ShardedDifferentiableLut6(torch.from_numpy(idx).cuda(), torch.from_numpy(W).cuda(), n_in, sharded=False))
        self.norm = LayerNormalization(CLASSES)
        self.adam = ops.Adam([layer.W for layer in self.layers] + [self.norm.gamma, self.norm.beta],
                             [layer.dW for layer in self.layers] + [self.norm.dgamma, self.norm.dbeta], lr=0.005)

    def step(self, x, t, index, frames):
        for layer in self.layers:
            ops.clamp_(layer.W)
            x = layer.forward(x, frames, frames)
        z = self.norm.forward(ops.reduce_forward(x, CLASSES, frames), frames)
        dz, loss, _ = ops.distillation_loss(z, t, index, frames, temperature=TEMPERATURE)
        g = ops.reduce_backward(self.norm.backward(dz), WIDTHS[-1], frames)
        for layer in reversed(self.layers):
            g = layer.backward(g)
        self.adam.update()
        return loss


def train(steps=300, frames=1000, seed=0, log=None):
    """The losses of `steps` steps on batches drawn from a set of 4 * `frames` inputs."""
    rng = np.random.default_rng(seed)
    teacher, student = Teacher(rng), Student(rng)
    losses = []
    batches = []
    for _ in range(4):
        x = torch.zeros((INPUTS, ops.fp32_stride(frames)), device="cuda")
        x[:, :frames] = torch.from_numpy(rng.random((INPUTS, frames), dtype=np.float32)).cuda()
        batches.append((x, *top_logits(teacher.logits(x, frames).float(), frames, TOP)))
    for step in range(steps):
        loss = student.step(*batches[step % len(batches)], frames)
        if step % 50 == 0 or step == steps - 1:
            losses.append(float(loss))
            if log:
                log(f"step {step:4d}  loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    train(int(sys.argv[1]) if len(sys.argv) > 1 else 300, log=print)
