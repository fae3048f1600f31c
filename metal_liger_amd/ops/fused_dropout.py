"""Fused dropout on MI355X: nn.Dropout, with the add of a residual after it, whose
mask is never stored (no counterpart in the reference, whose models keep
nn.Dropout and whose fused LoRA ignores lora_dropout).

The mask comes from a counter-based generator: an element's random number is a
function of the seed, the stream and the element's index, so that the backward
forms the forward's mask again instead of reading one. The rate is applied as
round(65536 p) / 65536, and kept elements are scaled by the inverse of exactly
that.

The seed is one int64 on the GPU. By default each call draws it from torch's
generator of the device, so that torch.manual_seed reproduces a run, activation
checkpointing recomputes the same mask and a captured step gets a new one at each
replay; where nothing is dropped none is drawn. A seed given as a tensor is read when
the kernels run: changing it between a forward and its backward is an error that
autograd reports, and changing it between replays gives each its own masks. An int is
the same mask at each call.

The backward can be differentiated again; forward mode and torch.func's transforms
are refused.
"""

from __future__ import annotations

import operator

import torch
import torch.nn as nn

from metal_liger_amd import _custom_ops as cops
from metal_liger_amd import hip_ops


def seed_tensor(seed, device) -> torch.Tensor:
    """A dropout seed as one int64 on `device`: given as a tensor or an int, or
    drawn from torch's generator."""
    if seed is None:
        return torch.randint(-(2 ** 63), 2 ** 63 - 1, (1,), dtype=torch.int64, device=device)
    if isinstance(seed, torch.Tensor):
        return seed
    wrapped = (operator.index(seed) + 2 ** 63) % 2 ** 64 - 2 ** 63
    return torch.full((1,), wrapped, dtype=torch.int64, device=device)


class _FusedDropoutFunction(torch.autograd.Function):
    """Dropout (+ residual); saves the seed alone."""

    @staticmethod
    def forward(ctx, x, residual, seed, threshold: int, stream: int):
        ctx.save_for_backward(seed)
        ctx.threshold, ctx.stream = threshold, stream
        return cops.dropout(x, residual, seed, threshold, stream, hip_ops.drop_scale(threshold))

    @staticmethod
    def backward(ctx, dy):
        seed, = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0] and ctx.threshold == 0:
            dx = dy
        elif ctx.needs_input_grad[0] and torch.is_grad_enabled():  # create_graph
            dx = _FusedDropoutFunction.apply(dy, None, seed, ctx.threshold, ctx.stream)
        elif ctx.needs_input_grad[0]:
            dx = cops.dropout(dy, None, seed, ctx.threshold, ctx.stream,
                              hip_ops.drop_scale(ctx.threshold))
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def fused_dropout(x: torch.Tensor, p: float = 0.5, training: bool = True,
                  residual: torch.Tensor | None = None, seed=None,
                  stream: int = 0) -> torch.Tensor:
    """x with a share p of its elements dropped and the others scaled by 1 / (1 - p),
    plus residual (of x's shape and dtype) where one is given.

    x of fp32, bf16 or fp16 and any shape and strides; the mask goes by row-major
    order. seed: one int64 on x's device, an int, or None (module docstring);
    stream: 0 .. 2^32 - 1, for several masks of one seed. Not training: x (+ residual),
    and no seed is drawn.
    """
    threshold = hip_ops.drop_threshold(p) if training else 0
    if not 0 <= stream < 2 ** 32:
        raise ValueError(f"dropout: stream {stream} outside 0 .. 2^32 - 1")
    if threshold == 0 and residual is None:
        return x
    hip_ops.ensure_rocm_device(x, residual)
    seed = seed_tensor(seed, x.device) if threshold else None
    return _FusedDropoutFunction.apply(x, residual, seed, threshold, stream)


class MetalLigerDropout(nn.Module):
    """Drop-in for nn.Dropout; forward also takes a residual to add. (There is no
    in-place form: inplace=True is refused.)"""

    def __init__(self, p: float = 0.5, inplace: bool = False):
        super().__init__()
        hip_ops.drop_threshold(p)
        if inplace:
            raise ValueError("MetalLigerDropout: inplace is not supported")
        self.p, self.inplace = p, False

    def forward(self, input: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        return fused_dropout(input, self.p, self.training, residual)

    def extra_repr(self) -> str:
        return f"p={self.p}"
