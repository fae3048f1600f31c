"""Fused linear layer on MI355X: y = act(x W^T + bias) + residual in one product with an
epilogue, and its backward (no counterpart in the reference, whose models keep
nn.Linear around their activations and residual adds).

The sum over K, the bias, the activation and the residual are added up in fp32 and y is
rounded once. The backward needs z = x W^T + bias where there is an activation: it is
kept in 16 bits (fp16 with a power of two as scale for every 32 columns of a row, which
rounds finer than bf16; in fp32 where the products run in fp32), or in 8 (checkpoint=
"fp8": e4m3 with such scales), formed of the fp32 sums. What is not needed (x where the
weight is frozen, W where x needs no gradient) is not kept. First derivatives only.

bf16 with sizes in multiples of 8 runs on the bf16 matrix cores, as fp16 does in forwards
of up to 64 rows that keep nothing, everything else on the fp32 ones (fp16 and other bf16
sizes are upcast, and rounded once at the end).
"""

from __future__ import annotations

import torch
import torch.nn as nn

from metal_liger_amd import _custom_ops as cops
from metal_liger_amd import hip_ops

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def check_checkpoint(checkpoint: str | None) -> None:
    if checkpoint not in (None, "fp8"):
        raise ValueError(f'checkpoint must be None or "fp8" (got {checkpoint!r})')


def keep_mode(checkpoint: str | None, dtype: torch.dtype) -> int:
    """How a backward's tensors are kept where the products are of `dtype`."""
    if checkpoint == "fp8":
        return hip_ops.KEEP_FP8
    return hip_ops.KEEP_FP16 if dtype == torch.bfloat16 else hip_ops.KEEP_F32


def compute_dtype(x: torch.Tensor, *features: int, infer: bool = False) -> torch.dtype:
    """bf16 where its matrix-core kernels take the sizes, fp16 in forwards of few rows
    with nothing to keep (infer), else fp32."""
    if x.dtype != torch.float32 and all(f % 8 == 0 for f in features):
        if x.dtype == torch.bfloat16:
            return x.dtype
        if infer and x.numel() <= hip_ops.FEW_ROWS * x.shape[-1]:
            return x.dtype
    return torch.float32


def rows(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """[..., C] -> [R, C] in dtype."""
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return t if t.dtype == dtype else t.to(dtype)


def check_input(what: str, x: torch.Tensor, *weights: torch.Tensor) -> None:
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: x must be fp32, bf16 or fp16 (got {x.dtype})")
    for w in weights:
        if w.dim() != 2 or 0 in w.shape:
            raise ValueError(f"{what}: a weight must be [out, in] (got {tuple(w.shape)})")
        if w.dtype != x.dtype:
            raise TypeError(f"{what}: weight of {w.dtype} with x of {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != weights[0].shape[1]:
        raise ValueError(f"{what}: x {tuple(x.shape)} does not fit a weight of "
                         f"{tuple(weights[0].shape)}")


def check_residual(what: str, residual, x: torch.Tensor, out: int) -> None:
    shape = (*x.shape[:-1], out)
    if residual is not None and (tuple(residual.shape) != shape or residual.dtype != x.dtype):
        raise ValueError(f"{what}: residual {tuple(residual.shape)} {residual.dtype}, needed is "
                         f"{shape} {x.dtype}")


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _forward(x, weight, bias, residual, act: int, keep: int):
    """(y, z, zscale), or y alone where nothing is kept."""
    none = keep == hip_ops.KEEP_NONE
    ct = compute_dtype(x, *weight.shape, infer=none)
    args = (rows(x, ct), rows(weight, ct), bias if bias is None or bias.dtype == ct else bias.to(ct),
            None if residual is None else rows(residual, ct), act)
    y, *kept = (cops.linear_infer(*args),) if none else cops.linear_fwd(*args, keep)
    if y.dtype != x.dtype:
        y = y.to(x.dtype)
    if x.dim() != 2:
        y = y.view(*x.shape[:-1], weight.shape[0])
    return y, *kept


class _FusedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int, keep: int):
        need_dx, need_dw, need_db = ctx.needs_input_grad[:3]
        if act == 0 or not (need_dx or need_dw or need_db):
            keep = hip_ops.KEEP_NONE
        y, *kept = _forward(x, weight, bias, residual, act, keep)
        ctx.save_for_backward(x if need_dw else None, weight if need_dx else None, *kept)
        ctx.act, ctx.keep, ctx.sizes = act, keep, tuple(weight.shape)
        ctx.x_shape, ctx.dtype = x.shape, x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        need_dx, need_dw, need_db, need_dr = ctx.needs_input_grad[:4]
        grads = [None, None, None]
        if need_dx or need_dw or need_db:
            x, weight, *kept = ctx.saved_tensors
            z, zscale = kept or (None, None)
            N, K = ctx.sizes
            g = rows(dy, compute_dtype(dy, N, K))
            out = cops.linear_bwd(None if x is None else rows(x, g.dtype),
                                  None if weight is None else rows(weight, g.dtype), g, ctx.act,
                                  ctx.keep, z, zscale, N, K, need_dx, need_dw, need_db)
            for i, need in enumerate((need_dx, need_dw, need_db)):
                if need:
                    grads[i] = out[i] if out[i].dtype == ctx.dtype else out[i].to(ctx.dtype)
            if need_dx and len(ctx.x_shape) != 2:
                grads[0] = grads[0].view(ctx.x_shape)
        return (*grads, dy if need_dr else None, None, None)


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 activation: str | None = None, residual: torch.Tensor | None = None,
                 checkpoint: str | None = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual.

    x [..., in], weight [out, in] (nn.Linear's), bias [out], residual [..., out]; all of
    x's dtype (fp32, bf16 or fp16) and on its device, any strides. activation: None,
    "silu", "gelu" (by the error function, nn.GELU's default) or "gelu_tanh" (nn.GELU's
    approximate="tanh"); the residual is added after it. checkpoint: None, or "fp8" to
    keep what the activation's backward needs in 8 bits (module docstring).
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"fused_linear: activation {activation!r} is not one of "
                         f"{list(ACTIVATIONS)}")
    act = ACTIVATIONS[activation]
    check_checkpoint(checkpoint)
    check_input("fused_linear", x, weight)
    if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.dtype != x.dtype):
        raise ValueError(f"fused_linear: bias {tuple(bias.shape)} {bias.dtype}, needed is "
                         f"({weight.shape[0]},) {x.dtype}")
    check_residual("fused_linear", residual, x, weight.shape[0])
    if not wants_grad(x, weight, bias, residual):
        return _forward(x, weight, bias, residual, act, hip_ops.KEEP_NONE)[0]
    keep = keep_mode(checkpoint, compute_dtype(x, *weight.shape))
    return _FusedLinearFunction.apply(x, weight, bias, residual, act, keep)


class MetalLigerLinear(nn.Module):
    """Drop-in for an nn.Linear with what follows it, whose parameters it shares
    (state_dict keys are unchanged); forward also takes a residual to add."""

    def __init__(self, original: nn.Linear, activation: str | None = None,
                 checkpoint: str | None = None):
        super().__init__()
        if type(original) is not nn.Linear:
            raise ValueError(f"MetalLigerLinear: a plain nn.Linear is needed (got {original})")
        if activation not in ACTIVATIONS:
            raise ValueError(f"MetalLigerLinear: activation {activation!r} is not one of "
                             f"{list(ACTIVATIONS)}")
        check_checkpoint(checkpoint)
        self.weight, self.bias = original.weight, original.bias
        self.activation, self.checkpoint = activation, checkpoint

    def forward(self, input: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        return fused_linear(input, self.weight, self.bias, self.activation, residual,
                            self.checkpoint)

    def extra_repr(self) -> str:
        out, ins = self.weight.shape
        return f"{ins}, {out}, bias={self.bias is not None}, activation={self.activation}"
