"""Fused gated feed-forward block on MI355X: y = (silu(x Wg^T) * (x Wu^T)) Wd^T
(+ residual), and its backward (the reference fuses the activation step only,
ops/fused_swiglu.py:59-75, and its LoRA block needs adapters).

The backward needs gate = x Wg^T and up = x Wu^T: they are kept in 16 bits (fp16 with a
power of two as scale for every 32 columns of a row; fp32 in fp32), or in 8
(checkpoint="fp8": e4m3 with such scales), formed of the fp32 sums. h = silu(gate) * up
is not kept; the backward forms it again of what was kept. What is not needed (x where
gate's and up's weights are frozen) is not kept. h and the gradients of gate, up and h
are rounded to bf16 between the products on the bf16 matrix cores. First derivatives
only, in reverse mode (forward mode is refused). Types and sizes as ops/fused_linear.py.
"""

from __future__ import annotations

import logging

import torch
import torch.nn as nn
import torch.nn.functional as F

from metal_liger_amd import _custom_ops as cops
from metal_liger_amd import hip_ops
from metal_liger_amd._forward_form import call, mul
from metal_liger_amd._model_walk import find_layers
from metal_liger_amd.ops.fused_linear import (activation_name, check_checkpoint, check_input,
                                              check_residual, computes, hooked, keep_mode,
                                              plain_linear, rows, takes, wants_grad)
from metal_liger_amd.ops.fused_swiglu import MetalLigerSwiGLU

logger = logging.getLogger(__name__)


def _forward(x, weights, residual, keep: int):
    """(y, gate, its scales, up, its scales), or y alone where nothing is kept."""
    args = (rows(x), *weights, rows(residual))
    y, *kept = (cops.swiglu_mlp_infer(*args),) if keep == hip_ops.KEEP_NONE else \
        cops.swiglu_mlp_fwd(*args, keep)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weights[2].shape[0]), *kept


class _FusedSwiGLUMLPFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, residual, keep: int):
        if not any(ctx.needs_input_grad[:4]):
            keep = hip_ops.KEEP_NONE
        y, *kept = _forward(x, (wg, wu, wd), residual, keep)
        need_dx, need_dwg, need_dwu = ctx.needs_input_grad[:3]
        ctx.save_for_backward(x if need_dwg or need_dwu else None, *((wg, wu) if need_dx else
                              (None, None)), wd, *kept)
        ctx.keep, ctx.x_shape = keep, x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        grads = [None] * 4
        if any(ctx.needs_input_grad[:4]):
            x, wg, wu, wd, *kept = ctx.saved_tensors
            outs = cops.swiglu_mlp_bwd(rows(x), wg, wu, wd, rows(dy), ctx.keep, *kept,
                                       *ctx.needs_input_grad[:4])
            grads = [g if need else None for g, need in zip(outs, ctx.needs_input_grad)]
            if grads[0] is not None and len(ctx.x_shape) != 2:
                grads[0] = grads[0].view(ctx.x_shape)
        return (*grads, dy if ctx.needs_input_grad[4] else None, None)


def fused_swiglu_mlp(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor,
                     down_weight: torch.Tensor, residual: torch.Tensor | None = None,
                     checkpoint: str | None = None) -> torch.Tensor:
    """(silu(x gate_weight^T) * (x up_weight^T)) down_weight^T + residual.

    x [..., hidden], gate_weight and up_weight [inter, hidden], down_weight [out, inter],
    residual [..., out]; all of x's dtype (fp32, bf16 or fp16; autocast casts none of
    them) and on its device, any strides. checkpoint: None, or "fp8" to keep gate and up in
    8 bits for the backward.
    """
    check_checkpoint(checkpoint)
    check_input("fused_swiglu_mlp", x, gate_weight, up_weight, down_weight)
    if up_weight.shape != gate_weight.shape or down_weight.shape[1] != gate_weight.shape[0]:
        raise ValueError(f"fused_swiglu_mlp: weights {tuple(gate_weight.shape)}, "
                         f"{tuple(up_weight.shape)} and {tuple(down_weight.shape)} do not fit")
    check_residual("fused_swiglu_mlp", residual, x, down_weight.shape[0])
    weights = (gate_weight, up_weight, down_weight)
    if not wants_grad(x, *weights, residual):
        return _forward(x, weights, residual, hip_ops.KEEP_NONE)[0]
    keep = keep_mode(checkpoint, x.dtype)
    return _FusedSwiGLUMLPFunction.apply(x, *weights, residual, keep)


_PROJECTIONS = ("gate_proj", "up_proj", "down_proj")


def _gated_formula(x):
    return call("down_proj", mul(call("act_fn", call("gate_proj", x)), call("up_proj", x)))


def _plain_projections(mlp: nn.Module) -> bool:
    """Three plain linear layers without bias."""
    projections = [getattr(mlp, name, None) for name in _PROJECTIONS]
    return all(plain_linear(m) and m.bias is None for m in projections)


def _gated(mlp: nn.Module) -> bool:
    """Three plain linear layers without bias, and SiLU."""
    if not _plain_projections(mlp):
        return False
    act = getattr(mlp, "act_fn", None)  # MetalLigerSwiGLU has none: SiLU
    return type(mlp) is MetalLigerSwiGLU if act is None else activation_name(act) == "silu"


def _fusable(mlp: nn.Module) -> bool:
    """A gated MLP of such parts whose own forward computes their formula and nothing
    else."""
    return _gated(mlp) and (type(mlp) is MetalLigerSwiGLU and "forward" not in mlp.__dict__
                            or computes(mlp, _gated_formula, *_PROJECTIONS, "act_fn"))


class MetalLigerSwiGLUMLP(nn.Module):
    """Drop-in for a gated MLP (gate_proj, up_proj, down_proj without bias, SiLU), whose
    projections it keeps under their names (state_dict keys are unchanged); forward also
    takes a residual to add. Where a projection has become something else since (an
    adapter's wrapper, a hook, a bias), under autocast, in forward mode and for inputs of
    another dtype, forward calls the projections themselves."""

    def __init__(self, original_mlp: nn.Module, checkpoint: str | None = None):
        super().__init__()
        check_checkpoint(checkpoint)
        # (a routed module is one already; one without a forward only holds the parts)
        if not (_fusable(original_mlp) or _gated(original_mlp) and
                (type(original_mlp).forward is nn.Module.forward or
                 isinstance(original_mlp.__dict__.get("forward"), _FusedMLPForward))):
            raise ValueError("MetalLigerSwiGLUMLP: gate_proj, up_proj and down_proj must be plain "
                             "nn.Linear layers without bias, on SiLU, in a forward of nothing else "
                             f"(got {original_mlp})")
        self.gate_proj = original_mlp.gate_proj
        self.up_proj = original_mlp.up_proj
        self.down_proj = original_mlp.down_proj
        self.checkpoint = checkpoint

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        gate, up, down = self.gate_proj, self.up_proj, self.down_proj
        if _plain_projections(self) and takes(x, gate, up, down):
            return fused_swiglu_mlp(x, gate.weight, up.weight, down.weight, residual,
                                    self.checkpoint)
        y = down(F.silu(gate(x)) * up(x))
        return y if residual is None else y + residual

    def extra_repr(self) -> str:
        return f"checkpoint={self.checkpoint}"


class _FusedMLPForward:
    """Forward of a routed MLP: the fused block, or the module's own forward where its
    parts, looked at in every call, are no longer what _gated asks for (an adapter was
    added since, a bias, a hook, another activation), under autocast, in forward mode and
    for inputs of another dtype."""

    def __init__(self, mlp: nn.Module, original, checkpoint: str | None):
        self.mlp, self.original, self.checkpoint = mlp, original, checkpoint

    def __call__(self, *args, **kwargs):
        x, = (*args, *kwargs.values())  # (by whatever name)
        if not _gated(self.mlp) or hooked(getattr(self.mlp, "act_fn", None)):
            return self.original(x)
        gate, up, down = (getattr(self.mlp, name) for name in _PROJECTIONS)
        if not takes(x, gate, up, down):
            return self.original(x)
        return fused_swiglu_mlp(x, gate.weight, up.weight, down.weight, checkpoint=self.checkpoint)


def patch_swiglu_mlp(model: nn.Module, checkpoint: str | None = None) -> int:
    """Routes the decoder layers' gated MLPs without adapters through the fused block and
    returns how many were routed. Only the instances' ``forward`` changes; modules
    already routed (here or to the LoRA block) are left as they are."""
    check_checkpoint(checkpoint)
    layers = find_layers(model)
    if layers is None:
        logger.warning("MetalLiger fused MLP: could not find transformer layers")
        return 0
    routed = 0
    for layer in layers:
        mlp = getattr(layer, "mlp", None)
        if mlp is None or not _fusable(mlp):
            continue
        mlp.forward = _FusedMLPForward(mlp, mlp.forward, checkpoint)
        routed += 1
    logger.info(f"MetalLiger fused MLP: activated on {routed} modules.")
    return routed
