"""Fused SwiGLU on MI355X (drop-in for the reference's ops/fused_swiglu.py).

One streaming HIP kernel each way. Unlike the reference, which kept
sigmoid(gate) as an extra fp32 tensor for backward (ops/fused_swiglu.py:34),
sigmoid is recomputed in the backward kernel: it costs no HBM traffic there,
while the saved tensor cost 4 bytes per element of memory and traffic.

checkpoint="fp8" keeps gate and up for the backward in 8 bits (e4m3 with a power of two
as scale for every 32 elements of the last dimension), written by the forward's kernel
and read by the backward's: 33 bytes for 32 elements of a tensor that takes 64 in bf16.
"""

import torch
import torch.nn as nn

from metal_liger_amd import _custom_ops as cops
from metal_liger_amd.ops.fused_linear import check_checkpoint


class _FusedSwiGLUFunction(torch.autograd.Function):
    """silu(gate) * up, computed in fp32 and rounded to gate's dtype
    (ops/fused_swiglu.py:18-50); grads in gate's / up's dtype."""

    @staticmethod
    def forward(ctx, gate: torch.Tensor, up: torch.Tensor):
        output = cops.swiglu_fwd(gate, up)
        ctx.save_for_backward(gate, up)
        return output

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor):
        gate, up = ctx.saved_tensors
        grad_gate, grad_up = cops.swiglu_bwd(gate, up, grad_output)
        return grad_gate, grad_up


class _FusedSwiGLUKeptFunction(torch.autograd.Function):
    """_FusedSwiGLUFunction with gate and up kept in 8 bits. First derivatives only."""

    @staticmethod
    def forward(ctx, gate: torch.Tensor, up: torch.Tensor):
        output, *kept = cops.swiglu_kept_fwd(gate, up)
        ctx.save_for_backward(*kept)
        ctx.dtypes = gate.dtype, up.dtype
        return output

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor):
        return cops.swiglu_kept_bwd(*ctx.saved_tensors, grad_output, *ctx.dtypes)


def fused_swiglu(gate: torch.Tensor, up: torch.Tensor,
                 checkpoint: str | None = None) -> torch.Tensor:
    """Functional: SiLU(gate) * up in a single fused op (ops/fused_swiglu.py:54-56).
    checkpoint: None, or "fp8" to keep gate and up in 8 bits for the backward, whose
    gradients are then those at the values that the 8 bits stand for."""
    check_checkpoint(checkpoint)
    if checkpoint is None or not (torch.is_grad_enabled()
                                  and (gate.requires_grad or up.requires_grad)):
        return _FusedSwiGLUFunction.apply(gate, up)
    return _FusedSwiGLUKeptFunction.apply(gate, up)


class MetalLigerSwiGLU(nn.Module):
    """Drop-in for a SwiGLU MLP block; fuses the activation step only
    (ops/fused_swiglu.py:59-75). Keeps gate_proj / up_proj / down_proj under
    their original names so state_dict keys are unchanged. checkpoint: as
    fused_swiglu's."""

    checkpoint = None

    def __init__(self, original_mlp: nn.Module, checkpoint: str | None = None):
        super().__init__()
        check_checkpoint(checkpoint)
        self.checkpoint = checkpoint
        self.gate_proj = original_mlp.gate_proj
        self.up_proj = original_mlp.up_proj
        self.down_proj = original_mlp.down_proj

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        gate = self.gate_proj(x)
        up = self.up_proj(x)
        activated = fused_swiglu(gate, up, self.checkpoint)
        return self.down_proj(activated)

    def extra_repr(self) -> str:
        return "fused=MetalLiger-Phase3"
