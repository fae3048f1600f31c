"""Fused linear layer on MI355X: y = act(x W^T + bias) + residual in one product with an
epilogue, and its backward (no counterpart in the reference, whose models keep
nn.Linear around their activations and residual adds).

The sum over K, the bias, the activation and the residual are added up in fp32 and y is
rounded once. The backward needs z = x W^T + bias where there is an activation: it is
kept in 16 bits (fp16 with a power of two as scale for every 32 columns of a row, which
rounds finer than bf16; fp32 in fp32), or in 8 (checkpoint="fp8": e4m3 with such
scales), formed of the fp32 sums. What is not needed (x where the
weight is frozen, W where x needs no gradient) is not kept. First derivatives only, in
reverse mode (forward mode is refused).

bf16 runs on the bf16 matrix cores, and dz is rounded to bf16 before its products (not in
db's sum); fp32 and fp16 run on the fp32 ones, with everything between input and output in
fp32 (fp16 forwards of up to 128 rows on the fp16 ones: the same products and sums, exact
and in fp32). The kernels take 16-bit sizes in multiples of 8, and
fp32 ones faster: others are padded with zeros, which add nothing.
"""

from __future__ import annotations

import inspect
import logging

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from metal_liger_amd import _custom_ops as cops
from metal_liger_amd import hip_ops
from metal_liger_amd._forward_form import add, arg, call, form, passed_on

logger = logging.getLogger(__name__)

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3}
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def check_checkpoint(checkpoint: str | None) -> None:
    if checkpoint not in (None, "fp8"):
        raise ValueError(f'checkpoint must be None or "fp8" (got {checkpoint!r})')


def keep_mode(checkpoint: str | None, dtype: torch.dtype) -> int:
    """How a backward's tensors are kept where the inputs are of `dtype`."""
    if checkpoint == "fp8":
        return hip_ops.KEEP_FP8
    return hip_ops.KEEP_F32 if dtype == torch.float32 else hip_ops.KEEP_FP16


def rows(t):
    """[..., C] -> [R, C]."""
    return t if t is None or t.dim() == 2 else t.reshape(-1, t.shape[-1])


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


def forward_mode() -> bool:
    """Whether forward-mode differentiation is at work (told by a private name; where
    torch has none, it is taken to be)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def wants_grad(*tensors) -> bool:
    """Whether a call goes through its autograd Function: for a backward, or to have
    forward mode refused there (the ops alone would drop the tangents)."""
    return forward_mode() or torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in tensors)


def _forward(x, weight, bias, residual, act: int, keep: int):
    """(y, z, zscale), or y alone where nothing is kept."""
    args = (rows(x), weight, bias, rows(residual), act)
    y, *kept = (cops.linear_infer(*args),) if keep == hip_ops.KEEP_NONE else \
        cops.linear_fwd(*args, keep)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0]), *kept


class _FusedLinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int, keep: int):
        need_dx, need_dw, need_db = ctx.needs_input_grad[:3]
        if act == 0 or not (need_dx or need_dw or need_db):
            keep = hip_ops.KEEP_NONE
        y, *kept = _forward(x, weight, bias, residual, act, keep)
        ctx.save_for_backward(x if need_dw else None, weight if need_dx else None, *kept)
        ctx.act, ctx.keep, ctx.sizes = act, keep, tuple(weight.shape)
        ctx.x_shape = x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        need_dx, need_dw, need_db, need_dr = ctx.needs_input_grad[:4]
        grads = [None, None, None]
        if need_dx or need_dw or need_db:
            x, weight, *kept = ctx.saved_tensors
            z, zscale = kept or (None, None)
            out = cops.linear_bwd(rows(x), weight, rows(dy), ctx.act, ctx.keep, z, zscale, *ctx.sizes,
                                  need_dx, need_dw, need_db)
            grads = [g if need else None for g, need in zip(out, ctx.needs_input_grad)]
            if need_dx and len(ctx.x_shape) != 2:
                grads[0] = grads[0].view(ctx.x_shape)
        return (*grads, dy if need_dr else None, None, None)


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 activation: str | None = None, residual: torch.Tensor | None = None,
                 checkpoint: str | None = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual.

    x [..., in], weight [out, in] (nn.Linear's), bias [out], residual [..., out]; all of
    x's dtype (fp32, bf16 or fp16; autocast casts none of them) and on its device, any
    strides. activation: None, "silu", "gelu" (by the error function, nn.GELU's default)
    or "gelu_tanh" (nn.GELU's approximate="tanh"); the residual is added after it.
    checkpoint: None, or "fp8" to keep what the activation's backward needs in 8 bits
    (module docstring).
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
    keep = keep_mode(checkpoint, x.dtype)
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


# ------------------------------------------------------------------ patching --

_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def hooked(module) -> bool:
    """Whether hooks want the module to be called, and to see what it returns."""
    return any(getattr(module, name, None) for name in _HOOKS)


def plain_linear(module) -> bool:
    """An nn.Linear as it is: an adapter's wrapper or a subclass may compute something
    else, and hooks (or a replaced forward) want the module to be called."""
    return (type(module) is nn.Linear and "forward" not in module.__dict__
            and not hooked(module))


_PLAIN = (torch.Tensor, nn.Parameter)


def takes(x, *linears) -> bool:
    """Whether a routed module's forward may run the fused op for x: its linear layers are
    of x's dtype, all are plain tensors (a subclass, sharded or quantized, has products of
    its own), autocast would not cast them, and no forward-mode derivative is wanted."""
    return (all(m.weight.dtype == x.dtype and type(m.weight) in _PLAIN for m in linears)
            and type(x) in _PLAIN and x.dtype in DTYPES and x.dim() > 0
            and not torch.is_autocast_enabled("cuda") and not forward_mode())


def activation_name(module) -> str | None:
    """The name in ACTIVATIONS of an activation module (nn's, or transformers' by its
    class name) as it is, None for any other: a subclass or a replaced forward may
    compute something else."""
    if "forward" in getattr(module, "__dict__", ()):
        return None
    if type(module) is nn.SiLU:
        return "silu"
    if type(module) is nn.GELU:
        return "gelu" if module.approximate == "none" else "gelu_tanh"
    if type(module).__module__ != "transformers.activations":
        return None
    # GELUTanh is gelu by tanh; GELUActivation is gelu, by torch or in Python
    return {"SiLUActivation": "silu", "GELUActivation": "gelu",
            "GELUTanh": "gelu_tanh", "PytorchGELUTanh": "gelu_tanh"}.get(type(module).__name__)


def computes(module: nn.Module, value, *parts: str) -> bool:
    """Whether a module's own forward has one argument x, returns value(x) and calls each
    of the parts once (_forward_form.py)."""
    f = form(type(module).forward) if "forward" not in module.__dict__ else None
    return (f is not None and len(f.params) == 1 and f.var_kw is None
            and sorted(f.calls) == sorted(parts) and f.value == value(arg(f.params[0])))


_VISION_PARTS = ("linear_fc1", "act_fn", "linear_fc2")


def _vision_formula(x):
    return call("linear_fc2", call("act_fn", call("linear_fc1", x)))


class _FusedVisionMLPForward:
    """Forward of a vision block's MLP, linear_fc2(act_fn(linear_fc1(x))), with the
    activation and (residual given) the block's addition in the products' epilogues. The
    module's own forward where its parts, looked at in every call, are no longer plain
    linear layers and an activation as it is, or takes() does not hold."""

    def __init__(self, mlp: nn.Module, original, checkpoint: str | None):
        self.mlp, self.original, self.checkpoint = mlp, original, checkpoint

    @property
    def activation(self) -> str | None:
        return activation_name(self.mlp.act_fn)

    def __call__(self, *args, residual=None, **kwargs):
        hidden_state, = (*args, *kwargs.values())  # (by whatever name)
        fc1, fc2, activation = self.mlp.linear_fc1, self.mlp.linear_fc2, self.activation
        if activation is None or hooked(self.mlp.act_fn) or \
                not (plain_linear(fc1) and plain_linear(fc2) and takes(hidden_state, fc1, fc2)):
            out = self.original(hidden_state)
            return out if residual is None else residual + out
        fused = residual is not None and residual.dtype == hidden_state.dtype and \
            residual.shape == (*hidden_state.shape[:-1], fc2.weight.shape[0])
        h = fused_linear(hidden_state, fc1.weight, fc1.bias, activation,
                         checkpoint=self.checkpoint)
        out = fused_linear(h, fc2.weight, fc2.bias, residual=residual if fused else None)
        return out if fused or residual is None else residual + out


_BLOCK_PARTS = ("norm1", "attn", "norm2", "mlp")


def _fusable_block(block: nn.Module) -> bool:
    """A vision block whose forward is h + attn(norm1(h), ...), then + mlp(norm2(h)), with
    every argument but h handed to attn."""
    if not all(hasattr(block, p) for p in _BLOCK_PARTS) or \
            not isinstance(block.mlp.__dict__.get("forward"), _FusedVisionMLPForward):
        return False
    f = form(type(block).forward)
    if f is None or f.calls != _BLOCK_PARTS or f.params[:1] != ("hidden_states",):
        return False
    h = arg("hidden_states")
    h = add(h, call("attn", call("norm1", h), **passed_on(f, "hidden_states")))
    return f.value == add(h, call("mlp", call("norm2", h)))


class _FusedVisionBlockForward:
    """Forward of a vision block, whose second addition its MLP makes. Every argument but
    hidden_states goes to attn, as the replaced forward passes them."""

    def __init__(self, block: nn.Module, original):
        self.block, self.signature = block, inspect.signature(original)
        self.var_kw = next((p.name for p in self.signature.parameters.values()
                            if p.kind is p.VAR_KEYWORD), None)

    def __call__(self, *args, **kwargs):
        bound = self.signature.bind(*args, **kwargs)
        bound.apply_defaults()
        rest = dict(bound.arguments)
        extra = rest.pop(self.var_kw, {}) if self.var_kw else {}
        h, b = rest.pop("hidden_states"), self.block
        h = h + b.attn(b.norm1(h), **rest, **extra)
        # (hooks see the MLP's own output; another MLP adds nothing)
        if hooked(b.mlp) or not isinstance(b.mlp.__dict__.get("forward"), _FusedVisionMLPForward):
            return h + b.mlp(b.norm2(h))
        return b.mlp(b.norm2(h), residual=h)


def patch_vision_mlp(model: nn.Module, checkpoint: str | None = None) -> int:
    """Routes the MLPs of a vision tower (modules with linear_fc1, act_fn and linear_fc2
    as Qwen3-VL's blocks have them, whose own forward computes linear_fc2(act_fn(
    linear_fc1(x))) and nothing else) through the fused linear layers, and the additions around them where a block's
    forward is transformers' (read from its source, _forward_form.py). Returns how many MLPs were routed; only the
    instances' ``forward`` changes, modules already routed are left as they are."""
    check_checkpoint(checkpoint)
    routed = 0
    for module in model.modules():
        if not all(hasattr(module, n) for n in _VISION_PARTS) or \
                getattr(module, "_metal_liger_vision_mlp", False):
            continue
        if not (plain_linear(module.linear_fc1) and plain_linear(module.linear_fc2)
                and activation_name(module.act_fn)
                and computes(module, _vision_formula, *_VISION_PARTS)):
            continue
        module.forward = _FusedVisionMLPForward(module, module.forward, checkpoint)
        module._metal_liger_vision_mlp = True
        routed += 1
    for module in model.modules():
        if "forward" not in module.__dict__ and _fusable_block(module):
            module.forward = _FusedVisionBlockForward(module, module.forward)
    logger.info(f"MetalLiger vision MLP: activated on {routed} modules.")
    return routed
