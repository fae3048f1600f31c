"""The feed-forward operators outside plain reverse mode, without a GPU: the ops are stood
in for by their formulas, registered as the ops are."""

import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from metal_liger_amd import _custom_ops as cops
from metal_liger_amd.ops.fused_linear import fused_linear, patch_vision_mlp
from metal_liger_amd.ops.fused_swiglu_mlp import (MetalLigerSwiGLUMLP, fused_swiglu_mlp,
                                                  patch_swiglu_mlp)
from tests import qwen_tiny
from tests.parity import seeded

_linear = cops._define(
    "test_linear_infer(Tensor x2, Tensor w, Tensor? bias, Tensor? residual, int act) -> Tensor",
    lambda x2, w, bias, residual, act: F.linear(x2, w, bias),
    lambda x2, w, bias, residual, act: x2.new_empty((x2.shape[0], w.shape[0])))
_mlp = cops._define(
    "test_swiglu_mlp_infer(Tensor x2, Tensor wg, Tensor wu, Tensor wd, Tensor? residual) -> Tensor",
    lambda x2, wg, wu, wd, residual: F.linear(F.silu(F.linear(x2, wg)) * F.linear(x2, wu), wd),
    lambda x2, wg, wu, wd, residual: x2.new_empty((x2.shape[0], wd.shape[0])))


@pytest.fixture
def cpu_ops(monkeypatch):
    monkeypatch.setattr(cops, "linear_infer", _linear)
    monkeypatch.setattr(cops, "swiglu_mlp_infer", _mlp)


CALLS = [lambda x, w: fused_linear(x, w), lambda x, w: fused_swiglu_mlp(x, w, w, w.t())]


@pytest.mark.parametrize("call", CALLS)
def test_forward_mode_is_refused(cpu_ops, call):
    """Frozen weights, an input with a tangent: an error, no output without its tangent."""
    x, w = seeded((3, 8), 1), seeded((4, 8), 2)
    want = call(x, w)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            for a, b in ((forward_ad.make_dual(x, x), w), (x, forward_ad.make_dual(w, w))):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call(a, b)
            assert torch.equal(call(x, w), want)  # no tangent, nothing to refuse
        with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(lambda t: call(t, w), (x,), (x,))
    assert torch.equal(call(x, w), want)


def test_routed_modules_have_their_own_tangents(cpu_ops):
    model, own = qwen_tiny.build_vl().requires_grad_(False), qwen_tiny.build_vl()
    assert patch_swiglu_mlp(model) == 2 and patch_vision_mlp(model) == 1
    for at, width in ((lambda m: m.model.language_model.layers[0].mlp, 128),
                      (lambda m: m.model.visual.blocks[0].mlp, 64)):
        x, dx = seeded((3, width), 1), seeded((3, width), 2)
        got, want = (torch.func.jvp(at(m), (x,), (dx,)) for m in (model, own))
        assert want[1].abs().max() > 0
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("call", CALLS)
def test_compiled_whole(call):
    """Traced without a break, up to the op itself, which refuses the CPU."""
    step = torch.compile(call, fullgraph=True, backend="eager")
    with pytest.raises(Exception, match="ROCm GPU"):
        step(seeded((3, 8), 1), seeded((4, 8), 2))


def test_compiled_modules():
    """Modules too, their checks in each call included."""
    model = qwen_tiny.build_vl()
    mlp, vision = model.model.language_model.layers[0].mlp, model.model.visual.blocks[0].mlp
    own = MetalLigerSwiGLUMLP(mlp)
    assert patch_swiglu_mlp(model) == 2 and patch_vision_mlp(model) == 1
    for m, width in ((own, 128), (mlp, 128), (vision, 64)):
        step = torch.compile(lambda x: m(x), fullgraph=True, backend="eager")
        with pytest.raises(Exception, match="ROCm GPU"):
            step(seeded((3, width), 1))
