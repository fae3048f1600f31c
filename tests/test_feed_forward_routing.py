"""Which MLPs the feed-forward patchers take, and what routed modules do once their parts
have changed (no GPU needed: the fused operators are stood in for by their formulas)."""

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from metal_liger_amd.ops import fused_linear as fl
from metal_liger_amd.ops import fused_swiglu_mlp as fm
from metal_liger_amd.ops.fused_swiglu import MetalLigerSwiGLU
from tests.parity import seeded
from tests.peft_shim import LoraLinear, init_lora

ACTS = {None: lambda z: z, "silu": F.silu, "gelu": F.gelu,
        "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}


@pytest.fixture
def formulas(monkeypatch):
    """The fused operators by their formulas; the calls that reach them."""
    calls = []

    def linear(x, weight, bias=None, activation=None, residual=None, checkpoint=None):
        calls.append("linear")
        y = ACTS[activation](F.linear(x, weight, bias))
        return y if residual is None else residual + y

    def mlp(x, wg, wu, wd, residual=None, checkpoint=None):
        calls.append("mlp")
        y = F.linear(F.silu(F.linear(x, wg)) * F.linear(x, wu), wd)
        return y if residual is None else y + residual

    monkeypatch.setattr(fl, "fused_linear", linear)
    monkeypatch.setattr(fm, "fused_swiglu_mlp", mlp)
    return calls


# ------------------------------------------------------------- own forwards --

class Gated(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj, self.up_proj = (nn.Linear(24, 40, bias=False) for _ in range(2))
        self.down_proj, self.act_fn = nn.Linear(40, 24, bias=False), nn.SiLU()
        self.dropout, self.scale = nn.Dropout(0.5), 0.5

    def forward(self, hidden):
        gate = self.act_fn(self.gate_proj(hidden))
        return self.down_proj(self.up_proj(hidden) * gate)


class GatedDropout(Gated):
    def forward(self, x):
        return self.dropout(self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)))


class GatedFactor(Gated):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)) * self.scale


class GatedOther(Gated):
    def forward(self, x):
        return self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x))


class GatedWithArguments(Gated):
    def forward(self, x, scale=1.0):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x) * scale)


class Vision(nn.Module):
    def __init__(self):
        super().__init__()
        self.linear_fc1, self.linear_fc2, self.act_fn = nn.Linear(24, 40), nn.Linear(40, 24), nn.GELU()
        self.dropout = nn.Dropout(0.5)

    def forward(self, x):
        x = self.act_fn(self.linear_fc1(x))
        return self.linear_fc2(x)


class VisionDropout(Vision):
    def forward(self, x):
        return self.linear_fc2(self.dropout(self.act_fn(self.linear_fc1(x))))


class VisionFactor(Vision):
    def forward(self, x):
        return self.linear_fc2(self.act_fn(self.linear_fc1(x))) * 0.5


class VisionAddition(Vision):
    def forward(self, x):
        return x + self.linear_fc2(self.act_fn(self.linear_fc1(x)))


class Doubled(nn.SiLU):
    def forward(self, x):
        return 2 * super().forward(x)


class DoubledGELU(nn.GELU):
    def forward(self, x):
        return 2 * super().forward(x)


class GELUActivation(nn.Module):
    """A name of transformers', another formula."""

    def forward(self, x):
        return x.clamp_min(0)


def _layers(mlp):
    root, layer = nn.Module(), nn.Module()
    layer.mlp, layer.self_attn = mlp, nn.Module()
    root.layers = nn.ModuleList([layer])
    return root


def test_same_formula_is_routed(formulas):
    mlp, x = Gated(), seeded((3, 24), 1)
    want = mlp(x)
    assert fm.patch_swiglu_mlp(_layers(mlp)) == 1
    for y in (mlp(x), mlp(hidden=x)):
        assert torch.allclose(y, want, atol=1e-6)
    vision = Vision()
    want = vision(x)
    assert fl.patch_vision_mlp(vision) == 1
    for y in (vision(x), vision(x=x), vision(x, residual=x) - x):
        assert torch.allclose(y, want, atol=1e-6)
    assert formulas == 2 * ["mlp"] + 6 * ["linear"]
    wrapped = MetalLigerSwiGLU(Gated())
    assert fm.patch_swiglu_mlp(_layers(wrapped)) == 1


@pytest.mark.parametrize("cls", [GatedDropout, GatedFactor, GatedOther, GatedWithArguments])
def test_other_gated_mlps_keep_their_forward(cls):
    mlp = cls()
    assert fm.patch_swiglu_mlp(_layers(mlp)) == 0 and "forward" not in mlp.__dict__
    with pytest.raises(ValueError, match="nothing else"):
        fm.MetalLigerSwiGLUMLP(mlp)


@pytest.mark.parametrize("cls", [VisionDropout, VisionFactor, VisionAddition])
def test_other_vision_mlps_keep_their_forward(cls):
    mlp = cls()
    assert fl.patch_vision_mlp(mlp) == 0 and "forward" not in mlp.__dict__


def test_replaced_forwards_are_kept():
    """A forward set on the instance (a framework's hook) is not what its class computes."""
    for mlp, patch in ((Gated(), lambda m: fm.patch_swiglu_mlp(_layers(m))),
                       (MetalLigerSwiGLU(Gated()), lambda m: fm.patch_swiglu_mlp(_layers(m))),
                       (Vision(), fl.patch_vision_mlp)):
        mlp.forward = lambda x: 2 * x
        assert patch(mlp) == 0 and torch.equal(mlp(torch.ones(3)), 2 * torch.ones(3))
    with pytest.raises(ValueError, match="nothing else"):
        mlp = Gated()
        mlp.forward = lambda x: 2 * x
        fm.MetalLigerSwiGLUMLP(mlp)


def test_activations_of_another_formula():
    for act in (Doubled(), DoubledGELU(), GELUActivation()):
        assert fl.activation_name(act) is None
        mlp, vision = Gated(), Vision()
        mlp.act_fn = vision.act_fn = act
        assert fm.patch_swiglu_mlp(_layers(mlp)) == fl.patch_vision_mlp(vision) == 0
    act = nn.SiLU()
    act.forward = lambda x: x
    assert fl.activation_name(act) is None and fl.activation_name(F.silu) is None


def test_a_module_that_only_holds_the_parts():
    parts, own = nn.Module(), Gated()
    for name in ("gate_proj", "up_proj", "down_proj", "act_fn"):
        setattr(parts, name, getattr(own, name))
    assert fm.MetalLigerSwiGLUMLP(parts).up_proj is own.up_proj
    assert fm.patch_swiglu_mlp(_layers(own)) == 1
    assert fm.MetalLigerSwiGLUMLP(own).up_proj is own.up_proj  # a routed one


# ------------------------------------------------- parts that change afterwards --

def _biased(linear):
    new = nn.Linear(linear.in_features, linear.out_features)
    new.weight = linear.weight
    return new


CHANGES = {
    "another layer, with a bias": lambda m: setattr(m, "up_proj", _biased(m.up_proj)),
    "a bias": lambda m: setattr(m.down_proj, "bias", nn.Parameter(torch.ones(24))),
    "another activation": lambda m: setattr(m, "act_fn", nn.GELU()),
    "an activation's forward": lambda m: setattr(m.act_fn, "forward", lambda x: x),
    "a subclass": lambda m: setattr(m, "act_fn", Doubled()),
    "another dtype": lambda m: m.double(),
}


@pytest.mark.parametrize("change", list(CHANGES))
def test_a_gated_mlp_changed_after_it_was_routed(formulas, change):
    mlp, own = Gated(), Gated()
    own.load_state_dict(mlp.state_dict())
    assert fm.patch_swiglu_mlp(_layers(mlp)) == 1
    x = seeded((3, 24), 1)
    mlp(x)
    with torch.random.fork_rng():
        for m in (mlp, own):
            torch.manual_seed(0)
            CHANGES[change](m)
    x = x.to(mlp.up_proj.weight.dtype)
    if change == "another dtype":  # (fp64 is none of the operator's)
        assert formulas == ["mlp"]
    assert torch.equal(mlp(x), own(x)) and formulas == ["mlp"]


def test_a_vision_mlp_changed_after_it_was_routed(formulas):
    x = seeded((3, 24), 1)
    for change, same_op in ((lambda m: setattr(m, "act_fn", nn.ReLU()), False),
                            (lambda m: setattr(m, "act_fn", Doubled()), False),
                            (lambda m: setattr(m, "act_fn", nn.SiLU()), True),
                            (lambda m: setattr(m.act_fn, "approximate", "tanh"), True)):
        mlp, own = Vision(), Vision()
        own.load_state_dict(mlp.state_dict())
        assert fl.patch_vision_mlp(mlp) == 1 and mlp.forward.activation == "gelu"
        change(mlp)
        change(own)
        del formulas[:]
        assert torch.allclose(mlp(x), own(x), atol=1e-6) and (formulas == 2 * ["linear"]) == same_op


def _with_adapter(m):
    m.gate_proj = LoraLinear(m.gate_proj, r=4, alpha=8)
    init_lora(m.gate_proj, 3, b_std=0.3)


def _with_hook(m):
    m.up_proj.register_forward_hook(lambda module, args, out: 2 * out)


@pytest.mark.parametrize("change", [None, _with_adapter, _with_hook, CHANGES["a bias"],
                                    CHANGES["another layer, with a bias"], CHANGES["another dtype"]])
def test_the_module_after_its_projections_changed(formulas, change):
    """What the projections have become counts, in the output and for the gradients."""
    own = Gated()
    m = fm.MetalLigerSwiGLUMLP(own)  # (the same projections)
    x, fused = seeded((3, 24), 1), ["mlp", "mlp"] if change is None else []
    if change is not None:
        with torch.random.fork_rng():
            torch.manual_seed(0)
            change(m)
        own.gate_proj, own.up_proj, own.down_proj = m.gate_proj, m.up_proj, m.down_proj
    x = x.to(own.up_proj.weight.dtype)
    for y, want in ((m(x), own(x)), (m(x, x), own(x) + x)):
        assert torch.allclose(y, want, atol=1e-6)
        y.sum().backward()
    assert formulas == fused and all(p.grad is not None for p in m.parameters())


def test_the_module_under_autocast(formulas, monkeypatch):
    m, x = fm.MetalLigerSwiGLUMLP(Gated()), seeded((3, 24), 1)
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device=None: True)
    m(x)
    assert formulas == []


class Sharded(torch.Tensor):
    """A tensor subclass: what its products are is its own matter."""


@pytest.mark.parametrize("part", ["x", "weight"])
def test_tensor_subclasses(formulas, part):
    x = seeded((3, 24), 1)
    mlp, vision, own = Gated(), Vision(), Gated()
    module = fm.MetalLigerSwiGLUMLP(own)
    wants = [m(x) for m in (mlp, vision, own)]
    assert fm.patch_swiglu_mlp(_layers(mlp)) == fl.patch_vision_mlp(vision) == 1
    if part == "x":
        x = x.as_subclass(Sharded)
    else:
        for m in (mlp.down_proj, vision.linear_fc2, module.gate_proj):
            m.weight = nn.Parameter(m.weight.detach().as_subclass(Sharded))
    for m, want in zip((mlp, vision, module), wants):
        assert torch.equal(m(x).as_subclass(torch.Tensor), want)
    assert formulas == []
