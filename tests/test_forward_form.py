"""What the patchers read of a forward, and which modules they leave alone for it."""

import copy
import functools

import pytest
import torch
import torch.nn as nn

from metal_liger_amd._forward_form import add, arg, call, form, item, mul, passed_on
from metal_liger_amd.ops import fused_add_rms_norm as fa
from metal_liger_amd.ops import fused_linear as fl
from metal_liger_amd.ops.fused_rms_norm import MetalLigerRMSNorm
from tests import qwen_tiny
from tests.parity import seeded

h = arg("h")


class Forms:
    def plain(self, h, n: int = 3, *, flag=None, **kw):
        """Text."""
        r = h
        h, _ = self.a(self.b(r), n, flag=flag, **kw)
        return r + h

    def product(self, h):
        return self.a(self.b(h) * self.c(h)) + h

    def chained(self, h):
        a = b = self.a(h)
        return a + b

    def twice(self, h):
        return self.a(h) + self.a(h)

    def branch(self, h):
        if self.flag:
            h = self.a(h)
        return h

    def early(self, h):
        return h
        return self.a(h)

    def in_place(self, h):
        r = self.a(h)
        r += h
        return r

    def statement(self, h):
        self.a(h)
        return h

    def scaled(self, h):
        return h + 0.5 * self.a(h)

    def attribute(self, h):
        return h + self.scale * self.a(h)

    def method(self, h):
        return self.a(h).float()

    def deeper(self, h):
        return self.a.b(h)

    def outside(self, h):
        return torch.relu(self.a(h))

    def state(self, h):
        self.last = self.a(h)
        return h

    def indexed(self, h):
        return self.a(h)[0]

    def star(self, *hs):
        return self.a(*hs)

    def nothing(self, h):
        self.a(h)

    def none(self, h):
        return


def test_forms():
    f = form(Forms.plain)
    assert f.params == ("h", "n", "flag") and f.var_kw == "kw"
    got = call("a", call("b", h), arg("n"), kwargs={"flag": arg("flag")}, star=arg("kw"))
    assert f.value == add(item(0, 2, got), h) and f.calls == ("b", "a") and f.adds == 1
    assert passed_on(f, "h") == dict(kwargs={"n": arg("n"), "flag": arg("flag")}, star=arg("kw"))
    f = form(Forms.product)
    assert f.value == add(h, call("a", mul(call("c", h), call("b", h)))) and f.var_kw is None
    # a result used twice, and a part called twice: the same value, other calls
    once, twice = form(Forms.chained), form(Forms.twice)
    assert once.value == twice.value and once.calls == ("a",) and twice.calls == ("a", "a")


@pytest.mark.parametrize("name", ["branch", "early", "in_place", "statement", "scaled", "attribute",
                                  "method", "deeper", "outside", "state", "indexed", "star",
                                  "nothing", "none"])
def test_other_forwards_have_no_form(name):
    assert form(getattr(Forms, name)) is None


def test_what_is_not_a_function_as_written():
    def doubling(fn):
        @functools.wraps(fn)
        def wrapper(*args, **kwargs):
            return 2 * fn(*args, **kwargs)
        return wrapper

    assert form(doubling(Forms.product)) is None  # the wrapper's own form counts
    assert form(len) is None and form(functools.partial(Forms.product)) is None
    assert form(lambda self, h: self.a(h)) is None
    scope = {}
    exec("def made(self, h):\n    return self.a(h)", scope)  # no source to read
    assert form(scope["made"]) is None


# ------------------------------------------------------------- vision blocks --

class Same(nn.Module):
    """transformers' block in other words."""

    def __init__(self, block):
        super().__init__()
        self.norm1, self.norm2, self.attn, self.mlp = block.norm1, block.norm2, block.attn, block.mlp
        self.ls1, self.half = nn.Linear(64, 64), 0.5
        self.drop_path = nn.Dropout(0.5)

    def forward(self, hidden_states, cu_seqlens, **kwargs):
        normed = self.norm1(hidden_states)
        h = self.attn(normed, cu_seqlens=cu_seqlens, **kwargs) + hidden_states
        return h + self.mlp(self.norm2(h))


class LayerScale(Same):
    def forward(self, hidden_states, **kwargs):
        hidden_states = hidden_states + self.ls1(self.attn(self.norm1(hidden_states), **kwargs))
        return hidden_states + self.mlp(self.norm2(hidden_states))


class DropPath(Same):
    def forward(self, hidden_states, **kwargs):
        hidden_states = hidden_states + self.drop_path(self.attn(self.norm1(hidden_states), **kwargs))
        hidden_states = hidden_states + self.drop_path(self.mlp(self.norm2(hidden_states)))
        return hidden_states


class Factor(Same):
    def forward(self, hidden_states, **kwargs):
        hidden_states = hidden_states + 0.5 * self.attn(self.norm1(hidden_states), **kwargs)
        hidden_states = hidden_states + self.mlp(self.norm2(hidden_states))
        return hidden_states


class Parallel(Same):
    def forward(self, hidden_states, **kwargs):
        h = hidden_states + self.attn(self.norm1(hidden_states), **kwargs)
        h = h + self.mlp(self.norm2(hidden_states))
        return h


class OwnArguments(Same):
    """One argument is not attn's, another is handed on changed."""

    def forward(self, hidden_states, layer=None, **kwargs):
        hidden_states = hidden_states + self.attn(self.norm1(hidden_states), **kwargs)
        hidden_states = hidden_states + self.mlp(self.norm2(hidden_states))
        return hidden_states


class OtherResidual(Same):
    def forward(self, hidden_states, **kwargs):
        normed = self.norm1(hidden_states)
        h = normed + self.attn(normed, **kwargs)
        h = h + self.mlp(self.norm2(h))
        return h


def _tower(cls):
    model = qwen_tiny.build_vl()
    block = cls(model.model.visual.blocks[0])
    model.model.visual.blocks[0] = block
    block.attn.forward = lambda h, **kw: 0.25 * h  # (its arguments do not matter here)
    return model, block


@pytest.mark.parametrize("cls", [LayerScale, DropPath, Factor, Parallel, OwnArguments, OtherResidual])
def test_other_blocks_keep_their_forward(cls, monkeypatch):
    model, block = _tower(cls)
    own = copy.deepcopy(block).eval()
    assert fl.patch_vision_mlp(model) == 1  # the MLP, not the block
    assert "forward" not in block.__dict__
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device=None: True)
    x = seeded((4, 64), 1)
    assert torch.equal(block.eval()(x), own(x))


def test_blocks_that_compute_the_same_are_routed(monkeypatch):
    model, block = _tower(Same)
    own = copy.deepcopy(block)
    assert fl.patch_vision_mlp(model) == 1
    assert type(block.forward) is fl._FusedVisionBlockForward
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device=None: True)
    x = seeded((4, 64), 1)
    assert torch.equal(block(x, None), own(x, None))
    assert fl._fusable_block(fl_block := qwen_tiny.build_vl().model.visual.blocks[0]) is False
    fl.patch_vision_mlp(fl_block)
    assert type(fl_block.forward) is fl._FusedVisionBlockForward


def test_a_block_whose_mlp_was_replaced(monkeypatch):
    """After the block was routed, its MLP is wrapped or given another forward."""
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device=None: True)
    x = seeded((4, 64), 1)
    for change in (lambda b: setattr(b, "mlp", nn.Sequential(b.mlp)),
                   lambda b: setattr(b.mlp, "forward", lambda t: 2 * t)):
        model, block = _tower(Same)
        own = copy.deepcopy(block)
        assert fl.patch_vision_mlp(model) == 1
        change(block)
        change(own)
        assert torch.equal(block(x, None), own(x, None))


# ------------------------------------------------------------ decoder layers --

class DecoderLayer(nn.Module):
    def __init__(self):
        super().__init__()
        self.input_layernorm, self.post_attention_layernorm = MetalLigerRMSNorm(8), MetalLigerRMSNorm(8)
        self.self_attn, self.mlp, self.residual_multiplier = nn.Identity(), nn.Identity(), 0.5

    def forward(self, hidden_states, attention_mask=None, **kwargs):
        attn, _ = self.self_attn(hidden_states=self.input_layernorm(hidden_states),
                                 attention_mask=attention_mask, **kwargs)
        hidden_states = hidden_states + attn
        return hidden_states + self.mlp(self.post_attention_layernorm(hidden_states))


class ScaledLayer(DecoderLayer):
    def forward(self, hidden_states, **kwargs):
        residual = hidden_states
        hidden_states = self.input_layernorm(hidden_states)
        hidden_states, _ = self.self_attn(hidden_states=hidden_states, **kwargs)
        hidden_states = residual + hidden_states * self.residual_multiplier
        residual = hidden_states
        hidden_states = self.post_attention_layernorm(hidden_states)
        hidden_states = self.mlp(hidden_states)
        hidden_states = residual + hidden_states * self.residual_multiplier
        return hidden_states


class NormedResidualLayer(DecoderLayer):
    def forward(self, hidden_states, **kwargs):
        hidden_states = self.input_layernorm(hidden_states)
        attn, _ = self.self_attn(hidden_states=hidden_states, **kwargs)
        hidden_states = hidden_states + attn
        hidden_states = hidden_states + self.mlp(self.post_attention_layernorm(hidden_states))
        return hidden_states


def test_decoder_layers():
    assert fa.patch_residual_add_norm(DecoderLayer()) == 1
    for cls in (ScaledLayer, NormedResidualLayer):
        assert fa.patch_residual_add_norm(cls()) == 0
