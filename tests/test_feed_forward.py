"""The feed-forward operators without a GPU: the oracle against torch, refusals, fake
kernels, the patcher's flags."""

import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode

from metal_liger_amd import _hip, apply_metal_liger_to_qwen3vl, hip_ops
from metal_liger_amd.ops import fused_linear as fl
from metal_liger_amd.ops import fused_lora as flora
from metal_liger_amd.ops import fused_swiglu as fs
from metal_liger_amd.ops import fused_swiglu_mlp as fm
from oracle import feed_forward as ref
from tests import qwen_tiny
from tests.parity import seeded
from tests.peft_shim import LoraLinear

BF, F32 = torch.bfloat16, torch.float32
ACTS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"),
        None: lambda z: z}


# ------------------------------------------------------------------- oracle --

@pytest.mark.parametrize("name", list(ACTS))
def test_oracle_activations(name):
    z = torch.linspace(-30, 30, 4001, dtype=torch.float64).requires_grad_()
    y = ACTS[name](z)
    g, = torch.autograd.grad(y.sum(), z)
    # torch's erf leaves an absolute error of eps where ndtr does not
    assert torch.allclose(ref.act(z.detach(), name), y.detach(), rtol=1e-12, atol=1e-14)
    assert torch.allclose(ref.act_grad(z.detach(), name), g, rtol=1e-12, atol=1e-14)
    if name:
        d = ref.act_grad(z.detach(), name)
        assert d.abs().max() <= ref.ACT_GRAD_MAX
        step = (z[1] - z[0]).item()
        assert ((d[1:] - d[:-1]) / step).abs().max() <= ref.ACT_GRAD2_MAX


@pytest.mark.parametrize("shape", [(1,), (31,), (4, 64), (3, 70), (2, 3, 33)])
def test_oracle_held_bytes(shape):
    """The bytes against torch's own e4m3 of the scaled values, and what they stand for."""
    v = seeded(shape, 1, F32, 3.0) * torch.exp(3 * seeded(shape, 2))
    v.view(-1)[0] = 0.0
    codes, scales = ref.held_bytes(v)
    s = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)[..., :shape[-1]]
    want = (v.double() / s).float().to(torch.float8_e4m3fn)
    assert torch.equal(codes, want.view(torch.uint8))
    assert torch.equal(ref.held_values(codes, scales), want.double() * s)
    m = F.pad(v.abs(), (0, -shape[-1] % 32)).unflatten(-1, (-1, 32)).amax(-1).double()
    top = m / torch.exp2(scales.double() - 127)
    assert bool(((top >= 128) & (top < 256) | (m == 0)).all())


def test_oracle_held_bytes_of_special_values():
    v = torch.zeros(32 * 4)
    v[:32] = torch.tensor([float("inf"), float("nan"), -float("inf"), 1.0] + [0.5] * 28)
    v[64:96] = 1e-42
    v[96:] = 3e38
    codes, scales = ref.held_bytes(v)
    assert scales.tolist() == [127 - 7, 1, 1, 127 + 127 - 7]
    got = ref.held_values(codes, scales)
    assert got[:3].isnan().all() and got[3] == 1.0 and bool((got[4:32] == 0.5).all())
    assert bool((got[32:96] == 0).all())
    assert bool((got[96:].float() == torch.tensor(3e38).view(1)).logical_or(
        (got[96:] - 3e38).abs() <= 2.0 ** -4 * 3e38).all())


# ----------------------------------------------------------------- refusals --

def t(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,error,match", [
    (lambda: fl.fused_linear(t(2, 8), t(4, 9)), ValueError, "does not fit"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8, 1)), ValueError, r"\[out, in\]"),
    (lambda: fl.fused_linear(t(2, 0), t(4, 0)), ValueError, r"\[out, in\]"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8, dtype=BF)), TypeError, "weight of"),
    (lambda: fl.fused_linear(t(2, 8, dtype=torch.float64), t(4, 8, dtype=torch.float64)), TypeError,
     "fp32, bf16 or fp16"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8), t(5)), ValueError, "bias"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8), t(4, dtype=BF)), ValueError, "bias"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8), residual=t(4)), ValueError, "residual"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8), residual=t(2, 4, dtype=BF)), ValueError, "residual"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8), activation="relu"), ValueError, "relu"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8), checkpoint="int8"), ValueError, "checkpoint"),
    (lambda: fl.fused_linear(t(2, 8), t(4, 8)), ValueError, "ROCm GPU"),
    (lambda: fm.fused_swiglu_mlp(t(2, 8), t(4, 8), t(5, 8), t(8, 4)), ValueError, "do not fit"),
    (lambda: fm.fused_swiglu_mlp(t(2, 8), t(4, 8), t(4, 8), t(8, 5)), ValueError, "do not fit"),
    (lambda: fm.fused_swiglu_mlp(t(2, 7), t(4, 8), t(4, 8), t(8, 4)), ValueError, "does not fit"),
    (lambda: fm.fused_swiglu_mlp(t(2, 8), t(4, 8), t(4, 8), t(8, 4), t(2, 4)), ValueError, "residual"),
    (lambda: fm.fused_swiglu_mlp(t(2, 8), t(4, 8), t(4, 8), t(8, 4), checkpoint=8), ValueError,
     "checkpoint"),
    (lambda: fm.fused_swiglu_mlp(t(2, 8), t(4, 8), t(4, 8), t(8, 4)), ValueError, "ROCm GPU"),
    (lambda: fs.fused_swiglu(t(2, 8), t(2, 8), checkpoint="bf16"), ValueError, "checkpoint"),
    (lambda: fs.fused_swiglu(t(2, 8).requires_grad_(), t(2, 8), checkpoint="fp8"), ValueError,
     "ROCm GPU"),
    (lambda: fl.MetalLigerLinear(nn.Identity()), ValueError, "nn.Linear"),
    (lambda: fl.MetalLigerLinear(nn.Linear(2, 2), "relu"), ValueError, "relu"),
    (lambda: fm.MetalLigerSwiGLUMLP(nn.Identity()), ValueError, "plain"),
    (lambda: fs.MetalLigerSwiGLU(nn.Identity(), "x"), ValueError, "checkpoint"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_host_side_argument_errors():
    """The C entry points refuse on the host; no pointer is read."""
    L = _hip.lib()
    p, q = 4096, 8192

    def refused(rc, word):
        assert rc == 1 and word in L.ml_last_error(), L.ml_last_error()

    def linear(x=p, ldx=64, w=p, ldw=64, bias=None, res=None, ldr=0, act=0, y=p, ldy=64, keep=0, z=None,
               zs=None, M=100, N=64, K=64, ws=p, wsb=1 << 40, dtype=1):
        return L.ml_linear_fwd(x, ldx, w, ldw, bias, res, ldr, act, y, ldy, keep, z, zs, M, N, K, ws,
                               wsb, dtype, None)

    refused(linear(M=0), b"bad sizes")
    refused(linear(M=1 << 31), b"bad sizes")
    refused(linear(M=(1 << 31) - 1), b"bad sizes")
    refused(linear(x=None), b"null pointer")
    refused(linear(act=4), b"bad activation")
    refused(linear(ldx=56), b"row strides")
    refused(linear(res=p, ldr=8), b"row strides")
    refused(linear(keep=9), b"bad way")
    refused(linear(keep=2), b"buffer is null")
    refused(linear(keep=2, z=p), b"scales")
    refused(linear(keep=2, z=p + 8, zs=p), b"16-byte aligned")
    refused(linear(keep=1, z=p), b"not kept as 1")
    refused(linear(dtype=0, keep=2, z=p, zs=p), b"not kept as 2")
    refused(linear(x=p + 2), b"16-byte aligned")
    refused(linear(K=60, ldx=64), b"multiples of 8")
    refused(linear(ldx=68), b"multiples of 8")
    refused(linear(bias=p + 2), b"bias")
    refused(linear(res=p, ldr=68), b"residual")
    refused(linear(M=1000, wsb=0, N=8, ldy=8, K=4096, ldx=4096, ldw=4096), b"workspace")
    refused(linear(dtype=2, keep=1, z=p), b"not kept as 1")
    refused(linear(dtype=2, x=p + 2), b"16-byte aligned")
    refused(linear(ldx=(1 << 21) + 8), b"up to")
    refused(linear(dtype=7), b"dtype tag 7")

    def linear_bwd(x=p, w=p, dy=p, ldy=64, act=0, keep=0, z=None, zs=None, dx=q, dw=q, db=q, M=100, N=64,
                   K=64, wsb=1 << 40, dtype=1):
        return L.ml_linear_bwd(x, 64, w, 64, dy, ldy, act, keep, z, zs, dx, dw, db, M, N, K, p, wsb,
                               dtype, None)

    refused(linear_bwd(dy=None), b"null pointer")
    refused(linear_bwd(w=None), b"null pointer")
    refused(linear_bwd(x=None), b"null pointer")
    refused(linear_bwd(act=1), b"no z was kept")
    refused(linear_bwd(ldy=72, dy=p + 4), b"dy")
    refused(linear_bwd(dx=q + 8), b"dx")
    refused(linear_bwd(wsb=0), b"workspace")
    refused(linear_bwd(dtype=9), b"dtype tag 9")
    assert linear_bwd(dx=None, dw=None, db=None) == 0

    def mlp(fn, *args, keep=0, kept=(None,) * 4, M=100, H=64, I=128, O=64, wsb=1 << 40, dtype=1):  # noqa: E741
        return fn(*args, keep, *kept, M, H, I, O, p, wsb, dtype, None)

    fwd = (p, 64, p, 64, p, 64, p, 128, None, 0, q)
    refused(mlp(L.ml_swiglu_mlp_fwd, *fwd, M=0), b"bad sizes")
    refused(mlp(L.ml_swiglu_mlp_fwd, *fwd, I=1 << 30), b"bad sizes")
    refused(mlp(L.ml_swiglu_mlp_fwd, *fwd, I=136), b"row strides")
    refused(mlp(L.ml_swiglu_mlp_fwd, *fwd, keep=3, kept=(p, p, None, None)), b"up")
    refused(mlp(L.ml_swiglu_mlp_fwd, *fwd, wsb=0), b"workspace")
    refused(mlp(L.ml_swiglu_mlp_fwd, *fwd, dtype=-1), b"dtype tag -1")
    refused(mlp(L.ml_swiglu_mlp_fwd, *fwd[:-1], None), b"null pointer")

    def mlp_bwd(dx=q, keep=3, kept=(p,) * 4, dy=p, wsb=1 << 40, dtype=1):
        return L.ml_swiglu_mlp_bwd(p, 64, p, 64, p, 64, p, 128, dy, 64, keep, *kept, dx, q, q, q, 100, 64,
                                   128, 64, p, wsb, dtype, None)

    refused(mlp_bwd(keep=0), b"not kept")
    refused(mlp_bwd(kept=(p, None, p, p)), b"scales")
    refused(mlp_bwd(dy=None), b"null pointer")
    refused(mlp_bwd(dx=q + 2), b"dx")
    refused(mlp_bwd(wsb=16), b"workspace")

    def pads(n=1, any_=p, strides=(16, 1), sizes=(3, 5), wide=q, wide_sizes=(8, 8), dtype=1):
        return L.ml_pad_matrices(n, _hip.ptrs([any_]), _hip.geom(strides), _hip.geom(sizes),
                                 _hip.ptrs([wide]), _hip.geom(wide_sizes), 1, dtype, None)

    refused(pads(n=0), b"0 matrices")
    refused(pads(n=9), b"9 matrices")
    refused(pads(sizes=(3, 9)), b"[3, 9] in [8, 8]")
    refused(pads(sizes=(9, 5)), b"[9, 5] in [8, 8]")
    refused(pads(sizes=(-1, 5)), b"[-1, 5]")
    refused(pads(wide_sizes=(8, 12)), b"[8, 12]")
    refused(pads(any_=None), b"null pointer")
    refused(pads(wide=q + 8), b"16-byte aligned")
    refused(pads(dtype=5), b"dtype tag 5")
    assert L.ml_pad_matrices(1, _hip.ptrs([None]), _hip.geom((8, 1)), _hip.geom((0, 5)),
                             _hip.ptrs([None]), _hip.geom((0, 8)), 1, 1, None) == 0

    refused(L.ml_swiglu_kept_fwd(p, p, q, p, p, p, p, -1, 8, 1, None), b"negative")
    refused(L.ml_swiglu_kept_fwd(p, p, q, p, None, p, p, 1, 8, 1, None), b"scales")
    refused(L.ml_swiglu_kept_fwd(p, p, q, p + 1, p, p, p, 1, 8, 1, None), b"16-byte aligned")
    refused(L.ml_swiglu_kept_bwd(p, p, p, p, None, q, q, 1, 8, 1, None), b"null pointer")
    refused(L.ml_swiglu_kept_fwd(p, p, q, p, p, p, p, 1, 8, 9, None), b"dtype")
    refused(L.ml_held_values(p, p, None, 1, 8, 1, None), b"null pointer")
    assert L.ml_swiglu_kept_fwd(None, None, None, None, None, None, None, 0, 8, 1, None) == 0


def test_workspaces():
    L = _hip.lib()
    fwd = L.ml_linear_fwd_workspace_bytes
    # few rows, and products that run their step as an epilogue, need none
    assert fwd(1, 64, 64, 1) == fwd(64, 4304, 1152, 1) == fwd(8192, 4304, 1152, 1) == 0
    # K split over workgroups: fp32 sums
    assert fwd(200, 2048, 2048, 1) >= 2 * 4 * 200 * 2048
    assert fwd(65, 64, 64, 0) >= 4 * 65 * 64
    assert fwd(0, 64, 64, 1) == fwd(64, 0, 64, 1) == fwd(64, 64, 1 << 31, 1) == 0
    act, none = (L.ml_linear_bwd_workspace_bytes(8192, 4304, 1152, a, 1) for a in (1, 0))
    assert act >= none + 2 * 8192 * 4304 - 512
    assert L.ml_swiglu_mlp_bwd_workspace_bytes(100, 64, 128, 64, 1) >= 3 * 2 * 100 * 128
    assert L.ml_swiglu_mlp_fwd_workspace_bytes(100, 64, 128, 64, 1) >= 2 * 100 * 128


# -------------------------------------------------------------------- fakes --

def test_fake_kernels():
    ops = torch.ops.metal_liger_amd

    def e(*shape, dtype=BF):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    def look(ts):
        return [(tuple(t.shape), t.dtype) for t in ts]

    U8, F16 = torch.uint8, torch.float16
    with FakeTensorMode():
        x, w, b = e(10, 64), e(72, 64), e(72)
        assert look(ops.linear_fwd(x, w, b, None, 1, 2)) == [((10, 72), BF), ((10, 72), F16),
                                                             ((10, 3), U8)]
        assert look(ops.linear_fwd(x, w, b, None, 1, 3)) == [((10, 72), BF), ((10, 72), U8),
                                                             ((10, 3), U8)]
        f = ops.linear_fwd(e(10, 64, dtype=F32), e(72, 64, dtype=F32), None, None, 1, 1)
        assert look(f) == [((10, 72), F32), ((10, 72), F32), ((0,), U8)]
        assert look([ops.linear_infer(x, w, b, e(10, 72), 0)]) == [((10, 72), BF)]
        z = ops.linear_fwd(x, w, b, None, 1, 2)
        out = ops.linear_bwd(x, w, e(10, 72), 1, 2, *z[1:], 72, 64, True, True, True)
        assert look(out) == [((10, 64), BF), ((72, 64), BF), ((72,), BF)]
        out = ops.linear_bwd(None, w, e(10, 72), 0, 0, None, None, 72, 64, True, False, False)
        assert look(out) == [((10, 64), BF), ((0,), BF), ((0,), BF)]
        ws = (e(96, 64), e(96, 64), e(40, 96))
        y = ops.swiglu_mlp_fwd(x, *ws, None, 3)
        assert look(y) == [((10, 40), BF)] + 2 * [((10, 96), U8), ((10, 3), U8)]
        assert look([ops.swiglu_mlp_infer(x, *ws, None)]) == [((10, 40), BF)]
        out = ops.swiglu_mlp_bwd(x, *ws, e(10, 40), 3, *y[1:], True, False, True, True)
        assert look(out) == [((10, 64), BF), ((0,), BF), ((96, 64), BF), ((40, 96), BF)]
        y = ops.linear_fwd(e(10, 33), e(45, 33), None, None, 1, 3)  # (kept at the padded width)
        assert look(y) == [((10, 45), BF), ((10, 48), U8), ((10, 2), U8)]
        out = ops.linear_bwd(e(10, 33), e(45, 33), e(10, 45), 1, 3, *y[1:], 45, 33, True, True, True)
        assert look(out) == [((10, 33), BF), ((45, 33), BF), ((45,), BF)]
        y = ops.linear_fwd(e(10, 33, dtype=F32), e(45, 33, dtype=F32), None, None, 1, 1)
        assert look(y) == [((10, 45), F32), ((10, 45), F32), ((0,), U8)]
        y = ops.swiglu_kept_fwd(e(2, 5, 70), e(2, 5, 70))
        assert look(y) == [((2, 5, 70), BF)] + 2 * [((2, 5, 70), U8), ((2, 5, 3), U8)]
        out = ops.swiglu_kept_bwd(*y[1:], e(2, 5, 70), BF, F32)
        assert look(out) == [((2, 5, 70), BF), ((2, 5, 70), F32)]
        assert look([ops.held_values(y[1], y[2], F32)]) == [((2, 5, 70), F32)]


# ------------------------------------------------------------------ patching --

def _decoder(model):
    return model.base_model.model.model.layers


def test_patcher_routes_gated_mlps():
    model = qwen_tiny.build(lora=False)
    keys = list(model.state_dict())
    apply_metal_liger_to_qwen3vl(model)
    assert all("forward" not in layer.mlp.__dict__ and layer.mlp.checkpoint is None
               for layer in _decoder(model))
    apply_metal_liger_to_qwen3vl(model, fuse_swiglu=False, fuse_mlp=True, mlp_checkpoint="fp8")
    for layer in _decoder(model):
        assert type(layer.mlp.forward) is fm._FusedMLPForward
        assert layer.mlp.forward.checkpoint == "fp8"
    assert list(model.state_dict()) == keys
    first = [layer.mlp.forward for layer in _decoder(model)]
    assert fm.patch_swiglu_mlp(model) == 0  # already routed
    assert [layer.mlp.forward for layer in _decoder(model)] == first


def test_patcher_leaves_other_mlps():
    # adapters: the LoRA block takes them
    model = apply_metal_liger_to_qwen3vl(qwen_tiny.build(lora=True), fuse_mlp=True,
                                         mlp_checkpoint="fp8")
    for layer in _decoder(model):
        assert type(layer.mlp.forward) is flora._FusedMLPForward
        assert layer.mlp.forward.checkpoint == "fp8" and layer.mlp.checkpoint == "fp8"
    with pytest.raises(ValueError, match="lora_dropout"):
        apply_metal_liger_to_qwen3vl(qwen_tiny.build(), lora_dropout=True, mlp_checkpoint="fp8")
    with pytest.raises(ValueError, match="checkpoint"):
        apply_metal_liger_to_qwen3vl(qwen_tiny.build(), mlp_checkpoint="int4")
    # a bias, another activation, a hook
    for change in (lambda m: setattr(m, "up_proj", nn.Linear(128, 256)),
                   lambda m: setattr(m, "act_fn", nn.GELU()),
                   lambda m: m.gate_proj.register_forward_hook(lambda *a: None)):
        model = qwen_tiny.build(lora=False)
        change(_decoder(model)[0].mlp)
        assert fm.patch_swiglu_mlp(model) == 1


def test_routed_mlp_falls_back_to_its_own_forward(monkeypatch):
    """Autocast, another dtype, an adapter or a hook added after the patch."""
    model = qwen_tiny.build(lora=False)
    mlp, own = _decoder(model)[0].mlp, copy.deepcopy(_decoder(model)[0].mlp)
    fm.patch_swiglu_mlp(model)
    x = seeded((3, 128), 5)
    with pytest.raises(ValueError, match="ROCm GPU"):  # the fused path, as every op here
        mlp(x)
    seen = []
    with monkeypatch.context() as m:  # (there is no autocast without a GPU)
        m.setattr(torch, "is_autocast_enabled", lambda device=None: True)
        assert torch.equal(mlp(x), own(x))
    handle = mlp.up_proj.register_forward_hook(lambda *a: seen.append(1))
    assert torch.equal(mlp(x), own(x)) and seen == [1]
    handle.remove()
    adapted = LoraLinear(mlp.gate_proj, r=4, alpha=8)
    mlp.gate_proj = own.gate_proj = adapted
    assert torch.equal(mlp(x), own(x))


def test_patcher_routes_vision_mlps(monkeypatch):
    model = qwen_tiny.build_vl()
    keys = list(model.state_dict())
    apply_metal_liger_to_qwen3vl(model, fuse_vision_mlp=True, mlp_checkpoint="fp8")
    visual = model.model.visual
    block = visual.blocks[0]
    assert type(block.mlp.forward) is fl._FusedVisionMLPForward
    assert block.mlp.forward.activation == "gelu_tanh" and block.mlp.forward.checkpoint == "fp8"
    assert type(block.forward) is fl._FusedVisionBlockForward
    assert "forward" not in visual.merger.__dict__  # it has a norm of its own
    assert list(model.state_dict()) == keys
    assert fl.patch_vision_mlp(model) == 0
    x, r = seeded((4, 64), 1), seeded((4, 64), 2)
    want = block.mlp.linear_fc2(block.mlp.act_fn(block.mlp.linear_fc1(x)))
    with monkeypatch.context() as m:  # its own forward, the residual added after it
        m.setattr(torch, "is_autocast_enabled", lambda device=None: True)
        assert torch.equal(block.mlp(x), want)
        assert torch.equal(block.mlp(x, residual=r), r + want)


def test_hooks_see_what_their_module_returns(monkeypatch):
    """A hook on an activation is called, one on an MLP sees its output alone."""
    model = qwen_tiny.build_vl()
    apply_metal_liger_to_qwen3vl(model, fuse_vision_mlp=True)
    block = model.model.visual.blocks[0]
    x, seen = seeded((4, 64), 1), []
    own = block.mlp.linear_fc2(block.mlp.act_fn(block.mlp.linear_fc1(x)))
    handle = block.mlp.act_fn.register_forward_hook(lambda *a: seen.append("act"))
    assert torch.equal(block.mlp(x), own) and seen == ["act"]
    handle.remove()
    block.mlp.register_forward_hook(lambda module, args, out: seen.append(out))
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device=None: True)
    block.attn.forward = lambda h, **kw: torch.zeros_like(h)
    out = block(x, cu_seqlens=None)
    want = block.mlp.linear_fc2(block.mlp.act_fn(block.mlp.linear_fc1(block.norm2(x))))
    assert torch.equal(seen[-1], want) and torch.equal(out, x + want)

    decoder = qwen_tiny.build_vl()
    mlp = next(m for m in decoder.modules() if hasattr(m, "gate_proj"))
    routed = fm._FusedMLPForward(mlp, mlp.forward, None)
    x = seeded((4, mlp.gate_proj.weight.shape[1]), 2)
    mlp.act_fn.register_forward_hook(lambda *a: seen.append("act"))
    assert torch.equal(routed(x), mlp(x)) and seen[-2:] == ["act", "act"]


def test_current_device(monkeypatch):
    """Tensors on another device than the current one: the call is made under theirs."""
    entered = []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)

        def __exit__(self, *exc):
            entered.append("out")

    class OnDevice(torch.Tensor):
        is_cuda = True

        def get_device(self):
            return 1

    monkeypatch.setattr(torch.cuda, "device", Device)
    x = torch.ones(2).as_subclass(OnDevice)
    f = hip_ops._on_device(lambda *args: list(entered))
    for current, want in ((1, []), (0, [1])):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: current)
        assert f(None, x) == want
    assert entered == [1, "out"]
    assert f(None, 3) == [1, "out"]
    for name in ("swiglu_kept_fwd", "swiglu_kept_bwd", "held_values", "linear_fwd", "linear_infer",
                 "linear_bwd", "swiglu_mlp_fwd", "swiglu_mlp_infer", "swiglu_mlp_bwd"):
        assert hasattr(getattr(hip_ops, name), "__wrapped__")


def test_activation_names():
    from transformers.activations import ACT2FN
    names = {"gelu_pytorch_tanh": "gelu_tanh", "gelu": "gelu", "silu": "silu"}
    for hf, own in names.items():
        assert fl.activation_name(ACT2FN[hf]) == own
        z = torch.linspace(-4, 4, 101)
        assert torch.allclose(ACT2FN[hf](z), ref.act(z.double(), own).float(), atol=1e-6)
    assert fl.activation_name(nn.GELU("tanh")) == "gelu_tanh" and fl.activation_name(nn.GELU()) == "gelu"
    for other in ("relu", "quick_gelu", "gelu_new", "gelu_fast"):
        assert fl.activation_name(ACT2FN[other]) is None


def test_exports():
    import metal_liger
    for name in ("fused_linear", "MetalLigerLinear", "fused_swiglu_mlp", "MetalLigerSwiGLUMLP"):
        assert hasattr(metal_liger, name)
    from metal_liger.ops.fused_linear import fused_linear  # noqa: F401
    from metal_liger.ops.fused_swiglu_mlp import fused_swiglu_mlp  # noqa: F401
    assert hip_ops.kept_shapes((2, 33)) == ((2, 33), (2, 2))
