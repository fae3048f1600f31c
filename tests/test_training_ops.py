"""Dropout, LoRA dropout and the token embedding without a GPU: the oracle against
published numbers and torch, refusals, fake kernels and the patcher's flags."""

import copy

import numpy as np
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import training_ops as ref
from tests.peft_shim import LoraLinear
from tests.qwen_tiny import build

BF, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------ the oracle

@pytest.mark.parametrize("rounds, fill, want", [
    (7, 0, (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
    (7, 0xFFFFFFFF, (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662)),
    (10, 0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
])
def test_philox_known_answers(rounds, fill, want):
    """The known answers that the generator's authors publish."""
    got = ref.philox4x32(np.full((1, 4), fill, dtype=np.uint64), (fill, fill), rounds)
    assert tuple(int(w) for w in got[0]) == want


def test_oracle_mask_is_a_function_of_the_element():
    whole = ref.dropout_factors((1000,), 0.3, 5, stream=2)
    assert torch.equal(whole[13:913], ref.dropout_factors((900,), 0.3, 5, stream=2, first=13))
    assert not torch.equal(whole, ref.dropout_factors((1000,), 0.3, 5, stream=1))
    assert not torch.equal(whole, ref.dropout_factors((1000,), 0.3, 5 + 2 ** 32, stream=2))


@pytest.mark.parametrize("p", [0.0, 0.05, 0.5, 0.9])
def test_oracle_rate(p):
    """Shares of 2^18 draws within six standard deviations of the rate."""
    n = 1 << 18
    f = ref.dropout_factors((n,), p, 11)
    q = ref.dropout_threshold(p) / 65536
    assert abs((f == 0).double().mean().item() - q) <= 6 * (q * (1 - q) / n) ** 0.5
    assert torch.all(f == 0).item() is False


def test_oracle_lora_against_autograd():
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = rnd(9, 24).requires_grad_()
    params = [(rnd(o, 24), rnd(4, 24).requires_grad_(), rnd(o, 4).requires_grad_(), 1.7)
              for o in (16, 8)]
    fs = [ref.dropout_factors((9, 24), 0.4, 3, i) for i in range(2)]
    ys = [x @ w.t() + s * ((x * f) @ a.t()) @ b.t() for (w, a, b, s), f in zip(params, fs)]
    dys = [rnd(*y.shape) for y in ys]
    want = torch.autograd.grad(ys, [x, *(t for p in params for t in p[1:3])], dys)
    outs, dx, grads = ref.lora_dropout(x.detach(), [(w, a.detach(), b.detach(), s)
                                                    for w, a, b, s in params], dys, fs)
    for got, y in zip(outs, ys):
        assert torch.allclose(got, y, rtol=1e-12, atol=1e-12)
    for got, w in zip([dx, *(t for g2 in grads for t in g2)], want):
        assert torch.allclose(got, w, rtol=1e-12, atol=1e-12)


def test_oracle_embedding_against_autograd():
    g = torch.Generator().manual_seed(1)
    w = torch.randn(11, 5, generator=g, dtype=torch.float64).requires_grad_()
    ids = torch.randint(0, 11, (4, 6), generator=g)
    dy = torch.randn(4, 6, 5, generator=g, dtype=torch.float64)
    want, = torch.autograd.grad(3 * F.embedding(ids, w, padding_idx=2), w, dy)
    assert torch.allclose(ref.embedding_grad(ids, dy, 11, 3.0, 2), want, rtol=1e-13, atol=1e-13)
    outside = ids.clone()
    outside[0, :3] = torch.tensor([-1, 11, 1 << 20])
    dy[0, :3] = 0
    assert torch.allclose(ref.embedding_grad(outside, dy, 11),
                          ref.embedding_grad(ids, dy, 11), rtol=1e-13, atol=1e-13)


# -------------------------------------------------------------------- refusals

@pytest.mark.parametrize("p", [-0.1, 1.5, float("nan")])
def test_dropout_refuses_rates(p):
    from metal_liger_amd import MetalLigerDropout, fused_dropout
    with pytest.raises(ValueError, match="between 0 and 1"):
        fused_dropout(torch.zeros(4), p)
    with pytest.raises(ValueError, match="between 0 and 1"):
        MetalLigerDropout(p)


def test_dropout_refuses_inplace_and_seeds_that_are_no_integers():
    from metal_liger_amd import MetalLigerDropout
    from metal_liger_amd.ops.fused_dropout import seed_tensor
    with pytest.raises(ValueError, match="inplace"):
        MetalLigerDropout(0.1, inplace=True)
    with pytest.raises(TypeError):
        seed_tensor(1.5, "cpu")
    assert seed_tensor(2 ** 64 - 1, "cpu").tolist() == [-1]
    assert seed_tensor(None, "cpu").dtype == torch.int64


def test_dropout_refuses_streams_and_cpu_tensors():
    from metal_liger_amd import fused_dropout
    for stream in (-1, 1 << 32):
        with pytest.raises(ValueError, match="stream"):
            fused_dropout(torch.zeros(4), 0.5, stream=stream)
    with pytest.raises(ValueError, match="ROCm GPU"):
        fused_dropout(torch.zeros(4), 0.5)
    with pytest.raises(ValueError, match="ROCm GPU"):
        fused_dropout(torch.zeros(4), 0.5, residual=torch.zeros(4), training=False)


def test_dropout_without_effect_is_the_identity():
    from metal_liger_amd import MetalLigerDropout, fused_dropout
    x = torch.randn(5)
    assert fused_dropout(x, 0.0) is x and fused_dropout(x, 0.5, training=False) is x
    assert fused_dropout(x, 1e-7) is x                      # rounds to a rate of 0
    assert MetalLigerDropout(0.5).eval()(x) is x


def test_embedding_refusals():
    from metal_liger_amd import MetalLigerEmbedding, fused_embedding, hip_ops
    table = torch.zeros(10, 4)
    for idx in (10, -11):
        with pytest.raises(ValueError, match="padding_idx"):
            fused_embedding(torch.zeros(3, dtype=torch.long), table, padding_idx=idx)
    with pytest.raises(ValueError, match="ROCm GPU"):
        fused_embedding(torch.zeros(3, dtype=torch.long), table)
    with pytest.raises(TypeError, match="int64 or int32"):
        hip_ops._ids(torch.zeros(3))
    for bad in (nn.Embedding(4, 4, max_norm=1.0), nn.Embedding(4, 4, sparse=True),
                nn.Embedding(4, 4, scale_grad_by_freq=True)):
        with pytest.raises(ValueError, match="plain nn.Embedding"):
            MetalLigerEmbedding(bad)


def test_seed_refusals():
    from metal_liger_amd import hip_ops
    for bad in (torch.zeros(1), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(TypeError, match="one int64"):
            hip_ops.check_seed(bad)


def test_host_side_argument_errors():
    from metal_liger_amd import _hip
    L = _hip.lib()

    def refused(rc, text):
        assert rc == 1 and text in L.ml_last_error(), L.ml_last_error()

    refused(L.ml_dropout(None, None, None, -1, 0, 1.0, None, 0, 0, None), b"negative size")
    refused(L.ml_dropout(None, None, None, 8, 65537, 1.0, None, 0, 0, None), b"threshold")
    refused(L.ml_dropout(None, None, None, 8, 1, 1.0, None, 1 << 32, 0, None), b"stream id")
    refused(L.ml_dropout(None, None, None, 8, 1, 1.0, None, 0, 0, None), b"null pointer")
    refused(L.ml_dropout(4096, None, 4096, 8, 1, 1.0, 4096, 0, 9, None), b"dtype")
    refused(L.ml_embedding_fwd(4096, 2, 1, 4096, 4, 4096, 8, 4, 1.0, 0, None), b"4 or 8 bytes")
    refused(L.ml_embedding_fwd(4096, 8, 1, 4096, 3, 4096, 8, 4, 1.0, 0, None), b"row stride")
    refused(L.ml_embedding_fwd(4096, 8, 1, 4096, 4, 4096, 0, 4, 1.0, 0, None), b"bad table")
    refused(L.ml_embedding_fwd(None, 8, 1, 4096, 4, 4096, 8, 4, 1.0, 0, None), b"null pointer")
    refused(L.ml_embedding_bwd(4096, 8, 1, 4096, 4, 4096, 8, 4, 8, 1.0, 4096, 1 << 20, 0, None),
            b"padding index")
    refused(L.ml_embedding_bwd(4096, 8, 1, 4096, 4, 4096, 8, 4, -1, 1.0, None, 1 << 20, 0, None),
            b"workspace")
    refused(L.ml_embedding_bwd(4096, 8, 1, 4096, 4, 4096, 8, 4, -1, 1.0, 4096, 16, 0, None),
            b"workspace")
    refused(L.ml_embedding_bwd(4096, 8, 1, 4096, 4, 4096, 8, 4, -1, 1.0, 4100, 1 << 20, 0, None),
            b"misaligned")
    refused(L.ml_embedding_bwd(4096, 8, 1, None, 4, 4096, 8, 4, -1, 1.0, 4096, 1 << 20, 0, None),
            b"null pointer")


def test_lora_dropout_host_side_argument_errors():
    from metal_liger_amd import _hip
    L = _hip.lib()
    p = 4096  # (never read: every call is refused on the host)

    one = lambda *v: _hip.ptrs(v)  # noqa: E731
    for nadp, geometry, text in ((2, (16, 64, 64, 16, 64), b"fragment order"),
                                 (1, (8, 64, 64, 8, 64), b"16 x 32"),
                                 (1, (16, 40, 40, 16, 40), b"16 x 32")):
        rc = L.ml_lora_dropout_pack(1, nadp, one(p), _hip.geom(geometry), _hip.ints([1]),
                                    _hip.floats([1.0]), one(p), one(None), None)
        assert rc == 1 and text in L.ml_last_error(), L.ml_last_error()

    def xa(n=1, tokens=4, width=64, ldx=64, rank=16, thresholds=(0, 0, 0), first=0, ldo=48, x=p,
           seed=p):
        return L.ml_lora_dropout_xa(n, x, tokens, width, ldx, p, rank, _hip.geom(thresholds), seed,
                                    first, p, ldo, None)

    for kw, text in ((dict(n=4), b"1..3 adapters"), (dict(n=0), b"1..3 adapters"),
                     (dict(seed=None), b"null pointer"), (dict(thresholds=(65537,)), b"threshold"),
                     (dict(n=2, thresholds=(0, -1)), b"threshold"), (dict(first=-1), b"stream id"),
                     (dict(n=2, first=(1 << 32) - 1), b"stream id"), (dict(width=60), b"multiple of 8"),
                     (dict(rank=24), b"rank 16, 32, 48 or 64"), (dict(rank=80), b"rank 16"),
                     (dict(ldx=56), b"leading"), (dict(ldo=8), b"leading"),
                     (dict(x=None), b"null pointer"), (dict(x=p + 2), b"16-byte aligned")):
        assert xa(**kw) == 1 and text in L.ml_last_error(), (kw, L.ml_last_error())

    def bwd(n=1, tokens=4, width=64, outs=(64, 64, 64), rank=16, dx=p, w=p, ws=p, ws_bytes=1 << 30,
            grad=0):
        ptrs = _hip.ptrs([p] * 3)
        return L.ml_lora_dropout_bwd(n, p, tokens, width, ptrs, _hip.geom(outs), _hip.ptrs([w] * 3), p,
                                     ptrs, _hip.floats([1.0] * 3), p, rank, _hip.geom([0] * 3), p, 0,
                                     dx, p, ptrs, grad, ws, ws_bytes, None)

    for kw, text in ((dict(n=0), b"1..3 adapters"), (dict(tokens=0), b"token count"),
                     (dict(width=4), b"multiple of 8"), (dict(outs=(60,)), b"multiple of 8"),
                     (dict(rank=72), b"rank 16"), (dict(dx=None), b"null pointer"),
                     (dict(w=None), b"null pointer"), (dict(w=p + 8), b"16-byte aligned"),
                     (dict(dx=p + 2), b"16-byte aligned"), (dict(ws=None), b"workspace"),
                     (dict(grad=2), b"fp32 or bf16"),
                     (dict(ws_bytes=64), b"workspace"), (dict(ws=p + 4), b"workspace")):
        assert bwd(**kw) == 1 and text in L.ml_last_error(), (kw, L.ml_last_error())
    assert L.ml_lora_dropout_bwd_workspace_bytes(4, 4, 64, _hip.geom([64] * 4), 16) == 0
    assert L.ml_lora_dropout_bwd_workspace_bytes(1, 4, 64, _hip.geom([64]), 72) == 0


# ----------------------------------------------------------------- fake kernels

def e(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_fake_kernels():
    import metal_liger_amd._custom_ops  # noqa: F401
    ops = torch.ops.metal_liger_amd
    with FakeTensorMode():
        seed = e(1, dtype=torch.int64)
        y = ops.dropout(e(6, 4).t(), None, seed, 100, 0, 1.0)
        assert y.shape == (4, 6) and y.is_contiguous() and y.dtype == BF
        ids = e(2, 3, dtype=torch.int64)
        assert ops.embedding_fwd(ids, e(10, 4), 1.0).shape == (2, 3, 4)
        dw = ops.embedding_bwd(ids, e(2, 3, 4, dtype=F32), 10, -1, 1.0)
        assert dw.shape == (10, 4) and dw.dtype == F32
        x, ws, As, Bs = e(96, 128), [e(64, 128), e(32, 128)], [e(12, 128), e(16, 128)], [e(64, 12),
                                                                                       e(32, 16)]
        for rank, fwd, bwd in ((16, ops.lora_dropout_fwd, ops.lora_dropout_bwd),
                               (72, ops.lora_dropout_wide_fwd, ops.lora_dropout_wide_bwd)):
            q, k, xa, packed = fwd(x, ws, As, Bs, [2.0] * 2, rank, seed, [100, 0], 0)
            assert q.shape == (96, 64) and k.shape == (96, 32) and xa.shape == (96, 2 * rank)
            assert packed.shape == (rank * (2 * 128 + 2 * 96),)
            dx, g = bwd(x, [q, k], ws, packed, [2.0] * 2, xa, rank, seed, [100, 0], 0, [], F32)
            assert dx.shape == (96, 128) and g.dtype == F32
            assert g.shape == (2 * rank * 128 + 64 * rank + 32 * rank,)


# ------------------------------------------------------------------ the patcher

def with_dropout(model, p):
    for m in model.modules():
        if isinstance(m, LoraLinear):
            m.lora_dropout = nn.ModuleDict({m._adapter: nn.Dropout(p) if p else nn.Identity()})
    return model


def test_thresholds_of_peft_modules():
    from metal_liger_amd.ops.fused_lora import _drop_threshold
    lin = LoraLinear(nn.Linear(8, 8), r=4)
    assert _drop_threshold(lin) == 0
    lin.lora_dropout = nn.ModuleDict({"default": nn.Identity()})
    assert _drop_threshold(lin) == 0
    lin.lora_dropout = nn.ModuleDict({"default": nn.Dropout(0.25)})
    assert _drop_threshold(lin) == 16384
    assert _drop_threshold(lin.eval()) == 0
    lin.lora_dropout = nn.ModuleDict({"default": nn.AlphaDropout(0.25)})
    with pytest.raises(TypeError, match="nn.Dropout"):
        _drop_threshold(lin.train())


def test_patcher_flags():
    from metal_liger_amd import apply_metal_liger_to_qwen3vl
    model = with_dropout(build(), 0.1)
    keys = set(model.state_dict())
    embed = model.base_model.model.get_input_embeddings()
    plain = apply_metal_liger_to_qwen3vl(copy.deepcopy(model), fuse_swiglu=False)
    layer = plain.base_model.model.model.layers[0]
    assert not layer.mlp.forward.lora_dropout and not layer.self_attn.forward.lora_dropout
    assert "forward" not in vars(plain.base_model.model.get_input_embeddings())

    apply_metal_liger_to_qwen3vl(model, fuse_swiglu=False, lora_dropout=True, fuse_embedding=True)
    layer = model.base_model.model.model.layers[0]
    assert layer.mlp.forward.lora_dropout and layer.self_attn.forward.lora_dropout
    assert set(model.state_dict()) == keys
    assert model.base_model.model.get_input_embeddings() is embed and "forward" in vars(embed)


def test_patch_embedding_is_routed_once_and_only_where_it_fits():
    from metal_liger_amd.ops.fused_embedding import patch_embedding

    class Wrapper(nn.Module):              # as PEFT wraps a module that is saved whole
        def __init__(self, m):
            super().__init__()
            self.original_module = m
            self.modules_to_save = nn.ModuleDict({"default": copy.deepcopy(m)})

    class Scaled(nn.Embedding):
        pass

    root = nn.Module()
    root.model = nn.Module()
    root.model.embed_tokens = Wrapper(nn.Embedding(8, 4))
    root.visual = nn.Module()
    root.visual.pos_embed = nn.Embedding(8, 4)
    assert patch_embedding(root) == 2 and patch_embedding(root) == 0
    assert "forward" not in vars(root.visual.pos_embed)
    root.model.embed_tokens = Scaled(8, 4)
    assert patch_embedding(root) == 0


def test_public_names():
    import metal_liger
    import metal_liger_amd as ml
    for name in ("MetalLigerDropout", "MetalLigerEmbedding", "fused_dropout", "fused_embedding"):
        assert name in ml.__all__ and getattr(metal_liger, name) is getattr(ml, name)
    from metal_liger.ops.fused_dropout import fused_dropout
    from metal_liger.ops.fused_embedding import MetalLigerEmbedding
    assert fused_dropout is ml.fused_dropout and MetalLigerEmbedding is ml.MetalLigerEmbedding


def test_embedding_module_shares_the_parameter():
    from metal_liger_amd import MetalLigerEmbedding
    old = nn.Embedding(8, 4, padding_idx=3)
    new = MetalLigerEmbedding(old, scale=2.0)
    assert new.weight is old.weight and set(new.state_dict()) == {"weight"}
    assert new.padding_idx == 3 and "scale=2.0" in repr(new)
