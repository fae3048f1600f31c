"""Dropout, LoRA dropout and the embedding where two of their paths meet: the types
that one projection hands to the next, evaluation beside training, rows of unusual
strides, second derivatives, sizes past the limits of one launch and ids that need
several levels of merging. Bounds as in the operators' own tests."""

import pytest
import torch

from oracle import training_ops as ref
from tests.parity import seeded
from tests.test_gpu_embedding import _check_grad, _ids
from tests.test_gpu_lora_dropout import (
    _block,
    _half,
    _linear,
    _mlp,
    _params,
)

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ------------------------------------------------- the MLP on the fp32 products

def _mlp_grads(dev, mlp, lins, x, dy, ps, seed=11):
    """(y, dx, adapters' gradients) of the block and the same in 64 bits, with the
    largest |h| of its inner activations."""
    from metal_liger_amd import apply_fused_lora_mlp
    xd = x.to(dev).requires_grad_()
    adapters = [t for m in lins for t in (m.lora_A["default"].weight, m.lora_B["default"].weight)]
    y = apply_fused_lora_mlp(mlp, xd, lora_dropout=True, seed=seed)
    got = [y, *torch.autograd.grad(y, [xd, *adapters], dy.to(dev))]
    x64 = x.double().requires_grad_()
    leaves, out, h = [], [], 0.0
    for k, m in enumerate(lins):
        w, a, b, s = _params(m)
        a, b = (v.double().requires_grad_() for v in (a, b))
        leaves += [a, b]
        t = out[0] * torch.sigmoid(out[0]) * out[1] if k == 2 else x64
        h = t.detach().abs().max().item()
        f = ref.dropout_factors(tuple(t.shape), ps[k], seed, k)
        out.append(t @ w.double().t() + s * ((t * f) @ a.t()) @ b.t())
    return got, [out[2], *torch.autograd.grad(out[2], [x64, *leaves], dy.double())], h


@pytest.mark.parametrize("dtype, H, I", [(F16, 256, 512), (F16, 99, 203), (BF, 99, 203)])
def test_mlp_holds_its_inner_tensors_in_fp32(dev, dtype, H, I):  # noqa: E741
    """On the fp32 products only the block's output and dX are rounded to the
    activations' type (norms: eps / 2 of them), as in the block without dropout; the
    adapters' gradients, in fp32, are sums of at most 512 terms (2e-5 of their norms,
    as where the activations are fp32 too)."""
    ps = (0.2, 0.1, 0.3)
    lins, mlp = _mlp(dev, dtype, (8, 8, 8), ps, H, I, adapter=F32)
    x, dy = (seeded((90, H), k, dtype) for k in (1, 2))
    got, want, _ = _mlp_grads(dev, mlp, lins, x, dy, ps)
    assert got[0].dtype == got[1].dtype == dtype
    for k, (g, w) in enumerate(zip(got, want)):
        tol = 2e-5 + (_half(dtype) if k < 2 else 0.0)
        assert (g.double().cpu() - w).norm() <= tol * w.norm(), k


def test_mlp_inner_activations_past_fp16(dev):
    """silu(gate) * up beyond 65504 under a down projection that brings it back: the
    fp16 block is finite and near the 64-bit form (output rounded once, sums of 512
    terms in fp32), with dropout as without."""
    from metal_liger_amd import apply_fused_lora_mlp
    ps = (0.1, 0.1, 0.1)
    lins, mlp = _mlp(dev, F16, (8, 8, 8), ps, adapter=F32)
    with torch.no_grad():
        lins[2].base_layer.weight.mul_(2.0 ** -7)
        lins[2].lora_B["default"].weight.mul_(2.0 ** -7)
    x, dy = seeded((40, 256), 1, F16, scale=400.0), seeded((40, 256), 2, F16)
    got, want, h = _mlp_grads(dev, mlp, lins, x, dy, ps)
    assert h > 65504 and want[0].abs().max() < 65504
    assert torch.isfinite(apply_fused_lora_mlp(mlp, x.to(dev))).all()
    for k, (g, w) in enumerate(zip(got, want)):
        tol = 2e-5 + (_half(F16) if k < 2 else 0.0)
        assert torch.isfinite(g).all() and (g.double().cpu() - w).norm() <= tol * w.norm(), k


# ------------------------------------------------------------------ odd strides

@pytest.mark.parametrize("rank", [16, 96])
def test_one_row_of_an_odd_stride(dev, rank):
    """A batch of one token cut out of a wider buffer: its row stride, which no access
    uses, need not be a multiple of 8."""
    from metal_liger_amd import apply_fused_lora_mlp, apply_fused_lora_qkv
    from metal_liger_amd.ops.fused_lora import _lora_linear, apply_fused_lora_linear
    lins = [_linear(dev, 128, o, rank, 0.4, BF, 10 * k) for k, o in enumerate((128, 64, 64))]
    attn = _block(q_proj=lins[0], k_proj=lins[1], v_proj=lins[2])
    _, mlp = _mlp(dev, BF, (rank,) * 3, (0.3,) * 3, 128, 256)
    wide = seeded((3, 131), 1, BF).to(dev)
    w, a, b, s = (lins[0].base_layer.weight, lins[0].lora_A["default"].weight,
                  lins[0].lora_B["default"].weight, 2.0)
    calls = [lambda x, drop=drop, f=f: f(x, drop) for drop in (True, False) for f in (
        lambda x, drop: apply_fused_lora_qkv(attn, x, lora_dropout=drop, seed=3),
        lambda x, drop: (apply_fused_lora_mlp(mlp, x, lora_dropout=drop, seed=3),),
        lambda x, drop: (apply_fused_lora_linear(lins[0], x, lora_dropout=drop, seed=3),),
        lambda x, drop: (_lora_linear(x, w, a, b, s),),
        lambda x, drop: (_lora_linear(x, w, None, None, s),))]
    for i, call in enumerate(calls):
        odd = wide[1:2, :128]
        assert odd.stride(0) == 131
        for x in (odd, odd.unsqueeze(0), wide[:1, :128]):
            runs = []
            for dense in (False, True):
                t = x.clone(memory_format=torch.contiguous_format) if dense else x
                t = t.detach().requires_grad_()
                assert t.stride(-2) == (128 if dense else 131)
                ys = call(t)
                dys = [wide.flatten()[5:5 + y.numel()].view(y.shape) for y in ys]
                dx = () if i % 5 > 2 else torch.autograd.grad(ys, t, dys)  # (_lora_linear: none)
                runs.append([*ys, *dx])
            assert all(torch.equal(p, q) for p, q in zip(*runs)), i


def test_one_row_of_an_odd_stride_through_the_loss(dev):
    """As above for the fused cross-entropy's hidden state and the products."""
    from metal_liger_amd import hip_ops
    from metal_liger_amd.ops.fused_linear_cross_entropy import MetalLigerFusedLinearCrossEntropy
    wide = seeded((3, 131), 1, BF).to(dev)
    x = wide[1:2, :128]
    weight = seeded((64, 128), 2, BF, scale=0.1).to(dev)
    labels = torch.tensor([5], device=dev)
    head = torch.nn.Linear(128, 64, bias=False)
    head.weight = torch.nn.Parameter(weight)
    loss = MetalLigerFusedLinearCrossEntropy(head)
    dense = x.clone(memory_format=torch.contiguous_format)
    runs = []
    first = wide[:1, :128]
    for t in (x, dense, first, first.clone(memory_format=torch.contiguous_format)):
        t = t.detach().requires_grad_()
        y = loss(t, labels)
        runs.append([y, *torch.autograd.grad(y, [t, head.weight])])
    for k in (0, 2):
        assert all(torch.equal(p, q) for p, q in zip(runs[k], runs[k + 1]))
    assert torch.equal(hip_ops.matmul(x, weight, b_t=True), hip_ops.matmul(dense, weight, b_t=True))
    f = wide.float()[1:2, :128]
    flat = torch.ones(128, device=dev).as_strided((1, 128), (1, 1))
    for t in (f, flat):
        assert torch.equal(hip_ops.gemm_f32([t], [weight.float()], b_t=True),
                           hip_ops.gemm_f32([t.clone(memory_format=torch.contiguous_format)],
                                            [weight.float()], b_t=True))


# ------------------------------------------------------------------ evaluation

def test_evaluation_with_a_residual_draws_no_seed(dev):
    """Nothing is dropped: torch's generator stays where it was, the sum is the one
    rounding of x + residual, and both gradients are dy's values."""
    from metal_liger_amd import MetalLigerDropout, fused_dropout
    for dtype in (F32, BF, F16):
        x, res, dy = (seeded((33, 65), k, dtype).to(dev).requires_grad_() for k in (1, 2, 3))
        torch.manual_seed(3)
        state = torch.cuda.get_rng_state()
        for y in (fused_dropout(x, 0.5, training=False, residual=res),
                  fused_dropout(x, 1e-7, residual=res), MetalLigerDropout(0.5).eval()(x, res)):
            assert torch.equal(y, x + res) and y.is_contiguous()
            dx, dr = torch.autograd.grad(y, [x, res], dy)
            assert torch.equal(dx, dy) and torch.equal(dr, dy)
        assert torch.equal(torch.cuda.get_rng_state(), state)
    with pytest.raises(ValueError, match="residual"):
        fused_dropout(x, 0.5, training=False, residual=res[:1])
    with pytest.raises(ValueError, match="residual"):
        fused_dropout(x, 0.5, training=False, residual=res.float())
    with pytest.raises(TypeError, match="dtype"):
        fused_dropout(x.double(), 0.5, training=False, residual=res.double())


# ------------------------------------------------- sizes past one launch's threads

def test_dropout_past_one_launch(dev):
    """More blocks of 16 bytes than a launch has threads (2^35 elements of 16 bits and
    some, in place): the ends, and both sides of where the second launch begins."""
    from metal_liger_amd import _hip
    n = 2 ** 35 + 1003
    x = torch.ones(n, dtype=BF, device=dev)
    seed = torch.tensor([10], device=dev)
    _hip.call("ml_dropout", x.data_ptr(), None, x.data_ptr(), n, 32768, 2.0, seed.data_ptr(), 7,
              _hip.DTYPE_TAG[BF], _hip.stream_of(x))
    for first in (0, 2 ** 34 - 512, 2 ** 35 - 512, n - 1003):
        f = ref.dropout_factors((1003,), 0.5, 10, 7, first=first)
        assert torch.equal(x[first:first + 1003].double().cpu(), f), first


def test_lookup_past_one_launch(dev):
    """More workgroups of four rows than a launch holds."""
    from metal_liger_amd import fused_embedding
    n, vocab, hidden = 2 ** 26 + 1029, 501, 129
    w = seeded((vocab, hidden), 1, F16).to(dev)
    ids = (torch.arange(n, dtype=torch.int32, device=dev) * 7) % vocab
    y = fused_embedding(ids, w)
    for first in (0, 2 ** 25 - 4096, n - 8192):
        part = slice(first, first + 8192)
        assert torch.equal(y[part], w[ids[part].long()]), first


# --------------------------------------------------------------- ranks above 64

@pytest.mark.parametrize("n", [1, 3])
def test_wide_ranks_round_dx_once(dev, n):
    """dX at ranks above 64, from whole numbers whose products and sums are exact in
    fp32 and whose P = c s dY B is exact in bf16 (at most 2 x 3 x 40 in magnitude): the
    large products' sum and every adapter's part, rounded once."""
    from metal_liger_amd.ops.fused_lora import _dropped
    outs, rank = (192, 64, 72)[:n], 96
    lins = [_linear(dev, 320, o, rank, 0.5, BF, 10 * k, alpha=float(rank)) for k, o in
            enumerate(outs)]
    g = torch.Generator().manual_seed(1)
    whole = lambda *s: torch.randint(-3, 4, s, generator=g).to(BF)  # noqa: E731
    with torch.no_grad():
        for lin, o in zip(lins, outs):
            lin.base_layer.weight.copy_(whole(o, 320))
            lin.lora_A["default"].weight.copy_(whole(rank, 320))
            b = torch.zeros(o, rank)
            b[:40] = whole(40, rank).sign()
            lin.lora_B["default"].weight.copy_(b)
    x, dys = whole(130, 320), [whole(130, o) for o in outs]
    xd = x.to(dev).requires_grad_()
    dx, = torch.autograd.grad(_dropped(lins, xd, 5), xd, [d.to(dev) for d in dys])
    fs = [ref.dropout_factors((130, 320), 0.5, 5, k) for k in range(n)]
    _, want, _ = ref.lora_dropout(x, [_params(m) for m in lins], dys, fs)
    assert want.abs().max() < 2 ** 24
    assert torch.equal(dx.cpu(), want.to(BF))


# ------------------------------------------------------------ second derivatives

@pytest.mark.parametrize("training", [True, False])
def test_dropout_twice_differentiable(dev, training):
    """d/dy of dx's product with v is the mask over v (and v for the residual)."""
    from metal_liger_amd import fused_dropout
    x, res, dy, v = (seeded((33, 65), k).to(dev).requires_grad_() for k in (1, 2, 3, 4))
    y = fused_dropout(x, 0.3, training, res, seed=77, stream=5)
    dx, dr = torch.autograd.grad(y, [x, res], dy, create_graph=True)
    ddy, = torch.autograd.grad([dx, dr], dy, [v, v])
    f = ref.dropout_factors((33, 65), 0.3, 77, 5).to(dev) if training else 1.0
    want = v.double() * f + v.double()
    assert bool(((ddy - want).abs() <= 4 * 2.0 ** -24 * (want.abs() + v.abs())).all())


def test_embedding_twice_differentiable(dev):
    """d/d(dy) of the table's gradient's product with v is the lookup of v: zero for
    the padding index and for ids outside the table; a third derivative follows."""
    from metal_liger_amd import fused_embedding
    w, v = (seeded((20, 24), k).to(dev).requires_grad_() for k in (1, 2))
    ids = torch.tensor([[3, -1, 20], [5, 7, 3]], device=dev)
    dy = seeded((2, 3, 24), 3).to(dev).requires_grad_()
    dw, = torch.autograd.grad(fused_embedding(ids, w, 1.5, 7), w, dy, create_graph=True)
    _check_grad(dw, ids, dy.detach(), 20, 1.5, 7)
    ddy, = torch.autograd.grad(dw, dy, v, create_graph=True)
    keep = torch.tensor([[1, 0, 0], [1, 0, 1]], device=dev, dtype=torch.bool)
    want = torch.where(keep[..., None], 1.5 * v[ids.clamp(0, 19)], torch.zeros((), device=dev))
    assert torch.equal(ddy, want)
    u = seeded((2, 3, 24), 4).to(dev)
    _check_grad(torch.autograd.grad(ddy, v, u)[0], ids, u, 20, 1.5, 7)


def test_other_derivatives_are_refused(dev):
    """Forward mode and torch.func say so instead of leaving a derivative out."""
    import torch.autograd.forward_ad as fw

    from metal_liger_amd import fused_dropout, fused_embedding
    x = seeded((20, 24), 1).to(dev)
    ids = torch.tensor([3, 5], device=dev)
    for fn in (lambda t: fused_dropout(t, 0.5, seed=3), lambda t: fused_embedding(ids, t),
               lambda t: fused_dropout(t, 0.5, training=False, residual=x)):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: fn(t).sum())(x)
        with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
            fn(fw.make_dual(x, torch.ones_like(x)))


def test_lookup_without_a_gradient(dev):
    """A frozen table, or a trained one where no gradient is formed: the same values,
    nothing kept for a backward; a routed module follows its table."""
    from metal_liger_amd import fused_embedding
    from metal_liger_amd.ops.fused_embedding import patch_embedding
    root = torch.nn.Module()
    root.embed_tokens = torch.nn.Embedding(50, 24, device=dev)
    assert patch_embedding(root) == 1
    w, ids = root.embed_tokens.weight, torch.randint(0, 50, (3, 7), device=dev)
    y = root.embed_tokens(ids)
    assert "FusedEmbedding" in type(y.grad_fn).__name__ and torch.equal(y, w[ids])
    with torch.no_grad():
        assert torch.equal(fused_embedding(ids, w, 2.0), 2 * w[ids])
    w.requires_grad_(False)
    for y in (fused_embedding(ids, w), root.embed_tokens(ids)):
        assert y.grad_fn is None and torch.equal(y, w[ids])
    step = torch.compile(lambda i: fused_embedding(i, w, 2.0), fullgraph=True, backend="aot_eager")
    assert torch.equal(step(ids), 2 * w[ids])


# -------------------------------------------------------------- compiled, drawn

def test_compile_with_a_drawn_seed(dev):
    """The seed is drawn inside the compiled step: one mask both ways, another at the
    next call, and the same again from the same state of torch's generator."""
    from metal_liger_amd import apply_fused_lora_qkv, fused_dropout
    x = torch.ones(64, 128, device=dev, requires_grad=True)
    step = torch.compile(lambda t: fused_dropout(t, 0.5), fullgraph=True, backend="aot_eager")
    torch.manual_seed(1)
    a, b = step(x), step(x)
    for y in (a, b):
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(dx, y)
        assert set(y.unique().tolist()) == {0.0, 2.0}
    torch.manual_seed(1)
    assert torch.equal(step(x), a) and not torch.equal(a, b)

    lins = [_linear(dev, 128, o, 16, 0.4, BF, 10 * k) for k, o in enumerate((128, 64, 64))]
    attn = _block(q_proj=lins[0], k_proj=lins[1], v_proj=lins[2])
    xb = seeded((50, 128), 1, BF).to(dev).requires_grad_()
    fn = torch.compile(lambda t: apply_fused_lora_qkv(attn, t, lora_dropout=True), fullgraph=True,
                       backend="aot_eager")
    dys = [seeded((50, o), 2, BF).to(dev) for o in (128, 64, 64)]
    runs = []
    for _ in range(2):
        torch.manual_seed(2)
        ys = fn(xb)
        runs.append([*ys, *torch.autograd.grad(ys, xb, dys)])
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    assert not torch.equal(fn(xb)[0], runs[0][0])


# ----------------------------------------------- several tiles of ids, and merges

@pytest.mark.parametrize("kind", ["uniform", "same", "half"])
@pytest.mark.parametrize("vocab, tokens", [
    (262144, 8193), (262145, 70001),          # 64-bit entries: two tiles, a full merge
    (30011, 140003), (262143, 131073),        # 32-bit entries, two levels of merging
    (262144, 65537), (300007, 150001)])       # 64-bit entries, two levels
def test_merged_orders(dev, vocab, tokens, kind):
    """Scattered ids over more tokens than one sorted tile, or one merge, holds; every
    token's row is another one, so that a wrong or repeated position shows."""
    ids = _ids(kind, tokens, vocab, seed=tokens)
    dy = seeded((tokens, 8), 2)
    dw = torch.ops.metal_liger_amd.embedding_bwd(ids.to(dev), dy.to(dev), vocab, -1, 1.0)
    _check_grad(dw, ids, dy, vocab)


def test_offsets_of_a_gradient_past_32_bits(dev):
    """An output's gradient of more than 2^31 elements with scattered ids: the rows
    past that, and those that a wrapped offset would read instead, have values of
    their own."""
    n, hidden, vocab = (1 << 19) + 3, 4104, 5003
    dy = torch.zeros(n, hidden, dtype=BF, device=dev)
    special = torch.tensor([0, 1, 2, 777, (1 << 31) // hidden - 1, (1 << 31) // hidden,
                            (1 << 31) // hidden + 1, n - 3, n - 2, n - 1])
    for k, t in enumerate(special.tolist()):
        dy[t] = float(k + 1)
    ids = _ids("uniform", n, vocab, seed=9)
    dw = torch.ops.metal_liger_amd.embedding_bwd(ids.to(dev), dy, vocab, -1, 1.0)
    want = torch.zeros(vocab)                           # sums of small whole numbers: exact
    want.index_add_(0, ids[special], torch.arange(1.0, len(special) + 1))
    assert torch.equal(dw.float().cpu(), want[:, None].expand(vocab, hidden))
