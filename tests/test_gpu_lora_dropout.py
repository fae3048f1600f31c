"""LoRA projections with dropout on the adapters' input against the oracle in fp64.

Bounds, element by element, from the roundings of the method (u = half a step of the
activation dtype, a = (K + 16) 2^-24 for a sum of K terms in fp32, both times the sum
of the terms' magnitudes): XA is rounded once (u), s B once (u), P once (u), the
outputs once (u), dX twice (the large products alone, then with the adapters' part)
and the adapters' part once before that at ranks above 64; dA and dB are fp32 sums rounded to the parameters' dtype. Second-order terms are
covered by a factor of 1.05.
"""

import pytest
import torch
import torch.nn as nn

from oracle import training_ops as ref
from tests.parity import seeded
from tests.peft_shim import LoraLinear

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _linear(dev, i, o, r, p, dtype, seed, adapter=None, alpha=None):
    lin = LoraLinear(nn.Linear(i, o, bias=False), r=r, alpha=alpha or 2.0 * r)
    adapter = adapter or dtype
    with torch.no_grad():
        lin.base_layer.weight.copy_(seeded((o, i), seed, scale=0.05))
        lin.lora_A["default"].weight.copy_(seeded((r, i), seed + 1, scale=i ** -0.5))
        lin.lora_B["default"].weight.copy_(seeded((o, r), seed + 2, scale=0.05))
    lin.base_layer.weight.requires_grad_(False)
    lin.base_layer.to(dtype)
    for m in (lin.lora_A, lin.lora_B):
        m.to(adapter)
    lin.lora_dropout = nn.ModuleDict({"default": nn.Dropout(p) if p else nn.Identity()})
    return lin.to(dev)


def _params(lin):
    return (lin.base_layer.weight.detach().cpu(), lin.lora_A["default"].weight.detach().cpu(),
            lin.lora_B["default"].weight.detach().cpu(), lin.scaling["default"])


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _bounds(x, params, dys, fs, dtype, adapter, composed):
    """Element-wise bounds of (outs, dx, [(dA, dB)])."""
    u = _half(dtype if dtype == BF else F32)
    ud, ua = _half(dtype), _half(adapter)
    x = x.double()
    N = x.shape[0]
    acc = lambda k: (k + 16) * 2.0 ** -24  # noqa: E731
    outs, grads = [], []
    base = torch.zeros_like(x)
    base_abs, extra = torch.zeros_like(x), torch.zeros_like(x)
    want_outs, want_dx, want_grads = ref.lora_dropout(x, params, dys, fs)
    ks = sum(dy.shape[1] for dy in dys)
    for (w, a, b, s), dy, f, wo, (wa, wb) in zip(params, dys, fs, want_outs, want_grads):
        w, a, b, dy = (t.double() for t in (w, a, b, dy))
        ca = _half(dtype) if adapter != dtype and dtype == BF else 0.0  # A, B cast to bf16
        xd = x * f
        xa, xa_abs = xd @ a.t(), xd.abs() @ a.abs().t()
        xa_err = u * xa.abs() + (acc(x.shape[1]) + ca) * xa_abs
        q, q_abs = s * (dy @ b), s * (dy.abs() @ b.abs())
        q_err = u * q.abs() + (acc(dy.shape[1]) + ca) * q_abs
        outs.append(ud * wo.abs() + acc(x.shape[1] + a.shape[0]) *
                    (x.abs() @ w.abs().t() + s * (xa_abs @ b.abs().t()))
                    + s * (xa_err @ b.abs().t()) + s * ((u + ca) * xa.abs() @ b.abs().t()))
        grads.append((ua * wa.abs() + q_err.t() @ xd.abs() + (acc(N)) * (q_abs.t() @ xd.abs()),
                      ua * wb.abs() + s * (dy.abs().t() @ xa_err)
                      + acc(N) * s * (dy.abs().t() @ xa_abs)))
        base += dy @ w
        base_abs += dy.abs() @ w.abs()
        extra += f * (q_err @ a.abs() + (acc(a.shape[0]) + ca) * (q_abs @ a.abs()))
        if composed or dtype != BF:
            extra += 2 * u * f * (q @ a).abs()
    # the products' rounding, one more for each adapter that is added by itself
    adds = 1 + (len(params) if composed or dtype != BF else 1)
    dx = ud * want_dx.abs() + adds * u * (base.abs() + want_dx.abs() + extra) \
        + acc(ks) * base_abs + extra
    return outs, dx, grads


def _near(got, want, bound, what):
    err = (got.detach().double().cpu().reshape(want.shape) - want).abs()
    worst = (err / (1.05 * bound + 1e-30)).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} times the bound"


def _check(dev, tokens, i, outs, ranks, ps, dtype=BF, adapter=None, seed=5, first=0, lead=None,
           alpha=None):
    from metal_liger_amd.ops.fused_lora import _dropped
    adapter = adapter or dtype
    lins = [_linear(dev, i, o, r, p, dtype, 10 * k, adapter, alpha)
            for k, (o, r, p) in enumerate(zip(outs, ranks, ps))]
    x = seeded((tokens, i), 100, dtype)
    dys = [seeded((tokens, o), 101 + k, dtype) for k, o in enumerate(outs)]
    xd = (x.view(*lead, i) if lead else x).to(dev).requires_grad_()
    ys = _dropped(lins, xd, seed, first)
    adapters = [t for m in lins for t in (m.lora_A["default"].weight, m.lora_B["default"].weight)]
    got = torch.autograd.grad(ys, [xd, *adapters],
                              [dy.to(dev).view(y.shape) for dy, y in zip(dys, ys)])
    fs = [ref.dropout_factors((tokens, i), p, seed, first + k) for k, p in enumerate(ps)]
    params = [_params(m) for m in lins]
    want, wdx, wg = ref.lora_dropout(x, params, dys, fs)
    composed = max(ranks) > 64 or any(v % 8 for v in (i, *outs))
    bo, bdx, bg = _bounds(x, params, dys, fs, dtype, adapter, composed)
    for k, y in enumerate(ys):
        assert y.dtype == dtype and y.shape[:-1] == xd.shape[:-1]
        _near(y, want[k], bo[k], f"out {k}")
    _near(got[0], wdx, bdx, "dx")
    for k in range(len(lins)):
        assert got[1 + 2 * k].dtype == adapter
        _near(got[1 + 2 * k], wg[k][0], bg[k][0], f"dA {k}")
        _near(got[2 + 2 * k], wg[k][1], bg[k][1], f"dB {k}")


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 31, 33, 64, 200, 257, 777])
def test_qkv_token_counts(dev, tokens):
    _check(dev, tokens, 256, (128, 64, 64), (16, 16, 16), (0.1, 0.1, 0.1))


@pytest.mark.parametrize("rank", [1, 4, 8, 16, 24, 32, 40, 48, 64, 72, 96, 128])
@pytest.mark.parametrize("n", [1, 2, 3])
def test_ranks(dev, rank, n):
    _check(dev, 130, 320, (192, 64, 72)[:n], (rank,) * n, (0.3,) * n)


@pytest.mark.parametrize("i", [8, 16, 24, 72, 104, 248, 264, 520, 1032, 2048])
@pytest.mark.parametrize("tokens", [3, 190])
def test_widths(dev, tokens, i):
    _check(dev, tokens, i, (40, 264), (16, 8), (0.2, 0.5))


@pytest.mark.parametrize("ps", [(0.0, 0.5, 0.0), (1.0, 0.1, 1e-5), (0.9, 0.0, 0.05)])
def test_rates_of_one_block(dev, ps):
    """Each projection has its own rate, none and one among them."""
    _check(dev, 130, 264, (128, 64, 64), (16, 8, 16), ps)


@pytest.mark.parametrize("adapter", [BF, F32])
def test_adapter_dtypes_and_scales(dev, adapter):
    _check(dev, 300, 512, (256, 128, 128), (12, 8, 16), (0.1, 0.2, 0.3), adapter=adapter, alpha=7.0)


@pytest.mark.parametrize("dtype", [F32, torch.float16])
@pytest.mark.parametrize("tokens, i, outs", [(1, 64, (32,)), (70, 99, (51, 7)),
                                             (130, 256, (128, 64, 64))])
def test_other_dtypes(dev, dtype, tokens, i, outs):
    _check(dev, tokens, i, outs, (8,) * len(outs), (0.25,) * len(outs), dtype, adapter=F32)


def test_odd_widths_in_bf16(dev):
    _check(dev, 70, 99, (51, 7), (8, 8), (0.25, 0.25))


def test_leading_dimensions(dev):
    _check(dev, 6 * 35, 128, (64,), (16,), (0.1,), lead=(2, 3, 35))


def test_large_block(dev):
    _check(dev, 2100, 2048, (2048, 1024, 1024), (16, 16, 16), (0.05, 0.05, 0.05), seed=2 ** 61 + 7)


def _block(**parts):
    m = nn.Module()
    for name, part in parts.items():
        setattr(m, name, part)
    return m


def test_entry_points_and_streams(dev):
    """qkv takes streams 0, 1, 2; a single projection 0; eval mode and lora_dropout
    False are the projections without dropout, bit for bit."""
    from metal_liger_amd import apply_fused_lora_qkv
    from metal_liger_amd.ops.fused_lora import _dropped, apply_fused_lora_linear
    lins = [_linear(dev, 128, o, 16, 0.4, BF, 10 * k) for k, o in enumerate((128, 64, 64))]
    attn = _block(q_proj=lins[0], k_proj=lins[1], v_proj=lins[2])
    x = seeded((50, 128), 1, BF).to(dev)
    got = apply_fused_lora_qkv(attn, x, lora_dropout=True, seed=3)
    for a, b in zip(got, _dropped(lins, x, 3)):
        assert torch.equal(a, b)
    y = apply_fused_lora_linear(lins[0], x, lora_dropout=True, seed=3)
    assert torch.equal(y, _dropped(lins[:1], x, 3)[0])
    assert not torch.equal(y, apply_fused_lora_linear(lins[0], x, lora_dropout=True, seed=4))
    plain = apply_fused_lora_qkv(attn, x)
    attn.eval()
    for a, b in zip(apply_fused_lora_qkv(attn, x, lora_dropout=True), plain):
        assert torch.equal(a, b)


def _mlp(dev, dtype, ranks, ps, H=256, I=512, adapter=None):  # noqa: E741
    shapes = ((H, I), (H, I), (I, H))
    lins = [_linear(dev, i, o, r, p, dtype, 10 * k, adapter)
            for k, ((i, o), r, p) in enumerate(zip(shapes, ranks, ps))]
    return lins, _block(gate_proj=lins[0], up_proj=lins[1], down_proj=lins[2])


@pytest.mark.parametrize("dtype, tokens, ranks, ps", [
    (F32, 300, (16, 16, 16), (0.2, 0.2, 0.2)), (BF, 300, (16, 16, 16), (0.2, 0.2, 0.2)),
    (BF, 1, (8, 8, 8), (0.5, 0.5, 0.5)), (BF, 777, (32, 16, 12), (0.1, 0.3, 0.2)),
    (BF, 65, (64, 64, 64), (0.1, 0.1, 0.1)), (BF, 130, (96, 16, 16), (0.2, 0.1, 0.3)),
    (BF, 200, (16, 16, 16), (0.0, 0.0, 0.4)), (BF, 200, (16, 16, 16), (0.4, 0.0, 0.0)),
    (torch.float16, 90, (8, 8, 8), (0.2, 0.2, 0.2))])
def test_mlp(dev, dtype, tokens, ranks, ps):
    """The MLP block: streams 0, 1, 2 for gate, up, down. Its inner tensors are
    rounded to the activation dtype, so that the norms of the errors are compared:
    about ten roundings of eps / 2 each in bf16 and fp16's fp32 products (rounded
    between), sums of 256 to 512 terms in fp32."""
    from metal_liger_amd import apply_fused_lora_mlp
    tol = {F32: 2e-5, BF: 2e-2, torch.float16: 2.5e-3}[dtype]
    lins, mlp = _mlp(dev, dtype, ranks, ps, adapter=F32 if dtype == torch.float16 else None)
    H = 256
    x = seeded((tokens, H), 1, dtype)
    dy = seeded((tokens, H), 2, dtype)
    xd = x.to(dev).requires_grad_()
    adapters = [t for m in lins for t in (m.lora_A["default"].weight, m.lora_B["default"].weight)]
    y = apply_fused_lora_mlp(mlp, xd, lora_dropout=True, seed=11)
    got = [y, *torch.autograd.grad(y, [xd, *adapters], dy.to(dev))]

    x64 = x.double().requires_grad_()
    leaves, t = [], x64
    out = []
    for k, m in enumerate(lins):
        w, a, b, s = _params(m)
        a, b = (v.double().requires_grad_() for v in (a, b))
        leaves += [a, b]
        t = out[0] * torch.sigmoid(out[0]) * out[1] if k == 2 else x64
        f = ref.dropout_factors(tuple(t.shape), ps[k], 11, k)
        out.append(t @ w.double().t() + s * ((t * f) @ a.t()) @ b.t())
    want = [out[2], *torch.autograd.grad(out[2], [x64, *leaves], dy.double())]
    assert y.dtype == dtype and [g.dtype for g in got[2:]] == [t.dtype for t in adapters]
    for g, w in zip(got, want):
        assert (g.double().cpu() - w).norm() <= tol * w.norm()


def test_mlp_without_dropout_is_the_plain_block(dev):
    from metal_liger_amd import apply_fused_lora_mlp
    _, mlp = _mlp(dev, BF, (16, 16, 16), (0.3, 0.3, 0.3))
    x = seeded((70, 256), 1, BF).to(dev)
    want = apply_fused_lora_mlp(mlp, x)
    assert not torch.equal(apply_fused_lora_mlp(mlp, x, lora_dropout=True), want)
    assert torch.equal(apply_fused_lora_mlp(mlp.eval(), x, lora_dropout=True), want)


def test_mlp_empty_batch(dev):
    from metal_liger_amd import apply_fused_lora_mlp
    lins, mlp = _mlp(dev, BF, (16, 16, 16), (0.3, 0.3, 0.3))
    x = torch.empty(0, 256, dtype=BF, device=dev, requires_grad=True)
    y = apply_fused_lora_mlp(mlp, x, lora_dropout=True)
    dx, db = torch.autograd.grad(y, [x, lins[2].lora_B["default"].weight], torch.empty_like(y))
    assert y.shape == dx.shape == (0, 256) and not db.any()


def test_dropped_infinities_stay_out_of_the_adapters(dev):
    """An element that every mask drops reaches no adapter, whatever it holds: XA and
    dA are those of a zero there."""
    from metal_liger_amd import hip_ops
    lins = [_linear(dev, 256, 64, 16, 0.5, BF, 10 * k) for k in range(2)]
    x = seeded((40, 256), 1, BF).to(dev)
    fs = [ref.dropout_factors((40, 256), 0.5, 21, k) for k in range(2)]
    gone = ((fs[0] == 0) & (fs[1] == 0)).to(dev)
    bad = torch.where(gone, torch.tensor(float("inf"), dtype=BF, device=dev), x)
    zero = torch.where(gone, torch.zeros((), dtype=BF, device=dev), x)
    seed = torch.tensor([21], device=dev)
    args = [[m.base_layer.weight.detach() for m in lins],
            [m.lora_A["default"].weight.detach() for m in lins],
            [m.lora_B["default"].weight.detach() for m in lins], [2.0, 2.0], 16, seed,
            [32768, 32768], 0]
    (*_, xa, packed), (*_, xa0, _) = (hip_ops.lora_dropout_fwd(t, *args) for t in (bad, zero))
    assert torch.equal(xa, xa0)
    dys = [seeded((40, 64), 2, BF).to(dev)] * 2
    _, g = hip_ops.lora_dropout_bwd(bad, dys, args[0], packed, [2.0, 2.0], xa, 16, seed,
                                    [32768, 32768], 0, [], BF)
    _, g0 = hip_ops.lora_dropout_bwd(zero, dys, args[0], packed, [2.0, 2.0], xa, 16, seed,
                                     [32768, 32768], 0, [], BF)
    assert torch.equal(g, g0)


@pytest.mark.parametrize("rank", [16, 96])
def test_strided_and_misaligned_operands(dev, rank):
    from metal_liger_amd.ops.fused_lora import _LoRA_Dropout
    lin = _linear(dev, 128, 64, rank, 0.3, BF, 0)
    seed = torch.tensor([4], device=dev)
    base = seeded((60, 300), 1, BF).to(dev)
    dys = seeded((60, 200), 2, BF).to(dev)
    w, a, b, s = (lin.base_layer.weight, lin.lora_A["default"].weight,
                  lin.lora_B["default"].weight, 2.0)

    def step(x, dy, w):
        x = x.detach().requires_grad_()
        y, = _LoRA_Dropout.apply(x, seed, (19661,), 0, w, a, b, s)
        return [y, *torch.autograd.grad(y, [x, a, b], dy)]

    x, dy = base[:, 3:131], dys[:, 5:69]
    want = step(x.contiguous(), dy.contiguous(), w)
    wide = torch.zeros(64, 140, dtype=BF, device=dev)
    wide[:, 1:129] = w.detach()
    for args in ((x, dy, w), (x.t().contiguous().t(), dy, w), (x, dy, wide[:, 1:129])):
        for got, ref_ in zip(step(*args), want):
            assert torch.equal(got, ref_)


def test_compile_and_opcheck(dev):
    from metal_liger_amd import _custom_ops as cops
    from metal_liger_amd import apply_fused_lora_mlp, apply_fused_lora_qkv, hip_ops
    lins = [_linear(dev, 128, o, 16, 0.4, BF, 10 * k) for k, o in enumerate((128, 64, 64))]
    attn = _block(q_proj=lins[0], k_proj=lins[1], v_proj=lins[2])
    mlp_lins, mlp = _mlp(dev, BF, (16, 16, 16), (0.3, 0.3, 0.3), 128, 256)
    x = seeded((50, 128), 1, BF).to(dev).requires_grad_()
    seed = torch.tensor([7], device=dev)
    for fn, ms in ((lambda t: apply_fused_lora_qkv(attn, t, lora_dropout=True, seed=seed), lins),
                   (lambda t: (apply_fused_lora_mlp(mlp, t, lora_dropout=True, seed=seed),),
                    mlp_lins)):
        leaves = [x, *(w for m in ms for w in (m.lora_A["default"].weight,
                                              m.lora_B["default"].weight))]
        want = fn(x)
        got = torch.compile(fn, fullgraph=True, backend="aot_eager")(x)
        dys = [seeded(tuple(y.shape), 3, BF).to(dev) for y in want]
        for p, q in zip([*got, *torch.autograd.grad(got, leaves, dys)],
                        [*want, *torch.autograd.grad(want, leaves, dys)]):
            assert torch.equal(p, q)
    checks = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    xd = x.detach()
    for rank, fwd, bwd in ((16, cops.lora_dropout_fwd, cops.lora_dropout_bwd),
                           (72, cops.lora_dropout_wide_fwd, cops.lora_dropout_wide_bwd)):
        m = _linear(dev, 128, 64, rank, 0.4, BF, 3)
        args = (xd, [m.base_layer.weight.detach()], [m.lora_A["default"].weight.detach()],
                [m.lora_B["default"].weight.detach()], [2.0], rank, seed, [1000], 1)
        torch.library.opcheck(fwd, args, test_utils=checks)
        y, xa, packed = fwd(*args)
        for spec, dtype in (([], F32), ([], BF), ([0, rank, 128, 128], BF)):
            if rank == 16 or spec or dtype == F32:
                torch.library.opcheck(bwd, (xd, [y], args[1], packed, [2.0], xa, rank, seed, [1000],
                                            1, spec, dtype), test_utils=checks)
    args = (xd, [m.base_layer.weight.detach() for m in mlp_lins],
            [m.lora_A["default"].weight.detach() for m in mlp_lins],
            [m.lora_B["default"].weight.detach() for m in mlp_lins], [2.0] * 3, 16, seed, [1000] * 3)
    torch.library.opcheck(cops.lora_dropout_mlp_fwd, args, test_utils=checks)
    y, gate, up, h, xa, xa_d, packed = cops.lora_dropout_mlp_fwd(*args)
    torch.library.opcheck(cops.lora_dropout_mlp_bwd,
                          (xd, gate, up, h, y, args[1], packed, [2.0] * 3, xa, xa_d, 16, seed,
                           [1000] * 3, [], BF), test_utils=checks)
    f32 = [t.float() for t in (xd, lins[0].base_layer.weight.detach(),
                               lins[0].lora_A["default"].weight.detach(),
                               lins[0].lora_B["default"].weight.detach())]
    args = (f32[0], [f32[1]], [f32[2]], [f32[3]], [2.0], seed, [1000], 0)
    torch.library.opcheck(cops.lora_dropout_f32_fwd, args, test_utils=checks)
    y, xa = cops.lora_dropout_f32_fwd(*args)
    torch.library.opcheck(cops.lora_dropout_f32_bwd, (f32[0], [y], [f32[1]], [f32[2]], [f32[3]], [2.0],
                                                      [xa], seed, [1000], 0), test_utils=checks)
    assert hip_ops.drop_scale(65536) == 0.0


def test_drawn_seeds(dev):
    from metal_liger_amd.ops.fused_lora import apply_fused_lora_linear
    lin = _linear(dev, 128, 64, 8, 0.5, BF, 0)
    x = seeded((40, 128), 1, BF).to(dev)
    torch.manual_seed(5)
    a, b = (apply_fused_lora_linear(lin, x, lora_dropout=True) for _ in range(2))
    torch.manual_seed(5)
    assert torch.equal(a, apply_fused_lora_linear(lin, x, lora_dropout=True))
    assert not torch.equal(a, b)


@pytest.mark.parametrize("rank", [16, 96])
def test_gradient_is_reproducible_and_accumulates(dev, rank):
    from metal_liger_amd.ops.fused_lora import _dropped
    lins = [_linear(dev, 264, o, rank, 0.3, BF, 10 * k) for k, o in enumerate((128, 64))]
    x = seeded((500, 264), 1, BF).to(dev).requires_grad_()
    dys = [seeded((500, o), 2, BF).to(dev) for o in (128, 64)]
    leaves = [x, *(t for m in lins for t in (m.lora_A["default"].weight,
                                            m.lora_B["default"].weight))]
    ys = _dropped(lins, x, 7)
    first = torch.autograd.grad(ys, leaves, dys, retain_graph=True)
    for got in (torch.autograd.grad(ys, leaves, dys),
                torch.autograd.grad(_dropped(lins, x, 7), leaves, dys)):
        for a, b in zip(first, got):
            assert torch.equal(a, b)


def test_gradient_by_differences(dev):
    """d loss along a direction in x, A and B, in fp32: a central difference of step h
    is off by O(h^2) of the loss's curvature (none in x, and bilinear in A, B along
    one of them at a time) and by the loss's rounding over h."""
    from metal_liger_amd.ops.fused_lora import _dropped
    lin = _linear(dev, 96, 64, 8, 0.3, F32, 0)
    x = seeded((40, 96), 1).to(dev).requires_grad_()
    dy = seeded((40, 64), 2).to(dev)
    leaves = [x, lin.lora_A["default"].weight, lin.lora_B["default"].weight]
    loss = lambda: (_dropped([lin], x, 9)[0].double() * dy.double()).sum()  # noqa: E731
    grads = torch.autograd.grad(loss(), leaves)
    h = 2.0 ** -4
    for leaf, g in zip(leaves, grads):
        d = seeded(tuple(leaf.shape), 3).to(dev)
        d *= leaf.detach().norm() / d.norm()
        with torch.no_grad():
            leaf.add_(d, alpha=h)
            up = loss().item()
            leaf.sub_(d, alpha=2 * h)
            down = loss().item()
            leaf.add_(d, alpha=h)
        want = (g.double() * d.double()).sum().item()
        # outputs rounded to fp32 after sums of 96 + 8 terms, 40 x 64 of them
        size = (_dropped([lin], x, 9)[0].double().abs() * dy.double().abs()).sum().item()
        assert abs((up - down) / (2 * h) - want) <= 2 * 120 * 2.0 ** -24 * size / h


def test_captured_step(dev):
    """A captured forward and backward, its seed advanced by the step itself."""
    from metal_liger_amd import apply_fused_lora_qkv
    lins = [_linear(dev, 264, o, 16, 0.3, BF, 10 * k) for k, o in enumerate((128, 64, 64))]
    attn = _block(q_proj=lins[0], k_proj=lins[1], v_proj=lins[2])
    x = seeded((200, 264), 1, BF).to(dev).requires_grad_()
    dys = [seeded((200, o), 2, BF).to(dev) for o in (128, 64, 64)]
    leaves = [x, *(t for m in lins for t in (m.lora_A["default"].weight,
                                            m.lora_B["default"].weight))]
    seed = torch.tensor([50], device=dev)

    def step(s):
        ys = apply_fused_lora_qkv(attn, x, lora_dropout=True, seed=s)
        return [*ys, *torch.autograd.grad(ys, leaves, dys)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(seed)
        seed.add_(1)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(50 + i)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_empty_batch(dev):
    from metal_liger_amd.ops.fused_lora import apply_fused_lora_linear
    lin = _linear(dev, 64, 32, 8, 0.5, BF, 0)
    x = torch.empty(0, 64, dtype=BF, device=dev, requires_grad=True)
    y = apply_fused_lora_linear(lin, x, lora_dropout=True)
    dx, da = torch.autograd.grad(y, [x, lin.lora_A["default"].weight],
                                 torch.empty(0, 32, dtype=BF, device=dev))
    assert y.shape == (0, 32) and dx.shape == (0, 64) and not da.any()


def test_refusals(dev):
    from metal_liger_amd.ops.fused_lora import apply_fused_lora_linear
    lin = _linear(dev, 64, 32, 8, 0.5, BF, 0)
    with pytest.raises(ValueError, match="do not fit"):
        apply_fused_lora_linear(lin, torch.zeros(4, 72, dtype=BF, device=dev), lora_dropout=True)
    with pytest.raises(TypeError, match="floating point"):
        apply_fused_lora_linear(lin, torch.zeros(4, 64, dtype=torch.int64, device=dev),
                                lora_dropout=True)
    with pytest.raises(ValueError, match="ROCm GPU"):
        apply_fused_lora_linear(lin, torch.zeros(4, 64, dtype=BF), lora_dropout=True)


def test_patched_model_against_peft_formula(dev, monkeypatch):
    """A tiny model with a trained embedding and LoRA dropout, patched, against the
    unpatched one in which each LoRA Linear drops by the oracle's masks: loss, adapter
    and embedding gradients in fp32 (relative norms, sums of up to 512 terms through
    two layers)."""
    from metal_liger_amd import apply_metal_liger_to_qwen3vl
    from metal_liger_amd.ops import fused_lora
    from tests.qwen_tiny import build
    from tests.test_training_ops import with_dropout
    p = 0.25
    fused, plain = (with_dropout(build(seed=3), p).to(dev).train() for _ in range(2))
    seeds = iter(range(1000, 2000))
    monkeypatch.setattr(fused_lora, "seed_tensor", lambda seed, device: (
        torch.tensor([next(seeds)], device=device) if seed is None else seed))
    apply_metal_liger_to_qwen3vl(fused, lora_dropout=True, fuse_embedding=True, fuse_swiglu=False)
    drawn = 1000
    for layer in plain.base_model.model.model.layers:  # one seed for q, k, v, one for o, one for the MLP
        for names, parent in ((("q_proj", "k_proj", "v_proj"), layer.self_attn),
                              (("o_proj",), layer.self_attn),
                              (("gate_proj", "up_proj", "down_proj"), layer.mlp)):
            for k, name in enumerate(names):
                lin = getattr(parent, name)

                def forward(x, lin=lin, key=drawn, k=k):
                    f = ref.dropout_factors(tuple(x.shape), p, key, k).to(x)
                    w, a, b, s = fused_lora._get_lora_params(lin)
                    return x @ w.t() + s * ((x * f) @ a.t()) @ b.t()

                lin.forward = forward
            drawn += 1
    ids = torch.randint(0, 512, (2, 48), generator=torch.Generator().manual_seed(1)).to(dev)
    grads = []
    for model in (fused, plain):
        for n, q in model.named_parameters():
            q.requires_grad_("lora_" in n or "embed_tokens" in n)
        lm = model.base_model.model
        out = lm(ids, labels=ids, use_cache=False)
        out.loss.backward()
        named = dict(model.named_parameters())
        grads.append([out.loss.detach(), *(named[n].grad for n in sorted(named)
                                           if "lora_" in n or "embed_tokens" in n)])
    assert next(seeds) == drawn
    for a, b in zip(*grads):
        assert (a - b).double().norm() <= 1e-4 * b.double().norm() + 1e-12
