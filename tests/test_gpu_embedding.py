"""The token embedding and its gradient on the GPU against fp64.

Bounds: a looked-up element is one fp32 product (two roundings of 2^-24, of the
scale and of the product) rounded to its type (eps / 2). A gradient element is a sum
of m terms in fp32, off by at most (m + 2) 2^-24 of the terms' magnitudes, times the
scale, and rounded to its type (fp16 below its smallest normal number: half of 2^-24).
"""

import pytest
import torch

from oracle import training_ops as ref
from tests.parity import seeded

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _op():
    from metal_liger_amd import fused_embedding
    return fused_embedding


def _ids(kind, n, vocab, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), generator=g)
    if kind == "same":
        return torch.full((n,), vocab // 2)
    if kind == "ends":
        return torch.randint(0, 2, (n,), generator=g) * (vocab - 1)
    ids = torch.randint(0, vocab, (n,), generator=g)          # half of them one id
    ids[torch.rand(n, generator=g) < 0.5] = vocab // 3
    return ids


def _check(got, want, terms, counts):
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = want.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 1e-3) \
        + (counts + 2) * 2.0 ** -24 * terms + tiny
    err = (got.detach().double().cpu() - want).abs()
    assert got.shape == want.shape
    assert bool((err <= bound).all()), (err - bound).max()


def _check_grad(got, ids, dy, vocab, scale=1.0, pad=None):
    ids, dy = ids.cpu(), dy.cpu()
    _check(got, ref.embedding_grad(ids, dy, vocab, scale, pad),
           ref.embedding_grad(ids, dy.abs(), vocab, scale, pad),
           ref.embedding_grad(ids, torch.ones(*dy.shape[:-1], 1), vocab, 1.0, pad))


def _run(dev, ids, vocab, hidden, dtype, scale=1.0, pad=None, id_type=torch.int64):
    w = seeded((vocab, hidden), 1, dtype).to(dev).requires_grad_()
    dy = seeded((*ids.shape, hidden), 2, dtype).to(dev)
    y = _op()(ids.to(dev, id_type), w, scale, pad)
    want = w.detach().double().cpu()[ids] * scale
    assert y.dtype == dtype
    _check(y, want, want.abs(), torch.ones(()))
    dw, = torch.autograd.grad(y, w, dy)
    assert dw.dtype == dtype
    _check_grad(dw, ids, dy, vocab, scale, pad)
    return dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hidden", [1, 7, 64, 250, 1001, 2048])
@pytest.mark.parametrize("kind", ["uniform", "same", "ends", "half"])
def test_values_and_gradients(dev, kind, hidden, dtype):
    _run(dev, _ids(kind, 777, 503), 503, hidden, dtype, scale=1.7)


@pytest.mark.parametrize("kind", ["uniform", "same", "half"])
@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 8191, 8192, 8193, 20000, 70001])
def test_token_counts(dev, tokens, kind):
    _run(dev, _ids(kind, tokens, 30011), 30011, 40, torch.float32)


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 4096, 262143, 262145, 1 << 22])
def test_vocabularies(dev, vocab):
    _run(dev, _ids("uniform", 3000, vocab), vocab, 8, torch.bfloat16)


@pytest.mark.parametrize("pad", [0, 17, -1])
def test_padding_row_gets_no_gradient(dev, pad):
    ids = _ids("uniform", 500, 40)
    ids[100:200] = pad % 40
    dw = _run(dev, ids, 40, 72, torch.bfloat16, pad=pad)
    assert not dw[pad].any()


@pytest.mark.parametrize("id_type", [torch.int64, torch.int32])
def test_shapes_and_id_types(dev, id_type):
    for shape in ((), (1,), (3, 5), (2, 3, 4)):
        _run(dev, _ids("uniform", 24, 50)[:torch.Size(shape).numel()].view(shape), 50, 33,
             torch.float32, id_type=id_type)


def test_empty(dev):
    w = seeded((10, 16), 1).to(dev).requires_grad_()
    y = _op()(torch.empty(0, 3, dtype=torch.int64, device=dev), w)
    dw, = torch.autograd.grad(y, w, torch.empty(0, 3, 16, device=dev))
    assert y.shape == (0, 3, 16) and dw.shape == (10, 16) and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dev, dtype):
    """Strided ids, misaligned and strided tables and gradients."""
    big = seeded((60, 91), 3, dtype).to(dev)
    ids = torch.randint(0, 25, (30, 4), generator=torch.Generator().manual_seed(4)).to(dev)
    grads = seeded((40, 91), 5, dtype).to(dev)
    for w in (big[:, 1:65], big[::2, :64], big.t()[:64, :].t(), big[1:, 3:67]):
        w = w.detach().requires_grad_()
        i = ids[::3, 1]
        for dy in (grads[:10, 2:66], grads[::4, :64], grads.t()[:64, :10].t(),
                   grads[:1, :64].expand(10, 64)):
            y = _op()(i, w)
            assert torch.equal(y, w[i])
            dw, = torch.autograd.grad(y, w, dy)
            _check_grad(dw, i, dy, w.shape[0])


def test_ids_outside_the_table(dev):
    """They give rows of NaN and no gradient; the others are as without them."""
    w = seeded((20, 24), 1).to(dev).requires_grad_()
    ids = torch.tensor([3, -1, 20, 5, 2 ** 31 - 1, -(2 ** 31), 3], device=dev)
    for i in (ids, ids.int(), torch.where(ids == 20, 2 ** 40, ids)):
        y = _op()(i, w)
        bad = torch.tensor([1, 2, 4, 5], device=dev)
        good = torch.tensor([0, 3, 6], device=dev)
        assert torch.isnan(y[bad]).all() and torch.equal(y[good], w[i[good].long()])
        dy = seeded((7, 24), 2).to(dev)
        dw, = torch.autograd.grad(y, w, dy)
        _check_grad(dw, i[good].cpu(), dy[good], 20)


def test_gradient_is_reproducible(dev):
    ids = _ids("half", 30000, 5000).to(dev)
    dy = seeded((30000, 72), 2, torch.bfloat16).to(dev)
    op = torch.ops.metal_liger_amd.embedding_bwd
    first = op(ids, dy, 5000, -1, 1.0)
    for _ in range(5):
        assert torch.equal(op(ids, dy, 5000, -1, 1.0), first)


def test_offsets_past_32_bits(dev):
    """A table and a gradient of more elements than a signed 32-bit index holds."""
    vocab, hidden = 1 << 19, 4104
    w = torch.zeros(vocab, hidden, dtype=torch.bfloat16, device=dev)
    ids = torch.tensor([vocab - 1, 0, vocab - 1, vocab - 2], device=dev)
    w[vocab - 1] = 3.0
    y = _op()(ids, w)
    assert torch.equal(y[0], w[vocab - 1]) and torch.equal(y[3], w[vocab - 2])
    dy = seeded((4, hidden), 2, torch.bfloat16).to(dev)
    dw = torch.ops.metal_liger_amd.embedding_bwd(ids, dy, vocab, -1, 1.0)
    assert torch.equal(dw[vocab - 1], (dy[0].float() + dy[2].float()).bfloat16())
    assert torch.equal(dw[0], dy[1]) and torch.equal(dw[vocab - 2], dy[3])
    assert not dw[1:vocab - 2].any()


def test_many_tokens_past_32_bits(dev):
    """A gradient of the output with more than 2^31 elements."""
    n, hidden = (1 << 19) + 3, 4104
    dy = torch.ones(1, 1, dtype=torch.bfloat16, device=dev).expand(n, hidden).contiguous()
    ids = torch.zeros(n, dtype=torch.int64, device=dev)
    ids[-1] = 1
    dw = torch.ops.metal_liger_amd.embedding_bwd(ids, dy, 4, -1, 1.0)
    assert torch.all(dw[1] == 1) and not dw[2:].any()
    assert torch.all(dw[0].float() == torch.tensor(float(n - 1)).bfloat16().float().item())


def test_other_stream(dev):
    ids = _ids("half", 9000, 3000).to(dev)
    w = seeded((3000, 64), 1).to(dev).requires_grad_()
    dy = seeded((9000, 64), 2).to(dev)
    want = torch.autograd.grad(_op()(ids, w), w, dy)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = torch.autograd.grad(_op()(ids, w), w, dy)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_captured_step(dev):
    w = seeded((3000, 64), 1).to(dev).requires_grad_()
    ids = _ids("half", 9000, 3000).to(dev)
    dy = seeded((9000, 64), 2).to(dev)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.autograd.grad(_op()(ids, w), w, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _op()(ids, w)
        dw, = torch.autograd.grad(y, w, dy)
    for k in range(4):
        ids.copy_(_ids("half" if k % 2 else "uniform", 9000, 3000, seed=k))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(_op()(ids, w), w, dy)[0]
        assert torch.equal(dw, want) and torch.equal(y, w[ids])


def test_refusals(dev):
    w = torch.zeros(4, 8, device=dev)
    i = torch.zeros(3, dtype=torch.int64, device=dev)
    with pytest.raises(TypeError, match="int64 or int32"):
        _op()(i.float(), w)
    with pytest.raises(ValueError, match="table"):
        _op()(i, torch.zeros(0, 8, device=dev))
    with pytest.raises(TypeError, match="dtype"):
        _op()(i, w.double())
    with pytest.raises(ValueError, match="different devices|ROCm GPU"):
        _op()(i.cpu(), w)
    with pytest.raises(ValueError, match="does not match ids"):
        torch.ops.metal_liger_amd.embedding_bwd(i, torch.zeros(2, 8, device=dev), 4, -1, 1.0)


def test_compile(dev):
    w = seeded((50, 24), 1).to(dev).requires_grad_()
    ids = _ids("half", 60, 50).to(dev)
    dy = seeded((60, 24), 2).to(dev)
    step = lambda i, t: _op()(i, t, 2.0, 3)  # noqa: E731
    want = step(ids, w)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(ids, w)
    assert torch.equal(got, want)
    assert torch.equal(*(torch.autograd.grad(t, w, dy)[0] for t in (got, want)))
    checks = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    ops = torch.ops.metal_liger_amd
    torch.library.opcheck(ops.embedding_fwd.default, (ids, w.detach(), 1.0), test_utils=checks)
    torch.library.opcheck(ops.embedding_bwd.default, (ids, dy, 50, -1, 1.0), test_utils=checks)
