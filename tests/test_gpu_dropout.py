"""Dropout on the GPU against the oracle's masks: values, gradients, layouts, seeds,
captured steps.

Bounds: a kept element is x times the factor (itself rounded to fp32), plus the
residual where there is one, in fp32 (at most three roundings of 2^-24 of the terms),
and rounded once to its type (half a step, eps / 2; fp16 below its smallest normal
number: half of 2^-24)."""

import pytest
import torch

from oracle import training_ops as ref
from tests.parity import seeded

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1,), (7,), (8,), (9,), (1, 2048), (37, 999), (3, 5, 64), (513, 264)]


def _op():
    from metal_liger_amd import fused_dropout
    return fused_dropout


def _check(got, x, f, res=None):
    """got against x * f (+ res) in fp64, elementwise."""
    want = x.double().cpu() * f
    terms = want.abs()
    if res is not None:
        want = want + res.double().cpu()
        terms = terms + res.double().cpu().abs()
    bound = want.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 1e-3) + 3 * terms * 2.0 ** -24
    bound += 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    err = (got.detach().double().cpu() - want).abs()
    assert got.shape == want.shape
    assert bool((err <= bound).all()), (err - bound).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_values_and_gradients(dev, shape, dtype, residual):
    x = seeded(shape, 1, dtype).to(dev).requires_grad_()
    res = seeded(shape, 2, dtype).to(dev).requires_grad_() if residual else None
    dy = seeded(shape, 3, dtype).to(dev)
    y = _op()(x, 0.3, residual=res, seed=77, stream=5)
    y.backward(dy)
    f = ref.dropout_factors(shape, 0.3, 77, 5)
    assert y.dtype == dtype and y.is_contiguous()
    _check(y, x.detach(), f, None if res is None else res.detach())
    _check(x.grad, dy, f)
    if residual:
        assert torch.equal(res.grad, dy)


@pytest.mark.parametrize("p", [1e-5, 0.05, 0.5, 0.99999, 1.0])
def test_rates(dev, p):
    x = seeded((64, 129), 4).to(dev)
    _check(_op()(x, p, seed=3), x, ref.dropout_factors((64, 129), p, 3))


@pytest.mark.parametrize("seed", [0, -1, 2 ** 63 - 1, -(2 ** 63), 2 ** 64 - 5, 2 ** 40 + 3])
def test_seeds(dev, seed):
    x = torch.ones(4096, device=dev)
    f = ref.dropout_factors((4096,), 0.5, seed).float()
    assert torch.equal(_op()(x, 0.5, seed=seed).cpu(), f)
    signed = (seed + 2 ** 63) % 2 ** 64 - 2 ** 63
    assert torch.equal(_op()(x, 0.5, seed=torch.tensor([signed], device=dev)).cpu(), f)


def test_streams_differ(dev):
    x = torch.ones(4096, device=dev)
    for s in (0, 1, 2 ** 32 - 1):
        assert torch.equal(_op()(x, 0.5, seed=9, stream=s).cpu(),
                           ref.dropout_factors((4096,), 0.5, 9, s).float())


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dev, dtype):
    """Strided, misaligned and broadcast inputs go by row-major order."""
    base = seeded((40, 57), 5, dtype).to(dev)
    views = [base.t(), base[:, 1:], base[::2, ::3], base[3:4].expand(9, 57), base.flatten()[1:],
             base.flatten()[3:1027]]
    for v in views:
        f = ref.dropout_factors(tuple(v.shape), 0.4, 6)
        _check(_op()(v, 0.4, seed=6), v, f)
        _check(_op()(v, 0.4, seed=6, residual=v), v, f, v)
    x = base.clone().requires_grad_()
    _op()(x, 0.4, seed=6).sum().backward()            # an expanded gradient
    _check(x.grad, torch.ones_like(base), ref.dropout_factors((40, 57), 0.4, 6))


def test_empty(dev):
    x = torch.empty(0, 8, device=dev, requires_grad=True)
    y = _op()(x, 0.5)
    y.sum().backward()
    assert y.shape == (0, 8) and x.grad.shape == (0, 8)


def test_dropped_infinities_and_nan_give_zero(dev):
    x = torch.full((4096,), float("inf"), device=dev)
    x[::2] = float("nan")
    f = ref.dropout_factors((4096,), 0.5, 8)
    y = _op()(x, 0.5, seed=8).cpu()
    assert torch.equal(y == 0, f == 0) and torch.equal(torch.isfinite(y), f == 0)


def test_offsets_past_32_bits(dev):
    """More elements than a signed 32-bit index holds: the ends of the tensor."""
    n = 2 ** 31 + 1001
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    y = _op()(x, 0.5, seed=10)
    for first in (0, 2 ** 31 - 512, n - 1001):
        f = ref.dropout_factors((1001,), 0.5, 10, first=first)
        assert torch.equal(y[first:first + 1001].double().cpu(), f), first


def test_drawn_seeds_follow_torch_generator(dev):
    x = torch.ones(4096, device=dev)
    torch.manual_seed(1)
    a, b = _op()(x, 0.5), _op()(x, 0.5)
    torch.manual_seed(1)
    assert torch.equal(a, _op()(x, 0.5)) and not torch.equal(a, b)


def test_module_and_checkpointing(dev):
    from torch.utils.checkpoint import checkpoint

    from metal_liger_amd import MetalLigerDropout
    drop = MetalLigerDropout(0.5)
    x = seeded((64, 32), 7).to(dev).requires_grad_()
    y = checkpoint(lambda t: drop(t * 2), x, use_reentrant=False)
    y.sum().backward()
    assert torch.equal(x.grad != 0, y != 0)
    assert torch.equal(drop.eval()(x), x)
    assert torch.equal(drop(x, residual=x), x + x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [4099, 4096])
def test_in_place_through_the_c_abi(dev, dtype, n):
    """out may be x or residual, aligned or not; what lies behind stays as it was."""
    from metal_liger_amd import _hip
    for shift in (0, 1):
        buf = [seeded((n + 16,), k, dtype).to(dev) for k in (1, 2)]
        seed = torch.tensor([4], device=dev)
        x, res = (b[shift:shift + n] for b in buf)
        want = _op()(x, 0.3, residual=res, seed=4)
        for out in (0, 1):
            t = [b.clone() for b in buf]
            p = [b[shift:].data_ptr() for b in t]
            _hip.call("ml_dropout", p[0], p[1], p[out], n, 19661, 65536 / (65536 - 19661),
                      seed.data_ptr(), 0, _hip.DTYPE_TAG[dtype], _hip.stream_of(seed))
            assert torch.equal(t[out][shift:shift + n], want)
            assert torch.equal(t[out][shift + n:], buf[out][shift + n:])
            assert torch.equal(t[1 - out], buf[1 - out])


def test_other_stream(dev):
    x = seeded((512, 512), 8).to(dev)
    want = _op()(x, 0.3, seed=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _op()(x, 0.3, seed=1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_seed_changed_before_the_backward_is_an_error(dev):
    x = seeded((64,), 9).to(dev).requires_grad_()
    seed = torch.tensor([5], device=dev)
    y = _op()(x, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("given", [False, True])
def test_captured_step(dev, given):
    """A captured forward and backward: new masks at each replay, the same in both
    directions, and those of the seed where one is given."""
    x = torch.ones(4096, device=dev, requires_grad=True)
    dy = torch.ones(4096, device=dev)
    seed = torch.tensor([100], device=dev) if given else None
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.autograd.grad(_op()(x, 0.5, seed=seed), x, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _op()(x, 0.5, seed=seed)
        dx, = torch.autograd.grad(y, x, dy)
        if given:
            seed.add_(1)
    seen = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dx)
        if given:
            assert torch.equal(y.detach().cpu(), ref.dropout_factors((4096,), 0.5, 100 + i).float())
        seen.append(y.detach().clone())
        _op()(x.detach(), 0.5)                       # the program's own eager work
        torch.cuda.synchronize()
    assert all(not torch.equal(a, b) for a, b in zip(seen, seen[1:]))


def test_refusals(dev):
    x = torch.ones(8, device=dev)
    with pytest.raises(ValueError, match="residual"):
        _op()(x, 0.5, residual=torch.ones(4, device=dev))
    with pytest.raises(ValueError, match="residual"):
        _op()(x, 0.5, residual=x.bfloat16())
    with pytest.raises(TypeError, match="one int64"):
        _op()(x, 0.5, seed=torch.ones(1, device=dev))
    with pytest.raises(ValueError, match="ROCm GPU"):
        _op()(x, 0.5, seed=torch.ones(1, dtype=torch.int64))
    with pytest.raises(TypeError, match="dtype"):
        _op()(x.double(), 0.5)


def test_compile(dev):
    def step(x, res, seed):
        return _op()(x, 0.3, residual=res, seed=seed)

    x, res = (seeded((33, 65), k).to(dev).requires_grad_() for k in (1, 2))
    seed = torch.tensor([4], device=dev)
    want = step(x, res, seed)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(x, res, seed)
    assert torch.equal(got, want)
    dy = seeded((33, 65), 3).to(dev)
    for a, b in zip(torch.autograd.grad(got, [x, res], dy), torch.autograd.grad(want, [x, res], dy)):
        assert torch.equal(a, b)
    op = torch.ops.metal_liger_amd.dropout.default
    for r in (None, res.detach()):
        torch.library.opcheck(op, (x.detach(), r, seed, 1000, 3, 1.5), test_utils=(
            "test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))
