"""The feed-forward operators as they are used: layouts, frozen parts, several of them
in a step, captured steps, other streams, compilation, models that the patcher routed.

Criterion where bf16 modules are compared with fused ones ("no less accurate"): against
the same module in fp32 on the same bf16 parameters, the fused result's relative error
is at most 1.5 times the unfused bf16 module's plus 2e-3 (the two round at different
points)."""

import copy
import types

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from oracle import feed_forward as ref
from tests import qwen_tiny
from tests.parity import rel_fro, seeded

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
CHECKS = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")


def _linear(*args, **kw):
    from metal_liger_amd import fused_linear
    return fused_linear(*args, **kw)


def _mlp(*args, **kw):
    from metal_liger_amd import fused_swiglu_mlp
    return fused_swiglu_mlp(*args, **kw)


def _swiglu(*args, **kw):
    from metal_liger_amd.ops.fused_swiglu import fused_swiglu
    return fused_swiglu(*args, **kw)


def _leaf(shape, seed, dev, dtype=BF, scale=1.0):
    return seeded(shape, seed, dtype, scale).to(dev).requires_grad_()


def _grads(y, leaves, dy):
    return torch.autograd.grad(y, leaves, dy)


# ------------------------------------------------------------------ layouts --

@pytest.mark.parametrize("dtype", [torch.float32, BF, torch.float16])
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_layouts(dev, dtype, checkpoint):
    """Column slices, transposed and misaligned weights, broadcast residuals and
    gradients: the same values and gradients as dense copies."""
    M, K, N = 70, 72, 136
    big = seeded((M, 2 * K + 5), 1, dtype).to(dev)
    xs = [big[:, 3:3 + K], big[:, 8:8 + K], big.t()[:K].t(), big[::2, :K].repeat(2, 1)]
    wt = seeded((K, N), 2, dtype, 0.1).to(dev)
    wbig = seeded((N * K + 3,), 3, dtype, 0.1).to(dev)
    ws = [wt.t(), wbig[3:].view(N, K), wbig[:N * K].view(N, K)]
    bs = [seeded((N + 1,), 4, dtype).to(dev)[1:], seeded((2 * N,), 5, dtype).to(dev)[::2]]
    rs = [seeded((1, N), 6, dtype).to(dev), seeded((M, N + 3), 7, dtype).to(dev)[:, 3:]]
    for i in range(4):
        x, w, b, r = xs[i], ws[i % 3], bs[i % 2], rs[i % 2]
        dy = [torch.ones((), dtype=dtype, device=dev).expand(M, N),
              seeded((N, M), 8, dtype).to(dev).t()][i % 2]
        outs = []
        for dense in (False, True):
            ts = [t.detach().clone(memory_format=torch.contiguous_format) if dense else t.detach()
                  for t in (x, w, b, r)]
            ts = [t.requires_grad_() for t in ts]
            g = dy.clone(memory_format=torch.contiguous_format) if dense else dy
            y = _linear(ts[0], ts[1], ts[2], "gelu", ts[3].expand(M, N), checkpoint)
            outs.append([y, *_grads(y, ts, g)])
        for a, b_ in zip(*outs):
            assert a.shape == b_.shape and torch.equal(a, b_)


def test_leading_dimensions(dev):
    x, w, b = _leaf((2, 3, 5, 64), 1, dev), _leaf((40, 64), 2, dev), _leaf((40,), 3, dev)
    r, dy = _leaf((2, 3, 5, 40), 4, dev), seeded((2, 3, 5, 40), 5, BF).to(dev)
    y = _linear(x, w, b, "silu", r)
    flat = _linear(x.reshape(30, 64), w, b, "silu", r.reshape(30, 40))
    assert y.shape == (2, 3, 5, 40) and torch.equal(y.reshape(30, 40), flat)
    for a, c in zip(_grads(y, [x, w, b, r], dy), _grads(flat, [x, w, b, r], dy.reshape(30, 40))):
        assert torch.equal(a, c)
    one = _linear(x[0, 0, 0], w, b, "silu", r[0, 0, 0])  # a vector
    assert one.shape == (40,)
    g = _grads(one, [x], dy[0, 0, 0])[0]
    assert g.shape == x.shape and bool((g.view(30, 64)[1:] == 0).all())
    wg, wu, wd = _leaf((48, 64), 6, dev), _leaf((48, 64), 7, dev), _leaf((40, 48), 8, dev)
    y = _mlp(x, wg, wu, wd, r)
    flat = _mlp(x.reshape(30, 64), wg, wu, wd, r.reshape(30, 40))
    assert torch.equal(y.reshape(30, 40), flat)
    assert _grads(y, [x], dy)[0].shape == x.shape


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, BF, torch.float16])
def test_no_rows(dev, shape, dtype):
    x = _leaf(shape, 1, dev, dtype)
    w, b = _leaf((40, 64), 2, dev, dtype), _leaf((40,), 3, dev, dtype)
    for held in (None, "fp8"):
        y = _linear(x, w, b, "gelu", checkpoint=held)
        assert y.shape == (*shape[:-1], 40)
        dx, dw, db = _grads(y, [x, w, b], torch.empty_like(y))
        assert dx.shape == x.shape and bool((dw == 0).all()) and bool((db == 0).all())
        ws = [_leaf(s, 4, dev, dtype) for s in ((48, 64), (48, 64), (40, 48))]
        y = _mlp(x, *ws, checkpoint=held)
        assert y.shape == (*shape[:-1], 40)
        dx, *dws = _grads(y, [x, *ws], torch.empty_like(y))
        assert dx.shape == x.shape and all(bool((g == 0).all()) for g in dws)
    with torch.no_grad():
        assert _linear(x, w, b).shape == _mlp(x, *ws).shape == (*shape[:-1], 40)


# ------------------------------------------------------------- frozen parts --

@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_frozen_parts(dev, dtype):
    """Whichever inputs want gradients, theirs are the same bits, and what no gradient
    needs is not kept."""
    M, K, N = 100, 72, 136
    make = [((M, K), 1.0), ((N, K), 0.1), ((N,), 1.0), ((M, N), 1.0)]
    dy = seeded((M, N), 9, dtype).to(dev)
    for act in (None, "gelu_tanh"):
        full = None
        for mask in range(15, 0, -1):
            ts = [seeded(s, i, dtype, c).to(dev).requires_grad_(bool(mask >> i & 1))
                  for i, (s, c) in enumerate(make)]
            y = _linear(ts[0], ts[1], ts[2], act, ts[3])
            saved = [t for t in y.grad_fn.saved_tensors if t is not None and t.numel()]
            assert len(saved) == bool(mask & 2) + bool(mask & 1) + (
                (1 if dtype == torch.float32 else 2) if act and mask & 7 else 0)
            got = _grads(y, [t for t in ts if t.requires_grad], dy)
            if full is None:
                full = got
            want = [g for i, g in enumerate(full) if mask >> i & 1]
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    H, I, O = 72, 104, 40  # noqa: E741
    make = [((M, H), 1.0), ((I, H), 0.1), ((I, H), 0.1), ((O, I), 0.1), ((M, O), 1.0)]
    dy, full = seeded((M, O), 9, dtype).to(dev), None
    for mask in range(31, 0, -1):
        ts = [seeded(s, i, dtype, c).to(dev).requires_grad_(bool(mask >> i & 1))
              for i, (s, c) in enumerate(make)]
        got = _grads(_mlp(*ts), [t for t in ts if t.requires_grad], dy)
        if full is None:
            full = got
        want = [g for i, g in enumerate(full) if mask >> i & 1]
        for a, b in zip(got, want):  # (fewer weights' gradients: their K may be split otherwise)
            assert torch.equal(a, b)


def test_what_is_kept(dev):
    """Bytes between forward and backward: 16 or 8 bits an element of z, gate and up, and
    a scale for 32 columns."""
    M, K, N = 128, 64, 256
    x, w = _leaf((M, K), 1, dev), _leaf((N, K), 2, dev)

    def kept(y, weights):
        total = sum(t.numel() * t.element_size() for t in y.grad_fn.saved_tensors)
        return total - sum(t.numel() * 2 for t in weights)

    for held, size in ((None, 2), ("fp8", 1)):
        assert kept(_linear(x, w, activation="silu", checkpoint=held), (x, w)) == M * N * size + M * N // 32
        ws = [_leaf(s, 3, dev) for s in ((N, K), (N, K), (K, N))]
        assert kept(_mlp(x, *ws, checkpoint=held), (x, *ws)) == 2 * (M * N * size + M * N // 32)
    assert kept(_linear(x, w), (x, w)) == 0
    g, u = _leaf((M, N), 4, dev), _leaf((M, N), 5, dev)
    assert kept(_swiglu(g, u, checkpoint="fp8"), ()) == 2 * (M * N + M * N // 32)


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_what_a_frozen_block_keeps(dev, dtype):
    """x is kept for the gradients of gate's and up's weights alone, these weights for x's."""
    M, H, I, O = 100, 72, 104, 40  # noqa: E741
    make = [((M, H), 1.0), ((I, H), 0.1), ((I, H), 0.1), ((O, I), 0.1), ((M, O), 1.0)]
    for mask in range(1, 32):
        ts = [seeded(s, i, dtype, c).to(dev).requires_grad_(bool(mask >> i & 1))
              for i, (s, c) in enumerate(make)]
        y = _mlp(*ts)
        saved = {t.data_ptr() for t in y.grad_fn.saved_tensors if t is not None}
        for t, needed in zip(ts, (mask & 6, mask & 1, mask & 1, True, False)):
            assert (t.data_ptr() in saved) == bool(needed)


def test_c_entry_of_weights_that_lie_differently(dev):
    """fp32 weights of which one is 16-byte aligned and one is not: their products run on
    different kernels, which may split K differently."""
    from metal_liger_amd import _hip
    M, H, I, O = 200, 2048, 264, 64  # noqa: E741
    x, wd = seeded((M, H), 1).to(dev), seeded((O, I), 4, scale=0.1).to(dev)
    wg = seeded((I, H), 2, scale=0.1).to(dev)
    wu = torch.empty(I * H + 1, device=dev)[1:].view(I, H).copy_(seeded((I, H), 3, scale=0.1))
    n = _hip.query("ml_swiglu_mlp_fwd_workspace_bytes", M, H, I, O, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    for a, b in ((wg, wu), (wu, wg)):
        y = torch.empty(M, O, device=dev)
        _hip.call("ml_swiglu_mlp_fwd", x.data_ptr(), H, a.data_ptr(), H, b.data_ptr(), H,
                  wd.data_ptr(), I, None, 0, y.data_ptr(), 0, None, None, None, None, M, H, I, O,
                  ws.data_ptr(), n, 0, torch.cuda.current_stream().cuda_stream)
        g, u, d = (t.double().cpu() for t in (a, b, wd))
        want = (F.silu(x.double().cpu() @ g.t()) * (x.double().cpu() @ u.t())) @ d.t()
        # (2048 roundings of a sum of 2048 products, and fewer after them)
        assert rel_fro(y, want) < 2048 * 2**-24


def test_repeatable(dev):
    """The same bits at every call (no sum depends on the order of workgroups)."""
    x, w, b = _leaf((3000, 264), 1, dev), _leaf((1160, 264), 2, dev), _leaf((1160,), 3, dev)
    ws = [_leaf(s, 4, dev, scale=0.1) for s in ((520, 264), (520, 264), (264, 520))]
    dy, dz = seeded((3000, 1160), 5, BF).to(dev), seeded((3000, 264), 6, BF).to(dev)

    def run():
        y, z = _linear(x, w, b, "gelu", checkpoint="fp8"), _mlp(x, *ws)
        return [y, *_grads(y, [x, w, b], dy), z, *_grads(z, [x, *ws], dz)]

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_rows_do_not_mix(dev):
    """Non-finite rows, and rows of another size: the others' results are the same bits."""
    M, H, I = 200, 128, 264  # noqa: E741
    ws = [seeded(s, 1, BF, 0.1).to(dev).requires_grad_() for s in ((I, H), (I, H), (H, I))]
    base = seeded((M, H), 2, BF).to(dev)
    dy = seeded((M, H), 3, BF).to(dev)
    bad = torch.zeros(M, dtype=torch.bool, device=dev)
    bad[::7] = True
    other = base.clone()
    other[bad] = torch.tensor([float("nan"), float("inf"), 1e30, -float("inf")], device=dev,
                              dtype=BF).repeat(H // 4)
    for held in (None, "fp8"):
        for op in (lambda x: _mlp(x, *ws, checkpoint=held),
                   lambda x: _linear(x, ws[0], activation="gelu", checkpoint=held) @ ws[2].t(),
                   lambda x: _swiglu(x, x * 2, checkpoint=held)):
            got = []
            for t in (base, other):
                x = t.clone().requires_grad_()
                y = op(x)
                got.append((y, _grads(y, [x], dy)[0]))
            for a, b in zip(*got):
                assert torch.equal(a[~bad], b[~bad])
            assert not torch.isfinite(got[1][0][bad]).all()
            assert not torch.isfinite(got[1][1][bad]).all()


# ---------------------------------------------------------- several in a step --

def _step(p, x, held):
    """A gated block and a vision MLP of the fused operators, each with its residual, and
    an activation."""
    h = _mlp(x, p["g"], p["u"], p["d"], residual=x, checkpoint=held)
    z = _linear(h, p["w1"], p["b1"], "gelu_tanh", checkpoint=held)
    h = _linear(z, p["w2"], p["b2"], residual=h)
    return _swiglu(h, x, checkpoint=held)


def _plain_step(p, x):
    h = x + F.linear(F.silu(F.linear(x, p["g"])) * F.linear(x, p["u"]), p["d"])
    z = F.gelu(F.linear(h, p["w1"], p["b1"]), approximate="tanh")
    h = h + F.linear(z, p["w2"], p["b2"])
    return F.silu(h) * x


def _params(dev, dtype=BF, H=128, I=264, V=520):  # noqa: E741
    shapes = {"g": (I, H), "u": (I, H), "d": (H, I), "w1": (V, H), "b1": (V,), "w2": (H, V), "b2": (H,)}
    return {k: seeded(s, 10 + i, dtype, s[-1] ** -0.5).to(dev).requires_grad_()
            for i, (k, s) in enumerate(shapes.items())}


@pytest.mark.parametrize("tokens", [1, 37, 300, 2100])
@pytest.mark.parametrize("held", [None, "fp8"])
def test_together(dev, tokens, held):
    p = _params(dev)
    x = seeded((tokens, 128), 1, BF).to(dev).requires_grad_()
    dy = seeded((tokens, 128), 2, BF).to(dev)
    names = ["x", *p]
    leaves = [x, *p.values()]
    y = _step(p, x, held)
    got = dict(zip(["y", *names], [y, *_grads(y, leaves, dy)]))
    y = _plain_step(p, x)
    plain = dict(zip(["y", *names], [y, *_grads(y, leaves, dy)]))
    exact_leaves = [t.detach().double().requires_grad_() for t in leaves]
    y = _plain_step(dict(zip(p, exact_leaves[1:])), exact_leaves[0])
    exact = dict(zip(["y", *names], [y, *_grads(y, exact_leaves, dy.double())]))
    for k, want in exact.items():
        bound = 1.5 * rel_fro(plain[k], want) + 2e-3
        if held and k != "y":
            # e4m3 is off by at most 2^-4 of each kept value; a gradient reads up to three
            # kept tensors, and its relative error stays below their sum
            bound += 3 * 2.0 ** -4
        assert rel_fro(got[k], want) <= bound, (k, rel_fro(got[k], want), bound)


def test_gradients_against_differences(dev):
    """fp32 gradients along random directions against central differences of the oracle's
    forward in 64 bits (their error: below 1e-8 of the value here; fp32's: 1e-4)."""
    torch.manual_seed(0)
    x, w, b = (torch.randn(s, dtype=torch.float64) for s in ((33, 40), (24, 40), (24,)))
    wg, wu, wd = (torch.randn(s, dtype=torch.float64) * 0.2 for s in ((56, 40), (56, 40), (24, 56)))
    dy = torch.randn(33, 24, dtype=torch.float64)

    def f_linear(x, w, b):
        return (ref.act(x @ w.t() + b, "gelu") * dy).sum()

    def f_mlp(x, wg, wu, wd):
        return (((ref.act(x @ wg.t(), "silu") * (x @ wu.t())) @ wd.t()) * dy).sum()

    cases = [(f_linear, (x, w, b), lambda t: _linear(*t, activation="gelu")),
             (f_mlp, (x, wg, wu, wd), lambda t: _mlp(*t))]
    for f, args, op in cases:
        ts = [t.float().to(dev).requires_grad_() for t in args]
        args = [t.detach().double().cpu() for t in ts]
        grads = _grads(op(ts), ts, dy.float().to(dev))
        for i, g in enumerate(grads):
            d = torch.randn_like(args[i])
            e = 1e-5
            hi = f(*[a + e * d if j == i else a for j, a in enumerate(args)])
            lo = f(*[a - e * d if j == i else a for j, a in enumerate(args)])
            want = (hi - lo) / (2 * e)
            terms = (g.double().cpu() * d).abs().sum()
            assert abs((g.double().cpu() * d).sum() - want) <= 1e-5 * terms


# ------------------------------------------------- captured, streams, compiled --

@pytest.mark.parametrize("tokens", [1, 40, 700])
@pytest.mark.parametrize("held", [None, "fp8"])
def test_captured_step(dev, tokens, held):
    """A captured training step, replayed with the program's own work in between, new
    inputs each time: the eager step's bits."""
    p = _params(dev)
    x = seeded((tokens, 128), 1, BF).to(dev).requires_grad_()
    dy = seeded((tokens, 128), 2, BF).to(dev)
    leaves = [x, *p.values()]

    def step():
        y = _step(p, x, held)
        return [y, *_grads(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(seeded((tokens, 128), 20 + i, BF))
            p["w1"].add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in outs]
        # the program's own eager work, on the same values
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float32, BF, torch.float16])
def test_captured_padded_step(dev, dtype):
    """Sizes that are no multiples of 8: the padding belongs to the graph."""
    x, w, b = (_leaf(s, i, dev, dtype) for i, s in enumerate(((70, 61), (75, 61), (75,))))
    ws = [_leaf(s, 5, dev, dtype, 0.1) for s in ((45, 75), (45, 75), (61, 45))]
    dy, leaves = seeded((70, 61), 6, dtype).to(dev), [x, w, b, *ws]

    def step():
        y = _mlp(_linear(x, w, b, "gelu", checkpoint="fp8"), *ws, residual=x)
        return [y, *_grads(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(seeded((70, 61), 20 + i, dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i
        torch.cuda.synchronize()


def test_two_threads(dev):
    """Calls of two threads at once, each on a stream of its own: a call's bits alone."""
    from concurrent.futures import ThreadPoolExecutor
    sizes = [(300, 264, 136), (33, 61, 75)]
    cases = [[seeded(s, i, BF).to(dev) for i, s in enumerate(((M, K), (N, K), (N,), (M, N)))]
             for M, K, N in sizes]
    want = [_linear(c[0], c[1], c[2], "gelu", c[3]) for c in cases]
    torch.cuda.synchronize()

    def run(j):
        stream, same = torch.cuda.Stream(), True
        with torch.cuda.stream(stream):
            for _ in range(20):
                c = cases[j]
                same &= torch.equal(_linear(c[0], c[1], c[2], "gelu", c[3]), want[j])
        return same

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(run, (0, 1)))


def test_two_captured_graphs(dev):
    """Two graphs of the same shapes, replayed in turn and on two streams at once: each
    has workspaces of its own."""
    p = _params(dev)
    xs = [seeded((500, 128), i, BF).to(dev) for i in (1, 2)]

    def forward(x):
        with torch.no_grad():
            return _step(p, x, None)

    want = [forward(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        forward(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(forward(x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_another_stream(dev):
    p = _params(dev)
    x, dy = seeded((700, 128), 1, BF).to(dev).requires_grad_(), seeded((700, 128), 2, BF).to(dev)
    y = _step(p, x, "fp8")
    want = [y, *_grads(y, [x, *p.values()], dy)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = _step(p, x, "fp8")
        got = [y, *_grads(y, [x, *p.values()], dy)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("held", [None, "fp8"])
def test_compile(dev, held):
    import torch._dynamo
    torch._dynamo.reset()
    p = _params(dev)
    x, dy = seeded((300, 128), 1, BF).to(dev).requires_grad_(), seeded((300, 128), 2, BF).to(dev)
    leaves = [x, *p.values()]
    names = list(p)

    def step(x, *ts):
        return _step(dict(zip(names, ts)), x, held)

    y = step(*leaves)
    want = [y, *_grads(y, leaves, dy)]
    y = torch.compile(step, fullgraph=True, backend="aot_eager")(*leaves)
    got = [y, *_grads(y, leaves, dy)]
    for a, b in zip(got, want):  # the same kernels run; sums of gradients in another order
        assert torch.equal(a, b) or (a - b).abs().max() <= 2.0 ** -6 * b.abs().max()
    with torch.no_grad():
        assert torch.equal(torch.compile(step, fullgraph=True, backend="aot_eager")(*leaves), want[0])


def test_opcheck(dev):
    from metal_liger_amd import hip_ops
    ops = torch.ops.metal_liger_amd
    x, w, b, r = (seeded(s, i, BF).to(dev) for i, s in enumerate(((70, 64), (72, 64), (72,), (70, 72))))
    check = lambda op, args: torch.library.opcheck(op.default, args, test_utils=CHECKS)  # noqa: E731
    check(ops.linear_infer, (x, w, b, r, 1))
    for keep in (hip_ops.KEEP_NONE, hip_ops.KEEP_FP16, hip_ops.KEEP_FP8):
        check(ops.linear_fwd, (x, w, b, None, 2, keep))
    z = ops.linear_fwd(x, w, b, None, 2, hip_ops.KEEP_FP8)[1:]
    check(ops.linear_bwd, (x, w, r, 2, hip_ops.KEEP_FP8, *z, 72, 64, True, True, True))
    check(ops.linear_bwd, (None, w, r, 0, 0, None, None, 72, 64, True, False, True))
    ws = [seeded(s, 5, BF, 0.1).to(dev) for s in ((104, 64), (104, 64), (72, 104))]
    check(ops.swiglu_mlp_infer, (x, *ws, r))
    check(ops.swiglu_mlp_fwd, (x, *ws, None, hip_ops.KEEP_FP16))
    kept = ops.swiglu_mlp_fwd(x, *ws, r, hip_ops.KEEP_FP8)[1:]
    check(ops.swiglu_mlp_bwd, (x, *ws, r, hip_ops.KEEP_FP8, *kept, True, True, False, True))
    odd = (x[:, :61], w[:70, :61], b[:70], None, 2, hip_ops.KEEP_FP8)
    check(ops.linear_fwd, odd)
    z = ops.linear_fwd(*odd)[1:]
    check(ops.linear_bwd, (*odd[:2], r[:, :70], 2, hip_ops.KEEP_FP8, *z, 70, 61, True, True, True))
    check(ops.swiglu_mlp_bwd, (None, *ws, r, hip_ops.KEEP_FP8, *kept, True, False, False, True))
    check(ops.swiglu_mlp_bwd, (None, None, None, ws[2], r, hip_ops.KEEP_FP8, *kept, False, False, False, True))
    out = ops.swiglu_kept_fwd(x, x)
    check(ops.swiglu_kept_fwd, (x, x))
    check(ops.swiglu_kept_bwd, (*out[1:], x, BF, BF))
    check(ops.held_values, (out[1], out[2], torch.float32))


def test_first_derivatives_only(dev):
    x, w, r = _leaf((8, 64), 1, dev), _leaf((64, 64), 2, dev), _leaf((8, 64), 3, dev)
    for y in (_linear(x, w, activation="silu"), _mlp(x, w, w, w), _swiglu(x, r, checkpoint="fp8")):
        with pytest.raises(RuntimeError):
            g = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)[0]
            torch.autograd.grad(g.float().sum(), x)


def test_refusals(dev):
    x, w = torch.ones(2, 8, device=dev), torch.ones(4, 8, device=dev)
    with pytest.raises(ValueError, match="ROCm GPU"):
        _linear(x, w.cpu())
    with pytest.raises(ValueError, match="ROCm GPU"):
        _linear(x, w, residual=torch.ones(2, 4))
    with pytest.raises(TypeError, match="weight of"):
        _mlp(x, w.bfloat16(), w.bfloat16(), w.t())


# ------------------------------------------------------------- large tensors --

def test_past_32_bits(dev):
    """More than 2^31 elements: the last rows are those of a call on them alone."""
    rows, cols = 33000, 65568
    gate = torch.empty(rows, cols, dtype=BF, device=dev).normal_()
    up = torch.empty_like(gate).normal_().requires_grad_()
    gate.requires_grad_()
    y = _swiglu(gate, up, checkpoint="fp8")
    dy = torch.empty_like(y).normal_()
    dg, du = _grads(y, [gate, up], dy)
    at = torch.tensor([0, 7, 32767, rows - 2, rows - 1], device=dev)
    g, u = (t.detach()[at].requires_grad_() for t in (gate, up))
    small = _swiglu(g, u, checkpoint="fp8")
    assert torch.equal(small, y.detach()[at])
    for a, b in zip(_grads(small, [g, u], dy[at]), (dg, du)):
        assert torch.equal(a, b[at])


def test_linear_past_32_bits(dev):
    M, K, N = 66000, 64, 32776
    x = torch.empty(M, K, dtype=BF, device=dev).normal_().requires_grad_()
    w = (torch.empty(N, K, dtype=BF, device=dev).normal_() * 0.1).requires_grad_()
    at = torch.tensor([0, 5, 32768, M - 2, M - 1], device=dev)
    y = _linear(x, w, activation="silu")
    dy = torch.empty_like(y).normal_()
    dx, = _grads(y, [x], dy)
    xs, W = x.detach()[at].double(), w.detach().double()
    z = xs @ W.t()
    s = torch.sigmoid(z)
    want_y, want_dx = z * s, (dy[at].double() * s * (1 + z * (1 - s))) @ W
    assert rel_fro(y[at], want_y) <= 4e-3 and rel_fro(dx[at], want_dx) <= 4e-3


# ------------------------------------------------------------------- LoRA --

@pytest.mark.parametrize("dtype,ranks", [(BF, (16, 16, 16)), (BF, (8, 4, 24)), (torch.float32, (8, 8, 8)),
                                         (torch.float16, (4, 4, 4))])
def test_lora_mlp_kept_in_8_bits(dev, dtype, ranks):
    """The LoRA block whose gate and up are kept in 8 bits: its output is the block's, its
    gradients are those at the values that the 8 bits stand for."""
    from metal_liger_amd.ops import fused_lora as fl
    from metal_liger_amd import _custom_ops as cops
    N, H, I = 150, 128, 264  # noqa: E741
    params = []
    for i, ((o, n), r) in enumerate(zip(((I, H), (I, H), (H, I)), ranks)):
        params += [seeded((o, n), 3 * i, dtype, 0.1).to(dev), _leaf((r, n), 3 * i + 1, dev, dtype, 0.2),
                   _leaf((o, r), 3 * i + 2, dev, dtype, 0.1), 2.0]
    x, dy = _leaf((N, H), 30, dev, dtype), seeded((N, H), 31, dtype).to(dev)
    leaves = [x] + [t for t in params if isinstance(t, torch.Tensor) and t.requires_grad]
    y0 = fl._LoRA_MLP.apply(x, *params)
    y1 = fl._LoRA_MLP.apply(x, *params, "fp8")
    assert torch.equal(y0, y1)
    plain, saved = list(y0.grad_fn.saved_tensors), y1.grad_fn.saved_tensors
    held = []
    for t, q, s in ((plain[0], *saved[:2]), (plain[1], *saved[2:4])):
        codes, scales = ref.held_bytes(t.double().cpu())
        assert torch.equal(codes, q.cpu()) and torch.equal(scales, s.cpu())
        v = cops.held_values(q, s, t.dtype)
        assert torch.equal(v.double().cpu(), ref.held_values(q.cpu(), s.cpu()))
        held.append(v)
    got = _grads(y1, leaves, dy)
    # the whole block's backward on its own saved tensors, gate and up (in fp32 h too,
    # which is kept there) at those values
    plain[:2] = held
    if dtype != BF:
        plain[2] = cops.swiglu_fwd(*held)
    node, ctx = y0.grad_fn, types.SimpleNamespace(saved_tensors=tuple(plain))
    for name in ("held", "fp32", "n_kept", "scales", "orig_shape", "x_dtype", "param_dtypes", "ranks",
                 "rank_p"):
        if hasattr(node, name):
            setattr(ctx, name, getattr(node, name))
    with torch.no_grad():
        want = [t for t in fl._LoRA_MLP.backward(ctx, dy) if t is not None]
    for a, b in zip(got, want):
        assert torch.equal(a, b.to(a.dtype))


# ------------------------------------------------------------------- models --

def _train(model, ids):
    model.train()
    model.zero_grad(set_to_none=True)
    out = model(input_ids=ids, labels=ids)
    out.loss.backward()
    return out.loss.detach().float(), {n: p.grad.detach().float().clone()
                                       for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("held", [None, "fp8"])
def test_patched_model_full_training(dev, held):
    """All parameters of a model without adapters trained one step, the MLPs routed."""
    from metal_liger_amd import apply_metal_liger_to_qwen3vl
    attn = qwen_tiny.register_fp32_attention()
    base = qwen_tiny.build(seed=5, lora=False, attn=attn, dtype=BF).to(dev)
    exact = copy.deepcopy(base).float()
    patched = apply_metal_liger_to_qwen3vl(copy.deepcopy(base), fuse_mlp=True, mlp_checkpoint=held)
    ids = torch.randint(0, 512, (2, 96), generator=torch.Generator().manual_seed(7)).to(dev)
    (l_ex, g_ex), (l_bf, g_bf), (l_pt, g_pt) = (_train(m, ids) for m in (exact, base, patched))
    assert set(g_pt) == set(g_ex)
    assert abs(l_pt - l_ex) <= 1.5 * abs(l_bf - l_ex) + 2e-3 * abs(l_ex)
    for n in g_ex:
        bound = 1.5 * rel_fro(g_bf[n], g_ex[n]) + 2e-3 + (3 * 2.0 ** -4 if held else 0.0)
        assert rel_fro(g_pt[n], g_ex[n]) <= bound, n
    with torch.autocast("cuda", dtype=BF):  # the modules' own forwards
        fp32 = apply_metal_liger_to_qwen3vl(copy.deepcopy(exact), fuse_mlp=True)
        own = apply_metal_liger_to_qwen3vl(copy.deepcopy(exact))
        assert torch.equal(fp32(input_ids=ids).logits, own(input_ids=ids).logits)
    patched.eval()
    with torch.no_grad():  # single tokens through the cache
        out = patched.base_model.model.generate(ids[:1, :8], max_new_tokens=4, do_sample=False)
    assert out.shape == (1, 12)


@pytest.mark.parametrize("held", [None, "fp8"])
def test_patched_vision_tower(dev, held):
    from metal_liger_amd import apply_metal_liger_to_qwen3vl
    from metal_liger_amd.ops.fused_linear import _FusedVisionBlockForward
    base = qwen_tiny.build_vl(seed=3, dtype=BF).to(dev)
    exact = copy.deepcopy(base).float()
    patched = apply_metal_liger_to_qwen3vl(copy.deepcopy(base), fuse_vision_mlp=True,
                                           mlp_checkpoint=held)
    towers = [m.model.visual.blocks[0] for m in (exact, base, patched)]
    assert type(towers[2].forward) is _FusedVisionBlockForward
    x = seeded((80, 64), 1, BF).to(dev)
    cu = torch.tensor([0, 32, 80], device=dev, dtype=torch.int32)
    angles = torch.randn(80, 32, generator=torch.Generator().manual_seed(2)).to(dev)
    dy = seeded((80, 64), 4, BF).to(dev)
    outs = []
    for t in towers:
        dtype = t.mlp.linear_fc1.weight.dtype
        emb = (angles.cos().to(dtype), angles.sin().to(dtype))
        xi = x.to(dtype).requires_grad_()
        y = t(xi, cu_seqlens=cu, position_embeddings=emb)
        params = dict(t.mlp.named_parameters())
        outs.append(dict(zip(["y", "x", *params], [y, *_grads(y, [xi, *params.values()], dy.to(dtype))])))
    for k, want in outs[0].items():
        bound = 1.5 * rel_fro(outs[1][k], want) + 2e-3 + (3 * 2.0 ** -4 if held and k != "y" else 0)
        assert rel_fro(outs[2][k], want) <= bound, k


def test_modules(dev):
    from metal_liger_amd import MetalLigerLinear, MetalLigerSwiGLUMLP
    lin = nn.Linear(64, 40).to(dev, BF)
    m = MetalLigerLinear(lin, "gelu")
    assert list(m.state_dict()) == ["weight", "bias"] and m.weight is lin.weight
    x, r = seeded((9, 64), 1, BF).to(dev), seeded((9, 40), 2, BF).to(dev)
    with torch.no_grad():
        assert rel_fro(m(x), F.gelu(lin.float()(x.float()))) <= 4e-3
        lin.bfloat16()
        assert rel_fro(m(x, r), F.gelu(F.linear(x.float(), lin.weight.float(), lin.bias.float()))
                       + r.float()) <= 4e-3
    tiny = qwen_tiny.build(lora=False, dtype=BF).to(dev).base_model.model.model.layers[0].mlp
    m = MetalLigerSwiGLUMLP(tiny, "fp8")
    assert list(m.state_dict()) == ["gate_proj.weight", "up_proj.weight", "down_proj.weight"]
    x = seeded((2, 30, 128), 3, BF).to(dev).requires_grad_()
    y = m(x, x)
    want = x.float() + copy.deepcopy(tiny).float()(x.float())
    assert rel_fro(y, want) <= 6e-3
    y.sum().backward()
    assert m.gate_proj.weight.grad is not None and x.grad.shape == x.shape
