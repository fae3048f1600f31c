"""The feed-forward operators on the GPU against 64 bits on the CPU.

Bounds, elementwise, of the sizes that the inputs themselves give (u = eps / 2 of the
operators' type, v = 2^-24 of fp32):
  a product of K terms in fp32: K v |a| |b| (and one v for each term added after it);
  a value rounded to its type: u |value| (fp16 below its smallest normal number: 2^-25);
  fp16 with a scale that puts a row's largest magnitude at 2^14 or more: its smallest
  normal number lies 2^28 below that, half its smallest step 2^-25 - 14 of it;
  act at z + d: 1.13 |d| (the largest |act'|), act' at z + d: 0.8 |d| (the largest
  |act''|); the activations' own fp32 arithmetic: 32 v (|z| + 1) (exp, a reciprocal and
  at most ten more roundings, and an exponent's rounding error that grows with |z|).
A value that a formula multiplies carries its bound through it.
"""

import pytest
import torch

from oracle import feed_forward as ref
from tests.parity import seeded

pytestmark = pytest.mark.gpu
V = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "silu", "gelu", "gelu_tanh"]


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _matrix_cores(dtype, *sizes):
    """Whether the products read bf16 (else everything between input and output is fp32)."""
    return dtype == torch.bfloat16


def _cpu(t):
    return t.detach().double().cpu()


def _check(got, want, bound, what):
    """bound without the output's own rounding."""
    u = _u(got.dtype)
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    total = bound * (1 + u) + want.abs() * u + tiny + 1e-30
    err = (_cpu(got) - want).abs()
    assert got.shape == want.shape, what
    assert bool((err <= total).all()), (what, (err / total).max())


def _mm(a, ea, b, eb, K):
    """a b and its bound, of operands with bounds."""
    A, B = a.abs(), b.abs()
    return a @ b, ea @ (B + eb) + A @ eb + (K + 2) * V * (A @ B)


def _act_noise(z):
    return 32 * V * (z.abs() + 1)


def _kept(saved, i, checkpoint, cols):
    """The i-th kept tensor of an autograd node's saved ones, as its backward reads it
    (without the columns that pad it)."""
    v, s = saved[i:i + 2]
    if checkpoint is None and v.dtype == torch.float32:
        return _cpu(v)[:, :cols]
    return ref.held_values(v.cpu(), s.cpu())[:, :cols]


# ------------------------------------------------------------------- linear --

def _linear_case(M, K, N, dtype, bias, residual, dev, seed=0, scale=1.0):
    x = seeded((M, K), seed, dtype, scale).to(dev).requires_grad_()
    w = seeded((N, K), seed + 1, dtype, K ** -0.5).to(dev).requires_grad_()
    b = seeded((N,), seed + 2, dtype).to(dev).requires_grad_() if bias else None
    r = seeded((M, N), seed + 3, dtype).to(dev).requires_grad_() if residual else None
    dy = seeded((M, N), seed + 4, dtype).to(dev)
    return x, w, b, r, dy


def _linear_check(x, w, b, r, dy, act, checkpoint, call):
    M, K, N = x.shape[0], x.shape[1], w.shape[0]
    y = call()
    saved = y.grad_fn.saved_tensors
    leaves = [t for t in (x, w, b, r) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    dtype, low = x.dtype, _matrix_cores(x.dtype, K, N)
    X, W, D = _cpu(x), _cpu(w), _cpu(dy)
    zero = torch.zeros(())
    z, ez = _mm(X, torch.zeros_like(X), W.t(), torch.zeros_like(W.t()), K)
    if b is not None:
        z, ez = z + _cpu(b), ez + V * (z + _cpu(b)).abs()
    want = ref.act(z, act)
    bound = 1.13 * ez + (_act_noise(z) if act else zero)
    if r is not None:
        want = want + _cpu(r)
        bound = bound + V * want.abs()
    _check(y, want, bound, "y")
    # the backward, at z as it was kept
    if act is None:
        dz, edz = D, torch.zeros_like(D)
    else:
        zk = _kept(saved, 2, checkpoint, N)
        err = (zk - z).abs()
        if checkpoint == "fp8":
            e = torch.ldexp(torch.ones((), dtype=torch.float64), ref.held_exponents(z))
            e = e.repeat_interleave(32, -1)[..., :N]
            # half a step, a smallest step of half 2^-9, where z's own error may move the scale
            assert bool((err <= 2 * ez + z.abs() * 2.0 ** -4 + 2 * e * 2.0 ** -10).all()), "kept"
        else:
            assert bool((err <= ez + z.abs() * (V if dtype == torch.float32 else _u(torch.float16))
                        + 2.0 ** -38 * z.abs().max()).all()), "kept"
        d = ref.act_grad(zk, act)
        dz, edz = D * d, D.abs() * _act_noise(zk)
        edz = edz + dz.abs() * (_u(dtype) if low else 2 * V)
    out = [(*_mm(dz, edz, W, torch.zeros_like(W), N), "dx"),
           (*_mm(dz.t(), edz.t(), X, torch.zeros_like(X), M), "dw")]
    if b is not None:
        out.append((dz.sum(0), edz.sum(0) + (M + 2) * V * dz.abs().sum(0), "db"))
    if r is not None:
        assert torch.equal(grads[-1], dy)
    for g, (want, bound, what) in zip(grads, out):
        assert g.dtype == dtype
        _check(g, want, bound, what)


SIZES = [(1, 64, 64), (3, 72, 8), (37, 128, 96), (129, 264, 136), (300, 200, 520), (5, 13, 7),
         (64, 33, 65), (257, 100, 31), (1, 1, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("act", ACTS)
def test_linear(dev, dtype, size, act):
    from metal_liger_amd.ops.fused_linear import fused_linear
    M, K, N = size
    x, w, b, r, dy = _linear_case(M, K, N, dtype, (M + N) % 2 == 0, K % 2 == 0, dev)
    _linear_check(x, w, b, r, dy, act, None,
                  lambda: fused_linear(x, w, b, activation=act, residual=r))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("act", ACTS[1:])
def test_linear_kept_in_8_bits(dev, dtype, size, act):
    from metal_liger_amd.ops.fused_linear import fused_linear
    M, K, N = size
    x, w, b, r, dy = _linear_case(M, K, N, dtype, (M + N) % 2 == 1, K % 2 == 1, dev)
    _linear_check(x, w, b, r, dy, act, "fp8",
                  lambda: fused_linear(x, w, b, activation=act, residual=r, checkpoint="fp8"))


# ------------------------------------------------------------- gated block --

def _mlp_case(M, H, I, O, dtype, residual, dev, seed=0):  # noqa: E741
    x = seeded((M, H), seed, dtype).to(dev).requires_grad_()
    ws = [seeded(s, seed + 1 + i, dtype, s[1] ** -0.5).to(dev).requires_grad_()
          for i, s in enumerate([(I, H), (I, H), (O, I)])]
    r = seeded((M, O), seed + 5, dtype).to(dev).requires_grad_() if residual else None
    return x, ws, r, seeded((M, O), seed + 6, dtype).to(dev)


def _gated(g, eg, u, eu):
    """silu(g) u and its bound."""
    s = ref.act(g, "silu")
    es = 1.13 * eg + _act_noise(g)
    h = s * u
    return h, es * (u.abs() + eu) + s.abs() * eu + V * h.abs()


def _mlp_check(x, ws, r, dy, checkpoint, call):
    (M, H), (O, I) = x.shape, ws[2].shape  # noqa: E741
    y = call()
    saved = y.grad_fn.saved_tensors
    leaves = [x, *ws] + ([] if r is None else [r])
    grads = torch.autograd.grad(y, leaves, dy)
    low = _matrix_cores(x.dtype, H, I, O)
    u16 = _u(torch.bfloat16) if low else V  # what is rounded between the products
    X, (Wg, Wu, Wd), D = _cpu(x), map(_cpu, ws), _cpu(dy)
    zx = torch.zeros_like(X)
    g, eg = _mm(X, zx, Wg.t(), torch.zeros_like(Wg.t()), H)
    u, eu = _mm(X, zx, Wu.t(), torch.zeros_like(Wu.t()), H)
    h, eh = _gated(g, eg, u, eu)
    want, bound = _mm(h, eh + u16 * h.abs(), Wd.t(), torch.zeros_like(Wd.t()), I)
    if r is not None:
        want = want + _cpu(r)
        bound = bound + V * want.abs()
    _check(y, want, bound, "y")
    gk = _kept(saved, 4, checkpoint, I)
    uk = _kept(saved, 6, checkpoint, I)
    for k, z, e in ((gk, g, eg), (uk, u, eu)):
        if checkpoint == "fp8":
            s = torch.ldexp(torch.ones((), dtype=torch.float64), ref.held_exponents(z))
            s = s.repeat_interleave(32, -1)[..., :I]
            assert bool(((k - z).abs() <= 2 * e + z.abs() * 2.0 ** -4 + 2 * s * 2.0 ** -10).all())
        else:
            v = V if x.dtype == torch.float32 else _u(torch.float16)
            assert bool(((k - z).abs() <= e + v * z.abs()
                        + 2.0 ** -38 * z.abs().max()).all())
    zero = torch.zeros_like(gk)
    h, eh = _gated(gk, zero, uk, zero)
    dh, edh = _mm(D, torch.zeros_like(D), Wd, torch.zeros_like(Wd), O)
    d, s = ref.act_grad(gk, "silu"), ref.act(gk, "silu")
    noise = _act_noise(gk) + 3 * V
    dg, du = dh * uk * d, dh * s
    edg = (edh * d.abs() + dh.abs() * noise) * uk.abs() + u16 * dg.abs()
    edu = edh * s.abs() + dh.abs() * noise + u16 * du.abs()
    a, ea = _mm(dg, edg, Wg, torch.zeros_like(Wg), I)
    b, eb = _mm(du, edu, Wu, torch.zeros_like(Wu), I)
    eb = eb + I * V * (a.abs() + b.abs())  # one sum over both
    eh = eh + u16 * h.abs()
    out = [(a + b, ea + eb, "dx"), (*_mm(dg.t(), edg.t(), X, zx, M), "dwg"),
           (*_mm(du.t(), edu.t(), X, zx, M), "dwu"),
           (*_mm(D.t(), torch.zeros_like(D.t()), h, eh, M), "dwd")]
    if r is not None:
        assert torch.equal(grads[-1], dy)
    for t, (want, bound, what) in zip(grads, out):
        assert t.dtype == x.dtype
        _check(t, want, bound, what)


MLP_SIZES = [(1, 64, 64, 64), (3, 72, 104, 8), (37, 128, 96, 40), (129, 264, 136, 264),
             (300, 200, 520, 200), (5, 13, 7, 9), (65, 33, 70, 33), (1, 1, 1, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", MLP_SIZES)
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_mlp(dev, dtype, size, checkpoint):
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    M, H, I, O = size  # noqa: E741
    x, ws, r, dy = _mlp_case(M, H, I, O, dtype, M % 2 == 0 or H % 2 == 1, dev)
    _mlp_check(x, ws, r, dy, checkpoint,
               lambda: fused_swiglu_mlp(x, *ws, residual=r, checkpoint=checkpoint))


# -------------------------------------------------- SwiGLU kept in 8 bits --

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (31,), (32,), (33,), (4, 64), (3, 5, 40), (7, 333),
                                   (129, 96), (2, 8), (5, 0), (0, 8)])
def test_swiglu_kept(dev, dtype, shape):
    from metal_liger_amd.ops.fused_swiglu import fused_swiglu
    gate = seeded(shape, 1, dtype, 3.0).to(dev).requires_grad_()
    up = (seeded(shape, 2, dtype) * torch.exp(seeded(shape, 3)).to(dtype)).to(dev).requires_grad_()
    dy = seeded(shape, 4, dtype).to(dev)
    y = fused_swiglu(gate, up, checkpoint="fp8")
    assert torch.equal(y, fused_swiglu(gate.detach(), up.detach()))
    gq, gs, uq, us = y.grad_fn.saved_tensors
    if y.numel():
        for t, q, s in ((gate, gq, gs), (up, uq, us)):
            want = ref.held_bytes(_cpu(t))
            assert torch.equal(q.cpu(), want[0]) and torch.equal(s.cpu(), want[1])
    dg, du = torch.autograd.grad(y, [gate, up], dy)
    if not y.numel():
        assert dg.shape == du.shape == gate.shape
        return
    g, u, D = ref.held_values(gq.cpu(), gs.cpu()), ref.held_values(uq.cpu(), us.cpu()), _cpu(dy)
    noise = _act_noise(g) + 3 * V
    _check(dg, D * u * ref.act_grad(g, "silu"), (D * u).abs() * noise, "dgate")
    _check(du, D * ref.act(g, "silu"), D.abs() * noise, "dup")


@pytest.mark.parametrize("dtype", DTYPES)
def test_8_bits_of_every_value(dev, dtype):
    """Every bf16 or fp16 (a spread of fp32) magnitude as an element of a block whose
    largest one sets the scale, infinities, NaN and zeros among them."""
    from metal_liger_amd import hip_ops
    bits = torch.arange(0, 2 ** 16, dtype=torch.int32)
    v = (bits - 2 ** 15).to(torch.int16).view(torch.float16 if dtype == torch.float16
                                              else torch.bfloat16).to(dtype)
    if dtype == torch.float32:
        g = torch.Generator().manual_seed(3)
        v = torch.randint(-2 ** 31, 2 ** 31, (2 ** 16,), generator=g).to(torch.int32).view(dtype)
    scattered = v[torch.randperm(2 ** 16, generator=torch.Generator().manual_seed(1))]
    top = torch.where((torch.arange(2 ** 16) % 32 == 5) & (v.abs() < 300), v, v * 0.01).to(dtype)
    for t in (v.view(64, 1024), scattered.view(64, 1024), top.view(-1, 32), v[:65535].view(-1, 15)):
        out = hip_ops.swiglu_kept_fwd(t.to(dev), t.to(dev))
        codes, scales = ref.held_bytes(t)
        got, want = out[1].cpu(), codes
        nan = ~torch.isfinite(t)
        assert torch.equal(out[2].cpu(), scales)
        assert torch.equal(got[~nan], want[~nan])
        assert bool(((got[nan] & 0x7F) == 0x7F).all())
        assert torch.equal(out[3].cpu(), got) and torch.equal(out[4].cpu(), scales)


# ------------------------------------- every tile, K whole and split, at edges --
# (a 256 x 256 tile where there are enough of them, 128 x 128 below, K split where
# those do not fill the GPU either)

@pytest.mark.parametrize("size", [(1025, 72, 4104), (2048, 136, 2056), (4099, 264, 1160),
                                  (700, 520, 1000)])
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_linear_tiles(dev, size, checkpoint):
    from metal_liger_amd.ops.fused_linear import fused_linear
    x, w, b, r, dy = _linear_case(*size, torch.bfloat16, True, True, dev)
    _linear_check(x, w, b, r, dy, "gelu_tanh", checkpoint,
                  lambda: fused_linear(x, w, b, "gelu_tanh", r, checkpoint))


@pytest.mark.parametrize("size", [(1025, 72, 2056, 136), (2050, 136, 1160, 520), (520, 264, 1000, 264),
                                  (4100, 64, 1032, 64)])
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_mlp_tiles(dev, size, checkpoint):
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    x, ws, r, dy = _mlp_case(*size, torch.bfloat16, True, dev)
    _mlp_check(x, ws, r, dy, checkpoint,
               lambda: fused_swiglu_mlp(x, *ws, residual=r, checkpoint=checkpoint))


@pytest.mark.parametrize("tokens,hidden,inter,out", [(1100, 264, 520, 264), (4097, 72, 264, 136),
                                                     (1600, 1032, 4104, 520)])
@pytest.mark.parametrize("frozen", ["", "gate", "up", "down", "gate up", "gate down", "up down"])
def test_weight_gradients_together(dev, tokens, hidden, inter, out, frozen):
    """Weights' gradients of one launch, tiles of a partial round split over the tokens,
    whichever of them are wanted: the same as each alone, up to the sums' order."""
    from metal_liger_amd import hip_ops
    x, ws, _, dy = _mlp_case(tokens, hidden, inter, out, torch.bfloat16, False, dev)
    x, ws = x.detach(), [w.detach() for w in ws]
    y, *kept = hip_ops.swiglu_mlp_fwd(x, *ws, None, hip_ops.KEEP_FP16)
    need = [name not in frozen.split() for name in ("gate", "up", "down")]
    got = hip_ops.swiglu_mlp_bwd(x, *ws, dy, hip_ops.KEEP_FP16, *kept, False, *need)
    g = ref.held_values(kept[0].cpu(), kept[1].cpu())
    u = ref.held_values(kept[2].cpu(), kept[3].cpu())
    dh = _cpu(dy) @ _cpu(ws[2])
    X, D, U = _cpu(x), _cpu(dy), _u(torch.bfloat16)
    noise = _act_noise(g) + (out + 6) * V
    dg, du = dh * u * ref.act_grad(g, "silu"), dh * ref.act(g, "silu")
    h = ref.act(g, "silu") * u
    big = D.abs() @ _cpu(ws[2]).abs()  # dh's error: (out + 2) V of this
    want = [(dg, U * dg.abs() + 1.2 * noise * big * u.abs(), X),
            (du, U * du.abs() + noise * big * (g.abs() + 1), X), None]
    for i in range(2):
        if need[i]:
            a, ea, b = want[i]
            _check(got[1 + i], *_mm(a.t(), ea.t(), b, torch.zeros_like(b), tokens), f"weight {i}")
        else:
            assert got[1 + i].numel() == 0
    if need[2]:
        eh = U * h.abs() + noise * u.abs()
        _check(got[3], *_mm(D.t(), torch.zeros_like(D.t()), h, eh, tokens), "down")
    assert got[0].numel() == 0


# ------------------------------------------------- few rows, nothing to keep --

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65])
@pytest.mark.parametrize("K,N", [(8, 8), (72, 40), (512, 264), (2056, 16), (1000, 1000)])
def test_linear_few_rows(dev, dtype, M, K, N):
    from metal_liger_amd.ops.fused_linear import fused_linear
    x, w, b, r, _ = _linear_case(M, K, N, dtype, K != 72, N != 16, dev)
    with torch.no_grad():
        y = fused_linear(x, w, b, "silu", r)
    X, W = _cpu(x), _cpu(w)
    z, ez = _mm(X, torch.zeros_like(X), W.t(), torch.zeros_like(W.t()), K)
    if b is not None:
        z = z + _cpu(b)
        ez = ez + V * z.abs()
    want, bound = ref.act(z, "silu"), 1.13 * ez + _act_noise(z)
    if r is not None:
        want = want + _cpu(r)
        bound = bound + V * want.abs()
    assert y.dtype == dtype
    _check(y, want, bound, "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 16, 31, 64, 65])
@pytest.mark.parametrize("H,I,O", [(64, 8, 8), (264, 520, 72), (520, 1032, 1000), (33, 40, 50)])
def test_mlp_few_rows(dev, dtype, M, H, I, O):  # noqa: E741
    """Without gradients; h past fp16's range (gate weights of one sign and size)."""
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    x, ws, r, _ = _mlp_case(M, H, I, O, dtype, M != 16, dev)
    with torch.no_grad():
        ws[0].mul_(100.0)
        ws[1].mul_(2000.0)
        ws[2].mul_(1e-3)
        y = fused_swiglu_mlp(x, *ws, residual=r)
    X, (Wg, Wu, Wd) = _cpu(x), map(_cpu, ws)
    zx, low = torch.zeros_like(X), _matrix_cores(dtype, H, I, O)
    g, eg = _mm(X, zx, Wg.t(), torch.zeros_like(Wg.t()), H)
    u, eu = _mm(X, zx, Wu.t(), torch.zeros_like(Wu.t()), H)
    h, eh = _gated(g, eg, u, eu)
    assert h.abs().max() > 65504 or H * I < 4000
    want, bound = _mm(h, eh + (_u(dtype) if low else V) * h.abs(), Wd.t(), torch.zeros_like(Wd.t()), I)
    if r is not None:
        want = want + _cpu(r)
        bound = bound + V * want.abs()
    keep = want.abs() < 65000
    _check(torch.where(keep.to(dev), y, 0), torch.where(keep, want, 0.0), torch.where(keep, bound, 0.0), "y")


# (rows shared out over workgroups by one tile of 16 and by two to four, the last
# workgroup's not full; on both sides of where the tiles take over)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(40, 264, 2056), (72, 136, 5000), (100, 520, 264), (113, 264, 4104),
                                   (128, 72, 8200), (128, 1000, 512), (129, 264, 264)])
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_linear_shared_rows(dev, dtype, M, K, N, checkpoint):
    from metal_liger_amd.ops.fused_linear import fused_linear
    case = _linear_case(M, K, N, dtype, True, True, dev, seed=7)
    _linear_check(*case, "gelu_tanh", checkpoint,
                  lambda: fused_linear(*case[:3], "gelu_tanh", case[3], checkpoint))
    test_linear_few_rows(dev, dtype, M, K, N)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,H,I,O", [(33, 72, 2056, 264), (80, 264, 1032, 520), (97, 136, 4104, 72),
                                     (128, 264, 520, 1000)])
def test_mlp_shared_rows(dev, dtype, M, H, I, O):  # noqa: E741
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    for checkpoint in (None, "fp8"):
        case = _mlp_case(M, H, I, O, dtype, True, dev, seed=7)
        _mlp_check(*case, checkpoint, lambda: fused_swiglu_mlp(case[0], *case[1], case[2], checkpoint))
    test_mlp_few_rows(dev, dtype, M, H, I, O)


@pytest.mark.parametrize("M", [5, 200])
@pytest.mark.parametrize("N", [8, 40, 72, 136])
def test_scales_of_short_blocks(dev, M, N):
    """A bias that cancels most of the sums: the scales of a row's last, short block go by
    its own columns alone."""
    from metal_liger_amd import hip_ops
    K = 64
    x, w, b, _, _ = _linear_case(M, K, N, torch.bfloat16, True, False, dev)
    x, w = torch.ones_like(x), torch.ones_like(w)
    b = torch.full_like(b, -float(K)) + b.detach() * 2.0 ** -6
    for keep in (hip_ops.KEEP_FP16, hip_ops.KEEP_FP8):
        _, v, s = hip_ops.linear_fwd(x, w, b, None, 1, keep)
        z = K + _cpu(b).expand(M, N)  # exact in fp32
        e = ref.held_exponents(z) - (7 if keep == hip_ops.KEEP_FP16 else 0)
        assert torch.equal(s.cpu().long() - 127, e.clamp_min(-126))
        half = z.abs() * (2.0 ** -11 if keep == hip_ops.KEEP_FP16 else 2.0 ** -4) + 2.0 ** -30
        assert bool(((ref.held_values(v.cpu(), s.cpu()) - z).abs() <= half).all())


# fp32 and fp16: 128 x 128 and 64 x 64 tiles, K whole and split, sizes that pad
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("size", [(1025, 72, 2056), (300, 1000, 264), (70, 2056, 136), (2100, 64, 520),
                                  (1030, 1001, 1043), (129, 40, 8)])
def test_linear_fp32_tiles(dev, dtype, size):
    from metal_liger_amd.ops.fused_linear import fused_linear
    for act in ("silu", None):
        x, w, b, r, dy = _linear_case(*size, dtype, True, act is None, dev)
        _linear_check(x, w, b, r, dy, act, None, lambda: fused_linear(x, w, b, act, r))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("size", [(1025, 72, 2056, 136), (520, 264, 1000, 264), (70, 1000, 1501, 999),
                                  (1100, 999, 1001, 64)])
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_mlp_fp32_tiles(dev, dtype, size, checkpoint):
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    x, ws, r, dy = _mlp_case(*size, dtype, True, dev)
    _mlp_check(x, ws, r, dy, checkpoint,
               lambda: fused_swiglu_mlp(x, *ws, residual=r, checkpoint=checkpoint))


def test_wide_strides(dev):
    """Rows further apart than the kernels address."""
    from metal_liger_amd.ops.fused_linear import fused_linear
    wide = 5 * (1 << 20)
    w = seeded((40, 64), 1, torch.bfloat16).to(dev)
    big = torch.zeros(300, wide, dtype=torch.bfloat16, device=dev)
    x = big[:, 8:72]
    x.copy_(seeded((300, 64), 2, torch.bfloat16))
    assert torch.equal(fused_linear(x, w), fused_linear(x.contiguous(), w))
    big = torch.zeros(150, wide, device=dev)
    x = big[:, 8:72]
    x.copy_(seeded((150, 64), 2))
    assert torch.equal(fused_linear(x, w.float()), fused_linear(x.contiguous(), w.float()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shapes", [[(1, 1)], [(13,), (7, 9), (0, 5), (8, 16), (1,)],
                                    [(3000, 1001), (517, 8), (1, 70001), (70001, 1), (4, 7), (9,), (2, 2), (65, 31)]])
def test_padding(dev, dtype, shapes):
    """Copies of any sizes and strides, in one launch: the same bits, zeros beside them."""
    from metal_liger_amd import hip_ops
    ts = []
    for i, s in enumerate(shapes):
        t = seeded(s, i, dtype).to(dev)
        if i % 3 == 1 and t.dim() == 2:
            t = t.t().contiguous().t()                            # columns apart
        elif i % 3 == 2:
            t = torch.cat([t, t, t], -1)[..., s[-1]:2 * s[-1]]    # a slice of longer rows
        elif t.dim() == 2 and i:
            t = t[:1].expand(s)                                   # one row for all
        ts.append(t)
    wide = hip_ops._Wide(ts[0])
    sizes = [(1 if t.dim() == 1 else t.shape[0] + 5 * (i % 2), hip_ops.padded8(t.shape[-1]))
             for i, t in enumerate(ts)]
    ins = [wide.operand(t, *s) for t, s in zip(ts, sizes)]
    wide.begin()
    for t, s, i in zip(ts, sizes, ins):
        want = torch.zeros(s, dtype=dtype, device=dev)
        want[:t.shape[0] if t.dim() == 2 else 1, :t.shape[-1]] = t
        if not isinstance(i, int):
            assert torch.equal(i.view(s), want)
            continue
        at = wide.rooms[i][0]
        n = s[0] * s[1] * t.element_size()
        assert wide.at(i) == (wide.base + at, s[1])
        assert torch.equal(wide.buffer[at:at + n].view(dtype).view(s), want)
    # back: each room into a result of the matrix's size
    outs = [torch.full(t.shape, 7.0, dtype=dtype, device=dev) for t in ts]
    wide.outs = [(o, i) for o, i in zip(outs, ins) if isinstance(i, int)]
    wide.end()
    for t, o, i in zip(ts, outs, ins):
        assert torch.equal(o, t) or not isinstance(i, int)


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("M,K,N", [(5, 13, 7), (70, 33, 65), (300, 201, 521), (129, 264, 131), (129, 131, 264)])
def test_fp32_padded(dev, monkeypatch, checkpoint, M, K, N):
    """fp32 sizes padded as large ones are."""
    from metal_liger_amd import hip_ops
    from metal_liger_amd.ops.fused_linear import fused_linear
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    monkeypatch.setattr(hip_ops, "PAD_F32", 1)
    case = _linear_case(M, K, N, torch.float32, True, True, dev, seed=3)
    _linear_check(*case, "silu", checkpoint,
                  lambda: fused_linear(*case[:3], "silu", case[3], checkpoint))
    x, ws, r, dy = _mlp_case(M, K, N, K + 3, torch.float32, True, dev, seed=3)
    _mlp_check(x, ws, r, dy, checkpoint, lambda: fused_swiglu_mlp(x, *ws, r, checkpoint))
    for frozen in range(15):  # (the padding of what is left)
        for i, t in enumerate((x, *ws)):
            t.requires_grad_(not frozen >> i & 1)
        leaves = [t for t in (x, *ws) if t.requires_grad]
        got = torch.autograd.grad(fused_swiglu_mlp(x, *ws, r, checkpoint), leaves, dy)
        for g, t in zip(got, leaves):
            assert g.shape == t.shape and bool(g.isfinite().all())
        if frozen == 0:
            full = dict(zip(map(id, leaves), got))
        # (fewer gradients may split K otherwise)
        for g, t in zip(got, leaves):
            assert torch.allclose(g, full[id(t)], rtol=0, atol=N * M * V * float(full[id(t)].abs().max()))
