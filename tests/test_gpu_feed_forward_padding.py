"""Infinities through sizes that the feed-forward operators pad: what is zero beside the
operands adds nothing, whatever is in them. (An infinity times a padded zero is NaN, which
no result may read.) Where a formula gives a number or an infinity, so does the kernel."""

import pytest
import torch

from tests.parity import seeded
from tests.test_gpu_feed_forward import DTYPES, V, _check, _cpu

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(autouse=True)
def _pad_fp32_too(monkeypatch):
    from metal_liger_amd import hip_ops
    monkeypatch.setattr(hip_ops, "PAD_F32", 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(5, 13, 7), (40, 72, 333), (200, 331, 1001), (3000, 72, 3763)])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh"])
def test_linear(dev, dtype, M, K, N, act):
    """z is infinite in whole rows of x, act'(z) there 1 or 0: dx is dy W or 0."""
    from metal_liger_amd.ops.fused_linear import fused_linear
    x, w = seeded((M, K), 1, dtype), seeded((N, K), 2, dtype, K ** -0.5)
    x[1, 2], x[3, 2] = INF, -INF
    w[:, 2] = w[:, 2].abs() + 0.125
    b, dy = seeded((N,), 3, dtype), seeded((M, N), 4, dtype)
    x, w, b, dy = (t.to(dev).requires_grad_() for t in (x, w, b, dy))
    y = fused_linear(x, w, b, act)
    dx, db = torch.autograd.grad(y, [x, b], dy.detach())
    assert bool((y[1] == INF).all())
    D, W = _cpu(dy), _cpu(w)
    _check(dx[1], D[1] @ W, (N + 2) * V * (D[1].abs() @ W.abs()), "dx where z is inf")
    assert bool((dx[3] == 0).all())
    assert bool(dx.isfinite().all()) and bool(db.isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,H,I,O", [(5, 13, 7, 9), (40, 72, 333, 64), (200, 64, 1001, 65),
                                     (2100, 72, 1003, 40)])
@pytest.mark.parametrize("checkpoint", [None, "fp8"])
def test_gated_block(dev, dtype, M, H, I, O, checkpoint):  # noqa: E741
    """Positive operands: an infinite x gives a row of infinities, an infinite dy one of
    dx."""
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    x, *ws = (seeded(s, i, dtype, s[1] ** -0.5).abs() + 2.0 ** -10
              for i, s in enumerate([(M, H), (I, H), (I, H), (O, I)]))
    x, *ws = (t.to(dev).requires_grad_() for t in (x, *ws))
    y = fused_swiglu_mlp(x, *ws, checkpoint=checkpoint)
    dy = torch.full_like(y, 2.0 ** -6)
    dy[2, 1] = INF
    grads = torch.autograd.grad(y, [x, *ws], dy)
    assert bool(y.isfinite().all())
    inf = torch.zeros(M, dtype=torch.bool, device=dev)
    inf[2] = True
    assert bool((grads[0][inf] == INF).all()) and bool(grads[0][~inf].isfinite().all())
    assert bool((grads[1] == INF).all()) and bool((grads[2] == INF).all())
    assert bool((grads[3][1] == INF).all()) and bool(grads[3][[0, 2]].isfinite().all())
    bad = x.detach().clone()
    bad[1, 3] = INF
    for t in (bad, bad.clone().requires_grad_()):  # (with and without gate and up kept)
        out = fused_swiglu_mlp(t, *ws, checkpoint=checkpoint)
        assert bool((out[1] == INF).all())
        rest = torch.arange(M, device=dev) != 1
        assert torch.equal(out[rest], y[rest])
    with torch.no_grad():
        out = fused_swiglu_mlp(bad, *ws)
    assert bool((out[1] == INF).all()) and bool(out[2:].isfinite().all())
