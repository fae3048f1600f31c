"""The feed-forward operators at sizes that take their large tiles and splits, with
remainders at every edge (test_feed_forward_plans.py says which, without a GPU), against 64
bits within test_gpu_feed_forward.py's bounds."""

import pytest
import torch

from tests import test_feed_forward_plans as plans
from tests.test_gpu_feed_forward import (_linear_case, _linear_check, _mlp_case, _mlp_check,
                                         test_linear_few_rows as _check_without_gradients)

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("size", [plans.LINEAR_256, *plans.LINEAR_SPLIT])
def test_linear(dev, size, checkpoint):
    from metal_liger_amd.ops.fused_linear import fused_linear
    x, w, b, r, dy = _linear_case(*size, BF, True, True, dev)
    _linear_check(x, w, b, r, dy, "gelu", checkpoint,
                  lambda: fused_linear(x, w, b, "gelu", r, checkpoint))


@pytest.mark.parametrize("size", [plans.LINEAR_256, *plans.LINEAR_SPLIT])
def test_linear_without_an_activation(dev, size):
    from metal_liger_amd.ops.fused_linear import fused_linear
    x, w, b, r, dy = _linear_case(*size, BF, True, True, dev)
    _linear_check(x, w, b, r, dy, None, None, lambda: fused_linear(x, w, b, None, r))


@pytest.mark.parametrize("checkpoint", [None, "fp8"])
@pytest.mark.parametrize("size", [*plans.MLP_256, *plans.MLP_SPLIT])
def test_gated_block(dev, size, checkpoint):
    from metal_liger_amd.ops.fused_swiglu_mlp import fused_swiglu_mlp
    x, ws, r, dy = _mlp_case(*size, BF, True, dev)
    _mlp_check(x, ws, r, dy, checkpoint, lambda: fused_swiglu_mlp(x, *ws, r, checkpoint))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("size", [plans.F32_FORWARD, plans.F32_DX, plans.F32_DW])
def test_fp32(dev, dtype, size):
    from metal_liger_amd.ops.fused_linear import fused_linear
    for act in ("silu", None):
        x, w, b, r, dy = _linear_case(*size, dtype, True, act is None, dev)
        _linear_check(x, w, b, r, dy, act, None, lambda: fused_linear(x, w, b, act, r))
    _check_without_gradients(dev, dtype, *size)
