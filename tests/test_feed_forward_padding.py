"""What the entry points for padded operands refuse on the host (no pointer is read)."""

import pytest

from metal_liger_amd import _hip


@pytest.mark.parametrize("data", [0, -1, 65, 1 << 40])
def test_columns_that_are_not_padding(data):
    L, p, q = _hip.lib(), 4096, 8192
    rcs = [lambda: L.ml_linear_fwd_padded(p, 64, p, 64, None, None, 0, 0, q, 64, 0, None, None, 100, 64,
                                          64, data, p, 1 << 40, 1, None),
           lambda: L.ml_swiglu_mlp_fwd_padded(p, 64, p, 64, p, 64, p, 64, None, 0, q, 0, *(None,) * 4,
                                              100, 64, 64, 64, data, p, 1 << 40, 1, None),
           lambda: L.ml_swiglu_mlp_bwd_padded(p, 64, p, 64, p, 64, p, 64, p, 64, 3, *(p,) * 4, q, q, q, q,
                                              100, 64, 64, 64, data, p, 1 << 40, 1, None)]
    for rc in rcs:
        assert rc() == 1 and b"of 64 columns are not padding" in L.ml_last_error()
