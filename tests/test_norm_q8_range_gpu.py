"""Rows of the int8 norm whose sum of squares passes fp32's range say so."""
import numpy as np
import pytest

from test_norm_q8_gpu import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0, 1])                # both kernels
@pytest.mark.parametrize("group", [0, 64])
def test_large_rows_have_nan_scales(group, offset):
    x = np.ones((4, 256), np.float32)
    x[1, 7] = 3e19                                        # its square passes 3.4e38
    x[2] = 2e18                                           # 256 of 4e36 do
    x[3] = 1e17
    _, s, _ = run(x, None, np.ones(256, np.float32), group, offset=offset)
    assert np.isnan(s[1:3]).all() and np.isfinite(s[[0, 3]]).all()
    assert np.abs(s[3] * 127 - 1).max() < 1e-5
