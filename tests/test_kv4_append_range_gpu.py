"""Heads whose sum of squares passes fp32's range are no zeros that nobody hears of."""
import pytest
import torch

import x100b
from test_kv4_gpu import ints, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_large_heads_are_reported(D):
    cache, pos, table, seq = x100b.Kv4Cache(1, 16, 1, D), ints([0, 1]), ints([[0]]), ints([0, 0])
    k = torch.ones(2, 1, D, device="cuda")
    q = torch.ones(2, 2, D, device="cuda")
    k[0, 0, 3], q[0, 1, 5] = 3e19, -3e19
    one = torch.ones(D, device="cuda")
    out = cache.append(k, k.clone().clamp(max=1), pos, table, seq=seq, q=q, q_norm=one, k_norm=one)
    assert status() == x100b.X100_E_ARG
    kb, vb = cache.read(pos, table, seq=seq)
    assert not kb[0].any() and (kb[1] - 1).abs().max() < 0.01 and (vb == 1).all()
    assert torch.isnan(out[0, 1]).all() and (out[0, 0] - 1).abs().max() < 1e-5 and (out[1] - 1).abs().max() < 1e-5
    # without a norm such a head is stored, and saturates
    cache.append(k, k, pos, table, seq=seq)
    assert status() == 0 and cache.read(pos, table, seq=seq)[0][0, 0, 3] == 65280
