"""fp32 queries of any size with a scale that keeps the scores ordinary."""
import numpy as np
import pytest

import kv4_ref as ref
from test_kv4_gpu import cache_of, dev, ints, page_table, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 4, 64])
@pytest.mark.parametrize("D,size", [(128, 1e-3), (64, 3e-4), (128, 1e-6), (64, 1e-12), (128, 1.0), (128, 1e3), (64, 1e7), (128, 1e20)])
def test_small_and_large_queries(D, size, T):
    """q of about `size` with scale = head_dim^-0.5 / size: the scores, and so the bound, are those of q of about 1."""
    rng = np.random.default_rng(T + D)
    kv, G, page, lens = 2, 8, 32, [3, 200, 1500]
    pool = ref.random_pool(rng, sum(-(-n // page) for n in lens), page, kv, D)
    table = page_table(rng, lens, page, pool.raw.shape[0])
    q = (size * rng.normal(size=(3 * T, kv * G, D))).astype(np.float32)
    scale = D ** -0.5 / size
    got = cache_of(pool).attend(dev(q), None, ints(table), ints(lens), q_start=ints(np.arange(4) * T), max_q=T, scale=scale).cpu().numpy()
    assert status() == 0
    for i, n in enumerate(lens):
        rows = slice(i * T, i * T + T)
        k, v = pool.values(table[i], n, False), pool.values(table[i], n, True)
        want = ref.attention(q[rows], k, v, n - T, scale)
        bound = (ref.attention_bound if T * G < 256 else ref.prompt_bound)(q[rows], k, v, scale, n, False)
        # the power of two leaves q between 0.7 and 1.4 of the usual size: elements under 1/8 are known to 2^-25, which moves a score by
        # 2^-25 sum |k| / sqrt(D) at most, or, for 0.7, 1.4 times that; numerator and sum carry it
        bound += 2 * 1.5 * 2.0 ** -25 * np.abs(k).max(0).sum(-1).max() / D ** 0.5 * np.abs(v).max()
        err = np.abs(got[rows].astype(np.float64) - want).max()
        assert err <= bound, (n, err, bound)
