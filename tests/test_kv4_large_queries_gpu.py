"""Attention over the 4-bit cache with a few elements of q and k far larger than the rest."""
import numpy as np
import pytest

import kv4_ref as ref
from test_kv4_gpu import cache_of, dev, ints, page_table, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("T", [1, 4, 64])
@pytest.mark.parametrize("D,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("how", ["k zero there", "both large"])
def test_outlying_channels(kind, T, D, page, how):
    """Two channels of q of 50 to 20000 where every key is zero add nothing, however large; of 50 to 200 against keys as large they
    make large scores, whose errors go by their own size.  The bound is that of ordinary values: no product counts more than itself."""
    rng = np.random.default_rng(T + D)
    kv, G, lens = 2, 8, [2, 5, 700, 4000]
    n_pages = sum(-(-n // page) for n in lens)
    pool = ref.Pages(n_pages, page, kv, D)
    table = page_table(rng, lens, page, n_pages)
    a, b = 3, D - 30                                      # two dims of two blocks
    k, v = (rng.normal(size=(n_pages * page, kv, D)).astype(np.float32) for _ in range(2))
    k[..., [a, b]] = 0 if how == "k zero there" else np.float32([100, -70]) + rng.normal(size=(n_pages * page, kv, 2))
    raw = pool.raw.reshape(n_pages, kv, page // 16, 18 * D)
    for is_v, x in ((False, k), (True, v)):               # whole tiles at once, by the formula
        c, d = ref.quantise(x)
        c = c.reshape(n_pages, page // 16, 16, kv, D)
        d = ref.scale16(d).reshape(n_pages, page // 16, 16, kv, D // 32)
        nib = np.zeros((n_pages, kv, page // 16, 36 * D), np.uint8)
        for s in range(16):
            at = (pool._v_nibble if is_v else pool._k_nibble)(s, np.arange(D))
            nib[..., at] = c[:, :, s].transpose(0, 2, 1, 3)
            for j in range(D // 32):
                o = pool._scale(is_v, s, j)
                raw[..., o:o + 2] = np.ascontiguousarray(d[:, :, s, :, j].transpose(0, 2, 1))[..., None].view(np.uint8)
        packed = nib[..., 0::2] | nib[..., 1::2] << 4
        part = slice(8 * D, 16 * D) if is_v else slice(0, 8 * D)
        raw[..., part] = packed[..., part]
    for size in (50, 200) if how == "both large" else (50, 200, 20000):
        q = rng.normal(size=(4 * T, kv * G, D)).astype(np.float32)
        q[..., a], q[..., b] = size, -size
        q = q.astype(np.float32 if kind == "f32" else np.float16)
        got = cache_of(pool).attend(dev(q), None, ints(table), ints(lens), q_start=ints(np.arange(5) * T), max_q=T).cpu().numpy()
        assert status() == 0
        for i, n in enumerate(lens):
            rows = slice(i * T, i * T + T)
            kk, vv = pool.values(table[i], n, False), pool.values(table[i], n, True)
            want = ref.attention(q[rows], kk, vv, n - T, D ** -0.5)
            bound = (ref.attention_bound if T * G < 256 else ref.prompt_bound)(q[rows], kk, vv, D ** -0.5, n, kind == "f16")
            bound += 2.0 ** -11 * np.abs(vv).max() if kind == "f16" else 0
            err = np.abs(got[rows].astype(np.float64) - want).max()
            assert err <= bound, (size, n, err, bound)
