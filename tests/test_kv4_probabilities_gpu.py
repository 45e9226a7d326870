"""Attention over the 4-bit cache where one position dominates the row: the small probabilities under it count."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
import x100b
from test_kv4_gpu import DT, cache_of, dev, ints, page_table, status

pytestmark = pytest.mark.gpu


def tail_bound(z, v, n, kind):
    """Largest error of rows of scores z (nats, [rows, n]) over values v >= 0 ([n]) in float64, and the rows' outputs.

    A probability relative to the row's largest, p, is held to 2^-36 of the largest (fp16's subnormal step 2^-24, half of it, under
    the factor 2^11) or, where that is more, to 2^-11 (fp16) or 2^-21 (both halves, and exp2) of itself; a score's own error is
    added to it: 40 fp32 steps of its largest product sum, which is the score here (one sign).  The tensor core's sums truncate,
    2^-23 of the sum for each of its additions: fp16 q n / 16 for prompts and no more for few rows; fp32 q 16 a tile and an fp32
    addition for each of n / 128.  The denominator is fp32 additions, n / 128 and 330 for the joins; both count with the output."""
    top = z.max(-1, keepdims=True)
    p = np.where(np.isfinite(z), np.exp(z - top), 0.0)
    total = p.sum(-1)
    out = p @ v / total
    score = 2 * 40 * 2.0 ** -24 * np.abs(top[:, 0])
    rel = 2.0 ** -11 if kind == "f16" else 2.0 ** -21
    held = np.maximum(rel * p, np.where(p > 0, 2.0 ** -36, 0.0)) @ v / total
    sums = n / 16 + 8 if kind == "f16" else 16 + n / 128
    bound = held + out * (score + sums * 2.0 ** -23 + (n / 128 + 330) * 2.0 ** -24)
    if kind == "f16":
        bound += np.maximum(out * 2.0 ** -11, 2.0 ** -25)
    return bound, out


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("T", [1, 3, 32, 300])
@pytest.mark.parametrize("n", [2600, 131072])
@pytest.mark.parametrize("nats,spread", [(16.85, 0.0), (24.0, 0.0), (17.0, 1.0), (12.0, 1.0), (5.0, 0.0)])
def test_a_tail_under_one_position(kind, T, n, nats, spread):
    """One position `nats` above the others (flat, or spread normally), its v zero and theirs one."""
    D, page, G, sink = 128, 64, 8, 5
    rng = np.random.default_rng(n + T)
    cache = x100b.Kv4Cache(-(-n // page), page, 1, D)
    score = spread * rng.normal(size=n)
    score[sink] = nats
    # every element of a key is one value and every q element 1 / 8: a score is D^-0.5 * D / 8 times it
    k = torch.from_numpy((score / (D ** 0.5 / 8)).astype(np.float32)).cuda()[:, None, None].expand(n, 1, D).contiguous()
    v = torch.ones(n, 1, D, device="cuda")
    v[sink] = 0
    pos, table = ints(np.arange(n)), ints(np.arange(-(-n // page))[None])
    seq = torch.zeros_like(pos)
    cache.append(k, v, pos, table, seq=seq)
    kb, vb = (t[:, 0, 0].double().cpu().numpy() for t in cache.read(pos, table, seq=seq))
    assert (np.delete(vb, sink) == 1).all() and vb[sink] == 0
    q = torch.full((T, G, D), 0.125, device="cuda", dtype=DT[kind])
    out = cache.attend(q, None, table, ints([n]), q_start=ints([0, T]), max_q=T).double().cpu().numpy()
    assert status() == 0 and (out == out[:, :1, :1]).all()
    rows = sorted({0, T // 2, T - 1})
    z = np.where(np.arange(n)[None] <= n - T + np.array(rows)[:, None], (D ** 0.5 / 8) * kb[None], -np.inf)
    bound, want = tail_bound(z, vb, n, kind)
    err = np.abs(out[rows, 0, 0] - want)
    assert (err <= bound).all(), (err / want, bound / want)


@pytest.mark.parametrize("D,page,kv,G,T", [(128, 64, 2, 8, 1), (64, 16, 2, 5, 1), (128, 32, 1, 7, 3), (64, 64, 2, 8, 4), (128, 64, 1, 8, 4), (64, 32, 1, 31, 1)])
def test_few_fp16_rows_are_off_by_the_outputs_rounding(D, page, kv, G, T):
    """Under 256 rows fp16 q is as near as fp32 q before the output is rounded: wherever that settles the rounding, it is the right one.

    Before it, as ref.attention_bound has it for fp32 q, row by row: the score's errors with A the row's own largest scale * sum |q k|, twice
    (numerator and sum), exp2 and the halves of p; then sums over n / 16 steps of a warp and the joins of 8 warps and n / 128 + 2 runs."""
    rng = np.random.default_rng(D + G)
    lens = [2, 5, 16, 33]
    pool = ref.random_pool(rng, sum(-(-n // page) for n in lens), page, kv, D)
    table = page_table(rng, lens, page, pool.raw.shape[0])
    q = rng.normal(size=(4 * T, kv * G, D)).astype(np.float16)
    checked = []
    for t in (table, np.concatenate([table, np.full((4, 6000), -1, np.int32)], 1)):          # clusters, and runs with a merge
        got = cache_of(pool).attend(dev(q), None, ints(t), ints(lens), q_start=ints(np.arange(5) * T), max_q=T).cpu().numpy()
        assert status() == 0
        for i, n in enumerate(lens):
            rows = slice(i * T, i * T + T)
            k, v = pool.values(table[i], n, False), pool.values(table[i], n, True)
            want = ref.attention(q[rows], k, v, n - T, D ** -0.5)
            size = np.abs(q[rows].astype(np.float64)).reshape(T, kv, G, D)
            A = D ** -0.5 * np.einsum("tkgd,nkd->tkgn", size, np.abs(k)).max(-1).reshape(T, kv * G, 1)
            rel = 2 * (A * (2.0 ** -22 + (D / 8 + D / 32 + 1) * 2.0 ** -23) + 2.0 ** -21) + (n / 16 + 2) * 2.0 ** -23 + (n / 128 + 10) * 2.0 ** -24
            off = rel * np.abs(v).max()
            near = want.astype(np.float16)
            step = np.spacing(np.abs(near)).astype(np.float64)
            sure = step / 2 - np.abs(want - near) > off          # so far from a tie that the rounding is known
            checked.append(sure.mean())
            assert np.array_equal(got[rows][sure], near[sure]), (n, (got[rows][sure] != near[sure]).mean())
    assert max(checked) > 0.25                                   # the bound settles enough of them to tell


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("T", [1, 3, 64])
@pytest.mark.parametrize("n", [300, 1024, 5000])
def test_large_common_scores_cancel(kind, T, n):
    """Scores of 163840 + 0 .. 60 in steps of 1/4, all exact sums in fp32: the softmax is that of the small part.

    What is left of a probability's error is the rounding of its exponent, which lies in -60 .. 15 (2^-19 of a power of two), exp2's
    and the halves' 2^-21 (fp16 prompts 2^-11), the scale's 2^-24 on the small part (8 powers of two), and the sums: n / 16 + 16 steps
    of 2^-23 (of 16 positions or fewer additions) and joins of 8 warps and n / 128 + 2 runs; numerator and sum carry it."""
    D, page, G = 128, 32, 8
    rng = np.random.default_rng(n + T)
    small = rng.integers(0, 241, n) / 4
    k = np.zeros((n, 1, D), np.float32)
    k[:, 0, :32], k[:, 0, 32:64] = 5120, small[:, None]
    v = rng.choice([-1.0, 1.0], (n, 1, D)).astype(np.float32)
    cache, pos, table = x100b.Kv4Cache(-(-n // page), page, 1, D), ints(np.arange(n)), ints(np.arange(-(-n // page))[None])
    seq = torch.zeros_like(pos)
    cache.append(dev(k), dev(v), pos, table, seq=seq)
    kb, vb = (t.double().cpu().numpy() for t in cache.read(pos, table, seq=seq))
    assert np.array_equal(kb, k)                          # 240 has 8 significant bits
    q = np.zeros((T, G, D), np.float32 if kind == "f32" else np.float16)
    q[..., :32], q[..., 32:64] = 1, 1 / 32
    out = cache.attend(dev(q), None, table, ints([n]), q_start=ints([0, T]), max_q=T).cpu().numpy()
    assert status() == 0
    rel = 2 * (2.0 ** -19 + (2.0 ** -11 if kind == "f16" and T * G >= 256 else 2.0 ** -21) + 8 * 2.0 ** -24) + (n / 16 + 16) * 2.0 ** -23 + (n / 128 + 10) * 2.0 ** -24
    for i in range(T):
        sees = n - T + i + 1
        p = np.exp(D ** -0.5 * (small[:sees] - small[:sees].max()))
        want = p @ vb[:sees, 0] / p.sum()
        bound = rel * np.abs(vb).max() + (np.abs(want) * 2.0 ** -11 if kind == "f16" else 0)
        assert (np.abs(out[i].astype(np.float64) - want) <= bound).all(), (i, np.abs(out[i] - want).max(), rel)
