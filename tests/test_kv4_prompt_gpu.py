"""Prompt-sized attention over the 4-bit cache (256 rows and more): ragged batches, cut items, long contexts, holes, graphs."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
import x100b
from test_kv4_gpu import DT, cache_of, dev, ints, page_table, status

pytestmark = pytest.mark.gpu


def poison(pool, table, lens):
    """Bytes past each length: codes 15 and scales NaN."""
    page = pool.page
    for b, n in enumerate(lens):
        for p in range(n, table.shape[1] * page):
            if table[b, p // page] >= 0:
                t, s = pool.raw[table[b, p // page], :, p % page // 16], p % 16
                for i in range(pool.NB):
                    for is_v in (False, True):
                        at = pool._scale(is_v, s, i)
                        t[:, at:at + 2] = 0xFF


def check(pool, table, lens, q_lens, heads, kind, rows=None, max_q=None, seed=0, wide=False):
    """attend() against the statement at `rows` of every sequence (all of them by default)."""
    rng = np.random.default_rng(seed)
    D = pool.D
    starts = np.concatenate([[0], np.cumsum(q_lens)])
    q = rng.normal(size=(starts[-1] + 2, heads, D)).astype(np.float32 if kind == "f32" else np.float16)
    qd = dev(q)
    if wide:                                              # heads of a wider row
        big = torch.randn(q.shape[0], heads + 3, D, device="cuda").to(DT[kind])
        big[:, 1:1 + heads] = qd
        qd = big[:, 1:1 + heads]
    out = torch.full((q.shape[0], heads + (2 if wide else 0), D), 7.0, dtype=DT[kind], device="cuda")
    cache_of(pool).attend(qd, out[:, :heads], ints(table), ints(lens), q_start=ints(starts), max_q=max_q or max(q_lens))
    assert status() == 0
    got = out.cpu().numpy()
    assert (got[starts[-1]:] == 7).all() and (got[:, heads:] == 7).all()
    for b, n in enumerate(lens):
        if q_lens[b] == 0:
            continue
        k, v = pool.values(table[b], n, False), pool.values(table[b], n, True)
        for i in range(q_lens[b]) if rows is None else sorted({r % q_lens[b] for r in rows}):
            at = starts[b] + i
            want = ref.attention(q[at:at + 1], k, v, n - q_lens[b] + i, D ** -0.5)
            bound = ref.prompt_bound(q[at:at + 1], k, v, D ** -0.5, n, kind == "f16") + (2.0 ** -11 * np.abs(want).max() if kind == "f16" else 0)
            err = np.abs(got[at:at + 1, :heads].astype(np.float64) - want).max()
            assert err <= bound, (b, i, n, err, bound)
            if n - q_lens[b] + i < 0:
                assert not got[at, :heads].any()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D,heads,kv,page", [(128, 8, 2, 16), (64, 14, 2, 64), (128, 3, 1, 128), (64, 5, 5, 32)])
def test_ragged_prompts(kind, D, heads, kv, page):
    """More than 32 sequences: of no tokens, of no positions, of fewer positions than tokens, whole tiles and ends inside one."""
    q_lens = [0, 1, 128, 0, 33, 300, 7, 64, 0, 256] + [1, 0, 5] * 9
    lens = [50, 1, 128, 0, 20, 700, 1000, 65, 0, 511] + [129, 3, 0] * 9
    rng = np.random.default_rng(D + heads)
    n_pages = sum(-(-n // page) for n in lens) + 2
    pool = ref.random_pool(rng, n_pages, page, kv, D)
    table = page_table(rng, lens, page, n_pages)
    poison(pool, table, lens)
    check(pool, table, lens, q_lens, heads, kind, rows=[0, 1, 15, 31, 100, 127, -1], max_q=400, wide=True)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D,heads,kv,T,n", [(128, 8, 1, 64, 9000), (64, 16, 2, 130, 5000), (128, 16, 4, 1000, 1400)])
def test_items_cut_by_runs(kind, D, heads, kv, T, n):
    """Few items of many key tiles: every item is several CTAs' work."""
    rng = np.random.default_rng(n)
    page = 64
    pool = ref.random_pool(rng, -(-n // page), page, kv, D)
    check(pool, page_table(rng, [n], page, pool.raw.shape[0]), [n], [T], heads, kind, rows=[0, 1, T // 2, -1])


@pytest.mark.parametrize("T,heads,kv,n", [(64, 40, 5, 70000), (320, 64, 8, 18000)])
def test_long_fp32_prompts(T, heads, kv, n):
    """Runs of many key tiles: parts of an item, and whole items."""
    rng = np.random.default_rng(n)
    page = 128
    pool = ref.random_pool(rng, 8, page, kv, 128)
    table = rng.integers(0, 8, (1, -(-n // page))).astype(np.int32)       # the same few pages over and over
    check(pool, table, [n], [T], heads, "f32", rows=[0, 17, -1])


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_equal_values_stay_equal(kind):
    """Every v is 1 (code 0, scale -1/8): so is every output, to what the sums lose.  Each of `steps` tensor-core additions drops
    less than 2^-23 of the sum; the denominator is fp32 additions of 128 at a time.  fp16: p's rounding 2^-11 and the output's."""
    kv, D, page, n = 2, 128, 128, 131072
    cache = x100b.Kv4Cache(4, page, kv, D)
    pos = ints(np.arange(4 * page))
    table = ints(np.arange(4)[None])
    cache.append(torch.randn(4 * page, kv, D, device="cuda"), torch.ones(4 * page, kv, D, device="cuda"), pos, table, seq=torch.zeros_like(pos))
    # the prompt kernel, then one token of 64 sequences; fp32 q: 16 or 2 steps a tile, then fp32 additions of the tiles
    for T, steps in ((64, 16 + n / 256), (1, 2 + n / 256)) if kind == "f32" else ((64, n / 16 + 8), (1, n / 128 + 2)):
        B = 1 if T > 1 else 64
        q = torch.randn(64, 8 * kv * (4 if T > 1 else 1), D, device="cuda").to(DT[kind])
        big = ints(np.tile(np.arange(4), (B, n // page // 4)))
        out = cache.attend(q, None, big, ints([n] * B), q_start=ints([0, 64]) if T > 1 else None, max_q=T)
        assert status() == 0
        err = (out.double() - 1).abs().max().item()
        # denominators: 1024 tiles' fp32 additions, each half an ulp
        bound = steps * 2.0 ** -23 + (n / 128 + 330) * 2.0 ** -24
        if kind == "f16":
            bound += 2 * 2.0 ** -11 + n * 2.0 ** -25
        assert err <= bound, (T, err, bound)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_holes_in_the_table(kind):
    """Pages out of range inside and at the ends of key tiles are masked, with one status."""
    rng = np.random.default_rng(21)
    page, D, n, T = 16, 128, 700, 80
    pool = ref.random_pool(rng, 50, page, 1, D)
    table = page_table(rng, [n], page, 50)
    bad = {0: -1, 9: 50, 15: 1 << 30, 16: -5, 43: 99}
    keep = np.ones(n, bool)
    holed = table.copy()
    for i, p in bad.items():
        holed[0, i] = p
        keep[i * page:(i + 1) * page] = False
    q = rng.normal(size=(T, 8, D)).astype(np.float32 if kind == "f32" else np.float16)
    got = cache_of(pool).attend(dev(q), None, ints(holed), ints([n]), q_start=ints([0, T]), max_q=T).cpu().numpy()
    assert status() == x100b.X100_E_ARG
    k, v = pool.values(table[0], n, False), pool.values(table[0], n, True)
    for i in (0, 11, 50, 79):
        sees = keep & (np.arange(n) <= n - T + i)
        want = ref.attention(q[i:i + 1], k[sees], v[sees], sees.sum() - 1, D ** -0.5)
        bound = ref.prompt_bound(q[i:i + 1], k, v, D ** -0.5, n, kind == "f16") + (2.0 ** -11 * np.abs(want).max() if kind == "f16" else 0)
        assert np.abs(got[i:i + 1].astype(np.float64) - want).max() <= bound


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_prompts_repeat_and_replay(kind):
    rng = np.random.default_rng(22)
    lens, q_lens = [2500, 300, 77], [200, 300, 1]
    pool = ref.random_pool(rng, 60, 64, 2, 128)
    cache, table, n = cache_of(pool), ints(page_table(rng, lens, 64, 60)), ints(lens)
    starts = ints(np.concatenate([[0], np.cumsum(q_lens)]))
    q = torch.randn(sum(q_lens), 16, 128, device="cuda").to(DT[kind])
    work = cache.attend_work(q.shape[0], 16, 3)
    first = cache.attend(q, None, table, n, q_start=starts, max_q=300, work=work)
    work.fill_(0xFF)                                      # what the scratch holds does not matter
    out = torch.zeros_like(first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(q, out, table, n, q_start=starts, max_q=300, work=work)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
        out.zero_()
    n.copy_(ints([1, 0, 78]))                             # lengths and starts are read when the graph runs
    starts.copy_(ints([0, 1, 1, 260]))
    out.fill_(3.0)
    g.replay()
    again = cache.attend(q, torch.full_like(out, 3.0), table, n, q_start=starts, max_q=300)
    assert status() == 0 and torch.equal(out, again) and (out[260:] == 3).all() and not (out[:260] == 3).any()


def test_bad_starts_of_prompts_are_reported():
    rng = np.random.default_rng(23)
    pool = ref.random_pool(rng, 4, 64, 1, 64)
    cache, table = cache_of(pool), ints([[0, 1], [2, 3]])
    q = torch.randn(300, 4, 64, device="cuda")
    for lens, starts, max_q in (([128, 5], [0, 200, 100], 300), ([128, 5], [0, 301, 302], 300), ([128, 5], [-1, 20, 300], 300), ([129, 5], [0, 64, 128], 64),
                                ([-4, 100], [0, 100, 200], 100), ([1 << 30, 100], [0, 100, 200], 100)):
        out = torch.full_like(q, 9.0)
        cache.attend(q, out, table, ints(lens), q_start=ints(starts), max_q=max_q)
        assert status() == x100b.X100_E_ARG and torch.isfinite(out).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_single_tokens_of_large_groups(kind):
    """300 query heads of one kv head are a prompt's rows, without q_start."""
    rng = np.random.default_rng(31)
    lens, D, G = [5, 400, 0, 129], 64, 300
    pool = ref.random_pool(rng, 30, 32, 1, D)
    table = page_table(rng, lens, 32, 30)
    q = rng.normal(size=(4, G, D)).astype(np.float32 if kind == "f32" else np.float16)
    got = cache_of(pool).attend(dev(q), None, ints(table), ints(lens)).cpu().numpy()
    assert status() == 0
    for b, n in enumerate(lens):
        k, v = pool.values(table[b], n, False), pool.values(table[b], n, True)
        want = ref.attention(q[b:b + 1], k, v, n - 1, D ** -0.5)
        bound = ref.prompt_bound(q[b:b + 1], k, v, D ** -0.5, n, kind == "f16") + (2.0 ** -11 * np.abs(want).max() if kind == "f16" else 0)
        assert np.abs(got[b:b + 1].astype(np.float64) - want).max() <= bound


def test_another_stream():
    """A call on a stream that is not the current one takes its outputs and scratch from the caller."""
    rng = np.random.default_rng(32)
    pool = ref.random_pool(rng, 10, 64, 2, 128)
    cache, table, n = cache_of(pool), ints(page_table(rng, [600], 64, 10)), ints([600])
    q, side = torch.randn(1, 8, 128, device="cuda"), torch.cuda.Stream()
    want, pos, seq = cache.attend(q, None, table, n), ints([599]), ints([0])
    kv = torch.randn(1, 2, 128, device="cuda")
    for call in (lambda: cache.attend(q, None, table, n, stream=side), lambda: cache.attend(q, torch.empty_like(q), table, n, stream=side),
                 lambda: cache.read(pos, table, seq=seq, stream=side), lambda: cache.append(kv, kv, pos, table, seq=seq, q=q, stream=side)):
        with pytest.raises(x100b.X100Error) as e:
            call()
        assert e.value.code == x100b.X100_E_ARG
    out, work = torch.empty_like(q), cache.attend_work(1, 8, 1)
    side.wait_stream(torch.cuda.current_stream())
    cache.attend(q, out, table, n, work=work, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and status() == 0


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("q_lens,width", [([1, 1, 1], None), ([1, 1, 1], 5000), ([40, 1, 500], None)])
def test_in_place(kind, q_lens, width):
    """out is q: clusters, runs with cut items, prompts."""
    rng = np.random.default_rng(len(q_lens))
    lens = [3000, 50, 900]
    pool = ref.random_pool(rng, 70, 64, 1, 128)
    table = page_table(rng, lens, 64, 70)
    if width:
        table = np.concatenate([table, np.full((3, width), -1, np.int32)], 1)
    cache, table, n = cache_of(pool), ints(table), ints(lens)
    starts = ints(np.concatenate([[0], np.cumsum(q_lens)]))
    q = torch.randn(sum(q_lens), 8, 128, device="cuda").to(DT[kind])
    want = cache.attend(q, None, table, n, q_start=starts, max_q=max(q_lens))
    assert torch.equal(cache.attend(q, q, table, n, q_start=starts, max_q=max(q_lens)), want) and status() == 0
