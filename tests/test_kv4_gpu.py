"""4-bit paged KV cache on the GPU: append, read and attention against plain numpy statements (kv4_ref)."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
import x100b

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def ints(a):
    return dev(np.asarray(a, np.int32))


def page_table(rng, lens, page, n_pages, width=None):
    need = [-(-n // page) for n in lens]
    order = rng.permutation(n_pages)[: sum(need)]
    t = np.full((len(lens), max(need + [1]) if width is None else width), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def cache_of(pool):
    n_pages, kv = pool.raw.shape[:2]
    return x100b.Kv4Cache(n_pages, pool.page, kv, pool.D, pages=dev(pool.raw))


def status():
    """The status that the next synchronising call reports (0 or an X100_E code)."""
    try:
        x100b.sync()
        return 0
    except x100b.X100Error as e:
        return e.code


# ---- append and read --------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_append_writes_the_formulas_bytes(kind, D, page):
    """Without a head norm every byte of the pool is the formula's, and no other byte changes."""
    rng = np.random.default_rng(D + page)
    kv, heads, lens = 3, 6, [page + 5, 1, 2 * page]
    n_pages = 8
    table = page_table(rng, lens, page, n_pages)
    pos = np.concatenate([np.arange(max(0, n - 7), n) for n in lens])
    seq = np.repeat(np.arange(3), [min(7, n) for n in lens])
    order = rng.permutation(len(pos))
    pos, seq = pos[order], seq[order]
    np_t = np.float32 if kind == "f32" else np.float16
    k, v = (rng.normal(size=(len(pos), kv, D)).astype(np_t) for _ in range(2))
    q = rng.normal(size=(len(pos), heads, D)).astype(np_t)
    k[0, 0, :32] = 0                                    # a block of zeros
    v[0, 1, 32:64] = np_t(2.0 ** -24)                   # the smallest halves
    v[1, 0, :32] = np.where(np.arange(32) % 2, 1, -1)   # a tie of +1 and -1
    rope = rng.normal(size=(2 * page, D // 2, 2)).astype(np.float32)
    pool = ref.Pages(n_pages, page, kv, D, fill=0xA5)
    cache = cache_of(pool)
    kr = ref.rotate(k.astype(np.float32), rope, pos)
    for i in range(len(pos)):
        for h in range(kv):
            for is_v, x in ((False, kr[i, h]), (True, v[i, h].astype(np.float32))):
                c, d = ref.quantise(x)
                pool.put(table[seq[i], pos[i] // page], pos[i], h, is_v, c, ref.scale16(d))
    q_out = cache.append(dev(k), dev(v), ints(pos), ints(table), seq=ints(seq), q=dev(q), rope=dev(rope))
    assert status() == 0
    assert np.array_equal(cache.pages.cpu().numpy(), pool.raw)
    qr = ref.rotate(q.astype(np.float32), rope, pos)
    assert np.array_equal(q_out.cpu().numpy(), qr.astype(np_t))
    kb, vb = cache.read(ints(pos), ints(table), seq=ints(seq))
    for i in range(len(pos)):
        row = table[seq[i]]
        assert np.array_equal(kb[i].cpu().numpy(), pool.values(row, pos[i] + 1, False)[-1].astype(np.float16))
        assert np.array_equal(vb[i].cpu().numpy(), pool.values(row, pos[i] + 1, True)[-1].astype(np.float16))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_append_with_head_norms(kind, D):
    """Codes do not depend on the rounding of 1 / rms; a scale may move by one of its 2^-8 steps, q by fp32 rounding."""
    rng = np.random.default_rng(5)
    n, kv, heads, page = 37, 2, 5, 32
    np_t = np.float32 if kind == "f32" else np.float16
    k, v, q = (3 * rng.normal(size=(n, h, D)) for h in (kv, kv, heads))
    k, v, q = (x.astype(np_t) for x in (k, v, q))
    qw, kw = (1 + 0.3 * rng.normal(size=D).astype(np.float32) for _ in range(2))
    rope = x100b.rope_table(64, D, 1e6)
    table = page_table(rng, [n], page, 3)
    cache = x100b.Kv4Cache(3, page, kv, D)
    q_out = cache.append(dev(k), dev(v), ints(np.arange(n)), ints(table), seq=ints(np.zeros(n)), q=dev(q), q_norm=dev(qw), k_norm=dev(kw), eps=1e-5,
                         rope=rope)
    assert status() == 0
    rope = rope.cpu().numpy()
    pool = ref.Pages(3, page, kv, D)
    pool.raw[...] = cache.pages.cpu().numpy().reshape(pool.raw.shape)
    got = pool.values(table[0], n, False).reshape(n, kv, -1, 32)
    c, d = ref.quantise(ref.rotate((k.astype(np.float32) * kw).astype(np.float32), rope, np.arange(n)))
    rms = np.sqrt((k.astype(np.float64) ** 2).mean(-1) + 1e-5)
    d = d / rms[..., None]
    step = got / np.where(d == 0, 1, d)[..., None] - (c.reshape(got.shape).astype(np.float64) - 8)
    assert np.abs(step).max() <= 8 * 2.0 ** -8            # 8 = the largest |code - 8|; 2^-9 rounding and a possible step
    want = ref.rotate((q.astype(np.float32) * qw).astype(np.float32), rope, np.arange(n)) / np.sqrt((q.astype(np.float64) ** 2).mean(-1) + 1e-5)[..., None]
    err = np.abs(q_out.cpu().numpy().astype(np.float64) - want)
    # sum of D squares, root, quotient, product: under (5 + log2 D + 4) fp32 roundings; then the output's half step
    assert (err <= np.abs(want) * (20 * 2.0 ** -24 + (2.0 ** -11 if kind == "f16" else 0)) + 2.0 ** -24).all()


def test_rope_table_far_positions():
    t = x100b.rope_table(131072, 128, 1e6).cpu().numpy().astype(np.float64)
    p = np.array([0, 1, 4095, 100003, 131071])
    a = p[:, None] * 1e6 ** (-np.arange(0, 128, 2) / 128)
    # half a step of fp32 values up to 1, and the 64-bit angle's own rounding (131071 * 2^-52 and a few)
    assert np.abs(t[p, :, 0] - np.cos(a)).max() <= 2.0 ** -25 + 1e-9 and np.abs(t[p, :, 1] - np.sin(a)).max() <= 2.0 ** -25 + 1e-9


def test_append_strided_in_place_and_padding():
    """q, k and v as slices of one projection, q rotated in place, padding tokens left out."""
    rng = np.random.default_rng(6)
    D, kv, heads, n, page = 128, 2, 4, 9, 16
    qkv = rng.normal(size=(n, heads + 2 * kv + 1, D)).astype(np.float32)   # one head more than used: a pitch of its own
    pos = np.array([3, -1, 0, 31, -7, 4, 5, 6, 7])
    table = page_table(rng, [32], page, 2)
    rope = x100b.rope_table(32, D, 1e4)
    t = dev(qkv)
    cache = x100b.Kv4Cache(2, page, kv, D, pages=torch.full((2 * kv * 18 * D,), 0x5A, dtype=torch.uint8, device="cuda"))
    cache.append(t[:, heads:heads + kv], t[:, heads + kv:heads + 2 * kv], ints(pos), ints(table), seq=ints(np.zeros(n)), q=t[:, :heads],
                 q_out=t[:, :heads], rope=rope)
    assert status() == 0
    got = t.cpu().numpy()
    live = pos >= 0
    assert np.array_equal(got[:, heads:], qkv[:, heads:]) and np.array_equal(got[~live], qkv[~live])
    assert np.array_equal(got[live][:, :heads], ref.rotate(qkv[live][:, :heads], rope.cpu().numpy(), pos[live]))
    want = ref.Pages(2, page, kv, D, fill=0x5A)
    kr = ref.rotate(qkv[live][:, heads:heads + kv], rope.cpu().numpy(), pos[live])
    for i, p in enumerate(pos[live]):
        for h in range(kv):
            for is_v, x in ((False, kr[i, h]), (True, qkv[live][i, heads + kv + h])):
                c, d = ref.quantise(x)
                want.put(table[0, p // page], p, h, is_v, c, ref.scale16(d))
    assert np.array_equal(cache.pages.cpu().numpy().reshape(want.raw.shape), want.raw)


def test_append_out_of_range_is_left_out_and_reported():
    D, kv, page = 64, 1, 16
    n = 6
    x = torch.ones(n, kv, D, device="cuda", dtype=torch.float16)
    table = ints([[0, 9, -1], [1, 1, 1]])                    # page 9 and -1 do not exist in a pool of 2
    rope = x100b.rope_table(40, D, 1e4)
    for pos, seq, fine in (([0, 16, 0, 0, 0, 0], [0, 0, 1, 1, 1, 1], [0, 1]), ([0, 32, 48, 1, 2, 3], [0] * 6, [0]),
                           ([0, 1, 2, 3, 4, 5], [0, 2, -1, 0, 0, 0], [0]), ([0, 39, 40, 1, 2, 3], [0, 1, 1, 0, 0, 0], [0, 1])):
        cache = x100b.Kv4Cache(2, page, kv, D)
        live = [i for i in range(n) if i < 3]
        idx = torch.tensor(live, device="cuda")
        cache.append(x[idx], x[idx], ints([pos[i] for i in live]), table, seq=ints([seq[i] for i in live]), rope=rope)
        assert status() == x100b.X100_E_ARG and status() == 0   # reported once
        touched = cache.pages.view(2, -1).any(1).cpu().tolist()
        assert [i for i, y in enumerate(touched) if y] == fine


def test_append_not_finite_blocks_are_zeros_and_reported():
    D = 128
    k = torch.ones(3, 1, D, device="cuda")
    v = torch.ones(3, 1, D, device="cuda")
    k[0, 0, 5] = float("nan")
    v[1, 0, 40] = float("inf")
    v[2, 0, 100] = -float("inf")
    cache = x100b.Kv4Cache(1, 16, 1, D)
    pos, table = ints([0, 1, 2]), ints([[0]])
    cache.append(k, v, pos, table, seq=ints([0, 0, 0]), k_norm=torch.ones(D, device="cuda"))
    assert status() == x100b.X100_E_ARG
    kb, vb = (t.cpu().numpy() for t in cache.read(pos, table, seq=ints([0, 0, 0])))
    assert status() == 0 and np.isfinite(kb).all() and np.isfinite(vb).all()
    assert not kb[0].any() and (kb[1:] != 0).all()
    assert not vb[1, 0, 32:64].any() and (vb[1, 0, :32] == 1).all() and (vb[1, 0, 64:] == 1).all() and not vb[2, 0, 96:].any()


def test_append_extremes_saturate():
    D = 64
    v = torch.full((2, 1, D), 3e38, device="cuda")
    v[0, 0, 32:] = 1e-45
    v[1] = -70000.0
    cache = x100b.Kv4Cache(1, 16, 1, D)
    cache.append(torch.zeros_like(v), v, ints([0, 1]), ints([[0]]), seq=ints([0, 0]))
    _, vb = cache.read(ints([0, 1]), ints([[0]]), seq=ints([0, 0]))
    assert status() == 0
    assert (vb[0, 0, :32] == 65280).all() and not vb[0, 0, 32:].any() and (vb[1] == -65280).all()


# ---- attention ------------------------------------------------------------------------------
def run_attention(pool, table, lens, q_lens, heads, kind, seed=0, extra=0, scale=None, q_scale=1.0):
    rng = np.random.default_rng(seed)
    D, kv = pool.D, pool.raw.shape[1]
    scale = D ** -0.5 if scale is None else scale
    starts = np.concatenate([[0], np.cumsum(q_lens)])
    np_t = np.float32 if kind == "f32" else np.float16
    q = (q_scale * rng.normal(size=(starts[-1] + extra, heads, D))).astype(np_t)
    out = torch.full(q.shape, 7.0, dtype=DT[kind], device="cuda")
    cache_of(pool).attend(dev(q), out, ints(table), ints(lens), q_start=ints(starts), max_q=max(max(q_lens), 1), scale=scale)
    return q, starts, out.cpu().numpy(), scale


def check_attention(pool, table, lens, q_lens, heads, kind, **kw):
    q, starts, got, scale = run_attention(pool, table, lens, q_lens, heads, kind, **kw)
    assert status() == 0
    for b, n in enumerate(lens):
        rows = slice(starts[b], starts[b + 1])
        if rows.start == rows.stop:
            continue
        k, v = pool.values(table[b], n, False), pool.values(table[b], n, True)
        want = ref.attention(q[rows], k, v, n - q_lens[b], scale)
        bound = ref.attention_bound(q[rows], k, v, scale, n, kind == "f16")
        err = np.abs(got[rows].astype(np.float64) - want).max()
        assert err <= bound, (b, n, q_lens[b], err, bound)
        for i in range(q_lens[b]):
            if n - q_lens[b] + i < 0:
                assert not got[starts[b] + i].any()
    assert (got[starts[-1]:] == 7.0).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D,page,kv,heads", [(128, 64, 4, 32), (128, 16, 1, 3), (64, 32, 2, 2), (64, 128, 2, 14), (128, 128, 1, 16), (64, 16, 1, 40)])
def test_decode_lengths(kind, D, page, kv, heads):
    """One token of sequences of no, one and many positions; bytes past a length are garbage with NaN scales."""
    lens = [0, 1, 2, 15, 16, 17, 31, 127, 128, 129, 255, 700, 1000, 64]
    rng = np.random.default_rng(heads)
    n_pages = sum(-(-n // page) for n in lens) + 2
    pool = ref.random_pool(rng, n_pages, page, kv, D)
    table = page_table(rng, lens, page, n_pages)
    for b, n in enumerate(lens):                          # 0xFF bytes: codes 15, scales NaN
        for p in range(n, table.shape[1] * page):
            if table[b, p // page] >= 0:
                t, s = pool.raw[table[b, p // page], :, p % page // 16], p % 16
                for i in range(pool.NB):
                    for is_v in (False, True):
                        at = pool._scale(is_v, s, i)
                        t[:, at:at + 2] = 0xFF
    check_attention(pool, table, lens, [1] * len(lens), heads, kind)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D,heads,kv,lens,q_lens", [(128, 8, 2, [300, 5, 0, 2100, 17, 640], [1, 2, 1, 3, 0, 1]), (64, 6, 2, [1500, 33], [1, 1]), (128, 7, 1, [4000], [1]),
                                                    (128, 12, 1, [900, 1, 700], [1, 1, 2]), (64, 30, 1, [200, 0, 1300], [1, 1, 4])])
def test_narrow_and_wide_tables(kind, D, heads, kv, lens, q_lens):
    """The same sequences over a table that just holds them (clusters) and one that could hold far longer ones (runs and a merge)."""
    rng = np.random.default_rng(heads + len(lens))
    page = 32
    n_pages = sum(-(-n // page) for n in lens) + 1
    pool = ref.random_pool(rng, n_pages, page, kv, D)
    table = page_table(rng, lens, page, n_pages)
    wide = np.full((len(lens), 6000), -1, np.int32)
    wide[:, :table.shape[1]] = table
    for t in (table, wide):
        check_attention(pool, t, lens, q_lens, heads, kind, extra=1)


def test_sequences_around_a_cluster():
    """Every count of items around those that fill the card with clusters of 16, 8 and 4 CTAs."""
    rng = np.random.default_rng(40)
    pool = ref.random_pool(rng, 24, 64, 1, 128)
    for B in (1, 6, 7, 8, 9, 13, 15, 16, 17, 30, 31, 32, 33, 36, 60, 64, 70, 74, 80):
        lens = [int(n) for n in rng.integers(0, 1500, B)]
        table = rng.integers(0, 24, (B, 24)).astype(np.int32)
        check_attention(pool, table, lens, [1] * B, 8, "f16", seed=B)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D,heads,kv", [(128, 8, 2), (64, 6, 2), (128, 7, 1)])
def test_several_tokens_each(kind, D, heads, kv):
    """Ragged token counts, none among them; a sequence shorter than its tokens has rows that see nothing."""
    lens = [5, 40, 300, 3, 17, 0, 129, 1]
    q_lens = [2, 0, 9, 5, 17, 2, 4, 1]
    rng = np.random.default_rng(D)
    page = 32
    n_pages = 40
    pool = ref.random_pool(rng, n_pages, page, kv, D)
    table = page_table(rng, lens, page, n_pages, width=12)
    check_attention(pool, table, lens, q_lens, heads, kind, extra=3)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D,heads,kv,T,n", [(128, 8, 1, 200, 200), (128, 4, 2, 131, 515), (64, 6, 2, 257, 300), (128, 5, 1, 77, 1024), (64, 1, 1, 64, 64),
                                            (128, 8, 1, 40, 25)])
def test_prompt_chunks(kind, D, heads, kv, T, n):
    rng = np.random.default_rng(T)
    page = 64
    n_pages = -(-n // page) + 3
    pool = ref.random_pool(rng, n_pages, page, kv, D)
    check_attention(pool, page_table(rng, [n], page, n_pages), [n], [T], heads, kind)


def test_two_prompts_and_a_decode_token():
    lens, q_lens = [260, 33, 700], [130, 33, 1]
    for kind in ("f16", "f32"):
        rng = np.random.default_rng(9)
        pool = ref.random_pool(rng, 80, 16, 2, 128)
        check_attention(pool, page_table(rng, lens, 16, 80), lens, q_lens, 16, kind)


def test_sharp_and_flat_scores():
    """Scores that grow along the sequence (the running max moves at every tile) and scores that are all equal."""
    for kind in ("f32", "f16"):
        rng = np.random.default_rng(3)
        pool = ref.random_pool(rng, 20, 64, 1, 128)
        table = page_table(rng, [1200], 64, 20)
        for q_scale in (0.0, 0.01, 8.0):
            check_attention(pool, table, [1200], [1], 8, kind, q_scale=q_scale)


def test_one_long_sequence_is_split():
    rng = np.random.default_rng(4)
    n, page = 40000, 128
    pool = ref.random_pool(rng, -(-n // page), page, 1, 128)
    table = page_table(rng, [n], page, pool.raw.shape[0])
    for kind, q_lens in (("f32", [1]), ("f16", [1]), ("f16", [3])):
        check_attention(pool, table, [n], q_lens, 8, kind)


def test_shared_pages_and_strides():
    """Two sequences over the same pages give the same rows; q and out are slices of wider tensors."""
    rng = np.random.default_rng(8)
    pool = ref.random_pool(rng, 4, 64, 2, 64)
    table = np.array([[2, 0, 3], [2, 0, 1]], np.int32)
    wide = torch.randn(2, 9, 64, device="cuda")
    wide[1] = wide[0]
    out = torch.full((2, 12, 64), 5.0, device="cuda")
    cache_of(pool).attend(wide[:, 1:5], out[:, 4:8], ints(table), ints([100, 100]))
    assert status() == 0 and torch.equal(out[0, 4:8], out[1, 4:8])
    assert (out[:, :4] == 5).all() and (out[:, 8:] == 5).all()
    want = ref.attention(wide[:1, 1:5].cpu().numpy(), pool.values(table[0], 100, False), pool.values(table[0], 100, True), 99, 0.125)
    assert np.abs(out[0, 4:8].cpu().numpy() - want[0]).max() < 1e-4


def test_bad_pages_are_masked_and_reported():
    rng = np.random.default_rng(10)
    page, D = 16, 128
    pool = ref.random_pool(rng, 4, page, 1, D)
    q = rng.normal(size=(1, 4, D)).astype(np.float32)
    for hole in (-1, 4, 1 << 30):
        table = np.array([[0, hole, 2]], np.int32)
        out = cache_of(pool).attend(dev(q), None, ints(table), ints([40])).cpu().numpy()
        assert status() == x100b.X100_E_ARG
        keep = np.r_[0:16, 32:40]
        fixed = np.array([[0, 0, 2]], np.int32)[0]
        k, v = (pool.values(fixed, 40, i)[keep] for i in (False, True))
        want = ref.attention(q, k, v, 39, D ** -0.5)
        assert np.abs(out - want).max() <= ref.attention_bound(q, k, v, D ** -0.5, 40, False)


def test_bad_lengths_and_starts_are_reported():
    rng = np.random.default_rng(11)
    pool = ref.random_pool(rng, 2, 16, 1, 64)
    cache = cache_of(pool)
    q = torch.randn(4, 2, 64, device="cuda")
    table = ints([[0, 1], [1, 0]])
    for lens, starts, max_q, alive in (([33, 5], [0, 1, 2], 1, None), ([-1, 5], [0, 1, 2], 1, None), ([20, 5], [0, 3, 4], 2, [3]),
                                       ([20, 5], [0, 5, 4], 4, []), ([20, 5], [-1, 3, 4], 4, [3])):
        out = torch.full_like(q, 9.0)
        cache.attend(q, out, table, ints(lens), q_start=ints(starts), max_q=max_q)
        assert status() == x100b.X100_E_ARG and torch.isfinite(out).all()
        if alive is not None:
            touched = [i for i in range(4) if not (out[i] == 9.0).all()]
            assert touched == alive


def test_runs_are_repeatable_and_graphs_replay():
    rng = np.random.default_rng(12)
    lens = [3000, 17, 900, 2049]
    pool = ref.random_pool(rng, 100, 64, 2, 128)
    cache, table = cache_of(pool), ints(page_table(rng, lens, 64, 100))
    q, n = torch.randn(4, 16, 128, device="cuda").half(), ints(lens)
    works = [cache.attend_work(4, 16, 4) for _ in range(2)]
    first = cache.attend(q, None, table, n, work=works[0])
    for w in works:
        w.fill_(0xFF)                                     # what the scratch holds does not matter
    outs = [torch.zeros_like(first) for _ in range(2)]
    side = torch.cuda.Stream()
    graphs = []
    for o, w in zip(outs, works):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.attend(q, o, table, n, work=w)
        graphs.append(g)
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
        for o in outs:
            o.zero_()
    n.copy_(ints([100, 0, 901, 1]))                      # lengths are read when the graph runs
    graphs[0].replay()
    assert torch.equal(outs[0], cache.attend(q, None, table, n)) and status() == 0


def test_pool_past_32_bits():
    """Pages whose bytes lie beyond 4 GB."""
    page, kv, D = 128, 8, 128
    per = page // 16 * kv * 18 * D
    n_pages = (5 << 30) // per
    cache = x100b.Kv4Cache(n_pages, page, kv, D)
    rng = np.random.default_rng(13)
    ids = np.array([n_pages - 1, 0, n_pages - 2, (1 << 31) // per, (1 << 32) // per], np.int32)
    pool = ref.random_pool(rng, 5, page, kv, D)
    cache.pages.view(n_pages, -1)[torch.from_numpy(ids.astype(np.int64)).cuda()] = dev(pool.raw.reshape(5, -1))
    q = rng.normal(size=(1, 16, D)).astype(np.float32)
    n = 5 * page - 3
    out = cache.attend(dev(q), None, ints(ids[None]), ints([n])).cpu().numpy()
    k, v = (pool.values(np.arange(5), n, i) for i in (False, True))
    assert status() == 0 and np.abs(out - ref.attention(q, k, v, n - 1, D ** -0.5)).max() <= ref.attention_bound(q, k, v, D ** -0.5, n, False)
    pos = ints([n - 1])
    cache.append(torch.zeros(1, kv, D, device="cuda"), torch.zeros(1, kv, D, device="cuda"), pos, ints(ids[None]))
    kb, vb = cache.read(pos, ints(ids[None]))
    assert status() == 0 and not kb.any() and not vb.any()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_prompt_then_decode_steps(kind):
    """The operators as a program uses them: a prompt appended and attended in two chunks, then tokens one at a time."""
    rng = np.random.default_rng(14)
    D, kv, heads, page, n0, steps = 128, 2, 8, 16, 75, 6
    total = n0 + steps
    np_t = np.float32 if kind == "f32" else np.float16
    q, k, v = (rng.normal(size=(total, h, D)).astype(np_t) for h in (heads, kv, kv))
    rope = x100b.rope_table(total, D, 1e6)
    table = page_table(rng, [total], page, 7)
    cache, tab = x100b.Kv4Cache(7, page, kv, D), ints(table)
    outs, at = [], 0
    for n in [40, n0 - 40] + [1] * steps:
        rows = slice(at, at + n)
        pos = ints(np.arange(at, at + n))
        qr = cache.append(dev(k[rows]), dev(v[rows]), pos, tab, seq=ints(np.zeros(n)), q=dev(q[rows]), rope=rope)
        at += n
        outs.append(cache.attend(qr, None, tab, ints([at]), q_start=ints([0, n]), max_q=n))
    assert status() == 0
    got = torch.cat(outs).cpu().numpy()
    pool = ref.Pages(7, page, kv, D)
    pool.raw[...] = cache.pages.cpu().numpy().reshape(pool.raw.shape)
    qr = ref.rotate(q.astype(np.float32), rope.cpu().numpy(), np.arange(total)).astype(np_t)
    kk, vv = (pool.values(table[0], total, i) for i in (False, True))
    want = ref.attention(qr, kk, vv, 0, D ** -0.5)
    assert np.abs(got.astype(np.float64) - want).max() <= ref.attention_bound(qr, kk, vv, D ** -0.5, total, kind == "f16")


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("D,G", [(128, 5), (64, 7)])
def test_row_tiles(kind, D, G):
    """Every number of tokens from one to where the prompt kernel begins: one to four groups of eight rows in one tile and in several."""
    rng = np.random.default_rng(G)
    pool = ref.random_pool(rng, 14, 32, 1, D)
    for T in [*range(1, 18), 25, 33, 255 // G]:
        lens = [T, 300 + T, T // 2]
        check_attention(pool, rng.integers(0, 14, (3, 20)).astype(np.int32), lens, [T, T, T], G, kind, seed=T)
