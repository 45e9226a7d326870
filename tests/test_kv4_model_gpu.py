"""The decode model over the paged 4-bit cache (x100q_model_create_kv4): append, attention and the layers around them together.

The statement is one layer in 64 bits over the keys and values read back from the layer's pool (their values are exact in
fp16).  What is left of the model's own arithmetic is what the fp16 cache's model has too, so the bar is the same:
relative L2 of 1e-3 of the oracle's step.
"""
import numpy as np
import pytest
import torch

import py_oracle as po
import x100b

pytestmark = pytest.mark.gpu

REL = 1e-3
CFG = dict(n_layers=2, d=512, n_heads=16, n_kv_heads=2, head_dim=128, vocab=256, n_exp=8, n_act=2, moe_ffn=256, attn_qtype=po.Q8_0, expert_qtype=po.Q3_K,
           lm_qtype=po.Q8_0, ctx=420, max_batch=4, expert_lo=0, expert_hi=8, rope_base=1e6, eps=1e-6)
PAGE, PAGES = 32, 60


def make_layer(rng, c):
    d, qd, kvd, hd, E, F = c["d"], c["n_heads"] * c["head_dim"], c["n_kv_heads"] * c["head_dim"], c["head_dim"], c["n_exp"], c["moe_ffn"]
    q = lambda qt, n, k: po.quantize(qt, rng.normal(0, 0.05, (n, k)).astype(np.float32))  # noqa: E731
    near1 = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
    return dict(attn_norm=near1(d), wq=q(po.Q8_0, qd, d), wk=q(po.Q8_0, kvd, d), wv=q(po.Q8_0, kvd, d), q_norm=near1(hd), k_norm=near1(hd),
                wo=q(po.Q8_0, d, qd), ffn_norm=near1(d), router=(0.3 * rng.standard_normal((E, d))).astype(np.float32),
                gate=q(po.Q3_K, E * F, d), up=q(po.Q3_K, E * F, d), down=q(po.Q3_K, E * d, F))


def np_layer(c, W, K, V, h, pos):
    """One token's layer in float64; K, V [kv heads, pos + 1, dim] as the cache holds them.  Also the token's own k and v."""
    nh, nkv, hd, E, F, d = (c[n] for n in ("n_heads", "n_kv_heads", "head_dim", "n_exp", "moe_ffn", "d"))
    rms = lambda x, w: x / np.sqrt(np.mean(x * x, -1, keepdims=True) + c["eps"]) * w  # noqa: E731
    a = pos * np.float64(c["rope_base"]) ** (-2.0 * np.arange(hd // 2) / hd)

    def rope(v):
        x, y = v[:, :hd // 2], v[:, hd // 2:]
        return np.concatenate([x * np.cos(a) - y * np.sin(a), x * np.sin(a) + y * np.cos(a)], -1)

    hn = rms(h, W["attn_norm"])
    q = rope(rms((W["wq"] @ hn).reshape(nh, hd), W["q_norm"]))
    k = rope(rms((W["wk"] @ hn).reshape(nkv, hd), W["k_norm"]))
    v = (W["wv"] @ hn).reshape(nkv, hd)
    s = np.einsum("gid,gnd->gin", q.reshape(nkv, nh // nkv, hd), K) / np.sqrt(hd)
    p = np.exp(s - s.max(-1, keepdims=True))
    att = np.einsum("gin,gnd->gid", p / p.sum(-1, keepdims=True), V)
    h = h + W["wo"] @ att.reshape(-1)
    hn = rms(h, W["ffn_norm"])
    lg = W["router"] @ hn
    p = np.exp(lg - lg.max())
    sel = np.argsort(-p, kind="stable")[: c["n_act"]]
    for e in sel:
        g, u = W["gate"][e] @ hn, W["up"][e] @ hn
        h = h + p[e] / p[sel].sum() * (W["down"][e] @ (g / (1 + np.exp(-g)) * u))
    return h, k, v


def fill(m, w):
    for li, lw in enumerate(w["layers"]):
        m.set_layer(li, *(lw[n] for n in ("attn_norm", "wq", "wk", "wv", "q_norm", "k_norm", "wo", "ffn_norm", "router", "gate", "up", "down")))
    m.set_output(w["emb"], w["out_norm"], w["lm"])
    return m


@pytest.fixture(scope="module")
def world():
    rng = np.random.default_rng(77)
    c = CFG
    w = dict(c=c, layers=[make_layer(rng, c) for _ in range(c["n_layers"])], emb=rng.standard_normal((c["vocab"], c["d"])).astype(np.float32),
             out_norm=(1 + 0.1 * rng.standard_normal(c["d"])).astype(np.float32), lm=po.quantize(po.Q8_0, rng.normal(0, 0.05, (c["vocab"], c["d"])).astype(np.float32)))
    qd, kvd, d, E, F = c["n_heads"] * c["head_dim"], c["n_kv_heads"] * c["head_dim"], c["d"], c["n_exp"], c["moe_ffn"]
    deq = lambda qt, b, n, k: po.dequant(qt, b, n, k).astype(np.float64)  # noqa: E731
    w["wide"] = [dict({n: lw[n].astype(np.float64) for n in ("attn_norm", "q_norm", "k_norm", "ffn_norm", "router")}, wq=deq(po.Q8_0, lw["wq"], qd, d),
                      wk=deq(po.Q8_0, lw["wk"], kvd, d), wv=deq(po.Q8_0, lw["wv"], kvd, d), wo=deq(po.Q8_0, lw["wo"], d, qd),
                      gate=deq(po.Q3_K, lw["gate"], E * F, d).reshape(E, F, d), up=deq(po.Q3_K, lw["up"], E * F, d).reshape(E, F, d),
                      down=deq(po.Q3_K, lw["down"], E * d, F).reshape(E, d, F)) for lw in w["layers"]]
    w["wide_lm"] = deq(po.Q8_0, w["lm"], c["vocab"], d)
    return w


def table_of(rng, c=CFG):
    """Every slot's pages, in no order; the table covers ctx."""
    n = -(-c["ctx"] // PAGE)
    return torch.from_numpy(rng.permutation(PAGES)[: c["max_batch"] * n].reshape(c["max_batch"], n).astype(np.int32)).cuda()


def paged(w, rng, **over):
    c = dict(w["c"], **over)
    return fill(x100b.Model(kv4=(PAGES, PAGE, table_of(rng)), **c), w)


def cached(m, layer, slot, n):
    """K, V [kv heads, n, dim] of a slot's first n positions, float64."""
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    k, v = m.kv4_cache(layer).read(pos, m.kv4_table, seq=torch.full_like(pos, slot))
    return (t.double().cpu().numpy().transpose(1, 0, 2) for t in (k, v))


def np_logits(w, m, slot, token, pos):
    h = w["emb"][token].astype(np.float64)
    for li, W in enumerate(w["wide"]):
        K, V = cached(m, li, slot, pos + 1)
        h, k, v = np_layer(w["c"], W, K, V, h, pos)
        # the cache holds the token's own: within a step of the scale (the code 15 clamps a whole step), and the scale's and fp32's roundings
        for have, x in ((K[:, pos], k), (V[:, pos], v)):
            top = np.abs(x).reshape(x.shape[0], -1, 32).max(-1).repeat(32, -1)
            assert (np.abs(have - x) <= top / 8 * 1.05).all()
    return w["wide_lm"] @ (h / np.sqrt(np.mean(h * h) + w["c"]["eps"]) * w["out_norm"])


def test_steps_of_several_slots(world):
    rng = np.random.default_rng(1)
    c, m = world["c"], paged(world, rng)
    B = c["max_batch"]
    toks = rng.integers(0, c["vocab"], (40, B))
    for t in range(40):
        got = m.forward(toks[t], [t] * B)
        if t in (0, 1, 15, 16, 31, 32, 39):
            for b in range(B):
                want = np_logits(world, m, b, toks[t, b], t)
                assert po.rel_l2(got[b], want) <= REL, (t, b, po.rel_l2(got[b], want))
    with pytest.raises(x100b.X100Error) as e:
        m.kv_read(0, 0, 0, 1)
    assert e.value.code == x100b.X100_E_UNSUPPORTED
    with pytest.raises(x100b.X100Error):
        m.kv4_cache(c["n_layers"])


@pytest.mark.parametrize("first,n", [(1, 4), (30, 3), (5, 20), (17, 40), (40, 333)])
def test_prefill_after_a_prompt(world, first, n):
    """Prompts of as many tokens as a step, of the decode kernel's rows and of the prompt kernel's, behind positions of an earlier call."""
    rng = np.random.default_rng(n)
    c, m = world["c"], paged(world, rng)
    toks = rng.integers(0, c["vocab"], first + n)
    m.prefill(2, toks[:first], 0, logits=False)
    got = m.prefill(2, toks[first:], first)
    for i in sorted({0, 1, n // 2, n - 1}):
        want = np_logits(world, m, 2, toks[first + i], first + i)
        assert po.rel_l2(got[i], want) <= REL, (i, po.rel_l2(got[i], want))
    # and the step after it
    got = m.forward([7] * 3, [0, 0, first + n])[2]
    want = np_logits(world, m, 2, 7, first + n)
    assert po.rel_l2(got, want) <= REL


def test_page_order_does_not_matter(world):
    rng = np.random.default_rng(3)
    toks = rng.integers(0, CFG["vocab"], 300)
    out = []
    for _ in range(2):
        m = paged(world, rng)
        out.append(np.concatenate([m.prefill(1, toks[:290], 0)] + [m.forward([3, toks[t]], [0, t])[1:] for t in range(290, 300)]))
    assert np.array_equal(out[0].view(np.uint32), out[1].view(np.uint32))


def test_captured_steps(world):
    """A captured step, replayed over advancing positions, against eager steps of a second model."""
    rng = np.random.default_rng(4)
    B, m, e = 3, paged(world, rng), paged(world, rng)
    tok, pos = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    h, logits = torch.zeros(B, CFG["d"], device="cuda"), torch.zeros(B, CFG["vocab"], device="cuda")
    m.forward_dev(tok, h, pos, logits, B)                    # attributes are set before the capture
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        m.forward_dev(tok, h, pos, logits, B)
        pos.add_(1)
    pos.zero_()
    for t in range(20):
        toks = rng.integers(0, CFG["vocab"], B)
        tok.copy_(torch.from_numpy(toks.astype(np.int32)))
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(logits.cpu().numpy(), e.forward(toks, [t] * B)), t


def test_padding_and_positions_out_of_range(world):
    rng = np.random.default_rng(5)
    c = CFG
    m = paged(world, rng)
    toks = rng.integers(0, c["vocab"], 4)
    for t in range(3):
        m.forward(toks, [t] * 4)
    before = m._pages.clone()
    ref = m.forward(toks[:1], [3])
    m._pages.copy_(before)
    got = m.forward(toks, [3, -1, -1, -1])                    # padding tokens beside it
    assert po.rel_l2(got[0], ref[0]) <= REL and x100b.last_error() == 0
    for slot in (1, 2, 3):
        p = m.kv4_table[slot].long()
        for li in range(c["n_layers"]):
            n = m._pages.shape[1] // PAGES
            assert torch.equal(m._pages[li].view(PAGES, n)[p], before[li].view(PAGES, n)[p])
    for bad in (c["ctx"], 1 << 30, 0x7fffffff):
        before.copy_(m._pages)
        with pytest.raises(x100b.X100Error) as e:
            m.forward(toks, [0, 0, 0, bad])
        assert e.value.code == x100b.X100_E_ARG
    one = torch.tensor([c["max_batch"]], dtype=torch.int32, device="cuda")
    h, zero = torch.zeros(1, c["d"], device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    before.copy_(m._pages)
    m.forward_slots_dev(zero, h, zero, one, None, 1)
    with pytest.raises(x100b.X100Error) as e:
        x100b.sync()
    assert e.value.code == x100b.X100_E_ARG and torch.equal(before, m._pages)


def test_loaded_from_a_file(world, tmp_path):
    import gguf_writer as gw
    c = dict(CFG, d=512, n_layers=1)
    path = str(tmp_path / "m.gguf")
    gw.qwen3moe_file(path, c, dict(q=po.Q8_0, k=po.Q8_0, v=po.Q8_0, o=po.Q8_0, exp=po.Q3_K, router=po.Q_F32, norm=po.Q_F32, embd=po.F16, lm=po.Q8_0), seed=9)
    g = x100b.Gguf(path)
    rng = np.random.default_rng(6)
    m, f = g.load_model(kv4=(PAGES, PAGE, table_of(rng)), ctx=CFG["ctx"], max_batch=4), g.load_model(ctx=CFG["ctx"], max_batch=4)
    # position 0 sees itself alone: the difference is v's 4 bits.  A later layer sees it through Wo: no equality, but the same token's k and v
    m.forward([5], [0]), f.forward([5], [0])
    k, v = f.kv_read(0, 0, 0, 1)
    K, V = cached(m, 0, 0, 1)
    for have, want in ((K, k), (V, v)):
        want = want.view(np.float16).astype(np.float64)
        top = np.abs(want).reshape(*want.shape[:2], -1, 32).max(-1).repeat(32, -1)
        assert (np.abs(have - want) <= top / 8 * 1.05).all() and np.abs(have).max() > 0
    m.close(), f.close(), g.close()
