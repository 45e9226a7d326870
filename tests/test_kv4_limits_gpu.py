"""Attention over the 4-bit cache at its limits: the longest runs, scores and queries of any size."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
import x100b
from test_kv4_gpu import DT, cache_of, dev, ints, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,T", [("f16", 640), ("f32", 640)])
def test_runs_past_16_bits_of_steps(kind, T):
    """Prompts of which every block takes more than 65536 steps of each kind, all rows checked.  The pages repeat, so a row's
    softmax is over 1024 positions, each weighted by how often the row sees it."""
    D, G, kv, page, unique, n = 64, 512, 8, 128, 1024, 131072
    rows_per_item, steps_per_tile = (256, 1) if kind == "f16" else (128, 0.5)
    tiles = kv * -(-T * G // rows_per_item) * ((n - T) // 128)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert tiles / sms * steps_per_tile > 65536 + 1024
    rng = np.random.default_rng(T)
    pool = ref.random_pool(rng, unique // page, page, kv, D)
    table = np.tile(np.arange(unique // page), n // unique)[None]
    q = torch.randn(T, kv * G, D, device="cuda", dtype=DT[kind], generator=torch.Generator("cuda").manual_seed(T))
    out = cache_of(pool).attend(q, None, ints(table), ints([n]), q_start=ints([0, T]), max_q=T)
    assert status() == 0
    k, v = (pool.values(table[0], unique, is_v) for is_v in (False, True))
    kd, vd = (torch.from_numpy(np.ascontiguousarray(x.transpose(1, 0, 2))).cuda() for x in (k, v))
    bound = ref.prompt_bound(q[:4].cpu().numpy(), k, v, D ** -0.5, n, kind == "f16") * q.abs().max().item() / q[:4].abs().max().item()
    bound += 2.0 ** -11 * np.abs(v).max() if kind == "f16" else 0.0
    worst = 0.0
    for i in range(T):
        sees = n - T + i + 1
        times = sees // unique + (torch.arange(unique, device="cuda") < sees % unique).double()
        z = D ** -0.5 * q[i].double().view(kv, G, D) @ kd.transpose(1, 2)
        p = times * torch.exp(z - z.amax(-1, keepdim=True))
        want = p @ vd / p.sum(-1, keepdim=True)
        worst = max(worst, (out[i].double().view(kv, G, D) - want).abs().max().item())
    assert worst <= bound, (worst, bound)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("T", [1, 3, 70])
def test_lists_that_end_in_nothing(kind, T):
    """More than 32 sequences of which few have tokens: the first, the last, one inside, none; clusters are too few for them."""
    rng = np.random.default_rng(T)
    D, kv, page, B = 64, 2, 16, 100
    pool = ref.random_pool(rng, 40, page, kv, D)
    table = ints(rng.integers(0, 40, (B, 20)))
    cache = cache_of(pool)
    for live in ([0], [B - 1], [31, 32], [40, 63, 64], []):
        counts, lens = np.zeros(B, int), rng.integers(0, 300, B)
        counts[live] = T
        starts = np.concatenate([[0], np.cumsum(counts)])
        q = rng.normal(size=(max(1, starts[-1]) + 1, 8 * kv, D)).astype(np.float32 if kind == "f32" else np.float16)
        out = torch.full(q.shape, 7.0, dtype=DT[kind], device="cuda")
        cache.attend(dev(q), out, table, ints(lens), q_start=ints(starts), max_q=T)
        assert status() == 0
        got = out.cpu().numpy()
        assert (got[starts[-1]:] == 7).all()
        for b in live:
            rows, row = slice(starts[b], starts[b + 1]), table[b].cpu().numpy()
            k, v = pool.values(row, lens[b], False), pool.values(row, lens[b], True)
            bound = ref.attention_bound if T * 8 < 256 else ref.prompt_bound
            bound = bound(q[rows], k, v, D ** -0.5, lens[b], kind == "f16") + (2.0 ** -11 * np.abs(v).max(initial=0) if kind == "f16" else 0)
            assert np.abs(got[rows].astype(np.float64) - ref.attention(q[rows], k, v, lens[b] - T, D ** -0.5)).max() <= bound


def test_as_many_sequences_as_a_call_takes():
    """65536 single tokens of no to 16 positions."""
    rng = np.random.default_rng(3)
    D, B = 64, 65536
    pool = ref.random_pool(rng, 5, 16, 1, D)
    page, lens = torch.arange(B, device="cuda") % 5, torch.arange(B, device="cuda") % 17
    q = torch.randn(B, 1, D, device="cuda")
    out = cache_of(pool).attend(q, None, page.int()[:, None], lens.int())
    assert status() == 0
    k, v = (torch.from_numpy(np.stack([pool.values(np.array([p]), 16, i)[:, 0] for p in range(5)])).cuda()[page] for i in (False, True))
    z = (q.double() @ k.transpose(1, 2))[:, 0] * D ** -0.5
    p = torch.where(torch.arange(16, device="cuda") < lens[:, None], torch.exp(z), 0.0)
    want = (p[:, None] @ v)[:, 0] / p.sum(-1, keepdim=True).clamp(min=1e-300)
    kn, vn = k[:5].cpu().numpy(), v[:5].cpu().numpy()
    assert (out[:, 0].double() - want).abs().max().item() <= ref.attention_bound(q.cpu().numpy(), kn, vn, D ** -0.5, 16, False)
    assert not out[lens == 0].any()
