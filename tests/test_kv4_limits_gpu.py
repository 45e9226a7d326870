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
