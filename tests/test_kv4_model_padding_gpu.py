"""Any negative position is a padding token of a model over the paged 4-bit cache."""
import numpy as np
import pytest
import torch

import py_oracle as po
import x100b
from test_kv4_model_gpu import CFG, REL, paged, world  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pad", [-1, -2, -7, -(1 << 20), -(1 << 31)])
def test_padding_positions(world, pad):  # noqa: F811
    rng = np.random.default_rng(11)
    m = paged(world, rng)
    toks = rng.integers(0, CFG["vocab"], 4)
    for t in range(3):
        m.forward(toks, [t] * 4)
    before = m._pages.clone()
    want = m.forward(toks[:1], [3])
    pages = m._pages.clone()
    m._pages.copy_(before)
    got = m.forward(toks, [3, pad, pad, pad])             # raises where the step reports
    assert po.rel_l2(got[0], want[0]) <= REL and torch.equal(m._pages, pages)


def test_padding_names_no_slot(world):  # noqa: F811
    """The slot of a padding token is not looked at, as its page is not."""
    m = paged(world, np.random.default_rng(12))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tok, h, pos, slot = i32(1, 2, 3), torch.zeros(3, CFG["d"], device="cuda"), i32(0, -5, -1), i32(2, 99, -(1 << 31))
    logits = torch.empty(3, CFG["vocab"], device="cuda")
    m.forward_slots_dev(tok, h, pos, slot, logits, 3)
    x100b.sync()
    assert torch.isfinite(logits[0]).all()
