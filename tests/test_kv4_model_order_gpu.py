"""The host calls of a model over the paged 4-bit cache come after what the caller's stream does to its table and pages."""
import contextlib

import numpy as np
import pytest
import torch

import x100b
from test_kv4_model_gpu import CFG, PAGE, PAGES, paged, world  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def other_rows(m):
    """A table of pages that the model's own does not name."""
    used = set(m.kv4_table.flatten().tolist())
    free = [p for p in range(PAGES) if p not in used]
    t = m.kv4_table.clone()
    t[0, 0] = free[0]
    return t


@pytest.mark.parametrize("where", ["default stream", "another stream"])
@pytest.mark.parametrize("call", ["forward", "prefill of a step", "prefill"])
def test_a_table_written_just_before(world, where, call):  # noqa: F811
    """Long work, then a change of the table and of a page on the current stream, then the call at once: what a call after a
    synchronisation gives, bit for bit, and the page that the row named before is left alone."""
    rng = np.random.default_rng(8)
    m = paged(world, rng)
    n = {"forward": 1, "prefill of a step": 3, "prefill": PAGE}[call]
    toks = rng.integers(0, CFG["vocab"], n)
    step = (lambda: m.forward(toks, [0])) if call == "forward" else (lambda: m.prefill(0, toks, 0))
    rows, new = m.kv4_table.clone(), other_rows(m)
    step()
    results = []
    for wait in (True, False):
        m.kv4_table.copy_(rows)
        m._pages.fill_(0x11)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream() if where == "another stream" else None
        with torch.cuda.stream(stream) if stream else contextlib.nullcontext():
            torch.cuda._sleep(200_000_000)                # about a tenth of a second
            m.kv4_table.copy_(new)
            m._pages.fill_(0x22)
            if wait:
                torch.cuda.synchronize()
            logits = step()
        torch.cuda.synchronize()
        results.append((logits, m._pages.clone()))
    (a, pa), (b, pb) = results
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32)) and torch.equal(pa, pb)
    page = pa.view(CFG["n_layers"], PAGES, -1)
    assert (page[:, int(rows[0, 0])] == 0x22).all() and not (page[:, int(new[0, 0])] == 0x22).all()


def test_the_c_call_waits_for_the_default_stream(world):  # noqa: F811
    rng = np.random.default_rng(9)
    m = paged(world, rng)
    new, tok, pos = other_rows(m), np.array([3], np.int32), np.zeros(1, np.int32)
    logits = np.empty((1, CFG["vocab"]), np.float32)
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    m.kv4_table.copy_(new)
    x100b.check(x100b.lib().x100q_model_forward(m.h, tok.ctypes.data, pos.ctypes.data, logits.ctypes.data, 1))
    page = m._pages.view(CFG["n_layers"], PAGES, -1)
    assert page[:, int(new[0, 0])].any(1).all()
