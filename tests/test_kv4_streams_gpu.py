"""What the 4-bit cache's Python calls do with a stream that is not the current one."""
import pytest
import torch

import x100b
from test_kv4_gpu import ints, status

pytestmark = pytest.mark.gpu


def test_rope_table_on_a_stream_takes_its_output():
    """A table made on the current stream would be written by another one that nothing orders: refused, as the other calls."""
    side, want = torch.cuda.Stream(), x100b.rope_table(100, 64, 1e4)
    with pytest.raises(x100b.X100Error) as e:
        x100b.rope_table(100, 64, 1e4, stream=side)
    assert e.value.code == x100b.X100_E_ARG
    out = torch.zeros(100, 32, 2, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    assert x100b.rope_table(100, 64, 1e4, stream=side, out=out) is out
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and status() == 0
    for bad in (torch.zeros(100, 64, device="cuda"), torch.zeros(99, 32, 2, device="cuda"), torch.zeros(100, 32, 2), torch.zeros(100, 32, 2, device="cuda").half(),
                torch.zeros(100, 32, 4, device="cuda")[:, :, :2]):
        with pytest.raises(x100b.X100Error) as e:
            x100b.rope_table(100, 64, 1e4, out=bad)
        assert e.value.code == x100b.X100_E_ARG


def test_a_new_pool_is_zeroed_before_another_stream_appends():
    side, pos, table, seq = torch.cuda.Stream(), ints([0]), ints([[0]]), ints([0])
    x = torch.ones(1, 1, 64, device="cuda")
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)                        # about a tenth of a second on the current stream
    cache = x100b.Kv4Cache(1, 16, 1, 64)
    cache.append(x, x, pos, table, seq=seq, stream=side)
    torch.cuda.synchronize()
    k, v = cache.read(pos, table, seq=seq)
    assert (k == 1).all() and (v == 1).all() and status() == 0
