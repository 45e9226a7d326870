"""The grouped form of the int8 norm with the library's int8 product: one product per group, each with its own scales."""
import numpy as np
import pytest
import torch

import x100b

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_groups_feed_a_product_each(kind, group):
    rng = np.random.default_rng(group)
    M, K, N = 70, 384, 96
    x, r = (torch.from_numpy(rng.normal(size=(M, K)).astype(np.float32)).cuda().to(kind) for _ in range(2))
    x[:, :group] *= 50                                    # a group that would take the other ones' bits with one scale per row
    w = torch.from_numpy((1 + 0.1 * rng.normal(size=K)).astype(np.float32)).cuda()
    B = torch.from_numpy(rng.integers(-127, 128, (K, N), np.int8)).cuda()
    q, s, h = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, K // group, device="cuda"), torch.empty_like(x)
    x100b.add_rmsnorm_q8(x, w, q, s, residual=r, residual_out=h, group=group)
    parts = torch.zeros(K // group, M, N, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for i in range(K // group):
        x100b.check(x100b.lib().gemm_ime_i8_dev_ld(M, N, group, q.data_ptr() + i * group, K, B.data_ptr() + i * group * N, N, parts[i].data_ptr(), N, stream))
    x100b.sync()
    want = torch.stack([q[:, i * group:(i + 1) * group].double() @ B[i * group:(i + 1) * group].double() for i in range(K // group)])
    assert torch.equal(parts.double(), want)
    y = (parts.double() * s.double().T[:, :, None]).sum(0)
    hd = h.double()
    exact = hd / (hd.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    # each element is off by at most half a step of its group (0.5001: the scale's own fp32 roundings): |error| <= sum scale / 2 * sum |B|
    bound = sum(0.5001 * s.double()[:, i:i + 1] * B[i * group:(i + 1) * group].double().abs().sum(0)[None] for i in range(K // group))
    assert ((y - exact @ B.double()).abs() <= bound).all()
