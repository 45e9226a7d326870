"""Residual RMS norm with int8 output on the GPU, against the formula in numpy (kv4_ref.norm_q8)."""
import numpy as np
import pytest
import torch

import kv4_ref as ref
import x100b

pytestmark = pytest.mark.gpu


def run(x, res, w, group, eps=1e-6, pad=0, offset=0, in_place=False):
    """Codes, scales and h, with a row pitch of d + pad elements and a first element `offset` elements into the storage."""
    rows, d = x.shape

    def put(a):
        t = torch.zeros(rows * (d + pad) + offset + 16, dtype=torch.from_numpy(a).dtype, device="cuda")
        v = torch.as_strided(t, (rows, d), (d + pad, 1), offset)
        v.copy_(torch.from_numpy(a))
        return v

    xt, rt = put(x), None if res is None else put(res)
    h = None if res is None else rt if in_place else put(np.zeros_like(res))
    q = put(np.full((rows, d), 77, np.int8))
    scales = torch.full((rows, d // group if group else 1), -1.0, device="cuda")
    x100b.add_rmsnorm_q8(xt, torch.from_numpy(w).cuda(), q, scales, residual=rt, residual_out=h, eps=eps, group=group)
    x100b.sync()
    return q.cpu().numpy(), scales.cpu().numpy(), None if h is None else h.cpu().numpy()


def check(x, res, w, group, **kw):
    q, s, h = run(x, res, w, group, **kw)
    wh, wq, ws = ref.norm_q8(x, res, w, kw.get("eps", 1e-6), group)
    assert np.array_equal(q, wq)
    if res is not None:
        assert np.array_equal(h, wh)
    # d squares summed in a tree of at most d / 1024 + 10 + 5 steps, then a quotient, a root, a quotient and two products
    d = x.shape[1]
    assert (np.abs(s - ws) <= ws * (d / 1024 + 25) * 2.0 ** -24 + 1e-44).all()


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,d,group", [(1, 2048, 0), (3, 64, 0), (5, 64, 32), (70, 512, 128), (9, 1000, 0), (2, 4096, 64), (4, 8192, 0), (3, 16384, 0),
                                          (2, 20000, 0), (7, 257, 0), (1, 1, 0), (300, 96, 32), (2, 160, 32), (33, 2688, 128), (5, 7, 0), (2, 24576, 128)])
def test_shapes(kind, rows, d, group):
    rng = np.random.default_rng(d + rows)
    x, r = ((3 * rng.normal(size=(rows, d))).astype(kind) for _ in range(2))
    w = (1 + 0.3 * rng.normal(size=d)).astype(np.float32)
    check(x, r, w, group)
    check(x, None, w, group)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 1), (16, 3)])
def test_pitches_and_alignment(kind, pad, offset):
    rng = np.random.default_rng(pad + offset)
    x, r = (rng.normal(size=(6, 384)).astype(kind) for _ in range(2))
    w = (1 + 0.3 * rng.normal(size=384)).astype(np.float32)
    for group in (0, 32, 128):
        check(x, r, w, group, pad=pad, offset=offset, in_place=True)


def test_zero_tiny_and_not_finite_rows():
    w = np.ones(256, np.float32)
    x = np.zeros((6, 256), np.float32)
    x[1] = 1e-36                                   # under 2^-110
    x[2, 3] = np.nan
    x[3, 200] = np.inf
    x[4] = 1e-30
    x[5, 0] = 3.0
    for offset in (0, 1):                          # both kernels
        q, s, _ = run(x, None, w, 0, offset=offset)
        assert not q[:4].any() and (s[:2] == 0).all() and np.isnan(s[2:4]).all()
        assert (q[4] == 127).all() and np.isfinite(s[4:]).all() and q[5, 0] == 127 and not q[5, 1:].any()
        q, s, _ = run(x, None, w, 64, offset=offset)
        assert not q[:4].any() and np.isnan(s[2, 0]) and np.isnan(s[3, 3])


def test_pad_of_q_stays_and_scale_sizes():
    rng = np.random.default_rng(1)
    x = torch.randn(5, 128, device="cuda")
    q = torch.full((5, 160), 9, dtype=torch.int8, device="cuda")
    s = torch.empty(5, device="cuda")
    x100b.add_rmsnorm_q8(x, torch.ones(128, device="cuda"), q[:, :128], s)
    x100b.sync()
    assert (q[:, 128:] == 9).all()
    del rng


def test_rows_feed_the_int8_product():
    """norm -> int8 GEMM -> scales: the product of the quantised rows is exact, and close to the unquantised one."""
    rng = np.random.default_rng(2)
    M, K, N = 130, 512, 96
    x, r = (torch.from_numpy(rng.normal(size=(M, K)).astype(np.float32)).cuda() for _ in range(2))
    w = torch.from_numpy((1 + 0.1 * rng.normal(size=K)).astype(np.float32)).cuda()
    B = torch.from_numpy(rng.integers(-127, 128, (K, N), np.int8)).cuda()
    q = torch.empty(M, K, dtype=torch.int8, device="cuda")
    s = torch.empty(M, device="cuda")
    h = torch.empty_like(x)
    x100b.add_rmsnorm_q8(x, w, q, s, residual=r, residual_out=h)
    Cm = torch.zeros(M, N, dtype=torch.int32, device="cuda")
    x100b.gemm_dev("gemm_ime_i8_dev", q, B, Cm)
    x100b.sync()
    assert np.array_equal(Cm.cpu().numpy(), q.cpu().numpy().astype(np.int64) @ B.cpu().numpy().astype(np.int64))
    hd = h.double()
    y = hd / (hd.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    # each element is off by at most half a step of its row: |error| <= scale / 2 * sum |B|
    bound = (s.double()[:, None] * 0.5001) * B.double().abs().sum(0)[None]
    assert ((Cm.double() * s.double()[:, None] - y @ B.double()).abs() <= bound).all()


def test_graph_replay_reads_new_inputs():
    x = torch.randn(64, 1024, device="cuda").half()
    w = torch.ones(1024, device="cuda")
    q, s = torch.empty(64, 1024, dtype=torch.int8, device="cuda"), torch.empty(64, device="cuda")
    x100b.add_rmsnorm_q8(x, w, q, s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x100b.add_rmsnorm_q8(x, w, q, s)
    x.normal_()
    g.replay()
    x100b.sync()
    _, wq, _ = ref.norm_q8(x.cpu().numpy(), None, w.cpu().numpy(), 1e-6, 0)
    assert np.array_equal(q.cpu().numpy(), wq)
