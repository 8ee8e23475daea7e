"""Kept calls whose weights want no gradient: g where the relu is open in one pass, nothing larger than g beside it."""
import pytest
import torch

from mpnn_amd import _lib


@pytest.mark.gpu
@pytest.mark.parametrize("n,m", [(1, 1), (3, 7), (40, 8), (33, 31), (64, 32), (65, 33), (129, 64), (50, 100), (1000, 128), (300, 257), (20000, 136)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_open_entries(n, m, dtype):
    from mpnn_amd.rows8 import open_entries, relu_bits
    gen = torch.Generator().manual_seed(n + m)
    y = torch.randn(n, m, generator=gen).relu().to(dtype)
    g = torch.randn(n, m, generator=gen).to(dtype)
    shut = (y <= 0).nonzero()
    if len(shut):                                  # nothing of a closed entry comes through, not even a NaN
        g[tuple(shut[0])] = float("nan")
        g[tuple(shut[-1])] = float("inf")
    want = torch.where(y > 0, g, torch.zeros((), dtype=dtype))
    bits = relu_bits(y.cuda())
    wider = torch.zeros(n, m + 16, dtype=dtype)
    wider[:, 8:m + 8] = g
    wider = wider.cuda()
    odd = torch.zeros(n, m + 1, dtype=dtype)
    odd[:, 1:] = g
    for view in (g.cuda(), wider[:, 8:m + 8], odd.cuda()[:, 1:], g.t().contiguous().cuda().t()):
        got = open_entries(view, bits)
        assert got.is_contiguous() and torch.equal(got.cpu(), want)
    row = torch.randn(1, m, generator=gen).to(dtype).cuda().expand(n, m)
    assert torch.equal(open_entries(row, bits).cpu(), torch.where(y > 0, row.cpu(), torch.zeros((), dtype=dtype)))


def test_open_entries_refuses_before_any_launch():
    """Addresses are never followed here: every call is rejected on the host."""
    lib, p = _lib.load(), 1 << 20
    call = lambda **k: lib.mpnn_open_entries(*{**dict(g=p, ldg=16, dt=0, bits=p, out=p, ldo=16, n=4, m=16, st=None), **k}.values())
    for bad in (dict(dt=2), dict(n=-1), dict(m=0), dict(ldg=15), dict(ldo=15), dict(g=None), dict(bits=None), dict(out=None)):
        assert call(**bad) == -1, bad
    assert call(n=0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_update_with_a_frozen_weight_takes_no_more_than_its_gradients(dtype):
    """At its largest the backward holds the gradient of the relu's input and the two input gradients, which are its results."""
    from mpnn_amd.dense import update
    n, f, h = 100000, 64, 128
    x, a = (torch.randn(n, c, device="cuda").to(dtype).requires_grad_() for c in (f, h))
    w = torch.randn(h, f + h, device="cuda").to(dtype)
    gy = torch.randn(n, h, device="cuda").to(dtype)
    y = update(x, a, w, checkpoint="int8")
    want = torch.autograd.grad(y, (x, a), gy, retain_graph=True)
    torch.cuda.synchronize()
    size = gy.element_size()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = torch.autograd.grad(y, (x, a), gy)
    assert torch.cuda.max_memory_allocated() - before <= size * n * (h + f + h) + (2 << 20)
    # the same product with a plain torch mask: gemm_nn takes it either way
    from mpnn_amd.rows8 import gemm_nn
    both = gemm_nn(torch.where(y > 0, gy, torch.zeros((), dtype=dtype, device="cuda")), w)
    for p, q in ((got, want), (got, (both[:, :f], both[:, f:]))):
        assert all(torch.equal(s, t) for s, t in zip(p, q))
