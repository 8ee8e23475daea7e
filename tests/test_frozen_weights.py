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
    # rows whose columns 32 bits cannot count with their padding
    wide = dict(m=(1 << 31) - 1, ldg=1 << 31, ldo=1 << 31)
    assert call(**wide) == -1
    assert lib.mpnn_relu_bits(p, 1 << 31, 0, 4, (1 << 31) - 1, p, None) == -1


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


def large_graph(n, e):
    gen = torch.Generator().manual_seed(7)
    return torch.randint(0, n, (2, e), generator=gen).cuda(), torch.rand(e, 4, generator=gen).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("f,h,dtype", [(64, 64, torch.float32), (11, 50, torch.float32), (300, 64, torch.float32), (64, 64, torch.bfloat16)])
def test_layer_with_frozen_weights_keeps_and_computes_what_is_wanted(f, h, dtype):
    """Only the weight gradients read 8-bit rows: x's for either weight, aggr's for the update's.  What is wanted is what the
    whole set of gradients has."""
    from mpnn_amd import MPNNLayerSum
    n = 3000
    ei, ea = large_graph(n, 15000)
    ea = ea.to(dtype)
    torch.manual_seed(0)
    layer = MPNNLayerSum(f, 4, h, checkpoint="int8").cuda().to(dtype)
    x = torch.randn(n, f, device="cuda").relu().to(dtype)
    gy = torch.randn(n, h, device="cuda").to(dtype)
    names = [k for k, _ in layer.named_parameters()]

    def grads(wanted, want_x):
        for k, p in layer.named_parameters():
            p.requires_grad_(k in wanted)
        leaf = x.clone().requires_grad_(want_x)
        held = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
            y = layer(leaf, ei, ea)
        ins = ([leaf] if want_x else []) + [p for k, p in layer.named_parameters() if k in wanted]
        out = torch.autograd.grad(y, ins, gy)
        return dict(zip((["x"] if want_x else []) + [k for k in names if k in wanted], out)), sum(t.dtype == torch.int8 for t in held)

    full, rows = grads(names, True)
    assert rows == 2
    tol = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -18     # the update's sums may run in another order without kept rows
    for wanted, rows_wanted in ((["linear_out.weight"], 2), (["fused_linear.weight"], 1), (["linear_3.weight"], 0), ([], 0),
                                (["fused_linear.weight", "linear_3.weight"], 1)):
        got, rows = grads(wanted, True)
        assert rows == rows_wanted, (wanted, rows)
        for k, g in got.items():
            assert float((g.double() - full[k].double()).norm()) <= tol * float(full[k].double().norm()), (wanted, k)
    got, rows = grads(["fused_linear.weight"], False)
    assert rows == 1 and float((got["fused_linear.weight"].double() - full["fused_linear.weight"].double()).norm()) <= tol * float(full["fused_linear.weight"].double().norm())
