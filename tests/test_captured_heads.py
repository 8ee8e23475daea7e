"""A head whose first backward of a size is captured: later eager calls do not read what the recorded graph has yet to fill."""
import pytest
import torch


@pytest.mark.gpu
def test_bias_gradient_after_a_capture_that_has_not_been_replayed():
    from mpnn_amd import dense
    dense._ONES.clear()
    n = 6000
    torch.manual_seed(0)
    linear = torch.nn.Linear(64, 10).cuda()
    x = torch.randn(n, 64, device="cuda")
    g = torch.randn(n, 10, device="cuda")

    def grads():
        return torch.autograd.grad(dense.head(x, linear), list(linear.parameters()), g)
    # the products' own first calls, at fewer rows
    small = torch.randn(5000, 64, device="cuda")
    torch.autograd.grad(dense.head(small, linear), list(linear.parameters()), g[:5000])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = grads()
    got = grads()                      # before any replay
    # 64-bit sums; float32 products in some order: 2 u per term, three pieces per operand
    want = (g.double().t() @ x.double(), g.double().sum(0))
    size = (g.double().abs().t() @ x.double().abs(), g.double().abs().sum(0))
    for a, w, s in zip(got, want, size):
        assert bool(((a.double() - w).abs() <= 2 * 3 * (n + 80) * 2.0 ** -24 * s).all())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, grads()))
