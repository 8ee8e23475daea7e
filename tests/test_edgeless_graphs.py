"""Graphs without any edge (a batch of single atoms): nothing is aggregated, y = relu(x W_out[:, :F]^T)."""
import pytest
import torch

U = 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 300])
@pytest.mark.parametrize("f,h", [(64, 64), (11, 128), (40, 24)])
@pytest.mark.parametrize("form", ["sum", "cat", "egnn", "kept"])
def test_layer_on_a_graph_without_edges(form, n, f, h):
    from mpnn_amd import EGNNLayer, MPNNLayerCat, MPNNLayerSum
    torch.manual_seed(0)
    make = {"sum": MPNNLayerSum, "cat": MPNNLayerCat, "egnn": EGNNLayer, "kept": lambda *a: MPNNLayerSum(*a, checkpoint="int8")}[form]
    layer = make(f, 4, h).cuda()
    x = torch.randn(n, f, device="cuda", requires_grad=True)
    ei, ea = torch.empty((2, 0), dtype=torch.int64, device="cuda"), torch.empty((0, 4), device="cuda")
    gy = torch.randn(n, h, device="cuda")
    if form == "egnn":
        pos = torch.randn(n, 3, device="cuda")
        y, moved = layer(x, pos, ei, ea)
        assert torch.equal(moved, pos)
    else:
        y = layer(x, ei, ea)
    w = layer.linear_out.weight.detach().double()[:, :f]
    z, size = x.detach().double() @ w.t(), x.detach().double().abs() @ w.abs().t()
    # sums of three pieces per operand in some order, 2 u of the magnitudes per addition
    assert bool(((y.detach().double() - z.clamp_min(0)).abs() <= 2 * 3 * (f + h + 80) * U * size).all())
    gx, g_out = torch.autograd.grad(y, (x, layer.linear_out.weight), gy, retain_graph=True)
    gz = gy.double() * (y.detach() > 0)
    assert bool(((gx.double() - gz @ w).abs() <= 2 * 3 * (h + 80) * U * (gz.abs() @ w.abs()) + 1e-30).all())
    size = gz.abs().t() @ x.detach().double().abs()
    half = 0.0 if form != "kept" else 0.501 * (gz.abs().t() @ (x.detach().double().abs().amax(1, keepdim=True) / 127).expand(n, f))
    assert bool(((g_out.double()[:, :f] - gz.t() @ x.detach().double()).abs() <= 2 * 3 * (n + 80) * U * size + half + 1e-30).all())
    assert not g_out[:, f:].any()
    for g in torch.autograd.grad(y, [p for p in layer.parameters() if p is not layer.linear_out.weight], gy, allow_unused=True):
        assert g is None or not g.any()
