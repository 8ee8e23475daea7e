"""A layer that keeps its inputs in 8 bits: a training step of it on another stream, and captured and replayed with eager work between."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("f,h,dtype", [(64, 64, torch.float32), (300, 64, torch.float32), (64, 64, torch.bfloat16)])
def test_kept_layer_step_on_another_stream_and_replayed(f, h, dtype):
    from mpnn_amd import MPNNLayerSum
    n, e = 6000, 50000
    gen = torch.Generator().manual_seed(3)
    ei, ea = torch.randint(0, n, (2, e), generator=gen).cuda(), torch.rand(e, 4, generator=gen).cuda().to(dtype)
    torch.manual_seed(0)
    layer = MPNNLayerSum(f, 4, h, checkpoint="int8").cuda().to(dtype)
    x = torch.randn(n, f, device="cuda").relu().to(dtype).requires_grad_()
    gy = torch.randn(n, h, device="cuda").to(dtype)

    def step():
        y = layer(x, ei, ea)
        return (y.detach(), *torch.autograd.grad(y, [x, *layer.parameters()], gy))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(1.25)
            gy.mul_(-0.5)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want)), k
