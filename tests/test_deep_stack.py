"""Layers, joins and 8-bit rows together, as a deep stack uses them: layers that keep their inputs in 8 bits against the
plain ones, a stack of layers with block_norm between them trained one step, and the same weights answering through 8-bit
products."""
import pytest
import torch

U = 2.0 ** -24


def graph(n, e, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, n, (2, e), generator=g).to(device), torch.rand(e, 4, generator=g).to(device)


def half_steps(g, *xs):
    """Bound of g^T [x ..] for every entry of x being off by half a step of its row (and the roundings of the scale)."""
    from mpnn_amd import quantize_rows
    s = [quantize_rows(t.detach()).scale.double().unsqueeze(1).expand(-1, t.size(1)) for t in xs]
    return g.double().abs().t() @ torch.cat(s, dim=1) * (0.5 + 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["sum", "cat"])
@pytest.mark.parametrize("n,e,f,h,dtype", [(3000, 24000, 64, 64, torch.float32), (2500, 20000, 500, 64, torch.float32),
                                           (3000, 9000, 11, 50, torch.float32), (3000, 24000, 128, 128, torch.bfloat16),
                                           (2100, 5000, 11, 64, torch.bfloat16)])
def test_layer_that_keeps_its_inputs_in_8_bits(mode, n, e, f, h, dtype):
    from mpnn_amd import MPNNLayerCat, MPNNLayerSum, aggregate_fused, graph_for
    from mpnn_amd.dense import project, update
    cls = MPNNLayerSum if mode == "sum" else MPNNLayerCat
    ei, ea = graph(n, e)
    ea = ea.to(dtype)
    torch.manual_seed(1)
    plain = cls(f, 4, h).cuda().to(dtype)
    kept = cls(f, 4, h, checkpoint="int8").cuda().to(dtype)
    kept.load_state_dict(plain.state_dict())
    x = torch.randn(n, f, device="cuda").relu().to(dtype).requires_grad_()
    gy = torch.randn(n, h, device="cuda").to(dtype)
    y0, y1 = plain(x, ei, ea), kept(x, ei, ea)
    g0 = dict(zip(["x"] + [k for k, _ in plain.named_parameters()], torch.autograd.grad(y0, [x, *plain.parameters()], gy)))
    g1 = dict(zip(["x"] + [k for k, _ in kept.named_parameters()], torch.autograd.grad(y1, [x, *kept.parameters()], gy)))
    if dtype == torch.bfloat16:
        # one rounding of a float32 sum each, taken in another order
        assert ((y0 - y1).double().abs() <= 2.0 ** -7 * y0.double().abs() + 1e-6).all()
        for k in g0:
            a, b = g0[k].double(), g1[k].double()
            # 127 steps: 2^-8 of a row's largest entry at most, where the rows' own roundings are 2^-9 of each entry
            assert float((a - b).norm()) <= 0.02 * float(a.norm()), k
        return
    if f < 2 * h:        # (a plain layer with wide inputs reads them once per direction, in another order of sums)
        assert torch.equal(y0, y1) and torch.equal(g0["x"], g1["x"])
    assert float((y0 - y1).norm()) <= 1e-6 * float(y0.norm())
    # the node weights' gradients: bounded by half a step of every kept entry, with the layer's inner gradients from its parts
    w = {k: v.detach() for k, v in plain.named_parameters()}
    if mode == "sum":
        w_nodes, w_edge = w["fused_linear.weight"], w["linear_3.weight"]
    else:
        lw = w["linear.weight"]
        w_nodes, w_edge = torch.cat([lw[:, :f], lw[:, f:2 * f]]), lw[:, 2 * f:].contiguous()
    ab = project(x.detach(), w_nodes).requires_grad_()
    aggr = aggregate_fused(ab, ea, w_edge, graph_for(ei, n))
    y = update(x.detach(), aggr, w["linear_out.weight"])
    (g_ab,) = torch.autograd.grad(y, ab, gy)
    slack = 1e-5
    d = (g0["linear_out.weight"] - g1["linear_out.weight"]).double().abs()
    assert (d <= half_steps(gy * (y > 0), x, aggr) + slack * g0["linear_out.weight"].abs().max()).all()
    bound = half_steps(g_ab, x)
    if mode == "sum":
        d = (g0["fused_linear.weight"] - g1["fused_linear.weight"]).double().abs()
        assert (d <= bound + slack * g0["fused_linear.weight"].abs().max()).all()
        if f < 2 * h:
            assert torch.equal(g0["linear_3.weight"], g1["linear_3.weight"])
    else:
        d = (g0["linear.weight"] - g1["linear.weight"]).double().abs()
        both = torch.cat([bound[:h], bound[h:]], dim=1)
        assert (d[:, :2 * f] <= both + slack * g0["linear.weight"].abs().max()).all()
        if f < 2 * h:
            assert torch.equal(g0["linear.weight"][:, 2 * f:], g1["linear.weight"][:, 2 * f:])


@pytest.mark.gpu
def test_kept_layer_holds_less_between_the_passes():
    from mpnn_amd import MPNNLayerSum
    n, h = 20000, 128
    ei, ea = graph(n, 60000)
    x = torch.randn(n, h, device="cuda", requires_grad=True)

    def held(checkpoint):
        layer = MPNNLayerSum(h, 4, h, checkpoint=checkpoint).cuda()
        layer(x, ei, ea)                              # the graph's own structures exist after this
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = layer(x, ei, ea)
        return torch.cuda.memory_allocated() - before - y.numel() * 4

    # plain: the projection (2 H) and aggr (H) in float32; kept: x and aggr in a byte each, the relu in bits
    saved = held(None) - held("int8")
    assert saved >= n * h * (4 * 3 - 2 - 1 / 8) - 2 * 4 * n - (1 << 20)


class Stack(torch.nn.Module):
    def __init__(self, f, h, depth, checkpoint):
        super().__init__()
        from mpnn_amd import MPNNLayerSum
        self.first = MPNNLayerSum(f, 4, h, checkpoint=checkpoint)
        self.layers = torch.nn.ModuleList([MPNNLayerSum(h, 4, h, checkpoint=checkpoint) for _ in range(depth)])
        self.norms = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(h)) for _ in range(depth + 1)])
        self.gates = torch.nn.ParameterList([torch.nn.Parameter(torch.full((h,), 0.5)) for _ in range(depth)])
        self.head = torch.nn.Linear(h, 7)

    def forward(self, x, ei, ea):
        from mpnn_amd import block_norm
        from mpnn_amd.dense import head
        stream = self.first(x, ei, ea)
        u = block_norm(stream, weight=self.norms[0], outputs="normed")
        for layer, gate, w in zip(self.layers, self.gates, self.norms[1:]):
            stream, u = block_norm(layer(u, ei, ea), stream, gate=gate, weight=w)
        return head(u, self.head)


@pytest.mark.gpu
@pytest.mark.parametrize("depth", [1, 4])
def test_stack_trains_alike_with_kept_inputs(depth):
    """Everything but the node weights' gradients is the same to the bit: forwards, input gradients, norms, gates, edge
    weights.  The node weights' gradients then differ by the 8-bit rows alone, 2^-8 of a row's largest entry per term."""
    n = 5000
    ei, ea = graph(n, 30000, seed=2)
    x = torch.randn(n, 40, device="cuda")
    target = torch.randint(0, 7, (n,), device="cuda")
    from mpnn_amd.loss import masked_cross_entropy
    torch.manual_seed(3)
    plain = Stack(40, 64, depth, None).cuda()
    kept = Stack(40, 64, depth, "int8").cuda()
    kept.load_state_dict(plain.state_dict())
    losses = []
    for model in (plain, kept):
        loss = masked_cross_entropy(model(x, ei, ea), target)
        loss.backward()
        losses.append(loss.detach())
    assert torch.equal(*losses)
    for (k, p), (_, q) in zip(plain.named_parameters(), kept.named_parameters()):
        if "fused_linear" in k or "linear_out" in k:
            assert float((p.grad - q.grad).norm()) <= 2.0 ** -6 * float(p.grad.norm()), k
        else:
            assert torch.equal(p.grad, q.grad), k


@pytest.mark.gpu
def test_stack_answers_through_8_bit_products():
    """The update's and the head's products of a trained layer from 8-bit weights: off by at most half a step of either
    operand per term."""
    from mpnn_amd import MPNNLayerSum, aggregate_fused, block_norm, graph_for, linear_int8, quantize_rows
    from mpnn_amd.dense import project, update
    n, f, h = 4000, 64, 64
    ei, ea = graph(n, 20000, seed=4)
    torch.manual_seed(5)
    layer, head = MPNNLayerSum(f, 4, h).cuda(), torch.nn.Linear(h, 7).cuda()
    x = torch.randn(n, f, device="cuda").relu()
    with torch.no_grad():
        ab = project(x, layer.fused_linear.weight)
        ab8 = linear_int8(x, quantize_rows(layer.fused_linear.weight))

        def bound(t, w):
            st = quantize_rows(t).scale.double().unsqueeze(1) * 0.501
            sw = quantize_rows(w).scale.double() * 0.501
            return t.double().abs().sum(1, keepdim=True) * sw + st * w.double().abs().sum(1) + t.size(1) * st * sw

        assert ((ab - ab8).double().abs() <= bound(x, layer.fused_linear.weight) + 1e-5).all()
        aggr = aggregate_fused(ab8, ea, layer.linear_3.weight, graph_for(ei, n))
        y = update(x, aggr, layer.linear_out.weight)
        u = block_norm(y, x, outputs="normed")
        out, out8 = head(u), linear_int8(u, quantize_rows(head.weight), bias=head.bias)
        assert ((out - out8).double().abs() <= bound(u, head.weight) + 1e-5).all()
        assert torch.equal(out8, linear_int8(quantize_rows(u), quantize_rows(head.weight), bias=head.bias))


@pytest.mark.gpu
def test_model_takes_the_option_and_refuses_others():
    from mpnn_amd import MPNN, MPNNLayerSum
    with pytest.raises(ValueError):
        MPNNLayerSum(8, 4, 8, checkpoint="int4")
    n = 3000
    ei, ea = graph(n, 9000, seed=6)
    x = torch.randn(n, 20, device="cuda")
    torch.manual_seed(0)
    a = MPNN(20, 32, 7, num_layers=3, mode="cat").cuda()
    b = MPNN(20, 32, 7, num_layers=3, mode="cat", checkpoint="int8").cuda()
    b.load_state_dict(a.state_dict())
    assert torch.equal(a(x, ei, ea), b(x, ei, ea))
    b.eval()
    with torch.no_grad():
        assert torch.equal(a(x, ei, ea), b(x, ei, ea))


def test_option_is_checked_without_a_gpu():
    from mpnn_amd import MPNN, MPNNLayerCat
    with pytest.raises(ValueError):
        MPNNLayerCat(8, 4, 8, checkpoint=True)
    assert MPNN(20, 32, 7, checkpoint="int8").layers[1].checkpoint == "int8"
    assert MPNN(20, 32, 7).layers[0].checkpoint is None


@pytest.mark.gpu
def test_captured_products_replay_side_by_side():
    """Two graphs recorded one after the other, replayed at once on two streams: neither uses the other's workspaces."""
    from mpnn_amd.dense import project
    n = 60000
    xs = [torch.randn(n, 64, device="cuda").requires_grad_() for _ in range(2)]
    ws = [torch.randn(200, 64, device="cuda").requires_grad_() for _ in range(2)]
    gy = torch.randn(n, 200, device="cuda")

    def step(k):
        y = project(xs[k], ws[k], checkpoint="int8")
        return (y.detach(), *torch.autograd.grad(y, (xs[k], ws[k]), gy))

    want = [step(0), step(1)]
    graphs, held = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(step(k))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, h in zip(want, held):
        assert all(torch.equal(a, b) for a, b in zip(w, h))


@pytest.mark.gpu
def test_operators_inside_a_traced_function():
    """A tracing compiler breaks its graph at the operators and takes their eager results."""
    from mpnn_amd import block_norm, linear_int8, quantize_rows
    from mpnn_amd.dense import project, update
    x, w = torch.randn(300, 64, device="cuda"), torch.randn(64, 64, device="cuda")
    wo, w8 = torch.randn(64, 128, device="cuda"), quantize_rows(w)

    def run(x):
        y = update(x, project(x, w, checkpoint="int8"), wo, checkpoint="int8")
        stream, u = block_norm(y * 2, x)
        with torch.no_grad():
            return stream + 1, linear_int8(u, w8)

    traced = torch.compile(run, backend="eager")
    for a, b in zip(traced(x), run(x)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matrices_beyond_32_bit_offsets(dtype):
    """More than 2^31 entries: the last rows are what they are by themselves."""
    from mpnn_amd import block_norm, linear_int8, quantize_rows
    from mpnn_amd.dense import project
    n, h, tail = (1 << 31) // 128 + 1001, 128, 1000
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((n, h), dtype=dtype, device="cuda").normal_(generator=gen)
    w = torch.randn(64, h, device="cuda", generator=gen).to(dtype).requires_grad_()
    last = x[-tail:].clone()

    def ends(t):
        return t[-tail:].clone()
    stream, normed = block_norm(x, x, norm="layer", post_norm=True)
    for p, q in zip((stream, normed), block_norm(last, last, norm="layer", post_norm=True)):
        assert torch.equal(ends(p), q)
    del stream, normed
    rows, rows_last = quantize_rows(x), quantize_rows(last)
    assert torch.equal(ends(rows.values), rows_last.values) and torch.equal(ends(rows.scale), rows_last.scale)
    w8 = quantize_rows(torch.randn(h, h, device="cuda", generator=gen).to(dtype))
    assert torch.equal(ends(linear_int8(x, w8)), linear_int8(last, w8))
    assert torch.equal(ends(linear_int8(rows, w8)), linear_int8(rows_last, w8))
    x.requires_grad_()
    last.requires_grad_()
    y, y_last = project(x, w, checkpoint="int8"), project(last, w, checkpoint="int8")
    assert torch.equal(ends(y.detach()), y_last)
    gy = torch.zeros((n, 64), dtype=dtype, device="cuda")
    gy[-tail:] = torch.randn(tail, 64, device="cuda", generator=gen)
    (gx, gw), (gx_last, gw_last) = (torch.autograd.grad(o, (i, w), g) for o, i, g in ((y, x, gy), (y_last, last, gy[-tail:])))
    assert torch.equal(ends(gx), gx_last) and not gx[:-tail].any()
    # the rows meet in other blocks: float32 sums of 1000 products each way, one rounding to the type
    size = gy[-tail:].double().abs().t() @ rows_last.dequantize().double().abs()
    assert bool(((gw - gw_last).double().abs() <= 2 * tail * 2.0 ** -24 * size + torch.finfo(dtype).eps * gw_last.double().abs()).all())
