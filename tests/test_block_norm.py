"""block_norm (residual join with the norms around it) against its definition in 64 bits, values and gradients.

Tolerances.  u = 2^-24 bounds the relative error of one float32 operation, a stored result is off by half a step of
its type (eps / 2) on top.  A row sum in the kernel adds at most 8 terms in a lane, then at most 8 levels of a tree: 16
roundings, so a mean is off by 16 u times the mean of the magnitudes; with the handful of operations after it 40 u
covers a normalised value.  An error e of a row v moves hat = norm(v) by at most inv * (e + mean e) + |hat| * inv *
rms(e) to first order.  The backward's row sums are of the same kind (100 u for two of them and the products), and an
error d of hat moves the gradient by at most 3 d times the terms it is made of.
"""
import itertools

import pytest
import torch

from mpnn_amd import _lib

U = 2.0 ** -24


def ref_norm(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    inv = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    return v * inv, inv


def reference(t, kind, eps, post, rs, bs):
    """(stream, normed) in float64 from a dict of float64 tensors."""
    n = t["block"]
    if post:
        n = ref_norm(n, kind, eps)[0]
        n = n * t.get("post_weight", 1.0) + t.get("post_bias", 0.0)
    s = bs * t.get("gate", 1.0) * n + (rs * t["residual"] if "residual" in t else 0.0)
    return s, ref_norm(s, kind, eps)[0] * t.get("weight", 1.0) + t.get("bias", 0.0)


def norm_error(v, e, kind, eps):
    """(hat, inv, bound on the error of hat) for a row v known to within e."""
    hat, inv = ref_norm(v, kind, eps)
    mean_abs = v.abs().mean(1, keepdim=True) if kind == "layer" else 0.0
    own = 40 * U * (hat.abs() * (1 + inv * mean_abs) + inv * mean_abs)
    moved = inv * (e + e.mean(1, keepdim=True)) + hat.abs() * inv * (e * e).mean(1, keepdim=True).sqrt()
    return hat, inv, own + moved


def back_error(gh, e_gh, hat, inv, e_hat):
    m = lambda x: x.mean(1, keepdim=True)
    size = inv * (gh.abs() + m(gh.abs()) + hat.abs() * (m((gh * hat).abs()) + m(gh.abs())))
    d = e_hat.max(1, keepdim=True).values
    return (100 * U + 3 * d) * size + inv * (e_gh + m(e_gh) + hat.abs() * m(e_gh * hat.abs()))


def bounds(t, kind, eps, post, rs, bs, gs, gn):
    """Error bounds (before the final rounding) of every output and gradient, by name."""
    zero = torch.zeros_like(t["block"])
    w, b = t.get("weight", zero[0] + 1), t.get("bias", zero[0])
    pw, pb = t.get("post_weight", zero[0] + 1), t.get("post_bias", zero[0])
    gate = t.get("gate", zero[0] + 1)
    n, e_n = t["block"], zero
    if post:
        hat1, inv1, e1 = norm_error(n, zero, kind, eps)
        n = hat1 * pw + pb
        e_n = e1 * pw.abs() + 4 * U * (n.abs() + pb.abs())
    res = t.get("residual", zero)
    s = rs * res + bs * gate * n
    e_s = (bs * gate).abs() * e_n + 4 * U * ((rs * res).abs() + (bs * gate * n).abs())
    hat2, inv2, e2 = norm_error(s, e_s, kind, eps)
    out = {"stream": e_s, "normed": e2 * w.abs() + 4 * U * ((hat2 * w).abs() + b.abs())}
    # rows per group, groups of a block and slabs are added one after the other: at most 64 roundings at these sizes
    col = lambda term, e: e.sum(0) + 64 * U * term.abs().sum(0)
    gh = gn * w
    out["weight"] = col(gn * hat2, gn.abs() * e2)
    out["bias"] = col(gn, 0 * gn)
    e_g = back_error(gh, U * gh.abs(), hat2, inv2, e2) + 4 * U * gs.abs()
    m = lambda x: x.mean(1, keepdim=True)
    g = gs + inv2 * (gh - (m(gh) if kind == "layer" else 0.0) - hat2 * m(gh * hat2))
    out["residual"] = abs(rs) * e_g + 2 * U * (rs * g).abs()
    g, e_g = bs * g, abs(bs) * e_g + 2 * U * (bs * g).abs()
    term, e_term = g * n, e_g * n.abs() + e_n * g.abs() + 2 * U * (g * n).abs()
    if "gate" in t:
        shape = t["gate"].shape
        if shape == term.shape:
            out["gate"] = e_term
        elif shape[-1] == 1 and t["block"].size(1) != 1:
            out["gate"] = e_term.sum(1, keepdim=True) + 40 * U * term.abs().sum(1, keepdim=True)
        else:
            out["gate"] = col(term, e_term)
    g, e_g = g * gate, e_g * gate.abs() + 2 * U * (g * gate).abs()
    if post:
        out["post_weight"] = col(g * hat1, e_g * hat1.abs() + g.abs() * e1)
        out["post_bias"] = col(g, e_g)
        gh = g * pw
        e_g = back_error(gh, e_g * pw.abs() + U * gh.abs(), hat1, inv1, e1)
    out["block"] = e_g
    return out


def make(n, h, dtype, gate, post, kind, seed, residual=True, vectors=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype)
    t = {"block": r(n, h)}
    if residual:
        t["residual"] = r(n, h) * 2
    shape = {"channel": (h,), "one": (1, h), "row": (n, 1), "full": (n, h)}.get(gate)
    if shape:
        t["gate"] = r(*shape)
    if vectors:
        t["weight"], t["bias"] = r(h) + 1, r(h)
        if post:
            t["post_weight"], t["post_bias"] = r(h) + 1, r(h)
    return t, r(n, h), r(n, h)


def close(got, want, bound, dtype, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + 1e-40
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((got - want).abs() / tol).max()))


def check(t, gs, gn, kind, post, eps=1e-5, rs=1.0, bs=1.0, place=lambda x: x.cuda()):
    from mpnn_amd import block_norm
    dtype = t["block"].dtype
    d = {k: v.double().requires_grad_() for k, v in t.items()}
    want = reference(d, kind, eps, post, rs, bs)
    want_g = torch.autograd.grad(want, list(d.values()), (gs.double(), gn.double()))
    dev = {k: place(v).requires_grad_() for k, v in t.items()}
    kw = {k: v for k, v in dev.items() if k != "block"}
    got = block_norm(dev["block"], norm=kind, eps=eps, post_norm=post, residual_scale=rs, branch_scale=bs, **kw)
    got_g = torch.autograd.grad(got, list(dev.values()), (place(gs), place(gn)))
    b = bounds({k: v.detach() for k, v in d.items()}, kind, eps, post, rs, bs, gs.double(), gn.double())
    for name, a, w in zip(("stream", "normed"), got, want):
        close(a, w.detach(), b[name], dtype, name)
    for name, a, w in zip(d, got_g, want_g):
        assert a.dtype == dtype
        close(a, w, b[name].view(w.shape), dtype, "gradient of " + name)
    return got


WIDTHS = [1, 3, 8, 16, 17, 63, 64, 65, 100, 128, 200, 256, 264, 500, 512, 513, 1000, 1024, 1031, 2040, 2048]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("h", WIDTHS)
def test_every_width(h, dtype):
    for (kind, post), gate in zip(itertools.product(("rms", "layer"), (False, True)), ("channel", "full", "row", None)):
        check(*make(37, h, dtype, gate, post, kind, h), kind, post)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [None, "channel", "one", "row", "full"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_every_form(kind, post, gate):
    for n in (1, 2, 1500):
        check(*make(n, 64, torch.float32, gate, post, kind, 3), kind, post, rs=0.5, bs=-1.25)
    check(*make(130, 64, torch.bfloat16, gate, post, kind, 4, residual=False), kind, post)
    check(*make(130, 24, torch.float32, gate, post, kind, 4, vectors=False), kind, post, eps=0.1)


@pytest.mark.gpu
def test_strided_rows_and_odd_addresses():
    def inside(x):
        """The same values as columns of a wider matrix, one element off a 16-byte boundary."""
        if x.dim() == 1:
            return torch.cat([x.new_zeros(1), x]).cuda()[1:]
        wide = torch.zeros(x.size(0), x.size(1) + 5, dtype=x.dtype).cuda()
        wide[:, 1:1 + x.size(1)] = x.cuda()
        return wide[:, 1:1 + x.size(1)]

    def by_columns(x):
        return x.cuda() if x.dim() == 1 else x.t().contiguous().cuda().t()

    for place in (inside, by_columns):
        for gate in ("channel", "row", "full"):
            check(*make(33, 64, torch.float32, gate, True, "layer", 5), "layer", True, place=place)
            check(*make(33, 48, torch.bfloat16, gate, True, "rms", 5), "rms", True, place=place)


@pytest.mark.gpu
def test_expanded_operands_take_the_gradient_of_every_use():
    from mpnn_amd import block_norm
    torch.manual_seed(0)
    row = torch.randn(1, 32, device="cuda", requires_grad=True)
    col = torch.randn(20, 1, device="cuda", requires_grad=True)
    block = torch.randn(20, 32, device="cuda")
    g = torch.randn(20, 32, device="cuda")
    s = block_norm(block, row.expand(20, 32), gate=col.expand(20, 32), outputs="stream")
    gr, gc = torch.autograd.grad(s, (row, col), g)
    assert torch.allclose(gr, g.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)
    assert torch.allclose(gc, (g * block).sum(1, keepdim=True), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("outputs", ["stream", "normed"])
def test_one_output_and_unused_outputs(outputs):
    from mpnn_amd import block_norm
    t, gs, gn = make(70, 64, torch.float32, "full", True, "layer", 6)
    if outputs == "stream":
        del t["weight"], t["bias"]
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    kw = {k: v for k, v in dev.items() if k != "block"}
    only = block_norm(dev["block"], norm="layer", post_norm=True, outputs=outputs, **kw)
    both = block_norm(dev["block"], norm="layer", post_norm=True, **kw)
    of_both = both[0] if outputs == "stream" else both[1]
    assert torch.equal(only, of_both)
    g = (gs if outputs == "stream" else gn).cuda()
    leaves = list(dev.values())
    for a, b in zip(torch.autograd.grad(only, leaves, g), torch.autograd.grad(of_both, leaves, g)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_no_rows():
    from mpnn_amd import block_norm
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    gate = torch.ones(0, 1, device="cuda", requires_grad=True)
    s, n = block_norm(x, x, weight=w, gate=gate)
    assert s.shape == n.shape == (0, 64)
    gx, gw, gg = torch.autograd.grad((s, n), (x, w, gate), (s, n))
    assert gx.shape == (0, 64) and gg.shape == (0, 1) and torch.equal(gw, torch.zeros_like(w))


@pytest.mark.gpu
def test_rows_of_zeros_infinities_and_nan_stay_in_their_rows():
    from mpnn_amd import block_norm
    t, gs, gn = make(40, 64, torch.float32, None, True, "rms", 7)
    clean = block_norm(t["block"].cuda(), t["residual"].cuda(), post_norm=True)
    t["block"][3] = 0.0
    t["block"][5, 7] = float("nan")
    t["block"][9, 1] = float("inf")
    got = block_norm(t["block"].cuda(), t["residual"].cuda(), post_norm=True)
    for a, c in zip(got, clean):
        assert a[5].isnan().all() and a[9].isnan().any()
        keep = [i for i in range(40) if i not in (3, 5, 9)]
        assert torch.equal(a[keep], c[keep])
    assert torch.equal(got[0][3], t["residual"][3].cuda())     # the norm of zeros is zeros


@pytest.mark.gpu
def test_gradient_against_differences():
    """The directional derivative of the 64-bit function, by central differences, against the kernel's gradient."""
    from mpnn_amd import block_norm
    t, gs, gn = make(12, 40, torch.float32, "row", True, "layer", 8)
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    out = block_norm(dev["block"], norm="layer", post_norm=True, **{k: v for k, v in dev.items() if k != "block"})
    grads = torch.autograd.grad(out, list(dev.values()), (gs.cuda(), gn.cuda()))
    gen = torch.Generator().manual_seed(1)
    for name, g in zip(t, grads):
        step = torch.randn(t[name].shape, generator=gen).double()
        def value(k):
            d = {a: v.double() for a, v in t.items()}
            d[name] = d[name] + k * step
            s, n = reference(d, "layer", 1e-5, True, 1.0, 1.0)
            return float((s * gs.double()).sum() + (n * gn.double()).sum())
        k = 1e-5
        want = (value(k) - value(-k)) / (2 * k)
        got = float((g.double().cpu() * step).sum())
        # central differences: k^2 times third derivatives (some 1e-8 here) and 2^-52 * |value| / k; the kernel's
        # float32 gradient: 1e-5 of the terms' magnitudes
        assert abs(got - want) <= 1e-5 * float((g.double().cpu() * step).abs().sum()) + 1e-6, name


@pytest.mark.gpu
def test_same_bits_twice_and_on_another_stream():
    from mpnn_amd import block_norm
    t, gs, gn = make(3000, 128, torch.float32, "channel", True, "rms", 9)
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    gs, gn = gs.cuda(), gn.cuda()

    def once():
        out = block_norm(dev["block"], post_norm=True, **{k: v for k, v in dev.items() if k != "block"})
        return (*out, *torch.autograd.grad(out, list(dev.values()), (gs, gn)))

    first = once()
    assert all(torch.equal(a, b) for a, b in zip(first, once()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))


@pytest.mark.gpu
def test_captured_step_replays():
    from mpnn_amd import block_norm
    t, gs, gn = make(500, 64, torch.float32, "full", True, "layer", 10)
    leaves = {k: v.cuda().requires_grad_() for k, v in t.items()}
    gs, gn = gs.cuda(), gn.cuda()

    def once():
        out = block_norm(leaves["block"], norm="layer", post_norm=True, **{k: v for k, v in leaves.items() if k != "block"})
        return (*(o.detach() for o in out), *torch.autograd.grad(out, list(leaves.values()), (gs, gn)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for k in range(3):
        with torch.no_grad():
            leaves["block"].mul_(1.5)
            gs.mul_(0.5)
        want = once()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k


@pytest.mark.gpu
def test_second_derivative_is_refused():
    from mpnn_amd import block_norm
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(block_norm(x, outputs="normed").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_refusals():
    from mpnn_amd import block_norm
    with pytest.raises(_lib.MpnnError, match="GPU"):
        block_norm(torch.zeros(4, 8))


@pytest.mark.gpu
def test_refusals_of_device_tensors():
    from mpnn_amd import block_norm
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    x = z(4, 8)
    for bad in (z(4, 8, dtype=torch.float16), z(4, 8, dtype=torch.int64)):
        with pytest.raises(TypeError):
            block_norm(bad)
    for bad in (z(8), z(4, 0), z(2, 4, 8), z(1, 2049)):
        with pytest.raises(ValueError):
            block_norm(bad)
    for kw in (dict(residual=z(3, 8)), dict(gate=z(4)), dict(gate=z(2, 8)), dict(weight=z(7)), dict(bias=z(1, 8)),
               dict(post_weight=z(8)), dict(norm="batch"), dict(outputs="none"), dict(eps=-1.0), dict(eps=float("nan")),
               dict(weight=z(8), outputs="stream")):
        with pytest.raises(ValueError):
            block_norm(x, **kw)
    for kw in (dict(residual=z(4, 8, dtype=torch.bfloat16)), dict(weight=z(8, dtype=torch.float64))):
        with pytest.raises(TypeError):
            block_norm(x, **kw)
    with pytest.raises(_lib.MpnnError):
        block_norm(x, residual=torch.zeros(4, 8))


def test_entry_points_refuse_before_any_launch():
    """Addresses are never followed here: every call is rejected on the host."""
    lib = _lib.load()
    fake = 1 << 20

    def desc(**kw):
        d = _lib.BlockNormDesc(block=fake, ldb=8, N=4, H=8, eps=1e-5, stream=fake, lds=8)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    for entry in (lib.mpnn_block_norm_fwd, lib.mpnn_block_norm_bwd):
        assert entry(None, None) == -1
        for kw in (dict(N=-1), dict(H=0), dict(H=2049), dict(dtype=2), dict(norm=2), dict(gate_kind=4), dict(gate_kind=-1),
                   dict(eps=float("nan")), dict(block=None), dict(ldb=7), dict(residual=fake, ldr=7), dict(gate_kind=1),
                   dict(gate=fake), dict(gate_kind=3, gate=fake, ldg=7), dict(gate_kind=2, gate=fake, ldg=0)):
            assert entry(desc(**kw), None) == -1, kw
            assert lib.mpnn_last_error()
    assert lib.mpnn_block_norm_fwd(desc(lds=7), None) == -1
    assert lib.mpnn_block_norm_fwd(desc(stream=None), None) == -1 and b"no output" in lib.mpnn_last_error()
    assert lib.mpnn_block_norm_bwd(desc(g_stream=fake, ldgs=7), None) == -1
    assert lib.mpnn_block_norm_bwd(desc(g_post_w=fake), None) == -1
    assert lib.mpnn_block_norm_bwd(desc(g_w=fake), None) == -1 and b"null" in lib.mpnn_last_error()     # no partial
    assert lib.mpnn_block_norm_partial_floats(-1, 8, 0) == -1 and lib.mpnn_block_norm_partial_floats(1, 2049, 0) == -1
    assert lib.mpnn_block_norm_partial_floats(0, 8, 0) == 0
