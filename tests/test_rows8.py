"""Rows in 8 bits: the format to the bit, the product with 8-bit weights, the weight gradient from 8-bit rows, and the
dense products that keep their inputs in them.

Tolerances.  u = 2^-24 per float32 operation, eps / 2 of the stored type on top.
  linear_int8   the integer sum is exact; its conversion, the product of the scales, their product and the bias are one
                rounding each: 3 u |sum * scales| + u |y|.
  gemm_tn8      g * scale is one rounding; its pieces are exact in float32 (3 of 8 bits) and off by at most 2^-17 in
                bfloat16 (2 of 8 bits); their products with whole numbers are exact.  Every addition rounds (or cuts) by
                at most 2 u of the partial sum: with d additions in a row, 2 d u times the sum of the magnitudes.  A row
                share is at most 256 rows at these sizes (3 pieces: d = 768) and slabs and blocks add at most 80 more.
                Whole numbers with scale 1 have no rounding at all: there the result is equal, which pins the indexing.
"""
import numpy as np
import pytest
import torch

from mpnn_amd import _lib

U = 2.0 ** -24
TINY = 2.0 ** -100


def quantized(x):
    """(q, scale) by the definition, in float64 with the roundings to float32 where the definition has them."""
    v = x.detach().cpu().double().numpy()
    top = np.abs(v).max(axis=1) if v.shape[1] else np.zeros(len(v))
    q, scale = np.zeros(v.shape, np.int8), np.zeros(len(v), np.float32)
    for i, t in enumerate(top):
        if not np.isfinite(t):
            scale[i] = np.nan
        elif t >= TINY:
            scale[i] = np.float32(t / 127.0)
            q[i] = np.rint(v[i] * np.float64(np.float32(127.0 / t))).astype(np.int8)
    return torch.from_numpy(q), torch.from_numpy(scale)


def same_rows(r, x):
    q, s = quantized(x)
    assert torch.equal(r.values.cpu(), q)
    assert torch.equal(r.scale.cpu().nan_to_num(nan=-1.0), s.nan_to_num(nan=-1.0))


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


WIDTHS = [1, 3, 8, 15, 16, 17, 32, 33, 64, 100, 128, 255, 256, 500, 512, 513, 1024, 1030, 2048, 2056, 4096, 5000, 8192]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", WIDTHS)
def test_quantize_every_width(k, dtype):
    from mpnn_amd import quantize_rows
    x = randn(37, k, seed=k, dtype=dtype) * torch.logspace(-3, 3, 37).unsqueeze(1).to(dtype)
    r = quantize_rows(x.cuda())
    same_rows(r, x)
    assert r.pitch % 16 == 0 and r.values.data_ptr() % 16 == 0
    store = torch.as_strided(r.values, (37, r.pitch), (r.pitch, 1))
    assert not store[:, k:].any()
    err = (r.dequantize().cpu().double() - x.double()).abs()
    # half a step, and the rounding of 127 / top and top / 127 on a number of at most 127 steps
    assert (err <= r.scale.cpu().double().unsqueeze(1) * (0.5 + 127 * 4 * U)).all()


@pytest.mark.gpu
def test_quantize_borders_and_special_rows():
    from mpnn_amd import quantize_rows
    n = float("nan")
    rows = [[0.0, -0.0, 0.0, 0.0], [127.0, 0.5, 1.5, -2.5], [127.0, -126.5, 125.5, 3.5], [2.0 ** -101] * 4,
            [2.0 ** -100, 2.0 ** -101, 0.0, 0.0], [3.4e38, -3.4e38, 1e38, 1.0], [1.0, n, 0.0, 0.0],
            [float("inf"), 1.0, 2.0, 3.0], [-float("inf"), n, 2.0, 3.0], [1e-45, 0.0, 0.0, 0.0]]
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.tensor(rows).to(dtype)
        r = quantize_rows(x.cuda())
        same_rows(r, x)
        assert r.dequantize()[6:9].isnan().all()
    # neighbours of every border between two whole numbers
    k = torch.arange(-126, 127).float() + 0.5
    x = torch.cat([torch.tensor([127.0]), k, k * (1 + 2 ** -23), k * (1 - 2 ** -23)]).view(1, -1)
    same_rows(quantize_rows(x.cuda()), x)
    x = x * 0.3
    same_rows(quantize_rows(x.cuda()), x)


@pytest.mark.gpu
def test_quantize_strides_and_no_rows():
    from mpnn_amd import quantize_rows
    x = randn(40, 70, seed=1)
    for view in (x.cuda()[:, 3:50], x.cuda().t(), x.cuda()[::2], x.cuda()[:1].expand(9, 70)):
        same_rows(quantize_rows(view), view)
    r = quantize_rows(torch.zeros(0, 5, device="cuda"))
    assert r.shape == (0, 5) and r.dequantize().shape == (0, 5)


def linear_reference(q, s, wq, ws, bias, relu):
    acc = q.double() @ wq.double().t()
    y = acc * s.double().unsqueeze(1) * ws.double()
    bound = 3 * U * y.abs()
    if bias is not None:
        y = y + bias.double()
    bound = bound + U * y.abs()
    return (y.clamp_min(0) if relu else y), bound


def close(got, want, bound):
    dtype = got.dtype
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    tol = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + 1e-40
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol).max()))


LINEAR = [(1, 1, 1), (1, 64, 128), (2, 11, 7), (18, 11, 128), (31, 16, 32), (32, 17, 33), (33, 48, 100), (63, 500, 192),
          (64, 64, 64), (65, 128, 256), (127, 129, 127), (128, 130, 130), (200, 256, 257), (257, 1000, 300), (100, 2048, 40),
          (5, 2048, 2048), (40, 8192, 20), (300, 100, 513), (1000, 64, 64), (515, 320, 640)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", LINEAR)
def test_linear_int8(n, k, m):
    from mpnn_amd import linear_int8, quantize_rows
    x, w, b = randn(n, k, seed=n), randn(m, k, seed=m), randn(m, seed=k)
    wq, ws = quantized(w)
    w8 = quantize_rows(w.cuda())
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype)
        q, s = quantized(xd)
        for out in (torch.float32, torch.bfloat16):
            for bias, relu in ((None, False), (b.to(out), True)):
                want, bound = linear_reference(q, s, wq, ws, bias, relu)
                bd = None if bias is None else bias.cuda()
                got = linear_int8(xd.cuda(), w8, bias=bd, relu=relu, dtype=out)
                assert got.dtype == out
                close(got, want, bound)
                held = linear_int8(quantize_rows(xd.cuda()), w8, bias=bd, relu=relu, dtype=out)
                assert torch.equal(held, got)
    assert linear_int8(x.cuda().bfloat16(), w8).dtype == torch.bfloat16
    assert linear_int8(quantize_rows(x.cuda()), w8).dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(4133, 520, 4091), (4096, 1040, 4160), (3000, 513, 70), (777, 1111, 777), (300, 4099, 130),
                                   (20000, 512, 300), (33, 512, 3000), (1100, 300, 1100), (50000, 500, 192), (70000, 64, 64)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_linear_int8_many_rows(n, k, m, out):
    """Every kernel at sizes with whole and ragged tiles; 64-bit products on the device."""
    from mpnn_amd import linear_int8, quantize_rows
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, k, generator=gen, device="cuda")
    w = torch.randn(m, k, generator=gen, device="cuda")
    b = torch.randn(m, generator=gen, device="cuda").to(out)
    xr, wr = quantize_rows(x), quantize_rows(w)
    want = (xr.values.double() @ wr.values.double().t()) * (xr.scale.double().unsqueeze(1) * wr.scale.double())
    bound = 3 * U * want.abs()
    want = want + b.double()
    bound += U * want.abs()
    bound += torch.finfo(out).eps / 2 * (want.abs() + bound)
    for rows in (x, xr):
        got = linear_int8(rows, wr, bias=b, dtype=out)
        assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(50, 21, 30), (50, 530, 30), (300, 530, 30)])
def test_linear_int8_bytes_behind_the_rows_do_not_count_anywhere(n, k, m):
    from mpnn_amd import Rows8, linear_int8, quantize_rows
    x, w = randn(n, k, seed=1), randn(m, k, seed=2)
    want = linear_int8(x.cuda(), quantize_rows(w.cuda()))
    dirty = []
    for t in (x, w):
        r = quantize_rows(t.cuda())
        store = torch.full((t.size(0), 560), 77, dtype=torch.int8, device="cuda")
        store[:, :k] = r.values
        rows = Rows8(store[:, :k], r.scale)
        assert rows.values.data_ptr() == store.data_ptr()
        dirty.append(rows)
    assert torch.equal(linear_int8(*dirty), want)


@pytest.mark.gpu
def test_linear_int8_layouts_that_cannot_be_read_in_place():
    from mpnn_amd import Rows8, linear_int8, quantize_rows
    x, w = randn(50, 21, seed=1), randn(30, 21, seed=2)
    want = linear_int8(x.cuda(), quantize_rows(w.cuda()))
    # layouts that cannot be read in place are copied: odd pitch, columns of a wider matrix, a last row that ends early
    tight = quantize_rows(w.cuda()).values.contiguous()
    assert tight.stride(0) == 21
    s = quantize_rows(w.cuda()).scale
    for v in (tight, torch.zeros(30, 64, dtype=torch.int8, device="cuda")[:, 3:24].copy_(tight)):
        r = Rows8(v, s)
        assert r.values.data_ptr() != v.data_ptr() and torch.equal(linear_int8(x.cuda(), r), want)
    short = torch.zeros(29 * 32 + 21, dtype=torch.int8, device="cuda").as_strided((30, 21), (32, 1))
    short.copy_(tight)
    r = Rows8(short, s)
    assert r.values.data_ptr() != short.data_ptr() and torch.equal(linear_int8(x.cuda(), r), want)


@pytest.mark.gpu
def test_linear_int8_strides_special_rows_and_no_rows():
    from mpnn_amd import linear_int8, quantize_rows
    w8 = quantize_rows(randn(40, 24, seed=3).cuda())
    x = randn(60, 30, seed=4)
    wide = x.cuda()[:, 5:29]
    assert torch.equal(linear_int8(wide, w8), linear_int8(wide.contiguous(), w8))
    assert torch.equal(linear_int8(x.cuda().t().contiguous().t()[:, 5:29], w8), linear_int8(wide.contiguous(), w8))
    y = wide.contiguous()
    y[7, 3] = float("nan")
    y[9] = 0.0
    y[11, 0] = float("inf")
    got, clean = linear_int8(y, w8), linear_int8(wide, w8)
    assert got[7].isnan().all() and got[11].isnan().all() and not got[9].any()
    assert linear_int8(y, w8, relu=True)[7].isnan().all()
    keep = [i for i in range(60) if i not in (7, 9, 11)]
    assert torch.equal(got[keep], clean[keep])
    assert linear_int8(torch.zeros(0, 24, device="cuda"), w8).shape == (0, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(18, 11, 128), (300, 700, 300), (16384, 520, 1024)])
def test_linear_int8_captured_and_on_another_stream(n, k, m):
    from mpnn_amd import linear_int8, quantize_rows
    x, w8 = randn(n, k, seed=1).cuda(), quantize_rows(randn(m, k, seed=2).cuda())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = linear_int8(x, w8)
    side = torch.cuda.Stream()
    for _ in range(3):
        x.mul_(-1.5)
        want = linear_int8(x, w8)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = linear_int8(x, w8)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(other, want)


@pytest.mark.gpu
def test_linear_int8_refusals():
    from mpnn_amd import Rows8, linear_int8, quantize_rows
    w8 = quantize_rows(randn(8, 16).cuda())
    x = randn(4, 16).cuda()
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_int8(x.clone().requires_grad_(), w8)
    with torch.no_grad():
        linear_int8(x.clone().requires_grad_(), w8)
    with pytest.raises(TypeError):
        linear_int8(x, x)
    with pytest.raises(TypeError):
        linear_int8(x.half(), w8)
    with pytest.raises(TypeError):
        linear_int8(x, w8, dtype=torch.float16)
    for args, kw in (((x[:, :8], w8), {}), ((x, w8), dict(bias=x[0, :7])), ((x, w8), dict(bias=x[0, :8].bfloat16())),
                     ((x[0], w8), {})):
        with pytest.raises(ValueError):
            linear_int8(*args, **kw)
    with pytest.raises(_lib.MpnnError):
        linear_int8(x.cpu(), w8)
    with pytest.raises(ValueError):
        quantize_rows(torch.zeros(2, 8193, device="cuda"))
    with pytest.raises(ValueError):
        Rows8(w8.values, w8.scale[:-1])
    with pytest.raises(ValueError):
        Rows8(w8.values.int(), w8.scale)


# ------------------------------------------------------------------------------------- weight gradient from 8-bit rows
SHAPES = [(1, 1, 1, 0), (1, 64, 64, 0), (5, 2, 3, 0), (16, 32, 128, 0), (17, 33, 127, 0), (127, 31, 129, 0), (128, 64, 64, 64),
          (129, 100, 11, 100), (200, 128, 128, 0), (256, 256, 128, 0), (257, 64, 200, 72), (300, 257, 40, 0), (400, 130, 130, 200),
          (1000, 300, 300, 0), (1500, 96, 64, 0), (64, 600, 20, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,k,k2", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gemm_tn8(n, m, k, k2, dtype):
    from mpnn_amd.rows8 import Rows8, gemm_tn8, quantize_rows, relu_bits
    if dtype == torch.bfloat16:
        m += m % 2
    gen = torch.Generator().manual_seed(n * m)
    y = randn(n, m, seed=n, dtype=dtype)
    is_open = (y > 0).double()
    # whole numbers: equal
    g = torch.randint(-8, 9, (n, m), generator=gen).to(dtype)
    q = [torch.randint(-127, 128, (n, c), generator=gen, dtype=torch.int8) for c in (k, k2) if c]
    rows = [Rows8(v.cuda(), torch.ones(n, device="cuda")) for v in q]
    g_out = torch.full((n, m), 3.0, dtype=dtype, device="cuda")
    bits = relu_bits(y.cuda())
    assert bits.shape == (n, (m + 31) // 32)
    both = torch.cat(q, dim=1).double()
    for b in (None, bits):
        gm = g.double() * (is_open if b is not None else 1.0)
        got = gemm_tn8(g.cuda(), *rows, bits=b, g_out=g_out if b is not None else None)
        want = gm.t() @ both
        assert got.dtype == dtype and torch.equal(got.cpu(), want.to(dtype))
        if b is not None:
            assert torch.equal(g_out.cpu().double(), gm)
    # random values
    g = randn(n, m, seed=7, dtype=dtype)
    xs = [randn(n, c, seed=8 + c) for c in (k, k2) if c]
    rows = [quantize_rows(x.cuda()) for x in xs]
    deq = torch.cat([r.values.cpu().double() * r.scale.cpu().double().unsqueeze(1) for r in rows], dim=1)
    want = g.double().t() @ deq
    size = g.double().abs().t() @ deq.abs()
    per_term = 2 * U if dtype == torch.float32 else 2.0 ** -17 + 2 * U
    got = gemm_tn8(g.cuda(), *rows)
    close(got, want, (per_term + 2 * (768 + 80) * U) * size)
    assert torch.equal(got, gemm_tn8(g.cuda(), *rows))


@pytest.mark.gpu
def test_gemm_tn8_strides_no_rows_and_rows_that_are_not_finite():
    from mpnn_amd.rows8 import gemm_tn8, quantize_rows
    x, g = randn(300, 40, seed=1), randn(300, 50, seed=2)
    r = quantize_rows(x.cuda())
    want = gemm_tn8(g.cuda(), r)
    wide = torch.zeros(300, 61, device="cuda")
    wide[:, 7:57] = g.cuda()
    assert torch.equal(gemm_tn8(wide[:, 7:57], r), want)
    one = gemm_tn8(g[:1].cuda().expand(300, 50), r)
    assert torch.equal(one, gemm_tn8(g[:1].repeat(300, 1).cuda(), r))
    b = g.bfloat16().cuda()
    off = torch.zeros(300, 53, dtype=torch.bfloat16, device="cuda")
    off[:, 1:51] = b
    assert torch.equal(gemm_tn8(off[:, 1:51], r), gemm_tn8(b, r))
    assert torch.equal(gemm_tn8(torch.zeros(0, 50, device="cuda"), quantize_rows(torch.zeros(0, 40, device="cuda"))),
                       torch.zeros(50, 40, device="cuda"))
    # a NaN of g reaches its own row of the result only; a row of x that is not finite reaches everything
    for where in (5, 299):
        bad = g.clone()
        bad[where, 3] = float("nan")
        got = gemm_tn8(bad.cuda(), r)
        assert got[3].isnan().all() and torch.equal(got[[i for i in range(50) if i != 3]], want[[i for i in range(50) if i != 3]])
    xb = x.clone()
    xb[299, 0] = float("inf")
    assert gemm_tn8(g.cuda(), quantize_rows(xb.cuda())).isnan().all()


# ----------------------------------------------------------------------------------------------- the dense products
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,f,h", [(777, 40, 24), (1, 8, 8), (130, 128, 128), (500, 64, 64), (300, 264, 32), (50, 16, 256), (129, 96, 200)])
def test_project_and_update_keep_their_inputs_in_8_bits(n, f, h, dtype):
    """Against 64 bits with the 8-bit rows in the weight gradient's place of the inputs.  Sums of c float32 terms in some
    order: 2 c u times the magnitudes (float32 inputs are cut into three pieces: 3 c terms); bfloat16 gradients of the
    update carry one rounding of g * open, which is exact."""
    from mpnn_amd import quantize_rows
    from mpnn_amd.dense import project, update
    leaf = lambda *s, seed: randn(*s, seed=seed, dtype=dtype).cuda().requires_grad_()
    x, a, w, wo = leaf(n, f, seed=1), leaf(n, h, seed=2), leaf(2 * h, f, seed=3), leaf(h, f + h, seed=4)
    gy, gy2 = randn(n, 2 * h, seed=5, dtype=dtype).cuda(), randn(n, h, seed=6, dtype=dtype).cuda()
    d = lambda t: t.detach().double().cpu()
    deq = lambda t: d(quantize_rows(t.detach()).values) * d(quantize_rows(t.detach()).scale).unsqueeze(1)

    def product(p, q):
        """p @ q and the bound of its error."""
        return p @ q, 2 * 3 * (p.size(1) + 80) * U * (p.abs() @ q.abs()) + 2.0 ** -16 * (0 if dtype == torch.float32 else 1) * (p.abs() @ q.abs())

    kept = project(x, w, checkpoint="int8")
    gx, gw = torch.autograd.grad(kept, (x, w), gy)
    close(kept, *product(d(x), d(w).t()))
    close(gx, *product(d(gy), d(w)))
    close(gw, *product(d(gy).t(), deq(x)))
    brought = project(x, w, checkpoint=quantize_rows(x))
    assert torch.equal(torch.autograd.grad(brought, w, gy)[0], gw)
    assert torch.equal(torch.autograd.grad(project(x, w.detach(), checkpoint="int8"), x, gy)[0], gx)
    (g,) = torch.autograd.grad(project(x, w, checkpoint="int8").sum(), w)       # an expanded upstream gradient
    assert torch.equal(g, torch.autograd.grad(project(x, w, checkpoint="int8"), w, torch.ones_like(gy))[0])

    kept = update(x, a, wo, checkpoint="int8")
    both = torch.cat([d(x), d(a)], dim=1)
    z, bound = product(both, d(wo).t())
    close(kept, z.clamp_min(0), bound)
    gz = d(gy2) * (d(kept) > 0)
    gx, ga, gw = torch.autograd.grad(kept, (x, a, wo), gy2)
    g_in, bound = product(gz, d(wo))
    close(gx, g_in[:, :f], bound[:, :f])
    close(ga, g_in[:, f:], bound[:, f:])
    close(gw, *product(gz.t(), torch.cat([deq(x), deq(a)], dim=1)))
    # with and without each gradient
    for needs in ((0, 1, 0), (1, 0, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1), (1, 1, 0)):
        ins = [t if k else t.detach() for t, k in zip((x, a, wo), needs)]
        part = torch.autograd.grad(update(*ins, checkpoint="int8"), [t for t, k in zip(ins, needs) if k], gy2)
        full = [t for t, k in zip((gx, ga, gw), needs) if k]
        for p, q, k in zip(part, full, [k for k in range(3) if needs[k]]):
            # the forward without a weight gradient may add in another order: its relu is the same unless z is zero to rounding
            if needs[2]:
                assert torch.equal(p, q) or k < 2
            close(p, d(q), 2 * bound.max() + torch.finfo(dtype).eps * d(q).abs())


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,k2,m", [(1, 8, 0, 8), (15, 32, 0, 40), (16, 40, 8, 32), (17, 64, 64, 64), (100, 128, 128, 128),
                                      (129, 256, 0, 64), (300, 256, 256, 56), (1000, 128, 0, 256), (3001, 72, 136, 104), (40000, 128, 128, 128)])
@pytest.mark.parametrize("relu", [False, True])
def test_kept_linear_leaves_what_the_separate_passes_do(n, k, k2, m, relu):
    from mpnn_amd.rows8 import kept_linear, quantize_rows, relu_bits
    x = randn(n, k, seed=n, dtype=torch.bfloat16).cuda()
    x2 = randn(n, k2, seed=n + 1, dtype=torch.bfloat16).cuda() if k2 else None
    w = randn(m, k + k2, seed=n + 2, dtype=torch.bfloat16).cuda()
    if n > 20:
        x[3] = 0
        x[5, 2] = float("inf")
        x[n - 1, k - 1] = float("nan")
    y, r, r2, bits = kept_linear(x, w, x2, relu=relu)
    for rows, t in ((r, x), (r2, x2)):
        if t is not None:
            q = quantize_rows(t)
            assert torch.equal(rows.values, q.values) and torch.equal(rows.scale.nan_to_num(nan=-1), q.scale.nan_to_num(nan=-1))
            assert torch.equal(torch.as_strided(rows.values, (n, rows.pitch), (rows.pitch, 1)), torch.as_strided(q.values, (n, q.pitch), (q.pitch, 1)))
    both = torch.cat([x] + ([x2] if k2 else []), dim=1).double()
    fine = torch.isfinite(both).all(dim=1)
    want = both[fine] @ w.double().t()
    size = both[fine].abs() @ w.double().abs().t()
    want = want.clamp_min(0) if relu else want
    bound = 2 * (k + k2) * U * size
    got = y[fine].double()
    assert bool(((got - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
    if relu:
        assert torch.equal(bits, relu_bits(y))
    else:
        assert bits is None
    if n > 20:
        assert not torch.isfinite(y[5]).all()
        assert y[n - 1].isnan().all()
        assert kept_linear(x.t().contiguous().t(), w, x2) is None          # rows that cannot be read in place


@pytest.mark.gpu
def test_kept_inputs_are_a_quarter():
    """What waits between the passes: the 8-bit rows, their scales and the relu's bits - not the float32 inputs."""
    from mpnn_amd.dense import update
    n, f, h = 4096, 128, 64
    wo = randn(h, f + h, seed=4).cuda().requires_grad_()
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        update(randn(n, f).cuda(), randn(n, h).cuda(), wo, checkpoint="int8")
    assert sum(t.numel() * t.element_size() for t in held) == n * (f + h) + 2 * 4 * n + n * h // 8 + 4 * h * (f + h)


@pytest.mark.gpu
def test_kept_product_against_differences():
    """The input gradient and, with inputs that 8 bits hold exactly, the weight gradient against central differences of
    the 64-bit function."""
    from mpnn_amd.dense import project
    gen = torch.Generator().manual_seed(3)
    x = torch.randint(-127, 128, (30, 16), generator=gen).float()
    x[:, 0] = 127.0
    w, gy = randn(12, 16, seed=1), randn(30, 12, seed=2)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    gx, gw = torch.autograd.grad(project(xd, wd, checkpoint="int8"), (xd, wd), gy.cuda())
    for t, g in ((x, gx), (w, gw)):
        step = torch.randn(t.shape, generator=gen).double()
        value = lambda k: float(((x.double() + (k * step if t is x else 0)) @ (w.double() + (k * step if t is w else 0)).t()
                                 * gy.double()).sum())
        want = (value(1e-3) - value(-1e-3)) / 2e-3          # linear in each: no error but 2^-52 * value / 1e-3
        got = float((g.double().cpu() * step).sum())
        assert abs(got - want) <= 1e-5 * float((g.double().cpu() * step).abs().sum()) + 1e-6


@pytest.mark.gpu
def test_kept_step_captured_and_on_another_stream():
    from mpnn_amd.dense import update
    x, a = randn(1000, 64, seed=1).cuda().requires_grad_(), randn(1000, 64, seed=2).cuda().requires_grad_()
    w, gy = randn(64, 128, seed=3).cuda().requires_grad_(), randn(1000, 64, seed=4).cuda()

    def once():
        y = update(x, a, w, checkpoint="int8")
        return (y.detach(), *torch.autograd.grad(y, (x, a, w), gy))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    graphs, held = [], []
    for _ in range(2):                                     # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(once())
        graphs.append(g)
    for k in range(3):
        with torch.no_grad():
            x.mul_(-1.25)
            gy.mul_(0.5)
        want = once()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for h in held:
            assert all(torch.equal(p, q) for p, q in zip(h, want)), k


@pytest.mark.gpu
def test_checkpoint_refusals():
    from mpnn_amd import quantize_rows
    from mpnn_amd.dense import project, update
    x, w = randn(6, 16).cuda(), randn(8, 16).cuda()
    a, wo = randn(6, 8).cuda(), randn(8, 24).cuda()
    for bad in ("int4", True, 8, quantize_rows(x[:5])):
        with pytest.raises(ValueError):
            project(x, w, checkpoint=bad)
    with pytest.raises(ValueError):
        update(x, a, wo, checkpoint=quantize_rows(x))
    with pytest.raises(ValueError):
        project(x, w[:, :8], checkpoint="int8")
    with pytest.raises(ValueError):
        update(x, a[:5], wo, checkpoint="int8")
    with pytest.raises(ValueError):
        project(torch.zeros(2, 8200, device="cuda"), torch.zeros(8, 8200, device="cuda"), checkpoint="int8")
    xr = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(project(xr, w.requires_grad_(), checkpoint="int8").square().sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), xr)


def test_cpu_tensors_are_refused():
    from mpnn_amd import Rows8, linear_int8, quantize_rows
    from mpnn_amd.dense import project
    x = torch.zeros(4, 16)
    for call in (lambda: quantize_rows(x), lambda: project(x, x, checkpoint="int8"),
                 lambda: linear_int8(x, Rows8(torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)))):
        with pytest.raises(_lib.MpnnError, match="GPU"):
            call()


def test_entry_points_refuse_before_any_launch():
    """Addresses are never followed here: every call is rejected on the host."""
    lib = _lib.load()
    p = 1 << 20
    q = lambda **k: lib.mpnn_quantize_rows(*{**dict(x=p, ldx=16, dt=0, n=4, k=16, q=p, ldq=16, s=p, st=None), **k}.values())
    for bad in (dict(dt=2), dict(n=-1), dict(k=0), dict(k=8193), dict(ldx=15), dict(ldq=15), dict(ldq=24), dict(x=None), dict(q=None),
                dict(s=None), dict(q=p + 8)):
        assert q(**bad) == -1, bad
    assert q(n=0) == 0
    b = lambda **k: lib.mpnn_relu_bits(*{**dict(y=p, ld=16, dt=0, n=4, m=16, b=p, st=None), **k}.values())
    for bad in (dict(dt=3), dict(n=-1), dict(m=0), dict(ld=15), dict(y=None), dict(b=None)):
        assert b(**bad) == -1, bad
    base = dict(x=p, ldx=608, xd=0, xs=None, w=p, ldw=608, ws=p, bias=None, y=p, ldy=8, yd=0, n=4, k=600, m=8, relu=0, space=p, st=None)
    li = lambda **k: lib.mpnn_linear_int8(*{**base, **k}.values())
    for bad in (dict(xd=2), dict(yd=3), dict(n=-1), dict(k=0), dict(k=8193), dict(m=0), dict(ldx=599), dict(ldw=600), dict(ldy=7),
                dict(x=None), dict(w=None), dict(ws=None), dict(y=None), dict(space=None), dict(xd=3), dict(w=p + 4), dict(ldw=612),
                dict(xd=3, xs=p, ldx=612), dict(xd=3, xs=p, x=p + 1), dict(space=p + 4)):
        assert li(**bad) == -1, bad
    assert li(n=0) == 0
    assert lib.mpnn_linear_int8_workspace_bytes(-1, 1, 1, 0) == -1 and lib.mpnn_linear_int8_workspace_bytes(4, 600, 8, 3) == 0
    assert lib.mpnn_linear_int8_workspace_bytes(4, 600, 8, 0) == 4 * 608 + 16 and lib.mpnn_linear_int8_workspace_bytes(4, 16, 8, 0) == 0
    base_t = dict(g=p, ldg=8, dt=0, bits=None, q=p, ldq=16, s=p, k=16, q2=None, ldq2=0, s2=None, k2=0, dw=p, lddw=16, scratch=p,
                  go=None, ldgo=0, n=4, m=8, st=None)
    tn = lambda **k: lib.mpnn_gemm_tn8(*{**base_t, **k}.values())
    for bad in (dict(dt=2), dict(n=-1), dict(m=0), dict(k=0), dict(k2=-1), dict(dw=None), dict(lddw=15), dict(g=None), dict(q=None),
                dict(s=None), dict(n=128, scratch=None), dict(k2=4, lddw=20), dict(ldg=7), dict(ldq=8), dict(go=p, ldgo=7), dict(ldg=1 << 22),
                dict(q=p + 2), dict(ldq=18), dict(dt=1, ldg=9), dict(dt=1, m=7), dict(dt=1, g=p + 2)):
        assert tn(**bad) == -1, bad
    assert lib.mpnn_gemm_tn8_scratch_floats(-1, 8, 8, 0, 0) == -1


# the kernel holds every value as three bfloat16 pieces (exact: 8 + 8 + 8 bits) and leaves out the products second x third,
# third x second and third x third: at most (2 * 2^-7 * 2^-15 + 2^-30) |x w|; six products per pair are added, each
# addition off by at most 2^-23 of a partial sum (a rounding or a truncation)
def kept_f32_bound(k, size):
    return (6 * k * 1.02 * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -30) * size


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,k2,m", [(1, 4, 0, 1), (1, 12, 0, 128), (31, 32, 0, 40), (32, 40, 8, 32), (33, 64, 64, 64), (63, 36, 0, 33),
                                      (65, 24, 20, 96), (100, 128, 64, 64), (129, 60, 124, 64), (257, 128, 128, 64), (500, 252, 0, 37),
                                      (1000, 128, 0, 256), (2049, 20, 100, 100), (3001, 72, 32, 104), (777, 100, 52, 70),
                                      (40000, 64, 64, 64), (70000, 128, 0, 128)])
@pytest.mark.parametrize("relu", [False, True])
def test_kept_linear_in_float32(n, k, k2, m, relu):
    from mpnn_amd.dense import gemm_nt
    from mpnn_amd.rows8 import kept_linear, quantize_rows, relu_bits
    x = randn(n, k, seed=n).cuda()
    x2 = randn(n, k2, seed=n + 1).cuda() if k2 else None
    w = randn(m, k + k2, seed=n + 2).cuda()
    if n > 20:
        x[3] = 0
        x[5, 2] = float("inf")
        x[n - 1, k - 1] = float("nan")
    both = torch.cat([x] + ([x2] if k2 else []), dim=1).double()
    fine = torch.isfinite(both).all(dim=1)
    want = both[fine] @ w.double().t()
    size = both[fine].abs() @ w.double().abs().t()
    want = want.clamp_min(0) if relu else want
    plain = gemm_nt(x, w[:, :k], x2, w[:, k:] if k2 else None, relu=relu)
    wider = torch.zeros((n, k + 8), device="cuda")             # rows inside a wider matrix
    wider[:, 4:k + 4] = x
    for xs in (x, wider[:, 4:k + 4]):
        y, r, r2, bits = kept_linear(xs, w, x2, relu=relu)
        for rows, t in ((r, x), (r2, x2)):
            if t is not None:
                q = quantize_rows(t)
                assert torch.equal(rows.values, q.values) and torch.equal(rows.scale.nan_to_num(nan=-1), q.scale.nan_to_num(nan=-1))
                assert torch.equal(torch.as_strided(rows.values, (n, rows.pitch), (rows.pitch, 1)), torch.as_strided(q.values, (n, q.pitch), (q.pitch, 1)))
        assert bool(((y[fine].double() - want).abs() <= kept_f32_bound(k + k2, size)).all())
        assert torch.equal(y[fine], plain[fine])
        assert torch.equal(bits, relu_bits(y)) if relu else bits is None
        if n > 20:
            assert not torch.isfinite(y[5]).all()
            assert y[n - 1].isnan().all()
    wider[:, 1:k + 1] = x
    assert kept_linear(wider[:, 1:k + 1], w, x2) is None       # off a 16-byte boundary


@pytest.mark.gpu
def test_float32_inputs_that_take_the_separate_passes(monkeypatch):
    from mpnn_amd.dense import project, update
    from mpnn_amd.rows8 import kept_linear
    x, a = randn(300, 128).cuda(), randn(300, 64, seed=1).cuda()
    w = randn(64, 192, seed=2).cuda()
    assert kept_linear(torch.cat([x, x, x], dim=1), torch.cat([w, w], dim=1)) is None       # 384 wide
    assert kept_linear(x[:, :11].contiguous(), w[:, :11].contiguous()) is None
    for mode in (None, "f32"):
        if mode:
            monkeypatch.setenv("MPNN_GEMM", mode)
        assert (kept_linear(x, w, a) is None) == (mode == "f32")
        assert torch.equal(update(x, a, w.requires_grad_(), checkpoint="int8"), update(x, a, w))
        x11, w11 = x[:, :11].contiguous(), w.detach()[:, :11].contiguous().requires_grad_()
        assert torch.equal(project(x11, w11, checkpoint="int8"), project(x11, w11))


def test_kept_linear_refuses_before_any_launch():
    """Addresses are never followed here: every call is rejected on the host."""
    lib = _lib.load()
    p = 1 << 20
    base = dict(x=p, ldx=64, k=64, q=p, ldq=64, s=p, x2=p, ldx2=32, k2=32, q2=p, ldq2=32, s2=p, w=p, ldw=96, y=p, ldy=64, bits=None,
                n=4, m=64, relu=0, dt=0, st=None)
    call = lambda **k: lib.mpnn_kept_linear(*{**base, **k}.values())
    shared = (dict(n=-1), dict(k=0), dict(k2=-1), dict(m=0), dict(dt=2), dict(k=264, ldx=264, ldq=272, ldw=296), dict(m=4104, ldy=4104),
              dict(ldx=60), dict(ldx2=24), dict(ldw=88), dict(ldy=56), dict(ldq=48), dict(ldq2=16), dict(q=p + 8), dict(ldq=72), dict(ldq2=40),
              dict(x=None), dict(q=None), dict(s=None), dict(x2=None), dict(q2=None), dict(s2=None), dict(w=None), dict(y=None),
              dict(x=p + 4), dict(x2=p + 8))
    for bad in shared + (dict(k=62), dict(k2=30), dict(ldx=66), dict(ldx2=34), dict(m=1024, ldy=1024)):
        assert call(**bad) == -1, bad
    for bad in shared + (dict(k=60), dict(m=60), dict(ldx=68), dict(ldw=100), dict(ldy=68), dict(w=p + 2), dict(y=p + 8)):
        assert call(**{**bad, "dt": bad.get("dt", 1)}) == -1, bad
    assert call(n=0) == 0 and call(n=0, dt=1) == 0
    assert lib.mpnn_kept_linear_fits(128, 0, 256, 0) == 1 and lib.mpnn_kept_linear_fits(128, 128, 128, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40, 500])
def test_saved_rows_that_come_back_in_another_layout(n):
    """A hook that moves what waits for the backward to the host returns it without the padding behind its rows."""
    from mpnn_amd.dense import project, update
    x, a = randn(n, 100).cuda().requires_grad_(), randn(n, 37, seed=1).cuda().requires_grad_()
    w, wo = randn(64, 100, seed=2).cuda().requires_grad_(), randn(50, 137, seed=3).cuda().requires_grad_()

    def grads():
        y, z = project(x, w, checkpoint="int8"), update(x, a, wo, checkpoint="int8")
        return lambda: torch.autograd.grad([y, z], [x, a, w, wo], [torch.ones_like(y), torch.ones_like(z)])
    want = grads()()
    with torch.autograd.graph.save_on_cpu():
        later = grads()
    for p, q in zip(later(), want):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_weights_with_many_rows_and_few_rows_of_x():
    from mpnn_amd.dense import project
    m = 262148                                            # more blocks than one grid dimension of 65,535 takes
    x, w = randn(3, 4).cuda(), randn(m, 4, seed=1).cuda().requires_grad_()
    g = randn(3, m, seed=2).cuda()
    (gw,) = torch.autograd.grad(project(x, w, checkpoint="int8"), [w], g)
    from mpnn_amd.rows8 import quantize_rows
    want = g.double().t() @ quantize_rows(x).dequantize(torch.float32).double()
    size = g.double().abs().t() @ x.double().abs()
    # three products of once rounded factors (scale, g * scale; q is exact) and their sums
    assert bool(((gw.double() - want).abs() <= 6 * 2.0 ** -24 * size + 1e-30).all())


@pytest.mark.gpu
def test_kept_rows_only_where_something_waits():
    from mpnn_amd.dense import project, update
    x, a = randn(300, 64).cuda(), randn(300, 32, seed=1).cuda()
    w, wo = randn(64, 64, seed=2).cuda().requires_grad_(), randn(32, 96, seed=3).cuda().requires_grad_()
    with torch.no_grad():
        y, z = project(x, w, checkpoint="int8"), update(x, a, wo, checkpoint="int8")
    assert not y.requires_grad and not z.requires_grad
    assert torch.equal(y, project(x, w, checkpoint="int8")) and torch.equal(z, update(x, a, wo, checkpoint="int8"))
    big = torch.empty(1, device="cuda").expand((1 << 21) + 1, 64)
    with pytest.raises(ValueError, match="at most"):
        project(x, big, checkpoint="int8")


@pytest.mark.gpu
def test_kept_calls_with_expanded_inputs():
    from mpnn_amd.dense import project, update
    row, a = randn(1, 64).cuda().requires_grad_(), randn(200, 32, seed=1).cuda()
    w, wo = randn(48, 64, seed=2).cuda().requires_grad_(), randn(32, 96, seed=3).cuda().requires_grad_()
    x = row.expand(200, 64)
    for f, full in ((lambda t: project(t, w, checkpoint="int8"), w), (lambda t: update(t, a, wo, checkpoint="int8"), wo)):
        y, y_full = f(x), f(x.contiguous())
        assert torch.equal(y, y_full)
        g = torch.ones_like(y)
        for p, q in zip(torch.autograd.grad(y, [row, full], g), torch.autograd.grad(y_full, [row, full], g)):
            assert torch.equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(1, 4, 1), (31, 32, 40), (33, 64, 11), (100, 128, 11), (129, 128, 64), (500, 124, 33), (1000, 100, 100),
                                   (4099, 64, 128), (40000, 128, 128), (9000, 96, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_input_gradient_from_the_weight_as_it_lies(n, k, m, dtype):
    from mpnn_amd.dense import gemm_nt
    from mpnn_amd.rows8 import gemm_nn
    bf = dtype == torch.bfloat16
    if bf:
        k, m = (k + 7) // 8 * 8, (m + 7) // 8 * 8
    g, w = randn(n, k, seed=n, dtype=dtype).cuda(), randn(k, m, seed=n + 1, dtype=dtype).cuda()
    wider = torch.zeros((k, m + 5), dtype=dtype, device="cuda")       # a column slice of a wider weight, at any alignment
    wider[:, 3:m + 3] = w
    gw = torch.zeros((n, k + 8), dtype=dtype, device="cuda")
    gw[:, :k] = g
    if n > 20:
        g[7, 1] = float("inf")
        gw[7, 1] = float("inf")
    fine = torch.isfinite(g).all(dim=1)
    want, size = g[fine].double() @ w.double(), g[fine].double().abs() @ w.double().abs()
    for gs, ws in ((g, w), (gw[:, :k], wider[:, 3:m + 3])):
        y = gemm_nn(gs, ws)
        if bf:
            bound = 2 * k * U * size
            assert bool(((y[fine].double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
        else:
            assert bool(((y[fine].double() - want).abs() <= kept_f32_bound(k, size)).all())
            assert torch.equal(y[fine], gemm_nt(g, w.t().contiguous())[fine])
        assert n <= 20 or not torch.isfinite(y[7]).any()
    assert gemm_nn(g[:, 1:], w[1:]) is None                           # off a 16-byte boundary, and a width that does not fit
    assert bf or gemm_nn(torch.ones((n, 256), device="cuda"), torch.ones((256, m), device="cuda")) is None


def test_gemm_nn_refuses_before_any_launch():
    """Addresses are never followed here: every call is rejected on the host."""
    lib = _lib.load()
    p = 1 << 20
    base = dict(x=p, ldx=64, w=p, ldw=40, y=p, ldy=40, n=4, k=64, m=40, dt=0, st=None)
    call = lambda **k: lib.mpnn_gemm_nn(*{**base, **k}.values())
    for bad in (dict(n=-1), dict(k=0), dict(m=0), dict(k=62), dict(k=264, ldx=264), dict(dt=2), dict(ldx=60), dict(ldw=39), dict(ldy=39),
                dict(x=None), dict(w=None), dict(y=None), dict(x=p + 4), dict(ldx=66), dict(dt=1, y=p + 8), dict(dt=1, ldy=44),
                dict(dt=1, ldx=68), dict(dt=1, m=36), dict(k=128, ldx=128, m=4096, ldw=4096, ldy=4096)):
        assert call(**bad) == -1, bad
    assert call(n=0) == 0 and call(n=0, dt=1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(300, 100, 100), (65, 500, 36), (33, 4, 12), (200, 252, 50), (300, 600, 300), (513, 1020, 1004)])
@pytest.mark.parametrize("first", [0, 4, 2])
def test_rows_on_8_byte_boundaries(n, k, m, first):
    """Widths and addresses that allow 8 bytes at a time but not 16 (and, first = 2, neither in bfloat16)."""
    from mpnn_amd import linear_int8, quantize_rows
    w, b = randn(m, k, seed=m), randn(m, seed=k)
    wq, ws = quantized(w)
    w8 = quantize_rows(w.cuda())
    for dtype in (torch.float32, torch.bfloat16):
        wider = torch.full((n, k + 8), float("nan"), dtype=dtype)
        wider[:, first:first + k] = randn(n, k, seed=n).to(dtype)
        x = wider.cuda()[:, first:first + k]
        q, s = quantized(wider[:, first:first + k])
        same_rows(quantize_rows(x), x)
        for out in (torch.float32, torch.bfloat16):
            want, bound = linear_reference(q, s, wq, ws, b.to(out), True)
            close(linear_int8(x, w8, bias=b.to(out).cuda(), relu=True, dtype=out), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kept_calls_without_rows_with_one_input_twice_and_a_transposed_weight(dtype):
    from mpnn_amd.dense import project, update
    wt, wot = randn(64, 32, seed=1, dtype=dtype).cuda(), randn(128, 32, seed=2, dtype=dtype).cuda()
    for n in (0, 1, 500):
        x = randn(n, 64, seed=3, dtype=dtype).cuda().requires_grad_()
        for f, w in ((lambda w: project(x, w, checkpoint="int8"), wt), (lambda w: update(x, x, w, checkpoint="int8"), wot)):
            got = []
            for v in (w.t(), w.t().contiguous()):                     # [32, 64], [32, 128]
                v = v.detach().requires_grad_()
                y = f(v)
                assert y.shape == (n, 32)
                got.append((y.detach(), *torch.autograd.grad(y, (x, v), torch.ones_like(y))))
            # a transposed weight takes the general product, whose sums may run in another order: some 10 units in size here, each
            # off by at most 128 * 2^-24 of 64, and one rounding to the type
            for p, q in zip(*got):
                assert bool(((p.double() - q.double()).abs() <= 4 * torch.finfo(dtype).eps * (q.double().abs() + 64)).all())
            assert n > 0 or not got[0][2].any()
        y = update(x, x, wot.t().contiguous().requires_grad_(), checkpoint="int8")
        (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        z = [x.detach().clone().requires_grad_() for _ in range(2)]
        ga, gb = torch.autograd.grad(update(z[0], z[1], wot.t().contiguous().requires_grad_(), checkpoint="int8"), z, torch.ones_like(y))
        assert torch.equal(gx, ga + gb)
