"""linear_int8 over its whole documented range of sizes: the plan of every launch fits a CU's LDS, and the widest heads answer a
few rows."""
import pytest
import torch

from mpnn_amd import _lib

U = 2.0 ** -24


def test_every_plan_fits_the_lds_of_a_cu():
    """On the host: every number of outputs up to 2^20 in steps of 32 (and one above), every form of the kernels."""
    size = _lib.load().mpnn_linear_int8_lds_bytes
    most = 160 * 1024
    for k in (64, 128, 256, 300, 512, 513, 8192):
        for n in (1, 32, 33, 100, 4096, 4097, 1000000):
            for out in (_lib.MPNN_F32, _lib.MPNN_BF16):
                worst = max(size(n, k, m, out) for m in range(32, (1 << 20) + 1, 32))
                assert 0 < worst <= most, (k, n, out, worst)
                assert size(n, k, 57345, out) <= most and size(n, k, 1, out) > 0
    for bad in ((-1, 8, 8, 0), (1, 0, 8, 0), (1, 8193, 8, 0), (1, 8, 0, 0), (1, 8, (1 << 20) + 1, 0), (1, 8, 8, 2)):
        assert size(*bad) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 32])
@pytest.mark.parametrize("k", [300, 512])
@pytest.mark.parametrize("m", [57344, 57345, 128256])
def test_few_rows_against_a_wide_head(n, k, m):
    """Sums of whole numbers are exact; the scales, their application and the bias round once each."""
    from mpnn_amd import linear_int8, quantize_rows
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    x, w = (torch.randn(r, k, generator=gen, device="cuda") for r in (n, m))
    b = torch.randn(m, generator=gen, device="cuda")
    xr, wr = quantize_rows(x), quantize_rows(w)
    exact = (xr.values.double() @ wr.values.double().t()) * (xr.scale.double().unsqueeze(1) * wr.scale.double())
    for out in (torch.float32, torch.bfloat16):
        bias = b.to(out)
        want = exact + bias.double()
        bound = 3 * U * exact.abs() + U * want.abs()
        bound = bound + torch.finfo(out).eps / 2 * (want.abs() + bound)
        first = None
        for rows in (x, xr):
            got = linear_int8(rows, wr, bias=bias, dtype=out)
            assert got.shape == (n, m) and bool(((got.double() - want).abs() <= bound).all())
            first = got if first is None else first
            assert torch.equal(got, first)


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", [(5, 64, 40), (40, 8192, 70)])
def test_scales_whose_product_leaves_the_range_of_float32(n, k, m):
    """A sum of zero stays zero where scale times scale would be infinite, and a result inside float32's range keeps its digits where
    scale times scale would be denormal: what the definition's factors make of it in 64 bits, three roundings off at most."""
    from mpnn_amd import linear_int8, quantize_rows
    U = 2.0 ** -24
    x = torch.zeros(n, k)
    w = torch.zeros(m, k)
    x[:, 0], w[:, 1] = 3e38, 1e5                      # disjoint columns: every sum is 0
    xs, ws = (t[0, c] / 127 for t, c in ((x, 0), (w, 1)))
    assert not torch.isfinite(xs * ws)
    b = torch.arange(m).float()
    assert torch.equal(linear_int8(x.cuda(), quantize_rows(w.cuda()), bias=b.cuda()).cpu(), b.expand(n, m))
    gen = torch.Generator().manual_seed(m)
    for up, down in ((2.0 ** -60, 2.0 ** -66), (2.0 ** -66, 2.0 ** -60), (2.0 ** 100, 2.0 ** -100), (2.0 ** -100, 2.0 ** 100),
                     (2.0 ** 120, 2.0 ** -90), (2.0 ** -90, 2.0 ** 120)):
        xr = quantize_rows((up * torch.rand(n, k, generator=gen)).cuda())
        wr = quantize_rows((down * torch.rand(m, k, generator=gen)).cuda())
        want = (xr.values.double() @ wr.values.double().t()) * xr.scale.double().unsqueeze(1) * wr.scale.double()
        got = linear_int8(xr, wr).double()
        # (the smallest step of float32's range, where the result itself lies below it)
        assert bool(((got - want).abs() <= 3.01 * U * want.abs() + 2.0 ** -149).all()), (up, down)


def test_every_operand_that_wants_a_gradient_is_refused():
    """On the host, before any device is asked for: a bias or a scale whose gradient would be dropped, not x alone."""
    from mpnn_amd import Rows8, linear_int8
    rows = lambda n, grad=False: Rows8(torch.zeros(n, 16, dtype=torch.int8), torch.ones(n, requires_grad=grad))
    x, b = torch.zeros(4, 16), torch.zeros(8)
    wanted = (((x.clone().requires_grad_(), rows(8)), {}), ((x, rows(8)), dict(bias=b.clone().requires_grad_())), ((x, rows(8, True)), {}),
              ((rows(4, True), rows(8)), {}), ((rows(4), rows(8)), dict(bias=torch.nn.Parameter(b))))
    for args, kw in wanted:
        with pytest.raises(RuntimeError, match="no gradient"):
            linear_int8(*args, **kw)
        with torch.no_grad(), pytest.raises(_lib.MpnnError, match="GPU"):      # as far as a host without a GPU gets
            linear_int8(*args, **kw)
