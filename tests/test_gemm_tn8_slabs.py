"""The weight gradient from 8-bit rows where a block walks many slabs of 128 rows: the next slab on its way while one is multiplied, two
sets of LDS in turn, float32 sums folded every 8 slabs.  Against 64-bit products on the device.

Whole numbers times powers of two are exact: g * scale has at most 5 bits, products at most 12, and sums of N random terms of size 2^10
or less stay far below 2^23 halves (a walk of 700,000 steps of at most 2032, of 300 on average, ends within some 10^6), so every order
of additions gives the same float32 number, rounded once to the type.

Random values: as in the tests of single slabs, with d additions in a row at most 2 d u times the sum of the magnitudes.  float32 adds
3 products per row for 1024 rows, then folds (one addition per 8 slabs), shares, and blocks: d <= 3 * 1024 + 20 + 8 + 80.  bfloat16 adds
2 products per row over all of a block's rows: d <= 2 * 128 * slabs + 88.  A slab that is lost or counted twice is off by some 1 / 20 of a
row's whole, a hundred times that."""
import pytest
import torch

U = 2.0 ** -24
SLABS = 20

# M, K, K2: every way the kernel shares strips, column tiles and rows among its waves, and outputs of many tiles
FORMS = [(32, 64, 0), (31, 100, 60), (64, 128, 0), (64, 40, 128), (100, 128, 0), (128, 128, 128), (130, 100, 0), (250, 64, 130), (256, 128, 0),
         (300, 96, 0), (520, 300, 200)]


def blocks(n, m, k, k2, bf16):
    """Blocks of a launch and slabs of the rows (the plan's own numbers: its scratch holds one tile of M x K per block)."""
    from mpnn_amd import _lib
    floats = _lib.load().mpnn_gemm_tn8_scratch_floats(n, m, k, k2, int(bf16))
    return floats // (m * (k + k2)), (n + 127) // 128


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,k2", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_slabs_per_block(m, k, k2, dtype):
    from mpnn_amd.rows8 import Rows8, gemm_tn8, quantize_rows, relu_bits
    bf = dtype == torch.bfloat16
    m += m % 2 if bf else 0
    per_launch, _ = blocks(1 << 20, m, k, k2, bf)
    n = SLABS * per_launch * 128 + 77                     # one more, ragged: it overlaps the one before
    assert blocks(n, m, k, k2, bf) == (per_launch, SLABS * per_launch + 1)
    gen = torch.Generator(device="cuda").manual_seed(m * k + k2)
    ints = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=gen, device="cuda")
    y = torch.randn(n, m, generator=gen, device="cuda").to(dtype)
    bits = relu_bits(y)
    g = ints(-8, 9, n, m).to(dtype)
    rows = []
    for c in (k, k2):
        if c:
            rows.append(Rows8(ints(-127, 128, n, c).to(torch.int8), torch.tensor([0.0, 0.5, 1.0, 2.0], device="cuda")[ints(0, 4, n)]))
    both = torch.cat([r.values.double() * r.scale.double().unsqueeze(1) for r in rows], dim=1)
    out = torch.full((n, m), 3.0, dtype=dtype, device="cuda")
    for b in (None, bits):
        gm = g if b is None else torch.where(y > 0, g, torch.zeros((), dtype=dtype, device="cuda"))
        want = (gm.double().t() @ both).to(dtype)
        got = gemm_tn8(g, *rows, bits=b, g_out=None if b is None else out)
        assert torch.equal(got, want), float((got.double() - want.double()).abs().max())
        if b is not None:
            assert torch.equal(out, gm)
        assert torch.equal(got, gemm_tn8(g, *rows, bits=b))
    del both
    # random values, scales of every size
    g = torch.randn(n, m, generator=gen, device="cuda").to(dtype)
    rows = [quantize_rows(torch.randn(n, c, generator=gen, device="cuda") * torch.exp(2 * torch.randn(n, 1, generator=gen, device="cuda")))
            for c in (k, k2) if c]
    both = torch.cat([r.values.double() * r.scale.double().unsqueeze(1) for r in rows], dim=1)
    want, size = g.double().t() @ both, g.double().abs().t() @ both.abs()
    per_term, d = (2.0 ** -17 + 2 * U, 2 * 128 * (SLABS + 1) + 88) if bf else (2 * U, 3 * 1024 + 20 + 8 + 80)
    bound = (per_term + 2 * d * U) * size
    bound = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound)
    got = gemm_tn8(g, *rows)
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_large_kept_step_gives_the_same_bits_again(dtype):
    from mpnn_amd.dense import update
    n, h = 700001, 128
    gen = torch.Generator(device="cuda").manual_seed(5)
    leaf = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype).requires_grad_()
    x, a, w, gy = leaf(n, h), leaf(n, h), leaf(h, 2 * h), leaf(n, h).detach()

    def once():
        y = update(x, a, w, checkpoint="int8")
        return (y.detach(), *torch.autograd.grad(y, (x, a, w), gy))
    first = once()
    for _ in range(3):
        junk = torch.randn(1 << 22, generator=gen, device="cuda").sum()      # other work between
        assert all(torch.equal(p, q) for p, q in zip(first, once())), junk
