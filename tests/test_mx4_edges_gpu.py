"""4-bit products at the ends of the scales' range and bias gradients of long batches, on the GPU against 64 bits."""
import numpy as np
import pytest
import torch

from tests import mx4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows', [8192, 8193, 8200, 16384, 16400, 128 * 8192 + 70])
@pytest.mark.parametrize('n', [1, 5, 130])
def test_bias_gradients_of_long_batches(rows, n, dtype):
    """One, two and three passes over the sums of 64 rows.  Whole numbers: sums of 64 rows stay below 2^24 (exact in 32 bits), all further ones
    below 2^53 (exact in 64), so the result is the exact sum rounded once.  Groups of 8192 rows sum to about 2^25 in turns of sign: rounded
    to 32 bits in between, they would not cancel to what is left."""
    from deepipr_amd import mx4
    if n == 130 and rows > 100000:
        rows = 3 * 8192 + 100
    g = torch.Generator(device=DEV).manual_seed(rows + n)
    dy = torch.randint(-8, 9, (rows, n), generator=g, device=DEV).float()
    r = torch.arange(rows, device=DEV)
    big = torch.where(r // 8192 % 2 == 0, 32768.0, -32768.0) * (r % 64 < 8)
    dy = torch.where(big[:, None] != 0, big[:, None], dy)
    dy = dy.to(dtype)
    assert torch.equal(dy.float().double().sum(0), dy.double().sum(0))
    bias = torch.zeros(n, device=DEV, requires_grad=True)
    y = mx4.linear(torch.ones(rows, 3, dtype=dtype, device=DEV), torch.ones(n, 3, dtype=dtype, device=DEV), bias)
    got, = torch.autograd.grad(y, bias, dy)
    assert torch.equal(got, dy.double().sum(0).float())


def _at_scales(rows, cols, seed, exponents, positive=False):
    """Values on the 4-bit grid, the blocks of 32 columns at 2^exponents (in turn); each block of a row holds a 6."""
    g = torch.Generator().manual_seed(seed)
    x = torch.tensor(oracle.VALUES)[torch.randint(0, 8, (rows, cols), generator=g)]
    if not positive:
        x = x * (torch.randint(0, 2, (rows, cols), generator=g) * 2 - 1)
    x[:, ::32] = 6.0
    e = torch.tensor(exponents, dtype=torch.float64).repeat(-(-cols // (32 * len(exponents))))[:-(-cols // 32)]
    return (x * torch.exp2(e).repeat_interleave(32)[:cols]).float()


# few rows, quantised inside the product and not; 64 x 32 and 64 x 64 tiles; 128 x 128 tiles, whole and with the columns shared out; 256 x 256
EDGE_SHAPES = [(1, 40, 100), (16, 33, 1000), (40, 70, 700), (100, 500, 3000), (250, 4000, 3000), (300, 520, 640), (128, 128, 20000), (4104, 4096, 4100)]


@pytest.mark.parametrize('mnk', EDGE_SHAPES)
def test_products_of_opposite_ends_are_exact(mnk):
    """A block at the lowest scale times one at the highest: every product is a multiple of 2^-4 (2^-2 times quarters), every partial sum below
    2^20: exact in 32 bits, whatever lies between."""
    from deepipr_amd import mx4
    m, n, k = mnk
    low = [-127, 125, -127, 0, -100, 64, -126, 125]
    high = [125, -127, 124, -1, 99, -65, 124, -126]
    a, b = _at_scales(m, k, 1, low).to(DEV), _at_scales(n, k, 2, high).to(DEV)
    qa, qb = mx4.quantize(a), mx4.quantize(b)
    assert torch.equal(qa.dequantize(), a) and torch.equal(qb.dequantize(), b)
    want = torch.mm(a.double(), b.double().t().contiguous())
    assert torch.equal(mx4.matmul(qa, qb), want.float())
    assert torch.equal(mx4.linear(a, qb), want.float())


@pytest.mark.parametrize('mnk', EDGE_SHAPES)
def test_products_past_the_range(mnk):
    """Beyond the largest float: infinity.  Below the smallest normal one: at most that far off for each of the K products (whether subnormal
    products are kept is the matrix instruction's)."""
    from deepipr_amd import mx4
    m, n, k = mnk
    top = mx4.quantize(_at_scales(m, k, 3, [125], True).to(DEV))
    assert bool((mx4.matmul(top, mx4.quantize(_at_scales(n, k, 4, [125], True).to(DEV))) == float('inf')).all())
    assert bool((mx4.matmul(top, mx4.quantize(-_at_scales(n, k, 4, [125], True).to(DEV))) == float('-inf')).all())
    # the largest sums that fit: K products of at most 36 * 2^s
    s = 127 - int(np.ceil(np.log2(36.0 * k)))
    a, b = _at_scales(m, k, 5, [125], True).to(DEV), _at_scales(n, k, 6, [s - 125], True).to(DEV)
    got, want = mx4.matmul(mx4.quantize(a), mx4.quantize(b)), torch.mm(a.double(), b.double().t().contiguous())
    assert bool(((got.double() - want).abs() <= want.abs() * (k + 1) * 2.0 ** -23).all())
    for ea, eb in ((-127, -127), (-127, 0), (-63, -63), (-64, -64), (-70, -62), (-100, -40)):
        a, b = _at_scales(m, k, 7, [ea]).to(DEV), _at_scales(n, k, 8, [eb]).to(DEV)
        got = mx4.matmul(mx4.quantize(a), mx4.quantize(b)).double()
        want = torch.mm(a.double(), b.double().t().contiguous())
        room = torch.mm(a.double().abs(), b.double().abs().t().contiguous()) * (k * 2.0 ** -23) + k * 2.0 ** -126
        assert bool(((got - want).abs() <= room).all()), (ea, eb)


@pytest.mark.parametrize('xt', TYPES)
@pytest.mark.parametrize('wt', TYPES)
def test_input_weight_and_bias_of_different_types(xt, wt):
    """Quantised in one launch only where the types are the same; every output in its own input's type, equal to the product of its parts."""
    from deepipr_amd import mx4
    g = torch.Generator(device=DEV).manual_seed(4)
    for m, n, k in ((3, 40, 70), (300, 200, 500)):
        x = torch.randn(m, k, generator=g, device=DEV).to(xt).requires_grad_()
        w = torch.randn(n, k, generator=g, device=DEV).to(wt).requires_grad_()
        for bt in TYPES:
            b = torch.randn(n, generator=g, device=DEV).to(bt).requires_grad_()
            y = mx4.linear(x, w, b)
            dy = torch.randn(m, n, generator=g, device=DEV).to(xt)
            dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
            assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (xt, xt, wt, bt)
            qx, qw, qy = mx4.quantize_both(x), mx4.quantize_both(w), mx4.quantize_both(dy)
            assert torch.equal(y, mx4.matmul(qx[0], qw[0], b.detach(), xt))
            assert torch.equal(dx, mx4.matmul(qy[0], qw[1], dtype=xt)) and torch.equal(dw, mx4.matmul(qy[1], qx[1], dtype=wt))
            exact = dy.double().sum(0)
            # sums of 32 and 64 rows in 32 bits, one rounding to 32 and one to the bias's type
            assert bool(((db.double() - exact).abs() <= 66 * 2.0 ** -24 * dy.double().abs().sum(0) + exact.abs() * torch.finfo(bt).eps / 2 * 1.001).all())
            with torch.no_grad():
                assert torch.equal(mx4.linear(x, w, b), y) and torch.equal(mx4.linear(x, qw[0], b), y)
            for keep in range(3):                                    # one gradient alone: other directions, other launches
                args = [t if i == keep else t.detach() for i, t in enumerate((x, w, b))]
                got, = torch.autograd.grad(mx4.linear(*args), args[keep], dy)
                assert torch.equal(got, (dx, dw, db)[keep])
