"""4-bit matrices on the GPU against the 64-bit definition (tests/mx4_oracle.py).

Quantisation is exact: codes, scales and values have to be equal.  Products: where every partial sum is a multiple of one power of two
and below 2^24 times it, 32-bit sums are exact in any order and the outputs have to be equal; elsewhere each of the K additions is off by
at most one step (2^-23) of a partial sum that is at most sum |a||b|, and the output is rounded once (eps / 2)."""
import numpy as np
import pytest
import torch

from tests import mx4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (1, 32), (3, 33), (33, 3), (64, 128), (65, 129), (63, 127), (200, 300), (1, 9216), (130, 31), (257, 1000), (1000, 96), (192, 261), (130, 391)]


def _random(shape, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    if spread:
        x = x * torch.exp2(torch.randint(-8, 8, shape[:1] + (1,) * (len(shape) - 1), generator=g).double())
    return x.to(dtype).to(DEV)


def _same(got, want):
    return np.array_equal(got, want, equal_nan=True)


def _check(q, x, dim):
    a = oracle.to64(x)
    a = a if dim == 1 else np.ascontiguousarray(a.T)
    code, scale, val = oracle.quantise(a)
    got_code, got_scale, clean = oracle.unpack(q.codes, q.scales, q.rows, q.cols)
    assert q.shape == x.shape and (q.rows, q.cols) == a.shape and clean
    assert np.array_equal(got_scale, scale)
    fine = np.repeat(scale != 255, 32, axis=1)[:, :a.shape[1]]
    assert np.array_equal(got_code[fine], code[fine])
    assert _same(oracle.to64(q.dequantize()), val if dim == 1 else val.T)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_quantise(shape, dtype):
    from deepipr_amd import mx4
    x = _random(shape, dtype, seed=shape[0] + shape[1])
    for dim in (0, 1):
        _check(mx4.quantize(x, dim), x, dim)
    along, down = mx4.quantize_both(x)
    _check(along, x, 1)
    _check(down, x, 0)


@pytest.mark.parametrize('dtype', TYPES)
def test_every_rounding_and_border(dtype):
    """Every value of a fine grid over [-8, 8] times powers of two, the largest of its block in each binade position."""
    from deepipr_amd import mx4
    grid = torch.arange(-127, 128, dtype=torch.float64) / 16
    rows = []
    for top in (4.0, 5.0, 6.0, 7.9375):
        for e in (-10, 0, 3):
            v = grid[grid.abs() <= top]
            v = torch.cat([v, torch.zeros(-len(v) % 31, dtype=torch.float64)]).reshape(-1, 31)
            rows.append(torch.cat([torch.full((len(v), 1), top, dtype=torch.float64), v], 1) * 2.0 ** e)
    x = torch.cat(rows).to(dtype).to(DEV)
    for dim in (0, 1):
        y = x if dim == 1 else x.t().contiguous()
        _check(mx4.quantize(y, dim), y, dim)


def test_ends_of_the_range():
    """Zeros of both signs, subnormals, the largest finite values, blocks whose scale is at its lower end."""
    from deepipr_amd import mx4
    tiny = 2.0 ** -149
    rows = [[0.0] * 32, [-0.0] * 32, [tiny] * 32, [2.0 ** -127] * 31 + [3 * 2.0 ** -129], [2.0 ** -126, 2.0 ** -128, 2.0 ** -129, 2.0 ** -130] * 8,
            [3.4028234663852886e38, 1e30, 2.0 ** 125, 2.0 ** 123] * 8, [1e-38 * i for i in range(32)], [2.0 ** -125 * i / 7 for i in range(32)]]
    x = torch.tensor(rows, dtype=torch.float64).float().to(DEV)
    _check(mx4.quantize(x, 1), x, 1)
    _check(mx4.quantize(x.t().contiguous(), 0), x.t().contiguous(), 0)
    h = torch.tensor([[65504.0, 2.0 ** -24, 1.0, -3.0] * 8, [2.0 ** -24] * 32, [2.0 ** -15, 2.0 ** -20] * 16], dtype=torch.float16, device=DEV)
    _check(mx4.quantize(h, 1), h, 1)
    b = torch.tensor([[3.38e38, -1e-40] * 16, [1e-40] * 32], dtype=torch.bfloat16, device=DEV)
    _check(mx4.quantize(b, 1), b, 1)


@pytest.mark.parametrize('dtype', TYPES)
def test_values_that_are_not_numbers_stay_in_their_block(dtype):
    from deepipr_amd import mx4
    x = _random((70, 200), dtype, seed=1)
    x[3, 40] = float('nan')
    x[66, 199] = float('inf')
    x[0, 0] = float('-inf')
    x[5, 64:96] = float('inf')
    for dim in (0, 1):
        _check(mx4.quantize(x, dim), x, dim)


@pytest.mark.parametrize('dtype', TYPES)
def test_strides_and_alignment(dtype):
    """Row strides, starts off the 16-byte grid, transposed matrices."""
    from deepipr_amd import mx4
    big = _random((140, 400), dtype, seed=2)
    for x in (big[:, :300], big[5:, 3:260], big[:, 1:], big[::2, 7:], big[:1, 3:200], big.t(), big[:, :130].t(), big[:7].t(), big[:, :1], big[:, 1:2], big[3:4].t()):
        for dim in (0, 1):
            _check(mx4.quantize(x, dim), x, dim)
        along, down = mx4.quantize_both(x)
        _check(along, x, 1)
        _check(down, x, 0)


def test_dequantise_types_and_refusals():
    from deepipr_amd import mx4
    x = _random((67, 203), torch.float32, seed=3)
    for dim in (0, 1):
        q = mx4.quantize(x, dim)
        val = torch.from_numpy(np.ascontiguousarray(oracle.values(x, dim)))
        for t in TYPES:
            got = q.dequantize(t)
            assert got.dtype == t and got.is_contiguous() and torch.equal(got.cpu(), val.to(t))
    for bad in (x[:, ::2], x[:, :1].expand(67, 5), x.double(), x.int()):
        with pytest.raises(RuntimeError):
            mx4.quantize(bad)
    with pytest.raises(RuntimeError, match='float32, bfloat16 and float16'):
        q.dequantize(torch.float64)
    for shape in ((0, 5), (5, 0), (0, 0)):
        for q in (mx4.quantize(x.new_zeros(shape), 0),) + mx4.quantize_both(x.new_zeros(shape)):
            assert q.shape == shape and q.dequantize().shape == shape


def _codes(rows, cols, seed, scales=(-1, 0, 1)):
    """A float matrix whose values are MX4 values already: every block's largest magnitude is 4 or 6 times its scale."""
    g = torch.Generator().manual_seed(seed)
    mag = torch.tensor(oracle.VALUES)[torch.randint(0, 8, (rows, cols), generator=g)]
    x = mag * (torch.randint(0, 2, (rows, cols), generator=g) * 2 - 1)
    x[:, ::32] = 6.0
    e = torch.tensor(scales)[torch.randint(0, len(scales), (rows, -(-cols // 32)), generator=g)]
    return (x * torch.exp2(e.double()).repeat_interleave(32, 1)[:, :cols]).float()


PRODUCTS = [(1, 1, 1), (1, 16, 128), (2, 3, 5), (16, 16, 32), (17, 33, 129), (64, 64, 128), (65, 63, 127), (128, 128, 256), (129, 257, 300),
            (1, 1000, 2048), (3, 130, 4224), (253, 515, 1000), (700, 8, 64), (8, 700, 96), (300, 520, 640), (16, 4096, 4096), (1030, 1100, 200)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('mnk', PRODUCTS)
def test_products_are_exact(mnk, dtype):
    """Scales 1/2, 1, 2: products are multiples of 1/16 and all partial sums stay below 2^20: 32 bits hold them exactly."""
    from deepipr_amd import mx4
    m, n, k = mnk
    a, b = _codes(m, k, 4), _codes(n, k, 5)
    bias = torch.randint(-8, 8, (n,), generator=torch.Generator().manual_seed(6)).float()
    qa, qb = mx4.quantize(a.to(DEV)), mx4.quantize(b.to(DEV))
    assert torch.equal(qa.dequantize().cpu(), a) and torch.equal(qb.dequantize().cpu(), b)
    want = a.double() @ b.double().t()
    got = mx4.matmul(qa, qb, dtype=dtype)
    assert torch.equal(got.cpu(), want.to(dtype))
    for t in TYPES:
        got = mx4.matmul(qa, qb, bias=bias.to(t).to(DEV), dtype=dtype)
        assert torch.equal(got.cpu(), (want + bias.double()).to(dtype))
    again = mx4.matmul(qa, qb, dtype=dtype)
    assert torch.equal(mx4.matmul(qa, qb, dtype=dtype), again)


@pytest.mark.parametrize('mnk', [(64, 4200, 1200), (65, 300, 9000), (128, 128, 20000), (4104, 4096, 130), (4160, 4000, 300), (4352, 4100, 250),
                                 (2500, 3000, 700), (4104, 4096, 4100), (2300, 3900, 5000), (300, 100, 20000), (512, 4000, 2050),
                                 (4000, 4001, 4100), (64, 9216, 4096), (48, 4096, 4096), (33, 70, 9000),
                                 (100, 500, 3000), (100, 500, 3100), (70, 30, 3900), (190, 490, 4200), (130, 510, 6300), (65, 33, 8200),
                                 (250, 4000, 3000), (250, 4001, 3100), (253, 3999, 3900), (200, 3900, 4200), (256, 4090, 6300), (129, 4050, 8200)])
def test_products_of_every_form_are_exact(mnk):
    """Few rows; 64 x 32 and 64 x 64 tiles over all counts of steps a wave; columns shared out over workgroups; whole tiles with a few rows
    behind them; large tiles with ragged ends."""
    from deepipr_amd import mx4
    m, n, k = mnk
    a, b = _codes(m, k, 4, (0,)).to(DEV), _codes(n, k, 5, (0,)).to(DEV)                # multiples of 1/4 below 2^20: exact
    bias = torch.randint(-8, 8, (n,), generator=torch.Generator().manual_seed(6)).float().to(DEV)
    want = torch.mm(a.double(), b.double().t().contiguous())
    for dtype in TYPES:
        got = mx4.matmul(mx4.quantize(a), mx4.quantize(b), dtype=dtype)
        assert torch.equal(got, want.to(dtype))
        assert torch.equal(mx4.linear(a.to(dtype), mx4.quantize(b), bias), (want + bias.double()).to(dtype))


def _bound(a, b, dtype, bias=None):
    """|out - exact| by the argument at the top of the file; a [M, K], b [N, K] float64 torch."""
    k = a.shape[1]
    exact = a @ b.t()
    room = (a.abs() @ b.abs().t()) * (k * 2.0 ** -23)
    if bias is not None:
        exact = exact + bias
        room = room + 2.0 ** -23 * (exact.abs() + room)
    half = torch.finfo(dtype).eps / 2
    return exact, room * (1 + half) + exact.abs() * half + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _values(x, dim):
    return torch.from_numpy(np.ascontiguousarray(oracle.values(x, dim)))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('mnk', [(1, 40, 100), (5, 70, 333), (65, 130, 257), (256, 300, 1024), (33, 1000, 2048), (512, 512, 4000)])
def test_linear_and_its_gradients(mnk, dtype):
    from deepipr_amd import mx4
    m, n, k = mnk
    x, w = _random((m, k), dtype, 7, False), _random((n, k), dtype, 8, False)
    bias, dy = _random((n,), torch.float32, 9, False), _random((m, n), dtype, 10)
    for t in (x, w, bias):
        t.requires_grad_()
    y = mx4.linear(x, w, bias)
    dx, dw, db = torch.autograd.grad(y, (x, w, bias), dy)
    for got, a, b, add in ((y, _values(x, 1), _values(w, 1), bias.detach().cpu().double()),
                           (dx, _values(dy, 1), _values(w, 0).t(), None), (dw, _values(dy, 0).t(), _values(x, 0).t(), None)):
        exact, room = _bound(a, b, dtype, add)
        assert got.dtype == dtype and bool(((got.detach().cpu().double() - exact).abs() <= room).all())
    exact = dy.double().sum(0).cpu()
    # sums of 64 rows in 32 bits, the rest in 64
    assert db.dtype == torch.float32 and bool(((db.cpu().double() - exact).abs() <= 65 * 2.0 ** -24 * dy.double().abs().sum(0).cpu()).all())
    # the same without a bias, and with the weight kept in 4 bits
    assert torch.equal(mx4.linear(x.detach(), w.detach(), bias.detach()), y.detach())
    with torch.no_grad():
        assert torch.equal(mx4.linear(x, mx4.quantize(w), bias), y)
    y2 = mx4.linear(x, w)
    dx2, = torch.autograd.grad(y2, x, dy)
    assert torch.equal(dx2, dx)


@pytest.mark.parametrize('mnk', [(40, 100, 200), (300, 2000, 1500), (512, 512, 4000), (600, 1000, 3000), (4104, 4096, 4096)])
def test_gradients_are_the_products_of_their_parts(mnk):
    """Two products in one launch give what each gives alone, in every form that they share."""
    from deepipr_amd import mx4
    m, n, k = mnk
    g = torch.Generator(device=DEV).manual_seed(m)
    x, w, dy = (torch.randn(s, generator=g, device=DEV).bfloat16() for s in ((m, k), (n, k), (m, n)))
    x.requires_grad_(), w.requires_grad_()
    y = mx4.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x, w = x.detach(), w.detach()
    assert torch.equal(y, mx4.matmul(mx4.quantize(x, 1), mx4.quantize(w, 1), dtype=x.dtype))
    assert torch.equal(dx, mx4.matmul(mx4.quantize(dy, 1), mx4.quantize(w, 0), dtype=x.dtype))
    assert torch.equal(dw, mx4.matmul(mx4.quantize(dy, 0), mx4.quantize(x, 0), dtype=x.dtype))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m', [1, 3, 16, 17, 40])
def test_rows_on_kept_weights(m, dtype):
    """Up to 16 rows are quantised inside the product, more by a launch of their own: the same codes, so the same sums, for every alignment,
    ragged last blocks and blocks that are not numbers."""
    from deepipr_amd import mx4
    for n, k in ((1, 1), (40, 31), (130, 300), (17, 2048), (300, 9216)):
        big = _random((m, k + 9), dtype, seed=m + k, spread=False)
        if k > 40 and m > 2:
            big[2, 37] = float('nan')
        q = mx4.quantize(_codes(n, k, 23, (0, 1)).to(DEV))
        bias = _random((n,), torch.float32, 24, False)
        for x in (big[:, :k].contiguous(), big[:, 1:k + 1], big[:, 8:k + 8], big[:, :k]):
            want = mx4.matmul(mx4.quantize(x), q, bias, dtype)
            got = mx4.linear(x, q, bias)
            assert got.dtype == dtype and torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got.nan_to_num(), want.nan_to_num())


def test_gradients_against_differences():
    """Inputs on the 4-bit grid in every direction: rounding changes nothing, the layer is the linear map, and one-sided differences of
    <y, dy> along steps that stay on the grid are the gradients."""
    from deepipr_amd import mx4
    m, n, k = 64, 32, 96
    g = torch.Generator().manual_seed(11)

    def on_grid(r, c):
        v = torch.tensor([-4.0, -3.0, -2.0, -1.0, 1.0, 2.0, 3.0, 4.0])[torch.randint(0, 8, (r, c), generator=g)]
        i, j = torch.arange(r)[:, None], torch.arange(c)[None, :]
        return torch.where((i + j) % 32 == 0, 6.0, v).to(DEV)         # every block of 32, either way, holds a 6: its scale is 1
    x, w, dy = on_grid(m, k), on_grid(n, k), on_grid(m, n)
    x.requires_grad_(), w.requires_grad_()
    y = mx4.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)

    def f(a, b):
        return float((mx4.linear(a, b).double() * dy.double()).sum())
    base = f(x.detach(), w.detach())
    for t, grad, other in ((x, dx, w), (w, dw, x)):
        for _ in range(6):
            i, j = int(torch.randint(0, t.shape[0], (1,), generator=g)), int(torch.randint(0, k, (1,), generator=g))
            s = t.detach().clone()
            if float(s[i, j]) == 6.0:
                continue
            s[i, j] += 1.0 if float(s[i, j]) < 4.0 and float(s[i, j]) != -1.0 else -1.0
            step = float(s[i, j] - t.detach()[i, j])
            got = f(s, w.detach()) if t is x else f(x.detach(), s)
            assert (got - base) / step == float(grad[i, j])           # whole numbers below 2^24 throughout


def test_shapes_of_linear_and_partial_gradients():
    from deepipr_amd import mx4
    w, bias = _random((40, 70), torch.float32, 12, False), _random((40,), torch.float32, 13, False)
    x = _random((3, 5, 70), torch.float32, 14, False)
    flat = mx4.linear(x.reshape(15, 70), w, bias)
    assert torch.equal(mx4.linear(x, w, bias), flat.reshape(3, 5, 40))
    assert torch.equal(mx4.linear(x[0, 0], w, bias), flat[0])
    assert torch.equal(mx4.linear(x.transpose(0, 1), w, bias), flat.reshape(3, 5, 40).transpose(0, 1))
    assert torch.equal(mx4.linear(x.reshape(15, 70).t().contiguous().t(), w.t().contiguous().t(), bias), flat)
    assert mx4.linear(x[:0], w, bias).shape == (0, 5, 40)
    e = mx4.linear(x.new_zeros(4, 0), w.new_zeros(40, 0), bias)
    assert torch.equal(e, bias.expand(4, 40))
    xg, wg, bg = x[0].clone().requires_grad_(), w.clone().requires_grad_(), bias.clone().requires_grad_()
    full = torch.autograd.grad(mx4.linear(xg, wg, bg).sum(), (xg, wg, bg))          # an expanded gradient
    assert torch.equal(full[2], torch.full((40,), 5.0, device=DEV))
    for keep in range(3):
        args = [t if i == keep else t.detach() for i, t in enumerate((xg, wg, bg))]
        got, = torch.autograd.grad(mx4.linear(*args).sum(), [args[keep]])
        assert torch.equal(got, full[keep])
    z = x.new_zeros(0, 70).requires_grad_()
    for a, b in zip(torch.autograd.grad(mx4.linear(z, wg, bg).sum(), (z, wg, bg)), (z, wg, bg)):
        assert a.shape == b.shape and not bool(a.any())


def test_refusals_of_products():
    from deepipr_amd import mx4
    x, w = _random((4, 64), torch.float32, 15), _random((8, 64), torch.float32, 16)
    q = mx4.quantize(w)
    with pytest.raises(RuntimeError, match='no backward'):
        mx4.linear(x.clone().requires_grad_(), q)
    with pytest.raises(ValueError, match='dim=1'):
        mx4.linear(x[:, :8], mx4.quantize(w.t().contiguous()[:8], 0))
    with pytest.raises(ValueError, match='features'):
        mx4.linear(x[:, :32], q)
    with pytest.raises(ValueError, match='bias'):
        mx4.linear(x, q, x[0])
    with pytest.raises(ValueError, match='blocks run'):
        mx4.matmul(q, mx4.quantize(w[:, :32]))
    with pytest.raises(TypeError):
        mx4.matmul(x, q)
    with pytest.raises(RuntimeError):
        mx4.linear(x.double(), q)
    with pytest.raises(RuntimeError, match='GPU only'):
        mx4.linear(x.cpu(), q)
    for codes, scales in ((q.codes[:-16], q.scales), (q.codes, q.scales[:-256]), (q.codes.int(), q.scales), (q.codes.cpu(), q.scales)):
        bad = mx4.Mx4Matrix(codes, scales, 8, 64, 1)
        for call in (bad.dequantize, lambda: mx4.matmul(mx4.quantize(x), bad), lambda: mx4.linear(x, bad)):
            with pytest.raises(RuntimeError):
                call()
    with pytest.raises(RuntimeError, match='twice|once_differentiable|marked'):
        a = x.clone().requires_grad_()
        g, = torch.autograd.grad(mx4.linear(a, w).square().sum(), a, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize('m', [1, 40, 300])
def test_a_bad_block_reaches_its_rows_and_columns_only(m):
    from deepipr_amd import mx4
    n, k = 70, 200
    x, w = _random((m, k), torch.float32, 17, False), _random((n, k), torch.float32, 18, False)
    good = mx4.linear(x, w)
    x[m - 1, 199] = float('nan')
    w[5, 3] = float('inf')
    y = mx4.linear(x, w)
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[m - 1] = True
    bad[:, 5] = True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], good[~bad])


def test_captured_training_passes_and_streams():
    """Two captured forward + backward passes on two streams, new inputs, eager work between the replays."""
    from deepipr_amd import mx4
    shapes = [(200, 130, 300), (64, 70, 2000)]

    def pieces(s, seed):
        m, n, k = shapes[s]
        return [_random((m, k), torch.float32, seed, False), _random((n, k), torch.float32, seed + 1, False),
                _random((n,), torch.float32, seed + 2, False), _random((m, n), torch.float32, seed + 3, False)]

    def go(x, w, b, dy):
        y = mx4.linear(x, w, b)
        return (y,) + torch.autograd.grad(y, (x, w, b), dy)
    held, graphs, outs = [], [], []
    for s in range(2):
        ts = pieces(s, 100 + 10 * s)
        for t in ts[:3]:
            t.requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go(*ts)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(go(*ts))
        held.append(ts)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(3):
        fresh = [pieces(s, 500 + 50 * rep + 10 * s) for s in range(2)]
        with torch.no_grad():
            for ts, fs in zip(held, fresh):
                for t, f in zip(ts, fs):
                    t.copy_(f)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        for t in fresh[0][:3] + fresh[1][:3]:
            t.requires_grad_()
        eager = [go(*fs) for fs in fresh]
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_launches_are_accounted():
    """The in-situ profile sees the launches of the new entry points."""
    from deepipr_amd import _lib, grad_clip, mx4
    x, w = _random((300, 500), torch.float32, 25), _random((200, 500), torch.float32, 26)
    _lib.profile_enable(True)
    try:
        mx4.linear(x, w)
        mx4.quantize(x).dequantize()
        grad_clip.clip_grads_([x], 0.5)
        got = _lib.profile_read()
    finally:
        _lib.profile_enable(False)
    for name, least in (('mx4_quantize', 2), ('mx4_dequantize', 1), ('mx4_matmul', 1), ('grad_norm', 1), ('grad_clip', 1)):
        assert got[name][1] >= least and got[name][0] > 0, (name, got[name])


def test_offsets_past_32_bits():
    """Codes of more than 2^32 bytes and an output of more than 2^32 elements."""
    from deepipr_amd import mx4
    rows, k = (1 << 20) + 77, 8320
    x = torch.ones((rows, k), dtype=torch.bfloat16, device=DEV)
    x[-3:] = _random((3, k), torch.bfloat16, 19, False)
    q = mx4.quantize(x)
    assert q.codes.numel() > 1 << 32
    w = _codes(3, k, 20).to(DEV)
    y = mx4.matmul(q, mx4.quantize(w))
    tail = _values(x[-3:], 1)
    del x, q
    assert torch.equal(y[:-3].cpu(), w.double().sum(1).float().cpu().expand(rows - 3, 3))
    exact, room = _bound(tail, w.double().cpu(), torch.float32)
    assert bool(((y[-3:].cpu().double() - exact).abs() <= room).all())
    del y
    a, b = _codes(rows, 1, 21, (0,)).to(DEV), _codes(4200, 1, 22, (0,)).to(DEV)
    y = mx4.matmul(mx4.quantize(a), mx4.quantize(b), dtype=torch.bfloat16)
    assert y.numel() > 1 << 32 and bool((y[-70:] == 36.0).all()) and bool((y[:70] == 36.0).all())
