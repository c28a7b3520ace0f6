"""Matrices in microscaled 4-bit floating point (MXFP4) and their products (csrc/deepipr_mx4.hip, include/deepipr_hip.h: deepipr_mx4_*).

The reference's classifiers are nn.Linear in fp32 (models/alexnet_passport.py:27-36, models/resnet_passport.py:127-129); the ImageNet
AlexNet keeps 58.6 of its 62 million parameters there.  Here they can be held and multiplied in 4 bits -- to train, to serve, or to see
what a 4-bit rounding of a trained net leaves of its signature (round_weights_).

  quantize(x, dim)     x -> Mx4Matrix: blocks of 32 values along `dim` share a power of two, every value is one of
                       0, 0.5, 1, 1.5, 2, 3, 4, 6 (and negatives) times it, rounded to nearest, ties to even, saturating at 6
  matmul(a, b, bias)   a b^T + bias of two quantised matrices: fp32 products and sums on the block-scaled matrix instructions
  linear(x, w, bias)   x quantised in the call; w a Mx4Matrix (weights kept in 4 bits, no gradient), or a float weight with gradients:
                           y  = Q(x) Q(w)^T + bias      blocks along the input features
                           dx = Q(dy) Q(w)              blocks along the output features
                           dw = Q(dy)^T Q(x)            blocks along the rows of the batch
                           dbias = the column sums of dy, not quantised
                       Q rounds; its own derivative is taken as 1 (straight-through).  Each of x, w and dy is read once for both of
                       its directions.

Calls only enqueue work on the current stream, allocate what they need from torch and can be captured into a hipGraph.
"""
import torch
from torch.autograd import forward_ad

from deepipr_amd import passport_ops as P

BLOCK = 32


class Mx4Matrix:
    """A matrix in 4 bits.  `shape`: that of the tensor it was made of; blocks run along its dimension `dim` (0 or 1).  `codes` and `scales`
    are the device buffers in the library's layout (include/deepipr_hip.h); `rows` x `cols` is the stored matrix, whose rows hold the blocks:
    the tensor itself for dim 1, its transpose for dim 0."""

    __slots__ = ('codes', 'scales', 'rows', 'cols', 'dim')

    def __init__(self, codes, scales, rows, cols, dim):
        self.codes, self.scales, self.rows, self.cols, self.dim = codes, scales, rows, cols, dim

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols) if self.dim == 1 else (self.cols, self.rows))

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def dequantize(self, dtype=torch.float32):
        """The values, [shape], rounded once to `dtype` (float32 holds them exactly)."""
        if self.rows == 0 or self.cols == 0:
            return torch.empty(self.shape, dtype=dtype, device=self.device)
        return P.kernels.mx4_dequantize(self.codes, self.scales, self.rows, self.cols, self.dim == 0, dtype)

    def __repr__(self):
        return 'Mx4Matrix(shape=%s, dim=%d, device=%s)' % (tuple(self.shape), self.dim, self.device)


def _matrix(x):
    if not isinstance(x, torch.Tensor):
        raise TypeError('mx4: a tensor is expected (got %s)' % type(x).__name__)
    if x.dim() != 2:
        raise ValueError('mx4: a matrix is expected (got %d dimensions)' % x.dim())
    return x.detach()


def _empty(x, rows, cols, dim):
    P.kernels._mx4_chk('mx4_quantize', x)
    z = torch.empty(0, dtype=torch.uint8, device=x.device)
    return Mx4Matrix(z, z, rows, cols, dim)


def _by_rows(x):
    """Whether x's rows are the contiguous direction; a matrix whose columns are is handled as its transpose, anything else refused
    by the kernel wrapper."""
    return x.stride(1) == 1 or x.shape[1] <= 1 or x.stride(0) != 1


def quantize(x, dim=-1):
    """x [R, C] (float32 / bfloat16 / float16, either direction contiguous) -> Mx4Matrix with blocks along `dim`.  Not differentiable."""
    x = _matrix(x)
    if dim not in (-2, -1, 0, 1):
        raise ValueError('mx4: dim 0 or 1 (got %r)' % (dim,))
    dim %= 2
    r, c = x.shape
    rows, cols = (r, c) if dim == 1 else (c, r)
    if r == 0 or c == 0:
        return _empty(x, rows, cols, dim)
    if _by_rows(x):
        a, b, _ = P.kernels.mx4_quantize(x, dim == 1, dim == 0)
    else:                                                   # the transpose has contiguous rows; its other direction is ours
        b, a, _ = P.kernels.mx4_quantize(x.t(), dim == 0, dim == 1)
    return Mx4Matrix(*(a if dim == 1 else b), rows, cols, dim)


def quantize_both(x):
    """-> (quantize(x, 1), quantize(x, 0)) with x read once."""
    x = _matrix(x)
    r, c = x.shape
    if r == 0 or c == 0:
        return _empty(x, r, c, 1), _empty(x, c, r, 0)
    if _by_rows(x):
        a, b, _ = P.kernels.mx4_quantize(x, True, True)
    else:
        b, a, _ = P.kernels.mx4_quantize(x.t(), True, True)
    return Mx4Matrix(*a, r, c, 1), Mx4Matrix(*b, c, r, 0)


def _bias_of(bias, n):
    if bias is None:
        return None
    if bias.shape != (n,):
        raise ValueError('mx4: the bias has shape %s, not (%d,)' % (tuple(bias.shape), n))
    return bias.detach().contiguous()


def _product(a, b, m, n, k, bias, dtype, like):
    """a b^T + bias with a [m, k], b [n, k] as (codes, scales)."""
    if m == 0 or n == 0 or k == 0:
        out = torch.zeros((m, n), dtype=dtype, device=like.device)
        return out if bias is None else out.add_(bias)
    return P.kernels.mx4_matmul(a, b, m, n, k, bias, dtype)


def matmul(a, b, bias=None, dtype=torch.float32):
    """a [M, K] times the transpose of b [N, K] (as STORED: a.rows x a.cols, b.rows x b.cols; the blocks of both run along K), plus
    bias [N]; -> [M, N] of `dtype`.  Not differentiable, in the bias neither."""
    if not isinstance(a, Mx4Matrix) or not isinstance(b, Mx4Matrix):
        raise TypeError('mx4.matmul takes quantised matrices (mx4.quantize)')
    if a.cols != b.cols:
        raise ValueError('mx4.matmul: the blocks run along %d and %d values' % (a.cols, b.cols))
    return _product((a.codes, a.scales), (b.codes, b.scales), a.rows, b.rows, a.cols, _bias_of(bias, b.rows), dtype, a)


def _forward(x, w, bias, need_dx, need_dw):
    """-> the output, what the backward pass needs (or None)."""
    (m, k), n = x.shape, w.shape[0]
    b = _bias_of(bias, n)
    if m == 0 or n == 0 or k == 0:
        P.kernels._mx4_chk('mx4_linear', x, w, bias)
        return _product(None, None, m, n, k, b, x.dtype, x), None
    return P.kernels.mx4_linear_fwd(x.detach(), w.detach(), None, b, need_dx, need_dw)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias):
        need_dx, need_dw, _ = ctx.needs_input_grad
        ctx.dims, ctx.types = (x.shape[0], w.shape[0], x.shape[1]), (x.dtype, w.dtype, None if bias is None else bias.dtype)
        y, saved = _forward(x, w, bias, need_dx, need_dw)
        ctx.save_for_backward(saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (m, n, k), (xtype, wtype, btype) = ctx.dims, ctx.types
        saved, = ctx.saved_tensors
        need_dx, need_dw, need_db = ctx.needs_input_grad
        if m == 0 or n == 0 or k == 0:
            zero = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=dy.device)
            return (zero(m, k, dtype=xtype) if need_dx else None, zero(n, k, dtype=wtype) if need_dw else None,
                    dy.sum(0, dtype=torch.float32).to(btype) if need_db else None)
        if not _rows_ok(dy):
            dy = dy.contiguous()                             # e.g. the expanded gradient of a sum
        dx, dw, db = P.kernels.mx4_linear_bwd(dy, saved, k, need_dx, need_dw, xtype, wtype, need_db)
        return dx, dw, (db.to(btype) if need_db else None)


def _rows_ok(x):
    """Rows of contiguous elements that do not overlap."""
    return (x.stride(1) == 1 or x.shape[1] <= 1) and (x.stride(0) >= x.shape[1] or x.shape[0] <= 1)


def _has_tangent(t):
    """Whether t takes part in forward-mode differentiation (no_grad() does not end that)."""
    return t is not None and forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def linear(x, weight, bias=None):
    """x [..., K] times weight^T plus bias [N], in 4 bits (see the module); -> [..., N] of x's type.  weight: Mx4Matrix [N, K] with blocks along
    K (frozen: asking for a gradient of x raises), or a float matrix [N, K]; gradients of x, weight and bias as the module states them.
    Forward-mode derivatives are refused."""
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise TypeError('mx4.linear: x is a tensor of at least one dimension')
    kept = isinstance(weight, Mx4Matrix)
    if not kept:
        _matrix(weight)
    n, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError('mx4.linear: x has %d features, the weight %d' % (x.shape[-1], k))
    if kept and weight.dim != 1:
        raise ValueError('mx4.linear: the weight must be quantised along its input features (dim=1)')
    if bias is not None and bias.shape != (n,):
        raise ValueError('mx4: the bias has shape %s, not (%d,)' % (tuple(bias.shape), n))
    rows = x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), k)
    if not _rows_ok(rows):
        rows = rows.contiguous()
    if kept:
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise RuntimeError('mx4.linear: a weight kept in 4 bits has no backward pass; pass the float weight, or use torch.no_grad()')
        if _has_tangent(x) or _has_tangent(bias):
            raise RuntimeError('mx4.linear has no forward-mode derivative')
        m = rows.shape[0]
        if m == 0 or n == 0 or k == 0:
            P.kernels._mx4_chk('mx4_linear', rows, weight.codes, bias)
            y = _product(None, None, m, n, k, _bias_of(bias, n), x.dtype, rows)
        else:
            y, _ = P.kernels.mx4_linear_fwd(rows.detach(), None, (weight.codes, weight.scales, n), _bias_of(bias, n), False, False)
    else:
        weight = weight if _rows_ok(weight) else weight.contiguous()
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:
            y = _Linear.apply(rows, weight, bias)
        else:                                                # (needs_input_grad names the tensors that require one, also without grad mode)
            y, _ = _forward(rows, weight, bias, False, False)
    return y if x.dim() == 2 else y.reshape(x.shape[:-1] + (n,))
