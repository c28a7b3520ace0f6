"""Which kernels a 4-bit product takes, pinned, and the products of every such form on the GPU.

The choice is made by estimated times; a refit of the estimates must not leave a form without a test unnoticed."""
import ctypes
import os

import pytest
import torch

from deepipr_amd import _lib
from tests.test_mx4_gpu import TYPES, _codes

DEV = 'cuda:0'
NAMES = ['rows', '64 x 32', '64 x 64', '128 x 128', '256 x 256']
# (M, N, K): (form, workgroups that share a tile's columns, rows at the end that go apart)
FORMS = {
    (1, 1000, 2048): ('rows', 1, 0), (17, 33, 129): ('rows', 1, 0), (32, 70, 9000): ('rows', 1, 0), (48, 17, 200): ('rows', 1, 0),
    (64, 4200, 1200): ('64 x 32', 1, 0), (65, 33, 8200): ('64 x 32', 1, 0), (190, 490, 4200): ('64 x 32', 1, 0),
    (250, 4001, 3100): ('64 x 64', 1, 0), (300, 2000, 1500): ('64 x 64', 1, 0),
    (2500, 3000, 700): ('128 x 128', 1, 0), (4104, 4099, 1000): ('128 x 128', 1, 0),
    # odd widths behind shared columns: partial sums and what adds them up at any alignment
    (128, 128, 20000): ('128 x 128', 13, 0), (128, 127, 20000): ('128 x 128', 13, 0), (300, 101, 20000): ('128 x 128', 13, 0),
    (600, 129, 20000): ('128 x 128', 9, 0),
    (4000, 4001, 4100): ('256 x 256', 1, 0),
    # up to 16, 32 and 64 rows behind whole tiles
    (4104, 4096, 4100): ('256 x 256', 1, 8), (4116, 4096, 4096): ('256 x 256', 1, 20), (4136, 4095, 4096): ('256 x 256', 1, 40),
    (4160, 4096, 4096): ('256 x 256', 1, 64), (8225, 4093, 4096): ('256 x 256', 1, 33), (8200, 4096, 4096): ('256 x 256', 1, 8),
}


def test_forms():
    """(256 CUs: those of the card, and what the library assumes without one)"""
    hooks = ctypes.CDLL(os.path.join(os.path.dirname(_lib.LIB_PATH), 'libdeepipr_hip_trace.so'))
    plan = (ctypes.c_longlong * 3)()
    for mnk, want in FORMS.items():
        assert hooks.deepipr_debug_mx4_plan(*map(ctypes.c_longlong, mnk), plan) == 0
        assert (NAMES[plan[0]], plan[1], plan[2]) == want, mnk
    for bad in ((0, 1, 1), (1, 1, 0), (1 << 41, 1, 1)):
        assert hooks.deepipr_debug_mx4_plan(*map(ctypes.c_longlong, bad), plan) == -1
    m, n, k = 600, 129, 20000
    assert _lib.lib().deepipr_mx4_matmul_workspace_bytes(m, n, k) == 9 * m * n * 4
    assert {v[0] for v in FORMS.values()} == set(NAMES)


@pytest.mark.gpu
@pytest.mark.parametrize('mnk', FORMS)
def test_products_of_every_form(mnk):
    """Whole-number multiples of 1 / 4 below 2^20: exact in 32 bits, in whatever order they are added."""
    from deepipr_amd import mx4
    m, n, k = mnk
    a, b = _codes(m, k, 14, (0,)).to(DEV), _codes(n, k, 15, (0,)).to(DEV)
    bias = torch.randint(-8, 8, (n,), generator=torch.Generator().manual_seed(16)).float().to(DEV)
    want = torch.mm(a.double(), b.double().t().contiguous())
    qa, qb = mx4.quantize(a), mx4.quantize(b)
    for dtype in TYPES:
        assert torch.equal(mx4.matmul(qa, qb, dtype=dtype), want.to(dtype))
        assert torch.equal(mx4.matmul(qa, qb, bias, dtype), (want + bias.double()).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('mnk', [(4136, 4096, 4096), (4116, 4160, 4096), (8225, 4096, 4096)])
def test_gradients_with_rows_behind_whole_tiles(mnk):
    """dx and dw in one launch, each with its own last rows: what the products give one by one."""
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
