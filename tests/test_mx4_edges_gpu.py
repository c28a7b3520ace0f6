"""Bias gradients of long batches on the GPU against 64 bits."""
import pytest
import torch

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
