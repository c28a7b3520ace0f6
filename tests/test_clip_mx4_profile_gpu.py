"""The in-situ profile of the gradient-list and 4-bit kernels: every launch timed, with the work that it does itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


class _Profile:
    """After the block: name -> (ms, launches, bytes or operations)."""

    def __enter__(self):
        from deepipr_amd import _lib
        torch.cuda.synchronize()
        _lib.profile_enable(True)
        return self

    def __exit__(self, *exc):
        from deepipr_amd import _lib
        times, work = _lib.profile_read(), _lib.profile_read_bytes()
        _lib.profile_enable(False)
        self.of = {k: times[k] + (work[k],) for k in times}
        return False


def _matrix(r, c, seed, dtype=torch.bfloat16):
    return torch.randn(r, c, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


@pytest.mark.parametrize('mnk,launches', [((4136, 4096, 4096), 2), ((8200, 4096, 4096), 2), ((128, 127, 20000), 2), ((250, 4000, 3000), 1), ((40, 70, 700), 1),
                                          ((2048, 2048, 2000), 1)])
def test_products(mnk, launches):
    """Large tiles with a few rows behind them, columns shared out over workgroups and added up, and forms of one launch."""
    from deepipr_amd import mx4
    m, n, k = mnk
    a, b = mx4.quantize(_matrix(m, k, 1)), mx4.quantize(_matrix(n, k, 2))
    mx4.matmul(a, b)
    with _Profile() as p:
        mx4.matmul(a, b)
    ms, count, work = p.of['mx4_matmul']
    assert count == launches and work == 2.0 * m * n * k
    assert work / ms < 1.0e13                                       # operations per ms: the card's dense 4-bit peak is 10 PFLOP/s


def test_training_layer():
    from deepipr_amd import mx4
    m, n, k = 8200, 1000, 500
    x, w, dy = _matrix(m, k, 3).requires_grad_(), _matrix(n, k, 4).requires_grad_(), _matrix(m, n, 5)
    b = torch.zeros(n, device=DEV, requires_grad=True)
    with _Profile() as p:
        y = mx4.linear(x, w, b)
        torch.autograd.grad(y, (x, w, b), dy)
    assert p.of['mx4_matmul'][2] == 6.0 * m * n * k
    # x and w in both directions (one launch), dy in both, and the sums of its 130 tiles in two passes
    _, count, work = p.of['mx4_quantize']
    assert count == 4 and work == (m * k + n * k + m * n) * (2 + 2 * 0.53125) + (130 * 4 + 2 * 8) * n


def test_lists():
    from deepipr_amd import grad_clip
    from deepipr_amd.flat_sgd import FlatSGD
    ts = [torch.randn(20000 + i, device=DEV) for i in range(300)]
    total = sum(t.numel() for t in ts)
    with _Profile() as p:
        grad_clip.grad_norm(ts)
    _, count, work = p.of['grad_norm']
    assert count == 3 and total * 4 < work <= total * 4 + 4096 * 8       # two lists, and what is left of them added up
    with _Profile() as p:
        grad_clip.clip_grads_(ts, 1.0)
    assert p.of['grad_norm'][1:] == (2, total * 4.0) and p.of['grad_clip'][1:] == (2, total * 8.0)
    params = [torch.nn.Parameter(t) for t in ts]
    opt = FlatSGD(params, lr=0.1, max_grad_norm=1.0)
    for q in params:
        q.grad = torch.ones_like(q)
    with _Profile() as p:
        opt.step()
    assert p.of['grad_norm'][1:] == (2, total * 4.0) and p.of['sgd'][1:] == (2, total * 20.0)
