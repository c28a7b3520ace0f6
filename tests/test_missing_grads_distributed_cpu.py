"""FlatSGD's gradient exchange where ranks do not all have the same gradients."""
import os

import pytest
import torch
import torch.distributed as dist

from tests.test_grad_clip_distributed_cpu import _data, _free_port, _net


@pytest.fixture
def world_of_one(monkeypatch):
    from deepipr_amd import passport_ops
    from tests.lm_kernels import LmKernels
    monkeypatch.setattr(passport_ops, 'kernels', LmKernels())
    for k, v in dict(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(_free_port()), RANK='0', WORLD_SIZE='1', DEEPIPR_FORCE_DDP='1').items():
        monkeypatch.setenv(k, v)
    dist.init_process_group('gloo', rank=0, world_size=1)
    yield
    dist.destroy_process_group()


@pytest.mark.parametrize('skip', [None, 0, 2, 4])
def test_buckets_travel_in_one_order(world_of_one, monkeypatch, skip):
    """Whatever gradients this rank misses: another rank may have them all, and its collectives have to meet these in the same order."""
    from deepipr_amd.flat_sgd import FlatSGD
    sent, real = [], dist.all_reduce

    def recorded(t, *args, **kwargs):
        sent.append(t.data_ptr())
        return real(t, *args, **kwargs)
    monkeypatch.setattr(dist, 'all_reduce', recorded)
    net = _net()
    opt = FlatSGD(net.parameters(), lr=0.1, bucket_fractions=(0.05, 0.5))
    assert opt._buckets == [(0, 2), (2, 4), (4, 6)] and len(opt._hooks) == 4
    for _ in range(2):
        opt.zero_grad(set_to_none=True)
        x, y = _data(0)
        h = x
        for i, m in enumerate(net):
            if i == skip:                                          # its weight has no gradient
                h = torch.nn.functional.linear(h, m.weight.detach(), m.bias)
            else:
                h = m(h)
        (h - y).square().mean().backward()
        opt.step()
        assert sent == sorted(sent) and len(sent) == 3
        sent.clear()


def _partly_used(net, x, y, rank):
    """Rank 1 leaves the last layer out; the extra layer is used nowhere."""
    h = net[2](net[1](net[0](x))) if rank else net[:5](x)
    return (h[:, :5] - y).square().mean() * 20


def _with_a_spare_layer():
    net = _net()
    return net.append(torch.nn.Linear(3, 3))


def _worker(rank, port, mode, top, out):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE='2', LOCAL_RANK=str(rank))
    from deepipr_amd import passport_ops
    from tests.lm_kernels import LmKernels
    passport_ops.kernels = LmKernels()
    dist.init_process_group('gloo', rank=rank, world_size=2)
    from deepipr_amd.flat_sgd import FlatSGD
    net = _with_a_spare_layer()
    opt = FlatSGD(net.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-2, max_grad_norm=top)
    if mode == 'single':
        opt.set_mode('single')
    elif mode == 'staged':
        ps = list(reversed(list(net.parameters())))
        assert opt.configure_stages([ps[:4], ps[4:6], ps[6:]])
    norms = []
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        _partly_used(net, *_data(rank), rank).backward()
        if mode == 'staged':
            opt.exchange_stages(0, 2, overlap=False)
        opt.step()
        norms.append(float(opt.grad_norm) if top else 0.0)
    torch.save((norms, [p.detach().clone() for p in net.parameters()], opt.flat_buf.clone()), '%s.%d' % (out, rank))
    dist.destroy_process_group()


@pytest.mark.parametrize('top', [None, 0.3])
@pytest.mark.parametrize('mode', ['hooks', 'single', 'staged'])
def test_ranks_stay_together_where_one_misses_a_gradient(mode, top, tmp_path):
    """A missing gradient counts as zero in the average, on every rank alike; what no rank uses stays as it is."""
    out = str(tmp_path / 'r')
    torch.multiprocessing.spawn(_worker, args=(_free_port(), mode, top, out), nprocs=2, join=True)
    (n0, p0, b0), (n1, p1, b1) = (torch.load('%s.%d' % (out, r)) for r in range(2))
    assert n0 == n1 and torch.equal(b0, b1) and all(torch.equal(a, b) for a, b in zip(p0, p1))
    net = _with_a_spare_layer()
    spare = [p.detach().clone() for p in net[5].parameters()]
    opt = torch.optim.SGD(net.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-2)
    for n in n0:
        opt.zero_grad(set_to_none=True)
        (sum(_partly_used(net, *_data(r), r) for r in range(2)) / 2).backward()
        if top:
            want = torch.nn.utils.clip_grad_norm_(net.parameters(), top)
            assert float(want) > top and n == pytest.approx(float(want), rel=1e-5)
        opt.step()
    # 32-bit steps on both sides, in another order: as in tests/test_grad_clip_distributed_cpu.py
    assert all(torch.allclose(a, b, rtol=1e-4, atol=1e-6) for a, b in zip(p0, net.parameters()))
    assert all(torch.equal(a, b) for a, b in zip(p0[-2:], spare))


def test_a_captured_step_that_would_have_to_read_the_flags_is_refused(world_of_one, monkeypatch):
    from types import SimpleNamespace

    from deepipr_amd.flat_sgd import FlatSGD
    opt = FlatSGD(_net().parameters(), lr=0.1, max_grad_norm=1.0)
    opt.flat_param = SimpleNamespace(is_cuda=True)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    assert opt._missing_everywhere([]) == []                           # nothing missing here: nothing to read
    with pytest.raises(RuntimeError, match='cannot be captured'):
        opt._missing_everywhere([1])
