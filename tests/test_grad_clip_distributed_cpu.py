"""FlatSGD(max_grad_norm=...) with two ranks (gloo, CPU stand-in of the kernels): norm and factor are those of the averaged gradients, the same
on both ranks, in every form of the exchange; a parameter without a gradient stays as it is."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _free_port():
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        return s.getsockname()[1]


def _net():
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(6, 80), torch.nn.ReLU(), torch.nn.Linear(80, 70), torch.nn.ReLU(), torch.nn.Linear(70, 5))


def _data(rank):
    g = torch.Generator().manual_seed(10 + rank)
    return torch.randn(8, 6, generator=g), torch.randn(8, 5, generator=g)


def _loss(net, x, y, unused):
    h = net[2](net[1](net[0](x))) if unused else net(x)
    return (h[:, :5] - y).square().mean() * 20


def _worker(rank, port, mode, unused, out):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE='2', LOCAL_RANK=str(rank))
    from deepipr_amd import passport_ops
    from tests.lm_kernels import LmKernels
    passport_ops.kernels = LmKernels()
    dist.init_process_group('gloo', rank=rank, world_size=2)
    from deepipr_amd.flat_sgd import FlatSGD
    net = _net()
    opt = FlatSGD(net.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-2, max_grad_norm=0.3)
    if mode == 'single':
        opt.set_mode('single')
    norms = []
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        _loss(net, *_data(rank), unused).backward()
        opt.step()
        norms.append(float(opt.grad_norm))
    torch.save((norms, [p.detach().clone() for p in net.parameters()]), '%s.%d' % (out, rank))
    dist.destroy_process_group()


@pytest.mark.parametrize('mode,unused', [('hooks', False), ('single', False), ('single', True)])
def test_two_ranks_clip_the_averaged_gradients(mode, unused, tmp_path):
    out = str(tmp_path / 'r')
    mp.spawn(_worker, args=(_free_port(), mode, unused, out), nprocs=2, join=True)
    (n0, p0), (n1, p1) = (torch.load('%s.%d' % (out, r)) for r in range(2))
    assert n0 == n1 and all(torch.equal(a, b) for a, b in zip(p0, p1))
    net = _net()
    opt = torch.optim.SGD(net.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-2)
    for n in n0:
        opt.zero_grad(set_to_none=True)
        (sum(_loss(net, *_data(r), unused) for r in range(2)) / 2).backward()
        want = torch.nn.utils.clip_grad_norm_(net.parameters(), 0.3)
        opt.step()
        assert float(want) > 0.3 and n == pytest.approx(float(want), rel=1e-5)
    assert all(torch.allclose(a, b, rtol=1e-4, atol=1e-6) for a, b in zip(p0, net.parameters()))
