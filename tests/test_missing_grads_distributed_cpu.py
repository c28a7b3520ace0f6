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
