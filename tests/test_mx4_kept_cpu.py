"""Mx4Linear.keep(): no answer out of codes whose weight has changed.  CPU stand-in of the kernels."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.nn as nn
import torch.nn.utils.parametrize

from deepipr_amd import mx4
from deepipr_amd import passport_ops as P
from deepipr_amd.flat_sgd import FlatSGD
from deepipr_amd.models.layers.linear import Mx4Linear, weights_written
from tests.lm_kernels import LmKernels
from tests.test_grad_clip_distributed_cpu import _free_port


@pytest.fixture(autouse=True)
def cpu_kernels(monkeypatch):
    monkeypatch.setattr(P, 'kernels', LmKernels())


def _layer():
    torch.manual_seed(0)
    return Mx4Linear(40, 8), torch.randn(3, 40)


OPTIMISERS = {'flat': lambda ps: FlatSGD(ps, lr=0.5), 'flat, clipped': lambda ps: FlatSGD(ps, lr=0.5, max_grad_norm=1.0),
              'plain': lambda ps: torch.optim.SGD(ps, lr=0.5), 'fused': lambda ps: torch.optim.SGD(ps, lr=0.5, fused=True)}


@pytest.mark.parametrize('name', OPTIMISERS)
def test_a_step_ends_the_kept_codes(name):
    lin, x = _layer()
    opt = OPTIMISERS[name](lin.parameters())
    lin(x).square().sum().backward()
    lin.keep()
    before = lin.weight.detach().clone()
    opt.step()
    assert not torch.equal(lin.weight, before)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match='keep'):
            lin(x)
        lin.keep()
        assert torch.equal(lin(x), mx4.linear(x, lin.weight, lin.bias))


@pytest.mark.parametrize('name', OPTIMISERS)
def test_a_step_that_leaves_the_weight_alone_does_not(name):
    lin, x = _layer()
    other = nn.Linear(4, 4)
    opt = OPTIMISERS[name](list(lin.parameters()) + list(other.parameters()))
    lin.keep()
    other(torch.randn(2, 4)).square().sum().backward()
    with torch.no_grad():
        want = lin(x)
        opt.step()                                                 # the layer has no gradients
        assert torch.equal(lin(x), want)
        weights_written(other.parameters())
        assert torch.equal(lin(x), want)


def test_a_step_that_only_other_ranks_have_a_gradient_for(monkeypatch):
    for k, v in dict(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(_free_port()), DEEPIPR_FORCE_DDP='1').items():
        monkeypatch.setenv(k, v)
    dist.init_process_group('gloo', rank=0, world_size=1)
    try:
        lin, x = _layer()
        opt = FlatSGD(lin.parameters(), lr=0.5)
        opt.set_mode('single')
        lin.keep()
        real = dist.all_reduce

        def with_another_rank(t, *args, **kwargs):
            t += 1.0
            return real(t, *args, **kwargs)
        monkeypatch.setattr(dist, 'all_reduce', with_another_rank)
        before = lin.weight.detach().clone()
        opt.step()
        assert not torch.equal(lin.weight, before)
        with torch.no_grad(), pytest.raises(RuntimeError, match='keep'):
            lin(x)
    finally:
        dist.destroy_process_group()


def _worker(rank, port, out):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE='2', LOCAL_RANK=str(rank))
    P.kernels = LmKernels()
    from deepipr_amd import distributed as D
    dist.init_process_group('gloo', rank=rank, world_size=2)
    torch.manual_seed(rank)
    lin = Mx4Linear(40, 8).keep()
    D.broadcast_state(lin)
    try:
        with torch.no_grad():
            lin(torch.ones(1, 40))
        said = ''
    except RuntimeError as e:
        said = str(e)
    torch.save(said, '%s.%d' % (out, rank))
    dist.destroy_process_group()


def test_weights_of_another_rank_end_the_kept_codes(tmp_path):
    out = str(tmp_path / 'r')
    torch.multiprocessing.spawn(_worker, args=(_free_port(), out), nprocs=2, join=True)
    assert all('keep' in torch.load('%s.%d' % (out, r)) for r in range(2))


def test_a_captured_evaluation_sees_a_changed_weight():
    """GraphedEval replays only while its signature stays: addresses alone would stay."""
    from deepipr_amd.experiments.graph_step import GraphedEval
    lin, x = _layer()
    net = nn.Sequential(lin, nn.ReLU()).eval()
    ev = GraphedEval(net)
    lin.keep()
    sig = ev._signature()
    with torch.no_grad():
        net(x)
        assert ev._signature() == sig
        lin.weight.mul_(2)
    assert ev._signature() != sig
    lin.keep()
    sig = ev._signature()
    lin.weight.grad = torch.ones_like(lin.weight)
    FlatSGD(lin.parameters(), lr=0.5).step()
    assert ev._signature() != sig


def test_another_type_of_weight_ends_the_kept_codes():
    lin, x = _layer()
    with torch.no_grad():
        lin.weight[0] = 2.0 ** -9 + 1.0                            # as bf16: 1
        lin.weight[0, 0] = 1.25                                    # between the codes 1 and 1.5 of scale 1 / 4
        want = lin.keep()(x)
        assert torch.equal(lin.cpu().float()(x), want) and lin.kept_codes is not None          # the same device, the same type
        lin.bfloat16()
        assert lin.kept_codes is None and torch.equal(lin(x.bfloat16()), mx4.linear(x.bfloat16(), lin.weight, lin.bias))
        lin.keep()
        assert torch.equal(lin.to(torch.bfloat16)(x.bfloat16()), mx4.linear(x.bfloat16(), lin.weight, lin.bias)) and lin.kept_codes is not None


def test_a_computed_weight_is_not_kept():
    """Its version says nothing: every call computes another tensor."""
    class Twice(nn.Module):
        def forward(self, w):
            return w * 2
    lin, x = _layer()
    lin.weight = nn.Parameter(lin.weight.detach().clone())          # version 0, as that of a computed tensor
    lin.keep()
    nn.utils.parametrize.register_parametrization(lin, 'weight', Twice())
    with torch.no_grad():
        with pytest.raises(RuntimeError, match='keep'):
            lin(x)
        with pytest.raises(RuntimeError, match='not a parameter'):
            lin.keep()
        lin.release()
        assert torch.equal(lin(x), mx4.linear(x, lin.weight, lin.bias))


def test_another_tensor_in_the_weights_place():
    """functional_call swaps the layer's tensors for one call."""
    from torch.func import functional_call
    lin, x = _layer()
    lin.weight = nn.Parameter(lin.weight.detach().clone())          # version 0, as that of a fresh tensor
    lin.keep()
    with torch.no_grad():
        want = lin(x)
        own = {'weight': lin.weight, 'bias': lin.bias}
        assert torch.equal(functional_call(lin, own, x), want)
        assert torch.equal(functional_call(lin, {k: v.detach() for k, v in own.items()}, x), want)
        other = {'weight': torch.randn(8, 40), 'bias': lin.bias}
        assert other['weight']._version == lin._kept_version
        with pytest.raises(RuntimeError, match='keep'):
            functional_call(lin, other, x)
        assert torch.equal(lin(x), want)
        FlatSGD(lin.parameters(), lr=0.5)                          # the same parameter at another address
        assert torch.equal(lin(x), want)


def test_kept_layers_can_be_pickled(tmp_path):
    lin, x = _layer()
    lin.keep()
    torch.save(lin, tmp_path / 'lin.pt')
    twin = torch.load(tmp_path / 'lin.pt', weights_only=False)
    with torch.no_grad():
        assert twin.kept_codes is None and torch.equal(twin(x), lin(x))
