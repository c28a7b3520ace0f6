"""The 4-bit layer, clipping and weight rounding inside the framework on the GPU: nets, captured steps, the command line."""
import os
import sys

import numpy as np
import pytest
import torch
import torch.nn as nn

from tests import mx4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _alexnet(classes=10):
    from deepipr_amd.models.alexnet_normal import AlexNetNormal
    torch.manual_seed(0)
    return AlexNetNormal(3, classes, 'bn').to(DEV)


def _batches(n, size=32, batch=16, classes=10):
    g = torch.Generator().manual_seed(5)
    return [(torch.randn(batch, 3, size, size, generator=g).to(DEV), torch.randint(0, classes, (batch,), generator=g).to(DEV)) for _ in range(n)]


def test_captured_step_of_the_set_together():
    """4-bit classifier, backward, clipped FlatSGD step, captured whole and replayed: follows the eager step batch by batch, from the same
    state (the state is copied over before every step, so that nothing but one step's rounding separates the two)."""
    from deepipr_amd.experiments.graph_step import GraphedTrainStep
    from deepipr_amd.experiments.trainer import train_step_v1
    from deepipr_amd.flat_sgd import FlatSGD
    from deepipr_amd.models.layers.linear import Mx4Linear

    def build():
        torch.manual_seed(1)
        net = nn.Sequential(nn.Flatten(), Mx4Linear(3 * 8 * 8, 256), nn.ReLU(), Mx4Linear(256, 10)).to(DEV)
        return net, FlatSGD(net.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-4, max_grad_norm=0.2)
    (na, oa), (nb, ob) = build(), build()
    data = [(x[:, :, :8, :8].contiguous(), y) for x, y in _batches(4)]
    step = GraphedTrainStep(train_step_v1, nb, ob, *data[0], warmup=0)
    for x, y in data:
        with torch.no_grad():
            ob.flat_param.copy_(oa.flat_param)
            ob.flat_buf.copy_(oa.flat_buf)
        la = train_step_v1(na, oa, x, y)[0]
        lb = step(x, y)[0]
        torch.cuda.synchronize()
        assert torch.equal(la, lb) and torch.equal(oa.grad_norm, ob.grad_norm) and float(oa.grad_norm) > 0.2
        assert torch.equal(oa.flat_param, ob.flat_param) and torch.equal(oa.flat_buf, ob.flat_buf)


def test_net_with_a_4_bit_classifier_and_kept_weights():
    from deepipr_amd.experiments.graph_step import GraphedEval
    from deepipr_amd.models.layers.linear import Mx4Linear, use_mx4_linear_
    net = _alexnet()
    seen = {}
    net.classifier.register_forward_hook(lambda m, i, o: seen.update(x=i[0].detach(), y=o.detach()))
    x, t = _batches(1)[0]
    net.eval()
    with torch.no_grad():
        net(x)
    feats = seen['x']
    assert use_mx4_linear_(net) == 1 and isinstance(net.classifier, Mx4Linear)
    lin = net.classifier
    with torch.no_grad():
        y = net(x)
        # 4 096 products, each sum off by at most a step of sum |a||b|
        a, b = (torch.from_numpy(np.ascontiguousarray(oracle.values(v, 1))) for v in (feats, lin.weight))
        want = a @ b.t() + lin.bias.cpu().double()
        room = (a.abs() @ b.abs().t()) * feats.shape[1] * 2.0 ** -23 + want.abs() * 2.0 ** -23
        assert bool(((y.cpu().double() - want).abs() <= room).all())
        ev = GraphedEval(net)
        top, loss, hits = (v.clone() for v in ev(x, t))
        lin.keep()
        assert torch.equal(net(x), y)
        got = ev(x, t)
        assert ev.captures == 2 and torch.equal(got[0], top) and torch.equal(got[1], loss)      # captured again on the kept codes
        lin.weight.mul_(-1)
        lin.keep()
        assert torch.equal(ev(x, t)[0], net(x).max(1, keepdim=True)[1]) and ev.captures == 3


def test_round_weights_of_a_passport_net():
    """Rounded weights are the 4-bit values; the signature check runs on them and agrees with the sign of gamma computed in 64 bits."""
    from deepipr_amd.experiments.runner import build_model
    from deepipr_amd.experiments.trainer_private import TesterPrivate
    from deepipr_amd.models.layers.linear import round_weights_
    from deepipr_amd.models.layers.passportconv2d import PassportBlock
    args = {'passport_config': os.path.join(ROOT, 'passport_configs', 'alexnet_passport.json'), 'norm_type': 'bn', 'key_type': 'random', 'sign_loss': 0.1,
            'arch': 'alexnet', 'train_passport': True}
    torch.manual_seed(0)
    np.random.seed(0)
    net = build_model(args, False, 10, DEV)
    x, _ = _batches(1)[0]
    net(x)                                                            # draws the random keys
    before = {k: v.clone() for k, v in net.state_dict().items()}
    change = round_weights_(net)
    assert len(change) >= 6 and all(0.01 < v < 0.3 for v in change.values())
    for k in change:
        flat = before[k].reshape(before[k].shape[0], -1)
        want = torch.from_numpy(np.ascontiguousarray(oracle.values(flat, 1))).float()
        assert torch.equal(net.state_dict()[k].reshape(flat.shape).cpu(), want)
    rates = TesterPrivate(net, DEV, verbose=False).test_signature()
    layers = [(n, m) for n, m in net.named_modules() if isinstance(m, PassportBlock)]
    assert layers and len(rates) == len(layers)
    for n, m in layers:
        w, k = m.conv.weight.double(), m.skey.double()
        gamma = torch.nn.functional.conv2d(k.cpu(), w.detach().cpu(), stride=m.conv.stride, padding=m.conv.padding).mean((0, 2, 3))
        assert rates['public_' + n] == pytest.approx(float((gamma.sign() == m.b.cpu().reshape(-1)).double().mean()), abs=2.0 / gamma.numel())


@pytest.mark.parametrize('eager', [False, True])
def test_command_line(tmp_path, eager, monkeypatch):
    monkeypatch.chdir(ROOT)
    sys.path.insert(0, ROOT)
    import train_v1
    from deepipr_amd.models.layers.linear import Mx4Linear
    argv = ['--arch', 'alexnet', '--train-passport', '--key-type', 'random', '--epochs', '1', '--batch-size', '16', '--synthetic-samples', '64',
            '--logdir', str(tmp_path), '--clip-grad-norm', '0.5', '--linear-format', 'mx4'] + (['--eager'] if eager else [])
    out = train_v1.main(argv)
    assert isinstance(out['model'].classifier, Mx4Linear) and np.isfinite(out['history'][0]['train_loss'])
    rep = train_v1.main(argv + ['--eval', '--exp-id', '1', '--round-weights', 'mx4'])
    assert set(rep['signature_before']) == set(rep['signature_after']) != set() and np.isfinite(rep['after']['loss'])


def test_work_on_a_side_stream():
    """Inputs made and consumed on a stream of the caller's own, work of another stream in between."""
    from deepipr_amd import grad_clip, mx4
    x, w = torch.randn(300, 500, device=DEV), torch.randn(200, 500, device=DEV)
    want, norm = mx4.linear(x, w), grad_clip.grad_norm([x, w])
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(other):
            noise = [torch.randn(1 << 20, device=DEV) for _ in range(4)]
            mx4.linear(noise[0].view(1024, 1024), noise[1].view(1024, 1024))
        with torch.cuda.stream(side):
            a, b = x * 1, w * 1
            y, n = mx4.linear(a, b), grad_clip.grad_norm([a, b])
            assert torch.equal(y, want) and torch.equal(n, norm)
    torch.cuda.synchronize()


def _flat_net():
    from deepipr_amd.models.layers.linear import Mx4Linear
    torch.manual_seed(2)
    return nn.Sequential(nn.Flatten(), Mx4Linear(3 * 8 * 8, 64), nn.ReLU(), Mx4Linear(64, 10)).to(DEV)


@pytest.mark.parametrize('fused', [False, True])
def test_a_replayed_step_ends_the_kept_codes(fused):
    """A layer that is kept between the replays of a train step: the replay runs no Python of the layer or of the optimiser."""
    from deepipr_amd.experiments.graph_step import GraphedTrainStep
    from deepipr_amd.experiments.trainer import train_step_v1
    from deepipr_amd.flat_sgd import FlatSGD
    net = _flat_net()
    opt = torch.optim.SGD(net.parameters(), lr=0.1, fused=True) if fused else FlatSGD(net.parameters(), lr=0.1)
    x, t = _batches(1, size=8)[0]
    step = GraphedTrainStep(train_step_v1, net, opt, x, t, warmup=0)
    step(x, t)
    with torch.no_grad():
        lin = net[3].keep()
        feats = torch.randn(4, 64, device=DEV)
        lin(feats)
        before = lin.weight.clone()
        step(x, t)
        torch.cuda.synchronize()
        assert not torch.equal(lin.weight, before)
        with pytest.raises(RuntimeError, match='keep'):
            lin(feats)


def test_a_captured_evaluation_refuses_a_changed_weight():
    from deepipr_amd.experiments.graph_step import GraphedEval
    from deepipr_amd.flat_sgd import FlatSGD
    net = _flat_net().eval()
    x, t = _batches(1, size=8)[0]
    lin, ev = net[3], GraphedEval(net)
    with torch.no_grad():
        lin.keep()
        for _ in range(3):
            assert torch.equal(ev(x, t)[0], net(x).max(1, keepdim=True)[1])
        assert ev.captures == 1
        lin.weight.mul_(-1)
        for _ in range(2):
            with pytest.raises(RuntimeError, match='keep'):
                ev(x, t)
        lin.keep()
        assert torch.equal(ev(x, t)[0], net(x).max(1, keepdim=True)[1])
        opt = FlatSGD(lin.parameters(), lr=1.0)                       # (moves the weight to the flat buffer)
        lin.keep()
        ev(x, t)
        lin.weight.grad = torch.randn_like(lin.weight)
        opt.step()
        with pytest.raises(RuntimeError, match='keep'):
            ev(x, t)
        lin.release()
        assert torch.equal(ev(x, t)[0], net(x).max(1, keepdim=True)[1])
