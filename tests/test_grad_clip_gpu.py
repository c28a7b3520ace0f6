"""Gradient norm, clipping and the clipped step on the GPU against the 64-bit definition.

Tolerances: the norm is a 64-bit sum (error far below 2^-40) rounded once to float32, half a step = 2^-24 of it; a clipped value is the
factor (rounded once to float32, 2^-24) times the gradient, rounded once to its type (eps / 2, or half the smallest subnormal)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _norm64(ts, kind):
    flat = torch.cat([t.detach().double().reshape(-1) for t in ts]) if ts else torch.zeros(0, dtype=torch.float64)
    return float(torch.linalg.vector_norm(flat, kind)) if flat.numel() else 0.0


def _tensors(sizes, dtype, seed=0, shift=0):
    """Tensors of odd sizes that start `shift` elements into their storage."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        base = torch.randn(n + shift, generator=g).mul_(10.0 ** (i % 3 - 1)).to(dtype).to(DEV)
        out.append(base[shift:])
    return out


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _check_clipped(got, before, factor):
    for t, b in zip(got, before):
        want = b.double() * factor
        tol = want.abs() * (_half_step(t.dtype) + 2 ** -23) + float(torch.finfo(t.dtype).smallest_normal) * torch.finfo(t.dtype).eps
        assert bool(((t.double() - want).abs() <= tol).all())


SIZES = [[1], [7], [64], [65, 1, 0, 3], [4096, 4095, 4097], [1 << 20, 5, 100003], [3] * 191, [1000 + 7 * i for i in range(400)],
         [8192], [8128, 1], [8192, 1], [100, 1, 1, 1, 1], [90] * 239]                    # around what one workgroup takes; many tiny ones


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', [2.0, 1.0, math.inf])
@pytest.mark.parametrize('sizes', range(len(SIZES)))
def test_norm_and_clip(sizes, kind, dtype):
    from deepipr_amd import grad_clip
    for shift in (0, 1):
        ts = _tensors(SIZES[sizes], dtype, seed=sizes, shift=shift)
        want = _norm64(ts, kind)
        n = grad_clip.grad_norm(ts, kind)
        assert n.dim() == 0 and n.dtype == torch.float32 and abs(float(n) - want) <= want * 2 ** -24 * 1.001
        before = [t.clone() for t in ts]
        assert float(grad_clip.clip_grads_(ts, 2 * want + 1, kind)) == float(n)
        assert all(torch.equal(t, b) for t, b in zip(ts, before))                      # within the norm: untouched
        got = grad_clip.clip_grads_(ts, 0.37 * want, kind)
        assert float(got) == float(n)
        _check_clipped(ts, before, 0.37 * want / (want + 1e-6))


def test_mixed_types_neighbours_and_reruns():
    """Types mixed in one list; what lies beside the tensors stays; twice the same inputs give the same bits."""
    from deepipr_amd import grad_clip
    base = [torch.full((1003,), 5.0, dtype=d, device=DEV) for d in TYPES]
    ts = [b[1:1000] for b in base]
    for i, t in enumerate(ts):
        t.copy_(torch.randn(999, generator=torch.Generator().manual_seed(i)))
    keep = [t.clone() for t in ts]
    want = _norm64(ts, 2)
    n = grad_clip.clip_grads_(ts, 0.5)
    assert abs(float(n) - want) <= want * 2 ** -24 * 1.001
    _check_clipped(ts, keep, 0.5 / (want + 1e-6))
    assert all(float(b[0]) == 5.0 and bool((b[1000:] == 5.0).all()) for b in base)
    first = [t.clone() for t in ts]
    for t, k in zip(ts, keep):
        t.copy_(k)
    assert torch.equal(grad_clip.clip_grads_(ts, 0.5), n) and all(torch.equal(t, f) for t, f in zip(ts, first))


def test_range_of_the_sum_and_values_that_are_not_numbers():
    from deepipr_amd import grad_clip
    for v in (1e30, 1e-30, 3e38):
        t = torch.full((1000,), v, device=DEV)
        want = _norm64([t], 2)
        n = float(grad_clip.clip_grads_([t], 1.0))
        assert (n == math.inf) if want > 3.4e38 else abs(n - want) <= want * 2 ** -23
        f = 1.0 / (want + 1e-6)
        assert torch.allclose(t.double(), torch.full((1000,), float(torch.tensor(v)) * min(1.0, f), dtype=torch.float64, device=DEV), rtol=2 ** -22, atol=0)
    t = [torch.ones(5, device=DEV), torch.tensor([1.0, math.nan], device=DEV)]
    assert math.isnan(float(grad_clip.grad_norm(t))) and math.isnan(float(grad_clip.grad_norm(t, math.inf)))
    assert math.isnan(float(grad_clip.clip_grads_(t, 1.0))) and bool(torch.isnan(t[0]).all())
    t = [torch.ones(5, device=DEV), torch.tensor([1.0, -math.inf], device=DEV)]
    assert float(grad_clip.grad_norm(t, math.inf)) == math.inf
    assert float(grad_clip.clip_grads_(t, 1.0)) == math.inf and bool((t[0] == 0).all()) and math.isnan(float(t[1][1]))
    z = torch.zeros(70, device=DEV)
    assert float(grad_clip.clip_grads_([z, z.new_zeros(0)], 1.0)) == 0.0 and float(grad_clip.clip_grads_([z], 0.0)) == 0.0
    p = torch.nn.Parameter(torch.ones(3, device=DEV))
    p.grad = torch.tensor([1.0, math.inf, 2.0], device=DEV)
    with pytest.raises(RuntimeError, match='norm is inf'):
        grad_clip.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert float(p.grad[2]) == 2.0


@pytest.mark.parametrize('rest', [0, 30000])                        # one workgroup, several launches
@pytest.mark.parametrize('dtype', TYPES)
def test_values_that_are_not_numbers_in_short_and_long_lists(dtype, rest):
    from deepipr_amd import grad_clip
    for bad, others in ((math.nan, math.nan), (math.inf, 0.0), (-math.inf, 0.0)):
        for kind in (2.0, 1.0, math.inf):
            ts = [torch.ones(5, dtype=dtype, device=DEV), torch.tensor([1.0, bad], dtype=dtype, device=DEV)]
            ts += [torch.ones(rest, dtype=dtype, device=DEV)] if rest else []
            n = float(grad_clip.clip_grads_(ts, 1.0, kind))
            assert math.isnan(n) if math.isnan(bad) else n == math.inf
            assert bool(ts[1].isnan()[1]) and all(bool(t.isnan().all() if math.isnan(others) else (t == 0).all()) for t in (ts[0], ts[-1]) if t is not ts[1])
    low = torch.full((max(rest, 6),), torch.finfo(dtype).min, dtype=dtype, device=DEV)      # the type's lowest value
    n = grad_clip.grad_norm([low], 1.0)
    want = low.double().abs().sum().item()
    assert float(n) == math.inf if want > 3.5e38 else abs(float(n) - want) <= want * 2 ** -23


def test_refusals_and_orders_of_dimensions():
    from deepipr_amd import grad_clip
    x = torch.randn(8, 6, device=DEV)
    for bad in ([x[:, ::2]], [x[:, :1].expand(8, 6)], [x.double()], [x.cpu(), x], [x.int()]):
        with pytest.raises(RuntimeError):
            grad_clip.grad_norm(bad)
    for bad in ([x, x], [x[:3], x[2:5]]):
        with pytest.raises(RuntimeError, match='share memory'):
            grad_clip.clip_grads_(bad, 1.0)
    want = _norm64([x], 2)
    version = x._version
    assert abs(float(grad_clip.clip_grads_([x.t()], 0.5)) - want) <= want * 2 ** -23
    assert x._version == version + 1                       # autograd sees the write
    with torch.inference_mode():
        y = torch.ones(7, device=DEV)
        grad_clip.clip_grads_([y], 1.0)
        assert abs(float(y.norm()) - 1.0) < 1e-5
    c = torch.randn(2, 5, 3, 4, device=DEV).to(memory_format=torch.channels_last)
    k = c.clone()
    grad_clip.clip_grads_([c], 0.5)
    _check_clipped([c], [k], 0.5 / (_norm64([k], 2) + 1e-6))


def test_large_list_past_32_bit_bytes():
    """One tensor of more than 2^31 elements (bf16): several entries, offsets past 32 bits."""
    from deepipr_amd import grad_clip
    n = (1 << 31) + 12345
    t = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    want = math.sqrt(n)
    assert abs(float(grad_clip.clip_grads_([t], want / 2)) - want) <= want * 2 ** -23
    # 1 * f, f just under 1/2: the nearest bf16 is 1/2
    assert bool((t[-20000:] == 0.5).all()) and bool((t[:20000] == 0.5).all()) and float(t[(1 << 29):(1 << 29) + 4096].float().sum()) == 2048.0


def test_captured_calls_share_nothing():
    """Two captured clips replayed in turn on two streams, with eager work between: each follows its own tensors' new values."""
    from deepipr_amd import grad_clip
    sets = [_tensors([1000, 77, 5000], torch.float32, seed=s) for s in (1, 2)]
    graphs, norms = [], []
    for ts in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            grad_clip.clip_grads_([t.clone() for t in ts], 1.0)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(grad_clip.clip_grads_(ts, 1.0))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for k in range(3):
        fresh = [_tensors([1000, 77, 5000], torch.float32, seed=10 * k + s) for s in (3, 4)]
        for ts, fs in zip(sets, fresh):
            for t, f in zip(ts, fs):
                t.copy_(f)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = [grad_clip.clip_grads_(fs, 1.0) for fs in fresh]
        torch.cuda.synchronize()
        for ts, fs, n, e in zip(sets, fresh, norms, eager):
            assert torch.equal(n, e) and all(torch.equal(t, f) for t, f in zip(ts, fs))


def _step64(params, bufs, grads, lr, mu, wd, top):
    n = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    f = min(1.0, top / (n + 1e-6))
    out = []
    for p, b, g in zip(params, bufs, grads):
        m = mu * b.double() + f * g.double() + wd * p.double()
        out.append((p.double() - lr * m, m))
    return n, out


@pytest.mark.parametrize('top', [0.5, 1e9])
def test_flat_sgd_step(top):
    """Eager steps, several: against the 64-bit definition from the state each step starts with."""
    from deepipr_amd.flat_sgd import FlatSGD
    sizes = [5, 64, 1000, 4097, 70000, 1]
    params = [torch.nn.Parameter(t) for t in _tensors(sizes, torch.float32, seed=5)]
    opt = FlatSGD(params, lr=0.1, momentum=0.9, weight_decay=1e-2, max_grad_norm=top)
    for k in range(3):
        grads = _tensors(sizes, torch.float32, seed=20 + k, shift=k)
        if k == 2:
            grads[2] = None                                    # a parameter without a gradient is left alone
        for p, g in zip(params, grads):
            p.grad = g
        slot = {id(p): off for p, off in opt._slots}
        before = [(p.detach().clone(), opt.flat_buf[slot[id(p)]:slot[id(p)] + p.numel()].clone()) for p in params]
        kept = [None if g is None else g.clone() for g in grads]
        opt.step()
        live = [i for i, g in enumerate(grads) if g is not None]
        n, want = _step64([before[i][0] for i in live], [before[i][1] for i in live], [kept[i] for i in live], 0.1, 0.9, 1e-2, top)
        assert abs(float(opt.grad_norm) - n) <= n * 2 ** -23
        for i, (wp, wm) in zip(live, want):
            got_m = opt.flat_buf[slot[id(params[i])]:slot[id(params[i])] + sizes[i]]
            # each of factor, factor * scale, its product, and three fused multiply-adds rounds once
            scale = before[i][1].double().abs() + kept[i].double().abs() + before[i][0].double().abs()
            assert bool(((got_m.double() - wm).abs() <= 6 * 2 ** -24 * scale).all())
            assert bool(((params[i].detach().double() - wp).abs() <= 6 * 2 ** -24 * (scale + wp.abs())).all())
            assert torch.equal(grads[i], kept[i])
        if k == 2:
            assert torch.equal(params[2], before[2][0])


def test_unclipped_step_is_the_plain_step_bit_for_bit():
    from deepipr_amd.flat_sgd import FlatSGD
    sizes = [5, 64, 1000, 4097]
    nets = [[torch.nn.Parameter(t) for t in _tensors(sizes, torch.float32, seed=5)] for _ in range(2)]
    a = FlatSGD(nets[0], lr=0.1, momentum=0.9, weight_decay=1e-2)
    b = FlatSGD(nets[1], lr=0.1, momentum=0.9, weight_decay=1e-2, max_grad_norm=1e9)
    for k in range(3):
        for ps in nets:
            for p, g in zip(ps, _tensors(sizes, torch.float32, seed=30 + k)):
                p.grad = g
        a.step()
        b.step()
        assert torch.equal(a.flat_param, b.flat_param) and torch.equal(a.flat_buf, b.flat_buf)


def test_captured_train_step_clips():
    """A whole captured train step (GraphedTrainStep) with clipping follows the eager one, and a changed max_grad_norm."""
    from deepipr_amd.experiments.graph_step import GraphedTrainStep
    from deepipr_amd.experiments.trainer import train_step_v1
    from deepipr_amd.flat_sgd import FlatSGD

    def build():
        torch.manual_seed(0)
        net = torch.nn.Sequential(torch.nn.Linear(40, 64), torch.nn.ReLU(), torch.nn.Linear(64, 10)).to(DEV)
        return net, FlatSGD(net.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-4, max_grad_norm=0.05)
    (na, oa), (nb, ob) = build(), build()
    g = torch.Generator().manual_seed(1)
    data = [(torch.randn(32, 40, generator=g).to(DEV), torch.randint(0, 10, (32,), generator=g).to(DEV)) for _ in range(4)]
    step = GraphedTrainStep(train_step_v1, nb, ob, *data[0], warmup=0)
    for k, (x, y) in enumerate(data):
        if k == 2:
            oa.max_grad_norm = ob.max_grad_norm = 10.0
        train_step_v1(na, oa, x, y)
        step(x, y)
        torch.cuda.synchronize()
        assert float(oa.grad_norm) == pytest.approx(float(ob.grad_norm), rel=1e-5) and float(oa.grad_norm) > 0.05
        assert torch.allclose(oa.flat_param, ob.flat_param, rtol=1e-5, atol=1e-7)
