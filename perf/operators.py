"""What is measured of the clipped optimiser step and of the 4-bit (microscaled, "MX4") matrix operators.

Each case is one pass through one operator:
  clip    the global norm of a list of gradients, and the gradients scaled down to `max_norm`      (deepipr_amd.grad_clip)
  step    SGD with momentum and weight decay behind the same clipping, on a net's parameters       (deepipr_amd.flat_sgd)
  round   a matrix in 4 bits and back: blocks of 32 values along `dim` share a power of two        (deepipr_amd.mx4)
  serve   activations quantised in the call, times weights that the program keeps in 4 bits        (deepipr_amd.mx4)
  train   a linear layer whose three products run in 4 bits: output and all gradients              (deepipr_amd.mx4)

`own` is set by whoever runs this file: False computes the plain form in elementary torch operations (32 bits), True calls the
framework.  `exact` restates every definition in 64 bits, apart from the plain form.
"""
import math

import torch

own = False

DEV = 'cuda'
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
BLOCK = 32                                     # values that share one scale
LR, MOMENTUM, DECAY = 0.01, 0.9, 1e-4          # the framework's own optimiser settings
ALIGN = 64                                     # floats: FlatSGD starts every parameter on a 256-byte boundary


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a classifier that is fine-tuned alone (weight + bias): launch latency is all there is
        {'name': 'clip-head', 'op': 'clip', 'net': 'head', 'tensors': 0, 'total': 0, 'dtype': 'float32', 'max_norm': 1.0},
        # every gradient of the ResNet50 variant, as views of one bucket
        {'name': 'clip-resnet50', 'op': 'clip', 'net': 'resnet50', 'tensors': 0, 'total': 0, 'dtype': 'float32', 'max_norm': 1.0},
        # many tensors of odd sizes in bf16, none of them aligned to a vector load: half a gigabyte
        {'name': 'clip-ragged-bf16', 'op': 'clip', 'net': 'ragged', 'tensors': 391, 'total': 268435459, 'dtype': 'bfloat16', 'max_norm': 5.0},
        # the optimiser step of the headline net, and of the ImageNet AlexNet (62 M parameters)
        {'name': 'step-resnet18', 'op': 'step', 'net': 'resnet18', 'tensors': 0, 'total': 0, 'dtype': 'float32', 'max_norm': 1.0},
        {'name': 'step-alexnet', 'op': 'step', 'net': 'alexnet', 'tensors': 0, 'total': 0, 'dtype': 'float32', 'max_norm': 1.0},
        # the 1000-class head of a ResNet50, as a removal attempt rounds it to 4 bits
        {'name': 'round-head', 'op': 'round', 'rows': 1000, 'cols': 2048, 'dim': 1, 'dtype': 'float32'},
        # activations of a 56x56 map of 64 images, odd width, blocks down the rows (the weight gradient's direction)
        {'name': 'round-map-bf16', 'op': 'round', 'rows': 200704, 'cols': 1021, 'dim': 0, 'dtype': 'bfloat16'},
        # one image through the widest hidden classifier layer of the ImageNet AlexNet
        {'name': 'serve-one', 'op': 'serve', 'm': 1, 'n': 4096, 'k': 9216, 'dtype': 'float32', 'bias': True},
        # a ragged batch through the same layer
        {'name': 'serve-batch', 'op': 'serve', 'm': 253, 'n': 4096, 'k': 9216, 'dtype': 'bfloat16', 'bias': True},
        # the largest product
        {'name': 'serve-large', 'op': 'serve', 'm': 8192, 'n': 8192, 'k': 8192, 'dtype': 'bfloat16', 'bias': False},
        # fine-tuning: the 1000-class head at batch 256, and a wide layer over a long batch of bf16 rows
        {'name': 'train-head', 'op': 'train', 'm': 256, 'n': 1000, 'k': 2048, 'dtype': 'float32', 'bias': True},
        {'name': 'train-wide-bf16', 'op': 'train', 'm': 8200, 'n': 4096, 'k': 4096, 'dtype': 'bfloat16', 'bias': True},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['clip', 'step', 'round', 'serve', 'train'])
    dtype = rng.choice(['float32', 'bfloat16', 'float16'])
    if op in ('clip', 'step'):
        tensors = _spread(rng, 1, 391)
        total = max(tensors, _spread(rng, 1000, 268435459 if op == 'clip' and dtype != 'float32' else 62000000))
        return {'op': op, 'net': 'ragged', 'tensors': tensors, 'total': total, 'dtype': dtype if op == 'clip' else 'float32',
                'max_norm': rng.choice([0.1, 1.0, 5.0, 1e6])}
    if op == 'round':
        cols = _spread(rng, 1, 9216)
        rows = _spread(rng, 1, max(1, min(802816, 200000000 // (cols * (2 if dtype == 'float32' else 1)))))
        return {'op': op, 'rows': rows, 'cols': cols, 'dim': rng.randrange(2), 'dtype': dtype}
    top = 8192 ** 3 if op == 'serve' else 8200 * 4096 * 4096
    n, k = _spread(rng, 10, 9216), _spread(rng, 20, 9216)
    m = _spread(rng, 1, max(1, min(8192, top // (n * k))))
    return {'op': op, 'm': m, 'n': n, 'k': k, 'dtype': dtype, 'bias': rng.random() < 0.5}


# --------------------------------------------------------------------------------------------------------------- the inputs
def _resnet_sizes(blocks, bottleneck, classes, stem):
    sizes, width = [64 * 3 * stem * stem, 64, 64], 64
    for stage, n in enumerate(blocks):
        mid = 64 << stage
        out = mid * (4 if bottleneck else 1)
        for b in range(n):
            kernels = [(width, mid, 1), (mid, mid, 9), (mid, out, 1)] if bottleneck else [(width, mid, 9), (mid, mid, 9)]
            for i, o, kk in kernels + ([(width, out, 1)] if b == 0 and (stage or bottleneck) else []):
                sizes += [i * o * kk, o, o]
            width = out
    return sizes + [width * classes, classes]


def _sizes(case, seed):
    """Elements of each tensor, in the order of the net's parameters."""
    net = case['net']
    if net == 'head':
        return [512 * 10, 10]
    if net == 'resnet18':
        return _resnet_sizes([2, 2, 2, 2], False, 10, 3)
    if net == 'resnet50':
        return _resnet_sizes([3, 4, 6, 3], True, 1000, 7)
    if net == 'alexnet':
        convs = [(3, 64, 121), (64, 192, 25), (192, 384, 9), (384, 256, 9), (256, 256, 9)]
        return [n for i, o, kk in convs for n in (i * o * kk, o, o)] + [9216 * 4096, 4096, 4096 * 4096, 4096, 4096 * 1000, 1000]
    g = torch.Generator().manual_seed(case['tensors'])
    cut = torch.rand(case['tensors'], generator=g, dtype=torch.float64).pow_(3).add_(1e-3)
    part = (cut / cut.sum() * (case['total'] - case['tensors'])).long() + 1
    part[0] += case['total'] - int(part.sum())
    return part.tolist()


def _starts(sizes, align):
    at, n = [], 0
    for s in sizes:
        at.append(n)
        n += -(-s // align) * align
    return at, n


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _activations(m, k, g, dtype):
    """What a ReLU leaves: half of it zero, features of very different size."""
    return torch.randn((m, k), generator=g, device=DEV).clamp_(min=0).mul_(torch.randn(k, generator=g, device=DEV).exp_()).to(dtype)


def _inputs(case, seed):
    g, op = _generator(seed), case['op']
    dtype = DTYPES[case['dtype']]
    if op in ('clip', 'step'):
        # FlatSGD keeps the parameters last to first, each on a boundary of its own; a bucket for `clip` is packed tight
        sizes = _sizes(case, seed)
        order = list(reversed(sizes)) if op == 'step' else sizes
        at, total = _starts(order, ALIGN if op == 'step' else 1)
        grad = torch.zeros(total, dtype=dtype, device=DEV)
        param, momentum = (torch.zeros(total, device=DEV) for _ in range(2)) if op == 'step' else (None, None)
        for s, n in zip(at, order):
            grad[s:s + n] = _normal(n, g).mul_(0.02 + 0.5 / math.sqrt(n)).to(dtype)
            if op == 'step':
                param[s:s + n] = _normal(n, g).mul_(1 / math.sqrt(n) + 0.01)
                momentum[s:s + n] = _normal(n, g).mul_(0.01)
        return {'grad': grad, 'param': param, 'momentum': momentum, 'at': at, 'order': order}
    if op == 'round':
        x = _normal((case['rows'], case['cols']), g).mul_(_normal((1, case['cols']), g).exp_())
        return {'x': x.to(dtype)}
    m, n, k = case['m'], case['n'], case['k']
    d = {'x': _activations(m, k, g, dtype), 'bias': _normal(n, g).mul_(0.1) if case['bias'] else None}
    w = _normal((n, k), g).mul_(1 / math.sqrt(k))
    d['w'] = w.to(dtype) if op == 'train' else w
    if op == 'train':
        d['dy'] = _normal((m, n), g).mul_(1 / m).mul_(_normal((m, 1), g).exp_()).to(dtype)
    return d


def prepare(case, seed):
    s = _inputs(case, seed)
    s['case'] = case
    op = case['op']
    if op == 'clip':
        # the gradients that a backward pass wrote, and the bucket whose views the parameters hold as `.grad`
        s['bucket'] = s['grad'].clone()
        s['views'] = [s['bucket'][a:a + n] for a, n in zip(s['at'], s['order'])]
    elif op == 'step':
        if own:
            from deepipr_amd.flat_sgd import FlatSGD
            params = [torch.nn.Parameter(s['param'][a:a + n].clone()) for a, n in zip(s['at'], s['order'])]
            for p, a in zip(params, s['at']):
                p.grad = s['grad'][a:a + p.numel()]
            s['opt'] = FlatSGD(list(reversed(params)), lr=LR, momentum=MOMENTUM, weight_decay=DECAY, max_grad_norm=case['max_norm'])
            s['opt'].flat_buf.copy_(s['momentum'])
    elif op == 'serve':
        # a program that serves keeps its weights as it uses them: in 4 bits, or (plain form) the values those stand for
        if own:
            from deepipr_amd import mx4
            s['kept'] = mx4.quantize(s['w'])
        else:
            s['kept'] = _rounded(s['w'], 1)
    elif op == 'train':
        if own:
            s['x'].requires_grad_()
            s['w'].requires_grad_()
            if s['bias'] is not None:
                s['bias'].requires_grad_()
    return s


# ----------------------------------------------------------------------------------------------------------- the plain forms
def _rounded(x, dim):
    """The values that x has in 4 bits: blocks of 32 along `dim` share the scale 2^(floor(log2 max|block|) - 2), limited to
    2^-127 .. 2^127; each value is rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, ties to the even code."""
    if dim == 0:
        return _rounded(x.t(), 1).t()
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    v = torch.ldexp(b, -e)
    a = v.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.copysign(torch.round(a / step) * step, v)
    return torch.ldexp(q, e).reshape(rows, -1)[:, :cols]


def _clip_factor(total, max_norm):
    """torch's rule: max_norm / (norm + 1e-6), never above 1."""
    return (max_norm / (total + 1e-6)).clamp(max=1.0)


def _run_clip(s):
    c = s['case']
    # the pass starts where a backward pass ends: with new gradients in the bucket
    s['bucket'].copy_(s['grad'])
    if own:
        from deepipr_amd import grad_clip
        norm = grad_clip.clip_grads_(s['views'], c['max_norm'])
        return {'norm': norm, 'grads': s['bucket']}
    squares = torch.stack([v.float().square().sum(dtype=torch.float64) for v in s['views']])
    norm = squares.sum().sqrt()
    factor = _clip_factor(norm, c['max_norm']).float()
    s['bucket'].mul_(factor)
    return {'norm': norm.float(), 'grads': s['bucket']}


def _run_step(s):
    if own:
        s['opt'].step()
        return {'norm': s['opt'].grad_norm, 'param': s['opt'].flat_param, 'momentum': s['opt'].flat_buf}
    norm = s['grad'].square().sum(dtype=torch.float64).sqrt()
    factor = _clip_factor(norm, s['case']['max_norm']).float()
    g = s['grad'] * factor + DECAY * s['param']
    s['momentum'].mul_(MOMENTUM).add_(g)
    s['param'].sub_(LR * s['momentum'])
    return {'norm': norm.float(), 'param': s['param'], 'momentum': s['momentum']}


def _run_round(s):
    dim = s['case']['dim']
    if own:
        from deepipr_amd import mx4
        return mx4.quantize(s['x'], dim=dim).dequantize()
    return _rounded(s['x'], dim).contiguous()


def _run_serve(s):
    if own:
        from deepipr_amd import mx4
        return mx4.linear(s['x'], s['kept'], s['bias'])
    y = _rounded(s['x'], 1) @ s['kept'].t()
    return (y if s['bias'] is None else y + s['bias']).to(s['x'].dtype)


def _run_train(s):
    x, w, bias, dy = s['x'], s['w'], s['bias'], s['dy']
    if own:
        from deepipr_amd import mx4
        y = mx4.linear(x, w, bias)
        grads = torch.autograd.grad(y, [x, w] + ([] if bias is None else [bias]), dy)
        return {'y': y.detach(), 'dx': grads[0], 'dw': grads[1], 'dbias': grads[2] if bias is not None else None}
    y = _rounded(x, 1) @ _rounded(w, 1).t()
    y = (y if bias is None else y + bias).to(x.dtype)
    dx = (_rounded(dy, 1) @ _rounded(w, 0)).to(x.dtype)
    dw = (_rounded(dy, 0).t() @ _rounded(x, 0)).to(w.dtype)
    return {'y': y, 'dx': dx, 'dw': dw, 'dbias': None if bias is None else dy.float().sum(0)}


_RUN = {'clip': _run_clip, 'step': _run_step, 'round': _run_round, 'serve': _run_serve, 'train': _run_train}


def run(state):
    return _RUN[state['case']['op']](state)


# ---------------------------------------------------------------------------------------------------------------------- work
def _mx4_bytes(rows, cols):
    return rows * (cols / 2 + cols / BLOCK)


def work(case):
    """Each input read once, each output written once."""
    op, size = case['op'], {'float32': 4, 'bfloat16': 2, 'float16': 2}[case['dtype']]
    if op in ('clip', 'step'):
        n = sum(_sizes(case, 0))
        # clip: new gradients in, clipped ones out; step: gradient, parameter and momentum in, the last two out
        return {'bytes': n * size * 2 + 4, 'flops': 3 * n} if op == 'clip' else {'bytes': n * 20 + 4, 'flops': 9 * n}
    if op == 'round':
        n = case['rows'] * case['cols']
        return {'bytes': n * (size + 4), 'flops': 4 * n}
    m, n, k = case['m'], case['n'], case['k']
    bias = 4 * n if case['bias'] else 0
    if op == 'serve':
        return {'bytes': m * k * size + _mx4_bytes(n, k) + m * n * size + bias, 'flops': 2 * m * n * k}
    return {'bytes': 2 * size * (m * k + n * k + m * n) + 2 * bias, 'flops': 6 * m * n * k}


# --------------------------------------------------------------------------------------------------------- 64-bit definitions
_CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_rounded(x, dim):
    x = x.double() if dim == 1 else x.double().t()
    rows, cols = x.shape
    codes = torch.tensor(_CODES, dtype=torch.float64, device=x.device)
    # a value on the border between two codes belongs to the even one: upwards where the lower code is odd
    border = (codes[1:] + codes[:-1]) / 2
    odd = torch.arange(7, device=x.device) % 2 == 1
    border = torch.where(odd, torch.nextafter(border, torch.zeros_like(border)), border)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    span = max(1, (1 << 25) // max(1, cols))
    for lo in range(0, rows, span):
        part = x[lo:lo + span]
        for c0, c1 in ((0, cols // BLOCK * BLOCK), (cols // BLOCK * BLOCK, cols)):
            if c1 > c0:
                b = part[:, c0:c1].reshape(part.shape[0], -1, min(BLOCK, c1 - c0))
                top = b.abs().amax(-1, keepdim=True)
                exponent = torch.where(top > 0, torch.frexp(top).exponent.double() - 3, torch.full_like(top, -127.0)).clamp(-127, 127)
                scale = torch.exp2(exponent)
                near = codes[torch.bucketize((b / scale).abs(), border)]
                out[lo:lo + span, c0:c1] = (near * scale * b.sign()).reshape(part.shape[0], -1)
    return out if dim == 1 else out.t()


def exact(case, seed):
    s, op = _inputs(case, seed), case['op']
    if op == 'round':
        return _exact_rounded(s['x'], case['dim']).contiguous()
    if op in ('clip', 'step'):
        g = s['grad'].double()
        norm = torch.linalg.vector_norm(g)
        factor = min(1.0, case['max_norm'] / (float(norm) + 1e-6))
        if op == 'clip':
            return {'norm': norm, 'grads': g * factor}
        p = s['param'].double()
        buf = MOMENTUM * s['momentum'].double() + factor * g + DECAY * p
        return {'norm': norm, 'param': p - LR * buf, 'momentum': buf}
    x, w = s['x'], s['w']
    y = torch.mm(_exact_rounded(x, 1), _exact_rounded(w, 1).t().contiguous())
    if s['bias'] is not None:
        y += s['bias'].double()
    if op == 'serve':
        return y
    dy = s['dy']
    dx = torch.mm(_exact_rounded(dy, 1), _exact_rounded(w, 0).contiguous())
    dw = torch.mm(_exact_rounded(dy, 0).t().contiguous(), _exact_rounded(x, 0).contiguous())
    return {'y': y, 'dx': dx, 'dw': dw, 'dbias': None if s['bias'] is None else dy.double().sum(0)}
