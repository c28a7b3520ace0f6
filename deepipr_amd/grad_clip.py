"""Global gradient norm and clipping over many tensors (csrc/deepipr_gradnorm.hip, include/deepipr_hip.h: deepipr_grad_*).

The reference steps without clipping (experiments/trainer.py:144-145); this is what stands in front of `optimizer.step()` when a run
clips.  n = (sum |g|^p)^(1/p) over every element of every tensor, f = min(1, max_norm / (n + 1e-6)), g *= f, in two launches (for up
to 240 tensors; two more for every further 240), without a host synchronisation, with the sum held in 64 bits and added in a fixed
order.  Calls only enqueue work on the current stream and can be captured into a hipGraph;
a captured call keeps the tensors' addresses.

FlatSGD(max_grad_norm=...) does the same inside its step: with several ranks the norm has to be that of the EXCHANGED gradients, which
only the optimiser sees -- clip_grad_norm_ on rank-local gradients in front of it clips something else.
"""
import math

import torch

from deepipr_amd import passport_ops as P

_NORMS = {2.0: 2, 1.0: 1, math.inf: 0}


def _norm_code(norm_type):
    try:
        return _NORMS[float(norm_type)]
    except KeyError:
        raise ValueError('norm_type: 1, 2 or infinity (got %r)' % (norm_type,)) from None


def _max_norm(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError('max_norm must not be negative or NaN (got %r)' % max_norm)
    return max_norm


def _as_list(tensors):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    layouts = {t.layout for t in tensors} - {torch.strided}
    if layouts:
        raise RuntimeError('deepipr_amd gradient norms take dense tensors (got layout %s)' % layouts.pop())
    return tensors


@torch.no_grad()
def grad_norm(tensors, norm_type=2.0):
    """0-d float32 tensor: the norm over all elements of `tensors` (float32 / bfloat16 / float16, mixed as they come, on one GPU)."""
    code, tensors = _norm_code(norm_type), _as_list(tensors)
    if not tensors:
        return torch.zeros(())
    return P.kernels.grad_norm(tensors, code)


@torch.no_grad()
def clip_grads_(tensors, max_norm, norm_type=2.0):
    """Scales `tensors` in place so that their common norm is at most `max_norm`; -> the norm before (0-d float32, no host read).
    A NaN norm makes every value NaN; an infinite one makes finite values 0.  Tensors that share memory are refused."""
    code, max_norm, tensors = _norm_code(norm_type), _max_norm(max_norm), _as_list(tensors)
    if not tensors:
        return torch.zeros(())
    norm = P.kernels.grad_clip(tensors, max_norm, code)
    if any(map(torch.Tensor.is_inference, tensors)):
        tensors = [t for t in tensors if not t.is_inference()]
    torch.autograd.graph.increment_version(tensors)
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """The gradients that the parameters have, clipped in place; -> their norm before.
    error_if_nonfinite=True reads the norm on the host first and raises, leaving the gradients as they were."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and grads:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError('the gradient norm is %s: not clipped (error_if_nonfinite=True)' % norm.item())
    return clip_grads_(grads, max_norm, norm_type)
