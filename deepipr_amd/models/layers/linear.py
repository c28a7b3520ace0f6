"""A linear layer whose products run in 4 bits (deepipr_amd.mx4): what the classifiers' nn.Linear (models/alexnet_passport.py:27-36,
models/resnet_passport.py:127-129) becomes under `--linear-format mx4`."""
import weakref

import torch
import torch.nn as nn
from torch.optim.optimizer import register_optimizer_step_post_hook

from deepipr_amd import mx4

_kept = weakref.WeakKeyDictionary()          # the layers that hold codes of their weight -> that weight (weakly)
_hook = None


def weights_written(params):
    """For code that writes parameters where autograd does not see it (kernels that take addresses, replayed graphs, collectives): a layer
    that keeps codes of one of `params` refuses to answer from them."""
    if _kept:
        ids = set(map(id, params))
        torch.autograd.graph.increment_version([m.weight for m in _kept if id(m.weight) in ids])


def _stepped(optimizer, args, kwargs):
    if _kept:
        weights_written(p for g in optimizer.param_groups for p in g['params'] if p.grad is not None)


class Mx4Linear(nn.Linear):
    """nn.Linear with the same parameters and state_dict.  Training and evaluation quantise weight and input in the call
    (mx4.linear: output, dx and dw in 4 bits, dbias exact).  A net that only answers can `keep()` its weight in 4 bits instead of
    quantising it per call; the kept codes are buffers outside the state_dict and are dropped by train(), load_state_dict(), release(),
    by a new `weight` or a new type of it and in copies of the layer.  A kept weight has no backward pass, and changing `weight` in place without a new
    keep() is an error, also where an optimiser or the framework's replayed train step does it (what neither autograd nor the framework sees,
    a write through `weight.data` or by a graph that a program captured itself, needs a keep() of its own)."""

    def __init__(self, in_features, out_features, bias=True, device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device, dtype)
        self._without_codes()

    def _without_codes(self):
        self.register_buffer('kept_codes', None, persistent=False)
        self.register_buffer('kept_scales', None, persistent=False)
        self._kept_version = None

    @classmethod
    def adopt_(cls, linear):
        """`linear` itself, from now on an Mx4Linear: parameters, hooks and every reference to it stay."""
        linear.__class__ = cls
        linear._without_codes()
        return linear

    def keep(self):
        global _hook
        if self._parameters.get('weight') is None:
            raise RuntimeError('Mx4Linear.keep: the weight is not a parameter of the layer (a parametrisation computes it anew in every call)')
        q = mx4.quantize(self.weight.detach())
        self.kept_codes, self.kept_scales, self._kept_version = q.codes, q.scales, self.weight._version
        _kept[self] = weakref.ref(self.weight)
        if _hook is None:                                    # fused optimisers write without raising a version
            _hook = register_optimizer_step_post_hook(_stepped)
        return self.eval()

    def release(self):
        self.kept_codes = self.kept_scales = self._kept_version = None
        _kept.pop(self, None)
        return self

    def register_parameter(self, name, param):               # (also what `layer.weight = ...` calls)
        if name == 'weight' and '_kept_version' in self.__dict__:
            self.release()
        super().register_parameter(name, param)

    def __setstate__(self, state):
        super().__setstate__(state)
        self.release()

    def train(self, mode=True):
        if mode:
            self.release()
        return super().train(mode)

    def _apply(self, fn, recurse=True):
        dtype = self.weight.dtype
        super()._apply(fn, recurse)
        if self.weight.dtype != dtype:                       # rounded to another type: other values (a device keeps them)
            self.release()
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        self.release()
        return super()._load_from_state_dict(*args, **kwargs)

    def forward(self, x):
        if self.kept_codes is None:
            return mx4.linear(x, self.weight, self.bias)
        weight, of = self._parameters.get('weight'), _kept[self]() if self in _kept else None
        # (torch.func.functional_call puts other tensors in the parameters' place, or detached ones of the same memory)
        if weight is None or of is None or weight._version != self._kept_version or (weight is not of and weight.data_ptr() != of.data_ptr()):
            raise RuntimeError('Mx4Linear: the weight changed after keep(); call keep() again, or release()')
        return mx4.linear(x, mx4.Mx4Matrix(self.kept_codes, self.kept_scales, self.out_features, self.in_features, 1), self.bias)

    def extra_repr(self):
        return super().extra_repr() + (', kept in 4 bits' if self.kept_codes is not None else ', mx4')


def use_mx4_linear_(model):
    """Every plain nn.Linear of `model` becomes an Mx4Linear in place (optimisers built before or after see the same parameters);
    -> how many.  Where two branches go through the layer as one batch (the lockstep form of schemes V2 and V3), the weight gradient's blocks of
    32 rows are those of that batch: unless a branch has a multiple of 32 rows, one block holds rows of both."""
    found = [m for m in model.modules() if type(m) is nn.Linear]
    for m in found:
        Mx4Linear.adopt_(m)
    return len(found)


@torch.no_grad()
def round_weights_(model):
    """The removal attempt: every convolution and linear weight is rounded to 4 bits in place, output channel by output channel in blocks
    of 32 -- what a thief who serves the net in 4 bits leaves of it.  Norm layers, biases, passports and signatures stay as they are.
    -> {parameter name: relative change (2-norm)}."""
    changed = {}
    for name, m in model.named_modules():
        if isinstance(m, (nn.Conv2d, nn.Linear)):
            w = m.weight
            flat = w.detach().reshape(w.shape[0], -1)
            new = mx4.quantize(flat).dequantize(w.dtype)
            norm = float(flat.double().norm())
            changed[(name + '.' if name else '') + 'weight'] = float((new.double() - flat.double()).norm()) / norm if norm else 0.0
            w.copy_(new.reshape(w.shape))
            if isinstance(m, Mx4Linear):
                m.release()
    return changed
