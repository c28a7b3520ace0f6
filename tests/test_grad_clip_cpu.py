"""Gradient norm and clipping, host side (no GPU): refusals of the public calls and of the C entries, and FlatSGD(max_grad_norm=...)
against torch's SGD behind torch's clipping on the CPU stand-in of the kernels."""
import ctypes
import math

import numpy as np
import pytest
import torch

from deepipr_amd import _lib, grad_clip
from deepipr_amd import passport_ops as P
from deepipr_amd.flat_sgd import FlatSGD
from tests.lm_kernels import LmKernels


def test_host_tensors_and_bad_arguments_are_refused():
    t = [torch.ones(3)]
    with pytest.raises(RuntimeError, match='GPU only'):
        grad_clip.grad_norm(t)
    with pytest.raises(RuntimeError, match='GPU only'):
        grad_clip.clip_grads_(t, 1.0)
    for bad in (3, 0.5, 'fro2', 0):
        with pytest.raises(ValueError):
            grad_clip.grad_norm(t, bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match='max_norm'):
            grad_clip.clip_grads_(t, bad)
        with pytest.raises(ValueError, match='max_grad_norm'):
            FlatSGD([torch.nn.Parameter(torch.ones(2))], max_grad_norm=bad)
    with pytest.raises(RuntimeError, match='dense'):
        grad_clip.grad_norm([torch.ones(2, 2).to_sparse()])
    assert torch.equal(t[0], torch.ones(3))
    assert float(grad_clip.grad_norm([])) == 0.0 and float(grad_clip.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0


def test_dense_means_every_element_once():
    dense = P.HipKernels._dense
    x = torch.zeros(4, 6)
    assert dense(x) and dense(x.t()) and dense(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last)) and dense(x[1:3])
    assert dense(torch.zeros(0, 3).t()) and dense(torch.zeros(3, 1, 4)[:, :1].transpose(0, 2))
    assert not dense(x[:, ::2]) and not dense(torch.zeros(1).expand(5)) and not dense(x[:, :5].t())


def _rows(*rows):
    return np.array(rows, dtype=np.int64).reshape(-1, 4)


def test_c_entries_refuse_before_any_launch():
    lib = _lib.lib()
    nbytes = lib.deepipr_grad_norm_workspace_bytes()
    buf = (ctypes.c_double * (nbytes // 8))()
    ws, norm = ctypes.addressof(buf), ctypes.addressof(ctypes.c_float(0))

    def norm_of(rows, n=None, kind=2, out=norm, ws=ws, size=nbytes):
        return lib.deepipr_grad_norm(rows.ctypes.data if rows is not None else None, len(rows) if n is None else n, kind, out, ws, size, None)

    good = _rows([4096, 10, 0, _lib.F32])
    for rc in (norm_of(good, out=None), norm_of(good, ws=None), norm_of(good, size=nbytes - 1), norm_of(good, kind=3), norm_of(good, ws=ws + 4),
               norm_of(None, n=1), norm_of(good, n=-1), norm_of(_rows([0, 10, 0, 0])), norm_of(_rows([4096, -1, 0, 0])), norm_of(_rows([4096, 1, 0, 3])),
               norm_of(_rows([4098, 1, 0, _lib.F32])), norm_of(_rows([4097, 1, 0, _lib.BF16])), norm_of(_rows([4096, 1 << 43, 0, 0]))):
        assert rc == -1 and b'grad_norm' in lib.deepipr_last_error()

    def clip(rows, top=1.0):
        return lib.deepipr_grad_clip(rows.ctypes.data, len(rows), 2, top, norm, ws, nbytes, None)
    assert clip(good, -1.0) == -1 and clip(good, math.nan) == -1
    for pair in ([[4096, 10, 0, 0], [4096, 10, 0, 0]], [[4096, 10, 0, 0], [4132, 4, 0, 0]], [[4096, 100, 0, 2], [4290, 1, 0, 1]]):
        assert clip(_rows(*pair)) == -1 and b'share memory' in lib.deepipr_last_error()
    many = _rows(*[[4096 + 40 * (i % 99), 10, 0, 0] for i in range(200)])
    assert clip(many) == -1 and b'share memory' in lib.deepipr_last_error()

    def step(rows, param=4096, buf=8192, hyper=12288):
        return lib.deepipr_sgd_momentum_step_clipped(param, buf, rows.ctypes.data, len(rows), hyper, norm, ws, nbytes, None)
    for rc in (step(good, param=None), step(good, buf=None), step(good, hyper=None), step(good, param=4100), step(good[:0]),
               step(_rows([4096, 10, 0, _lib.BF16])), step(_rows([4096, 10, 32, 0])), step(_rows([4096, 10, -64, 0])), step(_rows([4096, 0, 0, 0])),
               step(_rows([4096, 65, 0, 0], [8192, 4, 64, 0]))):
        assert rc == -1 and b'sgd_momentum_step_clipped' in lib.deepipr_last_error()


@pytest.mark.parametrize('top', [0.05, 1e6])
@pytest.mark.parametrize('unused', [False, True])
def test_flat_sgd_clips_like_torch(monkeypatch, top, unused):
    monkeypatch.setattr(P, 'kernels', LmKernels())
    torch.manual_seed(3)

    def net():
        torch.manual_seed(4)
        return torch.nn.Sequential(torch.nn.Linear(5, 7), torch.nn.Linear(7, 3), torch.nn.Linear(3, 3))
    a, b = net(), net()
    oa = torch.optim.SGD(a.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-2)
    ob = FlatSGD(b.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-2, max_grad_norm=top)
    for k in range(4):
        x = torch.randn(6, 5)
        for m, o in ((a, oa), (b, ob)):
            o.zero_grad(set_to_none=True)
            h = m[1](m[0](x)) if unused else m(x)
            (h.square().sum()).backward()
            if m is a:
                n = torch.nn.utils.clip_grad_norm_(a.parameters(), ob.max_grad_norm)
            o.step()
        # 64-bit sums on one side, 32-bit ones on the other: 100 terms of 2^-24 each
        assert float(ob.grad_norm) == pytest.approx(float(n), rel=1e-5)
        if k == 1:
            ob.max_grad_norm = 0.3 * top
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.allclose(p, q, rtol=1e-4, atol=1e-6)
    with pytest.raises(RuntimeError, match='chosen when'):
        ob.max_grad_norm = None
        ob.step()
