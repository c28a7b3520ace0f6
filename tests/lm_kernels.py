"""CPU stand-in of the clipping and 4-bit entry points (test infrastructure): the 64-bit definitions behind the kernels' python interface."""
import math

import numpy as np
import torch

from tests import mx4_oracle as oracle
from tests.oracle_kernels import OracleKernels


class LmKernels(OracleKernels):
    def _norm64(self, tensors, kind):
        flat = torch.cat([t.detach().double().reshape(-1) for t in tensors])
        return float(torch.linalg.vector_norm(flat, math.inf if kind == 0 else kind))

    def grad_norm(self, tensors, norm_type):
        return torch.tensor(self._norm64(tensors, norm_type))

    def grad_clip(self, tensors, max_norm, norm_type):
        n = self._norm64(tensors, norm_type)
        for t in tensors:
            t.mul_(min(1.0, max_norm / (n + 1e-6)))
        return torch.tensor(n)

    def clipped_rows(self, numels, offsets, size):
        return np.array([[0, n, off, 0] for n, off in zip(numels, offsets)], dtype=np.int64)

    def sgd_momentum_step_clipped(self, flat_param, flat_buf, grads, rows, hyper, norm):
        if not all(g.is_contiguous() for g in grads):
            return False
        lr, mu, wd, gs, top = [float(v) for v in hyper.tolist()]
        n = abs(gs) * math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        f = min(1.0, top / (n + 1e-6))
        norm.fill_(n)
        with torch.no_grad():
            for g, (_, _, off, _) in zip(grads, rows.tolist()):
                s = slice(off, off + g.numel())
                d = f * gs * g.reshape(-1) + wd * flat_param[s]
                flat_buf[s] = mu * flat_buf[s] + d
                flat_param[s] -= lr * flat_buf[s]
        return True

    def _mx4_chk(self, what, *tensors):
        return torch.device('cpu')

    @staticmethod
    def _quantise(a):
        code, scale, _ = oracle.quantise(a)
        return oracle.pack(code, scale)

    @staticmethod
    def _values(pair, rows, cols):
        code, scale, clean = oracle.unpack(pair[0], pair[1], rows, cols)
        assert clean
        x = np.repeat(np.exp2(scale.astype(np.float64) - 127), 32, axis=1)[:, :cols]
        x = np.where(np.repeat(scale == 255, 32, axis=1)[:, :cols], np.nan, x)
        return torch.from_numpy(oracle.VALUES[code & 7] * np.where(code & 8, -1.0, 1.0) * x)

    def mx4_quantize(self, x, along_rows, along_cols, col_sums=False):
        a = oracle.to64(x)
        return (self._quantise(a) if along_rows else None, self._quantise(np.ascontiguousarray(a.T)) if along_cols else None,
                x.double().sum(0).float() if col_sums else None)

    def mx4_dequantize(self, codes, scales, rows, cols, transposed, dtype):
        v = self._values((codes, scales), rows, cols)
        return (v.t() if transposed else v).contiguous().to(dtype)

    def mx4_matmul(self, a, b, m, n, k, bias, dtype):
        y = self._values(a, m, k) @ self._values(b, n, k).t()
        return (y if bias is None else y + bias.double()).to(dtype)

    def mx4_linear_fwd(self, x, w, kept, bias, need_dx, need_dw):
        m, k = x.shape
        n = w.shape[0] if kept is None else kept[2]
        wq = self.mx4_quantize(w, True, False)[0] if kept is None else kept[:2]
        y = self.mx4_matmul(self.mx4_quantize(x, True, False)[0], wq, m, n, k, bias, x.dtype)
        saved = None
        if need_dx or need_dw:
            saved = torch.cat([x.detach().reshape(-1).double(), w.detach().reshape(-1).double()])
        return y, saved

    def mx4_linear_bwd(self, dy, saved, k, need_dx, need_dw, dx_type, dw_type, want_db):
        m, n = dy.shape
        v = lambda t, dim: torch.from_numpy(np.ascontiguousarray(oracle.values(t, dim)))
        dx = dw = None
        if need_dx:
            dx = (v(dy, 1) @ v(saved[m * k:].reshape(n, k), 0)).to(dx_type)
        if need_dw:
            dw = (v(dy, 0).t() @ v(saved[:m * k].reshape(m, k), 0)).to(dw_type)
        return dx, dw, (dy.double().sum(0).float() if want_db else None)
