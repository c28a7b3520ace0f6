"""4-bit matrices, host side: sizes, refusals (C entries and public calls) before any launch."""
import pytest
import torch

from deepipr_amd import _lib, mx4


def test_sizes():
    lib = _lib.lib()
    assert [lib.deepipr_mx4_code_bytes(*s) for s in ((1, 1), (3, 128), (3, 129), (0, 5), (5, 0))] == [64, 192, 384, 0, 0]
    assert [lib.deepipr_mx4_scale_bytes(*s) for s in ((1, 1), (64, 128), (65, 129), (0, 5))] == [256, 256, 1024, 0]
    assert lib.deepipr_mx4_quantize_workspace_bytes(65, 10) == 2 * 10 * 4 and lib.deepipr_mx4_quantize_workspace_bytes(64 * 129, 10) == (130 + 2) * 10 * 4
    assert lib.deepipr_mx4_code_bytes(1 << 33, 200) == (1 << 33) * 128


def test_c_entries_refuse_before_any_launch():
    lib = _lib.lib()
    p = 1 << 12

    def quant(x=p, dtype=0, rows=4, cols=40, stride=40, rc=p, rs=p, cc=p, cs=p, sums=None, ws=None, n=0):
        return lib.deepipr_mx4_quantize(x, dtype, rows, cols, stride, rc, rs, cc, cs, sums, ws, n, None)
    for bad in (dict(x=None), dict(dtype=3), dict(rows=0), dict(cols=0), dict(rows=-1), dict(stride=39), dict(rc=None), dict(cs=None),
                dict(rc=None, rs=None, cc=None, cs=None), dict(x=p + 2), dict(rc=p + 8), dict(sums=p), dict(sums=p, ws=p, n=1),
                dict(sums=p, ws=p, n=1 << 20, cc=None, cs=None), dict(rows=1 << 41), dict(rows=1 << 27, cols=1 << 20, stride=1 << 20)):
        assert quant(**bad) == -1 and b'mx4_quantize' in lib.deepipr_last_error(), bad

    def deq(codes=p, scales=p, rows=4, cols=40, out=p, dtype=0):
        return lib.deepipr_mx4_dequantize(codes, scales, rows, cols, 0, out, dtype, None)
    for bad in (dict(codes=None), dict(scales=None), dict(out=None), dict(rows=0), dict(cols=0), dict(dtype=7), dict(codes=p + 4), dict(out=p + 2)):
        assert deq(**bad) == -1 and b'mx4_dequantize' in lib.deepipr_last_error(), bad

    def mm(a=p, sa=p, b=p, sb=p, bias=None, bt=0, m=4, n=5, k=6, out=p, dtype=0, ws=None, nbytes=0):
        return lib.deepipr_mx4_matmul(a, sa, b, sb, bias, bt, m, n, k, out, dtype, ws, nbytes, None)
    for bad in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(out=None), dict(m=0), dict(n=0), dict(k=0), dict(dtype=-1),
                dict(bias=p, bt=9), dict(a=p + 8), dict(bias=p + 1, bt=1), dict(out=p + 1, dtype=1), dict(m=1 << 41), dict(m=1 << 27, n=1 << 27),
                dict(n=1 << 27)):                                  # 2^23 workgroups of 512 threads: 2^32
        assert mm(**bad) == -1 and b'mx4_matmul' in lib.deepipr_last_error(), bad


def test_linear_entries_refuse_before_any_launch():
    lib = _lib.lib()
    p, big = 1 << 12, 1 << 30

    def fwd(x=p, xt=0, xs=70, w=p, wt=0, ws=70, wc=None, wsc=None, bias=None, bt=0, m=5, n=6, k=70, dx=1, dw=1, saved=p, sb=big, out=p, scratch=p, cb=big):
        return lib.deepipr_mx4_linear_fwd(x, xt, xs, w, wt, ws, wc, wsc, bias, bt, m, n, k, dx, dw, saved, sb, out, scratch, cb, None)
    for bad in (dict(x=None), dict(xt=3), dict(xs=69), dict(w=None), dict(w=None, wc=p, wsc=p), dict(w=None, wc=p, dx=0, dw=0), dict(wt=-1), dict(ws=1),
                dict(m=0), dict(n=0), dict(k=0), dict(out=None), dict(saved=None), dict(sb=1), dict(scratch=None), dict(cb=1), dict(scratch=p + 4),
                dict(bias=p, bt=5), dict(bias=p + 2), dict(m=1 << 41)):
        assert fwd(**bad) == -1 and b'mx4_linear_fwd' in lib.deepipr_last_error(), bad

    def bwd(dy=p, t=0, s=6, m=5, n=6, k=70, ndx=1, ndw=1, saved=p, sb=big, dx=p, dxt=0, dw=p, dwt=0, db=p, scratch=p, cb=big):
        return lib.deepipr_mx4_linear_bwd(dy, t, s, m, n, k, ndx, ndw, saved, sb, dx, dxt, dw, dwt, db, scratch, cb, None)
    for bad in (dict(dy=None), dict(t=4), dict(s=5), dict(m=0), dict(n=-1), dict(k=0), dict(ndx=0), dict(ndw=0), dict(saved=None), dict(sb=7), dict(dxt=9),
                dict(dwt=3), dict(db=p + 2), dict(dx=None, dw=None, db=None), dict(scratch=None), dict(cb=3)):
        assert bwd(**bad) == -1 and b'mx4_linear_bwd' in lib.deepipr_last_error(), bad
    assert lib.deepipr_mx4_linear_saved_bytes(5, 6, 70, 0, 0) == 0 and lib.deepipr_mx4_linear_scratch_bytes(0, 6, 70, 0) == 0
    # kept weights: none for rows that their product quantises (up to 4096 bytes x blocks), no room for the weight's codes otherwise
    assert lib.deepipr_mx4_linear_kept_scratch_bytes(0, 1, 6, 9216) == lib.deepipr_mx4_linear_kept_scratch_bytes(1, 16, 6, 4096) == 0
    assert 0 < lib.deepipr_mx4_linear_kept_scratch_bytes(0, 16, 600, 4096) < lib.deepipr_mx4_linear_scratch_bytes(16, 600, 4096, 0)
    assert fwd(w=None, wc=p, wsc=p, dx=0, dw=0, m=17, cb=1) == -1 and b'scratch' in lib.deepipr_last_error()
    assert lib.deepipr_mx4_linear_saved_bytes(5, 6, 70, 1, 1) == 2 * lib.deepipr_mx4_linear_saved_bytes(5, 6, 70, 1, 0)
    assert lib.deepipr_mx4_matmul_workspace_bytes(128, 128, 20000) > 0 == lib.deepipr_mx4_matmul_workspace_bytes(64, 128, 20000)


def test_host_tensors_and_shapes_are_refused():
    x = torch.ones(4, 40)
    for call in (lambda: mx4.quantize(x), lambda: mx4.quantize_both(x), lambda: mx4.linear(x, x), lambda: mx4.quantize(x[:0])):
        with pytest.raises(RuntimeError, match='GPU only'):
            call()
    for bad in (x[0], x[None], x.sum()):
        with pytest.raises(ValueError, match='matrix'):
            mx4.quantize(bad)
    with pytest.raises(ValueError, match='dim'):
        mx4.quantize(x, 2)
    with pytest.raises(TypeError):
        mx4.quantize([1.0])
    with pytest.raises(ValueError, match='features'):
        mx4.linear(x, x[:, :3])
    with pytest.raises(ValueError, match='bias'):
        mx4.linear(x, x, x[0])


def test_empty_host_tensors_are_refused_too():
    x, w = torch.ones(4, 40), torch.ones(3, 40)
    for a, b in ((x[:0], w), (x, w[:0]), (x[:, :0], w[:, :0])):
        for grad in (False, True):
            with pytest.raises(RuntimeError, match='GPU only'):
                mx4.linear(a, b.clone().requires_grad_(grad))
