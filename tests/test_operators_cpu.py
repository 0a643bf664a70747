"""What the sequence-memory operators refuse before anything is launched, and
the 64-bit forms of their gradients against differences: no GPU needed."""
import ctypes as C

import pytest
import torch

import operator_refs as R
from libnrn_b200 import _native as N


def linattn(**kw):
    a = N.LinAttn()
    a.dtype, a.seqs, a.heads, a.kv_heads, a.dk, a.dv, a.tokens, a.scale, a.log_decay = 0, 1, 4, 2, 64, 64, 10, 1.0, 256
    a.q = a.k = a.v = a.o = 256
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(seqs=-1), dict(tokens=-1), dict(heads=0), dict(kv_heads=3), dict(dk=0), dict(dk=257), dict(dv=257),
                                 dict(scale=0.0), dict(scale=float("inf")), dict(log_decay=None), dict(q=None), dict(o=None)], ids=str)
def test_linattn_refuses(bad):
    assert N.lib().nrn_cuda_linattn_forward(C.byref(linattn(**bad)), None) == 1
    assert b"nrn_cuda_linattn_forward" in N.lib().nrn_last_error()


def test_linattn_refuses_null_and_steps():
    L = N.lib()
    assert L.nrn_cuda_linattn_forward(None, None) == 1
    assert L.nrn_cuda_linattn_backward(C.byref(linattn()), None, None) == 1
    assert L.nrn_cuda_linattn_step(C.byref(linattn()), 256, 0, 1, None, None) == 1             # ten tokens
    assert L.nrn_cuda_linattn_step(C.byref(linattn(tokens=1, seqs=3)), 256, 0, 2, None, None) == 1   # two states
    assert L.nrn_cuda_linattn_step(C.byref(linattn(tokens=1)), None, 0, 1, None, None) == 1
    assert L.nrn_cuda_linattn_forward(C.byref(linattn(seqs=0)), None) == 0                     # nothing to do


def matrix(**kw):
    d = N.Scaled()
    d.values, d.scales, d.rows, d.cols, d.value_stride, d.row_block = 256, 256, 10, 100, 112, 1
    for n, v in kw.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=1 << 40), dict(row_block=2), dict(values=None), dict(scales=None), dict(values=8), dict(value_stride=100),
                                 dict(value_stride=96)], ids=str)
def test_scaled_refuses(bad):
    L = N.lib()
    a, b = matrix(**bad), matrix()
    assert L.nrn_cuda_scaled_product(C.byref(a), C.byref(b), 256, 0, 10, None, 0, None, None) == 1
    assert L.nrn_cuda_scaled_product(C.byref(b), C.byref(a), 256, 0, 10, None, 0, None, None) == 1
    assert L.nrn_cuda_scaled_quantize(256, 0, 10, 100, 100, 0, C.byref(a), None) == 1


def test_scaled_refuses_shapes():
    L = N.lib()
    a, b = matrix(), matrix(cols=99)
    assert L.nrn_cuda_scaled_product(C.byref(a), C.byref(b), 256, 0, 10, None, 0, None, None) == 1
    assert L.nrn_cuda_scaled_product(C.byref(a), C.byref(a), 256, 0, 9, None, 0, None, None) == 1
    assert L.nrn_cuda_scaled_product(C.byref(a), C.byref(a), 256, 9, 10, None, 0, None, None) == 1
    assert L.nrn_cuda_scaled_quantize(256, 0, 100, 10, 10, 0, C.byref(a), None) == 1
    assert L.nrn_cuda_scaled_transpose(C.byref(a), C.byref(a), None) == 1
    assert L.nrn_cuda_scaled_product(C.byref(matrix(rows=0)), C.byref(a), None, 0, 10, None, 0, None, None) == 0


def norm(**kw):
    a = N.GatedNorm()
    a.dtype, a.act, a.rows, a.d, a.eps, a.residual, a.h, a.y, a.z = 0, 0, 3, 64, 1e-6, 256, 256, 256, 256
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(act=2), dict(rows=-1), dict(d=0), dict(d=16385), dict(eps=-1.0), dict(eps=float("nan")), dict(residual=None),
                                 dict(h=None)], ids=str)
def test_gatednorm_refuses(bad):
    assert N.lib().nrn_cuda_gatednorm_forward(C.byref(norm(**bad)), None) == 1


def test_gatednorm_refuses_gradients():
    g = N.GatedNormGrad()
    assert N.lib().nrn_cuda_gatednorm_backward(C.byref(norm()), None, None) == 1
    g.dalpha = 256
    assert N.lib().nrn_cuda_gatednorm_backward(C.byref(norm(h=None, y=None)), C.byref(g), None) == 1


def test_recurrence_gradients_are_the_differences():
    g = torch.Generator().manual_seed(0)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    t, h, dk, dv = 9, 2, 5, 4
    x = {"q": r(t, h, dk), "k": r(t, h, dk), "v": r(t, h, dv), "s0": r(h, dk, dv)}
    do, ds, decay = r(t, h, dv), r(h, dk, dv), torch.tensor([-0.1, -0.7])

    def value(at):
        o, s = R.scan(at["q"], at["k"], at["v"], decay, 0.3, at["s0"])
        return float((o * do).sum() + (s * ds).sum())
    got = R.scan_backward(do, x["q"], x["k"], x["v"], decay, 0.3, x["s0"], ds)
    for n, d in zip(("q", "k", "v", "s0"), got):
        e = 1e-5 / float(d.norm())
        slope = (value({**x, n: x[n] + e * d}) - value({**x, n: x[n] - e * d})) / (2 * e)
        assert abs(slope - float(d.square().sum())) <= 1e-7 * abs(slope)
