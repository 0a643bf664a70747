"""Gradients of the 8-bit products in every type, with rows that lie apart, on
one another or on no 16-byte boundary, with no rows or outputs, on streams of
their own.  Tolerances as in test_gpu_scaled.py."""
import pytest
import torch

import operator_refs as R
from test_gpu_scaled import BF16, FP16, FP32, randn, tol

pytestmark = pytest.mark.gpu


def compare(dy, x, w, **kw):
    from libnrn_b200 import scaled
    dx, dw = scaled.product_backward(dy, x, w, **kw)
    m, n, k = dy.shape[0], dy.shape[1], x.shape[1]
    assert dx.shape == (m, k) and dx.dtype == (kw.get("dx_dtype") or dy.dtype)
    assert dw.shape == (n, k) and dw.dtype == kw.get("dw_dtype", FP32)
    wd = R.dequantized(w.values, w.scales, 128)
    rdx = R.dequantized(*R.quantized(dy)) @ wd
    rdw = R.dequantized(*R.quantized(dy.t())) @ R.dequantized(*R.quantized(x.t())).t()
    assert R.rel(dx, rdx) <= tol(dx.dtype, n), R.rel(dx, rdx)
    assert R.rel(dw, rdw) <= tol(dw.dtype, m), R.rel(dw, rdw)
    return dx, dw


def test_no_outputs_no_rows():
    """Empty sums are zero, also where a projection has no outputs."""
    from libnrn_b200 import scaled
    trash = torch.full((1 << 16,), float("nan"), device="cuda")
    del trash                                        # what an unwritten result would show
    none = scaled.quantize(torch.empty(0, 64, device="cuda"), row_block=128)
    dx, dw = scaled.product_backward(torch.empty(50, 0, device="cuda"), randn(50, 64), none)
    assert torch.equal(dx, torch.zeros(50, 64, device="cuda")) and dw.shape == (0, 64)
    trash = torch.full((1 << 16,), float("nan"), device="cuda")
    del trash
    w = scaled.quantize(randn(10, 64), row_block=128)
    dx, dw = scaled.product_backward(torch.empty(0, 10, device="cuda"), torch.empty(0, 64, device="cuda"), w)
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros(10, 64, device="cuda"))
    flat = scaled.Scaled.empty(10, 0, torch.device("cuda", torch.cuda.current_device()), 128)
    dx, dw = scaled.product_backward(randn(5, 10), torch.empty(5, 0, device="cuda"), flat)
    assert dx.shape == (5, 0) and dw.shape == (10, 0)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_one_row_for_all(dtype):
    """Rows that are one (a stride of 0), as the gradient of a sum over rows is."""
    from libnrn_b200 import scaled
    m, n, k = 150, 200, 136
    w = scaled.quantize(randn(n, k, seed=3), row_block=128)
    x, dy = randn(1, k, seed=1, dtype=dtype).expand(m, k), randn(1, n, seed=2, dtype=dtype).expand(m, n)
    got, want = compare(dy, x, w), compare(dy.contiguous(), x.contiguous(), w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for kw in ({}, {"transpose": True}, {"row_block": 128}):
        a, b = scaled.quantize(x, **kw), scaled.quantize(x.contiguous(), **kw)
        assert torch.equal(a.dequantize(), b.dequantize())


@pytest.mark.parametrize("size", [(1, 64, 64), (130, 257, 384), (600, 1001, 136)], ids=str)
@pytest.mark.parametrize("dw_dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
def test_types(dtype, dw_dtype, size):
    from libnrn_b200 import scaled
    m, n, k = size
    w = scaled.quantize(randn(n, k, seed=3), row_block=128)
    x, dy = randn(m, k, seed=1, dtype=dtype), randn(m, n, seed=2, dtype=dtype)
    compare(dy, x, w, dw_dtype=dw_dtype)
    compare(dy, x, w, dw_dtype=dw_dtype, dx_dtype=FP32 if dtype != FP32 else BF16)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
def test_strides(dtype):
    from libnrn_b200 import scaled
    m, n, k = 300, 200, 328
    w = scaled.quantize(randn(n, k, seed=3), row_block=128)
    wide = randn(m, n + k + 40, seed=4, dtype=dtype)
    compare(wide[:, :n], wide[:, n + 8:n + 8 + k], w)                        # rows on 16 bytes, apart
    odd = randn(m, n + k + 41, seed=5, dtype=dtype)
    compare(odd[:, 1:n + 1], odd[:, n + 4:n + 4 + k], w)                     # and off
    v = torch.zeros(n, 400, device="cuda", dtype=torch.uint8)
    v[:, 16:16 + k] = w.values.view(torch.uint8)
    apart = scaled.Scaled(v.view(torch.float8_e4m3fn)[:, 16:16 + k], w.scales.contiguous(), 128)
    got, want = compare(wide[:, :n], wide[:, n + 8:n + 8 + k], apart), compare(wide[:, :n], wide[:, n + 8:n + 8 + k], w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_on_streams_of_their_own():
    from libnrn_b200 import scaled
    w = scaled.quantize(randn(256, 640, seed=7), row_block=128)
    pairs = [(randn(300, 256, seed=8 + i, dtype=BF16), randn(300, 640, seed=18 + i, dtype=BF16)) for i in range(2)]
    want = [scaled.product_backward(dy, x, w) for dy, x in pairs]
    streams = [torch.cuda.Stream() for _ in pairs]
    torch.cuda.synchronize()
    got = [[scaled.product_backward(dy, x, w, stream=s) for (dy, x), s in zip(pairs, streams)] for _ in range(10)]
    torch.cuda.synchronize()
    for round_ in got:
        assert all(torch.equal(a, b) for g, r in zip(round_, want) for a, b in zip(g, r))
    scaled.check()
