"""Gradients of the 8-bit products at their ends (test_gpu_scaled.py has the
tolerances)."""
import pytest
import torch

import operator_refs as R
from test_gpu_scaled import BF16, FP32, randn, tol

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
