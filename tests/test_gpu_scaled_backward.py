"""Gradients of the 8-bit products at their ends (test_gpu_scaled.py has the
tolerances)."""
import pytest
import torch

from test_gpu_scaled import randn

pytestmark = pytest.mark.gpu


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
