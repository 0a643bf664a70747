"""What the operators refuse at their ends, before anything is launched: no GPU needed."""
import ctypes as C

from libnrn_b200 import _native as N


def weights(rows=10, cols=64):
    d = N.Scaled()
    d.values, d.scales, d.rows, d.cols, d.value_stride, d.row_block = 256, 256, rows, cols, max(cols, 16), 128
    d.scale_stride[0], d.scale_stride[1] = 1, 1
    return d


def test_gradients_of_an_unknown_type():
    def backward(dx, dw, w):
        return N.lib().nrn_cuda_scaled_backward(None, None, 0, 0, 0, 0, C.byref(w), None, dx, 256, dw, None, 0, None, None)
    for w in (weights(), weights(rows=0), weights(cols=0)):
        assert backward(9, 0, w) == 1 and b"dx" in N.lib().nrn_last_error()
        assert backward(0, -1, w) == 1 and b"dw" in N.lib().nrn_last_error()
    assert backward(0, 0, weights(rows=0)) == 0 and backward(0, 0, weights(cols=0)) == 0
