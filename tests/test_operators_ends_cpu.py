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


def test_steps_of_states_that_overlap():
    a = N.LinAttn()
    a.dtype, a.seqs, a.heads, a.kv_heads, a.dk, a.dv, a.tokens, a.scale, a.log_decay = 0, 0, 4, 2, 8, 16, 1, 1.0, 256
    step = lambda stride, n: N.lib().nrn_cuda_linattn_step(C.byref(a), 256, stride, n, None, None)      # noqa: E731
    assert step(0, 2) == 1 and step(511, 2) == 1 and b"one another" in N.lib().nrn_last_error()
    assert step(512, 2) == 0 and step(0, 1) == 0


def test_flag_of_no_device():
    p = C.c_void_p()
    for device in (-1, 64):
        assert N.lib().nrn_cuda_wait_flag(device, C.byref(p)) == 1 and p.value is None
    assert N.lib().nrn_cuda_wait_flag(0, None) == 1
