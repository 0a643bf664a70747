"""What the tensor operators (linattn, scaled, gatednorm) share: types, the
checks of their tensor arguments, and the device and stream of a call."""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _native as N

DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def require(cond: bool, msg: str) -> None:
    """Refuses an argument as the library does: NrnError with its status."""
    if not cond:
        raise N.NrnError(1, msg)


def check_tensor(t, name: str, dtype, device, shape=None) -> None:
    require(isinstance(t, torch.Tensor), f"{name}: a tensor is needed")
    require(t.is_cuda and t.device == device, f"{name}: must be on {device}, is on {t.device}")
    require(t.dtype == dtype, f"{name}: must be {dtype}, is {t.dtype}")
    if shape is not None:
        require(tuple(t.shape) == tuple(shape), f"{name}: shape must be {tuple(shape)}, is {tuple(t.shape)}")


def check_rows(t, name: str, dtype, device, shape) -> None:
    """A tensor whose innermost elements are next to each other; the other strides are free."""
    check_tensor(t, name, dtype, device, shape)
    require(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: the last dimension must have stride 1, has {t.stride(-1)}")


def check_vector(t, name: str, n: int, device) -> None:
    check_tensor(t, name, torch.float32, device, (n,))
    require(t.is_contiguous(), f"{name}: must be contiguous")


def check_state(t, name: str, device, shape) -> None:
    check_tensor(t, name, torch.float32, device, shape)
    require(t.is_contiguous(), f"{name}: must be contiguous")


def ptr(t):
    return None if t is None else t.data_ptr()


@contextlib.contextmanager
def _switched(device, stream):
    with torch.cuda.device(device):
        if stream is None:
            yield C.c_void_p(torch.cuda.current_stream().cuda_stream)
        else:
            with torch.cuda.stream(stream):
                yield C.c_void_p(stream.cuda_stream)


class _Current:
    """The context of a call on the current device and stream: nothing to switch."""

    def __enter__(self):
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)

    def __exit__(self, *exc):
        return False


_CURRENT = _Current()


def on(device, stream=None):
    """Context of a call on `device`: its kernels, results and workspaces belong to `stream` (default: the current one)."""
    if stream is None and torch.cuda.current_device() == device.index:
        return _CURRENT
    return _switched(device, stream)


# A flag on each device that kernels set when one of their bounded waits gives up.
_errors: dict = {}


def error_flag(device) -> int:
    """Address of the device's flag."""
    t = _errors.get(device.index)
    if t is None:
        t = _errors[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
    return t.data_ptr()


def check_waits(device=None) -> None:
    """Raises if a device-side wait of an earlier call on `device` (default: the current one) gave up.  Waits for the GPU."""
    i = torch.cuda.current_device() if device is None else torch.device(device).index
    t = _errors.get(i)
    if t is not None and int(t.item()) != 0:
        raise N.NrnError(7, f"a device-side wait timed out (code {int(t.item())})")
