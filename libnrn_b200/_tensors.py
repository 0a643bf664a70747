"""What the tensor operators (linattn, scaled, gatednorm) share: types, the
checks of their tensor arguments, and the device and stream of a call.

A call's checks depend on its arguments' layouts alone (shapes, strides,
types, devices), so each operator keeps the outcome by layout: a later call
with the same layouts fills a copy of the checked argument block with its
pointers (``Layouts``)."""
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


_recorded = torch.is_grad_enabled


def check_gradient(t, name: str) -> None:
    """The operators' results have no graph: a gradient would be lost without a word."""
    require(not (t.requires_grad and _recorded()), f"{name}: requires a gradient, which this call does not record: call it under torch.no_grad() and use the "
                                   "operator's backward")


def check_tensor(t, name: str, dtype, device, shape=None) -> None:
    require(isinstance(t, torch.Tensor), f"{name}: a tensor is needed")
    check_gradient(t, name)
    require(t.is_cuda and t.device == device, f"{name}: must be on {device}, is on {t.device}")
    require(t.dtype == dtype, f"{name}: must be {dtype}, is {t.dtype}")
    if shape is not None:
        require(tuple(t.shape) == tuple(shape), f"{name}: shape must be {tuple(shape)}, is {tuple(t.shape)}")


def check_rows(t, name: str, dtype, device, shape) -> None:
    """A tensor whose innermost elements are next to each other; the other strides are free."""
    check_tensor(t, name, dtype, device, shape)
    require(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: the last dimension must have stride 1, has {t.stride(-1)}")


def check_result(t, name: str, dtype, device, shape) -> None:
    """Rows that are written: no two elements at one place (each dimension steps over what lies inside it)."""
    check_rows(t, name, dtype, device, shape)
    inside = 1
    for stride, n in sorted((t.stride(i), n) for i, n in enumerate(t.shape) if n > 1):
        require(stride >= inside, f"{name}: elements lie on one another")
        inside += (n - 1) * stride


def check_vector(t, name: str, n: int, device) -> None:
    check_tensor(t, name, torch.float32, device, (n,))
    require(t.is_contiguous(), f"{name}: must be contiguous")


def check_state(t, name: str, device, shape) -> None:
    check_tensor(t, name, torch.float32, device, shape)
    require(t.is_contiguous(), f"{name}: must be contiguous")


def ptr(t):
    return None if t is None else t.data_ptr()


def number(x):
    """x as a Python number, read at every call: a tensor would stand in a key for what it held at its first use."""
    return x if x is None or type(x) is float else float(x)


def layout(t):
    """All of a tensor argument that its checks look at (None and anything else stand for themselves)."""
    if t is None:
        return None
    try:
        return t.shape, t.stride(), t.dtype, t.device, t.requires_grad and _recorded()
    except AttributeError:               # no tensor
        return type(t)


class Layouts:
    """Checked argument blocks by the layouts they were checked for."""

    def __init__(self, build, most: int = 4096):
        self.build, self.most, self.known = build, most, {}

    def get(self, key, *args):
        """What ``build(*args)`` gives for these layouts; it raises where they are refused."""
        got = self.known.get(key)
        if got is None:
            got = self.build(*args)
            if len(self.known) >= self.most:
                self.known.clear()
            self.known[key] = got
        return got


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


@contextlib.contextmanager
def _switched(device, stream):
    with torch.cuda.device(device):
        if stream is None:
            yield _raw_stream(device.index)
        else:
            with torch.cuda.stream(stream):
                yield stream.cuda_stream


class _Current:
    """The context of a call on the current device and stream: nothing to switch."""

    __slots__ = ("stream",)

    def __init__(self, stream):
        self.stream = stream

    def __enter__(self):
        return self.stream

    def __exit__(self, *exc):
        return False


def on(device, stream=None):
    """Context of a call on `device`: its kernels, results and workspaces belong to `stream` (default: the current one),
    whose handle it gives."""
    i = device.index
    if stream is None and _current_device() == i:
        return _Current(_raw_stream(i))
    if stream is not None:
        require(stream.device == device, f"stream: must be of {device}, is of {stream.device}")
    return _switched(device, stream)


def share(stream, device, inputs, results) -> None:
    """After a call on a stream of the caller's choice: the memory of its inputs, should they be dropped, is not given out again
    before that stream is past the call, nor that of its results before the current stream is past what it does with them."""
    here = torch.cuda.current_stream(device)
    if stream.cuda_stream == here.cuda_stream:
        return
    for of, tensors in ((stream, inputs), (here, results)):
        for t in tensors:
            if t is not None:
                t.record_stream(of)


class _Flag:
    """A device's word that kernels set when one of their bounded waits gives up, and the same as a tensor.  The library
    makes it: made here by the first call it could become part of a graph that is being captured, whose replays would clear
    it."""

    def __init__(self, index: int):
        p = C.c_void_p()
        N.check(N.lib().nrn_cuda_wait_flag(index, C.byref(p)), "nrn_cuda_wait_flag")
        self.index, self.address = index, p.value
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (p.value, False), "version": 2}

    def tensor(self) -> torch.Tensor:
        return torch.as_tensor(self, device=torch.device("cuda", self.index))


_flags: dict = {}


def flag(index: int) -> _Flag:
    f = _flags.get(index)
    if f is None:
        f = _flags[index] = _Flag(index)
    return f


def error_flag(device) -> int:
    """Address of the device's flag."""
    i = device.index
    return (_flags.get(i) or flag(i)).address


# Called with a device's index when a wait there gave up: what later calls would take over from the unfinished ones.
after_timeout: list = []


def check_waits(device=None) -> None:
    """Raises if a device-side wait of an earlier call on `device` (default: the current one) gave up.  Waits for the GPU.
    What gave up is told once: the flag is down afterwards and later calls start afresh.  Results of the calls before, and
    graphs that were captured, are the caller's to make again."""
    i = None if device is None else torch.device(device).index
    i = torch.cuda.current_device() if i is None else i
    f = _flags.get(i)
    if f is None:
        return
    torch.cuda.synchronize(i)            # a call on any stream
    code = int(f.tensor().item())
    if code != 0:
        for drop in after_timeout:
            drop(i)
        f.tensor().zero_()
        torch.cuda.synchronize(i)
        raise N.NrnError(7, f"a device-side wait timed out (code {code})")
