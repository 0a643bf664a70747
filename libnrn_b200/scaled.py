"""Matrix products in 8-bit floating point (e4m3) with a scale for each block
of 128 columns.

A ``Scaled`` matrix stands for values[r, c] * scales[r // row_block, c // 128].
Activations and gradients have a scale for each row (row_block 1), weights one
for each 128 x 128 block (row_block 128).  ``product`` is a @ b^T: 8-bit
products summed in fp32 within a block, scaled, and summed in fp32.

    w = scaled.quantize(weights, row_block=128)          # once
    y = scaled.product(scaled.quantize(x), w)            # x @ weights^T, bf16
    dx, dw = scaled.product_backward(dy, x, w)

What 8 bits save is memory: weights take half of bf16's.  In time a product
with its quantise is close to a bf16 one (8192 x 8192 over 4096 columns: 337 us
against 349, run for a second 383 against 398; three rows of 4096 x 4096 15
against 11), and both gradients are behind (4097 rows, 2048 x 4096: 170
against 98): they quantise and transpose first.

Results have no autograd graph: tensors that require gradients are refused
where these are recorded.  Calls on one stream share its workspace; threads
take turns at it.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _native as N
from ._tensors import DTYPE, Layouts, after_timeout, check_gradient, check_tensor, check_waits, error_flag, layout, on, require, share

BLOCK = 128


def _describe(values, scales, row_block):
    """The checked description of a matrix, without its pointers."""
    require(row_block in (1, BLOCK), f"row_block: must be 1 or {BLOCK}, is {row_block}")
    require(values.dim() == 2, "values: must be a matrix")
    check_tensor(values, "values", torch.float8_e4m3fn, values.device)
    rows, cols = values.shape
    check_tensor(scales, "scales", torch.float32, values.device, (-(-rows // row_block), -(-cols // BLOCK)))
    require(cols <= 1 or values.stride(1) == 1, "values: the last dimension must have stride 1")
    stride = values.stride(0)
    if rows <= 1 or cols == 0:           # the stride of a single row or of empty ones says nothing
        stride = -(-max(cols, 1) // 16) * 16
    require(stride % 16 == 0 and stride >= cols, "values: rows must start on 16-byte boundaries (Scaled.empty allocates them so)")
    d = N.Scaled()
    d.rows, d.cols, d.value_stride, d.row_block = rows, cols, stride, row_block
    d.scale_stride[0], d.scale_stride[1] = scales.stride(0), scales.stride(1)
    return bytes(d)


_matrices = Layouts(_describe)


def _describe_empty(rows, cols, row_block):
    """(bytes, where the scales start, row pitch, shape of the scales, description) of a matrix of Scaled.empty."""
    require(row_block in (1, BLOCK), f"row_block: must be 1 or {BLOCK}, is {row_block}")
    pitch, shape = -(-max(cols, 1) // 16) * 16, (-(-rows // row_block), -(-cols // BLOCK))
    at = -(-rows * pitch // 16) * 16
    d = N.Scaled()
    d.rows, d.cols, d.value_stride, d.row_block = rows, cols, pitch, row_block
    d.scale_stride[0], d.scale_stride[1] = 1, max(shape[0], 1)
    return max(at + 4 * shape[0] * shape[1], 16), at, pitch, shape, bytes(d)


_empties = Layouts(_describe_empty)


class Scaled:
    """``values`` (float8_e4m3fn [rows, cols], rows 16-byte aligned) and their ``scales`` (fp32
    [ceil(rows / row_block), ceil(cols / 128)], any strides).  ``quantize`` makes one; values and scales of a checkpoint
    can be given as they are."""

    __slots__ = ("_values", "_scales", "_base", "_at", "_pitch", "_scale_shape", "row_block", "desc", "shape", "device")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, row_block: int = 1):
        require(isinstance(values, torch.Tensor) and values.is_cuda, "values: a CUDA matrix is needed")
        block = _matrices.get((layout(values), layout(scales), row_block), values, scales, row_block)
        self._base, self._values, self._scales, self.row_block = None, values, scales, row_block
        self.shape, self.device = values.shape, values.device
        at = values.data_ptr()
        require(at % 16 == 0, "values: rows must start on 16-byte boundaries (Scaled.empty allocates them so)")
        self.desc = N.Scaled.from_buffer_copy(block)
        self.desc.values, self.desc.scales = at, scales.data_ptr()

    @classmethod
    def empty(cls, rows: int, cols: int, device, row_block: int = 1) -> "Scaled":
        """A matrix to be filled: one allocation, of which ``values`` and ``scales`` are views."""
        n, at, pitch, scale_shape, block = _empties.get((rows, cols, row_block), rows, cols, row_block)
        new = object.__new__(cls)
        new._base = base = torch.empty_strided((n,), (1,), dtype=torch.uint8, device=device)
        new._values = new._scales = None
        new._at, new._pitch, new._scale_shape = at, pitch, scale_shape
        new.row_block, new.shape, new.device = row_block, torch.Size((rows, cols)), base.device
        d = new.desc = N.Scaled.from_buffer_copy(block)
        p = base.data_ptr()
        d.values, d.scales = p, p + at
        return new

    @property
    def values(self) -> torch.Tensor:
        if self._values is None:
            rows, cols = self.shape
            self._values = self._base[:rows * self._pitch].view(torch.float8_e4m3fn).view(rows, self._pitch)[:, :cols]
        return self._values

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            # scales of neighbouring rows next to each other: as the product's threads read them
            rows, cols = self._scale_shape
            self._scales = self._base[self._at:self._at + 4 * rows * cols].view(torch.float32).view(cols, rows).t()
        return self._scales

    def memory(self) -> tuple:
        """The tensors that hold it."""
        return (self._values, self._scales) if self._base is None else (self._base,)

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """What the matrix stands for, by torch operations (for checks and export)."""
        rows, cols = self.shape
        s = self.scales.repeat_interleave(self.row_block, 0)[:rows] if self.row_block > 1 else self.scales
        return (self.values.float() * s.repeat_interleave(BLOCK, 1)[:, :cols]).to(dtype)


def _describe_quantize(x, row_block, transpose):
    require(x.dim() == 2, "x: must be a matrix")
    check_gradient(x, "x")
    require(x.dtype in DTYPE, f"x: must be bfloat16, float16 or float32, is {x.dtype}")
    require(row_block in (1, BLOCK), f"row_block: must be 1 or {BLOCK}, is {row_block}")
    rows, cols = x.shape
    require(cols <= 1 or x.stride(1) == 1, f"x: the last dimension must have stride 1, has {x.stride(1)}")
    require(not transpose or row_block == 1, "transpose: only with a scale for each row")
    return DTYPE[x.dtype], rows, cols, x.stride(0) if rows > 1 else max(cols, 1)


_quantized = Layouts(_describe_quantize)


def quantize(x: torch.Tensor, *, row_block: int = 1, transpose: bool = False, stream=None) -> Scaled:
    """x (bf16, fp16 or fp32 [rows, cols], last stride 1, rows anywhere) in 8 bits.  A block's scale is its largest magnitude / 448; an
    infinity or NaN makes its whole block NaN.  ``transpose`` gives x^T with a scale for each of its rows (row_block 1)."""
    require(isinstance(x, torch.Tensor) and x.is_cuda, "x: a CUDA tensor is needed")
    dtype, rows, cols, stride = _quantized.get((layout(x), row_block, transpose), x, row_block, transpose)
    dev = x.device
    with on(dev, stream) as st:
        out = Scaled.empty(cols, rows, dev) if transpose else Scaled.empty(rows, cols, dev, row_block)
        N.check(N.lib().nrn_cuda_scaled_quantize(x.data_ptr(), dtype, rows, cols, stride, int(transpose), C.byref(out.desc), st),
                "nrn_cuda_scaled_quantize")
    if stream is not None:
        share(stream, dev, (x,), out.memory())
    return out


def transpose(w: Scaled, *, stream=None) -> Scaled:
    """w^T of weights (row_block 128): the same values and scales."""
    require(isinstance(w, Scaled) and w.row_block == BLOCK, "w: must be Scaled with a row_block of 128")
    rows, cols = w.shape
    with on(w.device, stream) as st:
        pitch = -(-rows // 16) * 16
        values = torch.empty(cols, pitch, dtype=torch.float8_e4m3fn, device=w.device)
        out = Scaled(values[:, :rows], w.scales.t(), BLOCK)
        N.check(N.lib().nrn_cuda_scaled_transpose(C.byref(w.desc), C.byref(out.desc), st), "nrn_cuda_scaled_transpose")
    if stream is not None:
        share(stream, w.device, w.memory(), (values,))
    return out


_COUNTERS = 4096        # bytes at a workspace's start that are zero between calls


class _Stream:
    """What calls on one stream share: their workspace (they follow one another there), and whose turn it is to enqueue.  The
    library lets other threads run while it launches: without turns another thread's kernels could come between those of
    one call and overwrite what they hand on, or free the workspace before they are in the stream."""

    __slots__ = ("turn", "work")

    def __init__(self):
        self.turn, self.work = threading.Lock(), None

    def workspace(self, n: int, device) -> torch.Tensor:
        """n bytes; for the thread whose turn it is, which keeps hold of them until its launches are made."""
        capturing = torch.cuda.is_current_stream_capturing()     # then it belongs to the graph
        w = None if capturing else self.work
        if w is None or w.numel() < n:
            w = torch.empty(max(n, _COUNTERS), dtype=torch.uint8, device=device)
            w[:_COUNTERS].zero_()
            if not capturing:
                self.work = w
        return w


_streams: dict = {}


def _on_stream(device, stream: int) -> _Stream:
    key = (device.index, stream)
    return _streams.get(key) or _streams.setdefault(key, _Stream())


def _drop_workspaces(index: int) -> None:
    """A product that gave up leaves counters above zero: the next one on its stream gets a new workspace."""
    for (i, _), shared in list(_streams.items()):
        if i == index:
            with shared.turn:
                shared.work = None


after_timeout.append(_drop_workspaces)


check = check_waits


def _describe_product(a, b, dtype, out):
    """(type, row stride of the result, bytes of workspace)."""
    m, n = a.shape[0], b.shape[0]
    require(a.device == b.device, f"b: must be on {a.device}, is on {b.device}")
    require(a.shape[1] == b.shape[1], f"b: has {b.shape[1]} columns, a has {a.shape[1]}")
    if out is not None:
        require(isinstance(out, torch.Tensor) and out.dtype in DTYPE, "out: must be bfloat16, float16 or float32")
        check_tensor(out, "out", out.dtype, a.device, (m, n))
        require(n <= 1 or out.stride(1) == 1, "out: the last dimension must have stride 1")
        require(m <= 1 or out.stride(0) >= n, "out: rows overlap")
        dtype = out.dtype
    require(dtype in DTYPE, f"dtype: must be bfloat16, float16 or float32, is {dtype}")
    need = C.c_int64()
    N.check(N.lib().nrn_cuda_scaled_workspace(C.byref(a.desc), C.byref(b.desc), C.byref(need)), "nrn_cuda_scaled_workspace")
    return DTYPE[dtype], out.stride(0) if out is not None and m > 1 else max(n, 1), need.value


_products = Layouts(_describe_product)


def product(a: Scaled, b: Scaled, *, dtype=torch.bfloat16, out=None, stream=None) -> torch.Tensor:
    """a @ b^T, [a rows, b rows], in ``dtype`` (bf16, fp16 or fp32)."""
    require(isinstance(a, Scaled) and isinstance(b, Scaled), "a, b: must be Scaled (scaled.quantize)")
    dev = a.device
    key, given = (a.shape, b.shape, dev, b.device, dtype, layout(out)), out
    with on(dev, stream) as st:
        kind, stride, need = _products.get(key, a, b, dtype, out)
        if out is None:
            n = b.shape[0]
            out = torch.empty_strided((a.shape[0], n), (n, 1), dtype=dtype, device=dev)
        if need:
            shared = _on_stream(dev, st)
            with shared.turn:
                w = shared.workspace(need, dev)
                s = N.lib().nrn_cuda_scaled_product(C.byref(a.desc), C.byref(b.desc), out.data_ptr(), kind, stride, w.data_ptr(), need, error_flag(dev), st)
        else:
            s = N.lib().nrn_cuda_scaled_product(C.byref(a.desc), C.byref(b.desc), out.data_ptr(), kind, stride, None, 0, error_flag(dev), st)
        N.check(s, "nrn_cuda_scaled_product")
    if stream is not None:
        share(stream, dev, (*a.memory(), *b.memory(), given), (out,))
    return out


def _describe_backward(dy, x, w, dx_dtype, dw_dtype):
    """(row strides of dy and x, their type, types of the results, bytes of workspace)."""
    require(w.row_block == BLOCK, "w: must be Scaled with a row_block of 128")
    for name, t, cols in (("dy", dy, w.shape[0]), ("x", x, w.shape[1])):
        require(isinstance(t, torch.Tensor) and t.dim() == 2 and t.shape[1] == cols, f"{name}: must be [rows, {cols}]")
        check_tensor(t, name, dy.dtype, w.device)
        require(cols <= 1 or t.stride(1) == 1, f"{name}: the last dimension must have stride 1")
    rows = dy.shape[0]
    require(rows == x.shape[0], f"dy: has {rows} rows, x has {x.shape[0]}")
    for name, t in (("dy", dy.dtype), ("dx_dtype", dx_dtype), ("dw_dtype", dw_dtype)):
        require(t in DTYPE, f"{name}: must be bfloat16, float16 or float32, is {t}")
    need, zeroed = C.c_int64(), C.c_int64()
    N.check(N.lib().nrn_cuda_scaled_backward_workspace(rows, C.byref(w.desc), C.byref(need), C.byref(zeroed)),
            "nrn_cuda_scaled_backward_workspace")
    return (rows, *(t.stride(0) if rows > 1 else max(t.shape[1], 1) for t in (dy, x)), DTYPE[dy.dtype], DTYPE[dx_dtype], DTYPE[dw_dtype],
            need.value)


_backwards = Layouts(_describe_backward)


def product_backward(dy: torch.Tensor, x: torch.Tensor, w: Scaled, *, dx_dtype=None, dw_dtype=torch.float32, stream=None):
    """(dx, dw) of y = x @ w^T: dx = dy @ w and dw = dy^T @ x, with dy and x quantised along the axis that each of the two
    sums over (dy's rows for dx; the columns of dy and x for dw)."""
    require(isinstance(w, Scaled), "w: must be Scaled with a row_block of 128")
    require(isinstance(dy, torch.Tensor) and dy.is_cuda, "dy: a CUDA tensor is needed")
    dx_dtype = dx_dtype or dy.dtype
    key = (layout(dy), layout(x), w.shape, w.row_block, w.device, dx_dtype, dw_dtype)
    dev, (n, k) = w.device, w.shape
    with on(dev, stream) as st:
        rows, dy_stride, x_stride, kind, dx_kind, dw_kind, need = _backwards.get(key, dy, x, w, dx_dtype, dw_dtype)
        dx = torch.empty_strided((rows, k), (k, 1), dtype=dx_dtype, device=dev)
        dw = torch.empty_strided((n, k), (k, 1), dtype=dw_dtype, device=dev)
        shared = _on_stream(dev, st)
        with shared.turn:
            work = shared.workspace(need, dev)
            s = N.lib().nrn_cuda_scaled_backward(dy.data_ptr(), x.data_ptr(), kind, rows, dy_stride, x_stride, C.byref(w.desc), dx.data_ptr(),
                                                 dx_kind, dw.data_ptr(), dw_kind, work.data_ptr(), need, error_flag(dev), st)
        N.check(s, "nrn_cuda_scaled_backward")
    if stream is not None:
        share(stream, dev, (dy, x, *w.memory()), (dx, dw))
    return dx, dw
