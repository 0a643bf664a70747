"""The norms before and after a block with its gate and residual scale, in one
pass, and their gradients.  For rows of d elements, with
norm(x) = x / sqrt(mean(x^2) + eps):

    y = residual + alpha * act(gate) * norm(h) * w_post
    z = norm(y) * w_pre                         (what the next block reads)

h is the block's output; without it y is the residual and only z is computed.
gate (like h), alpha, w_post and w_pre (fp32 [d]) may be None: 1.  All sums
and z's input are fp32; y and z are rounded once.  Results have no autograd
graph: tensors that require gradients are refused where these are recorded.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _native as N
from ._tensors import DTYPE, Layouts, check_rows, check_vector, check_waits, error_flag, layout, number, on, ptr, require, share
from .scaled import Scaled

check = check_waits
ACTIVATION = {"silu": 0, "sigmoid": 1}


class Gradients(NamedTuple):
    residual: torch.Tensor
    h: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]
    alpha: Optional[torch.Tensor]
    w_post: Optional[torch.Tensor]
    w_pre: Optional[torch.Tensor]


def _stride(t):
    return 0 if t is None else t.stride(0)


def _describe(residual, h, gate, alpha, w_post, w_pre, eps, activation, dy, dz):
    """The checked argument block of a call (its pointers are set by each call), and the bytes of its backward's workspace."""
    require(residual.dim() == 2, "residual: must be [rows, d]")
    require(residual.dtype in DTYPE, f"residual: must be bfloat16, float16 or float32, is {residual.dtype}")
    require(activation in ACTIVATION, f"activation: must be one of {sorted(ACTIVATION)}, is {activation!r}")
    rows, d = residual.shape
    dev, dt = residual.device, residual.dtype
    check_rows(residual, "residual", dt, dev, (rows, d))
    for name, t in (("h", h), ("gate", gate), ("dy", dy), ("dz", dz)):
        if t is not None:
            check_rows(t, name, dt, dev, (rows, d))
    require(h is not None or (gate is None and alpha is None and w_post is None),
            "h: gate, alpha and w_post belong to a block's output")
    for name, t in (("alpha", alpha), ("w_post", w_post), ("w_pre", w_pre)):
        if t is not None:
            check_vector(t, name, d, dev)
    a = N.GatedNorm()
    a.dtype, a.act, a.rows, a.d, a.eps = DTYPE[dt], ACTIVATION[activation], rows, d, eps
    a.residual_stride, a.h_stride, a.gate_stride = residual.stride(0), _stride(h), _stride(gate)
    n = C.c_int64()
    N.check(N.lib().nrn_cuda_gatednorm_workspace(C.byref(a), C.byref(n)), "nrn_cuda_gatednorm_workspace")
    return bytes(a), max(n.value, 16)


_layouts = Layouts(_describe)


def _check_residual(residual):
    require(isinstance(residual, torch.Tensor) and residual.is_cuda, "residual: a CUDA tensor is needed")


def _call(residual, h, gate, alpha, w_post, w_pre, eps, activation, dy, dz):
    eps = number(eps)
    key = (layout(residual), layout(h), layout(gate), layout(alpha), layout(w_post), layout(w_pre), eps, activation, layout(dy), layout(dz))
    block, need = _layouts.get(key, residual, h, gate, alpha, w_post, w_pre, eps, activation, dy, dz)
    a = N.GatedNorm.from_buffer_copy(block)
    a.residual, a.h, a.gate = residual.data_ptr(), ptr(h), ptr(gate)
    a.alpha, a.w_post, a.w_pre, a.err = ptr(alpha), ptr(w_post), ptr(w_pre), error_flag(residual.device)
    return a, need


def forward(residual, h=None, gate=None, *, alpha=None, w_post=None, w_pre=None, eps=1e-6, activation="silu",
            scaled=False, want_z=True, stream=None):
    """(y, z) of [rows, d] tensors (bf16, fp16 or fp32; last stride 1).  z is None without ``want_z``, and a ``Scaled``
    matrix with ``scaled``: the next block's 8-bit input.  Without h, y is ``residual`` itself."""
    _check_residual(residual)
    dev = residual.device
    y, z = residual, None
    with on(dev, stream) as st:
        a, _ = _call(residual, h, gate, alpha, w_post, w_pre, eps, activation, None, None)
        rows, d = residual.shape
        if h is not None:
            y = torch.empty_strided((rows, d), (d, 1), dtype=residual.dtype, device=dev)
            a.y, a.y_stride = y.data_ptr(), d
        if want_z and scaled:
            z = Scaled.empty(rows, d, dev)
            a.z_scaled = C.pointer(z.desc)
        elif want_z:
            z = torch.empty_strided((rows, d), (d, 1), dtype=residual.dtype, device=dev)
            a.z, a.z_stride = z.data_ptr(), d
        N.check(N.lib().nrn_cuda_gatednorm_forward(C.byref(a), st), "nrn_cuda_gatednorm_forward")
    if stream is not None:
        share(stream, dev, (residual, h, gate, alpha, w_post, w_pre), (y, *z.memory()) if isinstance(z, Scaled) else (y, z))
    return y, z


def backward(dy, dz, residual, h=None, gate=None, *, alpha=None, w_post=None, w_pre=None, eps=1e-6, activation="silu",
             stream=None) -> Gradients:
    """Gradients of a ``forward`` call with these arguments, given those of y and z (None: zero).  Those of alpha, w_post
    and w_pre are fp32 sums over the rows, added in a fixed order."""
    _check_residual(residual)
    dev, dt = residual.device, residual.dtype
    with on(dev, stream) as st:
        a, need = _call(residual, h, gate, alpha, w_post, w_pre, eps, activation, dy, dz)
        rows, d = residual.shape
        g = N.GatedNormGrad()
        g.dy, g.dz, g.dy_stride, g.dz_stride = ptr(dy), ptr(dz), _stride(dy), _stride(dz)
        like = [torch.empty_strided((rows, d), (d, 1), dtype=dt, device=dev) if want else None for want in (True, h is not None, gate is not None)]
        sums = [torch.empty(d, dtype=torch.float32, device=dev) if t is not None else None for t in (alpha, w_post, w_pre)]
        g.dresidual, g.dh, g.dgate = (ptr(t) for t in like)
        g.dresidual_stride = g.dh_stride = g.dgate_stride = d
        g.dalpha, g.dw_post, g.dw_pre = (ptr(t) for t in sums)
        if any(t is not None for t in sums):
            w = torch.empty(need, dtype=torch.uint8, device=dev)
            g.workspace, g.workspace_bytes = w.data_ptr(), need
        N.check(N.lib().nrn_cuda_gatednorm_backward(C.byref(a), C.byref(g), st), "nrn_cuda_gatednorm_backward")
    if stream is not None:
        share(stream, dev, (dy, dz, residual, h, gate, alpha, w_post, w_pre), (*like, *sums))
    return Gradients(*like, *sums)
