"""Linear attention with a decay for each head: a fast Hebbian projection
with forgetting, for sequences (``forward``, ``backward``) and one token at a
time (``step``).  For each sequence and head, with lam = exp(log_decay[head]):

    S_t = lam S_{t-1} + k_t v_t^T          o_t = scale * S_t^T q_t

Tokens are [batch, tokens, heads, d] tensors with any strides but the last,
which is 1; bf16, fp16 or fp32.  A result given as ``out`` lies on none of the
inputs, and its elements not on one another.  k and v may have fewer heads (a
divisor of q's), each read by as many heads of q.  States are fp32
[batch, heads, dk, dv].  With ``cu_seqlens`` (int32 starts of packed
sequences, [sequences + 1], on the device, from 0 to the number of tokens) the
batch dimension is 1 and states have one entry for each sequence.  dk and dv
are at most 256; ``log_decay`` (fp32 [heads]) is at most 0, -inf forgets
everything at each token.  The decays are time constants, not learned: they
have no gradient.  States are summed in fp32.  For bf16 inputs the scores
q . k and the state as q reads it are rounded to bf16 on their way to the
tensor cores, so a result is about 1.4 times as far from the exact one as its
own rounding; a caller who wants every bit gives fp32 tensors (slower, one
token at a time).  Results have no autograd graph: tensors that require
gradients are refused where these are recorded, and ``backward`` gives them.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _native as N
from ._tensors import (DTYPE, Layouts, check_result, check_rows, check_state, check_tensor, check_vector, check_waits, error_flag, layout, number,
                       on, ptr, require, share)

check = check_waits


def _strides(t):
    return t.stride(0), t.stride(1), t.stride(2)


def _check_q(q):
    require(isinstance(q, torch.Tensor) and q.is_cuda, "q: a CUDA tensor is needed")
    require(q.dtype in DTYPE, f"q: must be bfloat16, float16 or float32, is {q.dtype}")


def _describe(q, k, v, log_decay, scale, cu_seqlens, state, dstate, do, out):
    """The checked argument block of a forward or backward call (its pointers are set by each call), and its workspace."""
    _check_q(q)
    for name, t in (("q", q), ("k", k), ("v", v)):
        require(isinstance(t, torch.Tensor) and t.dim() == 4, f"{name}: must be [batch, tokens, heads, d]")
    b, t, h, dk = q.shape
    hk, dv = k.shape[2], v.shape[3]
    require(h >= 1 and hk >= 1 and h % hk == 0, f"heads: {h} of q are no multiple of {hk} of k")
    dev, dt = q.device, q.dtype
    check_rows(q, "q", dt, dev, (b, t, h, dk))
    check_rows(k, "k", dt, dev, (b, t, hk, dk))
    check_rows(v, "v", dt, dev, (b, t, hk, dv))
    check_vector(log_decay, "log_decay", h, dev)
    a = N.LinAttn()
    a.dtype, a.heads, a.kv_heads, a.dk, a.dv, a.tokens = DTYPE[dt], h, hk, dk, dv, t
    if cu_seqlens is None:
        a.seqs = b
    else:
        require(b == 1, "cu_seqlens: packed sequences have a batch dimension of 1")
        check_tensor(cu_seqlens, "cu_seqlens", torch.int32, dev)
        require(cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1 and cu_seqlens.is_contiguous(),
                "cu_seqlens: must be a contiguous vector of sequences + 1 starts")
        a.seqs, a.cu_seqlens = cu_seqlens.numel() - 1, cu_seqlens.data_ptr()
        require(a.seqs > 0 or t == 0, f"cu_seqlens: no sequences for {t} tokens")
    shape = (a.seqs, h, dk, dv)
    for name, x in (("state", state), ("dstate", dstate)):
        if x is not None:
            check_state(x, name, dev, shape)
    if do is not None:
        check_rows(do, "do", dt, dev, (b, t, h, dv))
    if out is not None:
        check_result(out, "out", dt, dev, (b, t, h, dv))
    a.log_decay = log_decay.data_ptr()
    a.scale = dk ** -0.5 if scale is None else scale
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = _strides(q), _strides(k), _strides(v)
    if out is not None:
        a.o_stride[:] = _strides(out)
    elif do is None:
        a.o_stride[:] = (t * h * dv, h * dv, dv)
    n = C.c_int64()
    N.check(N.lib().nrn_cuda_linattn_workspace(C.byref(a), int(do is not None), C.byref(n)), "nrn_cuda_linattn_workspace")
    return bytes(a), n.value, shape


_sequences = Layouts(_describe)


def _call(q, k, v, log_decay, scale, cu_seqlens, state, dstate, do, out):
    """(argument block with the inputs' pointers, workspace bytes, shape of the states)."""
    scale = number(scale)
    key = (layout(q), layout(k), layout(v), layout(log_decay), scale, layout(cu_seqlens), layout(state), layout(dstate), layout(do),
           layout(out))
    block, need, shape = _sequences.get(key, q, k, v, log_decay, scale, cu_seqlens, state, dstate, do, out)
    a = N.LinAttn.from_buffer_copy(block)
    a.q, a.k, a.v, a.log_decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr()
    a.cu_seqlens, a.state_in, a.err = ptr(cu_seqlens), ptr(state), error_flag(q.device)
    return a, need, shape


def forward(q, k, v, log_decay, *, scale=None, state=None, cu_seqlens=None, out=None, stream=None):
    """(o, final states) of whole sequences that go on from ``state`` (default: zero states).
    o is like q with v's last dimension; ``scale`` defaults to dk ** -0.5."""
    _check_q(q)
    given = out
    with on(q.device, stream) as st:
        a, need, shape = _call(q, k, v, log_decay, scale, cu_seqlens, state, None, None, out)
        if out is None:
            out = torch.empty((*q.shape[:3], a.dv), dtype=q.dtype, device=q.device)
        end = torch.empty(shape, dtype=torch.float32, device=q.device)
        a.o, a.state_out = out.data_ptr(), end.data_ptr()
        if need:
            w = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = w.data_ptr(), need
        N.check(N.lib().nrn_cuda_linattn_forward(C.byref(a), st), "nrn_cuda_linattn_forward")
    if stream is not None:
        share(stream, q.device, (q, k, v, log_decay, cu_seqlens, state, given), (out, end))
    return out, end


def backward(do, q, k, v, log_decay, *, scale=None, state=None, dstate=None, cu_seqlens=None, stream=None):
    """(dq, dk, dv, dstate) of a ``forward`` call with these arguments, given the gradients of o (``do``) and of the final
    states (``dstate``, default: zero); the last result is the gradient of the states it started from."""
    _check_q(q)
    require(do is not None, "do: a tensor is needed")
    with on(q.device, stream) as st:
        a, need, shape = _call(q, k, v, log_decay, scale, cu_seqlens, state, dstate, do, None)
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        ds = torch.empty(shape, dtype=torch.float32, device=q.device)
        g = N.LinAttnGrad()
        g.d_o, g.dstate_out, g.dstate_in = do.data_ptr(), ptr(dstate), ds.data_ptr()
        g.dq, g.dk, g.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        g.d_o_stride[:], g.dq_stride[:] = _strides(do), _strides(dq)
        g.dk_stride[:], g.dv_stride[:] = _strides(dk), _strides(dv)
        if need:
            w = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = w.data_ptr(), need
        N.check(N.lib().nrn_cuda_linattn_backward(C.byref(a), C.byref(g), st), "nrn_cuda_linattn_backward")
    if stream is not None:
        share(stream, q.device, (do, q, k, v, log_decay, cu_seqlens, state, dstate), (dq, dk, dv, ds))
    return dq, dk, dv, ds


def _describe_step(q, k, v, log_decay, state, scale, slots, out):
    for name, x in (("q", q), ("k", k), ("v", v)):
        require(isinstance(x, torch.Tensor) and x.dim() == 3, f"{name}: must be [batch, heads, d]")
    b, h, dk = q.shape
    hk, dv = k.shape[1], v.shape[2]
    require(h >= 1 and hk >= 1 and h % hk == 0, f"heads: {h} of q are no multiple of {hk} of k")
    dev = q.device
    check_rows(q, "q", q.dtype, dev, (b, h, dk))
    check_rows(k, "k", q.dtype, dev, (b, hk, dk))
    check_rows(v, "v", q.dtype, dev, (b, hk, dv))
    check_vector(log_decay, "log_decay", h, dev)
    require(isinstance(state, torch.Tensor) and state.dim() == 4, "state: must be [states, heads, dk, dv]")
    check_tensor(state, "state", torch.float32, dev, (state.shape[0], h, dk, dv))
    require(state.shape[0] == 0 or state[0].is_contiguous(), "state: each state must be contiguous")
    require(state.shape[0] <= 1 or state.stride(0) >= h * dk * dv, "state: states lie on one another")
    if slots is not None:
        check_tensor(slots, "slots", torch.int32, dev, (b,))
        require(slots.is_contiguous(), "slots: must be contiguous")
    else:
        require(state.shape[0] >= b, f"state: {state.shape[0]} states for {b} sequences")
    if out is not None:
        check_result(out, "out", q.dtype, dev, (b, h, dv))
    a = N.LinAttn()
    a.dtype, a.seqs, a.heads, a.kv_heads, a.dk, a.dv, a.tokens = DTYPE[q.dtype], b, h, hk, dk, dv, 1
    a.scale = dk ** -0.5 if scale is None else scale
    for f, x in ((a.q_stride, q), (a.k_stride, k), (a.v_stride, v)):
        f[0], f[2] = x.stride(0), x.stride(1)
    a.o_stride[0], a.o_stride[2] = (out.stride(0), out.stride(1)) if out is not None else (h * dv, dv)
    return bytes(a), (b, h, dv), (h * dv, dv, 1), state.stride(0), state.shape[0]


_steps = Layouts(_describe_step)


def step(q, k, v, log_decay, state, *, scale=None, slots=None, out=None, stream=None):
    """o of one token for each sequence ([batch, heads, d] tensors), updating ``state`` in place.  Sequence i uses
    ``state[slots[i]]`` (int32, default: state[i]); a slot appears at most once in a call, a negative one is padding whose
    output is 0, and one past the states gives NaN."""
    _check_q(q)
    scale = number(scale)
    key = (layout(q), layout(k), layout(v), layout(log_decay), layout(state), scale, layout(slots), layout(out))
    block, shape, strides, stride, count = _steps.get(key, q, k, v, log_decay, state, scale, slots, out)
    given = out
    with on(q.device, stream) as st:
        if out is None:
            out = torch.empty_strided(shape, strides, dtype=q.dtype, device=q.device)
        a = N.LinAttn.from_buffer_copy(block)
        a.q, a.k, a.v, a.o, a.log_decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), log_decay.data_ptr()
        N.check(N.lib().nrn_cuda_linattn_step(C.byref(a), state.data_ptr(), stride, count, ptr(slots), st), "nrn_cuda_linattn_step")
    if stream is not None:
        share(stream, q.device, (q, k, v, log_decay, state, slots, given), (out,))
    return out
