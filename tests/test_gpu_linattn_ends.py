"""Linear attention at its ends.  Tolerances as in test_gpu_linattn.py."""
import pytest
import torch

import operator_refs as R
from libnrn_b200 import _native as N
from test_gpu_linattn import STATE_TOL, TOL, close, decays, make

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("t", [1, 16, 40, 150])
@pytest.mark.parametrize("kind", ["bf16", "bf16 off 16 bytes", "fp16", "fp32"])
def test_an_infinite_state_stays_infinite(kind, t):
    from libnrn_b200 import linattn
    dtype = {"fp16": FP16, "fp32": FP32}.get(kind, BF16)
    q, k, v, s0, _, _ = make(1, t, 3, 3, 64, 64, dtype)
    if kind == "bf16 off 16 bytes":
        q, k, v = (torch.cat([x[..., :1], x], -1)[..., 1:] for x in (q, k, v))
    q[q == 0] = 1
    s0[0, :, 5, 7] = float("inf")
    g = torch.tensor([0.0, -0.01, -0.5], device="cuda")      # the first decay has no error to take out
    o, end = linattn.forward(q, k, v, g, state=s0)
    ro, rend = R.linattn(q, k, v, g, 0.125, s0)
    assert bool(ro[..., 7].isinf().all())
    assert torch.equal(o[..., 7].double(), ro[..., 7]) and torch.equal(end[..., 5, 7].double(), rend[..., 5, 7])
    rest = [i for i in range(64) if i != 7]
    close(o[..., rest], ro[..., rest], TOL[dtype])
    end[..., 5, 7] = rend[..., 5, 7] = 0
    close(end, rend, STATE_TOL)


def test_states_on_one_another_are_refused(monkeypatch):
    """Sequences that would update one state, or states that overlap.  (Nothing is launched here.)"""
    from libnrn_b200 import linattn
    monkeypatch.setattr(N.lib(), "nrn_cuda_linattn_step", lambda *a: 0)
    q, k, v, _, _, _ = make(3, 1, 2, 2, 32, 32, BF16)
    q, k, v, g = q[:, 0], k[:, 0], v[:, 0], decays(2)
    one = torch.zeros(1, 2, 32, 32, device="cuda")
    linattn.step(q[:1], k[:1], v[:1], g, one)
    linattn.step(q[:1], k[:1], v[:1], g, one.expand(1, 2, 32, 32))
    for state in (one.expand(3, 2, 32, 32), torch.zeros(4 * 2048, device="cuda").as_strided((3, 2, 32, 32), (1024, 1024, 32, 1))):
        with pytest.raises(N.NrnError, match="state"):
            linattn.step(q, k, v, g, state)
        with pytest.raises(N.NrnError, match="state"):
            linattn.step(q[:1], k[:1], v[:1], g, state, slots=torch.zeros(1, dtype=torch.int32, device="cuda"))


def test_results_on_one_another_are_refused(monkeypatch):
    """An `out` whose tokens share memory.  (Nothing is launched here.)"""
    from libnrn_b200 import linattn
    for name in ("nrn_cuda_linattn_step", "nrn_cuda_linattn_forward"):
        monkeypatch.setattr(N.lib(), name, lambda *a: 0)
    q, k, v, s0, _, _ = make(2, 10, 2, 2, 32, 32, BF16)
    g = decays(2)
    for out in (torch.empty(2, 1, 2, 32, device="cuda", dtype=BF16).expand(2, 10, 2, 32), torch.empty(1, 10, 2, 32, device="cuda", dtype=BF16).expand(2, 10, 2, 32),
                torch.empty(2, 10, 1, 32, device="cuda", dtype=BF16).expand(2, 10, 2, 32),
                torch.empty(4000, device="cuda", dtype=BF16).as_strided((2, 10, 2, 32), (640, 32, 32, 1))):
        with pytest.raises(N.NrnError, match="out"):
            linattn.forward(q, k, v, g, out=out)
    for out in (torch.empty(1, 2, 32, device="cuda", dtype=BF16).expand(2, 2, 32), torch.empty(2, 1, 32, device="cuda", dtype=BF16).expand(2, 2, 32)):
        with pytest.raises(N.NrnError, match="out"):
            linattn.step(q[:, 0], k[:, 0], v[:, 0], g, s0, out=out)
    # heads outside tokens, parts of something wider
    linattn.forward(q, k, v, g, out=torch.empty(2, 2, 10, 32, device="cuda", dtype=BF16).transpose(1, 2))
    linattn.forward(q, k, v, g, out=torch.empty(2, 10, 2, 96, device="cuda", dtype=BF16)[..., 32:64])
    linattn.forward(q, k, v, g, out=torch.empty(10, 2, 2, 32, device="cuda", dtype=BF16).transpose(0, 1))


def test_tokens_without_a_sequence_are_refused():
    from libnrn_b200 import linattn
    q, k, v, _, do, _ = make(1, 10, 2, 2, 32, 32, BF16)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(N.NrnError, match="cu_seqlens"):
        linattn.forward(q, k, v, decays(2), cu_seqlens=none)
    with pytest.raises(N.NrnError, match="cu_seqlens"):
        linattn.backward(do, q, k, v, decays(2), cu_seqlens=none)
    e = q[:, :0]
    o, end = linattn.forward(e, e, e, decays(2), cu_seqlens=none)
    assert o.shape == (1, 0, 2, 32) and end.shape == (0, 2, 32, 32)


@pytest.mark.parametrize("scale", [2.0 ** -126, -2.0 ** -100, 2.0 ** 100])
def test_scales_far_from_one(scale):
    """The gradient of the final state passes through 1 / scale: scales whose inverse is no number are refused."""
    from libnrn_b200 import linattn
    q, k, v, s0, do, ds = make(1, 40, 1, 1, 32, 32, FP32)
    got = linattn.backward(do * 0, q, k, v, decays(1), scale=scale, state=s0, dstate=ds * scale)
    ref = R.linattn_backward(do * 0, q, k, v, decays(1), scale, s0, ds * scale)
    close(got[1] / scale, ref[1] / scale, TOL[FP32])
    for x in (2.0 ** -140, -2.0 ** -130):
        with pytest.raises(N.NrnError, match="scale"):
            linattn.backward(do, q, k, v, decays(1), scale=x, dstate=ds)
