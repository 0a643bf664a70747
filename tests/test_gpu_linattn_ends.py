"""Linear attention at its ends.  Tolerances as in test_gpu_linattn.py."""
import ctypes as C

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


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("kind", ["bf16", "bf16 off 16 bytes", "fp16", "fp32"])
def test_a_bad_token_in_the_gradients(kind, which, bad):
    """Keys and values before it see a token of q or do that is no number, queries after it one of k or v; nobody else does."""
    from libnrn_b200 import linattn
    dtype = {"fp16": FP16, "fp32": FP32}.get(kind, BF16)
    at, h = 77, 1
    q, k, v, _, do, _ = make(2, 200, 2, 2, 64, 64, dtype, seed=5)
    if kind == "bf16 off 16 bytes":
        q, k, v, do = (torch.cat([x[..., :1], x], -1)[..., 1:] for x in (q, k, v, do))
    g = decays(2)
    good = linattn.backward(do, q, k, v, g)
    {"q": q, "k": k, "v": v, "do": do}[which][1, at, h, 3] = bad
    got = linattn.backward(do, q, k, v, g)
    for n, x, y in zip(("q", "k", "v"), got, good):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1, :, 0], y[1, :, 0])
        later, earlier = slice(at + 1, None), slice(None, at)
        clean = {"q": {"q": [earlier, slice(at, None)], "k": [earlier], "v": [earlier], "do": [earlier, later]},
                 "k": {"q": [later], "k": [earlier, slice(at, None)], "v": [earlier, later], "do": [later]},
                 "v": {"q": [later], "k": [earlier, later], "v": [earlier, slice(at, None)], "do": [later]}}[n][which]
        for part in clean:
            z = x[1, part, h]
            assert bool(torch.isfinite(z).all()), (n, part)
            assert R.rel(z, y[1, part, h]) <= TOL[dtype]
    assert torch.equal(got[3][0], good[3][0]) and torch.equal(got[3][1, 0], good[3][1, 0])


@pytest.mark.parametrize("lens", [[0, 1, 64, 0, 65, 300, 2], [17, 16, 15, 1]], ids=str)
def test_packed_fp16(lens):
    from libnrn_b200 import linattn
    n = len(lens)
    q, k, v, _, do, _ = make(1, sum(lens), 4, 2, 64, 96, FP16, seed=1)
    _, _, _, s0, _, ds = make(n, 0, 4, 2, 64, 96, FP16, seed=2)
    g, cu = decays(4), torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    o, end = linattn.forward(q, k, v, g, state=s0, cu_seqlens=cu)
    ro, rend = R.linattn(q, k, v, g, 0.125, s0, lens)
    close(o, ro, TOL[FP16])
    close(end, rend, STATE_TOL)
    got = linattn.backward(do, q, k, v, g, state=s0, dstate=ds, cu_seqlens=cu)
    for x, y, tol in zip(got, R.linattn_backward(do, q, k, v, g, 0.125, s0, ds, lens), [TOL[FP16]] * 3 + [STATE_TOL]):
        close(x, y, tol)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_one_key_head_for_all(dtype):
    """k and v expanded over the heads (a stride of 0), as a caller without shared heads would give them."""
    from libnrn_b200 import linattn
    q, k, v, s0, do, ds = make(2, 150, 4, 1, 64, 64, dtype, seed=6)
    kx, vx, g = k.expand(2, 150, 4, 64), v.expand(2, 150, 4, 64), decays(4)
    o, end = linattn.forward(q, kx, vx, g, state=s0)
    ro, rend = R.linattn(q, k, v, g, 0.125, s0)
    close(o, ro, TOL[dtype])
    close(end, rend, STATE_TOL)
    got = linattn.backward(do, q, kx, vx, g, state=s0, dstate=ds)
    ref = R.linattn_backward(do, q, kx, vx, g, 0.125, s0, ds)
    for x, y, tol in zip(got, ref, [TOL[dtype]] * 3 + [STATE_TOL]):
        close(x, y, tol)


def test_sequences_are_split_by_their_own_kernels_costs():
    """Seen in the workspace of the segments' states: none where whole sequences are faster, many where they are long."""
    def states(dtype, seqs, tokens, heads, d):
        a, n = N.LinAttn(), C.c_int64()
        a.dtype, a.seqs, a.heads, a.kv_heads, a.dk, a.dv, a.tokens, a.scale, a.log_decay = dtype, seqs, heads, heads, d, d, tokens, 1.0, 256
        N.check(N.lib().nrn_cuda_linattn_workspace(C.byref(a), 0, C.byref(n)), "nrn_cuda_linattn_workspace")
        return n.value // (heads * d * d * 4)
    for dtype in (1, 2):                             # fp16, fp32: token by token
        assert states(dtype, 4, 2048, 16, 128) == 0          # 1.67 ms whole, 1.96 and more split
        assert states(dtype, 1, 65536, 8, 64) >= 32          # 18 segments 3.4 ms, 32 2.4, 64 2.2
        assert states(dtype, 1, 8192, 16, 64) >= 16          # 8 segments 0.92 ms, 16 0.61, 32 0.58


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16 off 16 bytes", "bf16 wide"])
def test_many_segments(kind):
    """Long sequences, packed too, on the kernels that are not the tensor cores' (whose segments test_gpu_linattn.py has)."""
    from libnrn_b200 import linattn
    dtype, d = {"fp32": FP32, "fp16": FP16}.get(kind, BF16), 136 if kind == "bf16 wide" else 32
    lens = [1201, 0, 700, 64, 1, 900]
    q, k, v, _, do, _ = make(1, sum(lens), 2, 1, d, d, dtype, seed=7)
    _, _, _, s0, _, ds = make(len(lens), 0, 2, 1, d, d, dtype, seed=8)
    if kind == "bf16 off 16 bytes":
        q, k, v, do = (torch.cat([x[..., :1], x], -1)[..., 1:] for x in (q, k, v, do))
    g, cu = decays(2), torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    tols = [TOL[dtype]] * 3 + [STATE_TOL]
    o, end = linattn.forward(q, k, v, g, state=s0, cu_seqlens=cu)
    ro, rend = R.linattn(q, k, v, g, d ** -0.5, s0, lens)
    close(o, ro, TOL[dtype])
    close(end, rend, STATE_TOL)
    for x, y, tol in zip(linattn.backward(do, q, k, v, g, state=s0, dstate=ds, cu_seqlens=cu), R.linattn_backward(do, q, k, v, g, d ** -0.5, s0, ds, lens), tols):
        close(x, y, tol)
    q, k, v, do = (x[:, :1201] for x in (q, k, v, do))
    o, end = linattn.forward(q, k, v, g, state=s0[:1])
    ro, rend = R.linattn(q, k, v, g, d ** -0.5, s0[:1])
    close(o, ro, TOL[dtype])
    close(end, rend, STATE_TOL)
    for x, y, tol in zip(linattn.backward(do, q, k, v, g, state=s0[:1], dstate=ds[:1]), R.linattn_backward(do, q, k, v, g, d ** -0.5, s0[:1], ds[:1]), tols):
        close(x, y, tol)
