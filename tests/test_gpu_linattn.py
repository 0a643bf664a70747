"""Linear attention with a decay for each head against the recurrence in 64
bits (tests/operator_refs.py).

Tolerances, relative in the 2-norm.  bf16: the scores, the state as an operand
and the result are each rounded to 8 bits, at most 2^-9 each: 3 * 2^-9.  fp16:
the same three to 11 bits, 3 * 2^-12.  fp32 results and all states: fp32
operations over the memory's length, here at most about 1,000 tokens whose
errors add like their root: 32 * 2 * 2^-24, doubled for the powers of the
decay: 2^-17."""
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu
TOL = {torch.bfloat16: 3 * 2.0 ** -9, torch.float16: 3 * 2.0 ** -12, torch.float32: 2.0 ** -17}
STATE_TOL = 2.0 ** -17
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def decays(h):
    return torch.log1p(-torch.exp2(-torch.linspace(2.0, 9.0, h, dtype=torch.float64))).float().cuda()


def make(b, t, h, hk, dk, dv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, device="cuda", generator=g)
    return (r(b, t, h, dk).to(dtype), r(b, t, hk, dk).to(dtype), r(b, t, hk, dv).to(dtype), r(b, h, dk, dv) * 2, r(b, t, h, dv).to(dtype),
            r(b, h, dk, dv))


def close(x, ref, tol):
    assert x.shape == ref.shape
    assert R.rel(x, ref) <= tol, R.rel(x, ref)


SHAPES = [
    # batch, tokens, heads, kv heads, dk, dv
    (1, 1, 1, 1, 8, 8), (2, 2, 3, 3, 64, 64), (3, 63, 2, 1, 64, 128), (2, 64, 4, 4, 128, 64), (1, 65, 2, 2, 128, 128),
    (2, 130, 4, 2, 96, 80), (1, 777, 2, 2, 32, 48), (1, 1501, 6, 2, 128, 128), (1, 4099, 1, 1, 64, 64),
    (2, 100, 3, 3, 33, 17), (1, 70, 2, 1, 200, 256), (1, 129, 2, 2, 1, 1), (40, 90, 8, 8, 64, 32),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
def test_forward_and_backward(shape, dtype):
    from libnrn_b200 import linattn
    b, t, h, hk, dk, dv = shape
    q, k, v, s0, do, ds = make(*shape, dtype)
    g, scale = decays(h), 0.7 * dk ** -0.5
    o, end = linattn.forward(q, k, v, g, scale=scale, state=s0)
    ro, rend = R.linattn(q, k, v, g, scale, s0)
    close(o, ro, TOL[dtype])
    close(end, rend, STATE_TOL)
    got = linattn.backward(do, q, k, v, g, scale=scale, state=s0, dstate=ds)
    ref = R.linattn_backward(do, q, k, v, g, scale, s0, ds)
    for x, y, like in zip(got[:3], ref[:3], (q, k, v)):
        assert x.dtype == dtype and x.shape == like.shape
        close(x, y, TOL[dtype])
    close(got[3], ref[3], STATE_TOL)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
@pytest.mark.parametrize("lens", [[0, 1, 64, 0, 65, 300, 2], [5], [0, 0], [1, 1, 1], [700, 0, 1301, 64, 128]], ids=str)
def test_packed(lens, dtype):
    from libnrn_b200 import linattn
    n = len(lens)
    q, k, v, _, do, _ = make(1, sum(lens), 4, 2, 64, 96, dtype, seed=1)
    _, _, _, s0, _, ds = make(n, 0, 4, 2, 64, 96, dtype, seed=2)
    g = decays(4)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    o, end = linattn.forward(q, k, v, g, state=s0, cu_seqlens=cu)
    ro, rend = R.linattn(q, k, v, g, 64 ** -0.5, s0, lens)
    close(o, ro, TOL[dtype])
    close(end, rend, STATE_TOL)
    for i, m in enumerate(lens):
        if m == 0:
            assert torch.equal(end[i], s0[i])
    got = linattn.backward(do, q, k, v, g, state=s0, dstate=ds, cu_seqlens=cu)
    for x, y, tol in zip(got, R.linattn_backward(do, q, k, v, g, 64 ** -0.5, s0, ds, lens), [TOL[dtype]] * 3 + [STATE_TOL]):
        close(x, y, tol)
    # the same sequences one by one
    at = 0
    for i, m in enumerate(lens):
        if m:
            one, e = linattn.forward(q[:, at:at + m], k[:, at:at + m], v[:, at:at + m], g, state=s0[i:i + 1])
            close(one, ro[:, at:at + m], TOL[dtype])
            close(e[0], rend[i], STATE_TOL)
        at += m


def test_no_state_no_tokens():
    from libnrn_b200 import linattn
    q, k, v, s0, do, _ = make(2, 200, 2, 2, 64, 64, BF16)
    g = decays(2)
    o, end = linattn.forward(q, k, v, g)
    ro, rend = R.linattn(q, k, v, g, 0.125, None)
    close(o, ro, TOL[BF16])
    close(end, rend, STATE_TOL)
    for x, y, tol in zip(linattn.backward(do, q, k, v, g), R.linattn_backward(do, q, k, v, g, 0.125, None, None), [TOL[BF16]] * 3 + [STATE_TOL]):
        close(x, y, tol)
    e = torch.empty(2, 0, 2, 64, device="cuda", dtype=BF16)
    o, end = linattn.forward(e, e, e, g, state=s0)
    assert o.shape == (2, 0, 2, 64) and torch.equal(end, s0)
    e = torch.empty(0, 5, 2, 64, device="cuda", dtype=BF16)
    o, end = linattn.forward(e, e, e, g)
    assert o.shape == (0, 5, 2, 64) and end.shape == (0, 2, 64, 64)


@pytest.mark.parametrize("t", [40, 300, 3000])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_decays_at_their_ends(t, dtype):
    """No forgetting, all of it at once, and decays whose powers vanish inside a chunk."""
    from libnrn_b200 import linattn
    g = torch.tensor([0.0, float("-inf"), -200.0, -3.0, -1e-4, -30.0], device="cuda")
    q, k, v, s0, do, ds = make(1, t, 6, 6, 64, 64, dtype, seed=3)
    o, end = linattn.forward(q, k, v, g, state=s0)
    ro, rend = R.linattn(q, k, v, g, 0.125, s0)
    got = linattn.backward(do, q, k, v, g, state=s0, dstate=ds)
    ref = R.linattn_backward(do, q, k, v, g, 0.125, s0, ds)
    for h in range(6):
        close(o[:, :, h], ro[:, :, h], TOL[dtype])
        close(end[:, h], rend[:, h], STATE_TOL)
        for x, y in zip(got[:3], ref[:3]):
            close(x[:, :, h], y[:, :, h], TOL[dtype])
        if float(ref[3][:, h].norm()) > 1e-30:
            close(got[3][:, h], ref[3][:, h], STATE_TOL)
        else:
            assert float(got[3][:, h].abs().max()) <= 1e-30


@pytest.mark.parametrize("kind", ["fused", "heads first", "one off"])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_strides(kind, dtype):
    from libnrn_b200 import linattn
    b, t, h, d = 2, 150, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(4)

    def r(*s):
        return torch.randn(*s, device="cuda", generator=gen).to(dtype)
    if kind == "fused":              # q, k, v as parts of one projection
        x = r(b, t, 3, h, d)
        q, k, v = x.unbind(2)
        out = r(b, t, h, 2 * d)[..., d:]
    elif kind == "heads first":
        q, k, v, out = (r(b, h, t, d).transpose(1, 2) for _ in range(4))
    else:                            # rows that start on no 16-byte boundary
        q, k, v, out = (r(b, t, h, d + 1)[..., 1:] for _ in range(4))
    do = torch.empty_strided(out.shape, out.stride(), dtype=dtype, device="cuda").normal_(generator=gen) if kind != "one off" else r(b, t, h, d + 1)[..., 1:]
    g = decays(h)
    o, end = linattn.forward(q, k, v, g, out=out)
    assert o is out
    ro, rend = R.linattn(q, k, v, g, 0.125, None)
    close(o, ro, TOL[dtype])
    close(end, rend, STATE_TOL)
    for x, y, tol in zip(linattn.backward(do, q, k, v, g), R.linattn_backward(do, q, k, v, g, 0.125, None, None), [TOL[dtype]] * 3 + [STATE_TOL]):
        close(x, y, tol)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
def test_nothing_reaches_earlier_tokens(bad, which, dtype):
    """A token that is no number is not seen by those before it, nor by other heads and sequences."""
    from libnrn_b200 import linattn
    q, k, v, _, _, _ = make(2, 200, 2, 2, 64, 64, dtype, seed=5)
    g = decays(2)
    good, _ = linattn.forward(q, k, v, g)
    x = k if which == "k" else v
    x[1, 77, 1, 3] = bad
    o, end = linattn.forward(q, k, v, g)
    assert torch.equal(o[0], good[0]) and torch.equal(o[1, :, 0], good[1, :, 0])
    assert R.rel(o[1, :77, 1], good[1, :77, 1]) <= TOL[dtype] and bool(torch.isfinite(o[1, :77, 1]).all())
    assert not bool(torch.isfinite(o[1, 77:, 1, 3]).any())
    assert not bool(torch.isfinite(end[1, 1]).all()) and bool(torch.isfinite(end[0]).all())


def test_runs_repeat_bit_for_bit():
    from libnrn_b200 import linattn
    q, k, v, s0, do, ds = make(1, 3000, 2, 1, 128, 128, BF16)
    g = decays(2)
    a = (*linattn.forward(q, k, v, g, state=s0), *linattn.backward(do, q, k, v, g, state=s0, dstate=ds))
    b = (*linattn.forward(q, k, v, g, state=s0), *linattn.backward(do, q, k, v, g, state=s0, dstate=ds))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("dims", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (5, 6, 1, 128, 96), (2, 2, 2, 256, 200), (4, 3, 3, 33, 18)], ids=str)
def test_steps_are_the_forward(dims, dtype):
    from libnrn_b200 import linattn
    b, h, hk, dk, dv = dims
    q, k, v, s0, _, _ = make(b, 9, h, hk, dk, dv, dtype)
    g = decays(h)
    state = s0.clone()
    ro, rend = R.linattn(q, k, v, g, dk ** -0.5, s0)
    for t in range(9):
        close(linattn.step(q[:, t], k[:, t], v[:, t], g, state), ro[:, t], TOL[dtype])
    close(state, rend, STATE_TOL)


def test_step_slots():
    from libnrn_b200 import linattn
    q, k, v, _, _, _ = make(4, 1, 2, 2, 64, 32, BF16)
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    big = torch.randn(7, 3, 2, 64, 32, device="cuda")
    state = big[:, 1]                               # states that lie apart
    before, g = big.clone(), decays(2)
    o = linattn.step(q, k, v, g, state, slots=torch.tensor([5, -1, 0, 7], device="cuda", dtype=torch.int32))
    for i, s in ((0, 5), (2, 0)):
        ro, rend = R.linattn(q[i][None, None], k[i][None, None], v[i][None, None], g, 0.125, before[s:s + 1, 1])
        close(o[i], ro[0, 0], TOL[BF16])
        close(state[s], rend[0], STATE_TOL)
    assert not o[1].any() and bool(torch.isnan(o[3]).all())
    rest = [1, 2, 3, 4, 6]
    assert torch.equal(state[rest], before[rest, 1]) and torch.equal(big[:, 0], before[:, 0]) and torch.equal(big[:, 2], before[:, 2])
    # nothing to do
    assert linattn.step(q[:0], k[:0], v[:0], g, state).shape == (0, 2, 32)


def test_states_past_32_bits():
    """A cache of more than 2^31 elements, used at both ends."""
    from libnrn_b200 import linattn
    n, h, d = 8300, 16, 128
    state = torch.empty(n, h, d, d, device="cuda")          # 2.18e9 elements
    at = torch.tensor([0, n - 1, 8191, 8192], device="cuda", dtype=torch.int32)
    q, k, v, s0, _, _ = make(4, 1, h, h, d, d, BF16)
    state[at.long()] = s0
    o = linattn.step(q[:, 0], k[:, 0], v[:, 0], decays(h), state, slots=at)
    ro, rend = R.linattn(q, k, v, decays(h), d ** -0.5, s0)
    close(o, ro[:, 0], TOL[BF16])
    close(state[at.long()], rend, STATE_TOL)


def test_tokens_past_32_bits():
    """Token rows of one tensor that lie more than 2^31 elements apart."""
    from libnrn_b200 import linattn
    t, d, gap = 70, 64, 33_000_000
    base = torch.zeros(t * gap, device="cuda", dtype=BF16)
    def spread(x, off):
        y = base.as_strided((1, t, 1, d), (t * gap, gap, d, 1), off)
        y.copy_(x)
        return y
    q, k, v, _, _, _ = make(1, t, 1, 1, d, d, BF16)
    g = decays(1)
    o, end = linattn.forward(spread(q, 0), spread(k, 64), spread(v, 128), g, out=base.as_strided((1, t, 1, d), (t * gap, gap, d, 1), 192))
    ro, rend = R.linattn(q, k, v, g, 0.125, None)
    close(o, ro, TOL[BF16])
    close(end, rend, STATE_TOL)


def test_on_another_stream_and_in_a_graph():
    from libnrn_b200 import linattn
    q, k, v, s0, do, ds = make(1, 1000, 2, 2, 64, 64, BF16)
    g = decays(2)
    want = linattn.forward(q, k, v, g, state=s0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = linattn.forward(q, k, v, g, state=s0, stream=side)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, end = linattn.forward(q, k, v, g, state=s0)
    q.copy_(q.flip(1))
    graph.replay()
    assert torch.equal(o, linattn.forward(q, k, v, g, state=s0)[0])


def test_refusals():
    from libnrn_b200 import _native as N
    from libnrn_b200 import linattn
    q, k, v, s0, do, _ = make(2, 10, 4, 2, 64, 32, BF16)
    g = decays(4)
    cu = torch.tensor([0, 10], device="cuda", dtype=torch.int32)
    ok = dict(q=q, k=k, v=v, log_decay=g)
    for bad in (dict(q=q.cpu()), dict(q=q.double()), dict(k=k.half()), dict(k=k[:, :9]), dict(k=k[..., :32]), dict(v=v[0]),
                dict(k=k[:, :, :1].expand(2, 10, 3, 64), v=v[:, :, :1].expand(2, 10, 3, 32)), dict(log_decay=g[:3]), dict(log_decay=g.double()),
                dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), dict(state=s0[:1]), dict(state=s0.half()),
                dict(state=s0.transpose(2, 3).contiguous().transpose(2, 3)), dict(cu_seqlens=cu), dict(scale=0.0), dict(scale=float("nan")),
                dict(out=torch.empty(2, 10, 4, 32, device="cuda"))):
        with pytest.raises(N.NrnError):
            linattn.forward(**{**ok, **bad})
    with pytest.raises(N.NrnError):
        linattn.forward(q[:1], k[:1], v[:1], g, cu_seqlens=cu.long())
    with pytest.raises(N.NrnError):
        linattn.backward(do[:, :9], q, k, v, g)
    big = torch.empty(1, 3, 1, 257, device="cuda", dtype=BF16)
    with pytest.raises(N.NrnError):
        linattn.forward(big, big, big, g[:1])
    with pytest.raises(N.NrnError):
        linattn.step(q[:, 0], k[:, 0], v[:, 0], g, s0[:1])
    with pytest.raises(N.NrnError):
        linattn.step(q[:, 0], k[:, 0], v[:, 0], g, s0, slots=torch.tensor([0, 1], device="cuda"))
