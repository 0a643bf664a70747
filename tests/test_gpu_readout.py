"""The readout: a simulated network's activity through all the sequence-memory
operators, whole, packed, step by step, and learning.

The two ways through (whole recordings and single steps) round their bf16
intermediates in other orders; each block's rounding is at most 2^-8 and e4m3's
2^-4 where a value falls to the other side: 2^-4 covers two blocks.  Gradients
are compared with those of the same readout in fp32 with unrounded activations,
weights as quantised: e4m3 activations and gradients, 2^-4 each way a block."""
import numpy as np
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -4


@pytest.fixture(scope="module")
def counts():
    from libnrn_b200 import readout, workloads
    from libnrn_b200.engine import Network
    spec = workloads.brunel(1600, 400, 160, 40)
    nw = Network.from_spec(spec)
    nw.run(6000)
    step, gid = nw.raster()
    nw.close()
    c = readout.bin_spikes(step, gid, 2000, 20, 300, group=20)
    want = np.zeros((300, 100), np.int64)
    np.add.at(want, (step // 20, gid // 20), 1)
    assert torch.equal(c, torch.from_numpy(want).cuda().to(torch.bfloat16)) and c.any()
    return c


def make(**kw):
    from libnrn_b200 import readout
    return readout.Readout(100, 40, width=192, heads=4, kv_heads=2, dk=32, dv=64, bin_s=2e-3, **kw)


def test_whole_packed_and_steps(counts):
    r = make()
    both = torch.stack([counts[:150], counts[150:]])
    answers, states = r.read(both)
    assert answers.shape == (2, 150, 40) and states[0].shape == (2, 4, 32, 64)
    cu = torch.tensor([0, 150, 300], device="cuda", dtype=torch.int32)
    packed, pstates = r.read(counts[None], cu_seqlens=cu)
    assert R.rel(packed.view(2, 150, 40), answers) <= TOL and all(R.rel(a, b) <= TOL for a, b in zip(pstates, states))
    # in two parts, the second from the states of the first
    first, mid = r.read(both[:, :70])
    second, end = r.read(both[:, 70:], states=mid)
    assert R.rel(torch.cat([first, second], 1), answers) <= TOL and all(R.rel(a, b) <= TOL for a, b in zip(end, states))
    # one bin at a time, the sessions in slots 3 and 1
    cache = r.new_states(5)
    slots = torch.tensor([3, 1], device="cuda", dtype=torch.int32)
    got = torch.stack([r.step(both[:, t], cache, slots=slots) for t in range(150)], 1)
    assert R.rel(got, answers) <= TOL
    assert all(R.rel(c[[3, 1]], s) <= TOL and not c[[0, 2, 4]].any() for c, s in zip(cache, states))


def plain(r, counts, targets):
    """The same readout in fp32 by torch, differentiable, with the weights that the 8-bit products use."""
    p = {n: (r.small(n).dequantize() if n.split(".")[0] in ("embed", "head", "in", "out") else w.clone()).requires_grad_(True)
         for n, w in r.weights.items()}

    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + r.eps)
    x = counts.float() @ p["embed"].t()
    t = x.shape[0]
    lag = torch.arange(t, device="cuda")
    lag = lag[:, None] - lag[None, :]
    inside = torch.where(lag >= 0, torch.exp(r.log_decay[:, None, None] * lag.clamp_min(0)), 0.0)
    for i in range(r.blocks):
        z = norm(x) * p["w_pre.%d" % i]
        q, k, v, gate = r._split(z @ p["in.%d" % i].t())
        k, v = (y.repeat_interleave(r.heads // r.kv_heads, 1) for y in (k, v))
        o = torch.einsum("ihd,jhd->hij", q, k) * inside * r.dk ** -0.5
        h = torch.einsum("hij,jhd->ihd", o, v).flatten(1) @ p["out.%d" % i].t()
        x = x + p["alpha.%d" % i] * torch.nn.functional.silu(gate) * norm(h) * p["w_post.%d" % i]
    answers = (norm(x) * p["w_pre.%d" % r.blocks]) @ p["head"].t()
    loss = (answers - targets.float()).square().mean()
    loss.backward()
    return loss.detach(), {n: w.grad for n, w in p.items()}


def test_gradients_and_learning(counts):
    r = make(blocks=1)
    past, future = counts[None, :-1], counts[None, 1:, :40]
    loss, grads = r.gradients(past, future)
    want, ref = plain(r, past[0], future[0])
    assert abs(float(loss) - float(want)) <= TOL * float(want)
    assert set(grads) == set(r.weights)
    for n, g in grads.items():
        assert g.shape == r.weights[n].shape
        assert R.rel(g, ref[n]) <= 2 * TOL, (n, R.rel(g, ref[n]))
    before = float(loss)
    for _ in range(15):
        loss, grads = r.gradients(past, future)
        r.learn(grads, 0.02)
    assert float(r.gradients(past, future)[0]) < 0.8 * before


def test_refusals(counts):
    from libnrn_b200 import _native as N
    from libnrn_b200 import readout
    r = make()
    for call in (lambda: r.read(counts[None].float()), lambda: r.read(counts[None, :, :50]), lambda: r.step(counts[:, :99], r.new_states(300)),
                 lambda: readout.Readout(10, 10, heads=3, kv_heads=2), lambda: readout.Readout(10, 10, width=100), lambda: readout.Readout(10, 10, tau=(1.0, 0.5))):
        with pytest.raises(N.NrnError):
            call()
