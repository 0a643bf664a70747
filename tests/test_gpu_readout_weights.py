"""A readout answers by the weights that it has at the call, and its ends."""
import numpy as np
import pytest
import torch

from libnrn_b200 import _native as N

pytestmark = pytest.mark.gpu


def make(seed=0, **kw):
    from libnrn_b200 import readout
    return readout.Readout(24, 16, width=64, heads=2, dk=32, dv=32, blocks=1, seed=seed, **kw)


def counts(*s):
    return torch.poisson(torch.full(s, 0.7, device="cuda"), generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)


@pytest.mark.parametrize("how", ["assign", "in place", "data", "update", "all"])
def test_answers_follow_the_weights(how):
    a, b, x = make(0), make(1), counts(2, 30, 24)
    before = a.read(x)[0]
    assert not torch.equal(before, b.read(x)[0])
    for n, w in b.weights.items():
        if how == "assign":
            a.weights[n] = w
        elif how == "in place":
            a.weights[n].copy_(w)
        elif how == "data":
            a.weights[n].data.copy_(w)
    if how == "update":
        a.weights.update(b.weights)
    elif how == "all":
        a.weights = dict(b.weights)
    assert torch.equal(a.read(x)[0], b.read(x)[0])
    sa, sb = a.new_states(2), b.new_states(2)
    assert torch.equal(a.step(x[:, 0], sa), b.step(x[:, 0], sb)) and torch.equal(sa[0], sb[0])
    la, ga = a.gradients(x[:1, :-1], x[:1, 1:, :16])
    lb, gb = b.gradients(x[:1, :-1], x[:1, 1:, :16])
    assert torch.equal(la, lb) and all(torch.equal(ga[n], gb[n]) for n in gb)


def test_a_captured_step_follows_the_weights():
    r, x = make(), counts(2, 24)
    states, mine = r.new_states(2), r.new_states(2)
    r.step(x, r.new_states(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = r.step(x, states)
    r.weights["head"].mul_(-2.0)
    graph.replay()
    assert torch.equal(got, r.step(x, mine))


def test_weights_that_the_caller_keeps():
    """8-bit weights made once are the caller's, and stay as they were."""
    r, x = make(), counts(2, 30, 24)
    kept, before = r.quantized(), r.read(x)[0]
    assert torch.equal(r.read(x, small=kept)[0], before)
    assert torch.equal(r.step(x[:, 0], r.new_states(2), small=kept), r.step(x[:, 0], r.new_states(2)))
    r.weights["head"].zero_()
    assert torch.equal(r.read(x, small=kept)[0], before) and not r.read(x)[0].any()


def test_counts_past_256():
    """bf16 has eight bits: larger counts are exact in the type that is asked for."""
    from libnrn_b200 import readout
    step, gid = np.repeat([3, 11], [257, 1001]), np.zeros(1258, np.int64)
    exact = readout.bin_spikes(step, gid, 4, 10, 2, group=4, dtype=torch.float32)
    assert exact.dtype == torch.float32 and exact.tolist() == [[257.0], [1001.0]]
    assert torch.equal(readout.bin_spikes(step, gid, 4, 10, 2, group=4), exact.to(torch.bfloat16))
    assert "256" in readout.bin_spikes.__doc__


def test_a_device_without_a_number():
    for device in ("cuda", torch.device("cuda"), "cuda:0", torch.device("cuda", 0)):
        r = make(device=device)
        assert r.device == torch.device("cuda", torch.cuda.current_device())
        r.read(counts(1, 5, 24))


def test_no_bins_and_no_sessions():
    r = make()
    answers, states = r.read(counts(2, 0, 24))
    assert answers.shape == (2, 0, 16) and not states[0].any()
    some = [s.normal_() for s in r.new_states(2)]
    assert torch.equal(r.read(counts(2, 0, 24), states=some)[1][0], some[0])
    assert r.read(counts(0, 7, 24))[0].shape == (0, 7, 16)
    assert r.step(counts(0, 24), r.new_states(3)).shape == (0, 16)
    with pytest.raises(N.NrnError):
        r.gradients(counts(1, 0, 24), counts(1, 0, 16))


def test_targets_of_another_shape_are_refused():
    """One target for all outputs would be taken for each of them."""
    r, x = make(), counts(1, 7, 24)
    r.gradients(x, x[..., :16])
    for bad in (x[..., :1], x, x[:, :6, :16]):
        with pytest.raises(N.NrnError, match="targets"):
            r.gradients(x, bad)
