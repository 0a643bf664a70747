"""What the tensor operators (linattn, scaled, gatednorm) share."""
import contextlib
import os
import subprocess
import sys
import threading
import time

import pytest
import torch

from libnrn_b200 import _native as N

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def randn(*s, seed=0, dtype=FP32):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def together(*calls):
    """Runs the calls in a thread each; the first error is raised here."""
    errors, start = [], threading.Barrier(len(calls))

    def run(f):
        try:
            start.wait()
            f()
        except BaseException as e:      # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(f,)) for f in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


# ------------------------------------------------------------------- threads

def test_threads_on_one_stream_take_turns(monkeypatch):
    """Two calls that use one workspace are never in the library at once, whatever their threads: between the launches of
    one, another's would overwrite its operands.  (Nothing is launched here.)"""
    from libnrn_b200 import scaled
    x, dy = randn(8, 4096, dtype=BF16), randn(8, 2048, seed=1, dtype=BF16)
    a, w = scaled.quantize(x), scaled.quantize(randn(2048, 4096, seed=2), row_block=128)
    guard, inside, most = threading.Lock(), [0], [0]

    def slowly(*_):
        with guard:
            inside[0] += 1
            most[0] = max(most[0], inside[0])
        time.sleep(0.02)
        with guard:
            inside[0] -= 1
        return 0
    for name in ("nrn_cuda_scaled_product", "nrn_cuda_scaled_backward"):
        monkeypatch.setattr(N.lib(), name, slowly)
    together(*[lambda: [scaled.product_backward(dy, x, w) for _ in range(4)]] * 2, lambda: [scaled.product(a, w) for _ in range(4)])
    assert most[0] == 1
    # on streams of their own they need not wait
    side = [torch.cuda.Stream() for _ in range(2)]
    together(*[lambda s=s: [scaled.product(a, w, stream=s) for _ in range(8)] for s in side])
    assert most[0] == 2


def test_threads_on_one_stream_are_right():
    from libnrn_b200 import scaled
    cases = []
    for i, (m, n, k) in enumerate([(200, 512, 1024), (300, 256, 640), (8, 2048, 4096), (16, 4096, 4096)]):
        x, dy = randn(m, k, seed=10 + i, dtype=BF16), randn(m, n, seed=20 + i, dtype=BF16)
        w = scaled.quantize(randn(n, k, seed=30 + i), row_block=128)
        cases.append((x, dy, w, scaled.product(scaled.quantize(x), w), scaled.product_backward(dy, x, w)))

    def work(x, dy, w, y, grads):
        for _ in range(40):
            assert torch.equal(scaled.product(scaled.quantize(x), w), y)
            assert all(torch.equal(a, b) for a, b in zip(scaled.product_backward(dy, x, w), grads))
    together(*[lambda c=c: work(*c) for c in cases])
    scaled.check()


# -------------------------------------------------------- numbers as tensors

@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_a_number_in_a_tensor_is_read_at_every_call(device):
    from libnrn_b200 import gatednorm, linattn
    q, k, v = (randn(1, 20, 2, 32, seed=i) for i in range(3))
    g = torch.full((2,), -0.1, device="cuda")
    scale, eps = torch.tensor(0.5, device=device), torch.tensor(1e-6, device=device)
    r, state = randn(4, 64), torch.zeros(1, 2, 32, 32, device="cuda")
    for s, e in ((0.5, 1e-6), (0.25, 0.5)):
        scale.fill_(s)
        eps.fill_(e)
        assert torch.equal(linattn.forward(q, k, v, g, scale=scale)[0], linattn.forward(q, k, v, g, scale=s)[0])
        assert all(torch.equal(a, b) for a, b in zip(linattn.backward(q, q, k, v, g, scale=scale), linattn.backward(q, q, k, v, g, scale=s)))
        one = [linattn.step(q[:, 0], k[:, 0], v[:, 0], g, state.clone(), scale=f) for f in (scale, s)]
        assert torch.equal(*one)
        assert torch.equal(gatednorm.forward(r, eps=eps)[1], gatednorm.forward(r, eps=float(eps))[1])
        assert torch.equal(gatednorm.backward(None, r, r, eps=eps).residual, gatednorm.backward(None, r, r, eps=float(eps)).residual)


# -------------------------------------------------- waits that gave up, graphs

FIRST = """
import torch
from libnrn_b200 import _native as N, _tensors, {module}
x = torch.randn(8, 4096, device="cuda"); big = torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda"); del big
torch.cuda.synchronize()
q = torch.randn(1, 70, 2, 64, device="cuda").bfloat16(); ld = torch.full((2,), -0.1, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    {call}
{module}.check()                                   # nothing ran yet: nothing gave up
graph.replay()
{module}.check()
_tensors.flag(0).tensor().fill_(5)
graph.replay()                                     # a replay takes no flag down
try:
    {module}.check()
    raise SystemExit("the flag was lost")
except N.NrnError:
    pass
print("told")
"""


@pytest.mark.parametrize("module,call", [("linattn", "linattn.forward(q, q, q, ld)"), ("gatednorm", "gatednorm.forward(x, x)"),
                                         ("scaled", "scaled.product(scaled.quantize(x), scaled.quantize(x, row_block=128))")], ids=["linattn", "gatednorm", "scaled"])
def test_the_first_call_of_a_process_may_be_captured(module, call):
    r = subprocess.run([sys.executable, "-c", FIRST.format(module=module, call=call)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "told" in r.stdout, r.stdout + r.stderr


def test_a_wait_that_gave_up_is_told_once_and_leaves_nothing():
    """After the flag is told it is down again, and products whose counters were left above zero are right."""
    from libnrn_b200 import _tensors, linattn, scaled
    a, w = scaled.quantize(randn(8, 4096)), scaled.quantize(randn(2048, 4096, seed=1), row_block=128)
    want = scaled.product(a, w)
    linattn.check()
    for shared in scaled._streams.values():
        if shared.work is not None:
            shared.work[:4096].view(torch.int32).fill_(1)
    _tensors.flag(torch.cuda.current_device()).tensor().fill_(5)
    with pytest.raises(N.NrnError, match="timed out"):
        scaled.check()
    scaled.check()
    assert torch.equal(scaled.product(a, w), want) and torch.equal(scaled.product(a, w), want)


def test_check_names_a_device_as_torch_does():
    from libnrn_b200 import _tensors, scaled
    scaled.product(scaled.quantize(randn(8, 256)), scaled.quantize(randn(20, 256), row_block=128))
    i = torch.cuda.current_device()
    for name in (None, "cuda", torch.device("cuda"), f"cuda:{i}", torch.device("cuda", i), i):
        scaled.check(name)
        _tensors.flag(i).tensor().fill_(5)
        with pytest.raises(N.NrnError):
            scaled.check(name)


def test_check_waits_for_every_stream():
    from libnrn_b200 import _tensors, scaled
    flag, side = _tensors.flag(torch.cuda.current_device()).tensor(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        flag.fill_(5)
    with pytest.raises(N.NrnError):
        scaled.check()
    scaled.check()


# ------------------------------------------------------------------ gradients

def test_tensors_that_want_gradients_are_refused():
    """Results have no graph: a call that would lose a gradient without a word is refused where gradients are recorded."""
    from libnrn_b200 import gatednorm, linattn, scaled
    q, k, v = (randn(1, 20, 2, 32, seed=i) for i in range(3))
    g, r, p = torch.full((2,), -0.1, device="cuda"), randn(4, 64), torch.ones(64, device="cuda")
    state = torch.zeros(1, 2, 32, 32, device="cuda")
    w = scaled.quantize(randn(16, 64), row_block=128)
    calls = [lambda q=q, k=k, v=v, state=state: linattn.forward(q, k, v, g, state=state),
             lambda q=q, k=k, v=v: linattn.backward(q, q, k, v, g),
             lambda q=q, k=k, v=v, state=state: linattn.step(q[:, 0], k[:, 0], v[:, 0], g, state),
             lambda r=r: scaled.quantize(r), lambda r=r: scaled.product_backward(r[:, :16].contiguous(), r, w),
             lambda r=r, p=p: gatednorm.forward(r, r, w_post=p), lambda r=r: gatednorm.backward(r, None, r)]
    for call in calls:
        call()
        for name in call.__code__.co_varnames[:call.__code__.co_argcount]:
            wants = {"q": q, "k": k, "v": v, "state": state, "r": r, "p": p}[name].clone().requires_grad_(True)
            with pytest.raises(N.NrnError, match="gradient"):
                call(**{name: wants})
            with torch.no_grad():
                call(**{name: wants})
            with pytest.raises(N.NrnError, match="gradient"):      # what was allowed there is not remembered here
                call(**{name: wants})


# -------------------------------------------------------------------- devices

def test_sizes_are_asked_for_on_the_tensors_device(monkeypatch):
    """The workspaces' sizes depend on the device: they are asked for after the switch to it."""
    from libnrn_b200 import gatednorm, scaled
    switched = [0]

    def watched(real):
        @contextlib.contextmanager
        def on(*a):
            with real(*a) as s:
                switched[0] += 1
                try:
                    yield s
                finally:
                    switched[0] -= 1
        return on
    asked = []

    def sizes(name):
        real = getattr(N.lib(), name)

        def call(*a):
            asked.append((name, switched[0]))
            return real(*a)
        return call
    for m in (scaled, gatednorm):
        monkeypatch.setattr(m, "on", watched(m.on))
    names = ["nrn_cuda_scaled_workspace", "nrn_cuda_scaled_backward_workspace", "nrn_cuda_gatednorm_workspace"]
    for n in names:
        monkeypatch.setattr(N.lib(), n, sizes(n))
    x = randn(37, 1111, dtype=BF16)                 # layouts that no other test has
    w = scaled.quantize(randn(53, 1111), row_block=128)
    scaled.product(scaled.quantize(x), w)
    scaled.product_backward(randn(37, 53, dtype=BF16), x, w)
    gatednorm.forward(x)
    assert sorted(n for n, _ in asked) == sorted(names) and all(s == 1 for _, s in asked), asked


def replayed(call, change):
    """The results of `call` captured and replayed after `change` of its inputs, and those of a call after it."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    change()
    graph.replay()
    return got, call()


def test_steps_norms_and_gradients_in_graphs():
    from libnrn_b200 import gatednorm, linattn, scaled
    # two sequences that are split, shared heads: every kernel of the chain
    q, k, v, do = (randn(2, 3000, h, 64, seed=i, dtype=BF16) for i, h in enumerate((4, 2, 2, 4)))
    g = torch.full((4,), -0.01, device="cuda")
    got, want = replayed(lambda: linattn.backward(do, q, k, v, g), lambda: do.copy_(do.flip(1)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, dy, w = randn(300, 640, seed=5, dtype=BF16), randn(300, 256, seed=6, dtype=BF16), scaled.quantize(randn(256, 640, seed=7), row_block=128)
    got, want = replayed(lambda: scaled.product_backward(dy, x, w), lambda: (dy.copy_(dy.flip(0)), x.copy_(x.flip(1))))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    p = torch.rand(640, device="cuda")
    got, want = replayed(lambda: gatednorm.forward(x, x, x, w_post=p, scaled=True), lambda: x.copy_(x.flip(0)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1].dequantize(), want[1].dequantize())
    got, want = replayed(lambda: gatednorm.backward(x, x, x, x, x, w_post=p, w_pre=p), lambda: x.copy_(x.flip(0)))
    assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)
    state = randn(5, 4, 64, 64, seed=8)
    slots = torch.tensor([4, 0], device="cuda", dtype=torch.int32)
    one = lambda s: linattn.step(q[:, 0], k[:, 0], v[:, 0], g, s, slots=slots)      # noqa: E731
    graph, mine = torch.cuda.CUDAGraph(), state.clone()
    one(mine)
    with torch.cuda.graph(graph):
        o = one(state)
    state.copy_(mine)
    for _ in range(3):
        graph.replay()
        assert torch.equal(o, one(mine)) and torch.equal(state, mine)
    linattn.check()


# ------------------------------------------------------------ other streams

def _on_side():
    """Calls on a stream of the caller's choice, by name: (input made anew, call of it and the stream that gives its results)."""
    from libnrn_b200 import gatednorm, linattn, scaled
    n = 1 << 19
    q, big = randn(1, n // 256, 4, 64, dtype=BF16), randn(n // 256, 256, dtype=BF16)
    g, w = torch.full((4,), -0.1, device="cuda"), scaled.quantize(randn(512, 256, seed=1), row_block=128)
    square = scaled.quantize(randn(256, 256, seed=2), row_block=128)
    return {
        "forward": (q.clone, lambda x, s: linattn.forward(x, x, x, g, stream=s)),
        "backward": (q.clone, lambda x, s: linattn.backward(x, x, x, x, g, stream=s)),
        "step": (q[0].clone, lambda x, s: [linattn.step(x, x, x, g, torch.zeros(n // 256, 4, 64, 64, device="cuda"), stream=s)]),
        "quantize": (big.clone, lambda x, s: [scaled.quantize(x, stream=s).values]),
        "transpose": (lambda: scaled.quantize(randn(2048, 1024), row_block=128), lambda x, s: [scaled.transpose(x, stream=s).values]),
        "product": (lambda: scaled.quantize(randn(8192, 256)), lambda x, s: [scaled.product(x, w, stream=s)]),
        "product_backward": (big.clone, lambda x, s: scaled.product_backward(x, x, square, stream=s)),
        "norm": (big.clone, lambda x, s: gatednorm.forward(x, x, x, stream=s)),
        "norm backward": (big.clone, lambda x, s: [t for t in gatednorm.backward(x, x, x, x, x, stream=s) if t is not None]),
    }


@pytest.mark.parametrize("name", ["forward", "backward", "step", "quantize", "transpose", "product", "product_backward", "norm", "norm backward"])
def test_memory_is_not_given_out_while_another_stream_uses_it(name):
    make, call = _on_side()[name]
    side = torch.cuda.Stream()
    call(make(), None)
    torch.cuda.synchronize()

    def busy(stream):
        with torch.cuda.stream(stream):
            torch.cuda._sleep(400_000_000)               # 0.2 s

    def fresh(n):
        """Addresses that the allocator gives the current stream for as much memory again."""
        got = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(4)]
        return [t.data_ptr() for t in got]
    # an input that is dropped after the call, before the call has run
    x = make()
    side.wait_stream(torch.cuda.current_stream())
    busy(side)
    held = x if isinstance(x, torch.Tensor) else x.values
    at, size = held.data_ptr(), held.numel() * held.element_size()
    results = call(x, side)
    del x, held
    assert at not in fresh(size)
    torch.cuda.synchronize()
    # a result that is dropped while the current stream may still read it
    busy(torch.cuda.current_stream())
    held = [(t.data_ptr(), t.numel() * t.element_size()) for t in results if t.numel() * t.element_size() >= 1 << 20]
    del results
    with torch.cuda.stream(side):
        for p, n in held:
            assert p not in fresh(n)
    torch.cuda.synchronize()


def test_another_stream_inside_a_captured_graph():
    from libnrn_b200 import gatednorm, linattn, scaled
    q, x = randn(1, 700, 2, 64, dtype=BF16), randn(8, 4096, seed=1, dtype=BF16)
    g, w = torch.full((2,), -0.1, device="cuda"), scaled.quantize(randn(2048, 4096, seed=2), row_block=128)
    side = torch.cuda.Stream()

    def calls(s):
        return (*linattn.forward(q, q, q, g, stream=s), scaled.product(scaled.quantize(x, stream=s), w, stream=s), gatednorm.forward(x, x, x, stream=s)[1],
                *scaled.product_backward(x[:, :2048], x, w, stream=s))
    calls(None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        got = calls(side)
        torch.cuda.current_stream().wait_stream(side)
    q.copy_(q.flip(1))
    x.copy_(x.flip(0))
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, calls(None)))
    scaled.check()
