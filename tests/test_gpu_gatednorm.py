"""The gated norms against their 64-bit form and its gradients by torch's
differentiation of that form (tests/operator_refs.py), and against differences.

Tolerances, in the 2-norm.  Outputs are compared with the 64-bit ones rounded
to their type, which they equal but where fp32's last bits decide a rounding:
2^-9 in bf16 and 2^-12 in fp16, relative.  fp32 outputs and the sums over rows:
about 30 fp32 operations an element, 2^-19, relative to the terms that are
added: h's gradient is a difference that cancels where a row has few elements
(for one element to nothing but eps), so its terms are counted, not the
difference.  8-bit outputs: equal scales to 2^-19, values that differ only
where fp32's last bits decide a rounding: fewer than 1 in 1,000."""
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TOL = {BF16: 2.0 ** -9 + 2.0 ** -19, FP16: 2.0 ** -12 + 2.0 ** -19, FP32: 2.0 ** -19}
EPS = 1e-5
SHAPES = [(1, 1), (3, 8), (5, 100), (7, 256), (130, 264), (9, 512), (4, 1000), (1, 2048), (33, 2052), (11, 2560), (6, 4096), (3, 8192), (2, 8200), (2, 16384),
          (1000, 64)]


def make(rows, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, device="cuda", generator=g)
    big = {n: (r(rows, d) * f).to(dtype) for n, f in (("residual", 1), ("h", 3), ("gate", 2), ("dy", 1), ("dz", 1))}
    return big, {"alpha": 0.5 + 0.1 * r(d), "w_post": 1 + 0.1 * r(d), "w_pre": 1 + 0.1 * r(d)}


def reference(x, p, act="silu", grads=True):
    leaf = {n: (t.double().clone().requires_grad_(True) if t is not None else None) for n, t in {**x, **p}.items()}
    y, z = R.gatednorm(leaf["residual"], leaf.get("h"), leaf.get("gate"), leaf.get("alpha"), leaf.get("w_post"), leaf.get("w_pre"), EPS, act)
    if not grads:
        return y.detach(), z.detach(), None
    total = 0.0
    if x.get("dy") is not None:
        total = total + (y * x["dy"].double()).sum()
    if x.get("dz") is not None:
        total = total + (z * x["dz"].double()).sum()
    total.backward()
    return y.detach(), z.detach(), {n: t.grad for n, t in leaf.items() if t is not None and n not in ("dy", "dz")}


def close(x, ref, tol, terms=0.0):
    """terms: the 2-norm of what was added to give ref, where that is larger than ref."""
    assert x.shape == ref.shape
    ref = ref.to(x.dtype).double()
    off = float((x.double() - ref).norm())
    assert off <= tol * float(ref.norm()) + 2.0 ** -19 * terms, (off, float(ref.norm()), terms)


def run(x, p, act="silu"):
    from libnrn_b200 import gatednorm
    args = (x["residual"], x.get("h"), x.get("gate"))
    kw = dict(eps=EPS, activation=act, **p)
    y, z = gatednorm.forward(*args, **kw)
    return y, z, gatednorm.backward(x.get("dy"), x.get("dz"), *args, **kw)


def compare(x, p, dtype, act="silu"):
    y, z, g = run(x, p, act)
    ry, rz, rg = reference(x, p, act)
    close(y, ry, TOL[dtype])
    close(z, rz, TOL[dtype])
    for n in ("residual", "h", "gate"):
        if x.get(n) is not None:
            assert getattr(g, n).dtype == dtype
            terms = 0.0
            if n == "h":      # inv_h dhh, of which its part along h is taken away
                h, d = x["h"].double(), rg["residual"]
                a = torch.ones_like(h) if x.get("gate") is None else x["gate"].double()
                a = a if x.get("gate") is None else (torch.sigmoid(a) * a if act == "silu" else torch.sigmoid(a))
                terms = float((d * a * (p["alpha"].double() if p.get("alpha") is not None else 1.0) * (p["w_post"].double() if p.get("w_post") is not None else 1.0)
                               / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt()).norm())
            close(getattr(g, n), rg[n], TOL[dtype], terms)
    for n in ("alpha", "w_post", "w_pre"):
        if p.get(n) is not None:
            close(getattr(g, n), rg[n] if rg[n] is not None else torch.zeros_like(p[n]).double(), 2.0 ** -19 * (1 + x["residual"].shape[0] ** 0.5 / 8))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, dtype):
    x, p = make(*shape, dtype)
    compare(x, p, dtype)


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("gone", [(), ("gate",), ("alpha",), ("w_post", "w_pre"), ("h", "gate", "alpha", "w_post"), ("dy",), ("dz",), ("gate", "alpha", "w_post", "w_pre")],
                         ids=str)
def test_parts_left_out(gone, act):
    x, p = make(37, 400, FP32, seed=1)
    compare({n: t for n, t in x.items() if n not in gone}, {n: t for n, t in p.items() if n not in gone}, FP32, act)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=str)
@pytest.mark.parametrize("kind", ["wide", "one off"])
def test_strides(kind, dtype):
    x, p = make(21, 321 if kind == "one off" else 640, dtype, seed=2)
    x = {n: (t[:, 1:] if kind == "one off" else t[:, 64:576]) for n, t in x.items()}
    p = {n: torch.randn(x["h"].shape[1], device="cuda") for n in p}
    compare(x, p, dtype)


@pytest.mark.parametrize("shape", [(1, 128), (3, 1000), (65, 2048), (2, 8200), (10, 264)], ids=str)
def test_scaled_output(shape):
    from libnrn_b200 import gatednorm, scaled
    x, p = make(*shape, BF16, seed=3)
    y, z = gatednorm.forward(x["residual"], x["h"], x["gate"], scaled=True, eps=EPS, **p)
    assert isinstance(z, scaled.Scaled) and z.shape == shape
    ry, rz, _ = reference(x, p, grads=False)
    v, s = R.quantized(rz)
    close(z.scales, s, 2.0 ** -19)
    assert float((z.values.float() != v.float()).float().mean()) <= 1e-3
    close(z.dequantize(), rz, 2.0 ** -4)
    close(y, ry, TOL[BF16])
    # it is the operand of the product
    w = scaled.quantize(torch.randn(50, shape[1], device="cuda"), row_block=128)
    close(scaled.product(z, w, dtype=FP32), R.dequantized(z.values, z.scales) @ R.dequantized(w.values, w.scales, 128).t(), shape[1] ** 0.5 * 2.0 ** -19)


def test_backward_is_the_differences():
    """sum(y dy + z dz) along each gradient, by central differences of the 64-bit form."""
    x, p = make(4, 96, FP32, seed=4)
    _, _, g = run(x, p)
    every = {**{n: x[n] for n in ("residual", "h", "gate")}, **p}

    def value(at):
        y, z = R.gatednorm(at["residual"], at["h"], at["gate"], at["alpha"], at["w_post"], at["w_pre"], EPS)
        return float((y * x["dy"].double()).sum() + (z * x["dz"].double()).sum())
    base = {n: t.double() for n, t in every.items()}
    for n in every:
        d = getattr(g, n).double()
        e = 1e-4 / float(d.norm())
        slope = (value({**base, n: base[n] + e * d}) - value({**base, n: base[n] - e * d})) / (2 * e)
        assert abs(slope - float(d.square().sum())) <= 1e-5 * abs(slope)


def test_rows_that_are_nothing():
    from libnrn_b200 import gatednorm
    x, p = make(5, 200, BF16, seed=5)
    x["h"][1] = 0
    x["residual"][2] = 0
    x["h"][2] = 0
    compare(x, p, BF16)
    x["h"][3, 7] = float("nan")
    y, z, g = run(x, p)
    keep = [0, 1, 2, 4]
    ry, rz, _ = reference({n: t[keep] for n, t in x.items()}, p)
    close(y[keep], ry, TOL[BF16])
    close(z[keep], rz, TOL[BF16])
    assert bool(torch.isnan(z[3]).all())
    e = {n: t[:0] for n, t in x.items()}
    y, z, g = run(e, p)
    assert y.shape == (0, 200) and not g.alpha.any() and not g.w_pre.any()
    # without h, y is the residual and z its norm
    y, z = gatednorm.forward(x["residual"], w_pre=p["w_pre"], eps=EPS)
    assert y is x["residual"]
    close(z, R.gatednorm(x["residual"].double(), None, None, None, None, p["w_pre"].double(), EPS)[1], TOL[BF16])
    assert gatednorm.forward(x["residual"], x["h"], want_z=False)[1] is None


def test_runs_repeat_and_streams():
    from libnrn_b200 import gatednorm
    x, p = make(3000, 2560, BF16, seed=6)
    a, b = run(x, p), run(x, p)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(s, t) for s, t in zip(a[2], b[2]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = gatednorm.backward(x["dy"], x["dz"], x["residual"], x["h"], x["gate"], eps=EPS, stream=side, **p)
    side.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(g, a[2]))


def test_refusals():
    from libnrn_b200 import _native as N
    from libnrn_b200 import gatednorm
    x, p = make(4, 64, BF16)
    r, h, gate = x["residual"], x["h"], x["gate"]
    for call in (lambda: gatednorm.forward(r.cpu()), lambda: gatednorm.forward(r.double()), lambda: gatednorm.forward(r.t()), lambda: gatednorm.forward(r[0]),
                 lambda: gatednorm.forward(r, h.half()), lambda: gatednorm.forward(r, h[:3]), lambda: gatednorm.forward(r, None, gate),
                 lambda: gatednorm.forward(r, h, gate, activation="tanh"), lambda: gatednorm.forward(r, h, alpha=p["alpha"][:63]),
                 lambda: gatednorm.forward(r, h, alpha=p["alpha"].half()), lambda: gatednorm.forward(r, h, eps=-1.0),
                 lambda: gatednorm.forward(r, h, eps=float("nan")), lambda: gatednorm.forward(r, w_post=p["w_post"]),
                 lambda: gatednorm.forward(torch.empty(1, 16385, device="cuda")), lambda: gatednorm.backward(x["dy"][:3], None, r, h)):
        with pytest.raises(N.NrnError):
            call()
