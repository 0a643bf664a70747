"""The norms' gates where they saturate, element by element, and rows with
an infinity as 8 bits.

Tolerances, relative and for each element.  fp32: the row's norm (a sum of 64
squares and a reciprocal root, 2^-21), the exponential (2 ulp) and its
reciprocal and products (2^-21), and for silu's derivative sg (1 + x (1 - sg)),
whose bracket loses a factor of at most 5 where gates keep 0.25 from its zero at
-1.2785: together below 2^-18.  16-bit: the result's rounding (2^-8, 2^-11), and
2^-16 for an exponential by ex2.approx, whose argument, up to 43, is rounded to
2^-19."""
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TOL = {BF16: 2.0 ** -8 + 2.0 ** -16, FP16: 2.0 ** -11 + 2.0 ** -16, FP32: 2.0 ** -18}
EPS = 1e-6


def off(x, ref):
    return float(((x.double() - ref).abs() / ref.abs()).max())


@pytest.mark.parametrize("d", [64, 1024, 1001], ids=str)
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
def test_saturated_gates(dtype, act, d):
    from libnrn_b200 import gatednorm
    most = 8.0 if dtype == FP16 else 30.0            # past that fp16 has no normal numbers left
    gate = torch.linspace(-most, most, d, device="cuda").to(dtype).expand(3, d).contiguous()
    near = (gate.double() + 1.2785).abs() < 0.25
    gate[near] = 1.0
    gate[gate.abs() < 2.0 ** -10] = 0.5              # nor below that
    gen = torch.Generator(device="cuda").manual_seed(0)
    h, dy = ((torch.rand(3, d, device="cuda", generator=gen) + 0.5).to(dtype) for _ in range(2))
    h[:, ::2] *= -1
    zero = torch.zeros_like(h)
    y, _ = gatednorm.forward(zero, h, gate, eps=EPS, activation=act, want_z=False)
    g = gatednorm.backward(dy, None, zero, h, gate, eps=EPS, activation=act)
    hh = h.double() / (h.double().pow(2).mean(1, keepdim=True) + EPS).sqrt()
    sg = 1.0 / (1.0 + torch.exp(-gate.double()))
    other = 1.0 / (1.0 + torch.exp(gate.double()))   # 1 - sg
    x = gate.double()
    assert off(y, hh * (x * sg if act == "silu" else sg)) <= TOL[dtype]
    ref = dy.double() * hh * (sg * (1.0 + x * other) if act == "silu" else sg * other)
    assert off(g.gate, ref) <= TOL[dtype], off(g.gate, ref)


@pytest.mark.parametrize("shape", [(5, 256), (4, 1000), (3, 4096)], ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_an_infinity_as_8_bits(bad, shape):
    """z's block that holds no number is NaN throughout, as the quantiser makes it; the row's other blocks are what z is."""
    from libnrn_b200 import gatednorm, scaled
    x = torch.randn(*shape, device="cuda")
    x[1, 140] = bad
    _, z = gatednorm.forward(x, scaled=True)
    _, plain = gatednorm.forward(x)
    want = scaled.quantize(plain)
    assert torch.equal(z.dequantize().isnan(), want.dequantize().isnan())
    assert bool(z.dequantize()[1, 128:256].isnan().all()) and torch.equal(z.scales.isnan(), want.scales.isnan())


@pytest.mark.parametrize("dtype", [FP16, FP32], ids=str)
def test_z_as_8_bits_from_other_types(dtype):
    from libnrn_b200 import gatednorm
    for rows, d in ((3, 200), (65, 2048), (2, 8200), (3, 16384)):
        gen = torch.Generator(device="cuda").manual_seed(2)
        r, h, gate = (torch.randn(rows, d, device="cuda", generator=gen).to(dtype) for _ in range(3))
        _, z = gatednorm.forward(r, h, gate, scaled=True, eps=EPS)
        _, ref = R.gatednorm(r.double(), h.double(), gate.double(), None, None, None, EPS)
        v, s = R.quantized(ref)
        assert R.rel(z.scales, s) <= 2.0 ** -19
        assert float((z.values.float() != v.float()).float().mean()) <= 1e-3
