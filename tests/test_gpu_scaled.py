"""8-bit products with block scales: the quantisers bit for bit against the
definition in torch operations, the products against 64-bit products of the
same 8-bit values (tests/operator_refs.py).

Tolerance of a product, relative in the 2-norm: the result's own rounding (2^-9
bf16, 2^-12 fp16) and fp32 sums of 8-bit products (their terms are exact; each
of the sums of a block of 128 and of the blocks errs by at most its depth times
2^-24 of the sum of magnitudes, which for random signs is about the root of the
number of terms above the result: sqrt(k) * 2^-24 * 32 covers it)."""
import pytest
import torch

import operator_refs as R

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF16: 2.0 ** -9, FP16: 2.0 ** -12, FP32: 0.0}


def tol(dtype, k):
    return ROUND[dtype] + max(k, 1) ** 0.5 * 2.0 ** -19


def randn(*s, seed=0, dtype=FP32):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 128), (5, 127), (130, 129), (64, 1000), (257, 300), (1, 4096)], ids=str)
def test_quantize(shape, dtype):
    from libnrn_b200 import scaled
    x = randn(*shape, seed=1, dtype=dtype)
    x[:, ::7] *= 30
    x[0] = 0
    for row_block in (1, 128):
        q = scaled.quantize(x, row_block=row_block)
        v, s = R.quantized(x, row_block)
        assert torch.equal(q.scales, s) and torch.equal(q.values.view(torch.uint8) if q.values.is_contiguous() else q.values.contiguous().view(torch.uint8), v.view(torch.uint8))
        assert torch.equal(q.dequantize(torch.float64), R.dequantized(v, s, row_block).float().double())
    q = scaled.quantize(x, transpose=True)
    v, s = R.quantized(x.t().contiguous())
    assert torch.equal(q.scales, s) and torch.equal(q.values.contiguous().view(torch.uint8), v.view(torch.uint8))
    w = scaled.quantize(x, row_block=128)
    t = scaled.transpose(w)
    assert t.shape == (shape[1], shape[0])
    assert torch.equal(t.values.contiguous().view(torch.uint8), w.values.contiguous().t().contiguous().view(torch.uint8)) and torch.equal(t.scales, w.scales.t())


@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_strides_and_ends(transpose):
    from libnrn_b200 import scaled
    x = randn(70, 333, seed=2)[:, 1:300]            # rows on no 16-byte boundary
    q = scaled.quantize(x, transpose=transpose)
    v, s = R.quantized(x.t() if transpose else x)
    assert torch.equal(q.scales, s) and torch.equal(q.values.contiguous().view(torch.uint8), v.contiguous().view(torch.uint8))
    for tiny in (0.0, 1e-30, 2.0 ** -70):           # far below the smallest scale
        d = scaled.quantize(torch.full((2, 130), tiny, device="cuda"), transpose=transpose).dequantize()
        assert bool(torch.isfinite(d).all()) and float(d.abs().max()) <= 2.0 ** -64
    big = torch.full((2, 130), 3e38, device="cuda")
    assert R.rel(scaled.quantize(big, transpose=transpose).dequantize(), big.t() if transpose else big) <= 2.0 ** -4
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = randn(200, 300, seed=3)
        y[4, 140] = bad
        d = scaled.quantize(y, transpose=transpose).dequantize()
        d = d.t() if transpose else d
        assert bool(torch.isnan(d[:128, 140] if transpose else d[4, 128:256]).all())
        assert int(torch.isnan(d).sum()) == 128
    # nothing to do
    assert scaled.quantize(torch.empty(0, 7, device="cuda"), transpose=transpose).values.numel() == 0


SIZES = [(1, 64, 128), (1, 4096, 4096), (2, 7, 16), (3, 128, 1), (16, 129, 130), (17, 1000, 640), (33, 256, 2048), (64, 64, 64), (100, 300, 500),
         (128, 2048, 1024), (129, 1, 129), (130, 257, 384), (515, 1001, 1400), (1000, 40, 3000), (1024, 2048, 256), (2050, 3000, 128)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_product(size, dtype):
    from libnrn_b200 import scaled
    m, n, k = size
    a, w = randn(m, k, seed=4), randn(n, k, seed=5)
    a[:, ::11] *= 20
    a = scaled.quantize(a)
    for row_block in (128, 1):
        b = scaled.quantize(w, row_block=row_block)
        y = scaled.product(a, b, dtype=dtype)
        ref = R.dequantized(a.values, a.scales) @ R.dequantized(b.values, b.scales, row_block).t()
        assert y.shape == (m, n) and y.dtype == dtype
        assert R.rel(y, ref) <= tol(dtype, k), R.rel(y, ref)
        assert torch.equal(y, scaled.product(a, b, dtype=dtype))
    aw = scaled.quantize(a.dequantize(), row_block=128)      # block scales on both sides
    b = scaled.quantize(w, row_block=128)
    ref = R.dequantized(aw.values, aw.scales, 128) @ R.dequantized(b.values, b.scales, 128).t()
    assert R.rel(scaled.product(aw, b, dtype=dtype), ref) <= tol(dtype, k)
    scaled.check()


def test_values_of_a_checkpoint():
    """Values and scales that were not made here: row-major scales, values in a wider buffer."""
    from libnrn_b200 import scaled
    v, s = R.quantized(randn(200, 300, seed=6), 128)
    buf = torch.zeros(200, 512, device="cuda", dtype=torch.uint8)
    buf[:, 16:316] = v.view(torch.uint8)
    b = scaled.Scaled(buf.view(torch.float8_e4m3fn)[:, 16:316], s.contiguous(), 128)
    a = scaled.quantize(randn(140, 300, seed=7))
    out = torch.zeros(140, 500, device="cuda", dtype=BF16)
    y = scaled.product(a, b, out=out[:, 3:203])
    ref = R.dequantized(a.values, a.scales) @ R.dequantized(v, s, 128).t()
    assert R.rel(y, ref) <= tol(BF16, 300)
    assert not out[:, :3].any() and not out[:, 203:].any()


@pytest.mark.parametrize("size", [(1, 64, 64), (100, 200, 300), (129, 1000, 136), (700, 256, 513)], ids=str)
def test_gradients(size):
    from libnrn_b200 import scaled
    m, n, k = size
    x, dy, w = randn(m, k, seed=8, dtype=BF16), randn(m, n, seed=9, dtype=BF16), scaled.quantize(randn(n, k, seed=10), row_block=128)
    dx, dw = scaled.product_backward(dy, x, w)
    wd = R.dequantized(w.values, w.scales, 128)
    qd = R.dequantized(*R.quantized(dy))
    assert dx.dtype == BF16 and R.rel(dx, qd @ wd) <= tol(BF16, n)
    assert dw.dtype == FP32
    assert R.rel(dw, R.dequantized(*R.quantized(dy.t())) @ R.dequantized(*R.quantized(x.t())).t()) <= tol(FP32, m)
    # and against the gradients of the product itself: each operand is off by at most half of e4m3's last bit, 2^-4
    assert R.rel(dx, dy.double() @ wd) <= 2.0 ** -4 and R.rel(dw, dy.double().t() @ x.double()) <= 2 * 2.0 ** -4
    # a change of the weights along dw changes sum(dy * y) by |dw|^2 a unit: differences of the product in 64 bits
    e = 1e-3
    f = lambda v: float((dy.double() * (x.double() @ v.t())).sum())      # noqa: E731
    d = (f(wd + e * dw.double()) - f(wd - e * dw.double())) / (2 * e)
    assert abs(d - float(dw.double().square().sum())) <= 2 * 2.0 ** -4 * abs(d)


def test_no_rows_no_columns():
    from libnrn_b200 import scaled
    e = scaled.quantize(torch.empty(0, 64, device="cuda"))
    w = scaled.quantize(randn(10, 64), row_block=128)
    assert scaled.product(e, w).shape == (0, 10) and scaled.product(w, e).shape == (10, 0)
    z = scaled.Scaled.empty(3, 0, torch.device("cuda", 0))
    assert torch.equal(scaled.product(z, scaled.Scaled.empty(5, 0, torch.device("cuda", 0))), torch.zeros(3, 5, device="cuda", dtype=BF16))


def test_a_bad_row_stays_alone():
    from libnrn_b200 import scaled
    x = randn(300, 256, seed=11)
    w = scaled.quantize(randn(200, 256, seed=12), row_block=128)
    good = scaled.product(scaled.quantize(x), w)
    x[7, 3] = float("nan")
    y = scaled.product(scaled.quantize(x), w)
    assert bool(torch.isnan(y[7]).all())
    keep = [i for i in range(300) if i != 7]
    assert torch.equal(y[keep], good[keep])


def test_streams_and_graphs():
    """Split products on two streams at once, and captured."""
    from libnrn_b200 import scaled
    a = [scaled.quantize(randn(8, 4096, seed=20 + i)) for i in range(2)]
    w = scaled.quantize(randn(2048, 4096, seed=22), row_block=128)
    want = [scaled.product(x, w) for x in a]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[scaled.product(a[i], w, stream=streams[i]) for i in range(2)] for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for pair in got for i, y in enumerate(pair))
    x = randn(8, 4096, seed=23)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = scaled.product(scaled.quantize(x), w)
    for s in (24, 25):
        x.copy_(randn(8, 4096, seed=s))
        graph.replay()
        assert torch.equal(y, scaled.product(scaled.quantize(x), w))
    scaled.check()


def test_refusals():
    from libnrn_b200 import _native as N
    from libnrn_b200 import scaled
    x = randn(64, 256)
    q, w = scaled.quantize(x), scaled.quantize(x, row_block=128)
    for call in (lambda: scaled.quantize(x.cpu()), lambda: scaled.quantize(x.double()), lambda: scaled.quantize(x.t()),
                 lambda: scaled.quantize(x, row_block=64), lambda: scaled.quantize(x, row_block=128, transpose=True),
                 lambda: scaled.quantize(x[None]), lambda: scaled.transpose(q), lambda: scaled.product(q, x),
                 lambda: scaled.product(q, scaled.quantize(x[:, :128].contiguous())), lambda: scaled.product(q, w, dtype=torch.float64),
                 lambda: scaled.product(q, w, out=torch.empty(64, 63, device="cuda")), lambda: scaled.product_backward(x, x, q),
                 lambda: scaled.product_backward(x, x[:10], w), lambda: scaled.Scaled(q.values, q.scales.half()),
                 lambda: scaled.Scaled(q.values, q.scales, 128), lambda: scaled.Scaled(q.values.view(torch.uint8), q.scales),
                 lambda: scaled.Scaled(q.values[:, 1:129], q.scales[:, :1])):
        with pytest.raises(N.NrnError):
            call()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize("shape", [(700, 1001, 130), (2100, 1344, 100), (2051, 2176, 300), (700, 129, 256), (1500, 264, 64)], ids=str)
def test_product_ragged_edges(shape, dtype):
    """Results that end inside a tile or inside one half of it, rows on 16 bytes and off: nothing beside them is written."""
    from libnrn_b200 import scaled
    m, n, k = shape
    a, b = scaled.quantize(randn(m, k, seed=3)), scaled.quantize(randn(n, k, seed=4), row_block=128)
    want = a.dequantize(torch.float64) @ b.dequantize(torch.float64).t()
    for first, pitch in ((0, n + 24 - n % 8), (5, n + 11)):
        out = torch.full((m + 2, pitch), 7.0, device="cuda", dtype=dtype)
        y = out[1:m + 1, first:first + n]
        scaled.product(a, b, out=y)
        scaled.check()
        assert R.rel(y, want) <= tol(dtype, k)
        y.fill_(7.0)
        assert bool((out == 7.0).all())
