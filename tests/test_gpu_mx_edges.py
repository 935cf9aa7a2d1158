"""The microscaled operators where a call is unlike the usual one: saved-tensor hooks, other streams, empty sides,
far scales, long sums."""
import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import turboloader_b200 as tb
from mx_reference import decode

pytestmark = pytest.mark.gpu

FORMATS = ("nvfp4", "mxfp4", "mxfp8")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


# ---- saved tensors that the node does not own --------------------------------------------------------------------

def _on_host_and_back():
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda())


@pytest.mark.parametrize("how", ["hooks", "checkpoint"])
@pytest.mark.parametrize("held", ["neither", "x", "weight"])
@pytest.mark.parametrize("m,n,k", [(40, 72, 200), (3000, 64, 96), (64, 2000, 130)])
def test_gradients_under_saved_tensor_hooks_and_checkpoints(how, held, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w, up = (torch.randn(*s, generator=g, device="cuda") for s in ((m, k), (n, k), (m, n)))
    x, w = (tb.mx_quantize(x, "mxfp4") if held == "x" else x.requires_grad_(True)), (tb.mx_quantize(w, "mxfp4") if held == "weight" else w.requires_grad_(True))
    leaves = [t for t in (x, w) if isinstance(t, torch.Tensor)]

    def layer(*leaves):
        a, b = x if held == "x" else leaves[0], w if held == "weight" else leaves[-1]
        return tb.mx_linear(a, b, "mxfp4", dtype=torch.float32)

    want = torch.autograd.grad(layer(*leaves), leaves, up)
    for _ in range(3):
        if how == "hooks":
            with _on_host_and_back():
                y = layer(*leaves)
        else:
            y = checkpoint(layer, *leaves, use_reentrant=False)
        got = torch.autograd.grad(y, leaves, up)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- empty sides -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lead", [(), (3,), (2, 3), (2, 0)])
@pytest.mark.parametrize("n", [0, 5])
def test_gradients_of_any_leading_dimensions_and_of_no_rows(lead, n):
    x = torch.randn(*lead, 40, device="cuda", requires_grad=True)
    w = torch.randn(n, 40, device="cuda", requires_grad=True)
    y = tb.mx_linear(x, w, "mxfp8")
    up = torch.randn(*lead, n, device="cuda")
    gx, gw = torch.autograd.grad(y, [x, w], up)
    xv, wv = (tb.mx_quantize(t.detach().reshape(-1, 40), "mxfp8").dequantize().double() for t in (x, w))
    u = up.double().reshape(xv.shape[0], n)
    assert y.shape == (*lead, n) and gx.shape == x.shape and gw.shape == w.shape
    # sums of at most 6 terms of three bf16 parts each, fp32
    assert ((gx.reshape(-1, 40).double() - u @ wv).abs() <= 24 * 2.0 ** -23 * (u.abs() @ wv.abs()) + 1e-38).all()
    assert ((gw.double() - u.T @ xv).abs() <= 24 * 2.0 ** -23 * (u.T.abs() @ xv.abs()) + 1e-38).all()


# ---- writes of one cache on several streams ----------------------------------------------------------------------

@pytest.mark.parametrize("wrapped", [False, True])
def test_first_long_writes_of_a_cache_on_two_streams(wrapped):
    """Different slots, nothing before them that would order the two: the first stream is kept busy, the second is not."""
    slots, cols = 1200, 96
    for round_ in range(4):
        cache = tb.MxCache.empty(slots, 1, cols, "mxfp8")
        if wrapped:
            cache = tb.MxCache(cache.codes, cache.scales, cols, "mxfp8", status=cache.status)
        x = torch.randn(slots, cols, device="cuda")
        order = torch.randperm(slots, device="cuda")
        parts = order[:600], order[600:]
        first, second = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(first):
            torch.cuda._sleep(20_000_000)
        for at, stream in zip(parts, (first, second)):
            with torch.cuda.stream(stream):
                rows = x[at]
                cache.write(at, rows)
        torch.cuda.synchronize()
        assert torch.equal(cache.read(None, torch.float32).view(slots, cols), tb.mx_quantize(x, "mxfp8").dequantize())
        assert cache.device_status() == 0


def test_a_first_long_write_that_is_captured():
    slots, cols = 700, 64
    cache = tb.MxCache.empty(slots, 1, cols)
    index, x = torch.arange(600, device="cuda"), torch.randn(600, 1, cols, device="cuda")
    index[599] = 3                                      # named twice: the last one stays
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(index, x)
    for _ in range(2):
        x.mul_(2)
        graph.replay()
        want = tb.mx_quantize(x.view(600, cols)).dequantize()
        got = cache.read(None, torch.float32).view(slots, cols)
        assert torch.equal(got[:3], want[:3]) and torch.equal(got[3], want[599]) and torch.equal(got[4:599], want[4:599])
        assert not got[599:].any()
        cache.write(index, x.flip(1) * 3)               # one that is not captured, between replays
        assert torch.equal(cache.read(index[:3], torch.float32).view(3, cols), tb.mx_quantize(x[:3].view(3, cols) * 3).dequantize())


def test_lengths_of_a_cache_that_are_out_of_range_are_clamped_and_reported():
    tokens, cols = 3, 40
    for bad, size in ((tokens + 2, tokens), (-1, 0)):
        cache = tb.MxCache.empty(5, tokens, cols, ragged=True)
        cache.write(torch.arange(5, device="cuda"), torch.randn(5, tokens, cols, device="cuda"))
        cache.lengths[2] = bad
        for read in (cache.read, cache.read_mx):
            values, lengths = read(torch.tensor([0, 1], device="cuda"))
            assert cache.device_status() == 0
            values, lengths = read(torch.tensor([1, 2], device="cuda"))
            assert lengths.tolist() == [tokens, size] and cache.device_status() == 16
            values = values.dequantize() if isinstance(values, tb.MxTensor) else values
            assert bool(values[1].any()) == (size > 0)
            cache.status.zero_()


def test_a_feature_loader_whose_consumer_changes_streams():
    """The last batch is read on a busy stream; what the first stream allocates meanwhile does not touch its indices."""
    n, dim = 4096, 32
    loader = tb.CudaFeatureLoader(n, 1, dim, n // 2, format="mxfp8", shuffle=True, dtype=torch.float32, return_indices=True)
    x = torch.randn(n, 1, dim, device="cuda")
    loader.write(np.arange(n), x)
    want = loader.cache.read(None, torch.float32)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    batches = iter(loader)
    next(batches)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        batch, index = next(batches)
    at = index.cpu()
    del index
    assert next(batches, None) is None                    # the epoch's order is free now
    del batches
    filler = [torch.full((n,), -1, dtype=torch.int64, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(batch, want[at.cuda()]) and loader.device_status() == 0 and len(filler) == 4


# ---- scales on the device that change --------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_on_the_device_may_change_after_the_forward_pass(fmt):
    x, w = torch.randn(70, 96, device="cuda", requires_grad=True), torch.randn(50, 96, device="cuda", requires_grad=True)
    up = torch.randn(70, 50, device="cuda")
    want = torch.autograd.grad(tb.mx_linear(x, w, fmt, scale=0.5, weight_scale=0.25), [x, w], up)
    sx, sw = torch.tensor([0.5], device="cuda"), torch.tensor([0.25], device="cuda")
    y = tb.mx_linear(x, w, fmt, scale=sx, weight_scale=sw)
    q = tb.mx_quantize(x.detach(), fmt, scale=sx)
    sx.fill_(7), sw.fill_(9)
    got = torch.autograd.grad(y, [x, w], up)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(q.dequantize(), tb.mx_quantize(x.detach(), fmt, scale=0.5).dequantize())


# ---- far scales ------------------------------------------------------------------------------------------------

def _values(q):
    """What an MxTensor stands for without its tensor scale, float64."""
    return torch.from_numpy(decode(q.codes.cpu().numpy(), q.scales.cpu().numpy(), q.format, q.shape[-1])).cuda()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 200])
def test_products_of_very_large_and_very_small_rows(fmt, m):
    """Rows near the end of fp32's range times a weight near its beginning, either way round: the products are ordinary."""
    n, k = 150, 320
    g = torch.Generator(device="cuda").manual_seed(m)
    for large, small in ((2.0 ** 120, 2.0 ** -100), (2.0 ** -110, 2.0 ** 124), (2.0 ** -126, 2.0 ** 123), (2.0 ** 60, 2.0 ** -60)):
        a, b = (tb.mx_quantize(torch.rand(r, k, generator=g, device="cuda") * s, fmt) for r, s in ((m, large), (n, small)))
        av, bv = _values(a), _values(b)
        want = av @ bv.T
        got = tb.mx_matmul(a, b, torch.float32)
        assert torch.isfinite(got).all()
        assert ((got.double() - want).abs() <= (k + 2) * 2.0 ** -23 * want).all()      # no value is negative
    for at in (0, k - 1):                               # a block of NaN beside scales of any size
        x = torch.rand(m, k, generator=g, device="cuda") * 2.0 ** -126
        x[m - 1, at] = float("nan")
        got = tb.mx_matmul(tb.mx_quantize(x, fmt), b, torch.float32)
        assert torch.isnan(got[m - 1]).all() and torch.isfinite(got[:m - 1]).all()
        w = torch.rand(n, k, generator=g, device="cuda") * 2.0 ** -126
        w[7, at] = float("inf")
        got = tb.mx_matmul(a, tb.mx_quantize(w, fmt), torch.float32)
        assert torch.isnan(got[:, 7]).all() and torch.isfinite(got[:, 8:]).all() and torch.isfinite(got[:, :7]).all()


@pytest.mark.parametrize("fmt", FORMATS[1:])
@pytest.mark.parametrize("e", [-110, -118, -122, -128, -131])
def test_gradients_of_very_small_values(fmt, e):
    """bf16 ends at 2^-133: less than that is lost of a value of the weight, or of the gradient's fp32."""
    m, n, k = 200, 64, 96
    g = torch.Generator(device="cuda").manual_seed(-e)
    x = torch.randn(m, k, generator=g, device="cuda", requires_grad=True)
    for w_exponent, up_exponent in ((e, 60), (60, e)):
        q = tb.mx_quantize(torch.randn(n, k, generator=g, device="cuda") * 2.0 ** w_exponent, fmt)
        up = torch.randn(m, n, generator=g, device="cuda") * 2.0 ** up_exponent
        got, = torch.autograd.grad(tb.mx_linear(x, q, fmt), [x], up)
        w, u = q.dequantize().double(), up.double()
        lost = u.abs().sum(1, keepdim=True) if w_exponent == e else w.abs().sum(0, keepdim=True)
        # 3 stages of 4 instructions, and the values
        assert ((got.double() - u @ w).abs() <= 2.0 ** -133 * lost + 16 * 2.0 ** -23 * (u.abs() @ w.abs()) + 2.0 ** -149).all()


# ---- long sums -------------------------------------------------------------------------------------------------

def _check_long_sum(got, want, magnitude, stages):
    """An accumulator holds 8 stages of 4 instructions (16-bit results: 32), each of which may cut 2^-23 of the partial
    sum; the accumulators, and the parts of a split sum (74 at most, not less than 16 stages each), are added rounding to
    nearest.  Beside it half a step of the result's type."""
    hold = 8 if got.dtype == torch.float32 else 32
    parts = stages / 8 + min(74, stages / 16)
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + (4 * hold + parts + 4) * 2.0 ** -23 * magnitude
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() / bound).max())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("m,n,k", [(64, 96, 20000), (300, 520, 60000), (257, 130, 5001), (3, 40, 70000)])
def test_products_of_long_rows(fmt, positive, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(k)
    draw = (lambda r: torch.rand(r, k, generator=g, device="cuda")) if positive else (lambda r: torch.randn(r, k, generator=g, device="cuda"))
    a, b = tb.mx_quantize(draw(m), fmt), tb.mx_quantize(draw(n), fmt)
    av, bv = a.dequantize().double(), b.dequantize().double()
    for dtype in DTYPES:
        _check_long_sum(tb.mx_matmul(a, b, dtype), av @ bv.T, av.abs() @ bv.abs().T, -(-k // (128 if fmt == "mxfp8" else 256)))


@pytest.mark.parametrize("fmt,m,n,k", [("nvfp4", 3000, 2570, 1000), ("mxfp4", 300, 5000, 131), ("mxfp8", 5000, 130, 250), ("nvfp4", 20000, 1300, 1000),
                                       ("mxfp4", 9000, 1027, 2045)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("positive", [False, True])
def test_gradients_of_long_sums(fmt, m, n, k, dtype, positive):
    """Tiles of 128 and of 256 columns, more tiles than pairs of CTAs, either sum split and not, odd rows."""
    g = torch.Generator(device="cuda").manual_seed(m)
    draw = (lambda *s: torch.rand(*s, generator=g, device="cuda")) if positive else (lambda *s: torch.randn(*s, generator=g, device="cuda"))
    x, w, up = (draw(*s).to(dtype) for s in ((m, k), (n, k), (m, n)))
    x.requires_grad_(True), w.requires_grad_(True)
    gx, gw = torch.autograd.grad(tb.mx_linear(x, w, fmt, dtype=dtype), [x, w], up)
    xv, wv = (tb.mx_quantize(t.detach(), fmt).dequantize().double() for t in (x, w))
    u, terms = up.double(), {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
    _check_long_sum(gx, u @ wv, u.abs() @ wv.abs(), -(-n // 64) * terms)
    _check_long_sum(gw, u.T @ xv, u.abs().T @ xv.abs(), -(-m // 64) * terms)
    for wanted, value in ((x, gx), (w, gw)):              # one alone is made in the same way
        assert torch.equal(torch.autograd.grad(tb.mx_linear(x, w, fmt, dtype=dtype), [wanted], up)[0], value)
