"""Microscaled operators on the GPU against their plain float64 form (tests/mx_reference.py)."""
import numpy as np
import pytest
import torch

import turboloader_b200 as tb
from mx_reference import BLOCK, decode, encode

pytestmark = pytest.mark.gpu

FORMATS = ("nvfp4", "mxfp4", "mxfp8")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _values(rows, cols, dtype, seed, special=True):
    """Features of mixed sizes: ties of the grids, zeros, tiny and huge blocks, infinities and NaN."""
    g = np.random.default_rng(seed)
    x = g.standard_normal((rows, cols)) * np.exp2(g.integers(-6, 6, (rows, 1)))
    x = np.where(g.random(x.shape) < 0.3, np.round(x * 4) / 4, x)
    if special:
        for kind, v in enumerate((0.0, 1e-41, 3e38, 1e4, np.inf, -np.inf, np.nan, 2.0 ** -127)):
            r = g.integers(0, rows)
            at = g.integers(0, cols)
            x[r, at:at + (1 if kind > 2 else 40)] = v
    with np.errstate(over="ignore"):
        return torch.from_numpy(x.astype(np.float32)).to(dtype)


def _np(t):
    return t.detach().float().cpu().numpy()


def _same(got, want):
    got, want = np.asarray(got), np.asarray(want)
    assert got.shape == want.shape
    assert np.array_equal(got, want), f"{(got != want).sum()} of {got.size} differ, first at {np.argwhere(got != want)[:3].tolist()}"


def _as_type(v64, scale, dtype):
    """code * block scale (exact in fp32), times the tensor scale in fp32, rounded to the type."""
    with np.errstate(over="ignore", invalid="ignore"):
        return torch.from_numpy((v64.astype(np.float32) * np.float32(scale)).astype(np.float32)).to(dtype)


def _equal_values(got, want):
    assert got.dtype == want.dtype and got.shape == want.shape
    got, want = got.cpu(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


# ---- quantisation ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (2, 15), (5, 16), (4, 17), (3, 31), (7, 32), (2, 33), (9, 127), (6, 128), (3, 129),
                                       (33, 1000), (1, 4096), (2, 4099), (260, 96)])
def test_quantize_gives_the_codes_of_exact_arithmetic(fmt, dtype, rows, cols):
    x = _values(rows, cols, dtype, rows * 1000 + cols)
    for scale in (1.0, 0.03125, 0.37):
        q = tb.mx_quantize(x.cuda(), fmt, scale=scale)
        codes, scales = encode(_np(x), fmt, scale)
        _same(q.codes.cpu().numpy(), codes)
        _same(q.scales.cpu().numpy(), scales)
        for out in DTYPES:
            _equal_values(q.dequantize(out), _as_type(decode(codes, scales, fmt, cols), scale, out))


def test_quantize_of_slices_scales_on_the_device_and_many_dimensions():
    wide = _values(64, 300, torch.bfloat16, 3).cuda()
    for lo, hi in ((0, 256), (1, 257), (7, 40), (8, 300)):
        q = tb.mx_quantize(wide[::2, lo:hi], "mxfp4")
        _same(q.codes.cpu().numpy(), encode(_np(wide[::2, lo:hi]), "mxfp4")[0])
    ts = torch.tensor([0.125], device="cuda")
    q = tb.mx_quantize(wide.view(4, 16, 300)[:, :, :64], "nvfp4", scale=ts)
    assert q.shape == (4, 16, 64) and q.dequantize().shape == (4, 16, 64)
    codes, scales = encode(_np(wide[:, :64]), "nvfp4", 0.125)
    _same(q.codes.cpu().numpy(), codes)
    _equal_values(q.dequantize(torch.bfloat16).view(64, 64), _as_type(decode(codes, scales, "nvfp4", 64), 0.125, torch.bfloat16))
    empty = tb.mx_quantize(wide[:0], "nvfp4")
    assert empty.dequantize().shape == (0, 300)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 7, 16, 17, 25, 31, 32, 33, 48, 63, 70, 100, 315])
def test_quantize_rows_that_end_anywhere_in_aligned_and_odd_matrices(fmt, dtype, cols):
    """Rows at multiples of 32 bytes, and at every other distance and start, cut off at any column."""
    for pitch, start in ((320, 0), (328, 0), (321, 0), (336, 3), (352, 16)):
        wide = _values(37, pitch, dtype, cols + pitch)
        x = wide[:, start:start + cols]
        q = tb.mx_quantize(wide.cuda()[:, start:start + cols], fmt)
        codes, scales = encode(_np(x), fmt)
        _same(q.codes.cpu().numpy(), codes)
        _same(q.scales.cpu().numpy(), scales)
        cache = tb.MxCache.empty(20, 2, cols, fmt)
        index = torch.arange(18, device="cuda")
        cache.write(index, wide[:36].cuda().view(18, 2, pitch)[:, :, start:start + cols])
        _same(cache.codes[:18].reshape(36, -1).cpu().numpy(), codes[:36])
        _same(cache.scales[:18].reshape(36, -1).cpu().numpy(), scales[:36])


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_float16_value_and_every_code(fmt):
    """All finite float16 values, one block each beside a fixed largest value, and every byte a row can hold."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    v = bits[torch.isfinite(bits)]
    x = torch.zeros(len(v), 32, dtype=torch.float16)
    x[:, 0], x[:, 5], x[:, 17] = 65504.0, v, v
    q = tb.mx_quantize(x.cuda(), fmt)
    codes, scales = encode(_np(x), fmt)
    _same(q.codes.cpu().numpy(), codes)
    _same(q.scales.cpu().numpy(), scales)
    n = 256
    codes = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 128 if fmt == "mxfp8" else 64))
    scales = np.tile(np.roll(np.arange(256), 97).astype(np.uint8)[:, None], (1, 128 // BLOCK[fmt]))
    if fmt != "nvfp4":
        scales = np.where((scales > 244) & (scales < 255), 244, scales)  # code * scale stays finite
    held = tb.MxTensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), (n, 128), fmt)
    _equal_values(held.dequantize(), _as_type(decode(codes, scales, fmt, 128), 1.0, torch.float32))


# ---- the cache ----------------------------------------------------------------------------------------------

def _expected_write(codes, scales, lengths, index, x, new, fmt, tokens):
    """numpy twin of MxCache.write on (slots, tokens, pitch) arrays, in place."""
    for i, s in enumerate(index):
        if not 0 <= s < codes.shape[0] or s in index[i + 1:]:
            continue
        size = tokens if new is None else min(max(int(new[i]), 0), tokens)
        if size:
            codes[s, :size], scales[s, :size] = encode(x[i, :size], fmt)
        if lengths is not None:
            lengths[s] = size


def _filled(slots, tokens, cols, fmt, ragged, seed):
    g = np.random.default_rng(seed)
    cache = tb.MxCache.empty(slots, tokens, cols, fmt, ragged=ragged)
    codes, scales = encode(_np(_values(slots * tokens, cols, torch.float32, seed, special=False)), fmt)
    cache.codes.copy_(torch.from_numpy(codes).view(cache.codes.shape))
    cache.scales.copy_(torch.from_numpy(scales).view(cache.scales.shape))
    lengths = None
    if ragged:
        lengths = g.integers(0, tokens + 1, slots).astype(np.int32)
        cache.lengths.copy_(torch.from_numpy(lengths))
    return cache, codes.reshape(slots, tokens, -1), scales.reshape(slots, tokens, -1), lengths


def _check_cache(cache, codes, scales, lengths):
    _same(cache.codes.cpu().numpy(), codes)
    _same(cache.scales.cpu().numpy(), scales)
    if lengths is not None:
        _same(cache.lengths.cpu().numpy(), lengths)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slots,tokens,cols,n,ragged", [(1, 1, 1, 1, False), (5, 1, 64, 3, True), (9, 7, 100, 9, True), (40, 3, 33, 17, False),
                                                        (700, 1, 48, 600, True), (300, 2, 16, 290, False), (4, 196, 768, 3, True)])
def test_cache_write_and_read(fmt, dtype, slots, tokens, cols, n, ragged):
    cache, codes, scales, lengths = _filled(slots, tokens, cols, fmt, ragged, n)
    g = np.random.default_rng(n + 1)
    x = _values(n * tokens, cols, dtype, n + 2).view(n, tokens, cols)
    index = g.permutation(slots)[:n]
    if n > 2:
        index[0], index[-2] = index[n // 2], -1       # one slot named twice, one index outside
    if n > 8:
        index[3], index[4], index[5] = index[6], index[6], slots  # a slot named three times
    new = g.integers(0, tokens + 1, n).astype(np.int32) if ragged else None
    if ragged and n > 1:
        new[1] = tokens + 3                            # clamped and reported
    for _ in range(2):                                 # the claims of the first call are gone in the second
        cache.write(torch.from_numpy(index).cuda(), x.cuda(), lengths=None if new is None else torch.from_numpy(new).cuda())
        _expected_write(codes, scales, lengths, index.tolist(), _np(x), new, fmt, tokens)
        _check_cache(cache, codes, scales, lengths)
    bad_length = 16 if ragged and n > 1 else 0
    assert cache.device_status() == (1 if n > 2 else 0) | bad_length
    cache.status.zero_()

    order = np.concatenate([g.permutation(slots), [slots + 5, -7, 0, 0]])
    want = decode(codes.reshape(slots * tokens, -1), scales.reshape(slots * tokens, -1), fmt, cols).reshape(slots, tokens, cols)
    sizes = np.array([(lengths[s] if ragged else tokens) if 0 <= s < slots else 0 for s in order], np.int32)
    values = np.zeros((len(order), tokens, cols))
    held_c, held_s = np.zeros((len(order), tokens, codes.shape[2]), np.uint8), np.zeros((len(order), tokens, scales.shape[2]), np.uint8)
    for j, s in enumerate(order):
        if sizes[j]:
            values[j, :sizes[j]] = want[s, :sizes[j]]
            held_c[j, :sizes[j]], held_s[j, :sizes[j]] = codes[s, :sizes[j]], scales[s, :sizes[j]]
    got = cache.read(torch.from_numpy(order).cuda(), dtype)
    got, got_sizes = got if ragged else (got, None)
    _equal_values(got, _as_type(values, 1.0, dtype))
    mx = cache.read_mx(torch.from_numpy(order).cuda())
    mx, mx_sizes = mx if ragged else (mx, None)
    _same(mx.codes.cpu().numpy(), held_c)
    _same(mx.scales.cpu().numpy(), held_s)
    if ragged:
        _same(got_sizes.cpu().numpy(), sizes)
        _same(mx_sizes.cpu().numpy(), sizes)
    assert cache.device_status() == 1
    everything = cache.read(None, torch.float32)
    _equal_values((everything[0] if ragged else everything), _as_type(
        np.where(np.arange(tokens)[None, :, None] < (lengths if ragged else np.full(slots, tokens))[:, None, None], want, 0.0), 1.0, torch.float32))


def test_cache_without_lengths_given_takes_whole_samples_and_strided_input():
    cache, codes, scales, lengths = _filled(6, 4, 40, "mxfp8", True, 5)
    wide = _values(6 * 9, 50, torch.float16, 6).view(6, 9, 50).cuda()
    x = wide[1:4, 2:6, 3:43]                            # misaligned rows, gaps between rows and samples
    cache.write(torch.tensor([5, 0, 2], device="cuda"), x)
    _expected_write(codes, scales, lengths, [5, 0, 2], _np(x), None, "mxfp8", 4)
    _check_cache(cache, codes, scales, lengths)
    cache.write(torch.zeros(0, dtype=torch.int64, device="cuda"), wide[:0, :4, :40])
    _check_cache(cache, codes, scales, lengths)
    assert cache.read(torch.zeros(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 4, 40)


def test_cache_refusals():
    cache = tb.MxCache.empty(4, 2, 32)
    x, i = torch.zeros(2, 2, 32, device="cuda"), torch.tensor([0, 1], device="cuda")
    n = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    for call, error in ((lambda: cache.write(i, x, lengths=n), ValueError), (lambda: cache.write(i.int(), x), TypeError),
                        (lambda: cache.write(i[:1], x), ValueError), (lambda: cache.write(i, x.double()), TypeError),
                        (lambda: cache.write(i, x[:, :1]), ValueError), (lambda: cache.write(i, x[..., ::2]), ValueError),
                        (lambda: cache.write(i, x[:, :1].expand(2, 2, 32)), ValueError), (lambda: cache.write(i.cpu(), x), TypeError),
                        (lambda: cache.read(i, torch.int8), TypeError), (lambda: cache.read(i, out=x), ValueError),
                        (lambda: tb.mx_quantize(x[..., ::2]), ValueError), (lambda: tb.mx_quantize(x.int()), TypeError),
                        (lambda: tb.mx_quantize(x[0, 0].expand(3, 32)), ValueError), (lambda: tb.mx_quantize(x, scale=0.0), ValueError),
                        (lambda: tb.mx_quantize(x, scale=torch.ones(2, device="cuda")), TypeError),
                        (lambda: tb.MxTensor(cache.codes, cache.scales, (4, 2, 200), "nvfp4"), ValueError),
                        (lambda: tb.mx_matmul(tb.mx_quantize(x[0]), tb.mx_quantize(x[0], "mxfp4")), ValueError),
                        (lambda: tb.mx_matmul(tb.mx_quantize(x[0]), tb.mx_quantize(x[0, :, :16])), ValueError),
                        (lambda: tb.mx_linear(x, x), ValueError), (lambda: tb.mx_linear(x, tb.mx_quantize(x[0]), "mxfp8"), ValueError)):
        with pytest.raises(error):
            call()


# ---- the product ---------------------------------------------------------------------------------------------

def _held(rows, cols, fmt, seed, spread=0, scale=1.0):
    """An MxTensor of normal values (rows of different sizes), and its values in float64 on the GPU."""
    g = np.random.default_rng(seed)
    x = (g.standard_normal((rows, cols)) * np.exp2(g.integers(-spread, spread + 1, (rows, 1)))).astype(np.float32)
    codes, scales = encode(x, fmt)
    held = tb.MxTensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), (rows, cols), fmt, scale=scale)
    return held, torch.from_numpy(decode(codes, scales, fmt, cols)).cuda()


def _close(got, want, magnitude, terms, dtype):
    """|error| <= half a step of the result's type + `terms` roundings of fp32 (a whole step each, for sums
    that cut instead of round) of the sum of the magnitudes."""
    bound = torch.finfo(dtype).eps / 2 * want.abs() + (terms + 2) * 2.0 ** -23 * magnitude + torch.finfo(dtype).tiny
    worst = ((got.double() - want).abs() - bound).max()
    assert got.dtype == dtype and torch.isfinite(got).all() and worst <= 0, f"over the bound by {worst}"


SHAPES = [(1, 1, 1), (1, 7, 33), (1, 1000, 4096), (1, 257, 129), (2, 129, 1000), (4, 300, 512), (5, 64, 96), (8, 520, 260), (9, 40, 4096), (13, 501, 200),
          (16, 128, 128), (17, 128, 256), (31, 1, 300), (64, 65, 64), (100, 333, 1003), (127, 255, 257), (128, 256, 512), (129, 257, 513),
          (300, 130, 90), (1000, 96, 640), (257, 1025, 1537), (700, 900, 2048)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(fmt, m, n, k):
    (a, av), (b, bv) = _held(m, k, fmt, m + k, 3), _held(n, k, fmt, n + 7 * k, 3)
    want, magnitude = av @ bv.T, av.abs() @ bv.abs().T
    for dtype in DTYPES:
        if dtype == torch.float16 and want.abs().max() > 60000:
            continue
        _close(tb.mx_matmul(a, b, dtype), want, magnitude, k, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 6, 40, 200])
def test_product_scales_nan_rows_and_out(fmt, m):
    n, k = 150, 320
    (a, av), (b, bv) = _held(m, k, fmt, 1, scale=0.37), _held(n, k, fmt, 2, scale=torch.tensor([0.11], device="cuda"))
    want, magnitude = av @ bv.T * float(np.float32(0.37)) * float(np.float32(0.11)), av.abs() @ bv.abs().T * 0.05
    out = torch.empty(m, n, device="cuda")
    assert tb.mx_matmul(a, b, torch.float32, out=out) is out
    _close(out, want, magnitude, k, torch.float32)
    a.scales[m - 1, 1] = 0x7F if fmt == "nvfp4" else 0xFF  # one block of NaN: its row, and no other
    b.scales[77, 0] = 0x7F if fmt == "nvfp4" else 0xFF
    got = tb.mx_matmul(a, b, torch.float32)
    assert torch.isnan(got[m - 1]).all() and torch.isnan(got[:, 77]).all()
    keep = torch.ones(n, dtype=torch.bool)
    keep[77] = False
    if m > 1:
        _close(got[:m - 1][:, keep], want[:m - 1][:, keep], magnitude[:m - 1][:, keep], k, torch.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k", [300, 4100])
def test_a_few_rows_are_the_first_rows_of_many(fmt, k):
    """Each row's sums are its own: what other rows hold, or what ran before on the device, changes no bit of them."""
    n, many = 330, 256
    (a, av), (b, bv) = _held(many, k, fmt, 1, 3), _held(n, k, fmt, 2, 3)
    whole = tb.mx_matmul(a, b, torch.float32)
    _close(whole, av @ bv.T, av.abs() @ bv.abs().T, k, torch.float32)
    nothing = tb.mx_quantize(torch.full((300, k), float("nan"), device="cuda"), fmt)
    up = torch.randn(many, n, device="cuda")
    for dtype in DTYPES:
        x = torch.randn(many, k, device="cuda", dtype=dtype, requires_grad=True)
        all_rows, = torch.autograd.grad(tb.mx_linear(x, b, fmt), [x], up.to(dtype))
        for m in (5, 8, 9, 24, 31, 32, 33, 63, 127, 128, 129, 250):
            part = tb.MxTensor(a.codes[:m], a.scales[:m], (m, k), fmt)
            assert torch.isnan(tb.mx_matmul(nothing, nothing, torch.float32)).all()
            assert torch.equal(tb.mx_matmul(part, b, torch.float32), whole[:m])
            few = x.detach()[:m].requires_grad_(True)
            lost = torch.full((m, n), float("nan"), device="cuda", dtype=dtype)
            y = tb.mx_linear(few, b, fmt)
            bad, = torch.autograd.grad(y, [few], lost, retain_graph=True)
            rows, = torch.autograd.grad(y, [few], up.to(dtype)[:m])
            assert torch.isnan(bad).all() and torch.equal(rows, all_rows[:m])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [2, 3, 4])
def test_two_to_four_rows_of_small_and_large_matrices(fmt, m):
    for n, k in ((70, 40), (9000, 2048), (17000, 2048)):
        (a, av), (b, bv) = _held(m, k, fmt, 1, 3), _held(n, k, fmt, 2, 3)
        _close(tb.mx_matmul(a, b, torch.float32), av @ bv.T, av.abs() @ bv.abs().T, k, torch.float32)


def test_product_of_nothing():
    x = torch.zeros(0, 64, device="cuda")
    w = tb.mx_quantize(torch.ones(5, 64, device="cuda"))
    assert tb.mx_matmul(tb.mx_quantize(x), w).shape == (0, 5)
    assert tb.mx_matmul(w, tb.mx_quantize(x)).shape == (5, 0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_product_gives_the_same_bits_every_time(fmt):
    for m, n, k in ((1, 512, 4096), (33, 700, 2048), (500, 300, 1000)):
        (a, _), (b, _) = _held(m, k, fmt, 5, 4), _held(n, k, fmt, 6, 4)
        first = tb.mx_matmul(a, b, torch.float32)
        for _ in range(5):
            assert torch.equal(first, tb.mx_matmul(a, b, torch.float32))


# ---- gradients --------------------------------------------------------------------------------------------------

TERMS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 5, 7), (1, 300, 64), (40, 1, 130), (129, 257, 100), (256, 128, 256), (300, 129, 515), (1000, 64, 72),
                                   (2050, 200, 136)])
def test_linear_and_its_gradients(fmt, dtype, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype).requires_grad_(True)
    w = (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).to(dtype).requires_grad_(True)
    up = torch.randn(m, n, generator=g, device="cuda").to(dtype)
    y = tb.mx_linear(x, w, fmt)
    y.backward(up)
    xv = torch.from_numpy(decode(*encode(_np(x), fmt), fmt, k)).cuda()
    wv = torch.from_numpy(decode(*encode(_np(w), fmt), fmt, k)).cuda()
    _close(y.detach(), xv @ wv.T, xv.abs() @ wv.abs().T, k, dtype)
    u = up.double()
    _close(x.grad, u @ wv, u.abs() @ wv.abs(), n * TERMS[dtype], dtype)
    _close(w.grad, u.T @ xv, u.abs().T @ xv.abs(), m * TERMS[dtype], dtype)


def test_gradients_of_mixed_types_held_operands_and_scales():
    k, n = 200, 72
    held, hv = _held(30, k, "nvfp4", 3, scale=0.5)
    w = (torch.randn(n, k, device="cuda") * 0.1).requires_grad_(True)            # float32 weight, bfloat16 result
    y = tb.mx_linear(held, w, "nvfp4", weight_scale=0.25, dtype=torch.bfloat16)
    up = torch.randn(30, n, device="cuda").to(torch.bfloat16)
    (gw,) = torch.autograd.grad(y, [w], up)
    assert gw.dtype == torch.float32
    _close(gw, up.double().T @ (hv * 0.5), up.double().abs().T @ (hv.abs() * 0.5), 30, torch.float32)
    qw, wv = _held(n, k, "nvfp4", 4, scale=2.0)
    x = torch.randn(2, 15, k, device="cuda", dtype=torch.float16, requires_grad=True)
    y = tb.mx_linear(x, qw, "nvfp4")
    assert y.shape == (2, 15, n) and y.dtype == torch.float16
    y.float().sum().backward()                                                    # an expanded gradient
    u = torch.ones(30, n, device="cuda", dtype=torch.float64)
    _close(x.grad.view(30, k), u @ (wv * 2), u.abs() @ (wv.abs() * 2), 2 * n, torch.float16)
    assert not tb.mx_linear(held, qw, "nvfp4").requires_grad
    with torch.no_grad():
        assert not tb.mx_linear(held, w, "nvfp4").requires_grad


def test_linear_of_nothing():
    w = torch.randn(5, 40, device="cuda", requires_grad=True)
    x = torch.randn(0, 40, device="cuda", requires_grad=True)
    y = tb.mx_linear(x, w, "mxfp4")
    assert y.shape == (0, 5)
    gx, gw = torch.autograd.grad(y, [x, w], torch.ones(0, 5, device="cuda"))
    assert gx.shape == (0, 40) and torch.equal(gw, torch.zeros(5, 40, device="cuda"))
    w = torch.randn(0, 40, device="cuda", requires_grad=True)
    x = torch.randn(3, 40, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = tb.mx_linear(x, w, "nvfp4")
    gx, gw = torch.autograd.grad(y, [x, w], torch.ones(3, 0, device="cuda"))
    assert y.shape == (3, 0) and gw.shape == (0, 40) and torch.equal(gx, torch.zeros_like(x))


def test_infinities_and_nan_in_the_gradient_stay_in_their_rows():
    g = torch.Generator(device="cuda").manual_seed(4)
    m, n, k = 130, 70, 64
    for dtype in DTYPES:
        x = torch.randn(m, k, generator=g, device="cuda").to(dtype).requires_grad_(True)
        w = torch.randn(n, k, generator=g, device="cuda").to(dtype).requires_grad_(True)
        clean = torch.randn(m, n, generator=g, device="cuda").to(dtype)
        dirty = clean.clone()
        dirty[3, 5], dirty[129, 7] = float("nan"), float("inf")
        y = tb.mx_linear(x, w, "mxfp8")
        ax, aw = torch.autograd.grad(y, [x, w], clean, retain_graph=True)
        bx, bw = torch.autograd.grad(y, [x, w], dirty)
        assert torch.isnan(bx[3]).all() and not torch.isfinite(bx[129]).any() and torch.isnan(bw[5]).all() and not torch.isfinite(bw[7]).any()
        rows, cols = torch.ones(m, dtype=torch.bool), torch.ones(n, dtype=torch.bool)
        rows[[3, 129]], cols[[5, 7]] = False, False
        assert torch.equal(ax[rows], bx[rows]) and torch.equal(aw[cols], bw[cols])


def test_gradients_against_differences():
    """The product is linear in each operand's values: moving one value between two points of its grid, scale
    unchanged, moves the result by the difference times the other operand."""
    k, n, m = 64, 24, 9
    g = np.random.default_rng(8)
    x = torch.from_numpy(g.choice([-3.0, -1.0, 0.5, 2.0], (m, k)).astype(np.float32)).cuda()
    w = torch.from_numpy(g.choice([-2.0, -0.5, 1.0, 1.5], (n, k)).astype(np.float32)).cuda()
    x[:, ::16], w[:, ::16] = 6.0, 6.0                                              # the blocks' scales are 1
    up = torch.randn(m, n, device="cuda")
    x.requires_grad_(True), w.requires_grad_(True)
    (tb.mx_linear(x, w, "nvfp4") * up).sum().backward()
    for t, at in ((x, (4, 17)), (w, (20, 33))):
        with torch.no_grad():
            before = (tb.mx_linear(x, w, "nvfp4").double() * up.double()).sum()
            old = float(t[at])
            t[at] = 4.0
            after = (tb.mx_linear(x, w, "nvfp4").double() * up.double()).sum()
            t[at] = old
        slope = float(after - before) / (4.0 - old)
        # both sides: sums of <= 24 products of values up to 6, fp32
        assert abs(slope - float(t.grad[at])) <= 64 * 2.0 ** -23 * 6 * float(up.abs().sum())


def test_shared_and_broadcast_inputs():
    k, n = 48, 40
    row = torch.randn(1, k, device="cuda", requires_grad=True)
    w = torch.randn(n, k, device="cuda", requires_grad=True)
    y = tb.mx_linear(row.expand(6, k), w, "mxfp8") + tb.mx_linear(row, w, "mxfp8")
    y.sum().backward()
    wv = torch.from_numpy(decode(*encode(_np(w), "mxfp8"), "mxfp8", k)).cuda()
    xv = torch.from_numpy(decode(*encode(_np(row), "mxfp8"), "mxfp8", k)).cuda()
    u = torch.ones(12, n, device="cuda", dtype=torch.float64)                      # y broadcast the second term: 6 + 6
    _close(row.grad, (u @ wv).sum(0, keepdim=True), (u @ wv.abs()).sum(0, keepdim=True), 3 * n + 12, torch.float32)
    _close(w.grad, (12 * xv).expand(n, k), (12 * xv.abs()).expand(n, k), 3 * 12 + 12, torch.float32)


# ---- together: streams, graphs, the loader ------------------------------------------------------------------------

def test_another_stream_gives_the_same_results():
    side = torch.cuda.Stream()
    x = torch.randn(200, 300, device="cuda")
    w = torch.randn(100, 300, device="cuda")
    index = torch.randperm(50, device="cuda")
    want_q = tb.mx_quantize(x)
    want = tb.mx_matmul(want_q, tb.mx_quantize(w), torch.float32)
    torch.cuda.synchronize()
    q = tb.mx_quantize(x, stream=side)
    cache = tb.MxCache.empty(50, 4, 300)
    side.wait_stream(torch.cuda.current_stream())
    cache.write(index, x.view(50, 4, 300), stream=side)
    back = cache.read(index, torch.float32, stream=side)
    got = tb.mx_matmul(q, tb.mx_quantize(w, stream=side), torch.float32, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(back.view(200, 300), want_q.dequantize())
    with torch.cuda.stream(side):
        assert torch.equal(tb.mx_matmul(q, tb.mx_quantize(w), torch.float32), want)
    torch.cuda.synchronize()


def test_calls_on_several_streams_at_once():
    """Products, gradients, writes and reads that overlap in time, each on data of its own."""
    streams = [torch.cuda.Stream() for _ in range(4)]
    work, want = [], []
    for i, fmt in enumerate(("nvfp4", "mxfp4", "mxfp8", "nvfp4")):
        g = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randn(700 + 64 * i, 640, generator=g, device="cuda")
        w = torch.randn(500, 640, generator=g, device="cuda")
        up = torch.randn(x.shape[0], 500, generator=g, device="cuda")
        cache = tb.MxCache.empty(400, 2, 640, fmt)
        index = torch.randperm(400, generator=g, device="cuda")[:300 + i]

        def step(x=x, w=w, up=up, cache=cache, index=index, fmt=fmt):
            a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
            y = tb.mx_linear(a, b, fmt)
            ga, gb = torch.autograd.grad(y, [a, b], up)
            cache.write(index, x[:600].view(300, 2, 640).repeat(2, 1, 1)[:index.shape[0]])
            return y.detach(), ga, gb, cache.read(index, torch.float32), tb.mx_matmul(tb.mx_quantize(x[:1], fmt), tb.mx_quantize(w, fmt), torch.float32)

        work.append(step)
        want.append(step())
    torch.cuda.synchronize()
    got = [None] * 4
    for _ in range(5):
        for i, step in enumerate(work):
            with torch.cuda.stream(streams[i]):
                got[i] = step()
    torch.cuda.synchronize()
    for have, expected in zip(got, want):
        for a, b in zip(have, expected):
            assert torch.equal(a, b)
    assert tb.mx_incomplete() == 0


def test_captured_and_replayed():
    """Two graphs of the whole path with their own workspaces, replayed in turn on changing inputs."""
    n, tokens, cols, out = 12, 3, 160, 200

    def make(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        s = {"cache": tb.MxCache.empty(20, tokens, cols, "mxfp4", ragged=True), "index": torch.arange(n, device="cuda"),
             "x": torch.randn(n, tokens, cols, generator=g, device="cuda"), "len": torch.full((n,), 2, dtype=torch.int32, device="cuda"),
             "w": torch.randn(out, cols, generator=g, device="cuda"), "up": torch.randn(n * tokens, out, generator=g, device="cuda")}

        def step():
            s["cache"].write(s["index"], s["x"], lengths=s["len"])
            mx, sizes = s["cache"].read_mx(s["index"])
            w = s["w"].detach().requires_grad_(True)
            y = tb.mx_linear(mx, w, "mxfp4", dtype=torch.float32).view(-1, out)
            (gw,) = torch.autograd.grad(y, [w], s["up"])
            return s["cache"].read(s["index"], torch.float32)[0], sizes, y.detach(), gw

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s["out"] = step()
        return s, step, graph

    made = [make(1), make(2)]
    for round_ in range(3):
        for s, _, _ in made:
            s["x"].mul_(1.7), s["index"].add_(1), s["len"].fill_(round_ + 1), s["w"].mul_(0.9)
        got = []
        for s, _, graph in made:
            graph.replay()
        for s, step, _ in made:
            got = [t.clone() for t in s["out"]]
            for have, want in zip(got, step()):
                assert torch.equal(have, want)


def test_captured_without_a_call_before():
    """In a fresh process: the first call of each kernel is a captured one."""
    import subprocess
    import sys

    code = """if 1:
        import torch, turboloader_b200 as tb
        x, w = torch.randn(300, 256, device="cuda"), torch.randn(64, 256, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a, b = tb.mx_quantize(x), tb.mx_quantize(w)
            y, z, v = tb.mx_matmul(a, b, torch.float32), tb.mx_matmul(tb.mx_quantize(x[:1]), b, torch.float32), a.dequantize()
        graph.replay()
        torch.cuda.synchronize()
        a, b = tb.mx_quantize(x), tb.mx_quantize(w)
        assert torch.equal(y, tb.mx_matmul(a, b, torch.float32)) and torch.equal(v, a.dequantize())
        assert torch.equal(z, tb.mx_matmul(tb.mx_quantize(x[:1]), b, torch.float32)) and tb.mx_incomplete() == 0
    """
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def test_offsets_beyond_32_bits():
    """A cache whose codes pass 4 GiB, and a result of more than 2^31 values: their far ends."""
    slots, tokens, cols = 8200, 256, 4096 + 32
    cache = tb.MxCache(torch.empty(slots, tokens, 2112, dtype=torch.uint8, device="cuda"), torch.empty(slots, tokens, 132, dtype=torch.uint8, device="cuda"),
                       cols, "mxfp4")
    assert cache.codes.numel() == slots * tokens * 2112 > 2 ** 32
    x = torch.randn(2, tokens, cols, device="cuda")
    index = torch.tensor([slots - 1, 0], device="cuda")
    cache.write(index, x)
    codes, scales = encode(_np(x[0]), "mxfp4")
    _same(cache.codes[-1].cpu().numpy(), codes[:, :2112])
    _same(cache.scales[-1].cpu().numpy(), scales[:, :132])
    want = tb.mx_quantize(x, "mxfp4")
    assert torch.equal(cache.read(index, torch.float32), want.dequantize())
    assert torch.equal(cache.read_mx(index).codes.view(-1), want.codes.view(-1))
    del cache
    m, n = 300_001, 8192
    a = tb.mx_quantize(torch.randn(m, 64, device="cuda"), "mxfp4")
    b = tb.mx_quantize(torch.randn(n, 64, device="cuda"), "mxfp4")
    y = tb.mx_matmul(a, b)
    assert y.numel() > 2 ** 31
    tail = tb.MxTensor(a.codes[m - 300:], a.scales[m - 300:], (300, 64), "mxfp4")
    assert torch.equal(y[m - 300:], tb.mx_matmul(tail, b))


def test_feature_loader_serves_what_was_written():
    n, tokens, dim, bs = 50, 5, 96, 8
    x = torch.randn(n, tokens, dim)
    lengths = np.random.default_rng(1).integers(0, tokens + 1, n).astype(np.int32)
    labels = np.arange(n) * 3
    loader = tb.CudaFeatureLoader(n, tokens, dim, bs, format="mxfp8", ragged=True, shuffle=True, seed=7, drop_last=False, labels=labels,
                                  return_indices=True, dtype=torch.float32)
    for i in range(0, n, 16):
        loader.write(np.arange(i, min(n, i + 16)), x[i:i + 16].cuda(), torch.from_numpy(lengths[i:i + 16]).cuda())
    want = decode(*encode(x.view(-1, dim).numpy(), "mxfp8"), "mxfp8", dim).reshape(n, tokens, dim)
    want[np.arange(tokens)[None, :] >= lengths[:, None]] = 0
    loader.set_epoch(3)
    order = np.random.default_rng(7 + 3).permutation(n)
    seen = []
    for b, (batch, sizes, labs, idx) in enumerate(loader):
        at = order[b * bs:(b + 1) * bs]
        seen.extend(idx.tolist())
        assert np.array_equal(idx.cpu().numpy(), at) and np.array_equal(labs.cpu().numpy(), labels[at])
        assert np.array_equal(sizes.cpu().numpy(), lengths[at])
        _equal_values(batch, torch.from_numpy(want[at].astype(np.float32)))
        if b == 3:
            state = loader.state_dict()
    assert len(loader) == 7 and sorted(seen) == list(range(n)) and loader.device_status() == 0
    assert state == {"version": 1, "epoch": 3, "batches_served": 4}
    loader.load_state_dict(state)
    assert [i for *_, idx in loader for i in idx.tolist()] == order[4 * bs:].tolist()
    with pytest.raises(IndexError):
        loader.write([n], x[:1].cuda())


def test_images_to_cached_features_to_a_projector():
    """The whole use: an image loader feeds a frozen encoder, its features fill the cache, and the projector
    trains on microscaled batches."""
    n, side, patch, dim, out = 24, 16, 8, 96, 80
    images = np.random.default_rng(0).integers(0, 256, (n, side, side, 3)).astype(np.uint8)
    source = tb.CudaResidentLoader.from_array(images, 8, shuffle=True, seed=1, return_indices=True)
    weight = torch.randn(dim, 3 * patch * patch, device="cuda") * 0.1

    def encoder(batch):
        p = batch.unfold(2, patch, patch).unfold(3, patch, patch).permute(0, 2, 3, 1, 4, 5).reshape(batch.shape[0], 4, -1)
        return p @ weight.T

    loader = tb.CudaFeatureLoader(n, 4, dim, 8, format="nvfp4", output="mx", shuffle=True, seed=2, return_indices=True)
    assert loader.fill(source, encoder) == n
    with pytest.raises(ValueError):
        loader.fill([images], encoder)
    plain = tb.CudaResidentLoader.from_array(images, n)
    features = encoder(torch.as_tensor(next(iter(plain)), device="cuda"))
    values = torch.from_numpy(decode(*encode(_np(features).reshape(-1, dim), "nvfp4"), "nvfp4", dim)).cuda().view(n, 4, dim)
    got = loader.cache.read(None, torch.float32)
    # the encoder's own sums may differ by a rounding between batch sizes, which can move a code to its neighbour
    assert ((got.double() - values).abs() <= features.abs().amax() / 3).all()
    projector = torch.nn.Parameter(torch.randn(out, dim, device="cuda") * 0.1)
    for mx, idx in loader:
        held = loader.cache.read(idx, torch.float32).double().view(-1, dim)
        y = tb.mx_linear(mx, projector, "nvfp4", dtype=torch.bfloat16)
        assert y.shape == (8, 4, out)
        up = torch.randn_like(y)
        (grad,) = torch.autograd.grad(y, [projector], up)
        u = up.double().view(-1, out)
        _close(grad, u.T @ held, u.abs().T @ held.abs(), 32, torch.float32)
        pv = torch.from_numpy(decode(*encode(_np(projector), "nvfp4"), "nvfp4", dim)).cuda()
        _close(y.detach().view(-1, out), held @ pv.T, held.abs() @ pv.abs().T, dim, torch.bfloat16)


def test_launches_are_counted():
    before = tb.launch_count()
    q = tb.mx_quantize(torch.randn(4, 64, device="cuda"))
    q.dequantize()
    assert tb.launch_count() == before + 2
    assert tb.mx_incomplete() == 0
