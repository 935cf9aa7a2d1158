"""The microscaled operators, measured: quantisation of rows, the feature cache, the product and the linear layer.

Every case is one call path of a program that trains or serves on cached features.  A block of 16 (``nvfp4``) or 32
(``mxfp4``, ``mxfp8``) consecutive values of a row shares one 8-bit scale; the values are e2m1 (4 bits) or e4m3 (8 bits).
``run`` computes the plain form in elementary torch operations, or, with ``own`` set, calls the framework.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BLOCK = {"nvfp4": 16, "mxfp4": 32, "mxfp8": 32}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One feature row quantised on arrival (a pooled embedding): launch latency is what counts.
        {"name": "quantize_row", "op": "quantize", "rows": 1, "cols": 4096, "pitch": 4096, "format": "nvfp4", "dtype": "bf16", "scale": 1.0},
        # A batch of 256 images' token features (14 x 14 patches of 224 x 224), whole.
        {"name": "quantize_batch", "op": "quantize", "rows": 256 * 196, "cols": 1024, "pitch": 1024, "format": "nvfp4", "dtype": "bf16", "scale": 0.03125},
        # A slice of a wider float32 matrix, odd sizes.
        {"name": "quantize_slice", "op": "quantize", "rows": 4099, "cols": 1000, "pitch": 1283, "format": "mxfp4", "dtype": "f32", "scale": 1.0},
        # One pooled feature vector written into a small cache and the cache read back.
        {"name": "cache_one", "op": "cache", "slots": 8, "write": 1, "read": 8, "tokens": 1, "cols": 1024, "format": "mxfp8", "dtype": "bf16", "ragged": False},
        # First epoch of a feature cache: a batch of images of different token counts is written, then a shuffled batch is served.
        {"name": "cache_fill", "op": "cache", "slots": 320, "write": 256, "read": 320, "tokens": 196, "cols": 768, "format": "nvfp4", "dtype": "bf16", "ragged": True},
        # Odd sizes, 16-bit floats, few tokens.
        {"name": "cache_odd", "op": "cache", "slots": 301, "write": 77, "read": 301, "tokens": 33, "cols": 1003, "format": "mxfp8", "dtype": "f16", "ragged": True},
        # Later epochs: only shuffled reads out of a large cache.
        {"name": "cache_serve", "op": "cache", "slots": 4096, "write": 0, "read": 512, "tokens": 256, "cols": 1024, "format": "mxfp4", "dtype": "bf16", "ragged": False},
        # A single token through a quantised weight.
        {"name": "product_token", "op": "product", "m": 1, "n": 4096, "k": 4096, "format": "nvfp4", "dtype": "bf16"},
        # A handful of odd-sized rows.
        {"name": "product_few", "op": "product", "m": 13, "n": 5001, "k": 2000, "format": "mxfp4", "dtype": "f32"},
        # A batch's cached features through the projector of a language model.
        {"name": "product_batch", "op": "product", "m": 256 * 196, "n": 4096, "k": 1024, "format": "nvfp4", "dtype": "bf16"},
        # A training step of the projector on cached (frozen) features: output and the weight's gradient.
        {"name": "linear_frozen", "op": "linear", "m": 64 * 196, "n": 4096, "k": 1024, "format": "nvfp4", "dtype": "bf16", "frozen": True},
        # A layer whose input is trained too, in float32, odd sizes.
        {"name": "linear_live", "op": "linear", "m": 1021, "n": 1000, "k": 1537, "format": "mxfp4", "dtype": "f32", "frozen": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "cache", "product", "linear"])
    fmt = rng.choice(["nvfp4", "mxfp4", "mxfp8"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quantize":
        cols = _log(rng, 33, 4096)
        rows = _log(rng, 1, min(256 * 196, 24_000_000 // cols))
        return {"op": op, "rows": rows, "cols": cols, "pitch": cols + rng.choice([0, 0, 1, 24]), "format": fmt, "dtype": dtype, "scale": 2.0 ** rng.randint(-6, 1)}
    if op == "cache":
        cols = _log(rng, 33, 2048)
        tokens = _log(rng, 1, 256)
        slots = _log(rng, 2, max(2, min(4096, 24_000_000 // (cols * tokens))))
        return {"op": op, "slots": slots, "write": rng.randint(0, slots), "read": rng.randint(1, slots), "tokens": tokens, "cols": cols, "format": fmt, "dtype": dtype, "ragged": rng.random() < 0.5}
    n, k = _log(rng, 48, 4096), _log(rng, 48, 4096)
    if op == "product":
        return {"op": op, "m": _log(rng, 1, min(20_000, 4_000_000_000 // (n * k) * 10 + 1)), "n": n, "k": k, "format": fmt, "dtype": dtype}
    return {"op": op, "m": _log(rng, 16, min(12_000, 2_000_000_000 // (n * k) * 10 + 16)), "n": n, "k": k, "format": fmt, "dtype": dtype, "frozen": rng.random() < 0.5}


# ---- layout: rows padded to 128 values; two 4-bit codes a byte, the even value in the low half ------------------------

def _padded(cols):
    return (cols + 127) // 128 * 128


def _code_bytes(fmt, cols):
    return _padded(cols) if fmt == "mxfp8" else _padded(cols) // 2


# ---- the plain form ----------------------------------------------------------------------------------------------------

def _power_of_two(e):
    """2 ** e exactly, in 64 bits, from the exponent's bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x, fmt, scale):
    """(rows, cols) -> codes (rows, code bytes) and scales (rows, blocks of the padded row), both uint8."""
    rows, cols = x.shape
    t = x.float() / scale
    t = torch.nn.functional.pad(t, (0, _padded(cols) - cols)).view(rows, -1, _BLOCK[fmt])
    a = t.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(t).all(-1, keepdim=True)
    t = torch.where(bad, torch.zeros_like(t), t)
    a = torch.where(bad, torch.zeros_like(a), a)
    if fmt == "nvfp4":
        s8 = (a / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
        byte = s8.view(torch.uint8)
        s = s8.float()
        r = torch.where(s > 0, t / s, torch.zeros_like(t))
    else:
        e = (torch.frexp(a)[1].int() - 1 - (2 if fmt == "mxfp4" else 8)).clamp(min=-127)
        e = torch.where(a > 0, e, torch.full_like(e, -127))
        byte = (e + 127).to(torch.uint8)
        r = (t.double() * _power_of_two(-e)).float()
    byte = torch.where(bad, torch.full_like(byte, 0x7F if fmt == "nvfp4" else 0xFF), byte).squeeze(-1)
    if fmt == "mxfp8":
        codes = r.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8).view(rows, -1)
    else:
        m = r.abs()
        c = (m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
        c = (c | (torch.signbit(r).to(torch.uint8) << 3)).view(rows, -1, 2)
        codes = c[..., 0] | (c[..., 1] << 4)
    return codes.contiguous(), byte.contiguous()


def _decode(codes, scales, fmt, cols):
    """Codes times block scales, float32, without the tensor's scale; leading dimensions as given."""
    if fmt == "mxfp8":
        c = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float32, device=codes.device)
        c = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], dim=-1).flatten(-2)
    if fmt == "nvfp4":
        s = scales.view(torch.float8_e4m3fn).float()
    else:
        s = _power_of_two(scales.int() - 127).float()
        s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (c.unflatten(-1, (-1, _BLOCK[fmt])) * s.unsqueeze(-1)).flatten(-2)[..., :cols]


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _features(g, rows, cols, dtype, spread=2.0):
    """Encoder features: near normal, each column with a strength of its own."""
    strength = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda")) * spread
    x = torch.empty((rows, cols), dtype=dtype, device="cuda")
    step = max(1, 32_000_000 // cols)
    for i in range(0, rows, step):
        x[i:i + step] = (torch.randn((min(step, rows - i), cols), generator=g, device="cuda") * strength).to(dtype)
    return x


def _encoded(g, rows, cols, fmt, spread=2.0):
    codes = torch.empty((rows, _code_bytes(fmt, cols)), dtype=torch.uint8, device="cuda")
    scales = torch.empty((rows, _padded(cols) // _BLOCK[fmt]), dtype=torch.uint8, device="cuda")
    step = max(1, 32_000_000 // cols)
    for i in range(0, rows, step):
        codes[i:i + step], scales[i:i + step] = _encode(_features(g, min(step, rows - i), cols, torch.float32, spread), fmt, 1.0)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    s = dict(case, dt=dtype)
    if case["op"] == "quantize":
        s["x"] = _features(g, case["rows"], case["pitch"], dtype)[:, :case["cols"]]
    elif case["op"] == "cache":
        slots, tokens, cols = case["slots"], case["tokens"], case["cols"]
        codes, scales = _encoded(g, slots * tokens, cols, case["format"])
        s["codes"], s["scales"] = codes.view(slots, tokens, -1), scales.view(slots, tokens, -1)
        s["lengths"] = torch.randint(0, tokens + 1, (slots,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        order = torch.randperm(slots, generator=g, device="cuda")
        s["put"] = order[:case["write"]].contiguous()
        s["put_lengths"] = torch.randint(0, tokens + 1, (case["write"],), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        s["x"] = _features(g, case["write"] * tokens, cols, dtype).view(case["write"], tokens, cols)
        s["get"] = torch.randperm(slots, generator=g, device="cuda")[:case["read"]].contiguous()
    elif case["op"] == "product":
        s["a"] = _encoded(g, case["m"], case["k"], case["format"])
        s["b"] = _encoded(g, case["n"], case["k"], case["format"], case["k"] ** -0.5)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["w"] = _features(g, n, k, dtype, k ** -0.5).requires_grad_(True)
        s["x"] = _encoded(g, m, k, case["format"]) if case["frozen"] else _features(g, m, k, dtype).requires_grad_(True)
        s["g"] = (torch.randn((m, n), generator=g, device="cuda") / m).to(dtype) * (64 if dtype == torch.float16 else 1)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def _run_plain(s):
    fmt, dt = s["format"], s["dt"]
    if s["op"] == "quantize":
        codes, scales = _encode(s["x"], fmt, s["scale"])
        return (_decode(codes, scales, fmt, s["cols"]) * s["scale"]).to(dt)
    if s["op"] == "cache":
        tokens, cols = s["tokens"], s["cols"]
        row = torch.arange(tokens, device="cuda")
        if s["write"]:
            codes, scales = _encode(s["x"].reshape(-1, cols), fmt, 1.0)
            slot = (s["put"][:, None] * tokens + row).reshape(-1)
            if s["put_lengths"] is not None:
                s["lengths"][s["put"]] = s["put_lengths"]
                fits = (row < s["put_lengths"][:, None]).reshape(-1)
                codes, scales, slot = codes[fits], scales[fits], slot[fits]
            s["codes"].view(-1, codes.shape[-1])[slot] = codes
            s["scales"].view(-1, scales.shape[-1])[slot] = scales
        v = _decode(s["codes"][s["get"]], s["scales"][s["get"]], fmt, cols)
        if s["lengths"] is None:
            return v.to(dt)
        lengths = s["lengths"][s["get"]]
        return torch.where((row < lengths[:, None])[..., None], v, torch.zeros_like(v)).to(dt), lengths
    if s["op"] == "product":
        return (_decode(*s["a"], fmt, s["k"]) @ _decode(*s["b"], fmt, s["k"]).T).to(dt)
    x = _decode(*(s["x"] if s["frozen"] else _encode(s["x"].detach(), fmt, 1.0)), fmt, s["k"])
    w = _decode(*_encode(s["w"].detach(), fmt, 1.0), fmt, s["k"])
    g = s["g"].float()
    out = [(x @ w.T).to(dt), (g.T @ x).to(dt)]
    return out if s["frozen"] else out + [(g @ w).to(dt)]


def _run_own(s):
    import turboloader_b200 as tb

    fmt, dt = s["format"], s["dt"]
    if s["op"] == "quantize":
        return tb.mx_dequantize(tb.mx_quantize(s["x"], fmt, scale=s["scale"]), dt)
    if s["op"] == "cache":
        cache = tb.MxCache(s["codes"], s["scales"], s["cols"], fmt, lengths=s["lengths"])
        if s["write"]:
            cache.write(s["put"], s["x"], lengths=s["put_lengths"])
        return cache.read(s["get"], dt)
    if s["op"] == "product":
        a = tb.MxTensor(*s["a"], (s["m"], s["k"]), fmt)
        b = tb.MxTensor(*s["b"], (s["n"], s["k"]), fmt)
        return tb.mx_matmul(a, b, dt)
    x = tb.MxTensor(*s["x"], (s["m"], s["k"]), fmt) if s["frozen"] else s["x"]
    y = tb.mx_linear(x, s["w"], fmt, dtype=dt)
    return [y.detach(), *torch.autograd.grad(y, [s["w"]] if s["frozen"] else [s["w"], s["x"]], s["g"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    e = _DTYPES[case["dtype"]].itemsize

    def held(rows, cols):
        return rows * (cols * (1.0 if case["format"] == "mxfp8" else 0.5) + -(-cols // _BLOCK[case["format"]]))

    if case["op"] == "quantize":  # values in, codes and scales out, values back
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * e + held(case["rows"], case["cols"]), "flops": 8 * n}
    if case["op"] == "cache":  # ragged: lengths are uniform, half of the rows are there on average
        part = 0.5 if case["ragged"] else 1.0
        put, get, cols = case["write"] * case["tokens"], case["read"] * case["tokens"], case["cols"]
        return {"bytes": part * (put * cols * e + held(put, cols) + held(get, cols)) + get * cols * e, "flops": 6 * part * put * cols + 2 * part * get * cols}
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "product":
        return {"bytes": held(m, k) + held(n, k) + m * n * e, "flops": 2.0 * m * n * k}
    live = not case["frozen"]
    inputs = (m * k * e if live else held(m, k)) + n * k * e + m * n * e
    return {"bytes": inputs + m * n * e + n * k * e + (m * k * e if live else 0), "flops": 2.0 * m * n * k * (3 if live else 2)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------

def _nearest(v, grid):
    """The nearest grid point (ascending grid; ties to the point of even place) of every |v|."""
    at = torch.searchsorted(grid, v.contiguous()).clamp(1, len(grid) - 1)
    lo, hi = grid[at - 1], grid[at]
    up = (v - lo > hi - v) | ((v - lo == hi - v) & (at % 2 == 0))
    return torch.where(up, hi, lo)


def _grid_e4m3():
    points = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(points[:-1], dtype=torch.float64, device="cuda")  # the last one is NaN's


def _rounded(x, fmt, scale):
    """What the quantised rows stand for, in 64 bits."""
    out = []
    small, wide = torch.tensor(_E2M1, dtype=torch.float64, device="cuda"), _grid_e4m3()
    step = max(1, 16_000_000 // x.shape[1])
    for i in range(0, x.shape[0], step):
        t = x[i:i + step].detach().double() / scale
        rows, cols = t.shape
        t = torch.nn.functional.pad(t, (0, -cols % _BLOCK[fmt])).view(rows, -1, _BLOCK[fmt])
        a = t.abs().amax(-1, keepdim=True)
        if fmt == "nvfp4":
            s = _nearest((a / 6).clamp(max=448.0), wide)
        else:
            powers = torch.tensor([2.0 ** i for i in range(-127, 130)], dtype=torch.float64, device="cuda")
            below = (torch.searchsorted(powers, a, right=True) - 1).clamp(min=0)  # the largest power of two up to a
            s = powers[(below - (2 if fmt == "mxfp4" else 8)).clamp(min=0)]
        top, grid = (448.0, wide) if fmt == "mxfp8" else (6.0, small)
        r = torch.where(s > 0, t.abs() / s.clamp(min=2.0 ** -150), torch.zeros_like(t)).clamp(max=top)
        out.append((torch.copysign(_nearest(r, grid), t) * s * scale).reshape(rows, -1)[:, :cols])
    return torch.cat(out)


def _stands(held, fmt, cols):
    codes, scales = held
    byte = torch.arange(256, device="cuda")
    small, wide = torch.tensor(_E2M1, dtype=torch.float64, device="cuda"), torch.cat([_grid_e4m3(), torch.full((1,), math.nan, dtype=torch.float64, device="cuda")])
    e4m3 = torch.where(byte < 128, wide[byte & 127], -wide[byte & 127])
    s = (e4m3 if fmt == "nvfp4" else torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan], dtype=torch.float64, device="cuda"))[scales.long()]
    if fmt == "mxfp8":
        c = e4m3[codes.long()]
    else:
        sign = torch.where(byte[:16] < 8, 1.0, -1.0).double() * small[byte[:16] & 7]
        c = torch.stack([sign[(codes % 16).long()], sign[(codes // 16).long()]], -1)
    return (c.view(codes.shape[0], -1, _BLOCK[fmt]) * s[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    fmt = case["format"]
    if case["op"] == "quantize":
        return _rounded(s["x"], fmt, case["scale"])
    if case["op"] == "cache":
        tokens, cols = case["tokens"], case["cols"]
        place = {int(p): i for i, p in enumerate(s["put"].tolist())}
        lengths = s["lengths"].tolist() if case["ragged"] else None
        new = s["put_lengths"].tolist() if case["ragged"] else [tokens] * case["write"]
        fresh = _rounded(s["x"].reshape(-1, cols), fmt, 1.0).view(-1, tokens, cols) if case["write"] else None
        got, sizes = torch.zeros((case["read"], tokens, cols), dtype=torch.float64, device="cuda"), []
        for j, p in enumerate(s["get"].tolist()):
            here = place.get(p)
            size = new[here] if here is not None else (lengths[p] if lengths else tokens)
            if size:
                got[j, :size] = fresh[here, :size] if here is not None else _stands((s["codes"][p, :size], s["scales"][p, :size]), fmt, cols)
            sizes.append(size)
        return (got, None) if case["ragged"] else got
    if case["op"] == "product":
        return _stands(s["a"], fmt, case["k"]) @ _stands(s["b"], fmt, case["k"]).T
    x = _stands(s["x"], fmt, case["k"]) if case["frozen"] else _rounded(s["x"], fmt, 1.0)
    w = _rounded(s["w"], fmt, 1.0)
    g = s["g"].double()
    out = [x @ w.T, g.T @ x]
    return out if case["frozen"] else out + [g @ w]
