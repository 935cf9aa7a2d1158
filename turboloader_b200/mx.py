"""Microscaled rows: quantisation of features to 4 or 8 bits, a cache that holds them, and the products on them.

A feature set -- the token outputs of a frozen image encoder -- is many times larger than the images it came
from.  Here it stays resident in HBM at 4.5 (``nvfp4``), 4.25 (``mxfp4``) or 8.25 (``mxfp8``) bits a value, is
written sample by sample, served in shuffled order, and goes through the next model's first linear layer without
being widened first.  The formats, the layout of the rows and the rules for special values stand in
``include/turboloader_b200.h`` ("microscaled rows").  torch allocates memory and names the current stream; every
computation happens inside the C-ABI library, on the current stream (or ``stream``), without synchronisation, so
all of it can be captured into CUDA graphs.  With ``stream``, what a call allocates belongs to that stream, and
ordering it behind the work that makes the inputs (and before what reads the results) is the caller's, as with
any torch call under ``torch.cuda.stream``.

No counterpart in the reference, whose resident loader keeps uint8 pixels (turboloader/cuda_loader.py:385-535).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math

import torch

from . import _capi

__all__ = ["MxTensor", "MxCache", "mx_quantize", "mx_dequantize", "mx_matmul", "mx_linear", "mx_incomplete"]

_FORMATS = {"nvfp4": 0, "mxfp4": 1, "mxfp8": 2}
_BLOCK = (16, 32, 32)
_raw_stream = torch._C._cuda_getCurrentRawStream  # the handle alone: a Stream object costs 3 us a call
_DTYPES = {torch.float32: _capi.TLB_F32, torch.bfloat16: _capi.TLB_BF16, torch.float16: _capi.TLB_F16}


def _format_id(format):
    try:
        return _FORMATS[format]
    except (KeyError, TypeError):
        raise ValueError(f"format must be one of {tuple(_FORMATS)}, got {format!r}") from None


def _dtype_id(dtype, what):
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {dtype}") from None


def _pitches(fmt, cols):
    if not 1 <= cols <= _capi.MX_MAX_COLS:
        raise ValueError(f"rows must have between 1 and {_capi.MX_MAX_COLS} values, got {cols}")
    padded = (cols + 127) // 128 * 128
    return (padded if fmt == 2 else padded // 2), padded // _BLOCK[fmt]


def _cuda(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{what} must be a CUDA tensor")
    return t


def _table(t, dtype, n, device, what):
    """A contiguous 1-D device table of ``n`` entries."""
    _cuda(t, what)
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise TypeError(f"{what} must be a contiguous 1-D {dtype} tensor")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{what} must have {n} entries, got {t.shape[0]}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")
    return t


def _check_scale(scale, device):
    if type(scale) is float and 0.0 < scale < float("inf"):
        return scale
    if isinstance(scale, torch.Tensor):
        if scale.device != device or scale.dtype != torch.float32 or scale.numel() != 1:
            raise TypeError(f"a scale tensor must be one float32 value on {device}")
        return scale.detach()
    scale = float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    return scale


def _own(scale):
    """A scale that the caller cannot change any more: what the rows stand for depends on it as long as they live."""
    return scale.clone() if isinstance(scale, torch.Tensor) else scale


def _away(device, stream):
    """Whether a call for tensors of ``device`` has to change the current device or stream first."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("the microscaled operators cannot be traced: torch would record the memory they allocate, not what their kernels write")
    return stream is not None or torch.cuda.current_device() != device.index


@contextlib.contextmanager
def _there(device, stream):
    """Makes ``device``, and ``stream`` where one is named, the current ones: what a call allocates then belongs to the
    stream that uses it."""
    if stream is not None and stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
    with torch.cuda.device(device):
        if stream is None:
            yield
        else:
            with torch.cuda.stream(stream):
                yield


def _rows_struct(codes, scales, rows, cols, fmt, scale):
    """tlb_mx_rows of two addresses."""
    if isinstance(scale, torch.Tensor):
        return _capi.MxRows(codes, scales, rows, cols, fmt, 1.0, scale.data_ptr())
    return _capi.MxRows(codes, scales, rows, cols, fmt, scale, None)


def _check_held(codes, scales, rows, cols, fmt):
    """codes (..., code pitch) and scales (..., scale pitch): uint8, contiguous, `rows` rows in all."""
    cp, sp = _pitches(fmt, cols)
    if (isinstance(codes, torch.Tensor) and isinstance(scales, torch.Tensor) and codes.is_cuda and codes.dtype is torch.uint8
            and scales.dtype is torch.uint8 and codes.dim() and scales.dim() and codes.size(-1) == cp and scales.size(-1) == sp
            and codes.numel() == rows * cp and scales.numel() == rows * sp and codes.get_device() == scales.get_device()
            and codes.is_contiguous() and scales.is_contiguous() and not codes.data_ptr() % 16 and not scales.data_ptr() % 4):
        return
    for t, pitch, what in ((codes, cp, "codes"), (scales, sp, "scales")):  # what is wrong
        _cuda(t, what)
        if t.dtype is not torch.uint8 or not t.is_contiguous() or t.dim() < 1 or t.shape[-1] != pitch:
            raise ValueError(f"{what} must be a contiguous uint8 tensor with rows of {pitch} bytes")
        if t.numel() != rows * pitch:
            raise ValueError(f"{what} must hold {rows} rows, got {t.numel() // pitch}")
    if codes.get_device() != scales.get_device():
        raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")
    if codes.data_ptr() % 16 or scales.data_ptr() % 4:
        raise ValueError("codes must be 16-byte and scales 4-byte aligned")


class MxTensor:
    """Microscaled rows: ``codes`` and ``scales`` (uint8 CUDA tensors, rows padded to 128 values as the C header
    says) standing for values of ``shape`` (the last dimension is the rows' length), times ``scale`` -- a float,
    or one float32 value on the device.  Holds the tensors it is given, without a copy."""

    __slots__ = ("shape", "format", "scale", "device", "_codes", "_scales", "_buf", "_lead", "_fmt", "_rows")

    def __init__(self, codes, scales, shape, format, *, scale=1.0):
        self._fmt = fmt = _format_id(format)
        self.shape = shape = tuple(shape)
        if not shape:
            raise ValueError("an MxTensor has at least one dimension")
        self._rows = rows = math.prod(shape[:-1])
        _check_held(codes, scales, rows, shape[-1], fmt)
        self._codes, self._scales, self.format, self.device, self._buf = codes, scales, format, codes.device, None
        self.scale = _check_scale(scale, self.device)

    @classmethod
    def _empty(cls, shape, lead, format, fmt, scale, device):
        """Room for rows of ``shape``, codes and then scales in one buffer; their tensors, with leading dimensions
        ``lead``, are made when they are asked for."""
        self = object.__new__(cls)
        rows = math.prod(lead)
        cp, sp = _pitches(fmt, shape[-1])
        self._buf = torch.empty(rows * (cp + sp), dtype=torch.uint8, device=device)
        self._codes = self._scales = None
        self.shape, self._lead, self._rows, self.format, self._fmt, self.scale, self.device = shape, lead, rows, format, fmt, scale, device
        return self

    def _views(self):
        cp, sp = _pitches(self._fmt, self.shape[-1])
        at = self._rows * cp
        self._codes, self._scales = self._buf[:at].view(*self._lead, cp), self._buf[at:].view(*self._lead, sp)

    @property
    def codes(self):
        if self._codes is None:
            self._views()
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            self._views()
        return self._scales

    def _at(self):
        """Addresses of codes and scales."""
        if self._buf is not None:
            base = self._buf.data_ptr()
            return base, base + self._rows * _pitches(self._fmt, self.shape[-1])[0]
        return self._codes.data_ptr(), self._scales.data_ptr()

    def _tensors(self):
        """What keeps the rows alive."""
        return [self._buf] if self._buf is not None else [self._codes, self._scales]

    def _struct(self):
        return _rows_struct(*self._at(), self._rows, self.shape[-1], self._fmt, self.scale)

    def dequantize(self, dtype=torch.float32):
        return mx_dequantize(self, dtype)

    def __repr__(self):
        return f"MxTensor(shape={self.shape}, format={self.format!r}, device={self.device})"


def _as_rows(x, what):
    """(rows, cols, row pitch) of (..., cols) values whose rows lie at equal distances."""
    _cuda(x, what)
    if x.dim() < 1:
        raise ValueError(f"{what} must have at least one dimension")
    cols = x.shape[-1]
    if x.stride(-1) != 1 and cols != 1:
        raise ValueError(f"the values of a row of {what} must be contiguous")
    if x.dim() == 2:
        rows, pitch = x.shape[0], x.stride(0)
    elif x.dim() == 1:
        rows, pitch = 1, cols
    else:
        try:
            flat = x.detach().view(-1, cols) if x.numel() else x.detach().reshape(-1, cols)
        except RuntimeError:
            raise ValueError(f"the rows of {what} must lie at equal distances") from None
        rows, pitch = flat.shape[0], flat.stride(0)
    if rows > 1 and pitch < cols:
        raise ValueError(f"the rows of {what} overlap (pitch {pitch}, {cols} values)")
    return rows, cols, pitch


def mx_quantize(x, format="nvfp4", *, scale=1.0, stream=None):
    """``x`` (..., cols), float32, bfloat16 or float16, as an ``MxTensor``.  The values of a row must be
    contiguous and the rows equally spaced (a slice of a wider matrix will do).  ``scale``: the tensor scale
    that values are divided by first, a float or one float32 value on the device (copied: the result keeps the
    value of this call); a power of two loses nothing.  For ``nvfp4``, ``max|x| / 2688`` rounded up to a power of
    two uses the range of its scales."""
    fmt = _format_id(format)
    rows, _, pitch = _as_rows(x, "x")
    dt = _dtype_id(x.dtype, "x")
    device = x.device
    scale = _check_scale(scale, device)
    if _away(device, stream):
        with _there(device, stream):
            return mx_quantize(x, format, scale=scale)
    q = MxTensor._empty(tuple(x.shape), (rows,), format, fmt, _own(scale), device)
    _capi.check(_capi.load().tlb_mx_quantize(q._struct(), x.data_ptr(), dt, pitch, _raw_stream(device.index)))
    return q


def _out(out, shape, dtype, device):
    if out is None:
        return torch.empty(*shape, dtype=dtype, device=device)  # sizes one by one parse faster than a tuple
    _cuda(out, "out")
    if out.dtype != dtype or tuple(out.shape) != tuple(shape) or not out.is_contiguous() or out.device != device:
        raise ValueError(f"out must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    if out.data_ptr() % 16:
        raise ValueError("out must be 16-byte aligned")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out must not require gradients")
    torch.autograd.graph.increment_version(out)  # torch does not see the kernel's writes; a graph that saved it has to
    return out


def mx_dequantize(q, dtype=torch.float32, *, out=None, stream=None):
    """The values that ``q`` stands for: code * block scale * tensor scale in fp32, rounded once to ``dtype``."""
    dt = _dtype_id(dtype, "dtype")
    device = q.device
    if _away(device, stream):
        with _there(device, stream):
            return mx_dequantize(q, dtype, out=out)
    out = _out(out, q.shape, dtype, device)
    cache = _capi.MxCache(q._struct(), 1, None, None, None)
    _capi.check(_capi.load().tlb_mx_read(cache, None, q._rows, out.data_ptr(), dt, None, _raw_stream(device.index)))
    return out


def _check_pair(a, b):
    if not isinstance(a, MxTensor) or not isinstance(b, MxTensor):
        raise TypeError("a and b must be MxTensors")
    if a._fmt != b._fmt:
        raise ValueError(f"a is {a.format}, b is {b.format}")
    if len(b.shape) != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError(f"shapes {a.shape} and {b.shape} do not multiply: b must be (n, {a.shape[-1]})")
    if a.device != b.device:
        raise ValueError(f"a is on {a.device}, b on {b.device}")


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size > 0 else None


def mx_matmul(a, b, dtype=torch.bfloat16, *, out=None, stream=None):
    """``a`` (..., k) times the transpose of ``b`` (n, k), two ``MxTensor`` of one format: (..., n) of ``dtype``.
    The products of the codes enter whole and are summed in fp32; the result is rounded once."""
    _check_pair(a, b)
    dt = _dtype_id(dtype, "dtype")
    device = a.device
    if _away(device, stream):
        with _there(device, stream):
            return mx_matmul(a, b, dtype, out=out)
    lib = _capi.load()
    out = _out(out, (*a.shape[:-1], b.shape[0]), dtype, device)
    sa, sb = a._struct(), b._struct()
    size = lib.tlb_mx_matmul_workspace(sa, sb, dt)
    ws = _workspace(size, device)
    _capi.check(lib.tlb_mx_matmul(sa, sb, out.data_ptr(), dt, None if ws is None else ws.data_ptr(), size, _raw_stream(device.index)))
    return out


def mx_incomplete() -> int:
    """Products and gradients on the current device whose kernels gave up a bounded wait and left NaN where they had not
    summed, since the library was loaded (synchronises): 0 in a healthy process."""
    count = C.c_uint32(0)
    _capi.check(_capi.load().tlb_mx_incomplete(C.byref(count)))
    return int(count.value)


def _grads(g, a, b, cols, a_dtype, b_dtype):
    """(grad_a, grad_b) of values(a) @ values(b).T for g (m, n); a, b: tlb_mx_rows, needed for the other one's
    gradient; a dtype of None: not wanted."""
    device = g.device
    if _away(device, None):
        with _there(device, None):
            return _grads(g, a, b, cols, a_dtype, b_dtype)
    lib = _capi.load()
    m, n = g.shape
    gt = _DTYPES[g.dtype]
    ga = None if a_dtype is None else torch.empty(m, cols, dtype=a_dtype, device=device)
    gb = None if b_dtype is None else torch.empty(n, cols, dtype=b_dtype, device=device)
    # an empty tensor has no address; any other one says that its gradient is wanted
    at = (a, b, None if ga is None else ga.data_ptr() or 16, _DTYPES.get(a_dtype, 0), None if gb is None else gb.data_ptr() or 16,
          _DTYPES.get(b_dtype, 0))
    size = lib.tlb_mx_grad_workspace(gt, m, n, *at)
    ws = _workspace(size, device)
    _capi.check(lib.tlb_mx_grad(g.data_ptr(), gt, m, n, *at, None if ws is None else ws.data_ptr(), size, _raw_stream(device.index)))
    return ga, gb


def _spaced(x):
    """``x`` as rows that can be quantised, and their number and pitch; a copy only where its strides demand one."""
    try:
        rows, _, pitch = _as_rows(x, "x")
    except ValueError:
        x = x.contiguous()
        rows, _, pitch = _as_rows(x, "x")
    return x, rows, pitch


def _align(n):
    return (n + 255) & ~255


def _linear(x, weight, held_x, held_w, fmt, scale, weight_scale, dtype, kept=(False, False)):
    """The product of mx_linear, and where its operands' rows lie: (out, buffer of the kept ones quantised here or None,
    for each operand (held one or None, offsets of codes and scales in its buffer, rows, scale)).  kept: whether the
    operand's rows are needed after this call; the others' memory is given back at its end."""
    lib = _capi.load()
    device = (held_x if x is None else x).device
    shape = held_x.shape if x is None else x.shape
    cols = shape[-1]
    cp, sp = _pitches(fmt, cols)
    at, given, plans = [0, 0], [], []  # sizes of the two buffers: of rows that end with the call, of kept ones
    for t, q, s, keep in ((x, held_x, scale, kept[0]), (weight, held_w, weight_scale, kept[1])):
        if t is None:
            given += None, 0, 0
            plans.append((q, 0, 0, q._rows, q.scale))
            continue
        t, rows, pitch = _spaced(t)
        codes, scales = at[keep], at[keep] + _align(rows * cp)
        at[keep] = scales + _align(rows * sp)
        given += t, _DTYPES[t.dtype], pitch
        s = _check_scale(s, device)
        plans.append((None, codes, scales, rows, _own(s) if keep else s))
    xt, xd, xp, wt, wd, wp = given
    dt = _DTYPES[dtype]
    bufs = [torch.empty(size, dtype=torch.uint8, device=device) if size else None for size in at]
    bases = [0 if buf is None else buf.data_ptr() for buf in bufs]
    a, b = [q._struct() if q is not None else _rows_struct(bases[keep] + c, bases[keep] + s, rows, cols, fmt, ts)
            for (q, c, s, rows, ts), keep in zip(plans, kept)]
    out = torch.empty(*shape[:-1], plans[1][3], dtype=dtype, device=device)
    size = lib.tlb_mx_matmul_workspace(a, b, dt)
    ws = _workspace(size, device)
    _capi.check(lib.tlb_mx_linear(a, None if xt is None else xt.data_ptr(), xd, xp, b, None if wt is None else wt.data_ptr(), wd, wp,
                                  out.data_ptr(), dt, None if ws is None else ws.data_ptr(), size, _raw_stream(device.index)))
    return out, bufs[True], plans


class _MxLinear(torch.autograd.Function):
    """`ctx.parts`: where the operands' rows lie that the backward pass needs, as (0, offsets of codes and scales in the
    first saved tensor, rows, scale); of a held operand the first number counts its saved tensors of rows, and a scale of
    None is the saved tensor behind them."""

    @staticmethod
    def forward(ctx, x, weight, held_x, held_w, fmt, scale, weight_scale, dtype):
        needs_x, needs_w = ctx.needs_input_grad[:2]
        out, buf, plans = _linear(x, weight, held_x, held_w, fmt, scale, weight_scale, dtype, (needs_w, needs_x))
        keep, parts = [] if buf is None else [buf], []
        for (q, c, s, rows, ts), needed in zip(plans, (needs_w, needs_x)):  # the gradient of one needs the other's codes
            count = 0
            if q is not None and needed:
                keep += q._tensors()
                count = len(q._tensors())
                if isinstance(ts, torch.Tensor):
                    keep.append(ts)
                    ts = None
            parts.append((count, c, s, rows, ts) if needed else None)
        ctx.save_for_backward(*keep)
        ctx.parts = parts
        ctx.one = buf is not None
        ctx.fmt, ctx.x_shape = fmt, held_x.shape if x is None else x.shape
        ctx.types = (x.dtype if needs_x else None, weight.dtype if needs_w else None)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        saved = ctx.saved_tensors  # held to the end: under hooks and checkpoints nothing else keeps the rows alive
        left = iter(saved)
        base = next(left).data_ptr() if ctx.one else 0
        cols = ctx.x_shape[-1]
        ops = []
        for part in ctx.parts:
            if part is None:
                ops.append(None)
                continue
            count, c, s, rows, ts = part
            if count == 0:
                c, s = base + c, base + s
            else:  # a held operand: one buffer, or its codes and its scales
                c = next(left).data_ptr()
                s = next(left).data_ptr() if count == 2 else c + rows * _pitches(ctx.fmt, cols)[0]
                ts = next(left) if ts is None else ts
            ops.append(_rows_struct(c, s, rows, cols, ctx.fmt, ts))
        if g.dim() != 2 or not g.is_contiguous():
            g = g.reshape(math.prod(ctx.x_shape[:-1]), g.shape[-1]).contiguous()
        if g.data_ptr() % 16:
            g = g.clone()
        gx, gw = _grads(g, *ops, cols, *ctx.types)
        return None if gx is None else gx.view(ctx.x_shape), gw, None, None, None, None, None, None


def mx_linear(x, weight, format="nvfp4", *, scale=1.0, weight_scale=1.0, dtype=None):
    """``x @ weight.T`` on microscaled operands, differentiable: (..., k), (n, k) -> (..., n) of ``dtype``.

    ``x`` and ``weight`` are float tensors, quantised to ``format`` by this call (``scale`` and ``weight_scale``
    are their tensor scales), or ``MxTensor`` of that format, used as they are (cached features, a frozen weight).
    Gradients flow to the float tensors, straight through their quantisation: ``dx = g @ values(weight)`` and
    ``dweight = g.T @ values(x)``, with every value of g entering whole (down to 2^-133), sums in fp32, in the operand's own type;
    for the backward pass only the codes are kept, and the tensor scales as they were.  An ``MxTensor`` and its scale
    must stay unchanged until then.  Forward-mode tangents and tracing are refused.  ``dtype`` (the result's): by default
    ``weight``'s, else ``x``'s, else bfloat16."""
    fmt = _format_id(format)
    held_x, held_w = (t if isinstance(t, MxTensor) else None for t in (x, weight))
    for t, held, what in ((x, held_x, "x"), (weight, held_w, "weight")):
        if held is not None:
            if held._fmt != fmt:
                raise ValueError(f"{what} is {held.format}, not {format}")
        else:
            _dtype_id(_cuda(t, what).dtype, what)
            if t.dim() < 1:
                raise ValueError(f"{what} must have at least one dimension")
    if len(weight.shape) != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"shapes {tuple(x.shape)} and {tuple(weight.shape)} do not multiply: weight must be (n, {x.shape[-1]})")
    device = x.device
    if device != weight.device:
        raise ValueError(f"x is on {device}, weight on {weight.device}")
    if dtype is None:
        dtype = weight.dtype if held_w is None else x.dtype if held_x is None else torch.bfloat16
    _dtype_id(dtype, "dtype")
    if _away(device, None):
        with _there(device, None):
            return mx_linear(x, weight, format, scale=scale, weight_scale=weight_scale, dtype=dtype)
    args = (None if held_x is not None else x, None if held_w is not None else weight, held_x, held_w, fmt, scale, weight_scale, dtype)
    # within forward-mode differentiation too: autograd then refuses a tangent instead of dropping it
    if torch.autograd.forward_ad._current_level >= 0 or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:2]):
        return _MxLinear.apply(*args)
    return _linear(*args)[0]


class MxCache:
    """Samples of ``tokens`` rows of ``cols`` values, held as microscaled rows: ``codes`` (slots, tokens, code
    pitch) and ``scales`` (slots, tokens, scale pitch), and for samples of different lengths ``lengths`` (slots,)
    int32.  Wraps the tensors it is given; ``MxCache.empty`` makes them.

    ``status``: one int32 value on the device that the kernels OR their TLB_DEV_* bits into (``empty`` gives one)."""

    def __init__(self, codes, scales, cols, format, *, lengths=None, scale=1.0, status=None):
        self._fmt = _format_id(format)
        self._owners = {}
        _cuda(codes, "codes")
        if codes.dim() != 3:
            raise ValueError("codes must be (slots, tokens, code pitch)")
        self.slots, self.tokens, self.cols, self.format = int(codes.shape[0]), int(codes.shape[1]), int(cols), format
        if self.tokens < 1:
            raise ValueError("a cache needs at least one row a sample")
        _check_held(codes, scales, self.slots * self.tokens, self.cols, self._fmt)
        self.codes, self.scales, self.device = codes, scales, codes.device
        self.lengths = None if lengths is None else _table(lengths, torch.int32, self.slots, codes.device, "lengths")
        self.scale = _check_scale(scale, codes.device)
        self.status = None if status is None else _table(status, torch.int32, 1, codes.device, "status")

    @classmethod
    def empty(cls, slots, tokens, cols, format="nvfp4", *, ragged=False, scale=1.0, device=None):
        """A cache of zero rows (``ragged``: of samples of length zero)."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        cp, sp = _pitches(_format_id(format), int(cols))
        return cls(torch.zeros((int(slots), int(tokens), cp), dtype=torch.uint8, device=device),
                   torch.zeros((int(slots), int(tokens), sp), dtype=torch.uint8, device=device), cols, format,
                   lengths=torch.zeros(int(slots), dtype=torch.int32, device=device) if ragged else None, scale=scale,
                   status=torch.zeros(1, dtype=torch.int32, device=device))

    def device_status(self) -> int:
        """Status bits the kernels OR-ed so far (synchronises); 0 when every index and length was valid."""
        return 0 if self.status is None else int(self.status.item())

    def _struct(self, owner=None):
        rows = _rows_struct(self.codes.data_ptr(), self.scales.data_ptr(), self.slots * self.tokens, self.cols, self._fmt, self.scale)
        return _capi.MxCache(rows, self.tokens, None if self.lengths is None else self.lengths.data_ptr(),
                             None if owner is None else owner.data_ptr(), None if self.status is None else self.status.data_ptr())

    def write(self, index, x, *, lengths=None, stream=None):
        """Quantises sample ``x[i]`` (tokens, cols) into slot ``index[i]`` (int64 CUDA tensor).  With ``lengths``
        (int32, for a cache that has lengths) only the first ``lengths[i]`` rows are read and written; the slot's
        other rows stay as they were.  Without, all rows are there.  A slot named twice takes the last of its
        samples; an index outside the cache is skipped and reported in ``status``.  Writes that overlap in time (on
        several streams) must not name the same slot."""
        device = self.device
        _cuda(x, "x")
        if x.dim() == 2 and self.tokens == 1:
            x = x.unsqueeze(1)
        if x.dim() != 3 or x.shape[1] != self.tokens or x.shape[2] != self.cols:
            raise ValueError(f"x must be (n, {self.tokens}, {self.cols}), got {tuple(x.shape)}")
        if x.device != device:
            raise ValueError(f"x is on {x.device}, the cache on {device}")
        n = x.shape[0]
        dt = _dtype_id(x.dtype, "x")
        _table(index, torch.int64, n, device, "index")
        if lengths is not None:
            if self.lengths is None:
                raise ValueError("lengths given for a cache without lengths")
            _table(lengths, torch.int32, n, device, "lengths")
        if n == 0:
            return
        if x.stride(2) != 1 and self.cols != 1:
            raise ValueError("the values of a row of x must be contiguous")
        if (self.tokens > 1 and x.stride(1) < self.cols) or (n > 1 and x.stride(0) < self.cols):
            raise ValueError("the rows of x overlap")
        if _away(device, stream):
            with _there(device, stream):
                return self.write(index, x, lengths=lengths)
        owner = self._claims() if n > _capi.MX_SCAN_SAMPLES else None
        torch.autograd.graph.increment_version([self.codes, self.scales] if self.lengths is None else [self.codes, self.scales, self.lengths])
        _capi.check(_capi.load().tlb_mx_write(self._struct(owner), index.data_ptr(), n, x.data_ptr(), dt, x.stride(1), x.stride(0),
                                              None if lengths is None else lengths.data_ptr(), _raw_stream(device.index)))

    def _claims(self):
        """The words that a long write decides with between samples naming the same slot, -1 each.  Every stream has its
        own, so that writes on several streams share nothing but the rows; a captured write too, whose words are filled
        when it is replayed."""
        stream = _raw_stream(self.device.index)
        owner = self._owners.get(stream)
        if owner is None or torch.cuda.is_current_stream_capturing():
            owner = torch.full((max(self.slots, 1),), -1, dtype=torch.int32, device=self.device)
            if not torch.cuda.is_current_stream_capturing():
                self._owners[stream] = owner
        return owner

    def _picked(self, index):
        if index is None:
            return self.slots, None
        _table(index, torch.int64, None, self.device, "index")
        return index.shape[0], index.data_ptr()

    def read(self, index=None, dtype=torch.bfloat16, *, out=None, stream=None):
        """Samples ``index`` (int64 CUDA tensor; None: all, in order) as values (n, tokens, cols) of ``dtype``, zeros
        behind a sample's length and for an index outside the cache (reported in ``status``).  A cache with
        lengths gives ``(values, lengths)``."""
        n, at = self._picked(index)
        dt = _dtype_id(dtype, "dtype")
        device = self.device
        if _away(device, stream):
            with _there(device, stream):
                return self.read(index, dtype, out=out)
        out = _out(out, (n, self.tokens, self.cols), dtype, device)
        lengths = None if self.lengths is None else torch.empty(n, dtype=torch.int32, device=device)
        _capi.check(_capi.load().tlb_mx_read(self._struct(), at, n, out.data_ptr(), dt, None if lengths is None else lengths.data_ptr(),
                                             _raw_stream(device.index)))
        return out if lengths is None else (out, lengths)

    def read_mx(self, index=None, *, stream=None):
        """The same samples as they are held: an ``MxTensor`` (n, tokens, cols) with memory of its own, zero rows
        where ``read`` gives zeros; with ``(…, lengths)`` for a cache that has them."""
        n, at = self._picked(index)
        device = self.device
        if _away(device, stream):
            with _there(device, stream):
                return self.read_mx(index)
        q = MxTensor._empty((n, self.tokens, self.cols), (n, self.tokens), self.format, self._fmt, _own(self.scale), device)
        lengths = None if self.lengths is None else torch.empty(n, dtype=torch.int32, device=device)
        _capi.check(_capi.load().tlb_mx_read_codes(self._struct(), at, n, *q._at(), None if lengths is None else lengths.data_ptr(),
                                                   _raw_stream(device.index)))
        return q if lengths is None else (q, lengths)
