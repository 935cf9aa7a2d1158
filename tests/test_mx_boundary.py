"""The microscaled entry points refuse bad arguments on the host, and their plain float64 form is what the
formats' definition says."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from mx_reference import BLOCK, E2M1, E4M3, decode, encode, padded
from turboloader_b200 import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FORMATS = {"nvfp4": 0, "mxfp4": 1, "mxfp8": 2}


def _fields(struct):
    text = open(os.path.join(ROOT, "include", "turboloader_b200.h")).read()
    start = text.index("typedef struct %s {" % struct)
    body = re.sub(r"/\*.*?\*/", "", text[start:text.index("} %s;" % struct)].split("{", 1)[1], flags=re.S)
    return [re.search(r"(\w+)\s*$", d.strip()).group(1) for d in body.split(";") if d.strip()]


def test_struct_layouts_match_the_header():
    assert _fields("tlb_mx_rows") == [f[0] for f in _capi.MxRows._fields_]
    assert _fields("tlb_mx_cache") == [f[0] for f in _capi.MxCache._fields_]
    text = open(os.path.join(ROOT, "include", "turboloader_b200.h")).read()
    assert "#define TLB_MX_MAX_COLS (1 << 20)" in text and _capi.MX_MAX_COLS == 1 << 20
    assert "#define TLB_MX_SCAN_SAMPLES %d" % _capi.MX_SCAN_SAMPLES in text


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("cols", [1, 16, 127, 128, 129, 1000])
def test_pitches(fmt, cols):
    lib = _capi.load()
    p = padded(cols)
    assert lib.tlb_mx_code_pitch(FORMATS[fmt], cols) == (p if fmt == "mxfp8" else p // 2)
    assert lib.tlb_mx_scale_pitch(FORMATS[fmt], cols) == p // BLOCK[fmt]
    assert lib.tlb_mx_code_pitch(3, cols) == lib.tlb_mx_scale_pitch(FORMATS[fmt], 0) == -1


def _rows(**kw):
    q = _capi.MxRows(0x1000, 0x2000, 8, 64, 0, 1.0, None)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize("kw,code", [
    (dict(format=3), 1), (dict(format=-1), 1), (dict(cols=0), 1), (dict(cols=(1 << 20) + 1), 1), (dict(rows=-1), 1),
    (dict(rows=(1 << 30) + 1), 7), (dict(codes=None), 1), (dict(scales=None), 1), (dict(codes=0x1008), 1),
    (dict(scales=0x2002), 1), (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1),
    (dict(scale=float("inf")), 1), (dict(scale_dev=0x3001), 1),
])
def test_bad_rows_are_refused_everywhere(kw, code):
    lib = _capi.load()
    q, good = _rows(**kw), _rows()
    cache = _capi.MxCache(q, 1, None, None, None)
    index, x = 0x4000, 0x5000
    assert lib.tlb_mx_quantize(C.byref(q), x, 0, 1 << 21, None) == code and lib.tlb_last_error()
    assert lib.tlb_mx_write(C.byref(cache), index, 1, x, 0, 1 << 21, 1 << 21, None, None) == code
    assert lib.tlb_mx_read(C.byref(cache), index, 1, x, 0, None, None) == code
    assert lib.tlb_mx_read_codes(C.byref(cache), index, 1, x, x, None, None) == code
    assert lib.tlb_mx_matmul(C.byref(q), C.byref(good), x, 0, None, 0, None) == code
    assert lib.tlb_mx_matmul(C.byref(good), C.byref(q), x, 0, None, 0, None) == code
    assert lib.tlb_mx_matmul_workspace(C.byref(q), C.byref(good), 0) == -1
    for a, b, ga, gb in ((q, None, None, x), (None, q, x, None), (good, q, x, x), (q, good, x, x)):
        a, b = (None if r is None else C.byref(r) for r in (a, b))
        assert lib.tlb_mx_grad(x, 0, 8, 8, a, b, ga, 0, gb, 0, None, 0, None) == code
        assert lib.tlb_mx_grad_workspace(0, 8, 8, a, b, ga, 0, gb, 0) == -1


def test_bad_calls_are_refused():
    lib = _capi.load()
    q = _rows()
    assert lib.tlb_mx_quantize(None, 0x5000, 0, 64, None) == 1
    assert lib.tlb_mx_quantize(C.byref(q), None, 0, 64, None) == 1
    assert lib.tlb_mx_quantize(C.byref(q), 0x5000, 3, 64, None) == 1          # dtype
    assert lib.tlb_mx_quantize(C.byref(q), 0x5000, 0, 63, None) == 1          # rows overlap
    assert lib.tlb_mx_quantize(C.byref(q), 0x5002, 0, 64, None) == 1          # fp32 at an odd address
    assert lib.tlb_mx_quantize(C.byref(_rows(rows=0)), None, 0, 0, None) == 0  # nothing to do

    def cache(rows=q, tokens=2, lengths=None, owner=None, status=None):
        return C.byref(_capi.MxCache(rows, tokens, lengths, owner, status))

    write = lib.tlb_mx_write
    assert write(None, 0x4000, 1, 0x5000, 0, 64, 128, None, None) == 1
    assert write(cache(tokens=0), 0x4000, 1, 0x5000, 0, 64, 128, None, None) == 1
    assert write(cache(tokens=3), 0x4000, 1, 0x5000, 0, 64, 128, None, None) == 1     # 8 rows are no whole samples of 3
    assert write(cache(), None, 1, 0x5000, 0, 64, 128, None, None) == 1
    assert write(cache(), 0x4000, 1, None, 0, 64, 128, None, None) == 1
    assert write(cache(), 0x4000, -1, 0x5000, 0, 64, 128, None, None) == 1
    assert write(cache(), 0x4000, 1 << 40, 0x5000, 0, 64, 128, None, None) == 7
    assert write(cache(), 0x4004, 1, 0x5000, 0, 64, 128, None, None) == 1             # index alignment
    assert write(cache(), 0x4000, 1, 0x5000, 0, 63, 128, None, None) == 1             # rows overlap
    assert write(cache(), 0x4000, 2, 0x5000, 0, 64, 63, None, None) == 1              # samples overlap
    assert write(cache(), 0x4000, 1, 0x5000, 0, 64, 128, 0x6000, None) == 1           # lengths, but the cache has none
    assert write(cache(), 0x4000, 257, 0x5000, 0, 64, 128, None, None) == 1           # owner is needed
    assert b"owner" in lib.tlb_last_error()
    assert write(cache(), 0x4000, 0, 0x5000, 0, 64, 128, None, None) == 0
    assert lib.tlb_mx_read(cache(), None, 5, 0x5000, 0, None, None) == 3              # more than the cache holds
    assert lib.tlb_mx_read(cache(), 0x4000, 1, None, 0, None, None) == 1
    assert lib.tlb_mx_read(cache(), 0x4000, 1, 0x5008, 0, None, None) == 1
    assert lib.tlb_mx_read(cache(), 0x4000, 1, 0x5000, 9, None, None) == 1
    assert lib.tlb_mx_read(cache(), 0x4000, 0, None, 0, None, None) == 0
    assert lib.tlb_mx_read_codes(cache(), 0x4000, 1, None, 0x5000, None, None) == 1
    assert lib.tlb_mx_matmul(C.byref(q), C.byref(_rows(format=1)), 0x5000, 0, None, 0, None) == 1
    assert lib.tlb_mx_matmul(C.byref(q), C.byref(_rows(cols=65)), 0x5000, 0, None, 0, None) == 1
    assert lib.tlb_mx_matmul(C.byref(q), C.byref(_rows(rows=(1 << 20) + 1)), 0x5000, 0, None, 0, None) == 7
    assert lib.tlb_mx_matmul(C.byref(q), C.byref(q), None, 0, None, 0, None) == 1
    assert lib.tlb_mx_matmul(C.byref(q), C.byref(q), 0x5000, 5, None, 0, None) == 1
    assert lib.tlb_mx_matmul(C.byref(q), C.byref(_rows(rows=0)), None, 0, None, 0, None) == 0
    r = C.byref(q)  # 8 rows

    def linear(a=r, x=0x5000, xd=0, xp=64, b=r, w=0x5800, wd=0, wp=64, out=0x6000, od=0, ws=None, size=0):
        return lib.tlb_mx_linear(a, x, xd, xp, b, w, wd, wp, out, od, ws, size, None)

    need = lib.tlb_mx_matmul_workspace(r, r, 0)
    assert need > 0 and linear() == 1 and b"workspace" in lib.tlb_last_error()
    ready = dict(ws=0x8000, size=need)
    assert linear(xd=3, **ready) == linear(wd=4, **ready) == linear(od=3, **ready) == linear(out=None, **ready) == 1
    assert linear(xp=63, **ready) == linear(wp=10, **ready) == linear(x=0x5002, **ready) == linear(w=0x5801, wd=1, **ready) == 1
    assert linear(a=None, **ready) == linear(b=C.byref(_rows(cols=65)), **ready) == linear(b=C.byref(_rows(format=2)), **ready) == 1
    none = C.byref(_rows(rows=0))
    assert linear(a=none, b=none, out=None) == 0

    def grad(g=0x5000, dtype=0, m=8, n=8, a=r, b=r, ga=0x6000, gb=0x7000, da=0, db=0, ws=None, size=0):
        return lib.tlb_mx_grad(g, dtype, m, n, a, b, ga, da, gb, db, ws, size, None)

    assert grad() == 1 and b"workspace" in lib.tlb_last_error()
    assert grad(dtype=3) == grad(da=-1) == grad(db=7) == grad(g=None) == grad(g=0x5004) == grad(ga=0x6008) == 1
    assert grad(m=7) == grad(n=7) == grad(m=-1) == grad(a=None) == grad(b=None) == grad(ga=None, gb=None) == 1
    assert grad(b=C.byref(_rows(format=2))) == grad(b=C.byref(_rows(cols=32))) == 1
    assert grad(m=1 << 30, a=C.byref(_rows(rows=1 << 30))) == 7
    assert grad(m=0, a=None, gb=None) == 0                                            # nothing to write
    need = lib.tlb_mx_grad_workspace(0, 8, 8, r, r, 0x6000, 0, 0x7000, 0)
    assert need > lib.tlb_mx_grad_workspace(0, 8, 8, None, r, 0x6000, 0, None, 0) > 0
    assert grad(ws=0x8000, size=need - 1) == grad(ws=0x8010, size=need) == 1


def test_host_tensors_and_unknown_formats_are_refused():
    import torch

    import turboloader_b200 as tb

    x = torch.zeros(4, 32)
    for call in (lambda: tb.mx_quantize(x), lambda: tb.mx_linear(x, x), lambda: tb.MxTensor(x, x, (4, 32), "nvfp4"),
                 lambda: tb.MxCache(x, x, 32, "nvfp4"), lambda: tb.mx_matmul(x, x)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        tb.mx_quantize(x, "fp4")
    with pytest.raises(ValueError):
        tb.mx_linear(x, x, None)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            tb.CudaFeatureLoader(4, 1, 32)


# ---- the reference itself ---------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
def test_points_of_the_grid_stand_for_themselves(fmt):
    grid = E4M3[E4M3 <= 448] if fmt == "mxfp8" else E2M1
    top = 6.0 if fmt != "mxfp8" else 448.0
    row = np.zeros(BLOCK[fmt] * len(grid), np.float32).reshape(len(grid), -1)
    row[:, 0], row[:, 1], row[:, 2] = top, grid, -grid
    codes, scales = encode(row, fmt)
    got = decode(codes, scales, fmt, row.shape[1])
    assert np.array_equal(got, row.astype(np.float64))


def test_ties_go_to_even_codes_and_large_values_saturate():
    x = np.zeros((1, 16), np.float32)
    x[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0]
    codes, scales = encode(x, "nvfp4")
    assert decode(codes, scales, "nvfp4", 9)[0].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -4]
    x = np.zeros((1, 32), np.float32)
    x[0, :3] = [7.9, -7.9, 1.0]                       # floor(log2 a) = 2: scale 1, 7.9 saturates at 6
    codes, scales = encode(x, "mxfp4")
    assert scales[0, 0] == 127 and decode(codes, scales, "mxfp4", 3)[0].tolist() == [6, -6, 1]


def test_special_blocks():
    for fmt in FORMATS:
        x = np.zeros((1, 4 * BLOCK[fmt]), np.float32)
        x[0, 0], x[0, BLOCK[fmt]], x[0, 2 * BLOCK[fmt]] = np.nan, np.inf, 1e-45
        got = decode(*encode(x, fmt), fmt, x.shape[1])[0].reshape(4, -1)
        assert np.isnan(got[:2]).all() and (got[3] == 0).all() and np.isfinite(got[2]).all()
