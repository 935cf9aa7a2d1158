"""The microscaled formats in plain float64 numpy, from their definition; rounding is a search for the nearest
point of the format's grid.  Inputs are float32 values (what any input type widens to)."""
import numpy as np

BLOCK = {"nvfp4": 16, "mxfp4": 32, "mxfp8": 32}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] +
                [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1], np.float64)  # 0x7f is NaN


def padded(cols):
    return -(-cols // 128) * 128


def nearest(v, grid):
    """Number of the grid point nearest to each v >= 0; ties to the even number, above the last point: the last."""
    hi = np.clip(np.searchsorted(grid, v), 1, len(grid) - 1)
    lo = hi - 1
    down, up = v - grid[lo], grid[hi] - v
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)


def encode(x, fmt, scale=1.0):
    """(rows, cols) float32 -> codes (rows, code pitch), scales (rows, padded / block)."""
    rows, cols = x.shape
    with np.errstate(all="ignore"):
        t = (x.astype(np.float32) / np.float32(scale)).astype(np.float32)
    t = np.pad(t.astype(np.float64), ((0, 0), (0, padded(cols) - cols))).reshape(rows, -1, BLOCK[fmt])
    bad = ~np.isfinite(t).all(-1)
    t = np.where(bad[..., None], 0.0, t)
    a = np.abs(t).max(-1)
    if fmt == "nvfp4":
        sb = nearest((a.astype(np.float32) * np.float32(1 / 6)).astype(np.float64), E4M3)
        s = E4M3[sb]
        sb[bad] = 0x7F
    else:
        emax = 2 if fmt == "mxfp4" else 8
        e = np.maximum(np.frexp(a)[1] - 1 - emax, -127)
        e = np.where(a > 0, e, -127)
        s = np.ldexp(1.0, e)
        sb = (e + 127).astype(np.uint8)
        sb[bad] = 0xFF
    r = np.divide(t, s[..., None], out=np.zeros_like(t), where=s[..., None] > 0)
    grid, sign = (E4M3, 0x80) if fmt == "mxfp8" else (E2M1, 8)
    c = nearest(np.abs(r), grid)
    c = np.where(np.signbit(r), c | sign, c).astype(np.uint8).reshape(rows, -1)
    if fmt != "mxfp8":
        c = c[:, 0::2] | (c[:, 1::2] << 4)
    return c, sb


def decode(codes, scales, fmt, cols):
    """The values without the tensor's scale, float64 (rows, cols)."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    signed8 = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])
    if fmt == "mxfp8":
        c = signed8[codes]
    else:
        signed4 = np.concatenate([E2M1, -E2M1])
        c = np.stack([signed4[codes & 15], signed4[codes >> 4]], -1).reshape(codes.shape[0], -1)
    s = signed8[scales] if fmt == "nvfp4" else np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (c.reshape(codes.shape[0], -1, BLOCK[fmt]) * s[..., None]).reshape(codes.shape[0], -1)[:, :cols]
