"""MXFP4 in numpy and 64 bits: quantisation from its definition, and the storage."""
from __future__ import annotations

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(x):
    """(codes 0..15, scale bytes) of a rows x cols array, blocks of 32 along the rows; the
    codes padded to whole blocks."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    nb = -(-cols // 32)
    b = np.zeros((rows, nb * 32))
    b[:, :cols] = x
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 1.0, np.abs(np.where(np.isfinite(b), b, 0)).max(-1))
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1))[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    with np.errstate(invalid="ignore"):
        a = np.abs(b) / np.ldexp(1.0, e)[..., None]
    mid = (GRID[1:] + GRID[:-1]) / 2
    up, down = np.searchsorted(mid, a, side="right"), np.searchsorted(mid, a, side="left")
    code = np.where(up == down, up, np.where(up % 2 == 0, up, down))
    code = code + 8 * np.signbit(b)
    return code.reshape(rows, -1).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(code, scale, cols):
    lut = np.concatenate([GRID, -GRID])
    s = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return (lut[code] * np.repeat(s, 32, 1))[:, :cols]


def pack_codes(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def tile_scales(scale, cuts=None):
    """Scale bytes (rows x blocks) in tiles of 128 x 4; ``cuts``: the first rows of the groups and the end."""
    rows, nb = scale.shape
    cuts = [0, rows] if cuts is None else cuts
    wide = -(-nb // 4)
    out = []
    for lo, hi in zip(cuts[:-1], cuts[1:]):
        tall = -(-(hi - lo) // 128)
        p = np.zeros((tall * 128, wide * 4), np.uint8)
        p[: hi - lo, :nb] = scale[lo:hi]
        out.append(p.reshape(tall, 4, 32, wide, 4).transpose(0, 3, 2, 1, 4).reshape(-1))
    return np.concatenate(out) if out else np.zeros(0, np.uint8)
