"""The microscaled 4-bit formats in numpy, 64 bits throughout (the checker of the fp4 tests)."""
import numpy as np

BLOCK = {"mxfp4": 32, "nvfp4": 16}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(b & 7) * 2.0 ** -9 if b < 8 else (8 + (b & 7)) * 2.0 ** ((b >> 3) - 10) for b in range(127)])


def nearest(v, grid):
    """Index of the nearest grid member, ties to the even index, beyond the last: the last."""
    v = np.asarray(v, np.float64)
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = np.searchsorted(mid, v, "left"), np.searchsorted(mid, v, "right")
    return np.where(lo % 2 == 0, lo, hi)


def quantize(x, fmt):
    """(codes [rows, cols], scale bytes [rows, blocks], g) of x (any float array)."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    bs = BLOCK[fmt]
    nb = -(-cols // bs)
    codes = np.zeros((rows, cols), np.uint8)
    scales = np.zeros((rows, nb), np.uint8)
    g = 1.0
    if fmt == "nvfp4":
        fin = np.abs(x[np.isfinite(x)])
        top = fin.max() if fin.size else 0.0
        if top > 0:
            g = 2.0 ** -126
            while top > 2688 * g:
                g *= 2
    for b in range(nb):
        blk = x[:, b * bs:(b + 1) * bs]
        amax = np.abs(blk).max(1)
        bad = ~np.isfinite(amax)
        amax = np.where(bad, 0.0, amax)
        if fmt == "mxfp4":
            e = np.full(rows, -127)
            for r in np.nonzero(amax)[0]:
                m, x2 = np.frexp(amax[r])
                e[r] = max(-127, x2 - (3 if m <= 0.75 else 2))
                while amax[r] > 6 * 2.0 ** e[r]:
                    e[r] += 1
                while e[r] > -127 and amax[r] <= 3 * 2.0 ** e[r]:
                    e[r] -= 1
            s = 2.0 ** e.astype(np.float64)
            scales[:, b] = np.where(bad, 255, e + 127)
        else:
            i = nearest(amax / (6 * g), E4M3)
            s = E4M3[i] * g
            scales[:, b] = np.where(bad, 127, i)
        v = np.where(s[:, None] > 0, blk / np.where(s > 0, s, 1.0)[:, None], 0.0)
        v = np.where(bad[:, None], 0.0, v)
        codes[:, b * bs:(b + 1) * bs] = nearest(np.abs(v), E2M1) | ((v < 0).astype(np.uint8) << 3)
    return codes, scales, g


def values(codes, scales, g, fmt):
    t = np.concatenate([E2M1, -E2M1])
    if fmt == "mxfp4":
        s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    else:
        s = np.concatenate([E4M3, [np.nan]])[scales & 127]
    return t[codes] * np.repeat(s, BLOCK[fmt], axis=1)[:, : codes.shape[1]] * g


def pack(codes):
    if codes.shape[1] % 2:
        codes = np.pad(codes, ((0, 0), (0, 1)))
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed, cols):
    out = np.empty((packed.shape[0], packed.shape[1] * 2), np.uint8)
    out[:, 0::2], out[:, 1::2] = packed & 15, packed >> 4
    return out[:, :cols]


def topk(va, vb, k, self_offset=None, fmt="nvfp4"):
    """Indices and float32 values by (value descending, index ascending); blocks add in order."""
    m, n = va.shape[0], vb.shape[0]
    bs = BLOCK[fmt]
    p = np.zeros((m, n))
    for c in range(0, va.shape[1], bs):
        p = p + va[:, c:c + bs] @ vb[:, c:c + bs].T
    idx = np.full((m, k), -1, np.int32)
    val = np.full((m, k), -np.inf, np.float32)
    for i in range(m):
        cols = np.nonzero(~np.isnan(p[i]))[0]
        if self_offset is not None:
            cols = cols[cols != self_offset + i]
        o = cols[np.lexsort((cols, -p[i, cols]))][:k]
        idx[i, :len(o)] = o
        val[i, :len(o)] = p[i, o].astype(np.float32)
    return idx, val
