"""The 4-bit formats from their definition, in 64 bits (NumPy); shared by the CPU and GPU tests."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def nearest(v, grid):
    """Index of the nearest value of an ascending grid; halfway goes to the even index, beyond the end to the last."""
    v = np.minimum(v, grid[-1])
    hi = np.minimum(np.searchsorted(grid, v), len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    below, above = v - grid[lo], grid[hi] - v
    return np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def encode(x, fmt):
    """``(codes [R,K], scale bytes [R,K/block], row scales [R] or None)`` of finite ``x``."""
    x = np.asarray(x, np.float64)
    R, K = x.shape
    xb = x.reshape(R, -1, BLOCK[fmt])
    amax = np.abs(xb).max(-1)
    floor_log2 = lambda a: np.frexp(a)[1] - 1
    if fmt == "mxfp4":
        e = np.where(amax > 0, np.maximum(floor_log2(np.where(amax > 0, amax, 1)) - 2, -127), -127)
        q, byte, rows = xb * 2.0 ** -e[..., None].astype(np.float64), e + 127, None
    else:
        top = amax.max(-1)
        rows = np.where(top > 0, 2.0 ** np.maximum(floor_log2(np.where(top > 0, top, 1)) - 10, -126).astype(np.float64), 1.0)
        byte = nearest(amax / rows[:, None] / 6, E4M3)
        s = E4M3[byte][..., None] * rows[:, None, None]
        q = np.where(s > 0, xb / np.where(s > 0, s, 1), 0)
    codes = nearest(np.abs(q), E2M1) | (np.signbit(q).astype(np.int64) << 3)
    return codes.reshape(R, K), byte.astype(np.int64), rows


def values(codes, byte, rows, fmt):
    s = 2.0 ** (byte - 127.0) if fmt == "mxfp4" else E4M3[byte] * rows[:, None]
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return v * np.repeat(s, BLOCK[fmt], axis=1)
