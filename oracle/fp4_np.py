"""float64 numpy statement of the 4-bit formats, of the product on them and of the gated norm (test infrastructure).

e2m1 grid, MX blocks of 32 with a power-of-two scale (the OCP microscaling rule), NV blocks of 16 with an e4m3 scale and
one scale for the tensor.  Written from the definitions: nearest grid value by distance, ties to the even code."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
# every finite e4m3 value in code order
E4M3 = np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127], dtype=np.float64)
BLOCK = {"mx": 32, "nv": 16}


def _nearest(v, grid):
    """Index of the nearest grid value; a tie takes the even index; above the top: the top."""
    i = np.clip(np.searchsorted(grid, v), 1, len(grid) - 1)
    lo, hi = v - grid[i - 1], grid[i] - v
    return np.where((lo < hi) | ((lo == hi) & (i % 2 == 1)), i - 1, i)


def quantise(x, fmt, ts=1.0):
    """f64 [rows, K] -> (codes uint8 [rows, blocks * bs], scale codes uint8 [rows, blocks])."""
    rows, K = x.shape
    bs = BLOCK[fmt]
    nb = -(-K // bs)
    xb = np.zeros((rows, nb * bs))
    xb[:, :K] = x
    xb = xb.reshape(rows, nb, bs)
    bad = ~np.isfinite(xb).all(-1)
    xb = np.where(bad[..., None], 0.0, xb)
    amax = np.abs(xb).max(-1)
    if fmt == "mx":
        e = np.maximum(np.frexp(amax)[1] - 3, -127)
        e = np.where(amax == 0, -127, e)
        code = (e + 127).astype(np.int64)
        scale = np.ldexp(1.0, e)
        nan_code = 255
    else:
        code = _nearest(amax / (6.0 * ts), E4M3)
        scale = E4M3[code] * ts
        nan_code = 127
    with np.errstate(divide="ignore", invalid="ignore"):
        t = np.where(scale[..., None] > 0, np.abs(xb) / scale[..., None], 0.0)
    q = _nearest(t, GRID)
    q = np.where(np.signbit(xb), q + 8, q)
    q = np.where((bad | (scale == 0))[..., None], 0, q)
    return q.reshape(rows, -1).astype(np.uint8), np.where(bad, nan_code, code).astype(np.uint8)


def scale_values(code, fmt):
    if fmt == "mx":
        return np.where(code == 255, np.nan, np.ldexp(1.0, code.astype(np.int64) - 127))
    return np.where(code == 127, np.nan, E4M3[np.minimum(code, 126)])


def values(q, code, fmt, K, ts=1.0):
    v = GRID[q & 7] * np.where(q & 8, -1.0, 1.0)
    return (v * np.repeat(scale_values(code, fmt), BLOCK[fmt], axis=1) * ts)[:, :K]


def row_bytes(K):
    return -(-K // 32) * 16


def pack(q, K):
    """codes [rows, >= K] -> packed bytes [rows, row_bytes(K)]."""
    full = np.zeros((q.shape[0], 2 * row_bytes(K)), dtype=np.uint8)
    full[:, :K] = q[:, :K]
    return full[:, 0::2] | (full[:, 1::2] << 4)


def scale_index(row, block, fmt, K):
    groups = -(-K // 256) * (256 // BLOCK[fmt] // 4)
    return ((row // 128) * groups + block // 4) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + block % 4


def lay_out_scales(code, fmt, K):
    rows, nb = code.shape
    out = np.zeros(-(-rows // 128) * -(-K // 256) * 128 * (256 // BLOCK[fmt]), dtype=np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    out[scale_index(r, b, fmt, K)] = code
    return out


def gated_norm(x, y, post=None, gate=None, mul=None, add=None, x_scale=1.0, eps=1e-6, mod_rows=0):
    """x_out and h in float64; gate, mul, add: [vectors, width]."""
    at = np.arange(x.shape[0]) // mod_rows if mod_rows else np.zeros(x.shape[0], dtype=np.int64)
    out = x_scale * x
    if y is not None:
        r = y if post is None else y / np.sqrt((y ** 2).mean(1, keepdims=True) + eps) * post
        out = out + (r if gate is None else gate[at] * r)
    if mul is None:
        return out, None
    h = out / np.sqrt((out ** 2).mean(1, keepdims=True) + eps) * mul[at]
    return out, h if add is None else h + add[at]
