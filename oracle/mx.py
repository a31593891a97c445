"""MXFP4 (OCP MX v1.0: e2m1 elements, one power-of-two scale per 32) in fp64: the oracle of lmi_mx_quantize and
lmi_mx_product."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def quantize(x):
    """x (rows, k) -> (codes uint8 (rows, B*32), scales uint8 (rows, B)); codes of a NaN block are not defined (0 here)."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    b = -(-k // BLOCK)
    v = np.zeros((rows, b * BLOCK))
    v[:, :k] = x
    v = v.reshape(rows, b, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    amax = np.abs(v).max(-1)
    exponent = np.where(amax > 0, np.frexp(amax)[1] - 1 - 2, -127).clip(-127)      # frexp: amax = m 2^e, m in [0.5, 1)
    u = np.abs(v) / np.exp2(exponent.astype(np.float64))[..., None]
    code = np.zeros(v.shape, np.uint8)
    for c in range(1, 8):       # nearest magnitude; the midpoint goes to the even code
        mid = (GRID[c - 1] + GRID[c]) / 2
        code += (u > mid) | ((u == mid) & (c % 2 == 0))
    code |= np.where(np.signbit(v), 8, 0).astype(np.uint8)
    return code.reshape(rows, b * BLOCK), np.where(bad, 255, exponent + 127).astype(np.uint8)


def dequantize(codes, scales, k):
    rows = codes.shape[0]
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(rows, -1, BLOCK) * s[..., None]).reshape(rows, -1)[:, :k]


def unpack(packed):
    """(rows, n) bytes -> (rows, 2n) codes, low half first."""
    p = np.asarray(packed)
    return np.stack([p & 15, p >> 4], -1).reshape(p.shape[0], -1)


def rows_of(packed, scales, rows, k):
    """The kernels' order -- packed (S, G, [2][32][16]), scales (Q, G, [2][32][4]): step of 64 along k (scales: four steps), group of 32 rows,
    block of the step, row, bytes (steps) -- as (bytes (rows, 16*B), scales (rows, B)); and whether all that lies beyond is zero."""
    packed, scales = np.asarray(packed), np.asarray(scales)
    packed, scales = packed.reshape(*packed.shape[:2], 2, 32, 16), scales.reshape(*scales.shape[:2], 2, 32, 4)
    b = -(-k // BLOCK)
    p = packed.transpose(1, 3, 0, 2, 4).reshape(packed.shape[1] * 32, -1)
    s = scales.transpose(1, 3, 0, 4, 2).reshape(scales.shape[1] * 32, -1)
    clean = not (p[rows:].any() or p[:, 16 * b:].any() or s[rows:].any() or s[:, b:].any())
    return p[:rows, :16 * b], s[:rows, :b], clean


def values(x):
    """What a quantised x (rows, k) stands for."""
    return dequantize(*quantize(x), np.asarray(x).shape[1])


def product(x, w, bias=None, act=None):
    """act(Q(x) Q(w)^T + bias), and the sum of |terms| that bounds the error of an fp32 sum."""
    a, b = values(x), values(w)
    y, size = a @ b.T, np.abs(a) @ np.abs(b).T
    if bias is not None:
        y, size = y + np.asarray(bias, np.float64), size + np.abs(np.asarray(bias, np.float64))
    with np.errstate(over="ignore", invalid="ignore"):
        return (y / (1 + np.exp(-y)) if act == "silu" else y), size
