"""The microscaled formats in numpy with 64-bit arithmetic, from their
definition; the oracle of tests/test_microscale*.py."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def blocks_of(cols):
    return -(-cols // 32)


def quantize(x, fmt):
    """x [rows, cols] (any float type) -> signed codes as values before the
    scale [rows, blocks, 32] and scale bytes [rows, blocks]."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    b = np.zeros((rows, blocks_of(cols) * 32))
    b[:, :cols] = x
    b = b.reshape(rows, -1, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(b).max(-1)
    fine = np.isfinite(top)
    safe = np.where(fine & (top > 0), top, 1.0)
    e = np.frexp(safe)[1] - 1
    e = np.where(top == 0, -2000, e)
    s = np.maximum(e - 2, -127) if fmt == "mxfp4" else np.maximum(e, -120)
    v = np.where(fine[..., None], b, 0.0)
    if fmt == "mxfp4":
        v = np.ldexp(v, -s[..., None])
        a = np.abs(v)
        # the nearest of the eight magnitudes, ties to the even code
        d = np.abs(np.minimum(a, 6.0)[..., None] - E2M1)
        best = d.min(-1, keepdims=True)
        tied = d == best
        even = np.arange(8) % 2 == 0
        k = np.where((tied & even).any(-1), np.argmax(tied & even, -1), np.argmax(tied, -1))
        q = np.where(np.signbit(v), -E2M1[k], E2M1[k])
    else:
        q = np.clip(np.rint(np.ldexp(v, 6 - s[..., None])), -127, 127)
    return q, np.where(fine, s + 127, 255).astype(np.uint8)


def values(q, scale, fmt, cols):
    """What codes and scale bytes stand for, [rows, cols] in 64 bits."""
    s = scale.astype(np.int64) - 127 - (0 if fmt == "mxfp4" else 6)
    v = np.ldexp(q, s[..., None])
    v[scale == 255] = np.nan
    return v.reshape(v.shape[0], -1)[:, :cols]


def rounded(x, fmt="mxfp4"):
    x = np.asarray(x)
    return values(*quantize(x, fmt), fmt, x.shape[1])


def code_bytes(q, fmt):
    """The stored codes of values before the scale, [rows, bytes]."""
    rows = q.shape[0]
    if fmt == "mxint8":
        return q.astype(np.int8).view(np.uint8).reshape(rows, -1)
    k = np.searchsorted(E2M1, np.abs(q)) | (np.signbit(q) * 8)
    k = k.astype(np.uint8).reshape(rows, -1, 2)
    return k[..., 0] | (k[..., 1] << 4)


def decode(codes, scale, fmt, cols):
    """Values of stored codes [rows, bytes] and row-major scales."""
    rows = codes.shape[0]
    if fmt == "mxint8":
        q = codes.view(np.int8).astype(np.float64)
    else:
        n = np.stack((codes & 15, codes >> 4), -1).reshape(rows, -1)
        q = E2M1[n & 7] * np.where(n >= 8, -1.0, 1.0)
    return values(q.reshape(rows, -1, 32), scale, fmt, cols)


def tile_scales(scale):
    """Row-major scales [rows, blocks] in tiles of 128 rows x 4 blocks; bytes
    that no block owns are 0."""
    rows, blocks = scale.shape
    tr, tq = -(-rows // 128), -(-blocks // 4)
    out = np.zeros(tr * tq * 512, np.uint8)
    for r in range(rows):
        for b in range(blocks):
            out[((r // 128) * tq + b // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4] = scale[r, b]
    return out
