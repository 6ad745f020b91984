"""Plain 64-bit implementations of the dropout and MXFP4 operators (numpy),
written from the definitions in include/sbx.h, for the tests.

Everything here is exact: a value of fp32, bf16 or fp16 is a double, and so
are its products with a power of two, its MXFP4 rounding and (with scale codes
near each other) whole dot products.
"""
import numpy as np

TAG = 0x44524F50
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def philox(counter, key):
    """Philox4x32-10: four uint64 arrays holding 32-bit words."""
    c = [np.asarray(x, dtype=np.uint64) for x in counter]
    k0, k1 = int(key) & 0xFFFFFFFF, int(key) >> 32
    m32 = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m32,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def threshold(p):
    return int(np.floor(65536.0 * p + 0.5))


def keep(rows, cols, p, seed, stream_id, row0=0):
    """The mask of rows row0 .. row0 + rows - 1."""
    chunks = (cols + 7) // 8
    chunk, row = np.meshgrid(np.arange(chunks), np.arange(row0, row0 + rows))
    w = philox((chunk, row, np.full_like(chunk, stream_id), np.full_like(chunk, TAG)), seed)
    h = np.stack([x for word in w for x in (word & np.uint64(0xFFFF), word >> np.uint64(16))], -1)
    return h.reshape(rows, chunks * 8)[:, :cols] >= threshold(p)


def dropped(x, p=0.0, seed=0, stream_id=0, gate=None):
    """The dropout of x in its arithmetic: float64 x in 64 bits, others in 32."""
    real = np.float64 if x.dtype == np.float64 else np.float32
    y = x.astype(real)
    if p > 0:
        t = threshold(p)
        scale = real(65536.0 / (65536 - t)) if t < 65536 else real(0)
        with np.errstate(invalid="ignore", over="ignore"):
            y = np.where(keep(*x.shape, p, seed, stream_id), y * scale, real(0))
    return y if gate is None else np.where(gate.astype(real) > 0, y, real(0))


def quantize(v):
    """Rows of v to MXFP4: element codes (rows x blocks x 32, 4 bits) and scale
    codes (rows x blocks)."""
    v = np.asarray(v, dtype=np.float64)
    rows, cols = v.shape
    nb = (cols + 31) // 32
    b = np.zeros((rows, nb * 32))
    b[:, :cols] = v
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    a = np.ldexp(np.abs(b), -e[..., None])
    # nearest of the eight magnitudes, a tie to the even code
    mid = (GRID[1:] + GRID[:-1]) / 2
    lo, hi = np.searchsorted(mid, a, side="left"), np.searchsorted(mid, a, side="right")
    n = np.where(lo % 2 == 1, hi, lo) | (np.signbit(b).astype(np.int64) << 3)
    n = np.where(bad[..., None], 0, n)
    return n.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def pack(n, code, ldp=None, lds=None, fill=0):
    """Element and scale codes in the library's layout (uint8 P, S)."""
    rows, nb = code.shape
    ldp, lds = ldp or 16 * nb, lds or 8 * rows
    P = np.full((rows, ldp), fill, dtype=np.uint8)
    P[:, :16 * nb] = (n[..., 0::2] | (n[..., 1::2] << 4)).reshape(rows, nb * 16)
    groups = (nb + 7) // 8
    c = np.zeros((rows, groups * 8), dtype=np.uint8)
    c[:, :nb] = code
    S = np.full((groups, lds), fill, dtype=np.uint8)
    S[:, :8 * rows] = c.reshape(rows, groups, 8).transpose(1, 0, 2).reshape(groups, rows * 8)
    return P, S


def unpack(P, S, rows, cols):
    """The values (rows x cols, float64) of packed arrays."""
    nb = (cols + 31) // 32
    P = P.reshape(rows, -1)[:, :16 * nb]
    n = np.stack([P & 15, P >> 4], -1).reshape(rows, nb, 32)
    groups = (nb + 7) // 8
    c = S.reshape(groups, -1)[:, :8 * rows].reshape(groups, rows, 8).transpose(1, 0, 2)
    return values(n, c.reshape(rows, groups * 8)[:, :nb], cols)


def values(n, code, cols):
    v = np.where(n & 8, -1.0, 1.0) * GRID[n & 7] * np.exp2(code.astype(np.float64) - 127)[..., None]
    v = np.where((code == 255)[..., None], np.nan, v)
    return v.reshape(n.shape[0], -1)[:, :cols]


def fake(v):
    """v to MXFP4 and back."""
    return values(*quantize(v), v.shape[1])
