"""Plain 64-bit implementations of the norm, the MXFP8 format, the few-token layer and the
mixture of experts (numpy), written from the definitions in include/sbx.h, for the tests.
Tensors come as float64 arrays of values that their type holds."""
import numpy as np

import mx4_reference as mx4

TYPES = ["f32", "bf16", "f16"]
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # finfo.eps / 2: of one rounding
TOP = {"f32": 2.0 ** 128 - 2.0 ** 104, "bf16": 2.0 ** 128 - 2.0 ** 120, "f16": 65504.0}
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}  # of one among subnormals


def types(name):
    import torch
    import sushiblas_amd as sbx
    return {"f32": (torch.float32, sbx.F32), "bf16": (torch.bfloat16, sbx.BF16), "f16": (torch.float16, sbx.F16)}[name]


def f64(t):
    return t.detach().cpu().double().numpy()


def norm(h, w, eps):
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        s = 1.0 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
        return h * s * w, s


def norm_grad(h, w, eps, dy, dr=None):
    """dx, dw, and for each the sum of its terms' magnitudes."""
    s = norm(h, w, eps)[1]
    g = dy * w
    along = (g * h).mean(-1, keepdims=True)
    dx = s * g - h * s ** 3 * along
    size = np.abs(s * g) + np.abs(h) * s ** 3 * np.abs(g * h).mean(-1, keepdims=True)
    if dr is not None:
        dx, size = dx + dr, size + np.abs(dr)
    terms = s * dy * h
    return dx, terms.sum(0), size, np.abs(terms).sum(0)


def e4m3(a):
    """|a| <= 448 to the nearest e4m3 value, ties to even: quanta of 2^-3 of the leading bit, 2^-9 at least."""
    m = np.abs(a)
    e = np.maximum(np.frexp(np.where(m == 0, 1.0, m))[1] - 1, -6)
    q = np.ldexp(1.0, e - 3)
    return np.sign(a) * np.round(m / q) * q


def e4m3_byte(v):
    """The byte of an e4m3 value."""
    m = np.abs(v)
    e = np.maximum(np.frexp(np.where(m == 0, 1.0, m))[1] - 1, -6)
    f = np.round(m / np.ldexp(1.0, e - 3)).astype(np.int64)  # 8 to 15, less among subnormals
    n = np.where(f >= 8, (e + 7) * 8 + f - 8, f)
    return (n | (np.signbit(v).astype(np.int64) << 7)).astype(np.uint8)


def quantize8(v):
    """Rows of v (64 bits, rounded to 32 here) to MXFP8: bytes (rows x blocks x 32), codes (rows x blocks)."""
    with np.errstate(over="ignore"):
        v = np.asarray(v).astype(np.float32).astype(np.float64)
    rows, cols = v.shape
    nb = (cols + 31) // 32
    b = np.zeros((rows, nb * 32))
    b[:, :cols] = v
    b = b.reshape(rows, nb, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    e = np.maximum(np.where(top > 0, np.frexp(top)[1] - 1 - 8, -127), -127)
    q = np.clip(np.ldexp(b, -e[..., None]), -448.0, 448.0)
    return e4m3_byte(np.copysign(e4m3(q), b)), np.where(bad, 255, e + 127).astype(np.uint8)


def codes(code, lds=None, fill=0):
    """Scale codes (rows x blocks) in the library's layout."""
    rows, nb = code.shape
    groups = (nb + 7) // 8
    c = np.zeros((rows, groups * 8), dtype=np.uint8)
    c[:, :nb] = code
    S = np.full((groups, lds or 8 * rows), fill, dtype=np.uint8)
    S[:, :8 * rows] = c.reshape(rows, groups, 8).transpose(1, 0, 2).reshape(groups, rows * 8)
    return S


def e4m3_values():
    n = np.arange(256)
    e, f = n >> 3 & 15, n & 7
    a = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0))
    a = np.where(n & 127 == 127, np.nan, a)
    return np.where(n & 128, -a, a)


def values8(n, code, cols):
    """The values of bytes (rows x blocks x 32) under codes."""
    v = e4m3_values()[n] * np.exp2(code.astype(np.float64) - 127)[..., None]
    v = np.where((code == 255)[..., None], np.nan, v)
    return v.reshape(n.shape[0], -1)[:, :cols]


def route(x, wr, topk, normalize):
    """Chosen experts (the highest logits, NaN first, ties by index) and their shares."""
    with np.errstate(invalid="ignore", over="ignore"):
        logits = x @ wr.T
        key = np.where(np.isnan(logits), np.inf, logits)
        first = ~np.isnan(logits)
        order = np.stack([np.lexsort((np.arange(len(k)), -k, f)) for k, f in zip(key, first)])[:, :topk]
        top = np.take_along_axis(logits, order, 1)
        e = np.exp(top - top[:, :1])
        total = e.sum(1) if normalize else np.exp(logits - top[:, :1]).sum(1)
    return order, e / total[:, None], logits


def moe(x, wr, w1, w2, topk, normalize, rounded):
    """y (tokens x width), a bound of its error before the last rounding, chosen, shares.
    w1: experts x 2 hidden x width, w2: experts x width x hidden; rounded: what an
    activation is rounded by before the second product, relative.

    Sums of n terms in 32 bits, in any order, are off by (n + 2) 2^-24 of their terms'
    magnitudes at most; silu's slope is at most 1.1, its value good to 2^-20."""
    order, p, _ = route(x, wr, topk, normalize)
    hidden = w2.shape[2]
    y, off = np.zeros((x.shape[0], w2.shape[1])), np.zeros((x.shape[0], w2.shape[1]))
    u = 2.0 ** -24
    with np.errstate(over="ignore", invalid="ignore"):
        for t in range(x.shape[0]):
            for j in range(topk):
                a1, a2 = w1[order[t, j]], w2[order[t, j]]
                z = a1 @ x[t]
                ez = (x.shape[1] + 2) * u * (np.abs(a1) @ np.abs(x[t]))
                g, v = z[:hidden], z[hidden:]
                silu = g / (1 + np.exp(-g))
                a = silu * v
                ea = 1.1 * ez[:hidden] * (np.abs(v) + ez[hidden:]) + np.abs(silu) * ez[hidden:]
                ea = ea + (2.0 ** -20 + rounded) * np.abs(a)
                y[t] += p[t, j] * (a2 @ a)
                off[t] += p[t, j] * (np.abs(a2) @ (ea + (hidden + topk + 4) * u * (np.abs(a) + ea)))
    return y, off, order, p


def random_mx4(rng, rows, cols, lo=124, hi=130):
    """Element and scale codes of a random matrix, zeros past the last column, and its values."""
    nb = (cols + 31) // 32
    n = rng.integers(0, 16, (rows, nb, 32)).astype(np.uint8)
    n.reshape(rows, nb * 32)[:, cols:] = 0
    code = rng.integers(lo, hi, (rows, nb)).astype(np.uint8)
    return n, code, mx4.values(n, code, cols)


def packed(cuda, n, code, pp=0, ps=0, fill=0xFF):
    """On the device, with pp blocks and ps rows of codes of padding; what lies beside the matrix,
    codes past the last block among it, is `fill` (0xFF: NaN, were it used)."""
    import torch
    rows, nb = code.shape
    P, S = mx4.pack(n, code, ldp=16 * (nb + pp), lds=8 * (rows + ps), fill=fill)
    if nb % 8:
        S[-1, :8 * rows].reshape(rows, 8)[:, nb % 8:] = fill
    return torch.from_numpy(P).to(cuda), torch.from_numpy(S).to(cuda)


def padded(cuda, a, dt, pad, fill=float("nan")):
    """a's values as a matrix of dt with `pad` columns beside it."""
    import torch
    t = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=dt)
    t[:, :a.shape[1]] = torch.from_numpy(np.ascontiguousarray(a)).to(dt)
    return t.to(cuda)


def rounded_to(a, dt):
    """a's values after rounding to dt, in 64 bits."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dt).double().numpy()
