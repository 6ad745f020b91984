"""Performance cases of the root-mean-square norm, of layers with MXFP4 weights for
a few tokens, and of the mixture-of-experts layer.

`listed()` gives the fixed cases, `draw(rng)` more of the same ranges; see the
comment at each.  `run` computes a case in plain torch operations where `own`
is false, and with the library's entry points where it is true.

Weights are MXFP4 matrices: 4-bit elements (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
sign) in blocks of 32 along a row, each block with a power-of-two scale in 8 bits
(e8m0).  Elements are packed two a byte, the even one in the low half, a row's
blocks padded with zeros; block b of row r has its scale at [b // 8][r][b % 8].  An
MXFP8 matrix is the same with 8-bit elements (e4m3, up to 448), one a byte.
"""
import math

import torch

own = False

F32, BF16, F16 = "f32", "bf16", "f16"
TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}
SIZE = {F32: 4, BF16: 2, F16: 2}
EPS = 1e-6


def _norm(dtype, rows, cols, residual=1, mx8=0, pad=0):
    return {"op": "norm", "dtype": dtype, "rows": rows, "cols": cols, "residual": residual, "mx8": mx8, "pad": pad}


def _grad(dtype, rows, cols, residual=1, pad=0):
    return {"op": "grad", "dtype": dtype, "rows": rows, "cols": cols, "residual": residual, "pad": pad}


def _linear(dtype, m, n, k, relu=0, pad=0):
    return {"op": "linear", "dtype": dtype, "m": m, "n": n, "k": k, "relu": relu, "pad": pad}


def _norm_linear(dtype, m, n, k):
    return {"op": "norm_linear", "dtype": dtype, "m": m, "n": n, "k": k}


def _moe(dtype, tokens, width, hidden, experts, topk, normalize=1):
    return {"op": "moe", "dtype": dtype, "tokens": tokens, "width": width, "hidden": hidden, "experts": experts,
            "topk": topk, "normalize": normalize}


def listed():
    return [
        # one token's norm, with the residual: a call costs its latency
        {"name": "norm_bf16_1x4096", **_norm(BF16, 1, 4096)},
        # a long batch's norm in training
        {"name": "norm_bf16_8192x8192", **_norm(BF16, 8192, 8192)},
        # a prompt's norm on its way into an 8-bit product, ragged, and its values
        {"name": "norm_mx8_f16_2047x4095", **_norm(F16, 2047, 4095, mx8=1)},
        # the norm's gradient in training, with the one that comes along the residual
        {"name": "norm_grad_bf16_8192x4096", **_grad(BF16, 8192, 4096)},
        # the same in 32 bits, odd sizes, rows without vector alignment
        {"name": "norm_grad_f32_4095x1001", **_grad(F32, 4095, 1001, pad=2)},
        # one token through a large layer: the weight is read once
        {"name": "linear_bf16_1x8192x8192", **_linear(BF16, 1, 8192, 8192)},
        # a few sequences' tokens through a layer and its ReLU, in 32 bits, odd sizes
        {"name": "linear_f32_7x4095x2047", **_linear(F32, 7, 4095, 2047, relu=1)},
        # a batch of sequences decoding: the norm to 8 bits, and the layer that reads it
        {"name": "norm_linear_bf16_16x8192x4096", **_norm_linear(BF16, 16, 8192, 4096)},
        # one token through a small mixture of experts
        {"name": "moe_bf16_1x2048x1024_8of64", **_moe(BF16, 1, 2048, 1024, 64, 8)},
        # a few tokens, ragged sizes, weights of the softmax over all experts
        {"name": "moe_f16_7x1000x700_2of9", **_moe(F16, 7, 1000, 700, 9, 2, normalize=0)},
        # the same layer in 32 bits
        {"name": "moe_f32_4x1024x2048_2of8", **_moe(F32, 4, 1024, 2048, 8, 2)},
        # a batch of sequences decoding: nearly every expert is read
        {"name": "moe_bf16_64x4096x2048_4of32", **_moe(BF16, 64, 4096, 2048, 32, 4)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case: norms of up to 2^26 values with 1 to 16384 on a side, layers
    with 1 to 64 tokens over 32 to 16384 terms, mixtures of 2 to 128 experts with 1
    to 64 tokens."""
    while True:
        op = rng.choice(["norm", "grad", "linear", "norm_linear", "moe"])
        dtype, pad, flag = rng.choice([F32, BF16, F16]), rng.choice([0, 0, 1, 8]), rng.randrange(2)
        if op in ("norm", "grad"):
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)
            residual = rng.randrange(2)
            c = _norm(dtype, rows, cols, residual, flag, pad) if op == "norm" else _grad(dtype, rows, cols, residual, pad)
            ok = rows * cols <= 1 << 26
        elif op in ("linear", "norm_linear"):
            m, n, k = _log_int(rng, 1, 64), _log_int(rng, 32, 16384), _log_int(rng, 32, 16384)
            c = _linear(dtype, m, n, k, flag, pad) if op == "linear" else _norm_linear(dtype, m, n, k)
            ok = n * k <= 1 << 27
        else:
            experts = _log_int(rng, 2, 128)
            c = _moe(dtype, _log_int(rng, 1, 64), _log_int(rng, 64, 4096), _log_int(rng, 64, 2048), experts,
                     rng.randint(1, min(8, experts)), flag)
            ok = experts * c["width"] * c["hidden"] <= 32 * 4096 * 2048
        if ok:
            return c


def _packed(rows, cols):
    """Bytes of an MXFP4 matrix: its elements and its blocks' scales."""
    return rows * -(-cols // 32) * 17


def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        # h is written where it is a sum; the values of the 8-bit form are what comes back
        n = case["rows"] * case["cols"]
        return {"bytes": n * e * (2 + 2 * case["residual"]) + case["cols"] * e, "flops": 6.0 * n}
    if op == "grad":
        n = case["rows"] * case["cols"]
        return {"bytes": n * e * (3 + case["residual"]) + case["cols"] * (e + 4), "flops": 12.0 * n}
    if op == "moe":
        t, w, h, x, k = (case[n] for n in ("tokens", "width", "hidden", "experts", "topk"))
        # as many different experts as that many choices name on average
        read = x * (1 - (1 - k / x) ** t)
        return {"bytes": int(read * (_packed(2 * h, w) + _packed(w, h))) + x * w * e + 2 * t * w * e,
                "flops": 6.0 * t * k * w * h + 2.0 * t * x * w}
    m, n, k = case["m"], case["n"], case["k"]
    extra = 2 * m * k * e + k * e if op == "norm_linear" else 0  # the residual and the sum
    return {"bytes": m * k * e + _packed(n, k) + m * n * e + extra, "flops": 2.0 * m * n * k}


# ---- the plain forms ---------------------------------------------------------


def _power(e):
    """2^e in 32 bits, exactly (e from -127 to 127)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _unpack(P, S, rows, cols):
    """The values an MXFP4 matrix stands for, in 32 bits."""
    nb = -(-cols // 32)
    n = torch.stack((P & 15, P >> 4), -1).reshape(rows, nb, 32).to(torch.int32)
    e, f = (n >> 1) & 3, (n & 1).float()
    a = torch.where(e == 0, f * 0.5, (1 + 0.5 * f) * _power(e - 1))
    q = torch.where(n >= 8, -a, a)
    code = S.permute(1, 0, 2).reshape(rows, -1)[:, :nb].to(torch.int32)
    return (q * _power(code - 127)[..., None]).reshape(rows, -1)[:, :cols]


def _fake8(v):
    """v (32 bits) to MXFP8 and back."""
    rows, cols = v.shape
    nb = -(-cols // 32)
    b = torch.nn.functional.pad(v, (0, nb * 32 - cols)).reshape(rows, nb, 32)
    top = b.abs().amax(-1)
    e = torch.where(top == 0, -127, (torch.frexp(top)[1] - 9).clamp(min=-127))  # frexp's exponent is floor(log2) + 1
    q = (b * _power(-e)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return (q * _power(e)[..., None]).reshape(rows, nb * 32)[:, :cols]


def _normed(x, r, w, dt):
    """The sum h and its norm; in 64 bits, for what is next to a border of the 8-bit form."""
    h = x if r is None else (x.float() + r.float()).to(dt)
    f = h.double()
    return h, (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * w.double()).float()


def _route(x, wr, topk, normalize):
    """Experts by their logits in 64 bits, the highest first and ties by index."""
    logits = x.double() @ wr.double().t()
    top, chosen = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, chosen = top[:, :topk], chosen[:, :topk]
    e = torch.exp(top - top[:, :1])
    total = e.sum(-1, keepdim=True) if normalize else torch.exp(logits - top[:, :1]).sum(-1, keepdim=True)
    return chosen, (e / total).float()


# ---- inputs ------------------------------------------------------------------


def _pack(x):
    """An MXFP4 matrix as a program holds it: packed elements and scales."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    v = torch.nn.functional.pad(x, (0, nb * 32 - cols)).reshape(rows, nb, 32)
    top = v.abs().amax(-1)
    code = torch.where(top == 0, 0, (torch.frexp(top)[1] + 124).clamp(0, 254))
    v = v * _power(127 - code)[..., None]
    # halves up to 2, wholes up to 4, then twos, each to the nearest; codes count up with the magnitude
    a = v.abs()
    n = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4))
    n = n.clamp(max=7).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    n = n.reshape(rows, nb * 16, 2)
    P = (n[..., 0] | (n[..., 1] << 4)).contiguous()
    S = torch.nn.functional.pad(code.to(torch.uint8), (0, -nb % 8)).reshape(rows, -1, 8).permute(1, 0, 2).contiguous()
    return P, S


def prepare(case, seed):
    """Activations are normal with a few large columns, weights normal with
    variance 1 / terms, a norm's around one, gradients small; weights are packed.
    Results go to memory that the program keeps."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dt = case["op"], TORCH[case["dtype"]]

    def normal(rows, cols, scale=1.0, loud=False):
        t = torch.randn((rows, cols), generator=gen, device="cuda") * scale
        if loud:
            t *= torch.where(torch.rand((1, cols), generator=gen, device="cuda") < 0.01, 8.0, 1.0)
        return t

    def padded(rows, cols, scale=1.0, loud=False):
        return normal(rows, cols + case["pad"], scale, loud).to(dt)[:, :cols]

    def empty(rows, cols, dtype=dt):
        return torch.empty((rows, cols), dtype=dtype, device="cuda")

    def room8(rows, cols):
        nb = -(-cols // 32)
        return empty(rows, nb * 32, torch.uint8), torch.empty((-(-nb // 8), rows, 8), dtype=torch.uint8, device="cuda")

    s = {"case": case}
    if op in ("norm", "grad"):
        rows, cols = case["rows"], case["cols"]
        s["w"] = (1.0 + normal(1, cols, 0.1))[0].to(dt)
        s["x"] = padded(rows, cols, loud=True)
        if op == "norm":
            s["r"] = padded(rows, cols, 2.0, loud=True) if case["residual"] else None
            s["h"], s["y"] = empty(rows, cols) if case["residual"] else None, empty(rows, cols)
            s["P"], s["S"] = room8(rows, cols) if case["mx8"] else (None, None)
        else:
            s["dy"] = padded(rows, cols, 1e-3)
            s["dr"] = padded(rows, cols, 1e-3) if case["residual"] else None
            s["dx"] = empty(rows, cols)
            s["dw"] = torch.empty(cols, dtype=torch.float32, device="cuda")
    elif op == "moe":
        t, w, h, x = case["tokens"], case["width"], case["hidden"], case["experts"]
        s["x"] = normal(t, w, loud=True).to(dt)
        s["wr"] = normal(x, w, w ** -0.5).to(dt)
        s["W1"], s["S1"] = _pack(normal(x * 2 * h, w, w ** -0.5))
        s["W2"], s["S2"] = _pack(normal(x * w, h, h ** -0.5))
        s["y"] = empty(t, w)
        s["chosen"], s["weights"] = empty(t, case["topk"], torch.int32), empty(t, case["topk"], torch.float32)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["B"], s["SB"] = _pack(normal(n, k, k ** -0.5))
        s["y"] = empty(m, n)
        if op == "linear":
            s["x"] = padded(m, k, loud=True)
        else:
            s["x"], s["r"] = normal(m, k, loud=True).to(dt), normal(m, k, 2.0, loud=True).to(dt)
            s["w"] = (1.0 + normal(1, k, 0.1))[0].to(dt)
            s["h"] = empty(m, k)
            s["P"], s["S"] = room8(m, k)
    return s


# ---- one pass ----------------------------------------------------------------


def _plain_moe(s):
    c = s["case"]
    t, w, h, x, k = (c[n] for n in ("tokens", "width", "hidden", "experts", "topk"))
    chosen, weights = _route(s["x"], s["wr"], k, c["normalize"])
    xf = s["x"].float()
    if t * k < x:  # the chosen experts' weights alone
        W1 = s["W1"].reshape(x, 2 * h, -1)[chosen.flatten()].flatten(0, 1)
        S1 = s["S1"].reshape(-1, x, 2 * h, 8)[:, chosen.flatten()].flatten(1, 2)
        W2 = s["W2"].reshape(x, w, -1)[chosen.flatten()].flatten(0, 1)
        S2 = s["S2"].reshape(-1, x, w, 8)[:, chosen.flatten()].flatten(1, 2)
        W1 = _unpack(W1, S1, t * k * 2 * h, w).reshape(t, k * 2 * h, w)
        gu = (W1 @ xf[:, :, None]).reshape(t * k, 2 * h)
        a = torch.nn.functional.silu(gu[:, :h]) * gu[:, h:]
        W2 = _unpack(W2, S2, t * k * w, h).reshape(t * k, w, h)
        y = ((W2 @ a[:, :, None]).reshape(t, k, w) * weights[..., None]).sum(1)
    else:  # every expert for every token, its weight zero where it was not chosen
        gu = (xf @ _unpack(s["W1"], s["S1"], x * 2 * h, w).t()).reshape(t, x, 2 * h)
        a = torch.nn.functional.silu(gu[..., :h]) * gu[..., h:]
        a = a * torch.zeros((t, x), device=a.device).scatter(1, chosen, weights)[..., None]
        W2 = _unpack(s["W2"], s["S2"], x * w, h).reshape(x, w, h).permute(1, 0, 2).reshape(w, x * h)
        y = a.reshape(t, x * h) @ W2.t()
    return {"y": y.to(s["x"].dtype), "chosen": chosen.to(torch.int32), "weights": weights}


def _run_plain(s):
    c, dt = s["case"], TORCH[s["case"]["dtype"]]
    op = c["op"]
    if op == "norm":
        h, y = _normed(s["x"], s["r"], s["w"], dt)
        y = (_fake8(y) if c["mx8"] else y).to(dt)
        return {"h": h, "y": y} if c["residual"] else {"y": y}
    if op == "grad":
        h, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
        rs = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
        n, g = h * rs, dy * w
        dx = rs * (g - n * (g * n).mean(-1, keepdim=True))
        if c["residual"]:
            dx = dx + s["dr"].float()
        return {"dx": dx.to(dt), "dw": (dy * n).sum(0)}
    if op == "moe":
        return _plain_moe(s)
    B = _unpack(s["B"], s["SB"], c["n"], c["k"])
    if op == "linear":
        y = s["x"].float() @ B.t()
        return (y.clamp_min(0.0) if c["relu"] else y).to(dt)
    h, v = _normed(s["x"], s["r"], s["w"], dt)
    return {"h": h, "y": (_fake8(v) @ B.t()).to(dt)}


def _workspace(s, size):
    if "workspace" not in s:
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _run_own(s):
    import sushiblas_amd as sbx

    c = s["case"]
    code = {F32: sbx.F32, BF16: sbx.BF16, F16: sbx.F16}[c["dtype"]]
    op = c["op"]

    def norm(x, r, h, y, P, S):
        optional = {} if r is None else {"R": r, "ldr": r.stride(0), "H": h, "ldh": h.stride(0)}
        if P is not None:
            optional |= {"P": P, "ldp": P.stride(0), "S": S, "lds": S.stride(0)}
        else:
            optional |= {"Y": y, "ldy": y.stride(0)}
        sbx.rms_norm(code, x.shape[0], x.shape[1], x, x.stride(0), s["w"], EPS, **optional)

    if op == "norm":
        norm(s["x"], s["r"], s["h"], s["y"], s["P"], s["S"])
        if c["mx8"]:
            P, S, y = s["P"], s["S"], s["y"]
            sbx.mx8_dequantize(code, c["rows"], c["cols"], P, P.stride(0), S, S.stride(0), y, y.stride(0))
        return {"h": s["h"], "y": s["y"]} if c["residual"] else {"y": s["y"]}
    if op == "grad":
        x, dy, dr, dx = s["x"], s["dy"], s["dr"], s["dx"]
        sbx.rms_norm_grad(code, c["rows"], c["cols"], x, x.stride(0), s["w"], EPS, dy, dy.stride(0), dx, dx.stride(0),
                          DW=s["dw"], DR=dr, lddr=0 if dr is None else dr.stride(0),
                          workspace=_workspace(s, sbx.rms_norm_grad_workspace(c["rows"], c["cols"])))
        return {"dx": dx, "dw": s["dw"]}
    if op == "moe":
        sizes = [c[n] for n in ("tokens", "width", "hidden", "experts", "topk")]
        x, y, wr, W1, S1, W2, S2 = (s[n] for n in ("x", "y", "wr", "W1", "S1", "W2", "S2"))
        sbx.mx4_moe(code, *sizes, x, x.stride(0), wr, wr.stride(0), W1, W1.stride(0), S1, S1.stride(0), W2,
                    W2.stride(0), S2, S2.stride(0), y, y.stride(0), normalize=c["normalize"], chosen=s["chosen"],
                    weights=s["weights"], workspace=_workspace(s, sbx.mx4_moe_workspace(*sizes)))
        return {"y": y, "chosen": s["chosen"], "weights": s["weights"]}
    x, y, B, SB = s["x"], s["y"], s["B"], s["SB"]
    if op == "linear":
        sbx.mx4_linear(code, c["m"], c["n"], c["k"], 1.0, x, x.stride(0), B, B.stride(0), SB, SB.stride(0), 0.0, y,
                       y.stride(0), epilogue=sbx.EPILOGUE_RELU if c["relu"] else sbx.EPILOGUE_NONE)
        return y
    P, S = s["P"], s["S"]
    norm(x, s["r"], s["h"], None, P, S)
    sbx.mx4_linear(code, c["m"], c["n"], c["k"], 1.0, P, P.stride(0), B, B.stride(0), SB, SB.stride(0), 0.0, y,
                   y.stride(0), SX=S, ldsx=S.stride(0))
    return {"h": s["h"], "y": y}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- 64 bits -----------------------------------------------------------------


def _exact_unpack(P, S, rows, cols):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=P.device)
    table = torch.cat((table, -table))
    v = torch.empty((rows, P.shape[1] * 2), dtype=torch.float64, device=P.device)
    v[:, 0::2], v[:, 1::2] = table[(P % 16).long()], table[(P // 16).long()]
    b = torch.arange(cols, device=P.device) // 32
    r = torch.arange(rows, device=P.device)[:, None]
    return v[:, :cols] * ((S[b // 8, r, b % 8].long() + 896) << 52).view(torch.float64)


def _exact_norm(s):
    h = s["x"].double()
    if s["r"] is not None:
        h = (h + s["r"].double()).float().to(s["x"].dtype).double()  # (as the sum of two values in 32 bits is)
    return h, h / (h.pow(2).sum(-1, keepdim=True) / h.shape[1] + EPS).sqrt() * s["w"].double()


def _exact_fake8(v):
    """To MXFP8 and back by the quantum of each magnitude."""
    rows, cols = v.shape
    v = v.float().double()
    out = torch.empty_like(v)
    whole = cols // 32 * 32
    for part, width in ((slice(0, whole), 32), (slice(whole, cols), cols - whole)):
        if part.start == part.stop:
            continue
        b = v[:, part].reshape(rows, -1, width)
        top = b.abs().amax(-1, keepdim=True)
        scale = (((top.view(torch.int64) >> 52) - 8).clamp(min=896) << 52).view(torch.float64)
        a = b.abs() / scale
        # three bits after the leading one, down to 2^-9
        quantum = (((a.view(torch.int64) >> 52).clamp(min=1023 - 6) - 3) << 52).view(torch.float64)
        q = (torch.round(a / quantum) * quantum).clamp(max=448.0)
        out[:, part] = (torch.sign(b) * q * scale).reshape(rows, -1)
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("norm", "norm_linear"):
        h, v = _exact_norm(s)
    if op == "norm":
        y = _exact_fake8(v) if case["mx8"] else v
        return {"h": h, "y": y} if case["residual"] else {"y": y}
    if op == "norm_linear":
        return {"h": h, "y": _exact_fake8(v) @ _exact_unpack(s["B"], s["SB"], case["n"], case["k"]).t()}
    if op == "linear":
        y = s["x"].double() @ _exact_unpack(s["B"], s["SB"], case["n"], case["k"]).t()
        return y.relu() if case["relu"] else y
    if op == "grad":
        h, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
        d = h.shape[1]
        m = h.pow(2).sum(1) / d + EPS
        along = (dy * w * h).sum(1) / (d * m)
        dx = (dy * w - h * along[:, None]) / m.sqrt()[:, None]
        return {"dx": dx if s["dr"] is None else dx + s["dr"].double(), "dw": ((1 / m.sqrt()) @ (dy * h))}
    w, h, x, k = (case[n] for n in ("width", "hidden", "experts", "topk"))
    logits = s["x"].double() @ s["wr"].double().t()
    prob = torch.softmax(logits, -1)
    order = torch.argsort(logits, dim=-1, descending=True, stable=True)[:, :k]
    weight = prob.gather(1, order)
    if case["normalize"]:
        weight = weight / weight.sum(1, keepdim=True)
    y = torch.zeros((case["tokens"], w), dtype=torch.float64, device="cuda")
    for e in range(x):  # each expert once, for the tokens that chose it
        t, j = (order == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        W1 = _exact_unpack(s["W1"][e * 2 * h:(e + 1) * 2 * h], s["S1"][:, e * 2 * h:(e + 1) * 2 * h], 2 * h, w)
        W2 = _exact_unpack(s["W2"][e * w:(e + 1) * w], s["S2"][:, e * w:(e + 1) * w], w, h)
        gu = s["x"][t].double() @ W1.t()
        g, u = gu[:, :h], gu[:, h:]
        y[t] += weight[t, j][:, None] * ((g / (1 + torch.exp(-g)) * u) @ W2.t())
    return {"y": y, "chosen": None, "weights": weight}
