"""Performance cases of the microscaled 4-bit (MXFP4) and dropout operators.

`listed()` gives the fixed cases, `draw(rng)` more of the same ranges; see the
comment at each.  `run` computes a case in plain torch operations where `own`
is false, and with the library's entry points where it is true.

An MXFP4 matrix holds 4-bit elements (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
sign) in blocks of 32 along a row, each block with a power-of-two scale in 8
bits (e8m0; 255 is NaN).  Elements are packed two a byte, the even one in the
low half, a row's blocks padded with zeros; block b of row r has its scale at
[b // 8][r][b % 8].
"""
import math

import torch

own = False

F32, F64, BF16, F16 = "f32", "f64", "bf16", "f16"
TORCH = {F32: torch.float32, F64: torch.float64, BF16: torch.bfloat16, F16: torch.float16}
SIZE = {F32: 4, F64: 8, BF16: 2, F16: 2}
TAG = 0x44524F50  # fourth counter word of the dropout's generator


def _dropout(dtype, rows, cols, p=0.1, gate=0, pad=0):
    return {"op": "dropout", "dtype": dtype, "rows": rows, "cols": cols, "p": p, "gate": gate, "pad": pad}


def _quantize(dtype, rows, cols, p=0.0, gate=0, pad=0):
    return {"op": "quantize", "dtype": dtype, "rows": rows, "cols": cols, "p": p, "gate": gate, "pad": pad}


def _product(dtype, m, n, k, alpha=1.0, beta=0.0, relu=0):
    return {"op": "product", "dtype": dtype, "m": m, "n": n, "k": k, "alpha": alpha, "beta": beta, "relu": relu}


def _linear(dtype, m, n, k, relu=0):
    return {"op": "linear", "dtype": dtype, "m": m, "n": n, "k": k, "relu": relu}


def _block(dtype, tokens, width, hidden, p=0.1):
    return {"op": "block", "dtype": dtype, "tokens": tokens, "width": width, "hidden": hidden, "p": p}


def listed():
    return [
        # dropout on the activations of a small layer: one call costs its latency
        {"name": "dropout_f32_512x1024", **_dropout(F32, 512, 1024)},
        # dropout forward on the activations of a long batch
        {"name": "dropout_bf16_8192x8192", **_dropout(BF16, 8192, 8192)},
        # its backward pass through the ReLU before it, odd sizes, rows without vector alignment
        {"name": "dropout_grad_bf16_4095x3001", **_dropout(BF16, 4095, 3001, p=0.2, gate=1, pad=2)},
        # a weight quantised along both of its axes, for the forward product and the gradient's
        {"name": "quantize_bf16_8192x8192", **_quantize(BF16, 8192, 8192)},
        # a gradient through dropout and ReLU on its way into both quantised forms, ragged
        {"name": "quantize_drop_f32_2047x4095", **_quantize(F32, 2047, 4095, p=0.1, gate=1)},
        # the smallest product of the benchmark
        {"name": "product_f32_512", **_product(F32, 512, 512, 512)},
        # ragged sizes, a result in 32 bits, as for a weight's gradient
        {"name": "product_f32_4095x3001x2047", **_product(F32, 4095, 3001, 2047)},
        # the largest product
        {"name": "product_bf16_8192", **_product(BF16, 8192, 8192, 8192)},
        # one token through a large layer: the weight is read once
        {"name": "linear_bf16_1x8192x8192", **_linear(BF16, 1, 8192, 8192)},
        # a few sequences' tokens through a layer and its ReLU
        {"name": "linear_f16_37x4096x1024", **_linear(F16, 37, 4096, 1024, relu=1)},
        # a batch of rows through a layer and its ReLU
        {"name": "linear_bf16_512x1024x1024", **_linear(BF16, 512, 1024, 1024, relu=1)},
        # a training step's feed-forward block: both layers, ReLU, dropout, and all gradients
        {"name": "block_bf16_4096x1024x4096", **_block(BF16, 4096, 1024, 4096)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case: dropout and quantisation of up to 2^26 values with 1 to
    16384 on a side, products of 1 to 8192 rows and columns over 32 to 16384
    terms, layers with 1 to 256 tokens, feed-forward blocks of up to 4096
    tokens."""
    while True:
        op = rng.choice(["dropout", "quantize", "product", "linear", "block"])
        gate, relu = rng.randrange(2), rng.randrange(2)
        p = rng.choice([0.05, 0.1, 0.2, 0.5])
        if op == "dropout":
            c = _dropout(rng.choice([F32, F64, BF16, F16]), _log_int(rng, 1, 16384), _log_int(rng, 1, 16384),
                         p=p, gate=gate, pad=rng.choice([0, 0, 1, 8]))
            ok = c["rows"] * c["cols"] <= 1 << 26
        elif op == "quantize":
            c = _quantize(rng.choice([F32, BF16, F16]), _log_int(rng, 1, 16384), _log_int(rng, 1, 16384),
                          p=rng.choice([0.0, p]), gate=gate, pad=rng.choice([0, 0, 1, 8]))
            ok = c["rows"] * c["cols"] <= 1 << 26
        elif op == "product":
            c = _product(rng.choice([F32, BF16, F16]), _log_int(rng, 1, 8192), _log_int(rng, 1, 8192),
                         _log_int(rng, 32, 16384), alpha=rng.choice([1.0, 1.5]), beta=rng.choice([0.0, 0.5, 1.0]),
                         relu=relu)
            ok = work(c)["flops"] <= 2.0 * 8192 ** 3
        elif op == "linear":
            c = _linear(rng.choice([F32, BF16, F16]), _log_int(rng, 1, 256), _log_int(rng, 64, 16384),
                        _log_int(rng, 64, 16384), relu=relu)
            ok = c["n"] * c["k"] <= 1 << 27
        else:
            c = _block(rng.choice([F32, BF16, F16]), _log_int(rng, 16, 4096), _log_int(rng, 64, 2048),
                       _log_int(rng, 64, 8192), p=p)
            ok = True
        if ok:
            return c


def _packed(rows, cols):
    """Bytes of an MXFP4 matrix: its elements and its blocks' scales."""
    nb = -(-cols // 32)
    return rows * nb * 17


def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * e * (2 + case["gate"]), "flops": float(n)}
    if op == "quantize":
        # the values of both forms are what comes back
        n = case["rows"] * case["cols"]
        return {"bytes": n * e * (3 + case["gate"]), "flops": 2.0 * n}
    if op == "block":
        t, d, h = case["tokens"], case["width"], case["hidden"]
        # x, dy in, y, dx out; both weights in, their gradients out in 32 bits
        return {"bytes": 4 * t * d * e + 2 * d * h * e + 2 * d * h * 4, "flops": 12.0 * t * d * h}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "product":
        reads_c = 1 if case["beta"] != 0 else 0
        return {"bytes": _packed(m, k) + _packed(n, k) + m * n * e * (1 + reads_c), "flops": 2.0 * m * n * k}
    return {"bytes": m * k * e + _packed(n, k) + m * n * e, "flops": 2.0 * m * n * k}


# ---- the plain forms ---------------------------------------------------------


def _philox_round(c, key):
    c0, c1, c2, c3 = c
    k0, k1 = key
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64; the shifts below keep their bits
    mask = 0xFFFFFFFF
    return ((b >> 32) & mask) ^ c1 ^ k0, b & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask


def _keep(rows, cols, p, seed, sid, device):
    """Which elements stay: 16 bits of Philox4x32-10 each, against p * 2^16."""
    chunks = -(-cols // 8)
    c = (torch.arange(chunks, device=device).expand(rows, chunks),
         torch.arange(rows, device=device)[:, None].expand(rows, chunks),
         torch.full((rows, chunks), sid, dtype=torch.int64, device=device),
         torch.full((rows, chunks), TAG, dtype=torch.int64, device=device))
    for r in range(10):
        key = ((seed & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF, ((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF
        c = _philox_round(c, key)
    w = torch.stack(c, -1)
    h = torch.stack((w & 0xFFFF, w >> 16), -1).reshape(rows, chunks * 8)[:, :cols]
    return h >= _threshold(p)


def _threshold(p):
    return int(math.floor(65536.0 * p + 0.5))


def _drop_scale(p):
    t = _threshold(p)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def _dropped(x, gate, p, seed, sid):
    """The dropout of x (and of the ReLU whose output `gate` is), unrounded."""
    y = x
    if p > 0:
        scale = torch.tensor(_drop_scale(p), dtype=x.dtype, device=x.device)
        y = torch.where(_keep(*x.shape, p, seed, sid, x.device), x * scale, torch.zeros_like(x))
    return y if gate is None else torch.where(gate > 0, y, torch.zeros_like(y))


def _power(e):
    """2^e in 32 bits, exactly (e from -127 to 127)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantized(x):
    """Rows of x in blocks of 32: elements (as their values) and scale codes."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    v = torch.nn.functional.pad(x, (0, nb * 32 - cols)).reshape(rows, nb, 32)
    top = v.abs().amax(-1)
    code = (torch.frexp(top)[1] + 124).clamp(0, 254)  # frexp's exponent is floor(log2) + 1
    code = torch.where(top == 0, 0, code)
    code = torch.where(torch.isfinite(top), code, 255)
    v = v * _power(127 - code)[..., None]
    a = v.abs()
    q = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
    return torch.copysign(q.clamp(max=6.0), v), code


def _values(q, code, cols):
    s = torch.where(code == 255, math.nan, _power((code - 127).clamp(max=127)))
    return (q * s[..., None]).reshape(q.shape[0], -1)[:, :cols]


def _unpack(P, S, rows, cols):
    """The values an MXFP4 matrix stands for, in 32 bits."""
    nb = -(-cols // 32)
    n = torch.stack((P & 15, P >> 4), -1).reshape(rows, nb, 32).to(torch.int32)
    e, f = (n >> 1) & 3, (n & 1).float()
    a = torch.where(e == 0, f * 0.5, (1 + 0.5 * f) * _power(e - 1))
    q = torch.where(n >= 8, -a, a)
    code = S.permute(1, 0, 2).reshape(rows, -1)[:, :nb].to(torch.int32)
    return _values(q, code, cols)


def _fake(x):
    """x to MXFP4 and back."""
    q, code = _quantized(x)
    return _values(q, code, x.shape[1])


# ---- inputs ------------------------------------------------------------------


def _pack(x):
    """An MXFP4 matrix as a program holds it: packed elements and scales."""
    q, code = _quantized(x)
    rows, nb = code.shape
    a = q.abs()
    n = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    n = n | (torch.signbit(q).to(torch.uint8) << 3)
    n = n.reshape(rows, nb * 16, 2)
    P = (n[..., 0] | (n[..., 1] << 4)).contiguous()
    S = torch.nn.functional.pad(code.to(torch.uint8), (0, -nb % 8)).reshape(rows, -1, 8).permute(1, 0, 2).contiguous()
    return P, S


def _room(rows, cols):
    """Memory for an MXFP4 matrix."""
    nb = -(-cols // 32)
    return (torch.empty((rows, nb * 16), dtype=torch.uint8, device="cuda"),
            torch.empty((-(-nb // 8), rows, 8), dtype=torch.uint8, device="cuda"))


def prepare(case, seed):
    """Activations are normal with a few large columns, weights normal with
    variance 1 / terms, gradients small; operands that a layer keeps quantised
    are packed.  Results go to memory that the program keeps."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dt = case["op"], TORCH[case["dtype"]]

    def normal(rows, cols, scale=1.0, loud=False):
        t = torch.randn((rows, cols), generator=gen, device="cuda") * scale
        if loud:
            t *= torch.where(torch.rand((1, cols), generator=gen, device="cuda") < 0.01, 8.0, 1.0)
        return t

    def empty(rows, cols, dtype=dt):
        return torch.empty((rows, cols), dtype=dtype, device="cuda")

    s = {"case": case, "seed": 0x5EED0000000 + int(seed) * 2654435761 % (1 << 40), "sid": int(seed) % 1000}
    if op in ("dropout", "quantize"):
        rows, cols, ld = case["rows"], case["cols"], case["cols"] + case["pad"]
        grad = case["gate"]
        s["x"] = normal(rows, ld, 1e-3 if grad else 1.0, loud=not grad).to(dt)[:, :cols]
        s["gate"] = normal(rows, ld).clamp_min(0.0).to(dt)[:, :cols] if grad else None
        if op == "dropout":
            s["y"] = empty(rows, cols)
        else:
            s["P"], s["S"] = _room(rows, cols)
            s["PT"], s["ST"] = _room(cols, rows)
            s["y"], s["yt"] = empty(rows, cols), empty(cols, rows)
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["A"], s["SA"] = _pack(normal(m, k, loud=True))
        s["B"], s["SB"] = _pack(normal(n, k, k ** -0.5))
        s["C"] = normal(m, n).to(dt)
        s["out"] = empty(m, n)
    elif op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = normal(m, k, loud=True).to(dt)
        s["B"], s["SB"] = _pack(normal(n, k, k ** -0.5))
        s["A"], s["SA"] = _room(m, k)
        s["y"] = empty(m, n)
    else:
        t, d, h = case["tokens"], case["width"], case["hidden"]
        s["x"] = normal(t, d, loud=True).to(dt)
        s["dy"] = normal(t, d, 1e-3).to(dt)
        s["w1"], s["w2"] = normal(h, d, d ** -0.5).to(dt), normal(d, h, h ** -0.5).to(dt)
        s["h"], s["dd"] = empty(t, h), empty(t, h)
        s["y"], s["dx"] = empty(t, d), empty(t, d)
        s["dw1"], s["dw2"] = empty(h, d, torch.float32), empty(d, h, torch.float32)
        for name, rows, cols in (("x", t, d), ("dy", t, d), ("w1", h, d), ("w2", d, h), ("h", t, h), ("dd", t, h)):
            s["q_" + name] = _room(rows, cols) + _room(cols, rows)
    return s


# ---- one pass ----------------------------------------------------------------


def _run_plain(s):
    c, dt = s["case"], TORCH[s["case"]["dtype"]]
    op = c["op"]
    if op == "dropout":
        x = s["x"] if c["dtype"] == F64 else s["x"].float()
        return _dropped(x, s["gate"], c["p"], s["seed"], s["sid"]).to(dt)
    if op == "quantize":
        v = _dropped(s["x"].float(), s["gate"], c["p"], s["seed"], s["sid"])
        return _fake(v).to(dt), _fake(v.t()).to(dt)
    if op == "product":
        y = c["alpha"] * (_unpack(s["A"], s["SA"], c["m"], c["k"]) @ _unpack(s["B"], s["SB"], c["n"], c["k"]).t())
        if c["beta"] != 0:
            y = y + c["beta"] * s["C"].float()
        return (y.clamp_min(0.0) if c["relu"] else y).to(dt)
    if op == "linear":
        y = _fake(s["x"].float()) @ _unpack(s["B"], s["SB"], c["n"], c["k"]).t()
        return (y.clamp_min(0.0) if c["relu"] else y).to(dt)
    x, dy, w1, w2 = (s[n].float() for n in ("x", "dy", "w1", "w2"))
    h = (_fake(x) @ _fake(w1).t()).clamp_min(0.0).to(dt)
    d = _dropped(h.float(), None, c["p"], s["seed"], s["sid"])
    y = _fake(d) @ _fake(w2).t()
    dd = (_fake(dy) @ _fake(w2.t()).t()).to(dt)
    dz = _dropped(dd.float(), h, c["p"], s["seed"], s["sid"])
    dx = _fake(dz) @ _fake(w1.t()).t()
    dw1 = _fake(dz.t()) @ _fake(x.t()).t()
    dw2 = _fake(dy.t()) @ _fake(d.t()).t()
    return {"y": y.to(dt), "dx": dx.to(dt), "dw1": dw1, "dw2": dw2}


def _run_own(s):
    import sushiblas_amd as sbx

    c = s["case"]
    code = {F32: sbx.F32, F64: sbx.F64, BF16: sbx.BF16, F16: sbx.F16}[c["dtype"]]
    op = c["op"]

    def quantize(x, P, S, PT=None, ST=None, p=0.0, gate=None):
        sbx.mx4_quantize(code, x.shape[0], x.shape[1], x, x.stride(0), P, P.stride(0), S, S.stride(0),
                         PT, 0 if PT is None else PT.stride(0), ST, 0 if ST is None else ST.stride(0),
                         p=p, seed=s["seed"], stream_id=s["sid"], gate=gate,
                         ldg=0 if gate is None else gate.stride(0))

    def product(dtype, A, SA, B, SB, C, k, alpha=1.0, beta=0.0, relu=0):
        sbx.mx4_gemm(dtype, 0, C.shape[0], C.shape[1], k, alpha, A, A.stride(0), SA, SA.stride(0), B, B.stride(0),
                     SB, SB.stride(0), beta, C, C.stride(0),
                     epilogue=sbx.EPILOGUE_RELU if relu else sbx.EPILOGUE_NONE)

    if op == "dropout":
        x, y, gate = s["x"], s["y"], s["gate"]
        sbx.dropout(code, c["rows"], c["cols"], x, x.stride(0), y, y.stride(0), c["p"], s["seed"], s["sid"],
                    gate=gate, ldg=0 if gate is None else gate.stride(0))
        return y
    if op == "quantize":
        quantize(s["x"], s["P"], s["S"], s["PT"], s["ST"], c["p"], s["gate"])
        for P, S, y in ((s["P"], s["S"], s["y"]), (s["PT"], s["ST"], s["yt"])):
            sbx.mx4_dequantize(code, y.shape[0], y.shape[1], P, P.stride(0), S, S.stride(0), y, y.stride(0))
        return s["y"], s["yt"]
    if op == "product":
        out = s["out"]
        if c["beta"] != 0:  # accumulates; C stays as it is for the next pass
            out.copy_(s["C"])
        product(code, s["A"], s["SA"], s["B"], s["SB"], out, c["k"], c["alpha"], c["beta"], c["relu"])
        return out
    if op == "linear":
        quantize(s["x"], s["A"], s["SA"])
        product(code, s["A"], s["SA"], s["B"], s["SB"], s["y"], c["k"], relu=c["relu"])
        return s["y"]
    t, d, h = c["tokens"], c["width"], c["hidden"]
    quantize(s["x"], *s["q_x"])
    quantize(s["w1"], *s["q_w1"])
    quantize(s["w2"], *s["q_w2"])
    product(code, *s["q_x"][:2], *s["q_w1"][:2], s["h"], d, relu=1)
    quantize(s["h"], *s["q_h"], p=c["p"])
    product(code, *s["q_h"][:2], *s["q_w2"][:2], s["y"], h)
    quantize(s["dy"], *s["q_dy"])
    product(code, *s["q_dy"][:2], *s["q_w2"][2:], s["dd"], d)
    product(sbx.F32, *s["q_dy"][2:], *s["q_h"][2:], s["dw2"], t)
    quantize(s["dd"], *s["q_dd"], p=c["p"], gate=s["h"])
    product(code, *s["q_dd"][:2], *s["q_w1"][2:], s["dx"], h)
    product(sbx.F32, *s["q_dd"][2:], *s["q_x"][2:], s["dw1"], t)
    return {"y": s["y"], "dx": s["dx"], "dw1": s["dw1"], "dw2": s["dw2"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- 64 bits -----------------------------------------------------------------


def _exact_keep(rows, cols, p, seed, sid):
    """The generator once more, its products from 16-bit halves."""
    def mul(a, m):
        al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
        mid = al * mh + ((al * ml) >> 16)
        up = ah * ml + (mid & 0xFFFF)
        return ah * mh + (mid >> 16) + (up >> 16), ((up & 0xFFFF) << 16) | ((al * ml) & 0xFFFF)

    n = -(-cols // 8)
    zero = torch.zeros((rows, n), dtype=torch.int64, device="cuda")
    x = [zero + torch.arange(n, device="cuda"), zero + torch.arange(rows, device="cuda")[:, None], zero + sid, zero + TAG]
    k = [seed % (1 << 32), seed // (1 << 32) % (1 << 32)]
    for _ in range(10):
        h0, l0 = mul(x[0], 0xD2511F53)
        h1, l1 = mul(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ k[0], l1, h0 ^ x[3] ^ k[1], l0]
        k = [(k[0] + 0x9E3779B9) % (1 << 32), (k[1] + 0xBB67AE85) % (1 << 32)]
    bits = torch.empty((rows, n, 8), dtype=torch.int64, device="cuda")
    for w in range(4):
        bits[..., 2 * w] = x[w] % 65536
        bits[..., 2 * w + 1] = x[w] // 65536
    return bits.reshape(rows, n * 8)[:, :cols] >= round(p * 65536)


def _exact_drop(x, gate, p, seed, sid, single):
    """In 64 bits; `single`: what goes on to the quantiser is the product in 32."""
    y = x.double()
    if p > 0:
        scale = 65536.0 / (65536 - round(p * 65536))
        if single:
            scale = float(torch.tensor(scale, dtype=torch.float32))
        y = y * scale
        if single:
            y = y.float().double()
        y = y * _exact_keep(*x.shape, p, seed, sid)
    return y if gate is None else y * (gate > 0)


def _exact_fake(x):
    """To MXFP4 and back by the midpoints between the eight magnitudes."""
    rows, cols = x.shape
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    mids = (grid[1:] + grid[:-1]) / 2
    out = torch.empty_like(x)
    whole = cols // 32 * 32
    for part, width in ((slice(0, whole), 32), (slice(whole, cols), cols - whole)):
        if part.start == part.stop:
            continue
        v = x[:, part].reshape(rows, -1, width)
        top = v.abs().amax(-1, keepdim=True)
        e = ((top.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127)
        scale = ((e + 1023) << 52).view(torch.float64)
        a = v.abs() / scale
        low, high = torch.bucketize(a, mids), torch.bucketize(a, mids, right=True)
        q = grid[torch.where(low % 2 == 1, high, low)]  # a tie goes to the even code
        out[:, part] = (q * torch.sign(v) * scale).reshape(rows, -1)
    return out


def _exact_unpack(P, S, rows, cols):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=P.device)
    table = torch.cat((table, -table))
    v = torch.empty((rows, P.shape[1] * 2), dtype=torch.float64, device=P.device)
    v[:, 0::2], v[:, 1::2] = table[(P % 16).long()], table[(P // 16).long()]
    b = torch.arange(cols, device=P.device) // 32
    r = torch.arange(rows, device=P.device)[:, None]
    return v[:, :cols] * ((S[b // 8, r, b % 8].long() + 896) << 52).view(torch.float64)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "dropout":
        return _exact_drop(s["x"], s["gate"], case["p"], s["seed"], s["sid"], False)
    if op == "quantize":
        v = _exact_drop(s["x"], s["gate"], case["p"], s["seed"], s["sid"], True)
        return _exact_fake(v), _exact_fake(v.t().contiguous())
    if op == "product":
        y = case["alpha"] * (_exact_unpack(s["A"], s["SA"], case["m"], case["k"]) @
                             _exact_unpack(s["B"], s["SB"], case["n"], case["k"]).t())
        y = y + case["beta"] * s["C"].double()
        return y.relu() if case["relu"] else y
    if op == "linear":
        y = _exact_fake(s["x"].double()) @ _exact_unpack(s["B"], s["SB"], case["n"], case["k"]).t()
        return y.relu() if case["relu"] else y
    # the block's two inner matrices, like the tensors they are, hold the case's type
    dt = TORCH[case["dtype"]]
    x, dy, w1, w2 = (s[n].double() for n in ("x", "dy", "w1", "w2"))
    turn = lambda a: a.t().contiguous()  # noqa: E731
    h = (_exact_fake(x) @ _exact_fake(w1).t()).relu().to(dt)
    d = _exact_drop(h, None, case["p"], s["seed"], s["sid"], True)
    dd = (_exact_fake(dy) @ _exact_fake(turn(w2)).t()).to(dt)
    dz = _exact_drop(dd, h, case["p"], s["seed"], s["sid"], True)
    return {"y": _exact_fake(d) @ _exact_fake(w2).t(), "dx": _exact_fake(dz) @ _exact_fake(turn(w1)).t(),
            "dw1": _exact_fake(turn(dz)) @ _exact_fake(turn(x)).t(),
            "dw2": _exact_fake(turn(dy)) @ _exact_fake(turn(d)).t()}
