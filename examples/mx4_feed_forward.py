"""Training a feed-forward block whose products run in MXFP4.

    Y = dropout(relu(X W1^T)) W2^T,   trained to a random target

All six products of a step (two forward, four backward) are sbx.mx4_gemm on
operands that sbx.mx4_quantize lays out along the axis each product sums over.
The dropout, and in the backward pass the ReLU's gradient with it, happen inside
the quantiser: neither a mask nor a dropped matrix is ever stored.  Weights are
kept in 32 bits and quantised anew each step.  Afterwards the trained block is
run for single tokens, with its weights quantised once.

    python examples/mx4_feed_forward.py            (needs the GPU)
"""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import sushiblas_amd as sbx  # noqa: E402

CODE = {torch.float32: sbx.F32, torch.bfloat16: sbx.BF16, torch.float16: sbx.F16}


class Mx4:
    """A matrix in MXFP4 along its rows (P, S), and of its transpose (PT, ST)."""

    def __init__(self, rows, cols, turned=True, device="cuda"):
        new = lambda shape: torch.empty(shape, dtype=torch.uint8, device=device)  # noqa: E731
        self.rows, self.cols = rows, cols
        self.P, self.S = (new(s) for s in sbx.mx4_shapes(rows, cols))
        self.PT, self.ST = (new(s) for s in sbx.mx4_shapes(cols, rows)) if turned else (None, None)

    def set(self, x, p=0.0, seed=0, stream_id=0, gate=None):
        """Quantise x, after dropout with probability p and, with a gate, where that is > 0."""
        ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
        sbx.mx4_quantize(CODE[x.dtype], self.rows, self.cols, x, x.stride(0), self.P, ld(self.P), self.S, ld(self.S),
                         self.PT, ld(self.PT), self.ST, ld(self.ST), p=p, seed=seed, stream_id=stream_id,
                         gate=gate, ldg=ld(gate))
        return self

    @property
    def along_rows(self):
        return self.P, self.S

    @property
    def along_columns(self):
        return self.PT, self.ST


def product(a, b, terms, out, relu=False):
    """out = a b^T over `terms` terms; a, b: (P, S) of matrices quantised along them."""
    (A, SA), (B, SB) = a, b
    sbx.mx4_gemm(CODE[out.dtype], 0, out.shape[0], out.shape[1], terms, 1.0, A, A.stride(0), SA, SA.stride(0), B,
                 B.stride(0), SB, SB.stride(0), 0.0, out, out.stride(0),
                 epilogue=sbx.EPILOGUE_RELU if relu else sbx.EPILOGUE_NONE)
    return out


class FeedForward:
    """The block for a fixed number of tokens; everything it needs is allocated here."""

    def __init__(self, tokens, width, hidden, p=0.1, seed=1, dtype=torch.bfloat16, device="cuda"):
        self.tokens, self.width, self.hidden, self.p, self.seed = tokens, width, hidden, p, seed
        gen = torch.Generator().manual_seed(seed)
        self.w1 = (torch.randn((hidden, width), generator=gen) * width ** -0.5).to(device)
        self.w2 = (torch.randn((width, hidden), generator=gen) * hidden ** -0.5).to(device)
        new = lambda r, c, t=dtype: torch.empty((r, c), dtype=t, device=device)  # noqa: E731
        self.h, self.dd = new(tokens, hidden), new(tokens, hidden)
        self.y, self.dx = new(tokens, width), new(tokens, width)
        self.dw1, self.dw2 = new(hidden, width, torch.float32), new(width, hidden, torch.float32)
        self.qx, self.qy = Mx4(tokens, width, device=device), Mx4(tokens, width, device=device)
        self.qh, self.qd = Mx4(tokens, hidden, device=device), Mx4(tokens, hidden, device=device)
        self.q1, self.q2 = Mx4(hidden, width, device=device), Mx4(width, hidden, device=device)

    def forward(self, x, step=0):
        """step selects the dropout's mask."""
        self.step = step
        self.qx.set(x)
        self.q1.set(self.w1)
        self.q2.set(self.w2)
        product(self.qx.along_rows, self.q1.along_rows, self.width, self.h, relu=True)
        self.qh.set(self.h, self.p, self.seed, step)
        return product(self.qh.along_rows, self.q2.along_rows, self.hidden, self.y)

    def backward(self, dy):
        self.qy.set(dy)
        product(self.qy.along_rows, self.q2.along_columns, self.width, self.dd)
        product(self.qy.along_columns, self.qh.along_columns, self.tokens, self.dw2)
        # the same mask again, and the ReLU's gradient: where its output was not 0
        self.qd.set(self.dd, self.p, self.seed, self.step, gate=self.h)
        product(self.qd.along_rows, self.q1.along_columns, self.hidden, self.dx)
        product(self.qd.along_columns, self.qx.along_columns, self.tokens, self.dw1)
        return self.dx


class Server:
    """The trained block for a few tokens at a time: no dropout, weights quantised once."""

    def __init__(self, block, dtype=torch.bfloat16):
        self.dtype = dtype
        self.q1 = Mx4(block.hidden, block.width, turned=False).set(block.w1)
        self.q2 = Mx4(block.width, block.hidden, turned=False).set(block.w2)

    def __call__(self, x):
        tokens, width, hidden = x.shape[0], self.q2.rows, self.q1.rows
        h = torch.empty((tokens, hidden), dtype=self.dtype, device=x.device)
        y = torch.empty((tokens, width), dtype=self.dtype, device=x.device)
        product(Mx4(tokens, width, turned=False).set(x).along_rows, self.q1.along_rows, width, h, relu=True)
        return product(Mx4(tokens, hidden, turned=False).set(h).along_rows, self.q2.along_rows, hidden, y)


def main(tokens=512, width=256, hidden=1024, steps=200, rate=0.004):
    gen = torch.Generator().manual_seed(7)
    x = torch.randn((tokens, width), generator=gen).bfloat16().cuda()
    target = torch.randn((tokens, width), generator=gen).cuda()
    block = FeedForward(tokens, width, hidden)
    first = last = None
    for step in range(steps):
        y = block.forward(x, step)
        error = y.float() - target
        last = float(error.square().mean())
        first = last if first is None else first
        block.backward((error * (2.0 / error.shape[0])).bfloat16())
        block.w1 -= rate * block.dw1
        block.w2 -= rate * block.dw2
        if step % 20 == 0 or step == steps - 1:
            print(f"step {step:4d}  mean squared error {last:.4f}", flush=True)
    served = Server(block)
    one = torch.cat([served(x[i:i + 1]) for i in range(4)])
    batch = served(x[:4])
    same = torch.equal(one, batch)
    print("single tokens and a batch of them:", "the same" if same else "DIFFERENT", flush=True)
    return first, last, same


if __name__ == "__main__":
    main()
