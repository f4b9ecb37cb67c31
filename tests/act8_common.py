"""Definition of activations in 8 bits in 64-bit arithmetic, written apart from the operators."""
import math

import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def held(x):
    """[rows, width] of any float type -> what 8 bits hold of it, fp64. Row by row, block by block: the smallest e >= -126 with
    round(amax / 2^e) <= 127, values round(x / 2^e) 2^e with ties to even; a block with an infinity or a NaN is NaN."""
    out = torch.empty(x.shape, dtype=torch.float64)
    x = x.double().cpu()
    for i in range(0, x.shape[1], 32):
        b = x[:, i:i + 32]
        top = b.abs().amax(1)
        e = torch.full_like(top, -126.0)
        for r, t in enumerate(top.tolist()):
            if math.isfinite(t) and t > 0:
                n = math.frexp(t)[1] - 8                     # t < 2^(n + 8): at least 128 steps of 2^n or fewer
                while round(t / 2.0 ** n) > 127:             # Python rounds ties to even
                    n += 1
                e[r] = max(n, -126)
        step = torch.exp2(e)[:, None]
        out[:, i:i + 32] = torch.where(torch.isfinite(top)[:, None], torch.round(b / step) * step, torch.nan)
    return out


def gate(g, act):
    """Value and derivative of the gate's function in 64 bits."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s + g * s * (1 - s)
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return g * (1 + t) / 2, (1 + t) / 2 + g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g) / 2


def inputs(rows, width, dtype, seed, edge=True, device="cpu"):
    """Columns of different size, and rows of the values where rounding turns: zeros, ties, the border of the exponent, tiny and huge ones."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * torch.exp(2 * torch.randn(width, generator=g))
    if edge and rows >= 8:
        x[0] = 0
        x[1] = 127.5 * 2.0 ** -3                             # rounds to 128: the next exponent
        x[2, ::2] = 1.0
        x[2, 1::2] = 0.5                                     # halves of the maximum: 64 and 32 steps of it
        x[3] = torch.arange(width) % 255 - 127.0
        x[4] = (torch.arange(width) % 255 - 127.0) / 2 + 0.25
        x[5] *= 2.0 ** -110
        x[6, width // 2] = 60000.0
        x[7] = -1.9921875
    return x.to(TYPES[dtype]).to(device)


def largest(dtype):
    """Blocks whose largest magnitude is at the top of a type's range, and what 8 bits hold of them, fp64: 64 steps of the exponent that the border between
    127 and 128 steps asks for would be the type's infinity, so the steps are 2^-6 of the largest power of two and end at 127."""
    t = TYPES[dtype]
    top = torch.finfo(t).max
    power = 2.0 ** math.floor(math.log2(top / 1.5))
    eps = torch.finfo(t).eps
    x = torch.zeros(9, 32, dtype=torch.float64)
    x[0] = top
    x[1, 0] = -top
    x[2, 3], x[2, 4:] = top, torch.arange(28.0, dtype=torch.float64) * power / 64
    x[3, 31], x[3, 30] = power * (255 / 128), power * (255 / 128 - eps)        # the border and what is below it
    x[4, 0] = power * (255 / 128 - eps)                                        # just below: 127 steps, as ever
    x[5, 0] = power
    x[6, 0], x[6, 1] = -power * 1.5, top
    x[7, 0], x[7, 1] = top, 1.0
    x[8, 7] = -power * (255 / 128)
    x = x.to(t)
    step = power / 64
    return x, torch.round(x.double() / step).clamp(-127, 127) * step, step


def check_glu_of_overflows(glu, act, dtype, device, f):
    """An infinite and a NaN gate, and an infinite up: the result is NaN where the definition's is, and the gradients of a whole block are NaN where one of its
    gates or ups overflowed, as the block is held as NaN. Nothing else is."""
    x = inputs(9, 2 * f, dtype, 9, edge=False, device=device).clamp(-8, 8)
    x[1, 3], x[2, 5], x[3, f + 7], x[4, 0] = math.inf, math.nan, math.inf, -math.inf
    x = x.requires_grad_()
    h = glu(x, act)
    h.backward(torch.ones_like(h))
    g, u = x.detach().double()[:, :f], x.detach().double()[:, f:]
    a = torch.relu(g) if act == "relu" else gate(g, act)[0]
    nan = torch.isnan(a * u)
    assert not torch.isfinite(h[3, 7])               # an infinite up times a gate that 32 bits may hold as 0 and 64 do not: infinite or NaN
    nan[3, 7] = torch.isnan(h[3, 7])
    assert torch.equal(torch.isnan(h), nan)
    block = lambda r, c: (torch.arange(9)[:, None] == r) & (torch.arange(f)[None] // 32 == c // 32)  # noqa: E731
    gates, ups = block(1, 3) | block(2, 5) | block(4, 0), block(3, 7)
    bad = torch.isnan(x.grad).cpu()                 # dgate = d up act'(gate), dup = d act(gate); 0 times NaN is NaN
    assert torch.equal(bad[:, f:], gates)
    assert torch.equal(bad[:, :f], gates | ups)
