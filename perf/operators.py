"""The operators at the two ends of a decoder's training step and of what it keeps between forward and backward, as cases that can be
timed and checked: the embedding lookup with its gradient by sorted tokens, the per-token loss over pieces of the vocabulary with its gradient,
activations held in 8 bits, and the gated activation that keeps its input so. Widths and vocabularies are those of the presets
(``models/config.py``); token counts run from one decode step to a training batch.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32          # values that share one exponent


def listed():
    return [
        # one decode step of 64 served sequences: 64 rows of the Llama-3 8B table, bound by the launch
        dict(name="embed_step", kind="embed", train=False, tokens=64, vocab=128256, width=4096, dtype="bf16", scale=1.0, pad=0.0, into=""),
        # a ragged prompt batch of a model that scales its embeddings by the root of the width, in fp16
        dict(name="embed_prompts", kind="embed", train=False, tokens=5003, vocab=32000, width=4096, dtype="fp16", scale=64.0, pad=0.0, into=""),
        # a training batch of the Llama-3 8B shape, a tenth of it padding: the dense gradient of the table is written once
        dict(name="embed_train_8b", kind="embed", train=True, tokens=8192, vocab=128256, width=4096, dtype="bf16", scale=1.0, pad=0.1, into=""),
        # tied table of the DeepSeek-V2-Lite shape: the lookup's gradient is added to the fp32 gradient that the head has already written
        dict(name="embed_tied", kind="embed", train=True, tokens=32768, vocab=102400, width=2048, dtype="bf16", scale=1.0, pad=0.0, into="fp32"),
        # the log-probabilities of one short reply under the small hybrid model: bound by launches
        dict(name="score_reply", kind="loss", train=False, tokens=77, vocab=32000, width=256, softcap=0.0, ignored=0.0),
        # a preference pair batch scored by the frozen reference model: 8 replies of 511 tokens, Llama-3 8B head
        dict(name="score_8b", kind="loss", train=False, tokens=4088, vocab=128256, width=4096, softcap=0.0, ignored=0.3),
        # training of the 130M Mamba-2 preset with soft-capped logits, an odd number of tokens and a vocabulary that no tile divides
        dict(name="loss_130m", kind="loss", train=True, tokens=4095, vocab=50280, width=768, softcap=30.0, ignored=0.05),
        # policy training on the Llama-3 8B head: per-token losses with their own weights, and the head's gradient
        dict(name="loss_8b", kind="loss", train=True, tokens=8192, vocab=128256, width=4096, softcap=0.0, ignored=0.05),
        # a short fp32 batch whose width is no multiple of the block
        dict(name="pack_odd", kind="pack", rows=77, width=500, dtype="fp32"),
        # the input of one Llama-3 8B layer for 16384 tokens, packed after forward and restored in backward
        dict(name="pack_layer", kind="pack", rows=16384, width=4096, dtype="bf16"),
        # the MLP of the tiny preset on a short batch
        dict(name="glu_short", kind="glu", rows=154, width=1024, act="silu", dtype="bf16"),
        # the MLP of the Llama-3 8B shape on 8192 tokens
        dict(name="glu_8b", kind="glu", rows=8192, width=14336, act="silu", dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "loss", "pack", "glu"])
    if kind == "embed":
        train = rng.random() < 0.7
        vocab, width = _spread(rng, 500, 152064), rng.choice([_spread(rng, 33, 4096), 8 * _spread(rng, 8, 512)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        tokens = _spread(rng, 1, max(2, min(65536, 32768 * 2048 // width)))
        return dict(kind=kind, train=train, tokens=tokens, vocab=vocab, width=width, dtype=dtype, scale=rng.choice([1.0, math.sqrt(width)]),
                    pad=rng.choice([0.0, 0.1, 0.6]), into=rng.choice(["", "fp32"]) if train else "")
    if kind == "loss":
        return dict(kind=kind, train=rng.random() < 0.6, tokens=_spread(rng, 1, 8192), vocab=_spread(rng, 500, 128256), width=8 * _spread(rng, 8, 512),
                    softcap=rng.choice([0.0, 0.0, 30.0]), ignored=rng.choice([0.0, 0.05, 0.5]))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "pack":
        width = _spread(rng, 20, 16384)
        return dict(kind=kind, rows=_spread(rng, 1, 16384 * 4096 // max(width, 1024)), width=width, dtype=dtype)
    width = rng.choice([_spread(rng, 20, 14336), 8 * _spread(rng, 8, 1792)])
    return dict(kind=kind, rows=_spread(rng, 1, 8192), width=width, act=rng.choice(["silu", "gelu", "relu"]), dtype=dtype)


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.bfloat16, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).mul_(std).to(dtype)


def _law(vocab, device):
    """Word frequencies fall with the rank."""
    p = 1.0 / torch.arange(1, vocab + 1, device=device, dtype=torch.float64)
    return p / p.sum()


def _words(g, n, vocab):
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    rank = torch.searchsorted(_law(vocab, DEV).cumsum(0), u).clamp_(max=vocab - 1)
    step = next(s for s in (7919, 7907, 7901, 1) if math.gcd(s, vocab) == 1)       # frequent words all over the table
    return (rank * step + 1) % vocab                # word 0 is a rare one


def _embed_inputs(case, seed):
    g = _gen(seed)
    n, vocab, width, dtype = case["tokens"], case["vocab"], case["width"], TYPES[case["dtype"]]
    table = _normal(g, vocab, width, dtype=dtype, std=0.02)
    ids = _words(g, n, vocab)
    if case["pad"]:
        ids[n - int(n * case["pad"]):] = 0          # a padded batch: word 0 is the padding
    dy = _normal(g, n, width, dtype=dtype) if case["train"] else None
    grad = _normal(g, vocab, width, dtype=torch.float32) if case["into"] else None
    return table, ids, dy, grad


def _loss_inputs(case, seed):
    g = _gen(seed)
    n, vocab, width = case["tokens"], case["vocab"], case["width"]
    w = _normal(g, vocab, width, std=1.0 / math.sqrt(width))
    target = _words(g, n, vocab)
    # from tokens that the model is sure of to tokens that it knows nothing about
    sure = 14.0 * torch.rand(n, 1, generator=g, device=DEV)
    h = (torch.randn(n, width, generator=g, device=DEV) + sure * w[target].float()).to(torch.bfloat16)
    gn, gz = _normal(g, n, dtype=torch.float32), _normal(g, n, dtype=torch.float32, std=0.1)
    target = torch.where(torch.rand(n, generator=g, device=DEV) < case["ignored"], -100, target)
    return h, w, target, gn, gz


def _glu_inputs(case, seed):
    g = _gen(seed)
    dtype = TYPES[case["dtype"]]
    return _normal(g, case["rows"], 2 * case["width"], dtype=dtype, std=1.5), _normal(g, case["rows"], case["width"], dtype=dtype)


def _pack_inputs(case, seed):
    """Activations of a residual stream: channels of very different size, a few of them huge."""
    g = _gen(seed)
    size = torch.exp(1.5 * torch.randn(case["width"], generator=g, device=DEV))
    return torch.randn(case["rows"], case["width"], generator=g, device=DEV).mul_(size).to(TYPES[case["dtype"]])


def prepare(case, seed):
    kind = case["kind"]
    if kind == "embed":
        table, ids, dy, grad = _embed_inputs(case, seed)
        table.requires_grad_(case["train"])
        if grad is not None:            # a training engine's gradient buffer, which the output projection has written already
            table.main_grad, table._main_grad_written = grad, True
        return dict(case=case, table=table, ids=ids, dy=dy, grad=grad)
    if kind == "loss":
        h, w, target, gn, gz = _loss_inputs(case, seed)
        return dict(case=case, h=h.requires_grad_(case["train"]), w=w.requires_grad_(case["train"]), target=target, gn=gn, gz=gz)
    if kind == "pack":
        return dict(case=case, x=_pack_inputs(case, seed))
    gu, dh = _glu_inputs(case, seed)
    return dict(case=case, gu=gu.requires_grad_(), dh=dh)


# ----------------------------------------------------------------------------- one pass: the framework's operators
def _own(s):
    from sneppx_alg_b200 import ops
    case = s["case"]
    kind = case["kind"]
    if kind == "embed":
        y = ops.embedding(s["ids"], s["table"], scale=case["scale"], padding_idx=0 if case["pad"] else None)
        if not case["train"]:
            return dict(y=y)
        (g,) = torch.autograd.grad(y, s["table"], s["dy"], allow_unused=True)
        return dict(y=y, grad=s["grad"] if case["into"] else g)
    if kind == "loss":
        nll, lse = ops.linear_token_loss(s["h"], s["w"], s["target"], softcap=case["softcap"])
        if not case["train"]:
            return dict(nll=nll, lse=lse)
        dh, dw = torch.autograd.grad((nll, lse), (s["h"], s["w"]), (s["gn"], s["gz"]))
        return dict(nll=nll, lse=lse, dh=dh, dw=dw)
    if kind == "pack":
        return dict(x=ops.unpack_8bit(ops.pack_8bit(s["x"])))
    h = ops.glu_8bit(s["gu"], case["act"])
    (dgu,) = torch.autograd.grad(h, s["gu"], s["dh"])
    return dict(h=h, dgu=dgu)


# ----------------------------------------------------------------------------- one pass: the plain form
def _plain_embed(s):
    case, ids, dtype = s["case"], s["ids"], s["table"].dtype
    y = (s["table"][ids].float() * case["scale"]).to(dtype)
    if not case["train"]:
        return dict(y=y)
    dy = s["dy"].float() * case["scale"]
    if case["pad"]:
        dy = dy * (ids != 0)[:, None]
    if case["into"]:
        return dict(y=y, grad=s["grad"].index_add_(0, ids, dy))
    return dict(y=y, grad=torch.zeros(s["table"].shape, dtype=torch.float32, device=dy.device).index_add_(0, ids, dy).to(dtype))


def _plain_loss(s):
    case, cap, target = s["case"], s["case"]["softcap"], s["target"]
    h, w = s["h"].float(), s["w"].float()
    z = h @ w.t()
    if cap:
        z = z.div_(cap).tanh_().mul_(cap)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    valid = target != -100
    at = target.clamp(min=0)[:, None]
    nll = torch.where(valid, lse - z.gather(1, at).squeeze(1), 0.0)
    if not case["train"]:
        return dict(nll=nll, lse=lse)
    gn = torch.where(valid, s["gn"], 0.0)[:, None]
    d = e.div_(total).mul_(gn + s["gz"][:, None]).scatter_add_(1, at, -gn)
    if cap:
        d = d.mul_(1 - (z / cap) ** 2)
    return dict(nll=nll, lse=lse, dh=(d @ w).to(torch.bfloat16), dw=(d.t() @ h).to(torch.bfloat16))


def _restored(x):
    """What 8 bits hold of x, in 32 bits: per 32 values of a row whole multiples, up to 127, of a power of two."""
    rows, width = x.shape
    n = -(-width // BLOCK) * BLOCK
    b = torch.zeros(rows, n, dtype=torch.float32, device=x.device)
    b[:, :width] = x.float()
    b = b.view(rows, -1, BLOCK)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))                       # amax = m 2^e, m in [1/2, 1)
    e = torch.clamp(e - 7 + (m * 128 >= 127.5).int(), min=-126)              # round(amax / 2^e) <= 127
    step = torch.ldexp(torch.ones_like(m), e)
    return ((b / step).round_() * step).view(rows, n)[:, :width]


def _plain_glu(s):
    case = s["case"]
    f, dtype = case["width"], s["gu"].dtype
    gu = s["gu"].detach()
    g, u = gu[:, :f].float(), gu[:, f:].float()
    h = (_act(g, case["act"]) * u).to(dtype)
    g, u, dh = _restored(gu[:, :f]), _restored(gu[:, f:]), s["dh"].float()
    return dict(h=h, dgu=torch.cat([dh * u * _slope(g, case["act"]), dh * _act(g, case["act"])], 1).to(dtype))


def _act(g, act):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    if act == "relu":
        return g * (g > 0)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _slope(g, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return s * (1 + g * (1 - s))
    if act == "relu":
        return (g > 0).to(g.dtype)
    t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))
    return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)


@torch.no_grad()
def _plain(s):
    kind = s["case"]["kind"]
    if kind == "embed":
        return _plain_embed(s)
    if kind == "loss":
        return _plain_loss(s)
    if kind == "pack":
        return dict(x=_restored(s["x"]).to(s["x"].dtype))
    return _plain_glu(s)


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "embed":
        e, n, vocab, width = TYPES[case["dtype"]].itemsize, case["tokens"], case["vocab"], case["width"]
        real = n - int(n * case["pad"])
        rows = float((1 - (1 - _law(vocab, "cpu")) ** real).sum())          # distinct words to be expected
        total = 8 * n + rows * width * e + n * width * e
        if case["train"]:           # the gradient of the rows; the words' sums, added to a buffer or written among zeros
            total += real * width * e + (2 * rows * width * 4 if case["into"] else vocab * width * e)
        return dict(bytes=total, flops=n * width * (2 if case["train"] else 1))
    if kind == "loss":
        n, vocab, width = case["tokens"], case["vocab"], case["width"]
        total = 2 * (n * width + vocab * width) + 8 * n + 8 * n
        if case["train"]:
            total += 2 * (n * width + vocab * width) + 8 * n
        return dict(bytes=total, flops=2 * n * vocab * width * (3 if case["train"] else 1))
    e, n = TYPES[case["dtype"]].itemsize, case["rows"] * case["width"]
    if kind == "pack":          # read, held, read again, written
        return dict(bytes=2 * n * e + 2 * n * (1 + 1 / BLOCK), flops=4 * n)
    return dict(bytes=2 * n * e + n * e + n * e + 2 * n * e + 4 * n * (1 + 1 / BLOCK), flops=30 * n)


# ----------------------------------------------------------------------------- the definition in 64 bits
def _exact_embed(case, seed):
    table, ids, dy, grad = _embed_inputs(case, seed)
    out = dict(y=torch.index_select(table, 0, ids).double().mul_(case["scale"]))
    if case["train"]:
        total = torch.zeros(table.shape, dtype=torch.float64, device=DEV) if grad is None else grad.double()
        keep = torch.nonzero(ids != 0).squeeze(1) if case["pad"] else torch.arange(ids.numel(), device=DEV)
        out["grad"] = total.index_put_((ids[keep],), dy[keep].double() * case["scale"], accumulate=True)
    return out


def _exact_loss(case, seed):
    h, w, target, gn, gz = _loss_inputs(case, seed)
    cap, wd = case["softcap"], w.double()
    nll, lse, dh, dw = [], [], [], torch.zeros_like(wd) if case["train"] else None
    for i in range(0, h.shape[0], 1024):
        hd, t = h[i:i + 1024].double(), target[i:i + 1024]
        raw = torch.mm(hd, wd.t())
        z = cap * torch.tanh(raw / cap) if cap else raw
        lse.append(torch.logsumexp(z, 1))
        ok = (t >= 0).double()
        row = torch.arange(t.numel(), device=DEV)
        nll.append((lse[-1] - z[row, t.clamp(min=0)]) * ok)
        if case["train"]:
            a = gn[i:i + 1024].double() * ok
            d = torch.softmax(z, 1) * (a + gz[i:i + 1024].double())[:, None]
            d[row, t.clamp(min=0)] -= a
            if cap:
                d /= torch.cosh(raw / cap) ** 2
            dh.append(torch.mm(d, wd))
            dw.addmm_(d.t(), hd)
    out = dict(nll=torch.cat(nll), lse=torch.cat(lse))
    if case["train"]:
        out.update(dh=torch.cat(dh), dw=dw)
    return out


def _held(x):
    """In 64 bits, by the smallest power of two of which 127 steps, and less than half a step more, reach the largest magnitude."""
    rows, width = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -width % BLOCK)).unflatten(1, (-1, BLOCK))
    top = x.abs().amax(2, keepdim=True)
    e = torch.ceil(torch.log2(top / 127.5))
    e = torch.where(top >= 127.5 * torch.exp2(e), e + 1, e)
    e = torch.where(top < 127.5 * torch.exp2(e - 1), e - 1, e)
    step = torch.exp2(e.clamp(min=-126))
    return (torch.round(x / step) * step).flatten(1)[:, :width]


def _exact_glu(case, seed):
    gu, dh = _glu_inputs(case, seed)
    h, dgu = [], []
    for i in range(0, gu.shape[0], 1024):
        g, u = gu[i:i + 1024].double().chunk(2, 1)
        h.append(_exact_act(g, case["act"])[0] * u)
        g, u = (_held(t) for t in gu[i:i + 1024].chunk(2, 1))
        a, da = _exact_act(g, case["act"])
        d = dh[i:i + 1024].double()
        dgu.append(torch.cat([d * u * da, d * a], 1))
    return dict(h=torch.cat(h), dgu=torch.cat(dgu))


def _exact_act(g, act):
    """Value and derivative."""
    with torch.enable_grad():
        x = g.clone().requires_grad_()
        a = dict(silu=lambda: x * torch.sigmoid(x), relu=lambda: torch.relu(x),
                 gelu=lambda: x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))[act]()
        (da,) = torch.autograd.grad(a.sum(), x)
    return a.detach(), da


@torch.no_grad()
def exact(case, seed):
    kind = case["kind"]
    if kind == "embed":
        return _exact_embed(case, seed)
    if kind == "loss":
        return _exact_loss(case, seed)
    if kind == "pack":
        return dict(x=_held(_pack_inputs(case, seed)))
    return _exact_glu(case, seed)
