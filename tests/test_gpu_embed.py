"""Embedding lookup and its gradient on the GPU against sums in 64 bits."""
import math

import pytest
import torch

from sneppx_alg_b200 import ops
from sneppx_alg_b200.ops._lib import KernelTimeout

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _ids(n, V, law, seed):
    g = torch.Generator().manual_seed(seed)
    if law == "one":
        return torch.full((n,), V // 2)
    if law == "few":
        return torch.randint(0, min(V, 3), (n,), generator=g) * max(1, (V - 1) // 3)
    if law == "skew":
        return (V * torch.rand(n, generator=g) ** 6).long().clamp(max=V - 1)
    return torch.randint(0, V, (n,), generator=g)


def _sums(ids, dy, V, scale, padding=None):
    """64-bit sums by word, and the sums of magnitudes that bound their rounding."""
    keep = ids != padding if padding is not None else torch.ones_like(ids, dtype=torch.bool)
    out, mag = (torch.zeros(V, dy.shape[-1], dtype=torch.float64, device=dy.device) for _ in range(2))
    d = dy[keep].double() * scale
    return out.index_add_(0, ids[keep], d), mag.index_add_(0, ids[keep], d.abs())


def _close(got, want, mag, dtype, n):
    """One rounding to the gradient's type; before it a sum of up to n terms in 32 bits and a product: n + 2 roundings of at most 2^-24 of the magnitudes
    (2^-25: the smallest step of fp16)."""
    assert ((got.double() - want).abs() <= _half(dtype) * want.abs() + (n + 2) * 2.0 ** -24 * mag + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 500, 8), (77, 300, 33), (64, 32000, 512), (513, 1000, 4096), (300, 70, 5003)])
@pytest.mark.parametrize("scale", [1.0, 22.5])
def test_lookup(n, V, d, scale, dtype):
    torch.manual_seed(0)
    w = torch.randn(V, d, device="cuda").to(TYPES[dtype])
    for ids in (_ids(n, V, "any", 1).cuda(), _ids(n, V, "one", 1).cuda().int()):
        y = ops.embedding(ids, w, scale)
        # the product in 32 bits is exact for 16-bit tables up to its one rounding
        want = w[ids.long()] if scale == 1.0 else (w[ids.long()].float() * scale).to(w.dtype)
        assert torch.equal(y, want)
    ops.check_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("law", ["any", "one", "few", "skew"])
@pytest.mark.parametrize("n,V,d", [(1, 1, 8), (2, 3, 1), (77, 300, 33), (500, 70, 1000), (4096, 5000, 256), (4097, 128256, 64), (9001, 300001, 40),
                                   (65536, 70000, 16), (65537, 3000, 24), (200003, 1000000, 8)])
def test_gradient(n, V, d, law, dtype):
    torch.manual_seed(0)
    t = TYPES[dtype]
    w = torch.randn(V, d, device="cuda").to(t).requires_grad_()
    ids = _ids(n, V, law, 2).cuda()
    dy = torch.randn(n, d, device="cuda").to(t)
    most = int(torch.bincount(ids).max())
    (g,) = torch.autograd.grad(ops.embedding(ids, w, 1.5), w, dy)
    want, mag = _sums(ids, dy, V, 1.5)
    assert g.dtype == t and g.shape == w.shape
    _close(g, want, mag, t, most)
    assert not g[torch.bincount(ids, minlength=V) == 0].any()
    (h,) = torch.autograd.grad(ops.embedding(ids, w, 1.5), w, dy)
    assert torch.equal(g, h)                                       # the same bits each time
    pad = int(ids[0])
    (g,) = torch.autograd.grad(ops.embedding(ids, w, 1.5, padding_idx=pad), w, dy)
    want, mag = _sums(ids, dy, V, 1.5, pad)
    _close(g, want, mag, t, most)
    assert not g[pad].any()
    ops.check_status()


@pytest.mark.parametrize("dtype,into", [("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("n,V,d", [(77, 300, 33), (3000, 500, 256), (40000, 2000, 128), (100000, 2000, 16)])
def test_main_grad_is_written_and_added_to(n, V, d, dtype, into):
    torch.manual_seed(0)
    t = TYPES[dtype]
    w = torch.randn(V, d, device="cuda").to(t).requires_grad_()
    buf = torch.full((V, d), math.nan, device="cuda", dtype=TYPES[into])
    w.main_grad, w._main_grad_written = buf, False
    ids = _ids(n, V, "skew", 3).cuda()
    dy = torch.randn(n, d, device="cuda").to(t)
    most = int(torch.bincount(ids).max())
    ops.embedding(ids, w).backward(dy)
    assert w.grad is None and w._main_grad_written
    want, mag = _sums(ids, dy, V, 1.0)
    _close(buf, want, mag, TYPES[into], most)                       # NaN was there: every element has been written
    start = torch.randn(V, d, device="cuda").to(TYPES[into])
    buf.copy_(start)
    ops.embedding(ids, w, padding_idx=1).backward(dy)
    want, mag = _sums(ids, dy, V, 1.0, 1)
    _close(buf, want + start.double(), mag + start.double().abs(), TYPES[into], most + 1)
    alone = torch.bincount(ids, minlength=V) == 0
    alone[1] = True
    assert torch.equal(buf[alone], start[alone])                    # rows of other words are left as they are


def test_layouts_shapes_and_empty_batches():
    torch.manual_seed(0)
    big = torch.randn(200, 300, device="cuda")
    ids = torch.randint(0, 200, (3, 7, 5), device="cuda")
    for w in (big[:, 8:264], big[:, 3:260], big[:, ::2], torch.randn(64, 200, device="cuda").t()):
        w = w.detach().requires_grad_()
        y = ops.embedding(ids, w, 2.0)
        assert torch.equal(y, w[ids] * 2)
        dy = torch.randn(7, 5, 3, w.shape[1], device="cuda").permute(2, 0, 1, 3)      # not contiguous
        (g,) = torch.autograd.grad(y, w, dy)
        want, mag = _sums(ids.reshape(-1), dy.reshape(-1, w.shape[1]), 200, 2.0)
        _close(g, want, mag, torch.float32, 105)
    w = big.detach().requires_grad_()
    t = torch.randint(0, 200, (8, 6), device="cuda", dtype=torch.int32).t()
    assert torch.equal(ops.embedding(t, w), w[t.long()])
    assert torch.equal(ops.embedding(t.to(torch.uint8), w), w[t.long()])
    e = ops.embedding(torch.zeros(0, 4, dtype=torch.int64, device="cuda"), w)
    assert e.shape == (0, 4, 300)
    (g,) = torch.autograd.grad(e, w, torch.zeros_like(e))
    assert g.shape == w.shape and not g.any()
    assert ops.embedding(torch.tensor(3, device="cuda"), w).shape == (300,)


def test_ids_out_of_range():
    w = torch.randn(50, 64, device="cuda", requires_grad=True)
    ids = torch.tensor([3, -1, 50, 3, 2 ** 40, 49, -2 ** 35], device="cuda")
    ok = torch.tensor([1, 0, 0, 1, 0, 1, 0], device="cuda", dtype=torch.bool)
    y = ops.embedding(ids, w)
    with pytest.raises(KernelTimeout):
        ops.check_status()
    assert torch.equal(y[ok], w[ids[ok]]) and not y[~ok].any()
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))          # the forward pass has sorted the ids and reported them
    ops.check_status()
    want = torch.zeros(50, 64, device="cuda")
    want[3], want[49] = 2, 1
    assert torch.equal(g, want)
    assert torch.equal(ops.embedding_backward_(torch.empty_like(w), ids, torch.ones_like(y)), want)
    with pytest.raises(KernelTimeout):
        ops.check_status()


def test_refusals():
    w = torch.randn(50, 64, device="cuda")
    with pytest.raises(ValueError):
        ops.embedding(torch.tensor([1]), w)
    with pytest.raises(ValueError):
        ops.embedding_backward_(torch.zeros(50, 64, device="cuda", dtype=torch.bfloat16), torch.tensor([1], device="cuda"), torch.zeros(1, 64, device="cuda"))
    with pytest.raises(ValueError):
        ops.embedding_backward_(torch.zeros(50, 64, device="cuda"), torch.tensor([1], device="cuda"), torch.zeros(2, 64, device="cuda"))


def test_backward_twice_and_changed_ids():
    """A graph that is kept may be gone through again, into main_grad too; ids changed in between are an error, as for any saved tensor."""
    torch.manual_seed(0)
    w = torch.randn(300, 64, device="cuda", requires_grad=True)
    ids = torch.randint(0, 300, (500,), device="cuda")
    y = ops.embedding(ids, w)
    dy = torch.randn_like(y)
    a, = torch.autograd.grad(y, w, dy, retain_graph=True)
    b, = torch.autograd.grad(y, w, dy, retain_graph=True)
    assert torch.equal(a, b)
    w.main_grad, w._main_grad_written = torch.empty_like(w), False
    y.backward(dy, retain_graph=True)
    y.backward(dy, retain_graph=True)
    assert torch.equal(w.main_grad, a + a)
    ids.add_(0)
    with pytest.raises(RuntimeError):
        y.backward(dy)


def test_expanded_gradient_and_no_grad():
    w = torch.randn(40, 24, device="cuda", dtype=torch.bfloat16).requires_grad_()
    ids = torch.randint(0, 40, (17,), device="cuda")
    ops.embedding(ids, w).sum().backward()                       # a gradient of stride 0
    assert torch.equal(w.grad.float(), torch.bincount(ids, minlength=40)[:, None].float().expand(40, 24))
    with torch.no_grad():
        assert not ops.embedding(ids, w).requires_grad
    assert not ops.embedding(ids, w.detach()).requires_grad


def test_other_stream_and_captured_graph():
    torch.manual_seed(0)
    w = torch.randn(1000, 256, device="cuda")
    ids = torch.randint(0, 1000, (600,), device="cuda")
    dy = torch.randn(600, 256, device="cuda")
    want = ops.embedding_backward_(torch.empty_like(w), ids, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.embedding_backward_(torch.empty_like(w), ids, dy)
    s.synchronize()
    assert torch.equal(got, want)
    # two graphs, replayed in turn: each has its own scratch
    outs, graphs = [torch.empty_like(w) for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    i2 = ids.clone()
    for o, gr in zip(outs, graphs):
        with torch.cuda.graph(gr):
            ops.embedding_backward_(o, i2, dy)
    for k in range(3):
        i2.copy_((ids + 17 * k) % 1000)
        for gr in graphs:
            gr.replay()
        want = ops.embedding_backward_(torch.empty_like(w), i2, dy)
        assert all(torch.equal(o, want) for o in outs)


def test_embedding_layer_in_a_model():
    """The layer's gradient is what autograd of the plain lookup gives, up to the rounding of the sums."""
    from sneppx_alg_b200.nn import Embedding
    torch.manual_seed(0)
    e = Embedding(300, 128, dtype=torch.bfloat16, device="cuda")
    ids = torch.randint(0, 300, (4, 200), device="cuda")
    dy = torch.randn(4, 200, 128, device="cuda").to(torch.bfloat16)
    y = e(ids)
    y.backward(dy)
    want, mag = _sums(ids.reshape(-1), dy.reshape(-1, 128), 300, 1.0)
    assert torch.equal(y, e.weight[ids])
    _close(e.weight.grad, want, mag, torch.bfloat16, 800)


@pytest.mark.parametrize("padding_idx", [None, 2])
def test_second_derivatives(padding_idx):
    w = torch.randn(11, 24, device="cuda")
    ids = torch.randint(0, 11, (3, 7), device="cuda")
    got = []
    for f in (lambda t: ops.embedding(ids, t, scale=1.5, padding_idx=padding_idx), lambda t: 1.5 * torch.nn.functional.embedding(ids, t, padding_idx)):
        t = w.clone().requires_grad_()
        (g,) = torch.autograd.grad((f(t) ** 3).sum(), t, create_graph=True)
        got += [g.detach(), torch.autograd.grad((g ** 2).sum(), t)[0]]
    # sums of at most 21 values in another order: 21 roundings of 2^-24, and a few of the products, of what is added up
    for a, b in zip(got[:2], got[2:]):
        assert ((a - b).abs() <= 32 * 2.0 ** -24 * 21 * b.abs().amax()).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [1, 7, 31, 33, 250, 257, 2049])
def test_sums_added_to_rows_that_end_a_buffer(d, dtype):
    """The last word's row is the last of an allocation of its own: no thread asks for what is behind it, and nothing there changes."""
    V, n = 9, 200
    buf = torch.full((V * d + 64,), 3.0, device="cuda")
    grad = buf[:V * d].view(V, d)
    grad.copy_(torch.randn(V, d, device="cuda"))
    start = grad.clone()
    ids = torch.randint(0, V, (n,), device="cuda")
    ids[:5] = V - 1
    dy = torch.randn(n, d, device="cuda").to(TYPES[dtype])
    ops.embedding_backward_(grad, ids, dy, add=True)
    want, mag = _sums(ids, dy, V, 1.0)
    _close(grad, want + start.double(), mag + start.double().abs(), torch.float32, int(torch.bincount(ids).max()) + 1)
    assert (buf[V * d:] == 3).all()


@pytest.mark.parametrize("offset", [0, 4, 8, 12])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_fp32_rows_at_any_16_byte_address(dtype, add, offset):
    """Rows of fp32 values that begin at a sector or in the middle of one: tables, gradients and what is looked up."""
    torch.manual_seed(0)
    V, d, n = 300, 40, 500
    t = TYPES[dtype]
    buf = torch.full((offset + V * d + 16,), 5.0, device="cuda")
    grad = buf[offset:offset + V * d].view(V, d)
    grad.copy_(torch.randn(V, d, device="cuda"))
    ids = _ids(n, V, "skew", 4).cuda()
    dy = torch.randn(n, d, device="cuda").to(t)
    start = grad.double() if add else torch.zeros(V, d, device="cuda", dtype=torch.float64)
    if dtype == "fp32":
        assert torch.equal(ops.embedding(ids, grad, 2.0), grad[ids] * 2)
    ops.embedding_backward_(grad, ids, dy, add=add)
    want, mag = _sums(ids, dy, V, 1.0)
    _close(grad, want + start, mag + start.abs(), torch.float32, int(torch.bincount(ids).max()) + 1)
    assert (buf[:offset] == 5).all() and (buf[offset + V * d:] == 5).all()


@pytest.mark.parametrize("d", [8, 33])
def test_small_values_of_fp32_tables(d):
    """Values and sums below 2^-126, the smallest normal number, are kept, scaled and not, as the library's lookup keeps them."""
    torch.manual_seed(0)
    w = (torch.randint(-100, 100, (20, d), device="cuda").double() * 2.0 ** -140).float().requires_grad_()
    ids = torch.randint(0, 20, (50,), device="cuda")
    dy = (torch.randint(-100, 100, (50, d), device="cuda").double() * 2.0 ** -145).float()
    assert w.abs().max() > 0 and w.abs().max() < torch.finfo(torch.float32).tiny
    for scale in (1.0, 4.0):
        y = ops.embedding(ids, w, scale)
        assert torch.equal(y.double(), w.double()[ids] * scale)
        (g,) = torch.autograd.grad(y, w, dy)
        want, _ = _sums(ids, dy, 20, scale)                    # whole multiples of 2^-145: exact
        assert torch.equal(g.double(), want)
        base = (torch.randint(-100, 100, (20, d), device="cuda").double() * 2.0 ** -143).float()
        start = base.double()
        assert torch.equal(ops.embedding_backward_(base, ids, dy, scale, add=True).double(), start + want)


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint8, torch.bool, torch.complex64, torch.float8_e4m3fn])
def test_tables_of_other_types(dtype):
    """They take the library's lookup, as they are."""
    w = torch.randint(0, 2, (30, 8), device="cuda").to(dtype)
    ids = torch.tensor([[3, 29], [0, 3]], device="cuda")
    y = ops.embedding(ids, w)
    assert y.dtype == dtype and torch.equal(y.to(torch.complex64), torch.nn.functional.embedding(ids, w).to(torch.complex64))
    ops.check_status()


def test_views_whose_sign_is_still_to_be_turned():
    """The imaginary part of a conjugate, as a table, as activations and as incoming gradients."""
    def turned(*shape):
        z = torch.randn(shape, dtype=torch.complex64, device="cuda").conj().imag
        assert z.is_neg()
        return z, z.clone()

    def plain(t):
        return torch.empty_like(t).copy_(t)

    table, t2 = turned(40, 16)
    dy, d2 = turned(7, 16)
    ids = torch.randint(0, 40, (7,), device="cuda")
    assert torch.equal(ops.embedding(ids, table, 2.0), table[ids] * 2)
    w = torch.randn(40, 16, device="cuda", requires_grad=True)
    want = torch.zeros(40, 16, device="cuda").index_add_(0, ids, plain(dy))
    assert torch.allclose(torch.autograd.grad(ops.embedding(ids, w), w, dy)[0], want, atol=1e-5)
    assert torch.allclose(ops.embedding_backward_(torch.empty_like(w), ids, dy), want, atol=1e-5)
    for shape in ((9, 64), (9, 1), (1,), ()):
        x, _ = turned(*shape)
        assert torch.equal(ops.unpack_8bit(ops.pack_8bit(x)), ops.unpack_8bit(ops.pack_8bit(plain(x))))
    x, _ = turned(9, 64)
    g, h = x.detach().requires_grad_(), plain(x).requires_grad_()
    dh, _ = turned(9, 32)
    a, b = ops.glu_8bit(g), ops.glu_8bit(h)
    assert torch.equal(a, b) and torch.equal(torch.autograd.grad(a, g, dh)[0], torch.autograd.grad(b, h, plain(dh))[0])
    hb, wb = (torch.randn(7, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    gn, _ = turned(7)
    t = torch.arange(7, device="cuda")
    got, want = (torch.autograd.grad(ops.linear_token_loss(hb, wb, t)[0], (hb, wb), v) for v in (gn, plain(gn)))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
