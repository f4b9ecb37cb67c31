"""Activations in 8 bits on the GPU against the definition in 64 bits."""
import pytest
import torch

from act8_common import TYPES, gate, held, inputs
from sneppx_alg_b200 import ops
from sneppx_alg_b200.ops import _lib

pytestmark = pytest.mark.gpu

SIZES = [(9, 1), (8, 31), (8, 32), (11, 33), (8, 500), (77, 512), (1, 4096), (300, 1000), (8, 4104), (13, 5001)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,width", SIZES)
def test_pack_and_unpack(rows, width, dtype):
    x = inputs(rows, width, dtype, 1)
    p, ref = ops.pack_8bit(x.cuda()), ops.pack_8bit(x)
    assert torch.equal(p.codes.cpu(), ref.codes) and torch.equal(p.exponents.cpu(), ref.exponents)
    want = held(x)
    assert torch.equal(ops.unpack_8bit(p, torch.float32).double().cpu(), want)
    assert torch.equal(ops.unpack_8bit(p).cpu(), want.to(x.dtype))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_strided_rows_odd_bases_and_overflows(dtype):
    big = inputs(64, 320, dtype, 2).cuda()
    for x in (big[:, 7:207], big[::3, 8:264], big[:, 16:], big.t(), big[5], big[:, :1], big.view(4, 16, 320)[:, 3:9]):
        assert torch.equal(ops.unpack_8bit(ops.pack_8bit(x)), ops.unpack_8bit(ops.pack_8bit(x.contiguous())))
        assert torch.equal(ops.unpack_8bit(ops.pack_8bit(x)).cpu(), ops.unpack_8bit(ops.pack_8bit(x.cpu())))
    big[3, 40], big[4, 0], big[5, 319] = float("inf"), float("nan"), -float("inf")
    y = ops.unpack_8bit(ops.pack_8bit(big))
    bad = torch.zeros_like(big, dtype=torch.bool)
    bad[3, 32:64], bad[4, :32], bad[5, 288:] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    for shape in ((0, 7), (3, 0), ()):
        z = torch.ones(shape, dtype=TYPES[dtype], device="cuda")
        assert torch.equal(ops.unpack_8bit(ops.pack_8bit(z)), z)


def test_every_exponent_byte():
    """2^(byte - 127) from the smallest on; 255 is NaN."""
    codes = torch.arange(-128, 128, dtype=torch.int16).to(torch.int8).repeat(256, 1).contiguous()
    exps = torch.arange(256, dtype=torch.int16).to(torch.uint8)[:, None].repeat(1, 8).contiguous()
    p = ops.Packed8bit(codes, exps, torch.Size((256, 256)), torch.float32)
    q = ops.Packed8bit(codes.cuda(), exps.cuda(), p.shape, p.dtype)
    want, got = ops.unpack_8bit(p), ops.unpack_8bit(q).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[:255], want[:255])


def test_refusals():
    with pytest.raises(TypeError):
        ops.pack_8bit(torch.zeros(4, 64, dtype=torch.float64, device="cuda"))
    p = ops.pack_8bit(torch.zeros(4, 64, device="cuda"))
    with pytest.raises(TypeError):
        ops.unpack_8bit(p, torch.float64)
    with pytest.raises(ValueError):
        ops.unpack_8bit(ops.Packed8bit(p.codes, p.exponents[:, :1], p.shape, p.dtype))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,f", [(1, 8), (9, 31), (8, 32), (77, 1000), (150, 1024), (5, 2503), (2, 16384)])
def test_glu(rows, f, act, dtype):
    half = torch.finfo(TYPES[dtype]).eps / 2
    gu = inputs(rows, 2 * f, dtype, 3, edge=False).clamp(-8, 8)
    dh = inputs(rows, f, dtype, 4, edge=False).clamp(-30, 30)
    x = gu.cuda().requires_grad_()
    h = ops.glu_8bit(x, act)
    h.backward(dh.cuda())
    g, u = gu[:, :f].double(), gu[:, f:].double()
    # a rounding of half a step, and before it functions in 32 bits: absolute errors of a few 2^-24 (1 + |g|^3); 2^-25: the smallest step of fp16
    want = gate(g, act)[0] * u
    assert ((h.double().cpu() - want).abs() <= half * want.abs() + 1e-6 * (1 + g.abs() ** 3) * u.abs() + 2.0 ** -25).all()
    g, u, d = held(gu[:, :f]), held(gu[:, f:]), dh.double()
    a, da = gate(g, act)
    want = torch.cat([d * u * da, d * a], 1)
    slack = 1e-6 * torch.cat([(1 + g.abs() ** 3) * (d * u).abs(), (1 + g.abs() ** 3) * d.abs()], 1)
    assert ((x.grad.double().cpu() - want).abs() <= half * want.abs() + slack + 2.0 ** -25).all()


def test_glu_strided_input_and_no_gradient():
    big = inputs(40, 300, "bf16", 5, edge=False).cuda()
    x = big[:, 20:276].detach().requires_grad_()
    h = ops.glu_8bit(x)
    y = big[:, 20:276].contiguous().requires_grad_()
    k = ops.glu_8bit(y)
    assert torch.equal(h, k)
    d = torch.randn_like(h)
    gx, = torch.autograd.grad(h, x, d.t().contiguous().t())       # an incoming gradient laid out the other way
    gy, = torch.autograd.grad(k, y, d)
    assert torch.equal(gx, gy)
    with torch.no_grad():
        assert torch.equal(ops.glu_8bit(y), ops.glu(y))
    e = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ops.glu_8bit(e).sum().backward()
    assert e.grad.shape == (0, 64)


def test_other_stream_and_captured_graph():
    x = inputs(64, 1024, "bf16", 6).cuda()
    want = ops.unpack_8bit(ops.pack_8bit(x))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.unpack_8bit(ops.pack_8bit(x))
    s.synchronize()
    assert torch.equal(y, want)
    graph, z = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = ops.unpack_8bit(ops.pack_8bit(z))
    for k in (1.0, -3.0):
        z.copy_(x * k)
        graph.replay()
        assert torch.equal(out, ops.unpack_8bit(ops.pack_8bit(z)))


def test_checkpoint_of_a_block():
    torch.manual_seed(0)
    w = torch.randn(256, 256, device="cuda", dtype=torch.bfloat16).mul_(0.06).requires_grad_()
    a = torch.randn(100, 256, device="cuda", dtype=torch.bfloat16).requires_grad_()
    x = a * 1
    y = ops.checkpoint_8bit(lambda t: ops.glu(ops.linear(t, w).repeat(1, 2)), x)
    assert torch.equal(y, ops.glu(ops.linear(x, w).repeat(1, 2)))
    y.float().sum().backward()
    b = ops.unpack_8bit(ops.pack_8bit(a.detach())).requires_grad_()
    ga, gw = torch.autograd.grad(ops.glu(ops.linear(b, w).repeat(1, 2)).float().sum(), (b, w))
    assert torch.equal(a.grad, ga) and torch.equal(w.grad, gw)


@pytest.mark.parametrize("width", [64, 72, 77])
@pytest.mark.parametrize("offset", [1, 4, 8, 16])
def test_codes_inside_a_larger_buffer(width, offset):
    """Held values may be views of any alignment; the entry point itself takes none that its loads could not."""
    x = torch.randn(5, width, device="cuda").bfloat16()
    p = ops.pack_8bit(x)
    buf = torch.zeros(offset + p.codes.numel(), device="cuda", dtype=torch.int8)
    view = buf[offset:].view(p.codes.shape)
    view.copy_(p.codes)
    assert torch.equal(ops.unpack_8bit(ops.Packed8bit(view, p.exponents, tuple(x.shape), x.dtype)), ops.unpack_8bit(p))
    if offset < 16:
        with pytest.raises(RuntimeError, match="code -1"):
            _lib.entry("sx_unpack8", "ppplilip")(view.data_ptr(), p.exponents.data_ptr(), x.data_ptr(), 5, width, width, 0, _lib.here(x))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("width", [1, 2, 15, 17, 33, 479, 511, 513, 1023, 1025, 1537])
def test_rows_that_begin_anywhere(width, dtype):
    """Every place of a row's first and last value in a word, and one and several warps a row; what stands before, between and behind the rows is not
    read (NaN) nor written."""
    rows = 10
    x = inputs(rows, width, dtype, 6)
    want = held(x)
    for before, pitch in ((0, width), (1, width), (0, width + 3), (3, width + 2)):
        big = torch.full((before + rows * pitch + 8,), float("nan"), dtype=x.dtype, device="cuda")
        v = big[before:before + rows * pitch].view(rows, pitch)[:, :width]
        v.copy_(x)
        p = ops.pack_8bit(v)
        assert torch.equal(ops.unpack_8bit(p, torch.float32).double().cpu(), want), (before, pitch)
        out = torch.full((rows * width + before + 8,), 7.0, dtype=x.dtype, device="cuda")
        y = out[before:before + rows * width].view(rows, width)
        _lib.entry("sx_unpack8", "ppplilip")(p.codes.data_ptr(), p.exponents.data_ptr(), y.data_ptr(), rows, width, width,
                                            {"bf16": 0, "fp16": 1, "fp32": 2}[dtype], _lib.here(y))
        assert torch.equal(y.cpu(), want.to(x.dtype)), (before, pitch)
        assert (out[:before] == 7).all() and (out[before + rows * width:] == 7).all()


@pytest.mark.parametrize("f", [1, 15, 257, 511, 513, 1025])
def test_glu_of_rows_that_begin_anywhere(f):
    gu, dh = inputs(9, 2 * f, "bf16", 7, edge=False).clamp(-8, 8).cuda(), inputs(9, f, "bf16", 8, edge=False).cuda()
    wide = -(-f // 32) * 32                        # the same values in rows of whole blocks take the other way through the kernels
    pad = lambda t: torch.nn.functional.pad(t, (0, wide - f))  # noqa: E731
    y = torch.cat([pad(gu[:, :f]), pad(gu[:, f:])], 1).requires_grad_()
    h2 = ops.glu_8bit(y)
    h2.backward(pad(dh))
    for before in (0, 1):
        x = torch.empty(9 * 2 * f + 1, dtype=torch.bfloat16, device="cuda")[before:before + 18 * f].view(9, 2 * f).copy_(gu).requires_grad_()
        h = ops.glu_8bit(x)
        h.backward(dh)
        assert torch.equal(h, h2[:, :f]) and torch.equal(x.grad, torch.cat([y.grad[:, :f], y.grad[:, wide:wide + f]], 1))


@pytest.mark.parametrize("bits", [8, 16])
def test_checkpoint_draws_the_same_random_numbers_again(bits):
    """Gradients are those of the mask that the forward pass drew, and the generator is where the forward pass left it."""
    from sneppx_alg_b200.training.extras import checkpoint
    w = torch.randn(40, 40, device="cuda").requires_grad_()
    a = (torch.randint(-100, 100, (9, 40), device="cuda") / 32.0)          # 8 bits hold whole multiples of a power of two
    a[:, ::32] = 127 / 32.0
    a.requires_grad_()

    def fn(t, rope):
        return torch.nn.functional.dropout(t, 0.5) @ w

    torch.manual_seed(3)
    y = checkpoint(fn, a * 1, (None, torch.zeros(1, device="cuda")), bits=bits)
    state = torch.cuda.get_rng_state()
    got = torch.autograd.grad(y.square().sum(), (a, w))
    assert torch.equal(torch.cuda.get_rng_state(), state)
    torch.manual_seed(3)
    want = torch.autograd.grad(fn(a * 1, None).square().sum(), (a, w))
    assert all(torch.equal(g, v) for g, v in zip(got, want))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("width", [32, 1000, 1001, 1008])
def test_the_largest_values_come_back_finite(width, dtype):
    """In every place of a row, through each way of reading rows."""
    from act8_common import largest
    block, want, _ = largest(dtype)
    x, y = (torch.cat([t.repeat(1, width // 32), t[:, :width % 32]], 1) for t in (block, want))
    if width % 32:                                # what is left of a block may have lost its largest value
        cut = width // 32 * 32
        y[:, cut:] = ops.unpack_8bit(ops.pack_8bit(x[:, cut:]), torch.float32).double()
    p = ops.pack_8bit(x.cuda())
    assert torch.equal(ops.unpack_8bit(p).cpu().double(), y)
    ref = ops.pack_8bit(x)
    assert torch.equal(p.codes.cpu(), ref.codes) and torch.equal(p.exponents.cpu(), ref.exponents)
    gu = torch.cat([x, torch.full_like(x, 2.0 ** -20)], 1).cuda().requires_grad_()
    h = ops.glu_8bit(gu, "relu")
    assert torch.isfinite(h).all()
    h.backward(torch.ones_like(h))
    assert torch.equal(gu.grad[:, width:].double().cpu(), y.clamp(min=0))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("f", [32, 1001, 96])
def test_glu_of_overflows(f, act, dtype):
    from act8_common import check_glu_of_overflows
    check_glu_of_overflows(ops.glu_8bit, act, dtype, "cuda", f)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("f", [31, 64, 1000, 1001])
def test_glu_without_a_gradient_keeps_nothing(f, dtype):
    x = inputs(77, 2 * f, dtype, 10, edge=False).clamp(-8, 8).cuda()
    want = ops.glu_8bit(x.clone().requires_grad_()).detach()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = ops.glu_8bit(x)
    used = torch.cuda.max_memory_allocated() - before
    assert torch.equal(got, want)
    # the result, in the allocator's blocks of 512 bytes, and no codes
    assert used <= (got.numel() * got.element_size() + 511) // 512 * 512
    with torch.no_grad():
        assert torch.equal(ops.glu_8bit(x.requires_grad_()), want)
    e = torch.zeros(0, 64, device="cuda", dtype=TYPES[dtype])
    assert ops.glu_8bit(e).shape == (0, 32)
