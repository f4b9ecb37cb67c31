"""Activations in 8 bits on the CPU: format, refusals, gradients, recomputation."""
import pytest
import torch

from act8_common import TYPES, gate, held, inputs
from sneppx_alg_b200 import ops


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,width", [(9, 1), (8, 31), (8, 32), (11, 33), (8, 500)])
def test_pack_holds_what_the_definition_says(rows, width, dtype):
    x = inputs(rows, width, dtype, 1)
    p = ops.pack_8bit(x)
    assert p.codes.shape == (rows, -(-width // 32) * 32) and p.exponents.shape == (rows, -(-width // 32))
    assert p.nbytes == p.codes.numel() + p.exponents.numel() and int(p.codes.abs().max()) <= 127
    assert torch.equal(ops.unpack_8bit(p, torch.float32).double(), held(x))
    assert torch.equal(ops.unpack_8bit(p).double(), held(x).to(x.dtype).double()) and ops.unpack_8bit(p).dtype == x.dtype


def test_a_block_with_an_overflow_is_restored_as_nan():
    x = torch.ones(3, 70)
    x[0, 5], x[1, 40], x[2, 69] = float("inf"), float("nan"), -float("inf")
    y = ops.unpack_8bit(ops.pack_8bit(x))
    bad = torch.zeros(3, 70, dtype=torch.bool)
    bad[0, :32], bad[1, 32:64], bad[2, 64:] = True, True, True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], x[~bad])


@pytest.mark.parametrize("shape", [(), (1,), (0, 7), (3, 0), (2, 3, 40), (4, 1)])
def test_any_shape_comes_back(shape):
    x = torch.full(shape, 3.0)
    y = ops.unpack_8bit(ops.pack_8bit(x))
    assert y.shape == x.shape and torch.equal(x, y)
    t = torch.arange(60.0).reshape(4, 15).t()          # columns of a transposed tensor
    assert torch.equal(ops.unpack_8bit(ops.pack_8bit(t)), ops.unpack_8bit(ops.pack_8bit(t.contiguous())))


def test_refusals():
    with pytest.raises(TypeError):
        ops.pack_8bit(torch.zeros(4, dtype=torch.int32))
    p = ops.pack_8bit(torch.zeros(4, 64))
    with pytest.raises(ValueError):
        ops.unpack_8bit(ops.Packed8bit(p.codes[:, :32], p.exponents, p.shape, p.dtype))
    with pytest.raises(ValueError):
        ops.unpack_8bit(ops.Packed8bit(p.codes, p.exponents, torch.Size((5, 64)), p.dtype))
    with pytest.raises(ValueError):
        ops.glu_8bit(torch.zeros(4, 63))
    with pytest.raises(ValueError):
        ops.glu_8bit(torch.zeros(4, 64), "tanh")
    with pytest.raises(TypeError):
        ops.glu_8bit(torch.zeros(4, 64, dtype=torch.int64))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("shape", [(6, 2), (2, 5, 70), (8, 128)])
def test_glu_gradient_is_that_of_the_restored_input(shape, act):
    f = shape[-1] // 2
    gu = inputs(torch.Size(shape[:-1]).numel(), shape[-1], "fp32", 3, edge=False).clamp(-8, 8)
    gu = gu.reshape(shape).requires_grad_()
    dh = torch.randn(*shape[:-1], f, generator=torch.Generator().manual_seed(4))
    h = ops.glu_8bit(gu, act)
    h.backward(dh)
    g2 = gu.detach().reshape(-1, 2 * f)
    a, _ = gate(g2[:, :f].double(), act)
    # 32-bit functions: an absolute error of a few 2^-24 (1 + |g|^3) before the last product
    assert ((h.reshape(-1, f).double() - a * g2[:, f:].double()).abs() <= 1e-6 * (1 + g2[:, :f].abs() ** 3) * (1 + g2[:, f:].abs())).all()
    g, u, d = held(g2[:, :f]), held(g2[:, f:]), dh.reshape(-1, f).double()
    a, da = gate(g, act)
    want = torch.cat([d * u * da, d * a], 1)
    tol = 1e-6 * torch.cat([(1 + g.abs() ** 3) * (1 + u.abs()), 1 + g.abs() ** 3], 1) * (1 + d.abs().repeat(1, 2))
    assert ((gu.grad.reshape(-1, 2 * f).double() - want).abs() <= tol).all()


def test_glu_gradient_against_differences():
    """On whole multiples of a power of two the 8 bits hold the input exactly, so the gradient is that of the function: central differences in 64 bits."""
    gen = torch.Generator().manual_seed(5)
    gu = torch.randint(-127, 128, (3, 64), generator=gen).double() / 32
    gu[:, 0], gu[:, 32] = 127 / 32, -127 / 32
    x = gu.clone().requires_grad_()
    ops.glu_8bit(x, "silu").sum().backward()
    f = lambda t: (gate(t[:, :32], "silu")[0] * t[:, 32:]).sum()  # noqa: E731
    step = 2.0 ** -12
    for i, j in [(0, 0), (1, 7), (2, 31), (0, 33), (1, 50), (2, 63)]:
        d = torch.zeros_like(gu)
        d[i, j] = step
        # error of the difference: step^2 / 6 times a third derivative below 4, and 32-bit functions
        assert abs(float((f(gu + d) - f(gu - d)) / (2 * step)) - float(x.grad[i, j])) < 4 * step ** 2 + 4e-5


def test_checkpoint_recomputes_from_the_held_arguments():
    gen = torch.Generator().manual_seed(6)
    w = torch.randn(48, 48, generator=gen).requires_grad_()
    a = torch.randn(7, 48, generator=gen).requires_grad_()
    mask = torch.arange(48) % 2
    calls = []

    def fn(x, m, k):
        calls.append(x.detach().clone())
        return torch.tanh(x @ w) * m * k, x

    x = a * 1.0
    y, same = ops.checkpoint_8bit(fn, x, mask, 2.0)
    assert torch.equal(same, x) and torch.equal(y, torch.tanh(x @ w) * mask * 2.0)
    (y.square().sum() + same.sum()).backward()
    restored = held(x).float()
    assert torch.equal(calls[0], x) and torch.equal(calls[1], restored)
    # the saved values are those of the restored argument, the incoming gradient that of y as it was
    t = torch.tanh(restored @ w)
    dz = 2 * y.detach() * mask * 2.0 * (1 - t * t)
    assert torch.allclose(w.grad, restored.t() @ dz, rtol=1e-5, atol=1e-5)
    assert torch.allclose(a.grad, dz @ w.detach().t() + 1, rtol=1e-5, atol=1e-5)


def test_checkpoint_without_gradients_and_with_leaves():
    lin = torch.nn.Linear(8, 8)
    x = torch.randn(3, 8)
    with torch.no_grad():
        assert torch.equal(ops.checkpoint_8bit(lin, x), lin(x))
    leaf = x.clone().requires_grad_()
    ops.checkpoint_8bit(lambda t: lin(t).square().sum(), leaf).backward()      # a leaf is kept as it is: the gradient is the function's own
    want, = torch.autograd.grad(lin(leaf).square().sum(), leaf)
    assert torch.equal(leaf.grad, want)


def test_checkpoint_is_told_the_devices_of_the_arguments(monkeypatch):
    """torch.utils.checkpoint saves and restores the generators of the devices of the tensors that it is handed, nested ones included."""
    import torch.utils.checkpoint as tc
    plain, seen = tc.checkpoint, []

    def spy(fn, *args, **kw):
        seen.append({t.device.type for t in args if torch.is_tensor(t)})
        assert not any(t.numel() for t in args)          # which are not kept through it
        return plain(fn, *args, **kw)

    monkeypatch.setattr(tc, "checkpoint", spy)
    x = torch.randn(3, 8, requires_grad=True) * 1
    ops.checkpoint_8bit(lambda t, k: t * 2, x, (torch.zeros(2, device="meta"), None))
    assert seen == [{"cpu", "meta"}]


def test_checkpoint_draws_the_same_random_numbers_again():
    a = (torch.randint(-100, 100, (9, 40)) / 32.0).requires_grad_()          # 8 bits hold whole multiples of a power of two
    a.data[:, ::32] = 127 / 32.0
    torch.manual_seed(3)
    y = ops.checkpoint_8bit(lambda t: torch.nn.functional.dropout(t, 0.5).square(), a * 1)
    state = torch.get_rng_state()
    y.sum().backward()
    assert torch.equal(torch.get_rng_state(), state)
    torch.manual_seed(3)
    want, = torch.autograd.grad(torch.nn.functional.dropout(a * 1, 0.5).square().sum(), a)
    assert torch.equal(a.grad, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_the_largest_values_come_back_finite(dtype):
    from act8_common import largest
    x, want, step = largest(dtype)
    p = ops.pack_8bit(x)
    y = ops.unpack_8bit(p)
    assert torch.equal(y.double(), want) and torch.equal(ops.unpack_8bit(p, torch.float32).double(), want) and int(p.codes.abs().max()) <= 127
    assert ((y.double() - x.double()).abs() < step).all()
    gu = torch.cat([x, torch.full_like(x, 2.0 ** -20)], 1).requires_grad_()
    ops.glu_8bit(gu, "relu").sum().backward()
    assert torch.equal(gu.grad[:, 32:].double(), want.clamp(min=0))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("f", [32, 70, 96])
def test_glu_of_overflows(f, act, dtype):
    from act8_common import check_glu_of_overflows
    check_glu_of_overflows(ops.glu_8bit, act, dtype, "cpu", f)
