"""Traces and function transforms through the embedding, the per-token loss and the 8-bit activations on the GPU."""
import math

import pytest
import torch

from sneppx_alg_b200 import jit, ops
from sneppx_alg_b200.nn import Embedding

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("cuda_graph", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_a_traced_lookup_replays_other_ids(dtype, cuda_graph):
    e = Embedding(100, 24, dtype=TYPES[dtype], device="cuda")
    first, second = (torch.randint(0, 100, (3, 9), device="cuda") for _ in range(2))
    tf = jit.trace(lambda i: e(i) * 2 + ops.embedding(i, e.weight, scale=0.5), first, cuda_graph=cuda_graph)
    with torch.no_grad():
        for ids in (first, second, first):
            assert torch.equal(tf(ids), e(ids) * 2 + ops.embedding(ids, e.weight, scale=0.5))
        e.weight.mul_(2)                                 # a trace follows its weights
        assert torch.equal(tf(second), e(second) * 2 + ops.embedding(second, e.weight, scale=0.5))
    assert tf.traces == 1


@pytest.mark.parametrize("cuda_graph", [False, True])
def test_traced_losses_and_8_bit_activations_replay_other_inputs(cuda_graph):
    w = (torch.randn(300, 64, device="cuda") / 8).to(torch.bfloat16)
    t = torch.randint(0, 300, (20,), device="cuda")

    def f(h):
        nll, lse = ops.linear_token_loss(h, w, t)
        held = ops.unpack_8bit(ops.pack_8bit(h))
        return nll + lse, held.float().sum(-1), ops.glu_8bit(h)

    first, second = (torch.randn(20, 64, device="cuda").to(torch.bfloat16) for _ in range(2))
    tf = jit.trace(f, first, cuda_graph=cuda_graph)
    with torch.no_grad():
        for h in (first, second):
            assert all(torch.equal(a, b) for a, b in zip(tf(h), f(h)))
    g = torch.zeros(50, 64, device="cuda")
    ids = torch.randint(0, 50, (20,), device="cuda")
    tf = jit.trace(lambda dy: ops.embedding_backward_(g, ids, dy) + 0, first.float(), cuda_graph=cuda_graph)
    with torch.no_grad():
        for dy in (first.float(), second.float()):
            got = tf(dy).clone()
            assert torch.equal(got, ops.embedding_backward_(torch.empty_like(g), ids, dy))
    ops.check_status()


def test_gradients_through_a_traced_lookup():
    w = torch.randn(50, 16, device="cuda", requires_grad=True)
    first, second = (torch.randint(0, 50, (9,), device="cuda") for _ in range(2))
    tf = jit.trace(lambda i, t: ops.embedding(i, t) ** 2, cuda_graph=False)
    for ids in (first, second):
        got, = torch.autograd.grad(tf(ids, w).sum(), w)
        want, = torch.autograd.grad((torch.nn.functional.embedding(ids, w) ** 2).sum(), w)
        assert torch.allclose(got, want, rtol=1e-6, atol=0)          # sums of at most 9 values in 32 bits


def test_a_default_device_does_not_change_the_lookup():
    w = torch.randn(50, 16, device="cuda")
    ids = torch.randint(0, 50, (9,), device="cuda")
    with torch.device("cuda"):                           # a function mode, too
        assert torch.equal(ops.embedding(ids, w, math.sqrt(16)), w[ids] * 4)


@pytest.mark.parametrize("dtype", ["fp16", "fp32", "fp64"])
def test_function_transforms_through_a_lookup(dtype):
    """Each against the same transform of the library's lookup."""
    torch.manual_seed(0)
    t = dict(TYPES, fp64=torch.float64)[dtype]
    e = Embedding(40, 8, dtype=t, device="cuda")
    w, v = e.weight.detach(), torch.randn(40, 8, device="cuda").to(t)
    ids = torch.randint(0, 40, (5, 6), device="cuda")

    def loss(look):
        return lambda i, x: (look(i, x).float() ** 2).sum()

    def own(i, x):
        return torch.func.functional_call(e, {"weight": x}, (i,))

    def plain(i, x):
        return torch.nn.functional.embedding(i, x)

    for f in (lambda look: jit.grad(loss(look), 1)(ids, w), lambda look: jit.vmap(look, (0, None))(ids, w), lambda look: jit.vmap(look, (None, 0))(ids, torch.stack([w, v])),
              lambda look: jit.jvp(lambda x: look(ids, x), (w,), (v,)), lambda look: jit.vmap(jit.grad(loss(look), 1), (0, None))(ids, w),
              lambda look: jit.hessian(lambda x: loss(look)(ids[0, :2], x))(w[:, :2].float()) if look is plain else
              jit.hessian(lambda x: loss(lambda i, y: ops.embedding(i, y))(ids[0, :2], x))(w[:, :2].float())):
        got, want = f(own), f(plain)
        for a, b in zip(*([x] if torch.is_tensor(x) else x for x in (got, want))):
            assert a.dtype == b.dtype and torch.equal(a, b)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        y = ops.embedding(ids, fwd.make_dual(w, v), scale=2.0)
        assert torch.equal(fwd.unpack_dual(y).tangent, v[ids] * 2)


def test_lookups_under_a_dispatch_mode():
    from torch.utils.flop_counter import FlopCounterMode
    w = torch.randn(40, 8, device="cuda", requires_grad=True)
    ids = torch.randint(0, 40, (7,), device="cuda")
    with FlopCounterMode(display=False):
        y = ops.embedding(ids, w)
        y.sum().backward()
    assert torch.equal(y, w[ids]) and torch.equal(w.grad, torch.bincount(ids, minlength=40)[:, None].float().expand(40, 8))


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
def test_ids_out_of_range_in_the_pytorch_form(dtype):
    """fp64 tables, and any table inside a transform: rows of zeros and no gradient, as from the kernels."""
    w = torch.randn(20, 8, device="cuda", dtype=dtype)
    ids = torch.tensor([3, -1, 20, 2 ** 40, 19], device="cuda")
    ok = torch.tensor([1, 0, 0, 0, 1], device="cuda", dtype=torch.bool)
    g, y = jit.value_and_grad(lambda x: ops.embedding(ids, x, scale=2.0).sum())(w)
    want = torch.zeros_like(w)
    want[3], want[19] = 2, 2
    assert torch.equal(g, want)
    ops.check_status()
    y = ops.embedding(ids, w)
    with pytest.raises(ops.KernelTimeout):
        ops.check_status()
    assert torch.equal(y[ok], w[ids[ok]]) and not y[~ok].any()


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_lookup_that_torch_compile_reads(backend):
    """In one graph, as it was when the layer called the library's lookup."""
    e = Embedding(50, 8, device="cuda")
    ids = torch.randint(0, 50, (7,), device="cuda")
    y = torch.compile(lambda i: e(i) * 2, fullgraph=True, backend=backend)(ids)
    y.sum().backward()
    assert torch.equal(y, e.weight[ids] * 2)
    assert torch.equal(e.weight.grad, 2 * torch.bincount(ids, minlength=50)[:, None].float().expand(50, 8))


class _Held(torch.Tensor):
    """A tensor class whose values are another tensor's and that has no address of its own, as sharded and lazily loaded weights are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device, strides=inner.stride())

    def __init__(self, inner):
        self.inner = inner

    __torch_function__ = torch._C._disabled_torch_function_impl

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        from torch.utils._pytree import tree_map
        args, kwargs = tree_map(lambda t: t.inner if isinstance(t, _Held) else t, (args, kwargs or {}))
        return func(*args, **kwargs)


def test_tensor_classes_without_an_address():
    w, h = torch.randn(40, 16, device="cuda"), torch.randn(7, 64, device="cuda").to(torch.bfloat16)
    v = (torch.randn(50, 64, device="cuda") / 8).to(torch.bfloat16)
    ids = torch.randint(0, 40, (7,), device="cuda")
    assert _Held(w).data_ptr() == 0
    for table, i in ((_Held(w), ids), (w, _Held(ids)), (_Held(w), _Held(ids))):
        assert torch.equal(ops.embedding(i, table, 2.0), w[ids] * 2)
    dy = torch.randn(7, 16, device="cuda")
    want = ops.embedding_backward_(torch.empty_like(w), ids, dy)
    for add in (False, True):
        got = ops.embedding_backward_(torch.zeros_like(w), _Held(ids), _Held(dy), add=add)
        assert torch.allclose(got, want, rtol=1e-6, atol=1e-6)
    # the PyTorch form's products in 32 bits against sums that the tensor cores cut: 64 additions, each off by 2^-23 of at most 64 x 4 x 0.6
    for args in ((_Held(h), v), (h, _Held(v))):
        for a, b in zip(ops.linear_token_loss(*args, ids), ops.linear_token_loss(h, v, ids)):
            assert torch.allclose(a, b, rtol=0, atol=64 * 2.0 ** -23 * 154)
    held = ops.pack_8bit(_Held(h))
    want = ops.pack_8bit(h)
    assert torch.equal(held.codes, want.codes) and torch.equal(held.exponents, want.exponents)
    assert torch.equal(ops.unpack_8bit(ops.Packed8bit(_Held(want.codes), want.exponents, want.shape, want.dtype)), ops.unpack_8bit(want))
    assert torch.allclose(ops.glu_8bit(_Held(h)).float(), ops.glu_8bit(h).float(), rtol=2.0 ** -7, atol=0)
    ops.check_status()


@pytest.mark.filterwarnings("ignore::DeprecationWarning", "ignore::torch.jit.TracerWarning")
def test_torch_jit_trace():
    e = Embedding(40, 64, dtype=torch.bfloat16, device="cuda").requires_grad_(False)          # torch.jit.trace takes no other constants
    w = (torch.randn(50, 64, device="cuda") / 8).to(torch.bfloat16)
    first, second = (torch.randint(0, 40, (7,), device="cuda") for _ in range(2))
    with torch.no_grad():
        f = torch.jit.trace(lambda i: e(i) * 2, (first,), check_trace=False)
        g = torch.jit.trace(lambda i: ops.linear_token_loss(e.weight[i], w, i)[0], (first,), check_trace=False)
        k = torch.jit.trace(lambda i: ops.unpack_8bit(ops.pack_8bit(e.weight[i])) + ops.glu_8bit(e.weight[i]).repeat(1, 2), (first,), check_trace=False)
        for ids in (first, second):
            x = e.weight[ids]
            assert torch.equal(f(ids), x * 2)
            assert torch.allclose(g(ids), ops.linear_token_loss(x, w, ids)[0], rtol=0, atol=1e-3)
            with torch.jit.optimized_execution(False):          # the tape as it was recorded: TorchScript's fuser drops the conversion to int8
                got = k(ids).float()
            # restored values are exact in both; the gated one may be a step of bf16 off, 2^-7 of it, and the sum is rounded
            a, b = ops.unpack_8bit(ops.pack_8bit(x)).float(), ops.glu_8bit(x).repeat(1, 2).float()
            assert ((got - (a + b)).abs() <= 2.0 ** -7 * (b.abs() + (a + b).abs())).all()


def test_backward_under_a_mode_that_forward_was_not_in():
    from torch.utils.flop_counter import FlopCounterMode
    w, x = torch.randn(40, 16, device="cuda", requires_grad=True), torch.randn(7, 64, device="cuda", requires_grad=True)
    h, v = torch.randn(7, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(50, 64, device="cuda").bfloat16().requires_grad_()
    ids = torch.randint(0, 40, (7,), device="cuda")

    def forward():
        return ops.embedding(ids, w).sum() + ops.glu_8bit(x).sum() + ops.linear_token_loss(h, v, ids)[0].sum()

    want = torch.autograd.grad(forward(), (w, x, h, v))
    loss = forward()
    with FlopCounterMode(display=False):
        got = torch.autograd.grad(loss, (w, x, h, v), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.device("cuda"):
        got = torch.autograd.grad(loss, (w, x, h, v))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
