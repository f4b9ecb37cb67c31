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
