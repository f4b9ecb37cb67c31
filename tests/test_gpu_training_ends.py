"""Embedding, 8-bit activations and the per-token loss together, as a training step of a decoder uses them."""
import math

import pytest
import torch

from sneppx_alg_b200 import ops
from sneppx_alg_b200.models import ModelConfig, build_model
from sneppx_alg_b200.training import extras
from sneppx_alg_b200.training.engine import TrainEngine
from sneppx_alg_b200.training.lora import sequence_logprob

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8            # half a step of bf16


def _model(tie, vocab=1000, layers=2, dtype=torch.bfloat16):
    torch.manual_seed(0)
    return build_model(ModelConfig(hidden_size=256, num_hidden_layers=layers, num_attention_heads=2, num_key_value_heads=1, intermediate_size=512,
                                   vocab_size=vocab, max_position_embeddings=256, rms_norm_eps=1e-5, tie_word_embeddings=tie), dtype=dtype, device="cuda").train()


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp(min=1e-30))


@pytest.mark.parametrize("tie", [True, False])
def test_a_step_from_the_table_to_the_losses(tie):
    """Lookup with scaling, a gated block whose activations are held in 8 bits, losses with weights of their own and a z-loss; the tied table's gradient
    is written by the loss and added to by the lookup. Against the same in 64 bits, from the same bf16 weights, with the held values restored."""
    torch.manual_seed(1)
    V, d, f, T = 701, 128, 192, 333
    table = (torch.randn(V, d, device="cuda") / math.sqrt(d)).to(torch.bfloat16).requires_grad_()
    head = table if tie else (torch.randn(V, d, device="cuda") / math.sqrt(d)).to(torch.bfloat16).requires_grad_()
    w1 = (torch.randn(2 * f, d, device="cuda") / math.sqrt(d)).to(torch.bfloat16).requires_grad_()
    w2 = (torch.randn(d, f, device="cuda") / math.sqrt(f)).to(torch.bfloat16).requires_grad_()
    ids, target = torch.randint(0, V, (T,), device="cuda"), torch.randint(0, V, (T,), device="cuda")
    target[::7] = -100
    weight = torch.rand(T, device="cuda")
    for p in {table, head, w1, w2}:
        p.main_grad, p._main_grad_written = torch.full(p.shape, math.nan, device="cuda"), False
    x = ops.embedding(ids, table, scale=4.0)
    gu = ops.linear(x, w1)
    h = ops.linear(ops.glu_8bit(gu), w2)
    nll, lse = ops.linear_token_loss(h, head, target, piece=256)
    ((nll * weight).sum() + 1e-2 * lse.square().sum()).backward()
    ops.check_status()
    assert all(p.grad is None and torch.isfinite(p.main_grad).all() for p in (table, head, w1, w2))

    t64, h64, a64, b64 = (p.detach().double().requires_grad_() for p in (table, head, w1, w2))
    h64 = t64 if tie else h64
    x64 = t64[ids] * 4.0
    gu64 = x64 @ a64.t()
    held = ops.unpack_8bit(ops.pack_8bit(gu.detach().view(T, 2, f))).double().view(T, 2 * f)
    g64, u64 = (gu64 + (held - gu64).detach()).chunk(2, 1)
    glu = torch.nn.functional.silu(g64) * u64
    exact = torch.nn.functional.silu(gu64[:, :f]) * gu64[:, f:]
    z = (glu + (exact - glu).detach()) @ b64.t() @ h64.t()
    l64 = torch.logsumexp(z, 1)
    n64 = torch.where(target >= 0, l64 - z.gather(1, target.clamp(min=0)[:, None]).squeeze(1), 0.0)
    ((n64 * weight.double()).sum() + 1e-2 * l64.square().sum()).backward()
    # each value that goes through the chain in bf16 is off by half a step at most, 2^-8 of it; up to eight of them lie one behind the other (x, gu, the
    # gate's value, h, then dz, dh, d of the gate's value, dgu, dx), and their errors do not all point one way
    assert _rel(nll, n64) < 4 * HALF and _rel(lse, l64) < 4 * HALF
    pairs = [(table, t64), (w1, a64), (w2, b64)] + ([] if tie else [(head, h64)])
    for p, p64 in pairs:
        assert _rel(p.main_grad, p64.grad) < 8 * HALF


@pytest.mark.parametrize("tie", [True, False])
def test_engine_step_writes_the_table_once(tie):
    """Gradients of an engine's step, embedding included, are in the flat buffer and are those of autograd without an engine."""
    model = _model(tie)
    ids = torch.randint(0, 1000, (4, 64), device="cuda")
    model(ids, labels=ids)["loss"].backward()
    want = {k: p.grad.clone() for k, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    engine = TrainEngine(model, lr=1e-3, grad_dtype=torch.float32)
    engine.step(ids, ids)
    ops.check_status()
    for k, p in engine.model.named_parameters():
        # the same sums, rounded to bf16 by autograd
        assert _rel(p.main_grad, want[k]) < 2 * HALF, k
    assert engine.model.embedding.weight.grad is None


def test_activations_in_8_bits_in_a_model():
    model = _model(True)
    ids = torch.randint(0, 1000, (4, 96), device="cuda")

    def grads():
        model.zero_grad(set_to_none=True)
        loss = model(ids, labels=ids)["loss"]
        loss.backward()
        ops.check_status()
        return loss.detach(), {k: p.grad.clone() for k, p in model.named_parameters()}

    loss, want = grads()
    extras.enable_8bit_activations(model)
    l8, got = grads()
    assert torch.equal(loss, l8)
    assert max(_rel(got[k], want[k]) for k in want) < 0.05          # half a step of 8 bits, 1/127 of a block's largest value
    extras.enable_activation_checkpointing(model, bits=8)
    l8, got = grads()
    assert torch.equal(loss, l8)
    assert max(_rel(got[k], want[k]) for k in want) < 0.1           # and once more for the layers' inputs
    # what is held between the passes: half of what 16-bit checkpoints hold, and the attention's part is recomputed
    def kept(bits):
        extras.enable_8bit_activations(model, False)
        extras.enable_activation_checkpointing(model, bits=bits)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_allocated()
        h = model.hidden_states(ids.repeat(8, 1))
        torch.cuda.synchronize()
        used = torch.cuda.memory_allocated() - before
        del h
        return used
    kept(16)
    assert kept(8) < kept(16)


def test_sequence_logprob_and_its_gradient():
    model = _model(False, vocab=1003)
    ids = torch.randint(0, 1003, (3, 40), device="cuda")
    mask = (torch.rand(3, 40, device="cuda") < 0.7).float()
    lp = sequence_logprob(model, ids, mask)
    logits = model(ids)["logits"]
    want = (torch.log_softmax(logits.double()[:, :-1], -1).gather(-1, ids[:, 1:, None]).squeeze(-1) * mask[:, 1:]).sum(-1)
    # logits are rounded to bf16 there: half a step of each of up to 39 of about 4
    assert ((lp.double() - want).abs() <= 39 * 4 * HALF).all()
    model.zero_grad(set_to_none=True)
    lp.sum().backward()
    got = {k: p.grad.clone() for k, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    logits = model(ids)["logits"].float()
    (torch.log_softmax(logits[:, :-1], -1).gather(-1, ids[:, 1:, None]).squeeze(-1) * mask[:, 1:]).sum().backward()
    for k, p in model.named_parameters():
        assert _rel(got[k], p.grad) < 8 * HALF, k


def test_two_streams_at_once():
    """The same operators on two streams at a time, each with scratch of its own."""
    torch.manual_seed(3)
    table = torch.randn(3000, 256, device="cuda").to(torch.bfloat16)
    sets = [(torch.randint(0, 3000, (2000,), device="cuda"), torch.randn(2000, 256, device="cuda").to(torch.bfloat16)) for _ in range(2)]

    def run(ids, dy):
        g = ops.embedding_backward_(torch.empty_like(table), ids, dy)
        nll, lse = ops.linear_token_loss(dy, table, ids)
        return g, nll, lse, ops.unpack_8bit(ops.pack_8bit(dy))

    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, st in zip(sets, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(run(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    ops.check_status()


def test_first_call_inside_a_capture():
    """A process whose first product, forward and backward, is captured into a graph: nothing on the way is a call that a capture does not allow."""
    import subprocess
    import sys
    code = """
import torch
from sneppx_alg_b200 import ops
w = torch.randn(3000, 256, device="cuda").to(torch.bfloat16).requires_grad_()
h = torch.randn(500, 256, device="cuda").to(torch.bfloat16).requires_grad_()
ids = torch.randint(0, 3000, (500,), device="cuda")
def step():
    nll, lse = ops.linear_token_loss(h, w, ids)
    return torch.autograd.grad((ops.embedding(ids, w), nll), (w, h), (h.detach(), torch.ones_like(nll)))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_sequence_logprob_calls_models_that_answer_otherwise():
    """A hook, a subclass's forward, a forward set on the model and a wrapper all change the logits, and with them the log-probabilities."""
    model = _model(False, vocab=203, layers=1)
    ids = torch.randint(0, 203, (2, 20), device="cuda")
    mask = torch.ones(2, 20, device="cuda")

    def of(logits):
        lp = torch.log_softmax(logits.float()[:, :-1], -1).gather(-1, ids[:, 1:, None]).squeeze(-1)
        return lp.sum(-1)

    def halved(out):
        return dict(out, logits=out["logits"] / 2)

    class Tempered(type(model)):
        def forward(self, *args, **kw):
            return halved(super().forward(*args, **kw))

    class Wrapper(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def __getattr__(self, name):
            try:
                return super().__getattr__(name)
            except AttributeError:
                return getattr(self.inner, name)

        def forward(self, ids):
            return halved(self.inner(ids))

    with torch.no_grad():
        plain, want = sequence_logprob(model, ids, mask), of(model(ids)["logits"] / 2)
        assert not torch.allclose(plain, want, rtol=1e-3)
        assert torch.equal(sequence_logprob(Wrapper(model), ids, mask), want)
        handle, seen = model.register_forward_hook(lambda m, a, out: halved(out)), []
        assert torch.equal(sequence_logprob(model, ids, mask), want)
        handle.remove()
        handle = model.register_forward_pre_hook(lambda m, a: seen.append(len(a)))
        sequence_logprob(model, ids, mask)
        assert seen == [1]
        handle.remove()
        first = model.forward
        model.forward = lambda *a, **k: halved(first(*a, **k))
        assert torch.equal(sequence_logprob(model, ids, mask), want)
        del model.forward
        model.__class__ = Tempered
        assert torch.equal(sequence_logprob(model, ids, mask), want)
        model.__class__ = Tempered.__mro__[1]
        assert torch.equal(sequence_logprob(model, ids, mask), plain)
    ops.check_status()
