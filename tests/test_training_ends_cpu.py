"""Callers of the embedding, the per-token loss and the 8-bit activations on the CPU."""
import copy

import pytest
import torch

from sneppx_alg_b200.models import ModelConfig, build_model
from sneppx_alg_b200.training import extras
from sneppx_alg_b200.training.lora import sequence_logprob


def _model(tie=True):
    torch.manual_seed(0)
    return build_model(ModelConfig(hidden_size=64, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, intermediate_size=96, vocab_size=50,
                                   max_position_embeddings=64, rms_norm_eps=1e-5, tie_word_embeddings=tie)).train()


def _grads(model, ids):
    model.zero_grad(set_to_none=True)
    loss = model(ids, labels=ids)["loss"]
    loss.backward()
    return float(loss.detach()), {k: p.grad.clone() for k, p in model.named_parameters()}


def _rel(a, b):
    return float((a - b).norm() / b.norm().clamp(min=1e-30))


@pytest.mark.parametrize("how", ["layers", "glu", "both"])
def test_8bit_activations_change_gradients_by_their_rounding_only(how):
    model, ids = _model(), torch.randint(0, 50, (2, 30), generator=torch.Generator().manual_seed(1))
    want_loss, want = _grads(model, ids)
    if how != "glu":
        assert extras.enable_activation_checkpointing(model, bits=8) is model
    if how != "layers":
        assert extras.enable_8bit_activations(model) == 2
    loss, got = _grads(model, ids)
    assert loss == want_loss                                   # the forward pass is the same
    # a held value is off by half a step, at most 1/127 of its block's largest, 1/220 of the values' size on average: a few of them meet in a gradient
    assert 0 < max(_rel(got[k], want[k]) for k in want) < 0.05
    model.eval()
    assert torch.equal(model(ids)["logits"], copy.deepcopy(model)(ids)["logits"])
    extras.enable_8bit_activations(model, False)
    extras.enable_activation_checkpointing(model, bits=16)
    loss, got = _grads(model.train(), ids)
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_refusals():
    with pytest.raises(ValueError):
        extras.enable_activation_checkpointing(_model(), bits=4)
    with pytest.raises(ValueError):
        extras.enable_activation_checkpointing(torch.nn.Linear(2, 2), bits=8)
    with pytest.raises(ValueError):
        extras.checkpoint(lambda x: x, torch.ones(2), bits=3)
    with pytest.raises(TypeError):
        extras.checkpoint(lambda x: x, torch.ones(2), bits=8, preserve_rng_state=False)


def test_next_token_logprobs_are_those_of_the_logits():
    model, ids = _model(False), torch.randint(0, 50, (3, 11), generator=torch.Generator().manual_seed(2))
    lp = torch.log_softmax(model(ids)["logits"][:, :-1], -1).gather(-1, ids[:, 1:, None]).squeeze(-1)
    assert torch.equal(model.next_token_logprobs(ids), lp)
    mask = torch.ones(3, 11)
    mask[0, 5:] = 0
    assert torch.equal(sequence_logprob(model, ids, mask), (lp * mask[:, 1:]).sum(-1))


def test_models_that_answer_with_their_logits():
    from sneppx_alg_b200.models.llama import MistralForCausalLM
    from sneppx_alg_b200.training.lora import _answers_with_its_logits, apply_lora
    model = _model()
    assert _answers_with_its_logits(model) and _answers_with_its_logits(copy.deepcopy(model))
    apply_lora(model)
    assert _answers_with_its_logits(model)
    model.__class__ = MistralForCausalLM
    assert _answers_with_its_logits(model)
    assert not _answers_with_its_logits(torch.nn.Linear(2, 2)) and not _answers_with_its_logits(torch.nn.DataParallel(model))
    handle = model.register_full_backward_hook(lambda *a: None)
    assert not _answers_with_its_logits(model)
    handle.remove()
    assert _answers_with_its_logits(model)


def test_models_saved_before_there_was_a_choice_of_bits():
    model, ids = _model(), torch.randint(0, 50, (2, 30), generator=torch.Generator().manual_seed(1))
    _, want = _grads(model, ids)
    model.activation_checkpointing = True
    vars(model).pop("checkpoint_bits", None)                   # what an object pickled earlier comes back without
    _, got = _grads(model, ids)
    assert all(torch.equal(got[k], want[k]) for k in want)
    assert extras.enable_activation_checkpointing(model, bits=8).checkpoint_bits == 8 and type(model).checkpoint_bits == 16
