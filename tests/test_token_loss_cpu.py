"""Per-token vocabulary loss on the CPU: values, gradients, refusals."""
import pytest
import torch
import torch.nn.functional as F

from sneppx_alg_b200 import ops


@pytest.mark.parametrize("softcap", [0.0, 5.0])
def test_values_and_gradients_against_differences(softcap):
    g = torch.Generator().manual_seed(0)
    h = torch.randn(2, 3, 5, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(7, 5, generator=g, dtype=torch.float64).requires_grad_()
    t = torch.tensor([[0, 6, -100], [3, 3, 1]])
    nll, lse = ops.linear_token_loss(h, w, t, softcap=softcap)
    z = h @ w.t()
    z = softcap * torch.tanh(z / softcap) if softcap else z
    assert torch.allclose(lse, torch.logsumexp(z, -1), rtol=0, atol=1e-13)
    assert torch.allclose(nll.reshape(-1), F.cross_entropy(z.reshape(-1, 7), t.reshape(-1), reduction="none"), rtol=0, atol=1e-13)
    assert nll[0, 2].item() == 0.0
    assert torch.autograd.gradcheck(lambda a, b: ops.linear_token_loss(a, b, t, softcap=softcap), (h, w))


def test_dtypes_and_empty_batches():
    h, w = torch.randn(4, 8).to(torch.bfloat16), torch.randn(9, 8).to(torch.bfloat16)
    nll, lse = ops.linear_token_loss(h, w, torch.tensor([0, 8, 2, 2]))
    assert nll.dtype == lse.dtype == torch.float32
    nll, lse = ops.linear_token_loss(h[:0], w, torch.zeros(0, dtype=torch.int64))
    assert nll.shape == lse.shape == (0,)


def test_refusals():
    h, w, t = torch.randn(4, 8), torch.randn(9, 8), torch.tensor([0, 8, 2, 2])
    for args in ((h[:, :7], w, t), (h, w[0], t), (h, w, t[:3]), (h, w[:0], t)):
        with pytest.raises(ValueError):
            ops.linear_token_loss(*args)
    with pytest.raises(ValueError):
        ops.linear_token_loss(h, w, t, softcap=-1.0)
    with pytest.raises(ValueError):
        ops.linear_token_loss(h, w, t, piece=-1)
    with pytest.raises(TypeError):
        ops.linear_token_loss(h, w, t.int())
    for bad in (t + 1, t - 1):
        with pytest.raises(IndexError):
            ops.linear_token_loss(h, w, bad)
