"""Embedding on the CPU: values, gradients, refusals."""
import pytest
import torch
import torch.nn.functional as F

from sneppx_alg_b200 import ops


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("scale,padding", [(1.0, None), (3.5, 2), (8.0, -1)])
def test_lookup_and_gradient(dtype, scale, padding):
    g = torch.Generator().manual_seed(0)
    w = torch.randn(11, 6, generator=g).to(dtype).requires_grad_()
    ids = torch.randint(0, 11, (4, 5), generator=g)
    dy = torch.randint(-8, 9, (4, 5, 6), generator=g).to(dtype)          # whole numbers: their sums are exact in every type
    y = ops.embedding(ids, w, scale, padding)
    assert y.dtype == dtype and torch.equal(y, (w.detach().double()[ids] * scale).to(dtype))
    y.backward(dy)
    want = torch.zeros(11, 6, dtype=torch.float64)
    for t, row in zip(ids.reshape(-1).tolist(), dy.reshape(-1, 6).double()):
        if padding is None or t != padding % 11:
            want[t] += scale * row
    assert torch.equal(w.grad.double(), want)


def test_plain_lookup_is_what_it_was():
    w = torch.randn(9, 4)
    for ids in (torch.tensor([[1, 2], [8, 0]]), torch.tensor([3, 3], dtype=torch.int32), torch.tensor([], dtype=torch.int64), torch.tensor(5)):
        assert torch.equal(ops.embedding(ids, w), F.embedding(ids, w))
    from sneppx_alg_b200.nn import Embedding
    e = Embedding(9, 4)
    assert torch.equal(e(torch.tensor([1, 7])), F.embedding(torch.tensor([1, 7]), e.weight))


def test_refusals():
    w = torch.randn(9, 4)
    with pytest.raises(TypeError):
        ops.embedding(torch.tensor([1.0]), w)
    with pytest.raises(TypeError):
        ops.embedding(torch.tensor([True]), w)
    with pytest.raises(ValueError):
        ops.embedding(torch.tensor([1]), w[0])
    with pytest.raises(ValueError):
        ops.embedding(torch.tensor([1]), w, padding_idx=9)
    with pytest.raises(IndexError):
        ops.embedding(torch.tensor([9]), w)
    with pytest.raises(IndexError):
        ops.embedding(torch.tensor([0]), torch.randn(0, 4))
    assert ops.embedding(torch.zeros(0, dtype=torch.int64), torch.randn(0, 4)).shape == (0, 4)


def test_graph_node_without_a_gpu():
    """The module in C++ can be built and loaded; it takes no tensors of the CPU, and says so."""
    from sneppx_alg_b200 import _build
    nodes = _build.load_torch()
    assert _build.load_torch() is nodes
    ids, w = torch.tensor([1, 2]), torch.randn(9, 4)
    for args in ((ids, w, 1.0), (ids, w, 1), (ids, w), (1, w, 1.0), (ids, None, 1.0), (w, ids, 1.0)):
        assert nodes.ordinary(*args) is None
    for args in ((ids, w, 1.0, -1, 0), (ids, w, 1.0, -1), (ids, "w", 1.0, -1, 0), ()):
        with pytest.raises(RuntimeError, match="lookup"):
            nodes.lookup(*args)
    with pytest.raises(RuntimeError, match="bind"):
        nodes.bind(1, 2)
