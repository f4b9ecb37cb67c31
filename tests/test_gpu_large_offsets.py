"""Tables, activations and gradients of more than 2^31 values: the last rows are as right as the first."""
import pytest
import torch

from sneppx_alg_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,width", [(70000, 32768), (140001, 16389)])
def test_8_bit_activations(rows, width):
    x = torch.empty(rows, width, device="cuda", dtype=torch.bfloat16).normal_()
    assert x.numel() > 2 ** 31
    y = ops.unpack_8bit(ops.pack_8bit(x))
    middle = 2 ** 31 // width
    for r in (slice(0, 20), slice(middle - 10, middle + 10), slice(rows - 20, rows)):
        assert torch.equal(y[r], ops.unpack_8bit(ops.pack_8bit(x[r].clone())))


def test_embedding():
    V, d = 600000, 4096
    w = torch.empty(V, d, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_()
    edge = 2 ** 31 // d
    ids = torch.cat([torch.randint(0, V, (3000,), device="cuda"), torch.tensor([V - 1, 0, edge - 1, edge, edge + 1, V - 1], device="cuda")])
    y = ops.embedding(ids, w, 2.0)
    assert torch.equal(y, (w.detach()[ids].float() * 2).to(torch.bfloat16))
    dy = torch.randn(len(ids), d, device="cuda").to(torch.bfloat16)
    g, = torch.autograd.grad(y, w, dy)
    words, at = ids.unique(return_inverse=True)
    want = torch.zeros(len(words), d, device="cuda", dtype=torch.float64).index_add_(0, at, dy.double() * 2)
    mag = torch.zeros_like(want).index_add_(0, at, dy.double().abs() * 2)
    # one rounding to bf16, before it sums of at most 8 values in 32 bits
    assert ((g[words].double() - want).abs() <= 2.0 ** -8 * want.abs() + 10 * 2.0 ** -24 * mag).all()
    assert sum(int(g[v:v + 50000].any(1).sum()) for v in range(0, V, 50000)) == len(words)          # and zeros elsewhere
    into = torch.ones(V, d, device="cuda")
    ops.embedding_backward_(into, ids, dy, 2.0, add=True)
    assert ((into[words].double() - 1 - want).abs() <= 11 * 2.0 ** -24 * (mag + 1)).all()
    assert sum(int((into[v:v + 50000] != 1).any(1).sum()) for v in range(0, V, 50000)) == len(words)
    ops.check_status()
