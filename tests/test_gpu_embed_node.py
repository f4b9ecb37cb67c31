"""The embedding's place in torch's graph: in C++, and in Python where that cannot be built. Both by the same kernels."""
import gc
import math
import threading
import weakref

import pytest
import torch

from sneppx_alg_b200 import _build, ops
from sneppx_alg_b200.ops import _lib, embed

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    assert embed._load_nodes()                             # it is built and loaded here
    if request.param == "python":
        monkeypatch.setattr(embed, "_nodes", False)
    return request.param


def _name(y):
    return y.grad_fn.name()


def test_which_one_is_taken(path):
    w = torch.randn(20, 8, device="cuda", requires_grad=True)
    n = _lib.launch_count
    y = ops.embedding(torch.tensor([1, 2], device="cuda"), w)
    assert _name(y) == ("EmbeddingBackward" if path == "native" else "_EmbeddingFnBackward")
    y.sum().backward()
    assert _lib.launch_count == n + 2                      # both count


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (77, 300, 33), (3000, 500, 256), (70000, 900, 16)])
def test_the_two_give_the_same_bits(n, V, d, dtype):
    torch.manual_seed(0)
    assert embed._load_nodes()
    w = torch.randn(V, d, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(n, d, device="cuda").to(dtype)
    for ids in (torch.randint(0, V, (n,), device="cuda"), torch.randint(0, V, (n,), device="cuda", dtype=torch.int32)):
        y = ops.embedding(ids, w, 1.5, padding_idx=-1)
        g, = torch.autograd.grad(y, w, dy)
        z = embed._EmbeddingFn.apply(ids, w, 1.5, V - 1)
        h, = torch.autograd.grad(z, w, dy)
        assert torch.equal(y, z) and torch.equal(g, h)
        with torch.no_grad():
            assert torch.equal(ops.embedding(ids, w, 1.5), z) and not ops.embedding(ids, w).requires_grad


@pytest.mark.parametrize("into", [torch.float32, torch.bfloat16])
def test_main_grad(path, into):
    torch.manual_seed(0)
    w = torch.randn(50, 16, device="cuda").bfloat16().requires_grad_()
    ids, dy = torch.randint(0, 50, (80,), device="cuda"), torch.randn(80, 16, device="cuda").bfloat16()
    w.main_grad = torch.full((50, 16), math.nan, device="cuda", dtype=into)      # without a mark that says whether it has been written
    y = ops.embedding(ids, w)
    y.backward(dy, retain_graph=True)
    want = ops.embedding_backward_(torch.empty_like(w.main_grad), ids, dy)
    assert w._main_grad_written is True and w.grad is None and torch.equal(w.main_grad, want)
    y.backward(dy)
    assert torch.equal(w.main_grad, ops.embedding_backward_(want, ids, dy, add=True))
    assert torch.autograd.grad(ops.embedding(ids, w), w, dy, allow_unused=True)[0] is None
    w.main_grad = None                                     # an engine that has let go of it
    ops.embedding(ids, w).backward(dy)
    assert w.grad is not None
    w.main_grad = torch.zeros(50, 16, device="cuda", dtype=torch.float64)        # of a type that sums are not written in
    w.grad = None
    ops.embedding(ids, w).backward(dy)
    assert w.grad is not None and not w.main_grad.any()


def test_a_graph_is_gone_through_once_unless_kept(path):
    w = torch.randn(50, 16, device="cuda", requires_grad=True)
    ids = torch.randint(0, 50, (8,), device="cuda")
    y = ops.embedding(ids, w)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = ops.embedding(ids, w)
    ids.add_(0)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    y, z = ops.embedding(ids, w), torch.zeros(3, device="cuda", requires_grad=True)
    assert torch.autograd.grad(z.sum(), w, allow_unused=True)[0] is None
    # nothing keeps the ids or the table behind a graph that is gone
    held = weakref.ref(w)
    del w, y
    gc.collect()
    assert held() is None


def test_batched_gradients(path):
    """A batch of incoming gradients at once, as vectorised jacobians take them."""
    w = torch.randn(20, 6, device="cuda", requires_grad=True)
    ids = torch.randint(0, 20, (4,), device="cuda")
    y = ops.embedding(ids, w, 2.0, padding_idx=int(ids[0]))
    dys = torch.randn(5, 4, 6, device="cuda")
    got, = torch.autograd.grad(y, w, dys, is_grads_batched=True, retain_graph=True)
    want = torch.stack([torch.autograd.grad(y, w, dy, retain_graph=True)[0] for dy in dys])
    assert torch.allclose(got, want, rtol=1e-6, atol=1e-6)
    jac = torch.autograd.functional.jacobian(lambda t: ops.embedding(ids, t), w.detach(), vectorize=True)
    assert torch.equal(jac, torch.autograd.functional.jacobian(lambda t: torch.nn.functional.embedding(ids, t), w.detach()))


def test_second_derivatives_and_hooks(path):
    w = torch.randn(11, 24, device="cuda", requires_grad=True)
    ids = torch.randint(0, 11, (3, 7), device="cuda")
    g, = torch.autograd.grad((ops.embedding(ids, w) ** 3).sum(), w, create_graph=True)
    got, = torch.autograd.grad((g ** 2).sum(), w)
    f, = torch.autograd.grad((torch.nn.functional.embedding(ids, w) ** 3).sum(), w, create_graph=True)
    want, = torch.autograd.grad((f ** 2).sum(), w)
    assert torch.allclose(g, f, rtol=1e-5) and torch.allclose(got, want, rtol=1e-5, atol=1e-4)
    seen = []
    w.register_hook(lambda t: seen.append(t.shape) or t * 2)
    with torch.autograd.detect_anomaly(check_nan=True):
        ops.embedding(ids, w).sum().backward()
    assert seen == [w.shape] and torch.equal(w.grad, 2 * torch.bincount(ids.reshape(-1), minlength=11)[:, None].float().expand(11, 24))


def test_backward_passes_of_several_threads(path):
    w = torch.randn(300, 32, device="cuda", requires_grad=True)
    ids, dy = torch.randint(0, 300, (500,), device="cuda"), torch.randn(500, 32, device="cuda")
    want = ops.embedding_backward_(torch.empty_like(w), ids, dy)
    torch.cuda.synchronize()
    out = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(40):
                g, = torch.autograd.grad(ops.embedding(ids, w), w, dy)
            torch.cuda.current_stream().synchronize()
            out.append(g)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert len(out) == 4 and all(torch.equal(g, want) for g in out)


def test_without_a_compiler(monkeypatch):
    """It is said once, and the calls do without."""
    def fails():
        raise RuntimeError("no compiler")

    monkeypatch.setattr(_build, "load_torch", fails)
    monkeypatch.setattr(embed, "_nodes", None)
    w = torch.randn(20, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 2], device="cuda")
    with pytest.warns(RuntimeWarning, match="no compiler"):
        y = ops.embedding(ids, w)
    assert _name(y) == "_EmbeddingFnBackward" and torch.equal(ops.embedding(ids, w), w[ids])
