"""Per-token vocabulary loss on the GPU against the definition in 64 bits.

Bounds. A logit is a sum of d products of bf16 numbers, exact in 32 bits, whose additions lose at most 2^-23 of the magnitudes' sum S each (the tensor cores
cut rather than round): ez = d 2^-23 S. The soft cap adds 2^-21 of the cap (exponential and quotient). lse then has ez, a relative error of the sum of
exponentials (each a few 2^-23, at most 300 additions one after another: 300 x 2^-24 < 2e-5) and its rounding; nll the target's ez more. dz has a
relative error of ez + elsa from its exponential and half a step of bf16, 2^-8; dh and dw add up its errors times the other factor, one rounding of
2^-24 for each addition, and half a step of their own.
"""
import ctypes
import math

import pytest
import torch

from sneppx_alg_b200 import ops
from sneppx_alg_b200.ops import _lib
from sneppx_alg_b200.ops._lib import KernelTimeout

pytestmark = pytest.mark.gpu


def _inputs(T, V, d, seed, sure=6.0, ignored=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(V, d, generator=g, device="cuda") / math.sqrt(d)).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), generator=g, device="cuda")
    h = (torch.randn(T, d, generator=g, device="cuda") + sure * torch.rand(T, 1, generator=g, device="cuda") * w[t].float()).to(torch.bfloat16)
    gn, gz = torch.randn(T, generator=g, device="cuda"), 0.1 * torch.randn(T, generator=g, device="cuda")
    return h, w, torch.where(torch.rand(T, generator=g, device="cuda") < ignored, -100, t), gn, gz


def _want(h, w, t, gn, gz, cap):
    """64-bit results, and what bounds their errors."""
    h, w = h.double(), w.double()
    T, d = h.shape
    raw = h @ w.t()
    z = cap * torch.tanh(raw / cap) if cap else raw
    lse = torch.logsumexp(z, 1)
    ok = t >= 0
    at = t.clamp(min=0)[:, None]
    nll = torch.where(ok, lse - z.gather(1, at).squeeze(1), 0.0)
    ez = d * 2.0 ** -23 * (h.abs() @ w.abs().t()).amax(1) + 2.0 ** -21 * cap
    el = ez + 2e-5 + 2.0 ** -23 * lse.abs()
    p = torch.exp(z - lse[:, None])
    a, b = (gn.double() * ok + gz.double())[:, None], (gn.double() * ok)[:, None]
    slope = 1 - (z / cap) ** 2 if cap else torch.ones_like(z)
    hot = torch.zeros_like(z).scatter_(1, at, 1.0)
    dz = (a * p - b * hot) * slope
    # errors of the exponential and of the slope (2 |z / cap| ez / cap), then the rounding to bf16
    mag = a.abs() * p + b.abs() * hot
    edz = mag * ((ez + el)[:, None] * 1.5 + 2.0 ** -21 + (4 * ez[:, None] / cap + 2.0 ** -20 if cap else 0.0)) + 2.0 ** -8 * dz.abs()
    out = dict(nll=nll, lse=lse, dh=dz @ w, dw=dz.t() @ h)
    tol = dict(nll=el + ez + 2.0 ** -23 * nll.abs(), lse=el,
               dh=edz @ w.abs() + w.shape[0] * 2.0 ** -23 * (dz.abs() @ w.abs()) + 2.0 ** -8 * out["dh"].abs(),
               dw=edz.t() @ h.abs() + T * 2.0 ** -23 * (dz.abs().t() @ h.abs()) + 2.0 ** -8 * out["dw"].abs())
    return out, tol


def _check(got, want, tol):
    for k, v in got.items():
        assert torch.isfinite(v).all() and v.shape == want[k].shape
        off = (v.double() - want[k]).abs()
        assert (off <= tol[k] + 1e-30).all(), (k, float((off - tol[k]).max()), float(off.max()))


def _run(h, w, t, gn, gz, cap, piece=0):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    nll, lse = ops.linear_token_loss(h, w, t, softcap=cap, piece=piece)
    dh, dw = torch.autograd.grad((nll, lse), (h, w), (gn, gz))
    ops.check_status()
    return dict(nll=nll.detach(), lse=lse.detach(), dh=dh, dw=dw)


@pytest.mark.parametrize("cap", [0.0, 3.0])
@pytest.mark.parametrize("T,V,d", [(1, 1, 8), (1, 300, 64), (3, 256, 72), (77, 1000, 256), (128, 257, 64), (129, 128, 640), (255, 4099, 128), (256, 512, 64),
                                   (257, 777, 192), (300, 33, 1024), (1000, 5000, 96), (520, 3001, 100), (33, 700, 7),
                                   (600, 20000, 256)])
def test_values_and_gradients(T, V, d, cap):
    x = _inputs(T, V, d, 1)
    got = _run(*x, cap)
    want, tol = _want(*x, cap)
    _check(got, want, tol)
    assert torch.equal(got["nll"][x[2] < 0], torch.zeros_like(got["nll"][x[2] < 0]))
    again = _run(*x, cap)
    assert all(torch.equal(got[k], again[k]) for k in got)          # the same bits each time


@pytest.mark.parametrize("piece", [1, 256, 512, 700, 4096])
def test_pieces_of_the_vocabulary(piece):
    x = _inputs(100, 2003, 128, 2)
    want, tol = _want(*x, 0.0)
    got = _run(*x, 0.0, piece)
    # the sums of dh over pieces are held in 32 bits: a rounding for each
    tol["dh"] = tol["dh"] + 8 * 2.0 ** -24 * want["dh"].abs().amax()
    _check(got, want, tol)


@pytest.mark.parametrize("T,V", [(700, 1300), (64, 20000)])
def test_which_gradients_are_asked_for(T, V):
    h, w, t, gn, gz = _inputs(T, V, 128, 3)
    full = _run(h, w, t, gn, gz, 0.0)
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
    nll, _ = ops.linear_token_loss(hg, w, t)
    assert torch.equal(nll, full["nll"])
    want, tol = _want(h, w, t, gn, torch.zeros_like(gz), 0.0)
    dh, = torch.autograd.grad(nll, hg, gn)
    _check(dict(dh=dh), want, tol)
    nll, _ = ops.linear_token_loss(h, wg, t)
    dw, = torch.autograd.grad(nll, wg, gn)
    _check(dict(dw=dw), want, tol)
    _, lse = ops.linear_token_loss(hg, wg, t)
    want, tol = _want(h, w, t, torch.zeros_like(gn), gz, 0.0)
    dh, dw = torch.autograd.grad(lse, (hg, wg), gz)
    _check(dict(dh=dh, dw=dw), want, tol)
    nll, lse = ops.linear_token_loss(h, w, t)
    assert not nll.requires_grad and not lse.requires_grad


@pytest.mark.parametrize("into", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [640, 1001])
def test_main_grad_is_written_and_added_to(V, into):
    h, w, t, gn, gz = _inputs(200, V, 128, 4)
    want, tol = _want(h, w, t, gn, gz, 0.0)
    w = w.detach().requires_grad_()
    w.main_grad, w._main_grad_written = torch.full((V, 128), math.nan, device="cuda", dtype=into), False
    half = torch.finfo(into).eps / 2
    for k in (1, 2):
        nll, lse = ops.linear_token_loss(h, w, t, piece=256)
        torch.autograd.backward((nll, lse), (gn, gz))
        assert w.grad is None and w._main_grad_written
        off = (w.main_grad.double() - k * want["dw"]).abs()
        assert (off <= k * tol["dw"] + 2 * half * k * want["dw"].abs()).all()


def test_layouts():
    """Rows of a wider tensor, an odd base address, a transposed weight, a batch of sequences with shifted targets."""
    g = torch.Generator(device="cuda").manual_seed(5)
    big = torch.randn(4, 60, 200, generator=g, device="cuda").to(torch.bfloat16)
    wide = (torch.randn(900, 300, generator=g, device="cuda") / 12).to(torch.bfloat16)
    ids = torch.randint(0, 900, (4, 61), generator=g, device="cuda")
    t = ids[:, 1:]                                           # not contiguous
    for h, w in ((big[..., 8:136], wide[:, 16:144]), (big[..., 3:131], wide[:, 5:133]), (big[:, :, :128], wide[:, :128].t().contiguous().t()),
                 (big[:, 1:, :128], wide[:, 100:228])):
        tt = t[:, :h.shape[1]]
        nll, lse = ops.linear_token_loss(h, w, tt)
        T = tt.numel()
        want, tol = _want(h.reshape(T, 128), w, tt.reshape(T), torch.ones(T, device="cuda"), torch.zeros(T, device="cuda"), 0.0)
        assert nll.shape == tt.shape
        _check(dict(nll=nll.reshape(-1), lse=lse.reshape(-1)), want, tol)
        hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
        dh, dw = torch.autograd.grad(ops.linear_token_loss(hg, wg, tt)[0].sum(), (hg, wg))
        _check(dict(dh=dh.reshape(T, 128), dw=dw), want, tol)
    # a single token out of wider rows with an odd pitch, a vocabulary of one word
    one = torch.randn(3, 131, generator=g, device="cuda").to(torch.bfloat16)
    for h, w in ((one[1:2, :128], wide[:, :128]), (one[:, :128], one[2:3, :128])):
        t = torch.zeros(h.shape[0], dtype=torch.int64, device="cuda")
        hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
        nll, lse = ops.linear_token_loss(hg, wg, t)
        dh, dw = torch.autograd.grad(nll.sum(), (hg, wg))
        want, tol = _want(h, w, t, torch.ones(len(t), device="cuda"), torch.zeros(len(t), device="cuda"), 0.0)
        _check(dict(nll=nll, lse=lse, dh=dh, dw=dw), want, tol)
    ops.check_status()


def test_everything_ignored_and_empty():
    h, w, _, gn, gz = _inputs(90, 500, 64, 6)
    t = torch.full((90,), -100, device="cuda")
    got = _run(h, w, t, gn, torch.zeros_like(gz), 0.0)
    assert not got["nll"].any() and not got["dh"].any() and not got["dw"].any()
    hg, wg = h[:0].detach().requires_grad_(), w.detach().requires_grad_()
    nll, lse = ops.linear_token_loss(hg, wg, t[:0])
    (nll.sum() + lse.sum()).backward()
    assert hg.grad.shape == (0, 64) and not wg.grad.any()


def test_targets_out_of_range_count_as_ignored_and_are_reported():
    h, w, t, gn, gz = _inputs(40, 500, 64, 7, ignored=0.0)
    bad = t.clone()
    bad[3], bad[4], bad[5] = 500, -1, 2 ** 40
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
    nll, lse = ops.linear_token_loss(hg, wg, bad)
    with pytest.raises(KernelTimeout):
        ops.check_status()
    dh, dw = torch.autograd.grad((nll, lse), (hg, wg), (gn, gz))
    t[3:6] = -100
    good = _run(h, w, t, gn, gz, 0.0)
    assert torch.equal(nll, good["nll"]) and torch.equal(lse, good["lse"]) and torch.equal(dh, good["dh"]) and torch.equal(dw, good["dw"])
    # a border value of ignore_index
    nll, _ = ops.linear_token_loss(h, w, torch.where(t < 0, 0, t), ignore_index=0)
    ops.check_status()
    assert not nll[(t <= 0)].any()


def test_other_types_on_the_gpu():
    """fp32 takes the PyTorch form: the same values, the same answer to targets out of range."""
    h, w, t, gn, gz = _inputs(30, 300, 64, 11)
    nll, lse = ops.linear_token_loss(h.float(), w.float(), t)
    want, tol = _want(h, w, t, gn, gz, 0.0)
    _check(dict(nll=nll, lse=lse), want, tol)
    ops.check_status()
    t[3] = 300
    nll, _ = ops.linear_token_loss(h.float(), w.float(), t)
    with pytest.raises(KernelTimeout):
        ops.check_status()
    assert nll[3] == 0 and torch.isfinite(nll).all()


def test_large_logits_and_infinities():
    h, w, t, _, _ = _inputs(50, 400, 64, 8)
    h = h * 300                                             # logits up to some thousands: exponentials of differences only
    nll, lse = ops.linear_token_loss(h, w, t)
    want, tol = _want(h, w, t, torch.zeros(50, device="cuda"), torch.zeros(50, device="cuda"), 0.0)
    _check(dict(nll=nll, lse=lse), want, tol)
    h[7, 3] = float("nan")
    nll2, lse2 = ops.linear_token_loss(h, w, t)
    rest = torch.arange(50, device="cuda") != 7
    assert torch.isnan(lse2[7]) and torch.equal(lse2[rest], lse[rest]) and torch.equal(nll2[rest], nll[rest])
    ops.check_status()


def test_other_stream_and_captured_graph():
    h, w, t, gn, gz = _inputs(200, 3000, 128, 9)
    want = ops.linear_token_loss(h, w, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_token_loss(h, w, t)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs, x = [torch.cuda.CUDAGraph() for _ in range(2)], [], h.clone()
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(ops.linear_token_loss(x, w, t))
    for k in (1.0, 0.5):
        x.copy_(h * k)
        for gr in graphs:
            gr.replay()
        want = ops.linear_token_loss(x, w, t)
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))
    ops.check_status()


@pytest.mark.parametrize("T,V,d", [(700, 1318, 328), (40, 5000, 1000), (2000, 700, 744), (257, 513, 3848), (5, 300, 24), (300, 4000, 136), (64, 9000, 264)])
def test_widths_between_multiples_of_64(T, V, d):
    x = _inputs(T, V, d, 21)
    got = _run(*x, 0.0)
    want, tol = _want(*x, 0.0)
    _check(got, want, tol)


@pytest.mark.parametrize("into", [torch.float32, torch.bfloat16])
def test_main_grad_of_a_width_between_multiples_of_64(into):
    h, w, t, gn, gz = _inputs(300, 1001, 328, 22)
    want, tol = _want(h, w, t, gn, gz, 0.0)
    w = w.detach().requires_grad_()
    w.main_grad = torch.full((1001, 328), math.nan, device="cuda", dtype=into)
    nll, lse = ops.linear_token_loss(h, w, t)
    assert torch.autograd.grad((nll, lse), w, (gn, gz), allow_unused=True)[0] is None
    _check(dict(dw=w.main_grad.float()), want, tol)


@pytest.mark.parametrize("M,N,K", [(72, 40, 64), (300, 200, 136), (1000, 328, 700), (264, 3848, 77), (520, 8, 300)])
@pytest.mark.parametrize("a_mn,b_mn", [(False, True), (True, False), (True, True)])
def test_products_of_ragged_operands(M, N, K, a_mn, b_mn):
    """Operands with K along their rows, whose rows are no whole groups of 64; behind each row of the storage stands NaN."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    full = [torch.full((r, c + 8 - c % 8 + 8), math.nan, device="cuda", dtype=torch.bfloat16) for r, c in ((K, M) if a_mn else (M, K), (K, N) if b_mn else (N, K))]
    a, b = (f[:, :c] for f, c in zip(full, (M if a_mn else K, N if b_mn else K)))
    for x in (a, b):
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
    d = torch.full((M, N), math.nan, device="cuda")
    p = _lib.SxGemmArgs()
    p.A, p.B, p.D, p.M, p.N, p.K, p.batch = a.data_ptr(), b.data_ptr(), d.data_ptr(), M, N, K, 1
    p.lda, p.ldb, p.ldd, p.a_mn, p.b_mn, p.out_fp32 = a.stride(0), b.stride(0), N, a_mn, b_mn, 1
    p.alpha, p.flags, p.status = 1.0, 2, _lib.status_ptr(d)
    _lib.call("sx_gemm_bf16", ctypes.byref(p), _lib.stream())
    ops.check_status()
    A, B = (a.T if a_mn else a).double(), (b if b_mn else b.T).double()
    assert ((d.double() - A @ B).abs() <= K * 2.0 ** -23 * (A.abs() @ B.abs())).all()       # K additions, each cut by at most 2^-23 of what is added up


@pytest.mark.parametrize("T,V,d", [(2, 1244, 72), (3, 1517, 656), (40, 5000, 1000), (300, 700, 64)])
def test_losses_of_tokens_that_the_model_is_sure_of(T, V, d):
    """nll down to 1e-9 is right to a part of itself, not of the logits: it is a sum of the other words' exponentials over the target's, each off by e^(2 ez)."""
    h, w, t, _, _ = _inputs(T, V, d, 23, ignored=0.0)
    h = (h + torch.linspace(6, 28, T, device="cuda")[:, None] * w[t].float() / (w[t].float() ** 2).sum(1, keepdim=True)).to(torch.bfloat16)
    nll, lse = ops.linear_token_loss(h, w, t)
    z = h.double() @ w.double().t()
    own = z.gather(1, t[:, None])
    want = torch.log1p(torch.exp(z - own).scatter(1, t[:, None], 0.0).sum(1))
    ez = d * 2.0 ** -23 * (h.double().abs() @ w.double().abs().t()).amax(1)
    # 2^-18: exponentials and their sums, a few 2^-23 each, and at most 30 additions one after another
    assert ((nll.double() - want).abs() <= want * (torch.expm1(2 * ez) + 2.0 ** -18)).all()
    assert ((lse.double() - torch.logsumexp(z, 1)).abs() <= ez + 2.0 ** -18 + 2.0 ** -23 * lse.abs()).all()
    assert want.min() < 1e-3


@pytest.mark.parametrize("d", [64, 1000])
def test_soft_cap_keeps_nan(d):
    """A word whose weights are NaN, beside logits on both sides of 0.6 of the cap; a hidden state that holds NaN, and one with infinities of both signs."""
    h, w, t, gn, gz = _inputs(40, 400, d, 31, ignored=0.0)
    clean = _run(h, w, t, gn, gz, 3.0)
    bad = w.clone()
    bad[77] = math.nan
    got = _run(h, bad, t, gn, gz, 3.0)
    assert torch.isnan(got["lse"]).all() and torch.isnan(got["nll"]).all() and torch.isnan(got["dh"]).all()
    for k in (0, 1):
        x = h.clone()
        x[7, :2] = torch.tensor([math.nan, 1.0] if k else [math.inf, -math.inf])
        wz = w.clone()
        wz[:, :2] = 0.5
        base, got = _run(h, wz, t, gn, gz, 3.0), _run(x, wz, t, gn, gz, 3.0)
        rest = torch.arange(40, device="cuda") != 7
        assert torch.isnan(got["lse"][7]) and torch.isnan(got["nll"][7])
        assert torch.isnan(got["dh"][7]).all()
        assert all(torch.equal(got[i][rest], base[i][rest]) for i in ("nll", "lse", "dh"))
    assert torch.isfinite(clean["lse"]).all()


@pytest.mark.parametrize("M", [4, 300])
def test_soft_capped_product_keeps_nan(M):
    """The same cap in the epilogues of the products."""
    from sneppx_alg_b200.ops.gemm import SoftCap
    x, w = (4 * torch.randn(M, 256, device="cuda")).to(torch.bfloat16), torch.randn(512, 256, device="cuda").to(torch.bfloat16)
    want = ops.gemm(x, w, act=SoftCap(30.0))
    w[5] = math.nan
    got = ops.gemm(x, w, act=SoftCap(30.0))
    rest = torch.arange(512, device="cuda") != 5
    assert torch.isnan(got[:, 5]).all() and torch.equal(got[:, rest], want[:, rest])


@pytest.mark.parametrize("cap", [0.0, 40.0])
@pytest.mark.parametrize("T,V,d", [(2, 1244, 72), (40, 5000, 1000), (300, 700, 64), (70, 3000, 4096)])
def test_gradients_of_tokens_that_the_model_is_sure_of(T, V, d, cap):
    """A target's dz is g_nll (p - 1) + g_lse p times the cap's slope, right to a part of itself where p is next to 1. Each token in its own direction: dw of a
    word that is one token's target and nobody else's is that token's dz times h."""
    g = torch.Generator(device="cuda").manual_seed(29)
    w = (torch.randn(V, d, generator=g, device="cuda") / math.sqrt(d)).to(torch.bfloat16)
    t = torch.randperm(V, generator=g, device="cuda")[:T]
    own = w[t].float()
    up = torch.linspace(8, 20, T, device="cuda")[:, None]
    h = (torch.randn(T, d, generator=g, device="cuda") * 0.1 + up * own / (own ** 2).sum(1, keepdim=True)).to(torch.bfloat16)
    gn, gz = torch.rand(T, generator=g, device="cuda") + 0.5, 1e-3 * torch.rand(T, generator=g, device="cuda")
    for zl in (torch.zeros_like(gz), gz):
        got = _run(h, w, t, gn, zl, cap)
        h64, w64 = h.double(), w.double()
        raw = h64 @ w64.t()
        z = cap * torch.tanh(raw / cap) if cap else raw
        others = torch.logsumexp(z.scatter(1, t[:, None], -math.inf), 1)
        zt = z.gather(1, t[:, None]).squeeze(1)
        nll = torch.nn.functional.softplus(others - zt, threshold=1e9)
        assert nll.min() < 1e-3
        slope = 1 - (z / cap) ** 2 if cap else torch.ones_like(z)
        p = torch.exp(z - (zt + nll)[:, None])
        rest = ((gn + zl).double()[:, None] * p)
        dz = rest.scatter(1, t[:, None], (gn.double() * torch.expm1(-nll) + zl.double() * torch.exp(-nll))[:, None]) * slope
        ez = d * 2.0 ** -23 * (h64.abs() @ w64.abs().t()).amax(1) + 2.0 ** -21 * cap
        # of dz itself: exponentials of logits off by ez, in the soft cap's slope 2 |z / cap| ez / cap and 2^-20, half a step of bf16; of the target's two
        # parts each, which may cancel. 2^-17: sums and functions, a few 2^-23 each and at most 30 additions one after another
        part = torch.expm1(3 * ez)[:, None] + 2.0 ** -17 + ((4 * ez[:, None] / cap + 2.0 ** -20) / slope.clamp(min=1e-9) if cap else 0.0)
        mag = rest.scatter(1, t[:, None], (gn.double() * -torch.expm1(-nll) + zl.double() * torch.exp(-nll))[:, None]) * slope
        edz = mag * part + 2.0 ** -8 * dz.abs()
        tol = dict(dh=edz @ w64.abs() + V * 2.0 ** -23 * (dz.abs() @ w64.abs()), dw=edz.t() @ h64.abs() + T * 2.0 ** -23 * (dz.abs().t() @ h64.abs()))
        want = dict(dh=dz @ w64, dw=dz.t() @ h64)
        _check({k: got[k] for k in tol}, want, {k: tol[k] + 2.0 ** -8 * want[k].abs() for k in tol})


def test_losses_may_be_written_over():
    """What backward needs of nll is its own."""
    h, w, t, gn, gz = _inputs(50, 400, 64, 30)
    want = _run(h, w, t, gn, torch.zeros_like(gz), 0.0)
    hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
    nll, _ = ops.linear_token_loss(hg, wg, t)
    nll.mul_(2.0)
    dh, dw = torch.autograd.grad(nll, (hg, wg), gn / 2)
    assert torch.equal(dh, want["dh"]) and torch.equal(dw, want["dw"])


@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_infinite_logits(cap):
    """A hidden state that overflowed, and products that do: lse, nll and gradients are infinite and NaN where the definition's are."""
    h, w, t, gn, gz = _inputs(60, 700, 64, 32, ignored=0.0)
    w[:, 3] = torch.where(w[:, 3] == 0, 0.25, w[:, 3])
    h[5, 3], h[6, 3], h[7] = math.inf, -math.inf, 0.0
    big = torch.finfo(torch.bfloat16).max
    w[100, :2] = big
    h[:, :2] = 0.0                                          # the word's logit is 0 but for one token, where it overflows
    h[9, 0], h[10, 0] = big, -big
    t[5], t[9] = 300, 100
    got = _run(h, w, t, gn, gz, cap)
    hg, wg = h.double().requires_grad_(), w.double().requires_grad_()
    z = (hg @ wg.t()).float().double()                       # where 32 bits overflow
    z = cap * torch.tanh(z / cap) if cap else z
    lse = torch.logsumexp(z, 1)
    nll = lse - z.gather(1, t[:, None]).squeeze(1)
    for k, v in dict(nll=nll, lse=lse).items():
        assert torch.equal(torch.isnan(got[k]), torch.isnan(v)), k
        assert torch.equal(torch.isposinf(got[k]), torch.isposinf(v)), k
    sure = torch.isfinite(nll)
    if not cap:
        assert torch.isposinf(lse[[5, 6]]).all() and torch.isnan(nll[9])
    # tokens whose lse is finite have finite gradients, the others none
    finite = torch.isfinite(lse) & torch.isfinite(hg).all(1)
    assert torch.isfinite(got["dh"][finite & sure][:, 2:]).all()
    if not cap:
        assert not torch.isfinite(got["dh"][~finite]).all(1).any()


@pytest.mark.parametrize("size", [1e3, 1e5, 1e8, 1e20, 1e36])
def test_logits_of_any_finite_size(size):
    """Losses of logits up to the type's range: right to what 32 bits hold of a logit, finite, and dz that of the word that stands out."""
    h, w, t, _, _ = _inputs(50, 700, 64, 33, ignored=0.0)
    h = (h.float() * size).to(torch.bfloat16)
    gn, gz = torch.ones(50, device="cuda"), torch.zeros(50, device="cuda")
    got = _run(h, w, t, gn, gz, 0.0)
    h64, w64 = h.double(), w.double()
    z = h64 @ w64.t()
    ez = 64 * 2.0 ** -23 * (h64.abs() @ w64.abs().t()).amax(1)
    lse = torch.logsumexp(z, 1)
    nll = lse - z.gather(1, t[:, None]).squeeze(1)
    assert ((got["lse"].double() - lse).abs() <= ez + 2e-5 + 2.0 ** -23 * lse.abs()).all()
    assert ((got["nll"].double() - nll).abs() <= 2 * ez + 2e-5 + 2.0 ** -23 * nll.abs()).all()
    # where one word stands out by more than the errors of two logits, dz is 1 for it and -1 for the target, or nothing
    top = z.topk(2, 1).values
    clear = top[:, 0] - top[:, 1] > 2 * ez + 120
    right = z.argmax(1) == t
    dh = torch.where(right[:, None], 0.0, w64[z.argmax(1)] - w64[t])
    assert clear.float().mean() > (0.5 if size > 2e3 else 0.1) and torch.isfinite(got["dh"]).all()
    off = (got["dh"].double() - dh).abs()[clear]
    assert (off <= 2.0 ** -7 * (w64[z.argmax(1)].abs() + w64[t].abs())[clear]).all()


@pytest.mark.parametrize("T,V,d", [(4, 16377, 640), (64, 3000, 4096), (256, 4000, 768), (200, 5000, 2304)])
def test_few_tokens_lose_little(T, V, d):
    """The tensor cores cut what they add to an accumulator, by as much as there are products in a part of the sum: of up to 256 tokens a part has half as many
    as of more, so that the same tokens' lse is off by about half of what it is among 600 (by less than three quarters, which leaves room for the rounding of
    lse itself, 2^-24 of it, on both sides)."""
    g = torch.Generator(device="cuda").manual_seed(41)
    few = many = 0.0
    for _ in range(8):
        w = (torch.randn(V, d, generator=g, device="cuda") / math.sqrt(d)).to(torch.bfloat16)
        t = torch.randint(0, V, (600,), generator=g, device="cuda")
        h = (torch.randn(600, d, generator=g, device="cuda") + 14 * torch.rand(600, 1, generator=g, device="cuda") * w[t].float()).to(torch.bfloat16)
        want = torch.logsumexp(h[:T].double() @ w.double().t(), 1)
        few += float((ops.linear_token_loss(h[:T], w, t[:T])[1].double() - want).square().sum())
        many += float((ops.linear_token_loss(h, w, t)[1][:T].double() - want).square().sum())
    assert math.sqrt(few) < 0.75 * math.sqrt(many)
