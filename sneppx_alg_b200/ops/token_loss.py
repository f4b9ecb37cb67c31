"""Per-token losses of a vocabulary projection without the logits (csrc/vocab_loss.cu). bf16 CUDA tensors take the kernels;
``linear_token_loss_reference`` states the same in PyTorch and serves everything else. The reference computes a softmax and its gradient over the
logits of a batch (kernel/cuda/autodiff_cuda.cu:519-608)."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _lib
from . import debug as _dbg
from .gemm import gemm

# Bytes of dz (bf16 gradients of the logits of one piece of the vocabulary) that backward holds where the caller does not say how wide a piece is.
PIECE_BYTES = 256 << 20


def linear_token_loss_reference(h, w, target, ignore_index=-100, softcap=0.0):
    ct = torch.promote_types(torch.promote_types(h.dtype, w.dtype), torch.float32)
    z = F.linear(h.to(ct), w.to(ct))
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    lse = torch.logsumexp(z, -1)
    valid = target != ignore_index
    zt = z.gather(-1, torch.where(valid, target, 0).unsqueeze(-1)).squeeze(-1)
    return torch.where(valid, lse - zt, 0.0), lse


def _rows16(t, d):
    """t [n, >= d] as the tensor maps take it: d columns, a multiple of 8 (padded with zeros), rows 16-byte aligned."""
    if t.shape[1] != d:
        return F.pad(t, (0, d - t.shape[1]))
    if t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < d or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


class _VocabSum:
    """dh = sum over pieces of the vocabulary of dz [T, n] times their rows of w [n, d], in 32 bits. The product has T d results only, and for narrow models
    these are too few tiles of 256 x 256 for 74 pairs of SMs: the vocabulary is then cut once more, into ``splits`` parts with sums of their own
    that run as one batch (4095 tokens of 768: 48 tiles, 3 x 48 fill two rounds)."""

    def __init__(self, T, d, n, dev):
        tiles = -(-T // 256) * -(-d // 256)
        use = lambda s: tiles * s / (74 * -(-tiles * s // 74))  # noqa: E731
        # from 512 rows on (smaller products have kernels of their own) and in parts of 2048 at least: shorter ones are bound by the sums' traffic
        fit = [s for s in range(1, 9) if s == 1 or (T >= 512 and d >= 256 and d % 64 == 0 and n // s >= 2048)]
        self.splits = next((s for s in fit if use(s) >= 0.9), max(fit, key=use))
        self.T, self.d, self.one = T, d, None
        self.acc = torch.empty(self.splits, T, d, dtype=torch.float32, device=dev)
        self.written = False

    def columns(self, n):
        """Columns that dz of n words has for ``add``: the parts are equal and whole groups of 8, those of dz whole groups of 64 in all."""
        return (-(-n // (8 * self.splits)) * 8 * self.splits + 63) // 64 * 64

    def add(self, z, w):
        """z [T, columns(n)], zeros from n on; w [n, d]. Pieces of one call are equally wide but for the last."""
        n, s = w.shape[0], self.splits
        k = -(-n // (8 * s)) * 8
        if s * k != n:                       # a last piece: zeros on both sides
            w = F.pad(w, (0, 0, 0, s * k - n))
        more = dict(c=self.acc, beta=1.0) if self.written else {}
        gemm(z.as_strided((s, self.T, k), (k, z.stride(0), 1)), w.unflatten(0, (s, k)), b_mn=True, out=self.acc, **more)
        self.written = True

    def result(self):
        out = self.acc.new_empty((self.T, self.d), dtype=torch.bfloat16)
        _lib.entry("sx_vocab_loss_sum", "ppilp")(self.acc.data_ptr(), out.data_ptr(), self.splits, self.T * self.d, _lib.here(out))
        return out


def _forward(h, w, target, ignore_index, softcap):
    """(nll, lse) in target's shape."""
    T, V, d = target.numel(), w.shape[0], (w.shape[1] + 7) // 8 * 8
    h2, w2 = _rows16(h.reshape(-1, h.shape[-1]), d), _rows16(w, d)
    tgt = target.contiguous()
    nll, lse = (h2.new_empty(target.shape, dtype=torch.float32) for _ in range(2))
    scratch = h2.new_empty(T * (2 * -(-V // 256) + 1), dtype=torch.float32)          # pairs of a row's maximum and sum, and its target's logit
    with _lib.on_device(h):
        _lib.entry("sx_vocab_loss_fwd", "plplpllilfpppppp")(
            h2.data_ptr(), h2.stride(0), w2.data_ptr(), w2.stride(0), tgt.data_ptr(), T, V, d, ignore_index, softcap, scratch.data_ptr(),
            scratch.data_ptr() + 8 * T * -(-V // 256), nll.data_ptr(), lse.data_ptr(), _lib.status_ptr(h), _lib.here(h))
    return nll, lse


class _TokenLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, target, ignore_index, softcap, piece):
        nll, lse = _forward(h, w, target, ignore_index, softcap)
        tgt = target.reshape(-1).contiguous()
        ctx.save_for_backward(h, w, tgt, lse)
        ctx.w, ctx.meta = w, (ignore_index, softcap, piece)
        ctx.set_materialize_grads(False)
        return nll, lse

    @staticmethod
    @_lib.once
    def backward(ctx, g_nll, g_lse):
        none = (None,) * 6
        if g_nll is None and g_lse is None:
            return none
        h, w, tgt, lse = ctx.saved_tensors
        ignore_index, softcap, piece = ctx.meta
        need_h, need_w = ctx.needs_input_grad[:2]
        T, V, d0 = tgt.numel(), w.shape[0], w.shape[1]
        d = (d0 + 7) // 8 * 8
        dev = h.device
        with _lib.on_device(h):
            rows = (T + 7) // 8 * 8                    # the reduction of dw is over whole groups of 8 rows; those behind the last token are zeros
            h2 = h.reshape(-1, d0)
            h2 = F.pad(h2, (0, d - d0, 0, rows - T)) if need_w and rows != T else _rows16(h2, d)
            w2 = _rows16(w, d)
            gn, gz = (None if g is None else g.reshape(-1).float().contiguous() for g in (g_nll, g_lse))
            if not piece:
                piece = max(1024, PIECE_BYTES // (2 * rows))
            piece = min((piece + 255) // 256 * 256, V)
            sums = _VocabSum(T, d, piece, dev) if need_h else None
            if sums is not None and piece < V:         # equal parts of whole pieces
                piece = max(1, piece // (256 * sums.splits)) * 256 * sums.splits
            width = sums.columns if sums is not None else lambda n: (n + 63) // 64 * 64
            dz = torch.empty(rows * width(piece), dtype=torch.bfloat16, device=dev)
            mg = getattr(ctx.w, "main_grad", None) if need_w and d == d0 else None
            if mg is not None and (mg.dtype not in (torch.bfloat16, torch.float32) or mg.stride(1) != 1):
                mg = None
            add = mg is not None and getattr(ctx.w, "_main_grad_written", False)
            # rows behind the vocabulary's end: the product over a last piece writes whole groups of 64 rows
            full = torch.empty((V + 63) // 64 * 64, d, dtype=torch.bfloat16, device=dev) if need_w and mg is None else None
            for v0 in range(0, V, piece):
                v1 = min(V, v0 + piece)
                ld = width(v1 - v0)
                z = dz[: rows * ld].view(rows, ld)
                _lib.entry("sx_vocab_loss_grad", "plplpllilfppppllllpp")(
                    h2.data_ptr(), h2.stride(0), w2.data_ptr(), w2.stride(0), tgt.data_ptr(), T, V, d, ignore_index, softcap, lse.data_ptr(),
                    gn.data_ptr() if gn is not None else 0, gz.data_ptr() if gz is not None else 0, z.data_ptr(), ld, rows, v0, v1,
                    _lib.status_ptr(h), _lib.here(h))
                if need_h:
                    sums.add(z[:T], w2[v0:v1])
                if need_w and full is not None:
                    n64 = (v1 - v0 + 63) // 64 * 64
                    gemm(z[:, :n64], h2, a_mn=True, b_mn=True, out=full[v0: v0 + n64])
                elif need_w:
                    gemm(z[:, : v1 - v0], h2, a_mn=True, b_mn=True, out=mg[v0:v1], c=mg[v0:v1] if add else None, beta=1.0 if add else 0.0)
            dh = sums.result() if need_h else None
            dw = full[:V] if full is not None else None
        if need_h:
            dh = (dh if d == d0 else dh[:, :d0]).reshape(h.shape)
        if mg is not None:
            ctx.w._main_grad_written = True
        elif need_w and d != d0:
            dw = dw[:, :d0].contiguous()
        return dh, dw, None, None, None, None


def linear_token_loss(h, w, target, ignore_index=-100, softcap=0.0, piece=0):
    """(nll, lse) of every token, fp32: logits z = h @ w^T, with ``softcap`` c > 0 c * tanh(z / c); lse = log sum exp z over the vocabulary, nll = lse
    - z[target], 0 where target is ``ignore_index``. h [..., d], w [V, d], target [...] int64. Both results are differentiable (a z-loss is a function of
    lse), with any weight for each token; the logits exist in tiles only.

    Backward holds dz for ``piece`` columns of the vocabulary at a time (rounded up to 256; 0: as many as fit 256 MiB) and computes the logits again:
    it trades a fourth product of h and w for logits that ``linear_cross_entropy`` holds a chunk of, and need not know the tokens' weights beforehand.
    Where w carries ``main_grad`` its gradient is written or added there and ``.grad`` stays empty. On the GPU a target outside [0, V) counts as
    ignored and sets the status word (``check_status`` raises); on the CPU it raises at once."""
    if w.dim() != 2 or h.dim() == 0 or h.shape[-1] != w.shape[1]:
        raise ValueError(f"linear_token_loss: hidden states {tuple(h.shape)} and weights {tuple(w.shape)} do not fit")
    if target.shape != h.shape[:-1]:
        raise ValueError(f"linear_token_loss: targets {tuple(target.shape)} for hidden states {tuple(h.shape)}")
    if target.dtype != torch.int64:
        raise TypeError(f"linear_token_loss: targets of {target.dtype}, int64 expected")
    if not (h.get_device() == w.get_device() == target.get_device()):
        raise ValueError(f"linear_token_loss: tensors on {h.device}, {w.device} and {target.device}")
    if w.shape[0] == 0 or softcap < 0 or piece < 0:
        raise ValueError(f"linear_token_loss: vocabulary of {w.shape[0]}, softcap {softcap}, piece {piece}")
    if not (h.is_cuda and h.dtype == w.dtype == torch.bfloat16 and w.shape[1] > 0 and _lib.available()):
        return linear_token_loss_reference(h, w, target, ignore_index, softcap)
    if target.numel() == 0:                    # nothing to compute, but results that backward can be called on
        z = h.sum(-1).float() + 0.0 * w[0, 0].float()
        return z, z.clone()
    if _dbg.ENABLED:
        _dbg.check_indices(target, 0, w.shape[0], _dbg.SITE_CE_TARGET, also_ok=ignore_index)
    if not (torch.is_grad_enabled() and (h.requires_grad or w.requires_grad)):
        return _forward(h, w, target, int(ignore_index), float(softcap))
    return _TokenLossFn.apply(h, w, target, int(ignore_index), float(softcap), int(piece))
