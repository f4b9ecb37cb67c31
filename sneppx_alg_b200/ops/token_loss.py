"""Per-token losses of a vocabulary projection without the logits (csrc/vocab_loss.cu). bf16 CUDA tensors take the kernels;
``linear_token_loss_reference`` states the same in PyTorch and serves everything else. The reference computes a softmax and its gradient over the
logits of a batch (kernel/cuda/autodiff_cuda.cu:519-608)."""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib
from . import debug as _dbg
from ._lib import c_float, c_int, c_ll, ptr, stream
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


class _TokenLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, target, ignore_index, softcap, piece):
        T, V, d = target.numel(), w.shape[0], (w.shape[1] + 7) // 8 * 8
        h2, w2 = _rows16(h.reshape(-1, h.shape[-1]), d), _rows16(w, d)
        tgt = target.reshape(-1).contiguous()
        dev = h.device
        with _lib.on_device(h):
            out = torch.empty(3, T, dtype=torch.float32, device=dev)
            nll, lse, zt = out[0], out[1], out[2]
            part = torch.empty(2 * -(-V // 256), T, 2, dtype=torch.float32, device=dev)
            _lib.call("sx_vocab_loss_fwd", ptr(h2), c_ll(h2.stride(0)), ptr(w2), c_ll(w2.stride(0)), ptr(tgt), c_ll(T), c_ll(V), c_int(d),
                      c_ll(ignore_index), c_float(softcap), ptr(part), ptr(zt), ptr(nll), ptr(lse), ptr(_lib.status_word(dev)), stream())
        nll, lse = nll.view(target.shape), lse.view(target.shape)
        ctx.save_for_backward(h, w, tgt, lse)
        ctx.w, ctx.meta = w, (ignore_index, softcap, piece)
        ctx.set_materialize_grads(False)
        return nll, lse

    @staticmethod
    @once_differentiable
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
            piece = min((piece + 255) // 256 * 256, (V + 63) // 64 * 64)
            dz = torch.empty(rows * piece, dtype=torch.bfloat16, device=dev)
            dh = torch.empty(T, d, dtype=torch.bfloat16, device=dev) if need_h else None
            acc = torch.empty(T, d, dtype=torch.float32, device=dev) if need_h and piece < V else None
            mg = getattr(ctx.w, "main_grad", None) if need_w and d == d0 else None
            if mg is not None and (mg.dtype not in (torch.bfloat16, torch.float32) or mg.stride(1) != 1):
                mg = None
            add = mg is not None and getattr(ctx.w, "_main_grad_written", False)
            dw = (mg if mg is not None else torch.empty(V, d, dtype=torch.bfloat16, device=dev)) if need_w else None
            for v0 in range(0, V, piece):
                v1 = min(V, v0 + piece)
                n = v1 - v0
                ld = (n + 63) // 64 * 64
                z = dz[: rows * ld].view(rows, ld)
                _lib.call("sx_vocab_loss_grad", ptr(h2), c_ll(h2.stride(0)), ptr(w2), c_ll(w2.stride(0)), ptr(tgt), c_ll(T), c_ll(V), c_int(d),
                          c_ll(ignore_index), c_float(softcap), ptr(lse), ptr(gn), ptr(gz), ptr(z), c_ll(ld), c_ll(rows), c_ll(v0), c_ll(v1),
                          ptr(_lib.status_word(dev)), stream())
                if need_h:
                    n8 = (n + 7) // 8 * 8              # a ragged end of the vocabulary: zeros on both sides
                    wp = w2[v0:v1] if n8 == n else F.pad(w2[v0:v1], (0, 0, 0, n8 - n))
                    gemm(z[:T, :n8], wp, b_mn=True, out=dh if v1 == V else acc, c=acc if v0 else None, beta=1.0 if v0 else 0.0)
                if need_w:
                    gemm(z[:, :n], h2, a_mn=True, b_mn=True, out=dw[v0:v1], c=dw[v0:v1] if add else None, beta=1.0 if add else 0.0)
        if need_h:
            dh = (dh if d == d0 else dh[:, :d0]).reshape(h.shape)
        if mg is not None:
            ctx.w._main_grad_written = True
            dw = None
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
    if not (h.device == w.device == target.device):
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
    return _TokenLossFn.apply(h, w, target, int(ignore_index), float(softcap), int(piece))
