"""Per-token losses of a vocabulary projection without the logits (csrc/vocab_loss.cu). bf16 CUDA tensors take the kernels;
``linear_token_loss_reference`` states the same in PyTorch and serves everything else. The reference computes a softmax and its gradient over the
logits of a batch (kernel/cuda/autodiff_cuda.cu:519-608)."""
from __future__ import annotations

import ctypes as C

import torch
import torch.nn.functional as F
from torch.overrides import handle_torch_function, has_torch_function_variadic

from . import _lib
from . import debug as _dbg


def linear_token_loss_reference(h, w, target, ignore_index=-100, softcap=0.0):
    ct = torch.promote_types(torch.promote_types(h.dtype, w.dtype), torch.float32)
    z = F.linear(h.to(ct), w.to(ct))
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    lse = torch.logsumexp(z, -1)
    valid = target != ignore_index
    bad = valid & ((target < 0) | (target >= w.shape[0]))
    if not target.is_cuda:
        if bool(bad.any()):
            raise IndexError(f"linear_token_loss: a target outside a vocabulary of {w.shape[0]}")
    else:                                          # as the kernels do: ignored, and told by the status word
        if not _lib.elementary(h, w, target):
            word = _lib.status_word(target.device)[:1]
            word.copy_(torch.where(bad.any() & (word == 0), 5, word))
        valid = valid & ~bad
    zt = z.gather(-1, torch.where(valid, target, 0).unsqueeze(-1)).squeeze(-1)
    return torch.where(valid, lse - zt, 0.0), lse


def _rows16(t, d):
    """(t, pitch): t [..., <= d] as the tensor maps take it: rows of d columns, a multiple of 8 (padded with zeros), 16-byte aligned."""
    w = t.shape[-1]
    t = t.resolve_neg()                        # the imaginary part of a conjugate is a view whose sign is still to be turned
    if w == d and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, d
    if t.dim() != 2:
        t = t.reshape(-1, w)
    if w != d:
        t = F.pad(t, (0, d - w))
    one = t.shape[0] == 1                      # its pitch may be anything and means nothing
    if t.stride(1) != 1 or (not one and (t.stride(0) % 8 or t.stride(0) < d)) or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
    return t, d if one else t.stride(0)


def _forward(h, w, target, ignore_index, softcap, keep=False):
    """(nll, lse) in target's shape, the targets as they were read, and with ``keep`` nll once more for backward (the caller's may be written over)."""
    T, V, d = target.numel(), w.shape[0], (w.shape[1] + 7) // 8 * 8
    (h2, ldh), (w2, ldw) = _rows16(h, d), _rows16(w, d)
    tgt = target.contiguous()
    nll, lse = h2.new_empty(target.shape, dtype=torch.float32), h2.new_empty(target.shape, dtype=torch.float32)
    pairs = 2 * T * -(-V // 256)                          # of a row's maximum and sum, and behind them its target's logit
    scratch = h2.new_empty(pairs if keep else pairs + T, dtype=torch.float32)
    own = h2.new_empty(T, dtype=torch.float32) if keep else None
    _lib.launch(h, "sx_vocab_loss_fwd", "plplpllilfpppppp", h2.data_ptr(), ldh, w2.data_ptr(), ldw, tgt.data_ptr(), T, V, d, ignore_index, softcap,
                scratch.data_ptr(), own.data_ptr() if keep else scratch.data_ptr() + 4 * pairs, nll.data_ptr(), lse.data_ptr(), _lib.status_ptr(h))
    return nll, lse, tgt, own


class _TokenLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, target, ignore_index, softcap, piece):
        nll, lse, tgt, own = _forward(h, w, target, ignore_index, softcap, True)
        ctx.save_for_backward(h, w, tgt, lse, own)
        ctx.meta = ignore_index, softcap, piece
        ctx.set_materialize_grads(False)
        return nll, lse

    @staticmethod
    @_lib.once
    def backward(ctx, g_nll, g_lse):
        none = (None,) * 6
        if g_nll is None and g_lse is None:
            return none
        h, w, tgt, lse, own = ctx.saved_tensors
        ignore_index, softcap, piece = ctx.meta
        need_h, need_w = ctx.needs_input_grad[:2]
        T, V, d0 = tgt.numel(), w.shape[0], w.shape[1]
        d = (d0 + 7) // 8 * 8                          # what the products' pitches take
        (h2, ldh), (w2, ldw) = _rows16(h, d), _rows16(w, d)
        gn, gz = (g if g is None else g.contiguous().resolve_neg() for g in (g_nll, g_lse))       # fp32, as the results are
        dh = h2.new_empty(h.shape if d == d0 else (T, d)) if need_h else None
        mg = getattr(w, "main_grad", None) if need_w and d == d0 else None
        if mg is not None and (mg.dtype not in (torch.bfloat16, torch.float32) or mg.stride(1) != 1):
            mg = None
        dw = (mg if mg is not None else w2.new_empty((V, d))) if need_w else None
        a = _lib.SxVocabLossArgs()
        a.h, a.w, a.ldh, a.ldw = h2.data_ptr(), w2.data_ptr(), ldh, ldw
        a.target, a.lse, a.nll, a.status = tgt.data_ptr(), lse.data_ptr(), own.data_ptr(), _lib.status_ptr(h)
        a.T, a.V, a.d, a.ignore_index, a.cap, a.piece = T, V, d, ignore_index, softcap, piece
        if gn is not None:
            a.g_nll = gn.data_ptr()
        if gz is not None:
            a.g_lse = gz.data_ptr()
        if need_h:
            a.dh = dh.data_ptr()
        if need_w:
            a.dw, a.lddw, a.dw_fp32 = dw.data_ptr(), dw.stride(0), dw.dtype == torch.float32
            a.dw_add = mg is not None and getattr(w, "_main_grad_written", False)
        a.work_bytes = _lib.entry("sx_vocab_loss_bwd_workspace", "p", _lib.c_ll)(C.addressof(a))
        work = h2.new_empty(a.work_bytes, dtype=torch.uint8)
        a.work = work.data_ptr()
        _lib.launch(h, "sx_vocab_loss_bwd", "pp", C.addressof(a))
        if mg is not None:
            w._main_grad_written = True
            dw = None
        elif need_w and d != d0:
            dw = dw[:, :d0].contiguous()
        if need_h and d != d0:
            dh = dh[:, :d0].reshape(h.shape)
        return dh, dw, None, None, None, None


def linear_token_loss(h, w, target, ignore_index=-100, softcap=0.0, piece=0):
    """(nll, lse) of every token, fp32: logits z = h @ w^T, with ``softcap`` c > 0 c * tanh(z / c); lse = log sum exp z over the vocabulary, nll = lse
    - z[target], 0 where target is ``ignore_index``. h [..., d], w [V, d], target [...] int64. Both results are differentiable (a z-loss is a function of
    lse), with any weight for each token; the logits exist in tiles only. On the GPU nll is right to a part of itself also where it is small.

    Backward holds dz for about ``piece`` columns of the vocabulary at a time (0: as many as fit 256 MiB) and computes the logits again: it trades a
    fourth product of h and w for logits that ``linear_cross_entropy`` holds a chunk of, and need not know the tokens' weights beforehand.
    Where w carries ``main_grad`` its gradient is written or added there and ``.grad`` stays empty. On the GPU a target outside [0, V) counts as
    ignored and sets the status word (``check_status`` raises); on the CPU it raises at once. Ignored tokens take part in the products with weight 0:
    their hidden states have to be finite. Scratch of the forward pass: 8 bytes for a token and 256 words."""
    if has_torch_function_variadic(h, w, target):      # a trace records this call: of the kernels' it would see their allocations only
        return handle_torch_function(linear_token_loss, (h, w, target), h, w, target, ignore_index, softcap, piece)
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
    if not (h.is_cuda and h.dtype == w.dtype == torch.bfloat16 and w.shape[1] > 0 and not _lib.elementary(h, w, target) and _lib.available()):
        return linear_token_loss_reference(h, w, target, ignore_index, softcap)
    if target.numel() == 0:                    # nothing to compute, but results that backward can be called on
        z = h.sum(-1).float() + 0.0 * w[0, 0].float()
        return z, z.clone()
    if _dbg.ENABLED:
        _dbg.check_indices(target, 0, w.shape[0], _dbg.SITE_CE_TARGET, also_ok=ignore_index)
    if not (torch.is_grad_enabled() and (h.requires_grad or w.requires_grad)):
        return _forward(h, w, target, int(ignore_index), float(softcap))[:2]
    return _TokenLossFn.apply(h, w, target, int(ignore_index), float(softcap), int(piece))
