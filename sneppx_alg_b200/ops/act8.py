"""Activations held in 8 bits between forward and backward.

``pack_8bit`` / ``unpack_8bit`` hold any floating tensor as one exponent byte and 32 signed codes for each 32 values of its last dimension
(33 bytes for 32 values); ``glu_8bit`` is the gated activation that keeps its input so; ``checkpoint_8bit`` recomputes a function in backward from
arguments that were held so. CUDA tensors in bf16, fp16 and fp32 take the kernels (csrc/act8.cu); ``*_reference`` states the same in PyTorch and
serves CPU tensors. The reference recomputes layers from inputs kept in full (grad_checkpoint.py, kernel/autodiff/tape.c:80-87).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.overrides import handle_torch_function, has_torch_function_variadic

from . import _lib
from .functional import GLU_ACT, glu, glu_reference

BLOCK = 32
_NAMES = {v: k for k, v in GLU_ACT.items()}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _native(x) -> bool:
    if not x.is_cuda or has_torch_function_variadic(x) or _lib.elementary(x):      # a trace would see the kernels' allocations only
        return False
    if x.dtype not in _TYPES:
        raise TypeError(f"8-bit activations: {x.dtype} is not one of bfloat16, float16, float32")
    return _lib.available()


class Packed8bit:
    """What ``pack_8bit`` returns: ``codes`` int8 [rows, 32 * ceil(width / 32)], ``exponents`` uint8 [rows, ceil(width / 32)] with the value
    code * 2^(exponent - 127) (255: the block held an infinity or a NaN and is restored as NaN), ``shape`` and ``dtype`` of the tensor."""

    __slots__ = ("codes", "exponents", "shape", "dtype")

    def __init__(self, codes, exponents, shape, dtype):
        self.codes, self.exponents, self.shape, self.dtype = codes, exponents, torch.Size(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    @property
    def device(self):
        return self.codes.device


def _rows(x):
    """x as [rows, width] whose rows are contiguous (a view where x allows one)."""
    x = x.resolve_neg()                        # the imaginary part of a conjugate is a view whose sign is still to be turned
    if x.dim() > 1 and x.is_contiguous() and x.numel():
        return x.view(-1, x.shape[-1])
    w = x.shape[-1] if x.dim() else 1
    x2 = x.reshape(-1, w) if x.numel() else x.reshape(0, w)
    return x2 if x2.numel() == 0 or (x2.stride(1) == 1 or w == 1) and (x2.shape[0] == 1 or x2.stride(0) >= w) else x2.contiguous()


def pack_8bit_reference(x2):
    """[rows, width] -> (codes, exponents)."""
    rows, w = x2.shape
    nb = -(-w // BLOCK)
    b = F.pad(x2.float(), (0, nb * BLOCK - w)).view(rows, nb, BLOCK)
    top = b.abs().amax(-1) if nb else b.new_zeros(rows, 0)
    finite = torch.isfinite(top)
    m, e = torch.frexp(torch.where(finite, top, 1.0))                        # top = m 2^e with m in [1/2, 1)
    e = torch.where(top > 0, e - 7 + (m >= 127.5 / 128).int(), -126).clamp(-126, 9 if x2.dtype == torch.float16 else 121)      # 121: of values from 2^127 on
    codes = torch.where(finite[..., None], torch.round(torch.ldexp(b, -e[..., None])).clamp(-127, 127), 0.0)
    return codes.to(torch.int8).view(rows, nb * BLOCK), torch.where(finite, e + 127, 255).to(torch.uint8)


def unpack_8bit_reference(codes, exponents, width, dtype):
    rows, nb = exponents.shape
    step = torch.ldexp(torch.ones(rows, nb, device=codes.device), exponents.int() - 127)
    step = torch.where(exponents == 255, torch.nan, step)
    return (codes.view(rows, nb, BLOCK).float() * step[..., None]).view(rows, nb * BLOCK)[:, :width].to(dtype)


def pack_8bit(x) -> Packed8bit:
    """x (any shape, blocks along its last dimension; float types) in 8 bits. Finite values come back finite: steps are never so wide that whole ones leave
    the type. Not differentiable: what backward reads."""
    if not x.is_floating_point():
        raise TypeError(f"pack_8bit: {x.dtype} is not a floating type")
    x2 = _rows(x.detach())
    rows, w = x2.shape
    nb = -(-w // BLOCK)
    if not _native(x):
        return Packed8bit(*pack_8bit_reference(x2), x.shape, x.dtype)
    codes, exps = x2.new_empty((rows, nb * BLOCK), dtype=torch.int8), x2.new_empty((rows, nb), dtype=torch.uint8)
    _lib.launch(x, "sx_pack8", "ppplilip", x2.data_ptr(), codes.data_ptr(), exps.data_ptr(), rows, w, x2.stride(0), _TYPES[x.dtype])
    return Packed8bit(codes, exps, x.shape, x.dtype)


def unpack_8bit(p: Packed8bit, dtype=None):
    """The tensor that ``p`` stands for, in its own type or in ``dtype``."""
    dtype = dtype or p.dtype
    w = p.shape[-1] if len(p.shape) else 1
    rows, nb = p.exponents.shape
    if p.codes.shape != (rows, nb * BLOCK) or nb != -(-w // BLOCK) or rows * w != p.shape.numel() or p.codes.dtype != torch.int8 \
            or p.exponents.dtype != torch.uint8 or p.codes.device != p.exponents.device:
        raise ValueError(f"unpack_8bit: codes {tuple(p.codes.shape)} and exponents {tuple(p.exponents.shape)} do not hold {tuple(p.shape)}")
    if not (p.codes.is_cuda and _lib.available()) or has_torch_function_variadic(p.codes, p.exponents) or _lib.elementary(p.codes, p.exponents):
        return unpack_8bit_reference(p.codes, p.exponents, w, dtype).view(p.shape)
    if dtype not in _TYPES:
        raise TypeError(f"8-bit activations: {dtype} is not one of bfloat16, float16, float32")
    codes, exps = p.codes.contiguous(), p.exponents.contiguous()               # whole numbers: no sign is left to be turned
    if codes.data_ptr() % 16:                  # a view into something larger: the kernels read four words at once
        codes = codes.clone()
    x = codes.new_empty(p.shape, dtype=dtype)
    _lib.launch(x, "sx_unpack8", "ppplilip", codes.data_ptr(), exps.data_ptr(), x.data_ptr(), rows, w, w, _TYPES[dtype])
    return x


# ----------------------------------------------------------------------------- gated activation
def _gate(g, act):
    """Value and derivative of the gate's function, in 32 bits."""
    if act == 0:
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == 1:
        k0, k1 = 0.7978845608028654, 0.044715
        t = torch.tanh(k0 * (g + k1 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k0 * (1 + 3 * k1 * g * g)
    return torch.relu(g), torch.where(torch.isnan(g), g, (g > 0).to(g.dtype))


def glu_8bit_backward_reference(dh, gate, up, act):
    """(rows of dgate | dup) from restored gate and up."""
    a, da = _gate(gate.float(), act)
    d = dh.float()
    return torch.cat([d * up.float() * da, d * a], -1).to(dh.dtype)


def _glu_forward(gu, act, held=None):
    """The kernel's value of gu; with ``held`` (a buffer for the codes of gate and up for each row and then their exponents) packed there, too."""
    f = gu.shape[-1] // 2
    g2 = _rows(gu)
    h = gu.new_empty((*gu.shape[:-1], f))
    at = 0 if held is None else held.data_ptr()
    _lib.launch(gu, "sx_glu8_fwd", "ppppliliip", g2.data_ptr(), h.data_ptr(), at, at and at + g2.shape[0] * 2 * -(-f // BLOCK) * BLOCK, g2.shape[0], f,
                g2.stride(0), act, _TYPES[gu.dtype])
    return h


class _Glu8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu, act):
        f = gu.shape[-1] // 2
        native = _native(gu)
        ctx.meta = act, gu.shape, native
        if not native:
            g2 = _rows(gu)
            parts = [pack_8bit_reference(t) for t in (g2[:, :f], g2[:, f:])]
            ctx.save_for_backward(torch.cat([c for c, _ in parts], 1), torch.cat([e for _, e in parts], 1))
            return glu_reference(gu, _NAMES[act])
        held = gu.new_empty(gu.shape[:-1].numel() * 2 * -(-f // BLOCK) * (BLOCK + 1), dtype=torch.uint8)
        ctx.save_for_backward(held)
        return _glu_forward(gu, act, held)

    @staticmethod
    @_lib.once
    def backward(ctx, dh):
        act, shape, native = ctx.meta
        f = shape[-1] // 2
        if not native:
            codes, exps = ctx.saved_tensors
            rows = codes.shape[0]
            gate, up = (unpack_8bit_reference(c, e, f, torch.float32) for c, e in zip(codes.chunk(2, 1), exps.chunk(2, 1)))
            return glu_8bit_backward_reference(dh.reshape(rows, f), gate, up, act).view(shape), None
        (held,) = ctx.saved_tensors
        nb = -(-f // BLOCK)
        rows = held.numel() // (2 * nb * (BLOCK + 1)) if nb else 0
        dh = dh.contiguous().resolve_neg()
        dgu = dh.new_empty(shape)
        at = held.data_ptr()
        _lib.launch(dh, "sx_glu8_bwd", "ppppliiip", dh.data_ptr(), at, at + rows * 2 * nb * BLOCK, dgu.data_ptr(), rows, f, act, _TYPES[dh.dtype])
        return dgu, None


def glu_8bit(gu, act="silu"):
    """act(gate) * up with gu = [..., 2F] laid out (gate | up), as ``glu``; what backward needs of gu is held in 8 bits (2.06 bytes instead of
    4 for a gate and an up value of 16 bits), so the gradient is that of the restored gate and up. The result is computed from gu itself."""
    if has_torch_function_variadic(gu):
        return handle_torch_function(glu_8bit, (gu,), gu, act)
    if act not in GLU_ACT:
        raise ValueError(f"glu_8bit: act {act!r} is not one of {sorted(GLU_ACT)}")
    if gu.dim() == 0 or gu.shape[-1] % 2:
        raise ValueError(f"glu_8bit: the last dimension of {tuple(gu.shape)} does not split into gate and up")
    if not gu.is_floating_point():
        raise TypeError(f"glu_8bit: {gu.dtype} is not a floating type")
    if not (torch.is_grad_enabled() and gu.requires_grad):      # nothing is kept
        if gu.is_cuda and gu.dtype == torch.bfloat16:
            return glu(gu, act)
        return _glu_forward(gu, GLU_ACT[act]) if _native(gu) else glu_reference(gu, act)
    return _Glu8Fn.apply(gu, GLU_ACT[act])


# ----------------------------------------------------------------------------- recomputation
def checkpoint_8bit(fn, *args):
    """``fn(*args)``, whose inner activations are recomputed in backward from arguments that are held in 8 bits: of ``args``, the floating CUDA / CPU
    tensors that autograd reaches (those that require a gradient and are no leaves) are packed, the others are kept as they are. The first pass runs
    on the arguments themselves; gradients are those of ``fn`` at the restored ones. Random state and autocast are as in torch.utils.checkpoint."""
    from torch.utils._pytree import tree_leaves
    from torch.utils.checkpoint import checkpoint

    held, kept = list(args), list(args)
    if not torch.is_grad_enabled():
        return fn(*args)
    for i, a in enumerate(args):
        if torch.is_tensor(a) and a.is_floating_point() and a.requires_grad and not a.is_leaf and (a.dtype in _TYPES):
            kept[i] = pack_8bit(a)

    # generators are saved and set back for the devices of what checkpoint is handed: nothing of each device, as the arguments themselves go past it
    places = [torch.empty(0, device=d) for d in {t.device for t in tree_leaves(args) if torch.is_tensor(t)}]

    def run(*_):
        if held:                       # forward
            now = list(held)
            held.clear()
        else:                          # backward
            now = [unpack_8bit(a).requires_grad_() if isinstance(a, Packed8bit) else a for a in kept]
        return fn(*now)

    return checkpoint(run, *places, use_reentrant=False)
