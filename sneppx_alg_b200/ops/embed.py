"""Embedding lookup with scaling, and its gradient by sorted tokens (csrc/embed.cu). CUDA tables in bf16, fp16 and fp32 take the kernels;
``embedding_reference`` states the same in PyTorch and serves CPU tensors. The reference looks rows up and scatters their gradients in its Python
module (interface_bindings/nn.py, ``Embedding``)."""
from __future__ import annotations

import ctypes
import functools
import warnings

import torch
import torch.nn.functional as F
from torch.overrides import handle_torch_function, has_torch_function_variadic

from . import _lib
from . import debug as _dbg
from .. import _build

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def embedding_reference(ids, table, scale=1.0, padding_idx=None):
    if not table.is_cuda or not (table.dtype in _TYPES or table.dtype is torch.float64):
        y = F.embedding(ids, table, padding_idx)
    else:                                          # ids out of range as the kernels have them: rows of zeros, told by the status word
        ok = (ids >= 0) & (ids < table.shape[0])
        y = torch.where(ok.unsqueeze(-1), F.embedding(torch.where(ok, ids, 0), table, padding_idx), 0.0)
        if not _lib.elementary(ids, table):        # which nobody may write to there
            word = _lib.status_word(table.device)[:1]
            word.copy_(torch.where((~ok).any() & (word == 0), 5, word))
    return y if scale == 1.0 else (y.float() * scale).to(y.dtype) if y.dtype != torch.float64 else y * scale


@functools.lru_cache(1024)
def _sorted_bytes(n, V):
    return _lib.entry("sx_embed_sorted_bytes", "ll", _lib.c_ll)(n, V)


@functools.lru_cache(1024)
def _workspace(n, V, d, presorted):
    return _lib.entry("sx_embed_bwd_workspace", "llii", _lib.c_ll)(n, V, d, presorted)


_nodes = None        # the graph node in C++, False where it cannot be built


def _load_nodes():
    """ops/native/embed_node.cpp, which the calls take where it is there: the same kernels at less host time than the Python function below."""
    global _nodes
    try:
        nodes = _build.load_torch()
        L = _lib.lib()
        nodes.bind(_lib, *(ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in
                           ("sx_embed_sorted_bytes", "sx_embed_bwd_workspace", "sx_embed_fwd", "sx_embed_bwd")))
        _nodes = nodes
    except RuntimeError as e:
        warnings.warn(f"sneppx_alg_b200: embeddings take more host time without libsneppx_torch.so: {e}", RuntimeWarning, stacklevel=3)
        _nodes = False
    return _nodes


# Numbers are read once and nothing is wrapped: for few tokens the host's time is all that the calls take.
def _lookup(ids, table, scale, padding=-1, sort=False):
    """(rows, ids as they were read, those in the order of their words or None). padding: a word, or -1."""
    V, d = table.shape
    table = table.resolve_neg()                # the imaginary part of a conjugate is a view whose sign is still to be turned
    ldw, step = table.stride()
    if step != 1 or ldw < d:
        table, ldw = table.contiguous(), d
    ids = ids.contiguous()
    n = ids.numel()
    y = table.new_empty((*ids.shape, d))
    order, at = None, 0
    if sort and d:
        size = _sorted_bytes(n, V)
        if size:
            order = table.new_empty(size, dtype=torch.uint8)
            at = order.data_ptr()
    _lib.launch(table, "sx_embed_fwd", "piplplilfilppp", ids.data_ptr(), ids.dtype is torch.int64, table.data_ptr(), ldw, y.data_ptr(), n, d, V, scale,
                _TYPES[table.dtype], padding, at, _lib.status_ptr(table))
    return y, ids, order


def embedding_backward_(grad, ids, dy, scale=1.0, padding_idx=None, add=False):
    """grad [V, d] = scale * (sums of the rows of dy [.., d] by their word), or, with ``add``, grad += that (rows of other words are not touched
    then). Sums are in 32 bits and in the order of the tokens, so they are the same each time. grad has dy's type or is fp32."""
    if has_torch_function_variadic(grad, ids, dy):
        return handle_torch_function(embedding_backward_, (grad, ids, dy), grad, ids, dy, scale, padding_idx, add)
    V, d = grad.shape
    if dy.dtype not in _TYPES or grad.dtype not in (dy.dtype, torch.float32) or grad.stride(1) != 1 or (V > 1 and grad.stride(0) < d):
        raise ValueError(f"embedding_backward_: gradients {dy.dtype} into {grad.dtype} with strides {grad.stride()}")
    if dy.shape != (*ids.shape, d):
        raise ValueError(f"embedding_backward_: gradients of shape {tuple(dy.shape)} for ids {tuple(ids.shape)} and rows of {d}")
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"embedding_backward_: ids of {ids.dtype}")
    if not (grad.is_cuda and grad.get_device() == dy.get_device() == ids.get_device()):
        raise ValueError(f"embedding_backward_: tensors on {grad.device}, {dy.device} and {ids.device}")
    if V == 0:
        raise ValueError("embedding_backward_: a table of no rows")
    if padding_idx is not None and not 0 <= padding_idx < V:
        raise ValueError(f"embedding_backward_: padding_idx {padding_idx} outside a table of {V} rows")
    if _lib.elementary(grad, ids, dy) or grad.is_neg():
        sums = _differentiable_backward(ids, dy, V, scale, -1 if padding_idx is None else padding_idx, torch.float32)
        return grad.add_(sums) if add else grad.copy_(sums)
    return _backward(grad, ids.contiguous(), dy.contiguous(), float(scale), -1 if padding_idx is None else padding_idx, bool(add), None)


def _backward(grad, ids, dy, scale, padding, add, order):
    """ids and dy contiguous, all on one device; order: what the forward pass left, or None."""
    V, d = grad.shape
    dy = dy.resolve_neg()
    n = ids.numel()
    size = _workspace(n, V, d, order is not None)
    work = grad.new_empty(size, dtype=torch.uint8)
    _lib.launch(grad, "sx_embed_bwd", "pippllillfiiipplpp", ids.data_ptr(), ids.dtype is torch.int64, dy.data_ptr(), grad.data_ptr(), grad.stride(0), n, d, V,
                padding, scale, add, _TYPES[dy.dtype], _TYPES[grad.dtype], 0 if order is None else order.data_ptr(), work.data_ptr(), size,
                _lib.status_ptr(grad))
    return grad


def _differentiable_backward(ids, dy, V, scale, padding, dtype):
    counts = (ids >= 0) & (ids < V) & (ids != padding)
    rows = torch.where(counts[..., None], dy.float() * scale, 0.0).reshape(-1, dy.shape[-1])
    return rows.new_zeros(V, dy.shape[-1]).index_add(0, torch.where(counts, ids, 0).reshape(-1), rows).to(dtype)


class _EmbeddingFn(torch.autograd.Function):
    """What ops/native/embed_node.cpp does, where that cannot be built."""

    @staticmethod
    def forward(ctx, ids, table, scale, padding):
        y, ids, order = _lookup(ids, table, scale, padding, True)
        ctx.save_for_backward(ids)
        ctx.meta = table, scale, padding, order
        return y

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        table, scale, padding, order = ctx.meta
        if torch.is_grad_enabled() or type(dy) is not torch.Tensor or torch._C._functorch.is_legacy_batchedtensor(dy):
            # a graph of this pass, or of a batch of them, is wanted: the same sums by operations that have one
            return None, _differentiable_backward(ids, dy, table.shape[0], scale, padding, dy.dtype), None, None
        mg = getattr(table, "main_grad", None)
        dy = dy.contiguous()
        if mg is None or mg.dtype not in (dy.dtype, torch.float32) or mg.stride(1) != 1:
            return None, _backward(dy.new_empty(table.shape), ids, dy, scale, padding, False, order), None, None
        _backward(mg, ids, dy, scale, padding, getattr(table, "_main_grad_written", False), order)
        table._main_grad_written = True
        return None, None, None, None


def embedding(ids, table, scale=1.0, padding_idx=None):
    """scale * table[ids]: table [V, d], ids any shape of integers -> [*ids.shape, d] in the table's type.

    The gradient of the table is dense; where the table carries ``main_grad`` (a view into a flat gradient buffer, of its type or fp32) it is written
    there, or added to what is there already (a tied output projection's), and ``.grad`` stays empty. ``padding_idx`` (negative counts from the
    end): tokens of this word give no gradient. On the GPU an id outside [0, V) gives a row of zeros and sets the status word
    (``check_status`` raises); on the CPU it raises at once. Inside function transforms (``jit.grad``, ``vmap``, ``jvp``, ``hessian``), in forward-mode
    differentiation, under torch.compile and torch.jit.trace and for tensor classes with a dispatch of their own the PyTorch form is taken; the status word
    is left alone there."""
    if has_torch_function_variadic(ids, table):      # a trace records this call: of the kernel's it would see the allocation of the result only
        return handle_torch_function(embedding, (ids, table), ids, table, scale, padding_idx)
    if _nodes and padding_idx is None and not _dbg.ENABLED and not torch.compiler.is_compiling():
        y = _nodes.ordinary(ids, table, scale)
        if y is not None:
            return y
    if table.dim() != 2:
        raise ValueError(f"embedding: table of shape {tuple(table.shape)} is no matrix")
    V = table.shape[0]
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
            raise TypeError(f"embedding: ids of {ids.dtype}")
        ids = ids.long()
    if ids.get_device() != table.get_device():
        raise ValueError(f"embedding: ids on {ids.device}, table on {table.device}")
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"embedding: padding_idx {padding_idx} outside a table of {V} rows")
        padding_idx %= V
    if V == 0 and ids.numel():
        raise IndexError("embedding: ids for a table of no rows")
    if not table.is_cuda or table.dtype not in _TYPES or V == 0 or _lib.elementary(ids, table) or not _lib.available():
        return embedding_reference(ids, table, scale, padding_idx)
    if _dbg.ENABLED:
        _dbg.check_indices(ids, 0, V, _dbg.SITE_USER)
    padding = -1 if padding_idx is None else padding_idx
    nodes = _nodes if _nodes is not None else _load_nodes()
    if nodes:
        return nodes.lookup(ids, table, scale, padding, _lib.status_ptr(table))
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbeddingFn.apply(ids, table, float(scale), padding)
    return _lookup(ids, table, scale)[0]
