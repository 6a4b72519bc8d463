"""Embedding rows by token, scaled, with the table's gradient summed in the tokens' order (csrc/embedding.hip).

    embedding(ids, table, scale, padding_idx)             y[..., :] = scale * table[ids]        differentiable in `table`
    embedding_backward(ids, upstream, rows, ...)          the table's gradient, as a call of its own
    FastEmbedding                                         nn.Embedding with a scale (the de-noising queries' label table:
                                                          /root/reference/models/dino/dino.py:93, dn_components.py:99)

Tables are float32, float16 or bfloat16 device tensors.  The gradient adds a row's tokens in ascending order in 32 bits and
rounds once: it does not depend on the launch, where atomics would.  An id outside [0, rows) gives a row of zeros and no
gradient (no host synchronisation to look for one).  Both directions are linear and each is the other's derivative, so they
differentiate any number of times, in reverse and in forward mode."""
from __future__ import annotations

import torch
from torch.autograd import Function, forward_ad

from . import _native


def _check_ids(ids: torch.Tensor) -> None:
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"embedding: ids are int64 or int32, got {ids.dtype}")


def _ids64(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype is torch.int64 and ids.is_contiguous():
        return ids
    return ids.to(torch.int64).contiguous()


def _padding(padding_idx, rows: int) -> int:
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"embedding: padding_idx {padding_idx} is outside a table of {rows} rows")
    return padding_idx + rows if padding_idx < 0 else padding_idx


def _forward(ids: torch.Tensor, table: torch.Tensor, scale: float) -> torch.Tensor:
    V, D = table.shape
    apart, step = table.stride()
    if step != 1 or apart < D:
        table = table.contiguous()
        apart = D
    device = table.device
    out = torch.empty((*ids.shape, D), dtype=table.dtype, device=device)
    flat = _ids64(ids)
    with _native.on_device(device):
        rc = _native.lib.datr_embedding_forward(_native.DTYPE[table.dtype], flat.data_ptr(), table.data_ptr(), flat.numel(), V, D,
                                                apart, scale, out.data_ptr(), _native.current_stream_ptr(device))
    _native.check(rc, "embedding_forward")
    return out


def embedding_backward(ids: torch.Tensor, upstream: torch.Tensor, rows: int, scale: float = 1.0, padding_idx=None) -> torch.Tensor:
    """The gradient [rows, D] of `embedding`'s table for upstream [*ids.shape, D], in upstream's type."""
    _check_ids(ids)
    if upstream.dtype not in _native.DTYPE:
        raise TypeError(f"embedding_backward: float32, float16 or bfloat16, got {upstream.dtype}")
    shape = upstream.shape
    if not shape or shape[:-1] != ids.shape:
        raise ValueError(f"embedding_backward: upstream is ids' shape and a width, got {tuple(shape)} for ids {tuple(ids.shape)}")
    if rows < 0:
        raise ValueError(f"embedding_backward: a table of {rows} rows")
    pad = _padding(padding_idx, rows)
    if not upstream.is_cuda:
        raise RuntimeError("embedding_backward: Not implemented on the CPU")
    if ids.device != upstream.device:
        raise ValueError("embedding_backward: ids and upstream are on different devices")
    return _gradient(ids, upstream, rows, float(scale), pad)


def _backward(ids: torch.Tensor, upstream: torch.Tensor, rows: int, scale: float, pad: int) -> torch.Tensor:
    shape, device = upstream.shape, upstream.device
    D, flat = shape[-1], _ids64(ids)
    tokens = flat.numel()
    up = upstream if len(shape) == 2 else upstream.reshape(tokens, D)
    apart, step = up.stride()
    if step != 1 or apart < D:
        up, apart = up.contiguous(), D
    grad = torch.empty((rows, D), dtype=up.dtype, device=device)
    need = _native.lib.datr_embedding_backward_workspace_bytes(tokens, rows, D)
    ws = torch.empty(need, dtype=torch.int8, device=device) if need else None
    with _native.on_device(device):
        rc = _native.lib.datr_embedding_backward(_native.DTYPE[up.dtype], flat.data_ptr(), up.data_ptr(), tokens, rows, D, apart, scale,
                                                 pad, grad.data_ptr(), 0 if ws is None else ws.data_ptr(), need,
                                                 _native.current_stream_ptr(device))
    _native.check(rc, "embedding_backward")
    return grad


def _gradient(ids: torch.Tensor, upstream: torch.Tensor, rows: int, scale: float, pad: int) -> torch.Tensor:
    if (upstream.requires_grad and torch.is_grad_enabled()) or _native.carries_tangent(upstream):
        return _EmbeddingGradient.apply(ids, upstream, rows, scale, pad)
    return _backward(ids, upstream, rows, scale, pad)


class _Embedding(Function):
    """`pad` is -1 without a padding row."""

    @staticmethod
    def forward(ctx, ids, table, scale, pad):
        ctx.save_for_backward(ids)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(ids)
        ctx.rest = table.shape[0], scale, pad
        return _forward(ids, table, scale)

    @staticmethod
    def backward(ctx, upstream):
        return None, _gradient(*ctx.saved_tensors, upstream, *ctx.rest), None, None

    @staticmethod
    def jvp(ctx, _ids, table, _scale, _pad):
        ids, = ctx.saved_tensors
        return embedding(ids, table, ctx.rest[1])


class _EmbeddingGradient(Function):
    """embedding_backward as a node of its own, for derivatives of the gradient."""

    @staticmethod
    def forward(ctx, ids, upstream, rows, scale, pad):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.rest = rows, scale, pad
        return _backward(ids, upstream, rows, scale, pad)

    @staticmethod
    def backward(ctx, along):
        ids, = ctx.saved_tensors
        _, scale, pad = ctx.rest
        if pad >= 0:                                       # the padding row's tokens took no part
            ids = torch.where(ids == pad, -1, ids)
        return None, embedding(ids, along, scale), None, None, None

    @staticmethod
    def jvp(ctx, _ids, upstream, _rows, _scale, _pad):
        return _gradient(*ctx.saved_tensors, upstream, *ctx.rest)


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx=None) -> torch.Tensor:
    """scale * table[ids]: ids int64 / int32 of any shape, table [rows, D] with a unit last stride -> [*ids.shape, D] in the
    table's type.  `padding_idx`: the row that takes no gradient (its values are read like any other's)."""
    _check_ids(ids)
    if table.dim() != 2:
        raise ValueError(f"embedding: the table is [rows, width], got {tuple(table.shape)}")
    if table.dtype not in _native.DTYPE:
        raise TypeError(f"embedding: float32, float16 or bfloat16 tables, got {table.dtype}")
    pad = _padding(padding_idx, table.shape[0])
    if not table.is_cuda:
        raise RuntimeError("embedding: Not implemented on the CPU")
    if ids.device != table.device:
        raise ValueError("embedding: ids and table are on different devices")
    if (table.requires_grad and torch.is_grad_enabled()) or _native.carries_tangent(table):
        return _Embedding.apply(ids, table, float(scale), pad)
    return _forward(ids, table, float(scale))


class FastEmbedding(torch.nn.Embedding):
    """nn.Embedding (same parameters, same state_dict keys) with a scale, on the kernels above for device tables; host tables
    and nn.Embedding's max_norm / scale_grad_by_freq / sparse take its own path, and so does a call below a function transform
    (torch.func)."""

    def __init__(self, *args, scale: float = 1.0, **kw):
        super().__init__(*args, **kw)
        self.scale = float(scale)

    def forward(self, ids):
        if (self.weight.is_cuda and self.weight.dtype in _native.DTYPE and self.max_norm is None and not self.scale_grad_by_freq
                and not self.sparse and not torch._C._are_functorch_transforms_active()):
            return embedding(ids, self.weight, self.scale, self.padding_idx)
        y = super().forward(ids)
        return y if self.scale == 1.0 else y * self.scale
