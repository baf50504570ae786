"""Table lookup by token with its gradient and the sparse row update (csrc/embed.hip): what a model over tokens has in front
of its dense layers.

``embedding_lookup(table, ids, scale)`` is the differentiable operator (``tf.nn.embedding_lookup`` of a graph evaluates to it);
``lookup``, ``lookup_grad`` and ``lookup_sgd`` are the three launches behind it for code that manages its own gradients.
``lookup_sgd`` is the sparse apply of a table that lives next to the caller: only the rows that occur in the batch are read
and written, so a step costs what the batch holds and not what the table holds.

An id outside ``[0, rows)`` is padding: its output row is zero and it has no gradient.  Tables in float32, bfloat16 or
float16; sums in fp32 in a fixed order (the same bits on every run), rounded once.  GPU tensors of any other type are refused.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import hip_backend as hb


def _out_matrix(out: torch.Tensor, shape, like: torch.Tensor, name: str) -> int:
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device:
        raise hb.HipKernelError(f"{name} must be a {like.dtype} tensor of shape {tuple(shape)} on {like.device}, got {out.dtype} "
                                f"{tuple(out.shape)} on {out.device}")
    return hb.typed_rows(out, name)


def _gradient_rows(ids: torch.Tensor, grad: torch.Tensor):
    """The upstream gradient ``ids.shape + (dim,)`` as a matrix with one contiguous row per token, and its row stride."""
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape:
        raise hb.HipKernelError(f"the gradient of a lookup of {tuple(ids.shape)} ids has shape {tuple(ids.shape)} + (dim,), got "
                                f"{tuple(grad.shape)}")
    g = grad.reshape(-1, grad.shape[-1]) if grad.numel() else grad.reshape(ids.numel(), grad.shape[-1])
    if g.shape[1] > 1 and g.stride(1) != 1 or g.shape[0] > 1 and g.stride(0) < g.shape[1]:
        g = g.contiguous()          # (broadcast or transposed upstream gradients)
    return g, hb.typed_rows(g, "grad")


def lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[..., :] = scale * table[ids[...], :]`` in one launch; rows of zeros for ids outside the table.  ``out``: a matrix
    ``[ids.numel(), dim]`` to write into (returned as it is) instead of a new tensor ``ids.shape + (dim,)``."""
    lib = hb.require()
    ld = hb.typed_rows(table, "table")
    flat = hb.int_vector(ids, "ids", table.device)
    rows, dim = table.shape
    if out is None:
        dst, ldo = table.new_empty((*ids.shape, dim)), dim
    else:
        ldo = _out_matrix(out, (flat.numel(), dim), table, "out")
        if hb.overlap(out, table) or hb.overlap(out, flat):
            raise hb.HipKernelError("lookup: out must not overlap the table or the ids")
        dst = out
    hb._check(lib.dtf_embed_lookup(table.data_ptr(), hb.TYPE_CODES[table.dtype], rows, dim, ld, flat.data_ptr(),
                                   int(flat.dtype == torch.int64), flat.numel(), float(scale), dst.data_ptr(), ldo,
                                   hb._stream(table)), "dtf_embed_lookup")
    if out is not None:
        hb.written(out)
    return dst


def _workspace(lib, tokens: int, dim: int, device) -> torch.Tensor:
    need = lib.dtf_embed_workspace(tokens, dim)
    if need < 0:
        raise hb.HipKernelError(f"dtf_embed_workspace: {tokens} tokens of {dim} elements are not supported")
    return torch.empty(need, dtype=torch.uint8, device=device)


def lookup_grad(ids: torch.Tensor, grad: torch.Tensor, rows: int, scale: float = 1.0,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the whole table: ``out[v, :] = scale * sum of grad[t, :] over the t with ids[t] == v``, zeros in the rows that
    do not occur.  ``grad``: ``ids.shape + (dim,)`` in the table's type."""
    lib = hb.require()
    flat = hb.int_vector(ids, "ids", grad.device)
    g, ldg = _gradient_rows(ids, grad)
    dim = g.shape[1]
    if out is None:
        out = g.new_empty((rows, dim))
    ldt = _out_matrix(out, (rows, dim), g, "out")
    if hb.overlap(out, g) or hb.overlap(out, flat):
        raise hb.HipKernelError("lookup_grad: out must not overlap the upstream gradient or the ids")
    ws = _workspace(lib, flat.numel(), dim, g.device)
    hb._check(lib.dtf_embed_grad(flat.data_ptr(), int(flat.dtype == torch.int64), flat.numel(), g.data_ptr(), ldg, out.data_ptr(),
                                 hb.TYPE_CODES[g.dtype], rows, dim, ldt, float(scale), ws.data_ptr(), ws.numel(),
                                 hb._stream(g)), "dtf_embed_grad")
    hb.written(out)
    return out


def lookup_sgd(table: torch.Tensor, ids: torch.Tensor, grad: torch.Tensor, lr: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``table[v, :] -= lr * scale * sum of grad[t, :] over the t with ids[t] == v`` in place, for the rows that occur.  ``lr``: a
    one-element float32 tensor on the table's device."""
    lib = hb.require()
    ldt = hb.typed_rows(table, "table")
    flat = hb.int_vector(ids, "ids", table.device)
    g, ldg = _gradient_rows(ids, grad)
    if g.dtype != table.dtype or g.device != table.device or g.shape[1] != table.shape[1]:
        raise hb.HipKernelError(f"lookup_sgd: a gradient of {g.dtype} rows of {g.shape[1]} on {g.device} for a table of {table.dtype} "
                                f"rows of {table.shape[1]} on {table.device}")
    if hb._f32c(lr, "lr").numel() != 1 or lr.device != table.device:
        raise hb.HipKernelError("lookup_sgd: lr is one float32 on the table's device")
    if hb.overlap(table, g) or hb.overlap(table, flat) or hb.overlap(table, lr):
        raise hb.HipKernelError("lookup_sgd: the table must not overlap the gradient, the ids or the learning rate")
    ws = _workspace(lib, flat.numel(), table.shape[1], table.device)
    hb._check(lib.dtf_embed_sgd(flat.data_ptr(), int(flat.dtype == torch.int64), flat.numel(), g.data_ptr(), ldg, table.data_ptr(),
                                hb.TYPE_CODES[table.dtype], table.shape[0], table.shape[1], ldt, float(scale), lr.data_ptr(),
                                ws.data_ptr(), ws.numel(), hb._stream(table)), "dtf_embed_sgd")
    hb.written(table)
    return table


def update_rows(table: torch.Tensor, ids: torch.Tensor, grad: torch.Tensor, lr: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``lookup_sgd`` for tables on either kind of device (CPU tensors: torch, same rules)."""
    if table.is_cuda:
        return lookup_sgd(table, ids, grad, lr, scale)
    flat = ids.reshape(-1).long()
    inside = (flat >= 0) & (flat < table.shape[0])
    rows, step = grad.reshape(-1, table.shape[1])[inside], -float(lr) * float(scale)
    if table.dtype == torch.float32:
        return table.index_add_(0, flat[inside], rows, alpha=step)
    # (sums in fp32 and rounded once; rows that do not occur come back as they were)
    return table.copy_(table.float().index_add_(0, flat[inside], rows.float(), alpha=step))


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        return lookup(table, ids, scale)

    @staticmethod
    @hb.first_order
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        return lookup_grad(ids, g, ctx.rows, ctx.scale), None, None


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]`` with the gradient of the table (GPU: the kernels above; CPU tensors: torch, same rules)."""
    if table.is_cuda:
        return _Lookup.apply(hb.with_rows(table), ids, float(scale))
    inside = (ids >= 0) & (ids < table.shape[0])
    # (16-bit tables: the gradient's sums in fp32, rounded once)
    wide = table.float() if table.dtype in (torch.bfloat16, torch.float16) else table
    rows = torch.nn.functional.embedding(torch.where(inside, ids, torch.zeros_like(ids)).long(), wide) * scale
    return torch.where(inside.unsqueeze(-1), rows, torch.zeros_like(rows)).to(table.dtype)
