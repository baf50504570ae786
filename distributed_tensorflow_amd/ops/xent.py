"""Softmax cross-entropy against integer labels (csrc/xent.hip): the output end of a model over tokens, where the one-hot
labels of ``hip_backend.softmax_xent`` would be a matrix as large as the logits.

``sparse_softmax_xent(logits, labels)`` is the differentiable operator: the loss of every row
(``tf.nn.sparse_softmax_cross_entropy_with_logits`` of a graph evaluates to it).  ``sparse_softmax_xent_step`` is the training
step's form: losses and gradient in ONE launch that reads the logits once and keeps each row in registers in between (two
launches for up to 64 rows of more than 256 KB, one for every 2^21 rows).

A negative label is padding: loss 0, a gradient row of zeros, the row's logits are not looked at.  A label that is no class
(``>= classes``) gives NaN.  Logits in float32, bfloat16 or float16 with contiguous rows; losses in float32.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import hip_backend as hb


def _operands(logits: torch.Tensor, labels: torch.Tensor):
    ld = hb.typed_rows(logits, "logits")
    flat = hb.int_vector(labels, "labels", logits.device)
    if labels.dim() != 1 or flat.numel() != logits.shape[0]:
        raise hb.HipKernelError(f"sparse_softmax_xent: one label per row of the logits, got {tuple(labels.shape)} for "
                                f"{tuple(logits.shape)}")
    return ld, flat


def _dz_rows(dz: torch.Tensor, logits: torch.Tensor) -> int:
    if dz.shape != logits.shape or dz.dtype != logits.dtype or dz.device != logits.device:
        raise hb.HipKernelError("sparse_softmax_xent: dz must be shaped and typed like the logits, on their device")
    if (dz.data_ptr() != logits.data_ptr() or dz.stride() != logits.stride()) and hb.overlap(dz, logits):
        raise hb.HipKernelError("sparse_softmax_xent: dz may be the logits themselves, but not overlap them otherwise")
    return hb.typed_rows(dz, "dz")


LAUNCH_ROWS = 1 << 21        # of one native call


def _parts(rows: int):
    return [slice(a, min(a + LAUNCH_ROWS, rows)) for a in range(0, rows, LAUNCH_ROWS)]


def _launch(lib, logits, ld, flat, dz, ldz, grad_scale, loss, stats):
    rows, classes = logits.shape
    code = hb.TYPE_CODES[logits.dtype]
    args = (logits.data_ptr(), code, rows, classes, ld, flat.data_ptr(), int(flat.dtype == torch.int64), hb._ptr(dz), ldz,
            float(grad_scale), loss.data_ptr(), hb._ptr(stats))
    # few long rows: several blocks each, which need a workspace
    need = lib.dtf_sparse_xent_workspace(code, rows, classes) if rows <= 64 and classes >= 1 << 16 else 0
    if need > 0:
        ws = torch.empty(need, dtype=torch.uint8, device=logits.device)
        hb._check(lib.dtf_sparse_xent_cut(*args, ws.data_ptr(), need, hb._stream(logits)), "dtf_sparse_xent_cut")
    else:
        hb._check(lib.dtf_sparse_xent(*args, hb._stream(logits)), "dtf_sparse_xent")


def _forward(logits, labels, dz, grad_scale, stats):
    lib = hb.require()
    ld, flat = _operands(logits, labels)
    ldz = 0 if dz is None else _dz_rows(dz, logits)
    loss = torch.empty((logits.shape[0],), device=logits.device, dtype=torch.float32)
    if logits.shape[0] <= LAUNCH_ROWS:
        _launch(lib, logits, ld, flat, dz, ldz, grad_scale, loss, stats)
    else:
        for r in _parts(logits.shape[0]):
            _launch(lib, logits[r], ld, flat[r], None if dz is None else dz[r], ldz, grad_scale, loss[r],
                    None if stats is None else stats[r])
    return loss, flat


def sparse_softmax_xent_step(logits: torch.Tensor, labels: torch.Tensor, *, dz: Optional[torch.Tensor] = None,
                             grad_scale: float = 1.0) -> torch.Tensor:
    """Row losses (float32 ``[rows]``); ``dz`` (shaped like the logits, or the logits themselves) receives
    ``grad_scale * d(row loss)/d(logits)`` in the same launch."""
    loss = _forward(logits, labels, dz, grad_scale, None)[0]
    if dz is not None:
        hb.written(dz)
    return loss


class _SparseXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels):
        stats = torch.empty((logits.shape[0], 2), device=logits.device, dtype=torch.float32)
        loss, flat = _forward(logits, labels, None, 1.0, stats)
        ctx.save_for_backward(logits, flat, stats)
        return loss

    @staticmethod
    @hb.first_order
    def backward(ctx, g):
        z, flat, stats = ctx.saved_tensors
        g = g.to(torch.float32)
        dz = torch.empty(z.shape, device=z.device, dtype=z.dtype)
        lib, ld = hb.require(), hb.typed_rows(z, "logits")
        whole = (z, flat, stats, g, dz)
        for z, flat, stats, g, to in [whole] if dz.shape[0] <= LAUNCH_ROWS else [[t[r] for t in whole] for r in _parts(dz.shape[0])]:
            hb._check(lib.dtf_sparse_xent_grad(z.data_ptr(), hb.TYPE_CODES[z.dtype], z.shape[0], z.shape[1], ld, flat.data_ptr(),
                                               int(flat.dtype == torch.int64), stats.data_ptr(), g.data_ptr(), g.stride(0),
                                               to.data_ptr(), z.shape[1], hb._stream(z)), "dtf_sparse_xent_grad")
        return dz, None


def sparse_softmax_xent(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Loss of every row, differentiable in the logits (GPU: the kernels above; CPU tensors: torch, same rules)."""
    if logits.is_cuda:
        return _SparseXent.apply(hb.with_rows(logits), labels)
    if logits.dim() != 2 or labels.dim() != 1 or labels.shape[0] != logits.shape[0]:
        raise ValueError("sparse_softmax_xent: one label per row of 2-D logits")
    classes = logits.shape[1]
    known = (labels >= 0) & (labels < classes)
    at = torch.where(known, labels, torch.zeros_like(labels)).long()
    # (the rows without a class are left out before the softmax, so that their logits cannot reach anything)
    z = torch.where(known[:, None], logits.float(), torch.zeros_like(logits, dtype=torch.float32))
    loss = -torch.log_softmax(z, dim=1).gather(1, at[:, None])[:, 0]
    loss = torch.where(known, loss, torch.zeros_like(loss))
    wrong = labels >= classes
    nan = (torch.where(wrong[:, None], logits.float(), torch.zeros_like(z)) * float("nan")).sum(1)
    return torch.where(wrong, nan, loss)
