"""Orthogonalised updates of matrices (csrc/muon.hip): the Muon optimiser's step on the matrix cores.

``orthogonalize(x)`` is the factor alone: five Newton-Schulz steps of the odd quintic (3.4445, -4.7750, 2.0315) on
``x / (|x|_F + eps)``, with the accuracy of fp32 matrix products for any input type, also in rows and columns that are little next
to the others (down to 2^-100 of the norm).  ``MuonPlan`` + ``muon_step`` are the optimiser step over a fixed list of matrices, momentum
and weight update included, every launch shared by all of them;
``train.MuonOptimizer`` runs it for the matrices of a graph.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch

from . import hip_backend as hb

EPS = 1e-7
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
GROUP = 8           # matrices per native call (DTF_MUON_MAX)


def _workspace(lib, shapes, device) -> torch.Tensor:
    n = len(shapes)
    need = lib.dtf_muon_workspace(n, (C.c_int32 * n)(*[s[0] for s in shapes]), (C.c_int32 * n)(*[s[1] for s in shapes]))
    if need < 0:
        raise hb.HipKernelError(f"dtf_muon_workspace: shapes {[tuple(s) for s in shapes]} are not supported")
    return torch.empty(need, dtype=torch.uint8, device=device)


def orthogonalize(x: torch.Tensor, eps: float = EPS, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The Newton-Schulz factor of a matrix, in its type; the zero matrix for a zero matrix.  ``out`` may be ``x`` itself."""
    lib = hb.require()
    ldx = hb.typed_rows(x, "x")
    if out is None:
        out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise hb.HipKernelError(f"orthogonalize: out must be a {x.dtype} tensor of shape {tuple(x.shape)} on {x.device}")
    ldo = hb.typed_rows(out, "out")
    ws = _workspace(lib, [x.shape], x.device)
    hb._check(lib.dtf_orthogonalize(x.data_ptr(), hb.TYPE_CODES[x.dtype], x.shape[0], x.shape[1], ldx, out.data_ptr(), ldo,
                                    float(eps), ws.data_ptr(), ws.numel(), hb._stream(x)), "dtf_orthogonalize")
    hb.written(out)
    return out


class MuonPlan:
    """A fixed list of float32 matrices ``[in, out]`` with their gradients and momentum buffers, and the workspace their steps use.
    The steps read and write the memory that the tensors have when the plan is made (and keep it alive): write new gradients
    into the same tensors.  One step of a plan at a time: two streams, or two captured graphs that may overlap, need a plan each.
    A plan may be dropped while a step is under way on any stream; one whose steps a graph has captured has to outlive the graph."""

    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor]):
        params, grads, momenta = list(params), list(grads), list(momenta)
        if not params or len(grads) != len(params) or len(momenta) != len(params):
            raise hb.HipKernelError("MuonPlan: a gradient and a momentum buffer for every one of at least one matrix")
        for w, g, b in zip(params, grads, momenta):
            hb._f32c(w, "params"), hb._f32c(g, "grads"), hb._f32c(b, "momenta")
            if w.dim() != 2 or not w.numel() or g.shape != w.shape or b.shape != w.shape:
                raise hb.HipKernelError(f"MuonPlan: matrices of one shape, got {tuple(w.shape)}, {tuple(g.shape)}, {tuple(b.shape)}")
            if g.device != w.device or b.device != w.device or w.device != params[0].device:
                raise hb.HipKernelError("MuonPlan: all tensors on one device")
        written = params + momenta
        for i, a in enumerate(written):
            if any(hb.overlap(a, b) for b in written[i + 1:] + grads):
                raise hb.HipKernelError("MuonPlan: weights and momentum buffers must not overlap each other or the gradients")
        lib = hb.require()
        self.params, self.grads, self.momenta = ([t.detach() for t in ts] for ts in (params, grads, momenta))
        self.device = params[0].device
        self._written = [hb._span(t) for t in written]
        self._groups = []
        # streams whose work the allocator waits for before it gives the memory away
        self._streams = {torch.cuda.current_stream(self.device).cuda_stream}
        for i in range(0, len(params), GROUP):
            ws, gs, bs = params[i:i + GROUP], grads[i:i + GROUP], momenta[i:i + GROUP]
            n = len(ws)
            self._groups.append((n, (C.c_int32 * n)(*[t.shape[0] for t in ws]), (C.c_int32 * n)(*[t.shape[1] for t in ws]),
                                 *[(C.c_uint64 * n)(*[t.data_ptr() for t in ts]) for ts in (ws, gs, bs)],
                                 _workspace(lib, [t.shape for t in ws], self.device)))


def muon_step(plan: MuonPlan, lr: torch.Tensor, *, momentum: float = 0.95, nesterov: bool = True, eps: float = EPS) -> None:
    """``buf = momentum * buf + g;  w -= lr * sqrt(max(1, cols / rows)) * orthogonalize(g + momentum * buf)`` (``buf`` itself without
    ``nesterov``) for every matrix of the plan, in place.  ``lr``: a one-element float32 tensor on the plan's device."""
    lib = hb.require()
    if hb._f32c(lr, "lr").numel() != 1 or lr.device != plan.device:
        raise hb.HipKernelError("muon_step: lr is one float32 on the plan's device")
    at = lr.data_ptr()
    if any(first <= at < end for first, end in plan._written):
        raise hb.HipKernelError("muon_step: the learning rate lies in a weight or momentum that the step writes")
    stream = hb._stream(lr)
    if stream not in plan._streams:
        side = torch.cuda.current_stream(plan.device)
        for t in (*plan.params, *plan.grads, *plan.momenta, *[group[-1] for group in plan._groups]):
            t.record_stream(side)
        plan._streams.add(stream)
    for n, rows, cols, w, g, b, ws in plan._groups:
        hb._check(lib.dtf_muon_step(n, rows, cols, w, g, b, at, float(momentum), int(bool(nesterov)), float(eps),
                                    ws.data_ptr(), ws.numel(), stream), "dtf_muon_step")
    hb.written(plan.params + plan.momenta)
