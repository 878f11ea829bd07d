"""The global gradient norm over many tensors, and clipping, as native kernels.

``clip_grad_norm_(grads, max_norm)`` is what stands between ``loss.backward()`` and ``opt.step()``: one pass
over all gradients for their norm and, where it is above ``max_norm``, one that scales them, whatever
their number, sizes and types.  CUDA only, like every op here.
"""
from __future__ import annotations

import ctypes
from typing import Iterable, Optional, Sequence

import torch

from .. import _lib
from .flash_born import _DTYPE_CODE, _stream_handle

__all__ = ["clip_grad_norm_", "grad_norm"]


def _run(grads: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]], max_norm: float, eps: float,
         what: str) -> torch.Tensor:
    if not grads:
        raise ValueError(f"{what}: no gradients given (their device is the result's)")
    device = grads[0].device
    tensors = list(grads) if out is None or out is grads else list(grads) + list(out)
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError(f"{what} (B200): CUDA tensors required; there is no CPU path")
        if t.device != device:
            raise RuntimeError(f"{what}: all tensors must be on {device}; got one on {t.device}")
        if t.dtype not in _DTYPE_CODE:
            raise ValueError(f"{what}: gradients are dense float32 / float16 / bfloat16; got {t.dtype}")
    n = len(grads)
    a = _lib.FbClipArgs()
    a.count, a.max_norm, a.eps = n, max_norm, eps
    keep = [(ctypes.c_void_p * n)(*[g.data_ptr() for g in grads]), (ctypes.c_int64 * n)(*[g.numel() for g in grads]),
            (ctypes.c_int32 * n)(*[_DTYPE_CODE[g.dtype] for g in grads])]
    a.grads, a.numel, a.dtype = (ctypes.cast(x, ctypes.c_void_p) for x in keep)
    if out is not None:
        keep += [(ctypes.c_void_p * n)(*[o.data_ptr() for o in out]), (ctypes.c_int32 * n)(*[_DTYPE_CODE[o.dtype] for o in out])]
        a.out, a.out_dtype = (ctypes.cast(x, ctypes.c_void_p) for x in keep[3:])
    norm = torch.empty((), dtype=torch.float32, device=device)
    lib = _lib.load()
    need = lib.fb_clip_workspace_size(ctypes.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    a.norm, a.workspace, a.workspace_bytes = norm.data_ptr(), ws.data_ptr(), need
    with torch.cuda.device(device):
        _lib.check(lib.fb_clip_grad_norm(ctypes.byref(a), _stream_handle(device)), what)
    return norm


def _dense(t: torch.Tensor) -> bool:
    """Every element of the storage span used once: the kernels take elements in memory order."""
    if t.layout is not torch.strided:
        return False
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size == 1:
            continue
        if stride != want:
            return False
        want *= size
    return True


def grad_norm(grads: Iterable[torch.Tensor]) -> torch.Tensor:
    """``sqrt(sum g^2)`` over all tensors, a 0-d fp32 tensor on their device (no host synchronisation)."""
    gs = [g.detach() for g in grads]
    gs = [g if _dense(g) else g.contiguous() for g in gs]
    return _run(gs, None, 0.0, 0.0, "grad_norm")


def clip_grad_norm_(
    grads: Iterable[torch.Tensor],
    max_norm: float,
    eps: float = 1e-6,
    out: Optional[Iterable[torch.Tensor]] = None,
) -> torch.Tensor:
    """Scale all ``grads`` by ``min(1, max_norm / (norm + eps))``; returns the norm before, a 0-d fp32 tensor.

    grads are dense CUDA tensors of any sizes, float32 / float16 / bfloat16, mixed as they come (pass
    ``[p.grad for p in params if p.grad is not None]``), each listed once.  They change in place; with
    ``out`` they stay and the scaled gradients go there: same shapes and memory order, each of its gradient's
    dtype or float32 (16-bit gradients into an optimiser's 32-bit buffers).  In place, a norm at most
    ``max_norm`` writes nothing.  A NaN or inf among the gradients shows in the norm, and then in the results.
    The same gradients give the same norm, bit for bit.
    """
    gs = list(grads)
    if not (max_norm >= 0.0 and eps >= 0.0):
        raise ValueError(f"clip_grad_norm_: max_norm and eps must not be negative; got {max_norm}, {eps}")
    to = gs if out is None else list(out)
    if len(to) != len(gs):
        raise ValueError(f"clip_grad_norm_: {len(gs)} gradients, but out has {len(to)} tensors")
    for g in gs:
        if not _dense(g):
            raise ValueError(f"clip_grad_norm_: gradients must be dense; got strides {g.stride()} for {tuple(g.shape)}")
    if to is not gs:
        for g, o in zip(gs, to):
            if o.shape != g.shape or o.stride() != g.stride() or o.dtype not in (g.dtype, torch.float32):
                raise ValueError(f"clip_grad_norm_: out must match its gradient's shape and strides, and its dtype or "
                                 f"float32; got {tuple(o.shape)} {o.stride()} {o.dtype} for {tuple(g.shape)} "
                                 f"{g.stride()} {g.dtype}")
    return _run(gs, to, float(max_norm), float(eps), "clip_grad_norm_")
