"""Softmax cross entropy over many classes with its gradients (``csrc/softmax_loss.cu``): the scores of rows against the
classes are tiles of a tensor-core product that are reduced where they are made, so no matrix of rows × classes is kept."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _native as N
from . import dense

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

KEEP_MB = 2048      # of exponentials that the forward pass leaves for the gradients; the scores of further classes are made again


class _Args(C.Structure):
    _fields_ = [("x", C.c_void_p), ("w", C.c_void_p), ("y", C.c_void_p), ("coef", C.c_void_p), ("loss", C.c_void_p), ("gx", C.c_void_p),
                ("gw", C.c_void_p), ("ldx", C.c_int64), ("ldw", C.c_int64), ("n", C.c_int), ("V", C.c_int), ("d", C.c_int),
                ("dtype", C.c_int), ("want_grad", C.c_int), ("keep_mb", C.c_int), ("ws", C.c_void_p), ("ws_bytes", C.c_int64),
                ("status", C.c_void_p)]


def softmax_loss(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, coef: Optional[torch.Tensor] = None,
                 want_grad: bool = True, want_gx: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(loss, gx, gw) of rows ``x`` [n, d] against classes ``w`` [classes, d], both fp32, bf16 or fp16:
    ``loss[i] = coef[i]·(log Σ_j exp(x_i·w_j) − x_i·w_{y_i})`` in fp32 [n] and the gradients of its sum, in the type of the
    operands (None without ``want_grad``; ``want_gx`` False leaves gx out, for rows that are data).

    ``y``: int64 [n], 0 ≤ y < classes; -1 is a row without a class: whatever x and coef hold there, its loss is 0 and it has
    no part in the gradients.  Another label counts as -1 and is reported by :func:`dense.check_status`.  ``coef``: fp32 [n]
    (None: ones).  Rows of x and w are contiguous, their strides are free.  fp32 operands are multiplied with 22 bits
    (three fp16 products), 16-bit ones as they are; sums are fp32.  The gradients need a workspace of 2 bytes (fp32: 4) for
    each row and class, at most 2 GB: beyond it the classes come in pieces, whose scores are made twice, and n·d floats."""
    for name, t in (("x", x), ("w", w), ("y", y), ("coef", coef)):
        if t is not None and (not t.is_cuda or t.device != x.device):
            raise ValueError(f"softmax_loss: {name} has to be on the GPU of x")
    if x.dtype not in DTYPES or w.dtype != x.dtype:
        raise ValueError(f"softmax_loss takes x and w of one type, fp32, bf16 or fp16: got {x.dtype} and {w.dtype}")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"softmax_loss takes x [n, d] and w [classes, d]: got {tuple(x.shape)} and {tuple(w.shape)}")
    n, d = x.shape
    classes = w.shape[0]
    if classes == 0 or d == 0:
        raise ValueError("softmax_loss needs at least one class and one column")
    if max(n, d, classes) > 1 << 30:
        raise ValueError("softmax_loss takes at most 2^30 rows, classes and columns")
    if (n > 0 and d > 1 and x.stride(1) != 1) or (d > 1 and w.stride(1) != 1):
        raise ValueError("softmax_loss: rows of x and w have to be contiguous")
    if y.dtype != torch.int64 or y.shape != (n,) or (coef is not None and (coef.dtype != torch.float32 or coef.shape != (n,))):
        raise ValueError("softmax_loss takes labels int64 [n] and coefficients float32 [n]")
    with torch.cuda.device(x.device):
        loss = torch.empty(n, dtype=torch.float32, device=x.device)
        gx = torch.empty((n, d), dtype=x.dtype, device=x.device) if want_grad and want_gx else None
        gw = torch.empty((classes, d), dtype=w.dtype, device=x.device) if want_grad else None
        if n == 0:
            return loss, gx, gw.zero_() if want_grad else None
        y, coef = y.contiguous(), None if coef is None else coef.contiguous()
        a = _Args(x.data_ptr(), w.data_ptr(), y.data_ptr(), None if coef is None else coef.data_ptr(), loss.data_ptr(),
                  None if gx is None else gx.data_ptr(), gw.data_ptr() if want_grad else None, x.stride(0), w.stride(0), n, classes, d,
                  DTYPES[x.dtype], int(want_grad), KEEP_MB, None, 0, dense.status_ptr(x.device))
        lib = N.lib()
        lib.psb_softmax_loss_workspace.restype = C.c_int64
        size = lib.psb_softmax_loss_workspace(C.byref(a))
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        a.ws, a.ws_bytes = ws.data_ptr(), size
        N.check(lib.psb_softmax_loss(C.byref(a), N.stream_ptr()), "softmax_loss")
    return loss, gx, gw
