"""Softmax cross entropy over many classes with its gradients (``csrc/softmax_loss.cu``): the scores of rows against the
classes are tiles of a tensor-core product that are reduced where they are made, so no matrix of rows × classes is kept."""
from __future__ import annotations

import ctypes as C
import struct
from typing import Dict, Optional, Tuple

import torch

from . import _native as N
from . import dense

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

KEEP_MB = 2048      # of exponentials that the forward pass leaves for the gradients; the scores of further classes are made again


# the arguments of a call as csrc/softmax_loss.cu has them: x, w, y, coef, loss, gx, gw; strides of x and w; n, classes, d, type,
# want_grad, keep_mb; workspace and its bytes; status words.  A small call is host time: a packed struct is quicker than ctypes'.
_ARGS = struct.Struct("7Q2q6iQqQ")
_sizes: Dict[tuple, int] = {}


def softmax_loss(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, coef: Optional[torch.Tensor] = None,
                 want_grad: bool = True, want_gx: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(loss, gx, gw) of rows ``x`` [n, d] against classes ``w`` [classes, d], both fp32, bf16 or fp16:
    ``loss[i] = coef[i]·(log Σ_j exp(x_i·w_j) − x_i·w_{y_i})`` in fp32 [n] and the gradients of its sum, in the type of the
    operands (None without ``want_grad``; ``want_gx`` False leaves gx out, for rows that are data).

    ``y``: int64 [n], 0 ≤ y < classes; -1 is a row without a class: whatever x and coef hold there, its loss is 0 and it has
    no part in the gradients.  Another label counts as -1 and is reported by :func:`dense.check_status`.  ``coef``: fp32 [n]
    (None: ones).  Rows of x and w are contiguous, their strides are free.  fp32 operands are multiplied with 22 bits (three
    fp16 products) relative to the largest of their own row or class: elements below 2^-17 of it keep fewer, below 2^-39 none.
    In the gradients the same holds for a term beside the largest of its row (gx), or of its and up to 127 neighbouring classes
    (gw).  A small call is one launch, in fp32 throughout.

    16-bit operands are multiplied as they are, and summed in fp32 on the tensor cores, which cut a sum at every 16 elements (scores
    of 1024 columns: 3e-7 of the loss) and are left 4096 columns of scores, or 32,768 terms of gradients, at a time.  The gradient
    of the scores is rounded to the operands' type before its two products (bf16 gradients are off by 0.17 to 0.25 % instead of the
    0.17 % that their own rounding takes); fp16 keeps it relative to the call's largest coefficient, in units of 2^-38 of that.

    Workspace: 8 bytes (fp32 with gradients: 16) for each row and 32 to 128 classes, for losses alone too; fp32 operands once more,
    and 16-bit ones whose rows do not start at 16 bytes; for gradients x once more, 2 bytes (fp32: 8) for each row and class, at most
    2 GB (or 256 classes; beyond that the classes come in pieces, whose scores are made twice), and fp32 copies of gx, and of either
    gradient where its product is split."""
    gpu = x.get_device()
    for name, t in (("x", x), ("w", w), ("y", y), ("coef", coef)):
        if t is not None and (t.get_device() != gpu or gpu < 0):
            raise ValueError(f"softmax_loss: {name} has to be on the GPU of x")
    dtype = DTYPES.get(x.dtype)
    if dtype is None or w.dtype != x.dtype:
        raise ValueError(f"softmax_loss takes x and w of one type, fp32, bf16 or fp16: got {x.dtype} and {w.dtype}")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"softmax_loss takes x [n, d] and w [classes, d]: got {tuple(x.shape)} and {tuple(w.shape)}")
    n, d = x.shape
    classes = w.shape[0]
    if classes == 0 or d == 0:
        raise ValueError("softmax_loss needs at least one class and one column")
    if max(n, d, classes) > 1 << 30:
        raise ValueError("softmax_loss takes at most 2^30 rows, classes and columns")
    (ldx, sx), (ldw, sw) = x.stride(), w.stride()
    if d > 1 and ((n > 0 and sx != 1) or sw != 1):
        raise ValueError("softmax_loss: rows of x and w have to be contiguous")
    if y.dtype != torch.int64 or y.dim() != 1 or y.shape[0] != n or (coef is not None and (coef.dtype != torch.float32 or coef.shape != (n,))):
        raise ValueError("softmax_loss takes labels int64 [n] and coefficients float32 [n]")
    if torch.cuda.current_device() != gpu:
        with torch.cuda.device(gpu):
            return softmax_loss(x, w, y, coef, want_grad, want_gx)
    dev = x.device
    loss = torch.empty(n, dtype=torch.float32, device=dev)
    gx = torch.empty((n, d), dtype=x.dtype, device=dev) if want_grad and want_gx else None
    gw = torch.empty((classes, d), dtype=w.dtype, device=dev) if want_grad else None
    if n == 0:
        return loss, gx, gw.zero_() if want_grad else None
    y, coef = y.contiguous(), None if coef is None else coef.contiguous()
    px, pw, pgx, pgw = x.data_ptr(), w.data_ptr(), 0 if gx is None else gx.data_ptr(), 0 if gw is None else gw.data_ptr()
    want = 1 if want_grad else 0
    lib = N.lib()
    # the workspace depends on sizes, types and alignment alone
    key = (n, classes, d, dtype, want, pgx == 0, KEEP_MB, ldx, ldw, px & 15, pw & 15)
    size = _sizes.get(key)
    if size is None:
        lib.psb_softmax_loss_workspace.restype = C.c_int64
        size = lib.psb_softmax_loss_workspace(_ARGS.pack(px, pw, 0, 0, 0, pgx, pgw, ldx, ldw, n, classes, d, dtype, want, KEEP_MB, 0, 0, 0))
        if len(_sizes) >= 1024:
            _sizes.clear()
        _sizes[key] = size
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None      # small calls need none
    args = _ARGS.pack(px, pw, y.data_ptr(), 0 if coef is None else coef.data_ptr(), loss.data_ptr(), pgx, pgw, ldx, ldw, n, classes, d,
                      dtype, want, KEEP_MB, 0 if ws is None else ws.data_ptr(), size, dense.status_ptr(dev))
    N.check(lib.psb_softmax_loss(args, N.raw_stream(gpu)), "softmax_loss")
    return loss, gx, gw
