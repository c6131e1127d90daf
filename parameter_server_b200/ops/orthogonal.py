"""Orthogonalised weight updates (``csrc/orthogonal.cu``): Newton-Schulz steps with the polynomial of the Muon optimiser on
the tensor cores, alone and as an update rule next to :func:`dense.sgd_update`."""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Dict

import torch

from . import _native as N
from . import dense

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
EPS = 1e-7            # added to the Frobenius norm that the steps start from
MAX_STEPS = 64


# the arguments of a call as csrc/orthogonal.cu has them: x or the gradient, momentum, result or weights; batch, rows, cols, type,
# steps, nesterov; lr, momentum, eps; workspace and its bytes; status words
_ARGS = struct.Struct("3Q6i4fQqQ")


_sizes: Dict[tuple, int] = {}
_F32 = (torch.float32,)


def _check(what: str, t: torch.Tensor, gpu: int, shape, dtypes) -> None:
    if t.get_device() != gpu or gpu < 0:
        raise ValueError(f"{what} has to be on the GPU of the first tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} has to be {' or '.join(str(d) for d in dtypes)}: got {t.dtype}")
    if t.shape != shape or not 2 <= len(shape) <= 3:
        raise ValueError(f"{what}: matrices [rows, cols] or [batch, rows, cols] of one shape: got {tuple(t.shape)} and {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what} has to be contiguous")


def _run(x, m, out, gpu, shape, steps, lr, momentum, nesterov) -> None:
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"1 to {MAX_STEPS} steps: got {steps}")
    batch, rows, cols = (1, *shape) if len(shape) == 2 else shape
    if batch > 65535 or max(rows, cols) > 1 << 30:
        raise ValueError("at most 65,535 matrices of at most 2^30 rows and columns")
    if batch * rows * cols == 0:
        return
    if torch.cuda.current_device() != gpu:
        with torch.cuda.device(gpu):
            return _run(x, m, out, gpu, shape, steps, lr, momentum, nesterov)
    dev = x.device
    lib = N.lib()
    key = (gpu, batch, rows, cols)
    size = _sizes.get(key)
    if size is None:
        lib.psb_orthogonal_workspace.restype = C.c_int64
        size = lib.psb_orthogonal_workspace(_ARGS.pack(0, 0, 0, batch, rows, cols, 0, steps, 0, lr, momentum, EPS, 0.0, 0, 0, 0))
        if len(_sizes) >= 1024:
            _sizes.clear()
        _sizes[key] = size
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None      # small matrices need none
    args = _ARGS.pack(x.data_ptr(), 0 if m is None else m.data_ptr(), out.data_ptr(), batch, rows, cols, DTYPES[x.dtype], steps,
                      1 if nesterov else 0, lr, momentum, EPS, 0.0, 0 if ws is None else ws.data_ptr(), size, dense.status_ptr(dev))
    N.check(lib.psb_orthogonal(args, N.raw_stream(gpu)), "orthogonal")


def orthogonalize(x: torch.Tensor, steps: int = 5) -> torch.Tensor:
    """``steps`` Newton-Schulz steps on a contiguous matrix [rows, cols] or a batch [batch, rows, cols], fp32, bf16 or
    fp16: ``X = x / (|x|_F + 1e-7)``, then ``X ← 3.4445 X − 4.7750 (X Xᵀ) X + 2.0315 (X Xᵀ)² X`` each, which brings singular
    values into about [0.7, 1.2].  The result has the type of x; fp32 and fp16 results are computed with 22-bit operands, bf16 ones
    with 22 bits up to the last step and 11 bits in that (off by 0.18 to 0.21 % instead of the 0.17 % of their rounding); a short
    side of at most 16 is computed in fp32.  The workspace takes 8 bytes an element of x and 12 bytes or more an element of the
    smaller square, none where a short side of at most 128 keeps the matrix on the SMs."""
    gpu, shape = x.get_device(), x.shape
    _check("orthogonalize: x", x, gpu, shape, DTYPES)
    out = torch.empty_like(x)
    _run(x, None, out, gpu, shape, steps, 0.0, 0.0, False)
    return out


def orthogonal_update(w: torch.Tensor, g: torch.Tensor, m: torch.Tensor, lr: float, momentum: float = 0.95, nesterov: bool = True,
                      steps: int = 5) -> None:
    """One update of fp32 weights ``w`` [rows, cols] or [batch, rows, cols] with their gradient ``g`` (fp32, bf16 or fp16) and
    momentum ``m`` (fp32), in place: ``m ← momentum·m + g``, ``w ← w − lr·√max(1, rows/cols)·orthogonalize(u)`` with
    ``u = g + momentum·m`` (``nesterov``) or ``m``, all contiguous and apart in memory.  The momentum is written first and the weights
    last: where a launch between them fails, the call raises with the momentum moved on and the weights as they were."""
    gpu, shape = w.get_device(), w.shape
    _check("orthogonal_update: w", w, gpu, shape, _F32)
    _check("orthogonal_update: g", g, gpu, shape, DTYPES)
    _check("orthogonal_update: m", m, gpu, shape, _F32)
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (w, g, m))
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("orthogonal_update: w, g and m share memory")
    _run(g, m, w, gpu, shape, steps, lr * math.sqrt(max(1.0, shape[-2] / max(shape[-1], 1))), momentum, nesterov)
    dense._written(w)
    dense._written(m)
