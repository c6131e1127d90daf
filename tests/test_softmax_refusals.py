"""What the softmax loss refuses before a kernel sees it (no GPU needed: tensors that are not on one are refused first)."""
import ctypes

import pytest
import torch

from parameter_server_b200.ops import _native, softmax


def test_tensors_outside_the_gpu_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        softmax.softmax_loss(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("change", [
    dict(w=lambda t: t.bfloat16()), dict(x=lambda t: t.double(), w=lambda t: t.double()), dict(x=lambda t: t[0]), dict(w=lambda t: t[:, :3]),
    dict(w=lambda t: t[:0]), dict(x=lambda t: t[:, :0], w=lambda t: t[:, :0]), dict(x=lambda t: t.T.contiguous().T),
    dict(w=lambda t: t.T.contiguous().T), dict(y=lambda t: t.int()), dict(y=lambda t: t[:1]), dict(y=lambda t: t[:, None]),
    dict(y=lambda t: t.cpu()), dict(coef=lambda t: t.double()), dict(coef=lambda t: t[:1]), dict(coef=lambda t: t.cpu())])
def test_refusals(change):
    a = {"x": torch.zeros(2, 4, device="cuda"), "w": torch.zeros(3, 4, device="cuda"), "y": torch.zeros(2, dtype=torch.int64, device="cuda"),
         "coef": torch.ones(2, device="cuda")}
    softmax.softmax_loss(**a)
    for k, f in change.items():
        a[k] = f(a[k])
    with pytest.raises(ValueError):
        softmax.softmax_loss(**a)


@pytest.mark.parametrize("n,V,d", [(65_536, 131_072, 4096), (65_536, 131_072, 512), (1_000_000, 131_072, 64), (700, 900, 33), (3000, 257, 2000)])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("grad", [0, 1])
def test_workspace_is_the_stated_one(n, V, d, dtype, grad):
    """The bytes that the documentation of the loss gives, from the planning code on the host."""
    lib = _native.lib()
    lib.psb_softmax_loss_workspace.restype = ctypes.c_int64
    size = lib.psb_softmax_loss_workspace(softmax._ARGS.pack(256, 256, 0, 0, 0, 256 * grad, 256 * grad, d, d, n, V, d, dtype, grad, 2048, 0, 0, 0))
    aligned, pad = d % 8 == 0, 1 << 16
    part = 16 if dtype == 0 and grad else 8
    packed = (n + V) * (d + 7) * 4 if dtype == 0 else (0 if aligned else V * (d + 7) * 2) + (n * (d + 7) * 2 if grad or not aligned else 0)
    assert n * (V // 128) * part <= size
    most = n * (V / 32 + 8) * part + packed + n * 48 + V * 8 + pad
    if grad:
        each = 8 if dtype == 0 else 2
        most += max(2 << 30, 256 * n * each) + n * 8 * each
        most += 64 * n * d * 4 + 16 * V * d * 4 if n * V < 1 << 24 else 16 * max(n, V) * d * 4
    assert size <= most
