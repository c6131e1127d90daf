"""What the softmax loss refuses before a kernel sees it (no GPU needed: tensors that are not on one are refused first)."""
import pytest
import torch

from parameter_server_b200.ops import softmax


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
