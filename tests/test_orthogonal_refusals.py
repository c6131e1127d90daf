"""What the orthogonalised update refuses before a kernel sees it."""
import pytest
import torch

from parameter_server_b200.ops import orthogonal


def test_tensors_outside_the_gpu_are_refused():
    t = torch.zeros(4, 4)
    with pytest.raises(ValueError, match="GPU"):
        orthogonal.orthogonalize(t)
    with pytest.raises(ValueError, match="GPU"):
        orthogonal.orthogonal_update(t, t, t, 0.1)


@pytest.mark.gpu
def test_refusals():
    def t(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    for bad in (t(4), t(2, 2, 2, 2), t(4, 4, dtype=torch.float64), t(4, 4, dtype=torch.int32), t(4, 6).T, t(4, 6)[:, :4], t(65536, 1, 1)):
        with pytest.raises(ValueError):
            orthogonal.orthogonalize(bad)
    for steps in (0, -1, 65):
        with pytest.raises(ValueError):
            orthogonal.orthogonalize(t(4, 4), steps)
    w, g, m = t(4, 4), t(4, 4), t(4, 4)
    orthogonal.orthogonal_update(w, g, m, 0.1)
    for args in ((w.bfloat16(), g, m), (w, g, m.half()), (w, t(4, 5), m), (w, g, t(3, 4)), (w, g.cpu(), m), (w, w, m), (w, g, w), (w, g, g),
                 (w, g.double(), m), (w.T[:2], g[:2], m[:2])):
        with pytest.raises(ValueError):
            orthogonal.orthogonal_update(*args, 0.1)
