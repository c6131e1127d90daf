"""Newton-Schulz orthogonalisation and the weight update that uses it against their definition in 64 bits.

Bounds (Frobenius norms, |X| elementwise where a product of magnitudes is meant).  A step is f(X) = a X + (b A + c A²) X with
A = X Xᵀ.  On singular values up to 1.25, where they stay, |f'| and the divided differences of f are at most 4.3, so an
error E in X becomes at most 4.3 E.  A step adds
  e_a = u ‖|X||X|ᵀ‖ + r ‖A‖                                  the product, and A's rounding to its planes
  e_b = |b| e_a + 2 c ‖A‖₂ e_a + u ‖|A||A'|‖ + r (‖A‖₂ ‖A'‖ + ‖B‖)   the same for B = A A' + a I with A' = b I + c A
  ‖X‖₂ e_b + u ‖|B||X|‖ + r ‖X‖                              the same for the new X = B X
with r the rounding to planes (two: 2^-22, one: 2^-11) and u that of a product: r for either factor and for the product
that two planes leave out (one plane: operands are what they are, r is counted where they were rounded), 2^-23 for each of
24 steps on the tensor cores and 2^-24 a sum of 128 elements (one plane: 2^-23 for each of K/16 steps).  The planes' smallest
unit, 2^-25 of values scaled by 2^10, adds 2^-35 an element.  The norm that the steps start from is exact to fp32's rounding."""
import pytest
import torch

pytestmark = pytest.mark.gpu

COEFS = (3.4445, -4.7750, 2.0315)
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _reference(x, steps, dtype):
    """The result in fp64 and the bound of its error (2-norm over all elements), for one matrix."""
    a, b, c = COEFS
    X = x.double() / (x.double().norm() + 1e-7)
    tall = X.shape[0] > X.shape[1]
    X = X.T if tall else X
    err = 2.0 ** -22 * X.norm() + 2.0 ** -35 * X.numel() ** 0.5
    for k in range(steps):
        one = dtype == torch.bfloat16 and k == steps - 1
        r = 2.0 ** -11 if one else 2.0 ** -22

        def u(K):
            return 2.0 ** -23 * (K / 16 + 1) if one else 3 * 2.0 ** -22 + 24 * 2.0 ** -23 + 2.0 ** -24 * (K / 128 + 1)

        eye = torch.eye(X.shape[0], dtype=torch.float64, device=X.device)
        A = X @ X.T
        A2 = b * eye + c * A
        B = A @ A2 + a * eye
        tiny, na = 2.0 ** -35 * X.shape[0], torch.linalg.matrix_norm(A, 2)
        e_a = u(X.shape[1]) * (X.abs() @ X.abs().T).norm() + r * A.norm() + tiny
        e_b = (abs(b) + 2 * c * na) * e_a + u(A.shape[0]) * (A.abs() @ A2.abs()).norm() + r * (na * A2.norm() + B.norm()) + tiny
        nx = torch.linalg.matrix_norm(X, 2)
        if one:
            err = err + r * X.norm()                     # its low plane is left out from here on
        X, old = B @ X, X
        err = 4.3 * err + nx * e_b + u(B.shape[0]) * (B.abs() @ old.abs()).norm() + r * X.norm() + 2.0 ** -35 * X.numel() ** 0.5
    return (X.T if tall else X), err


def _data(shape, seed=0, strong=16, floor=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    k = min(strong, *shape[-2:])
    x = floor * torch.randn(*shape, generator=g, device="cuda")
    return x + torch.randn(*shape[:-1], k, generator=g, device="cuda") @ torch.randn(*shape[:-2], k, shape[-1], generator=g, device="cuda")


def _check(x, steps=5):
    from parameter_server_b200.ops import dense, orthogonal

    before = x.clone()
    got = orthogonal.orthogonalize(x, steps)
    torch.cuda.synchronize()
    dense.check_status(x.device)
    assert got.dtype == x.dtype and got.shape == x.shape and torch.equal(x, before)
    for o, i in zip(got, x) if x.dim() == 3 else [(got, x)]:
        ref, err = _reference(i, steps, x.dtype)
        off, tol = (o.double() - ref).norm().item(), (err + 1.01 * HALF_STEP[x.dtype] * ref.norm()).item()
        if x.dtype == torch.float16:
            tol += 2.0 ** -25 * ref.numel() ** 0.5
        assert off <= tol, (off, tol, ref.norm().item())
    return got


@pytest.mark.parametrize("shape", [(1, 1), (1, 5), (7, 1), (2, 2), (8, 9), (64, 64), (63, 65), (129, 127), (64, 8000), (8000, 65), (1, 9000),
                                   (1000, 520), (513, 2049), (1025, 1023), (2600, 2500), (3, 40, 72), (5, 72, 40), (2, 257, 1100), (300, 17, 5),
                                   # one CTA, clusters of 2 to 16, either way round, and what just does not fit
                                   (128, 128), (17, 512), (16, 513), (128, 200), (100, 400), (400, 100), (64, 1025), (128, 1024), (128, 1025),
                                   (1024, 127), (112, 2048), (3, 48, 3000), (2, 8192, 64), (64, 8193), (129, 130),
                                   # in registers: every number of rows, columns a thread and CTAs, and what just does not fit
                                   (2, 300), (3, 2), (4, 4097), (5, 70), (8, 512), (700, 9), (15, 1), (16, 16), (16, 257), (16, 16384), (16385, 16),
                                   (17, 17), (200, 3, 5), (40, 16, 1100), (150, 700, 2), (1, 16500)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize(shape, dtype):
    _check(_data(shape).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_steps(dtype, steps):
    _check(_data((200, 264), 1).to(dtype), steps)


@pytest.mark.parametrize("floor", [1e-1, 1e-2])
def test_a_few_strong_directions_over_weak_noise(floor):
    """What the two planes are for: weak directions are amplified by a^5 = 485, and so are roundings.  bf16 results stay
    within 1e-2 of the definition (their own rounding: 1.7e-3).  fp32 results are held to what the formula loses in fp32 with
    library products, where a product's terms are rounded by 2^-24: here they are cut by 2^-23 and operands keep 2^-22, four
    times that."""
    a, b, c = COEFS
    for dtype in (torch.float32, torch.bfloat16):
        x = _data((512, 768), 2, floor=floor).to(dtype)
        got = _check(x).double()
        ref, _ = _reference(x, 5, dtype)
        off = ((got - ref).norm() / ref.norm()).item()
        if dtype == torch.bfloat16:
            assert off < 1e-2
            continue
        X = x / (x.norm() + 1e-7)
        for _ in range(5):
            A = X @ X.T
            X = a * X + (b * A + c * A @ A) @ X
        assert off <= 4 * ((X.double() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("shape", [(256, 256), (100, 700), (700, 100)])
def test_singular_values(shape):
    """Singular values from 0.02 of the norm on come to [0.6, 1.3]."""
    u, _, v = torch.linalg.svd(torch.randn(*shape, device="cuda"), full_matrices=False)
    s = torch.linspace(0.3, 1.0, min(shape), device="cuda")
    got = torch.linalg.svdvals(_check(((u * s) @ v).contiguous()).double())
    assert 0.6 < got.min().item() and got.max().item() < 1.3


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e30])
def test_magnitudes(scale):
    """A gradient's size does not matter as long as it is above the epsilon; squares are summed in fp64."""
    x = _data((90, 130), 3)
    _check(x * scale)


def test_zero_matrix_and_zeros_in_a_batch():
    from parameter_server_b200.ops import orthogonal

    assert not orthogonal.orthogonalize(torch.zeros(70, 50, device="cuda")).any()
    x = _data((3, 70, 50), 4)
    x[1] = 0
    got = _check(x)
    assert not got[1].any() and bool(torch.isfinite(got).all())


def test_nan_stays_in_its_matrix():
    from parameter_server_b200.ops import orthogonal

    x = _data((3, 70, 50), 5)
    want = orthogonal.orthogonalize(x)
    x[1, 3, 4] = float("nan")
    got = orthogonal.orthogonalize(x)
    assert bool(torch.isnan(got[1]).any()) and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_empty():
    from parameter_server_b200.ops import orthogonal

    for shape in ((0, 5), (5, 0), (0, 4, 4)):
        assert orthogonal.orthogonalize(torch.empty(*shape, device="cuda")).shape == shape


@pytest.mark.parametrize("shape", [(64, 64), (33, 1000), (1000, 33), (4, 65, 130), (1030, 1100)])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update(shape, gtype, nesterov):
    from parameter_server_b200.ops import dense, orthogonal

    w, m = torch.randn(*shape, device="cuda") / shape[-1] ** 0.5, _data(shape, 6) * 1e-2
    g = (_data(shape, 7) * 1e-2).to(gtype)
    w0, m0, v = w.double(), m.double(), (w._version, m._version)
    orthogonal.orthogonal_update(w, g, m, 0.02, momentum=0.9, nesterov=nesterov)
    torch.cuda.synchronize()
    dense.check_status(w.device)
    assert w._version > v[0] and m._version > v[1]
    m1 = 0.9 * m0 + g.double()
    # 0.9 as fp32 (2^-24), the product and the sum rounded
    assert bool(((m.double() - m1).abs() <= 2.0 ** -24 * (3 * 0.9 * m0.abs() + m1.abs()) * 1.01 + 1e-40).all())
    u = g.double() + 0.9 * m1 if nesterov else m1
    step = 0.02 * max(1.0, shape[-2] / shape[-1]) ** 0.5
    for w1, wz, uz in zip(w, w0, u) if w.dim() == 3 else [(w, w0, u)]:
        ref, err = _reference(uz, 5, torch.float32)
        # the direction is rounded as the momentum is: 4 half steps of it, carried through five steps
        err = err + 4.3 ** 5 * 4 * 2.0 ** -24
        want = wz - step * ref
        tol = step * err + 2 * 2.0 ** -24 * want.norm() + 2.0 ** -22 * step * ref.norm()
        assert (w1.double() - want).norm().item() <= tol.item()


@pytest.mark.parametrize("shape", [(2, 264, 520), (130, 136), (203, 301), (300, 8000), (64, 64), (96, 700), (5, 72)])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offsets", [(0, 0, 0), (1, 2, 3), (0, 4, 0), (4, 0, 1), (2, 8, 4)])
def test_update_and_matrix_at_any_address(shape, gtype, offsets):
    """Tensors that start inside others, so that wide loads apply to all, some or none: the same result but for the order of the
    norm's fp64 sum, a last bit of its quotient in fp32 (2^-24), which five steps multiply by at most 4.3 each."""
    from parameter_server_b200.ops import orthogonal

    numel = torch.Size(shape).numel()
    data = [torch.randn(*shape, device="cuda"), (_data(shape, 8) * 1e-2).to(gtype), _data(shape, 9) * 1e-2]
    bound = 4.3 ** 5 * 2.0 ** -23 + (2 * HALF_STEP[gtype] * numel ** 0.5 if gtype != torch.float32 else 0)
    results = []
    for at in ((0, 0, 0), offsets):
        w, g, m = (torch.zeros(numel + 16, dtype=t.dtype, device="cuda")[o: o + numel].view(shape).copy_(t) for t, o in zip(data, at))
        orthogonal.orthogonal_update(w, g, m, 0.5, momentum=0.9)
        results.append((w, m, orthogonal.orthogonalize(g)))
    (w0, m0, x0), (w1, m1, x1) = results
    assert torch.equal(m0, m1)
    step = 0.5 * max(1.0, shape[-2] / shape[-1]) ** 0.5
    batch = shape[0] if len(shape) == 3 else 1
    assert (w1.double() - w0.double()).norm().item() <= step * 4.3 ** 5 * 2.0 ** -23 * batch + 2.0 ** -23 * w0.double().norm().item()
    assert (x1.double() - x0.double()).norm().item() <= bound * batch


def test_update_captured_and_on_another_stream():
    from parameter_server_b200.ops import orthogonal

    def state():
        g = torch.Generator(device="cuda").manual_seed(1)
        return [torch.randn(96, 200, generator=g, device="cuda") for _ in range(3)]

    w, g, m = state()
    for _ in range(3):
        orthogonal.orthogonal_update(w, g, m, 0.02)
    w2, g2, m2 = state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        orthogonal.orthogonal_update(w2, g2, m2, 0.02)
    w2.copy_(state()[0])
    m2.copy_(state()[2])
    w3, g3, m3 = state()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(stream):
            orthogonal.orthogonal_update(w3, g3, m3, 0.02)
    torch.cuda.synchronize()
    for a, b, c in ((w, w2, w3), (m, m2, m3)):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("shape", [(48, 48), (80, 80), (112, 100), (40, 1000), (700, 75), (110, 1500), (4, 80, 300)])
def test_short_sides_that_end_inside_a_warp(shape):
    """Rounded up to 16 they are 48, 80 or 112: of the warp that holds the last 16 rows, half has none."""
    _check(_data(shape, 10))


@pytest.mark.parametrize("shape", [(1, 7), (5, 72), (700, 9), (16, 5000), (3, 40, 12), (16385, 16), (200, 2, 3)])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update_of_thin_matrices(shape, gtype, nesterov):
    """A short side of at most 16, either way round, batched, on one CTA and on several, against the definition."""
    test_update(shape, gtype, nesterov)


@pytest.mark.parametrize("shape", [(2, 264, 520), (130, 136), (203, 301), (300, 8000), (64, 64), (96, 700), (5, 72), (3, 40, 12)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
def test_matrix_at_any_address(shape, dtype, offset):
    """Wide and single loads of all types, each against the definition: a bound relative to the result, matrix by matrix."""
    numel = torch.Size(shape).numel()
    x = (_data(shape, 11) * 1e-2).to(dtype)
    _check(torch.zeros(numel + 16, dtype=dtype, device="cuda")[offset: offset + numel].view(shape).copy_(x))


@pytest.mark.parametrize("shape", [(20, 2_000_000), (1_500_000, 24)])
def test_millions_of_columns(shape):
    """bf16, whose last step sums one plane of up to 32,768 columns at a time: its own rounding (1.7e-3 on average) and that of the
    operands of the last step (1.2e-3) are what is left."""
    x = _data(shape, 12).bfloat16()
    got = _check(x)
    ref, _ = _reference(x, 5, torch.bfloat16)
    assert ((got.double() - ref).norm() / ref.norm()).item() < 4e-3
