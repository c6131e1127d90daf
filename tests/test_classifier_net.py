"""Nets with a softmax loss over many classes and orthogonalised updates: what the layers hand to the operators, on the CPU with
PyTorch restatements, and whole training steps on the GPU."""
import pytest
import torch

from parameter_server_b200 import config as cfg
from parameter_server_b200.models import nn
from parameter_server_b200.ops import dense, orthogonal, softmax
from parameter_server_b200.parallel.peer import PeerGroup

NET = '''
neural_network {
  train { name: "train"
    layer { type: DATA name: "data" out: "x" out: "y" minibatch_size: %(batch)d %(data)s }
    layer { type: FULLY_CONNECTED name: "fc1" in: "x" out: "h" size: %(hidden)d activation { type: RELU } }
    layer { type: FULLY_CONNECTED name: "fc2" in: "h" out: "g" size: 24 activation { type: SCALED_TANH } }
    layer { type: SOFTMAX_LOSS name: "loss" in: "g" in: "y" size: %(classes)d lr_scale: 0.5 }
  }
  test { name: "test"
    layer { type: DATA name: "tdata" out: "x" out: "y" %(data)s }
    layer { type: FULLY_CONNECTED name: "fc1" in: "x" out: "h" size: %(hidden)d activation { type: RELU } }
    layer { type: FULLY_CONNECTED name: "fc2" in: "h" out: "g" size: 24 activation { type: SCALED_TANH } }
    layer { type: SOFTMAX_LOSS name: "loss" in: "g" in: "y" size: %(classes)d }
  }
  solver { type: SGD update: %(update)s lr { alpha: 0.1 beta: 1 } max_iteration: %(iters)d display: 50 validation: %(valid)d momentum: 0.9 }
}
'''


def _conf(**k):
    return cfg.parse_app_config(NET % dict(dict(batch=0, hidden=32, classes=10, update="ORTHOGONAL", iters=3, valid=0, data=""), **k)).neural_network


def _data(n, d=12, classes=10, seed=0):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn(n, d, generator=g)
    y = (X @ torch.randn(d, classes, generator=torch.Generator().manual_seed(5))).argmax(1).float()
    y[::9] = -1
    return X, y


def _reference(X, y, ws):
    """Loss sum and gradients in fp64 of the net above."""
    ws = [w.detach().double().requires_grad_(True) for w in ws]
    h = torch.relu(X.double() @ ws[0].T)
    h = 1.7159 * torch.tanh(2.0 / 3.0 * (h @ ws[1].T))
    live = y >= 0
    loss = torch.nn.functional.cross_entropy((h @ ws[2].T)[live], y[live].long(), reduction="sum")
    loss.backward()
    return loss.item(), [w.grad for w in ws]


@pytest.fixture
def cpu_ops(monkeypatch):
    """The operators in PyTorch, with a record of the calls."""
    calls = []

    def softmax_loss(x, w, y, coef=None, want_grad=True, want_gx=True):
        assert y.dtype == torch.int64 and y.dim() == 1
        calls.append(("softmax_loss", want_grad, want_gx))
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        losses = torch.nn.functional.cross_entropy(xr @ wr.T, y, reduction="none", ignore_index=-1)
        losses.sum().backward()
        return losses.detach(), xr.grad if want_grad and want_gx else None, wr.grad if want_grad else None

    def orthogonal_update(w, g, m, lr, momentum=0.95, nesterov=True, steps=5):
        calls.append(("orthogonal_update", tuple(w.shape), lr, momentum))
        m.mul_(momentum).add_(g)
        w.sub_(lr * m)

    def act_backward_t(g, y, act, want_z=True):
        z = g * (y > 0) if act == "RELU" else g * (1.7159 * 2 / 3 * (1 - (y / 1.7159) ** 2))
        return (z if want_z else None), z.T.contiguous()

    def gemm_tn(a, b, act="IDENTITY", out=None, pad_k=False, out_t=None, variant=0):
        r = a @ b.T
        r = torch.relu(r) if act == "RELU" else 1.7159 * torch.tanh(2.0 / 3.0 * r) if act == "SCALED_TANH" else r
        if out_t is not None:
            out_t.copy_(r.T)
        return r

    def sgd_update(w, g, h, alpha, beta, it):
        calls.append(("sgd_update", tuple(w.shape), h is not None, alpha))

    monkeypatch.setattr(softmax, "softmax_loss", softmax_loss)
    monkeypatch.setattr(orthogonal, "orthogonal_update", orthogonal_update)
    for f in (act_backward_t, gemm_tn, sgd_update):
        monkeypatch.setattr(dense, f.__name__, f)
    monkeypatch.setattr(dense, "transpose", lambda x: x.T.clone(memory_format=torch.contiguous_format))
    monkeypatch.setattr(dense, "check_status", lambda dev: None)
    monkeypatch.setattr(dense, "col_normalize", lambda x: None)
    return calls


def _solver(device, data, **k):
    sol = nn.SGDSolver(_conf(**k), PeerGroup.single(device))
    sol.train.layer("data").set_data(*data, normalize=False)
    sol.test.layer("tdata").set_data(*data, normalize=False)
    return sol


def test_gradients_and_update_on_the_cpu(cpu_ops):
    data = _data(60)
    sol = _solver(torch.device("cpu"), data)
    sol.train.forward()
    sol.train.backward()
    layers = [sol.train.layer(n) for n in ("fc1", "fc2", "loss")]
    loss, grads = _reference(*data, [l.model.value for l in layers])
    assert layers[2].loss.item() == pytest.approx(loss, rel=1e-5) and layers[2].n == 60
    for l, g in zip(layers, grads):
        torch.testing.assert_close(l.model.gradient.double(), g, rtol=1e-4, atol=1e-5)
    assert ("softmax_loss", True, True) in cpu_ops
    cpu_ops.clear()
    mean = sol.step(3)
    assert mean == pytest.approx(loss / 60, rel=1e-5)
    assert cpu_ops[1:] == [("orthogonal_update", (32, 12), 0.1 / 3, pytest.approx(0.9)), ("orthogonal_update", (24, 32), 0.1 / 3, pytest.approx(0.9)),
                           ("sgd_update", (10, 24), True, 0.1 * 0.5)]
    cpu_ops.clear()
    sol.evaluate()
    assert cpu_ops == [("softmax_loss", False, True)] and sol.test.layer("loss").model is layers[2].model and sol.test_loss() > 0


def test_rows_that_are_data_get_no_gradient(cpu_ops):
    conf = cfg.parse_app_config('''neural_network { train { name: "t"
      layer { type: DATA name: "data" out: "x" out: "y" minibatch_size: 0 }
      layer { type: SOFTMAX_LOSS name: "loss" in: "x" in: "y" size: 10 } }
      solver { type: SGD update: ADAGRAD lr { alpha: 0.1 beta: 1 } max_iteration: 1 } }''').neural_network
    sol = nn.SGDSolver(conf, PeerGroup.single(torch.device("cpu")))
    sol.train.layer("data").set_data(*_data(40), normalize=False)
    sol.step(0)
    assert cpu_ops == [("softmax_loss", True, False), ("sgd_update", (10, 12), True, 0.1)]


def test_number_of_classes_is_asked_for():
    with pytest.raises(ValueError, match="classes"):
        nn.SGDSolver(_conf(classes=0), PeerGroup.single(torch.device("cpu")))
    with pytest.raises(ValueError, match="classes"):                # labels are float32
        nn.SGDSolver(_conf(classes=(1 << 24) + 1), PeerGroup.single(torch.device("cpu")))


def _write_libsvm(path, X, y):
    path.write_text("\n".join(f"{int(c)} " + " ".join(f"{j + 1}:{v:.6f}" for j, v in enumerate(r)) for r, c in zip(X.tolist(), y.tolist())) + "\n")


def test_class_numbers_of_files(tmp_path, cpu_ops):
    """Labels of a data file are class numbers where the net has a softmax loss, and signs where it has not."""
    X, y = _data(30, classes=5)
    y = y.clamp(min=0)
    _write_libsvm(tmp_path / "part", X, y)
    data = f'data {{ format: TEXT text: LIBSVM file: "{tmp_path}/part" }}'
    sol = nn.SGDSolver(_conf(data=data), PeerGroup.single(torch.device("cpu")))
    assert torch.equal(sol.train.layer("data").y, y)


@pytest.mark.gpu
@pytest.mark.parametrize("n,hidden,classes", [(512, 64, 10), (300, 40, 3001), (64, 7, 1)])
def test_gradients_match_the_formula(n, hidden, classes):
    """Dense layers multiply TF32 operands (11 bits, 2^-11 a factor): hidden values are off by 2^-10 of their terms, and gradients
    through two layers and their products by a few times that."""
    data = _data(n, classes=classes)
    sol = _solver(torch.device("cuda", 0), data, hidden=hidden, classes=classes)
    sol.train.forward()
    sol.train.backward()
    layers = [sol.train.layer(n) for n in ("fc1", "fc2", "loss")]
    loss, grads = _reference(data[0].cuda(), data[1].cuda(), [l.model.value for l in layers])
    assert layers[2].loss.item() == pytest.approx(loss, rel=2e-3, abs=1e-3)
    for l, g in zip(layers, grads):
        assert (l.model.gradient.double() - g).norm().item() <= 2e-2 * g.norm().item() + 1e-6


@pytest.mark.gpu
def test_a_training_run_with_both(tmp_path):
    """Minibatches, softmax loss and orthogonalised updates together, as a job runs them: every step is the operators' own
    step on the gradients of that minibatch, and the losses are recorded."""
    data = _data(400, classes=50)
    sol = _solver(torch.device("cuda", 0), data, batch=64, classes=50, iters=4, valid=2)
    hist = sol.run(verbose=False)
    assert len(hist) == 4 and all(h["loss"] > 0 for h in hist) and [("test_loss" in h) for h in hist] == [False, True, False, True]
    layers = [sol.train.layer(n) for n in ("fc1", "fc2", "loss")]
    before = [l.model.value.clone() for l in layers]
    m = [l.model.momentum.clone() for l in layers[:2]]
    h = layers[2].model.hession.clone()
    sol.step(4)
    for l, w, mm in zip(layers[:2], before, m):
        orthogonal.orthogonal_update(w, l.model.gradient, mm, 0.1 / (1 + 5 ** 0.5), momentum=sol.momentum)
        assert torch.equal(l.model.value, w) and torch.equal(l.model.momentum, mm)
    dense.sgd_update(before[2], layers[2].model.gradient, h, 0.05, 1.0, 5)
    assert torch.equal(layers[2].model.value, before[2])


@pytest.mark.gpu
def test_a_job_from_files(tmp_path):
    X, y = _data(200, classes=7)
    y = y.clamp(min=0)
    _write_libsvm(tmp_path / "part", X, y)
    data = f'data {{ format: TEXT text: LIBSVM file: "{tmp_path}/part" }}'
    conf = cfg.parse_app_config(NET % dict(batch=64, hidden=32, classes=7, update="ORTHOGONAL", iters=3, valid=3, data=data))
    out = nn.run_nn_job(conf, None, PeerGroup.single(torch.device("cuda", 0)))
    assert len(out["history"]) == 3 and out["history"][-1]["test_loss"] > 0


@pytest.mark.parametrize("bad", [10.0, 2.5, -2.0, float("nan"), float("inf")])
def test_labels_that_are_no_classes_are_refused(bad):
    """They would count as rows without a class, and the job would learn of it at its end only."""
    X, y = _data(30)
    sol = nn.SGDSolver(_conf(), PeerGroup.single(torch.device("cpu")))
    sol.train.layer("data").set_data(X, y, normalize=False)
    wrong = y.clone()
    wrong[4] = bad
    with pytest.raises(ValueError, match="class numbers"):
        sol.train.layer("data").set_data(X, wrong, normalize=False)
    with pytest.raises(ValueError, match="class numbers"):
        sol.train.layer("data").set_sparse_data(torch.arange(31), torch.zeros(30), None, wrong, 5)
    assert torch.equal(sol.train.layer("data").y, y)
    sol.train.layer("data").set_data(X, y.long(), normalize=False)


def test_files_of_signs_are_pointed_out(tmp_path, cpu_ops):
    X, y = _data(30, classes=2)
    _write_libsvm(tmp_path / "part", X, torch.where(y > 0, 1.0, -1.0))
    with pytest.warns(UserWarning, match="numbered from 0"):
        nn.SGDSolver(_conf(data=f'data {{ format: TEXT text: LIBSVM file: "{tmp_path}/part" }}'), PeerGroup.single(torch.device("cpu")))
