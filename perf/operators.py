"""Operators of large nets that the framework offers next to its dense layers, as cases that can be timed: the softmax
cross entropy of rows over many classes with its gradients, and the orthogonalised weight update.

Kinds of cases
  loss        ``ops.softmax.softmax_loss``: rows x [rows, dim] against classes w [classes, dim], the loss of every row and,
              where ``grad`` is set, the gradients with respect to x and w.  A label of -1 is a row without a class: its
              loss and its part in the gradients are 0.  ``weighted``: every row has a coefficient.
  orthogonal  ``ops.orthogonal.orthogonalize``: five Newton-Schulz steps on one matrix or on a batch of them
  update      ``ops.orthogonal.orthogonal_update``: momentum, the same five steps, and the step of the weights
"""
import math

import torch

own = False

# odd polynomial of a Newton-Schulz step, and its number of steps (the published ones of the Muon optimiser)
COEFS, STEPS, EPS = (3.4445, -4.7750, 2.0315), 5, 1e-7
LR, MOMENTUM = 0.02, 0.95
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one example is scored against a long list of classes: a latency, bound by reading the classes
        _loss("loss_score_1_row", 1, 50_000, 1024, "bf16"),
        # the head of a small net: a minibatch of 16 rows, 100 classes, trained
        _loss("loss_16_rows_100_classes", 16, 100, 64, "fp32", grad=True),
        # an ordinary minibatch of a net in single precision, a thousand classes
        _loss("loss_256_rows_1k_classes", 256, 1000, 256, "fp32", grad=True),
        # odd sizes, rows that are weighted or have no class, single precision
        _loss("loss_1003_rows_odd", 1003, 32_003, 517, "fp32", grad=True, unlabelled=0.1, weighted=True),
        # a large minibatch is scored: the test net's loss
        _loss("loss_score_4096_rows", 4096, 131_072, 1024, "bf16"),
        # an ordinary training step in 16 bits, padded rows at the end of sequences without a class
        _loss("loss_2048_rows_50k_classes", 2048, 50_003, 1024, "bf16", grad=True, unlabelled=0.05),
        # the largest: many rows, a large vocabulary, wide rows
        _loss("loss_8192_rows_131k_classes", 8192, 131_072, 2048, "bf16", grad=True),
        # the weight matrix of the small perceptron: a latency
        _orth("update_64x64", "update", 1, 64, 64, "fp32"),
        # layers of one odd shape together, 16 bits
        _orth("orthogonal_6x1000x520", "orthogonal", 6, 1000, 520, "bf16"),
        # the wide layers of the perceptron benchmark
        _orth("update_1024x4096", "update", 1, 1024, 4096, "fp32"),
        # a square matrix in 16 bits
        _orth("orthogonal_4096x4096", "orthogonal", 1, 4096, 4096, "bf16"),
        # the largest: a wide projection with its weights and momentum in single precision
        _orth("update_4096x16384", "update", 1, 4096, 16_384, "fp32"),
    ]


def _loss(name, rows, classes, dim, dtype, grad=False, unlabelled=0.0, weighted=False):
    return {"name": name, "kind": "loss", "rows": rows, "classes": classes, "dim": dim, "dtype": dtype, "grad": grad,
            "unlabelled": unlabelled, "weighted": weighted}


def _orth(name, kind, batch, m, n, dtype):
    return {"name": name, "kind": kind, "batch": batch, "m": m, "n": n, "dtype": dtype}


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        if rng.random() < 0.55:
            c = _loss("", log(1, 8192), log(2, 131_072), log(8, 2048), rng.choice(["fp32", "bf16", "bf16", "fp16"]), rng.random() < 0.7,
                      rng.choice([0.0, 0.0, 0.05, 0.5]), rng.random() < 0.4)
            if rng.random() < 0.4:
                c["dim"] = -(-c["dim"] // 8) * 8
        else:
            kind = rng.choice(["update", "orthogonal"])
            c = _orth("", kind, rng.choice([1, 1, 1, 2, 3, 8]), log(1, 4096), log(1, 8192),
                      "fp32" if kind == "update" else rng.choice(["fp32", "bf16", "fp16"]))
            if rng.random() < 0.3:
                c["m"], c["n"] = c["n"], c["m"]
        del c["name"]
        w = work(c)
        # at most the largest listed ones' work, single precision counted three times for its cost; matrices of a batch fit
        if w["flops"] * (3 if c["dtype"] == "fp32" else 1) <= 1.3e13 and w["bytes"] <= 4e9:
            return c


def labelled(case):
    return case["rows"] - int(case["unlabelled"] * case["rows"])


def work(case):
    if case["kind"] == "loss":
        n, v, d, size = labelled(case), case["classes"], case["dim"], SIZE[case["dtype"]]
        grad = case["grad"]
        return {"bytes": (n + v) * d * size + case["rows"] * (12 + 4 * case["weighted"]) + ((case["rows"] + v) * d * size if grad else 0),
                "flops": 2 * n * v * d * (3 if grad else 1)}
    lo, hi = min(case["m"], case["n"]), max(case["m"], case["n"])
    mn, size = case["batch"] * lo * hi, SIZE[case["dtype"]]
    # a step: x xᵀ and its square are symmetric, half of each is enough; the third product is a full one
    flops = case["batch"] * STEPS * (lo * lo * hi + lo ** 3 + 2 * lo * lo * hi)
    return {"bytes": mn * (2 * size if case["kind"] == "orthogonal" else 5 * size), "flops": flops}


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dt = TYPES[case["dtype"]]
    if case["kind"] == "loss":
        n, v, d = case["rows"], case["classes"], case["dim"]
        # scores have a deviation of about 2: a net that has learned something
        x, w = normal(n, d).to(dt), (normal(v, d) * (2.0 / math.sqrt(d))).to(dt)
        # popular classes come first, as a frequency-sorted vocabulary has them
        y = ((v + 1.0) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64) - 1.0).long().clamp_(0, v - 1)
        gone = n - labelled(case)
        if gone:
            y[torch.randperm(n, generator=g, device="cuda")[:gone]] = -1
        coef = torch.rand(n, generator=g, device="cuda") + 0.5 if case["weighted"] else None
        return {"case": dict(case), "x": x, "w": w, "y": y, "coef": coef}
    b, m, n = case["batch"], case["m"], case["n"]
    shape = (m, n) if b == 1 else (b, m, n)
    # gradients of a minibatch: a few strong directions over a floor of noise
    k = min(m, n, 16)
    x = normal(*shape) + 0.5 * (normal(*shape[:-1], k) @ normal(*shape[:-2], k, n))
    if case["kind"] == "orthogonal":
        return {"case": dict(case), "x": (x * 1e-3).to(dt)}
    return {"case": dict(case), "w": normal(*shape) / math.sqrt(n), "g": x * 1e-3, "m": normal(*shape) * 5e-3}


# ------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if c["kind"] == "loss":
        if own:
            from parameter_server_b200.ops import softmax

            r = softmax.softmax_loss(state["x"], state["w"], state["y"], coef=state["coef"], want_grad=c["grad"])
        else:
            r = _plain_loss(state["x"], state["w"], state["y"], state["coef"], c["grad"])
        return {"loss": r[0], "gx": r[1], "gw": r[2]} if c["grad"] else {"loss": r[0]}
    if c["kind"] == "orthogonal":
        if own:
            from parameter_server_b200.ops import orthogonal

            return orthogonal.orthogonalize(state["x"])
        return _plain_orthogonal(state["x"].float()).to(state["x"].dtype)
    if own:
        from parameter_server_b200.ops import orthogonal

        orthogonal.orthogonal_update(state["w"], state["g"], state["m"], LR, momentum=MOMENTUM)
    else:
        _plain_update(state["w"], state["g"], state["m"])
    return {"w": state["w"], "m": state["m"]}


def _plain_loss(x, w, y, coef, grad):
    """Loss of row i: log Σ_j exp(x_i·w_j) − x_i·w_y;  its gradients through softmax minus the label's indicator."""
    live = y >= 0
    xf, wf = torch.where(live[:, None], x, torch.zeros_like(x)).float(), w.float()
    scores = xf @ wf.T
    at = torch.where(live, y, torch.zeros_like(y))[:, None]
    top = scores.max(dim=1, keepdim=True).values
    target = scores.gather(1, at)
    p = scores.sub_(top).exp_()
    total = p.sum(dim=1, keepdim=True)
    zero = torch.zeros((), device=x.device)
    c = live.float() if coef is None else torch.where(live, coef, zero)
    loss = torch.where(live, (total.log() + top - target)[:, 0], zero) * c
    if not grad:
        return loss, None, None
    p.div_(total)
    p.scatter_add_(1, at, torch.full_like(target, -1.0))
    p.mul_(c[:, None])
    return loss, (p @ wf).to(x.dtype), (p.T @ xf).to(w.dtype)


def _plain_orthogonal(x):
    a, b, c = COEFS
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(STEPS):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def _plain_update(w, g, m):
    m.mul_(MOMENTUM).add_(g)
    o = _plain_orthogonal(g + MOMENTUM * m)
    w.sub_(o, alpha=LR * math.sqrt(max(1.0, w.shape[-2] / w.shape[-1])))


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "loss":
        return _exact_loss(s, case)
    if case["kind"] == "orthogonal":
        return _exact_orthogonal(s["x"].double())
    w, g, m = s["w"].double(), s["g"].double(), s["m"].double()
    m = MOMENTUM * m + g
    o = _exact_orthogonal(MOMENTUM * m + g)
    return {"w": w - LR * max(1.0, case["m"] / case["n"]) ** 0.5 * o, "m": m}


def _exact_loss(s, case):
    n = case["rows"]
    w = s["w"].double()
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    gx = torch.zeros(n, case["dim"], dtype=torch.float64, device="cuda")
    gw = torch.zeros_like(w)
    rows = torch.nonzero(s["y"] >= 0)[:, 0]
    for part in rows.split(1024):
        x, y = s["x"][part].double(), s["y"][part]
        k = torch.ones(len(part), dtype=torch.float64, device="cuda") if s["coef"] is None else s["coef"][part].double()
        z = torch.mm(x, w.t())
        lse = torch.logsumexp(z, dim=1)
        loss[part] = k * (lse - z[torch.arange(len(part), device="cuda"), y])
        if case["grad"]:
            d = torch.exp(z - lse[:, None])
            d[torch.arange(len(part), device="cuda"), y] -= 1.0
            d *= k[:, None]
            gx[part] = torch.mm(d, w)
            gw += torch.mm(d.t(), x)
    return {"loss": loss, "gx": gx, "gw": gw} if case["grad"] else {"loss": loss}


def _exact_orthogonal(x):
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + EPS)
    a, b, c = COEFS
    eye = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device="cuda")
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            s = torch.matmul(x, x.mT)
            x = torch.matmul(a * eye + b * s + c * torch.matmul(s, s), x)
        else:
            s = torch.matmul(x.mT, x)
            x = torch.matmul(x, a * eye + b * s + c * torch.matmul(s, s))
    return x
