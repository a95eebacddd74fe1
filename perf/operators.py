"""Measured cases of the readout loss and the orthogonalised update.

Three operators of ``neurocell_b200``:

* ``ops.linear_softmax_ce_loss`` / ``ops.linear_softmax_ce_value_and_grad``: softmax
  cross-entropy of a linear readout (features of the output ports times a class matrix)
  over a large vocabulary, the value alone or with every gradient;
* ``ops.orthogonalize``: Newton-Schulz orthogonalisation of a matrix or a batch of them;
* ``ops.muon_``: momentum, orthogonalisation and the parameter update in place.

``own`` selects the framework's calls; otherwise ``run`` is their plain form.
"""
import math
import os
import sys

import torch

own = False

IGNORE = -100
COEFFS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _ops():
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(here, "neurocell-v2_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from neurocell_b200 import ops
    return ops


def _ce(kind, rows, dim, classes, dtype, bias, ignored):
    return {"op": kind, "rows": rows, "dim": dim, "classes": classes, "dtype": dtype, "bias": bias,
            "ignored": ignored}


def _mat(kind, batch, rows, cols, dtype):
    return {"op": kind, "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # the ALU chip's 8 output ports read as one of 256 byte values, its batch of 128
        dict(_ce("ce_train", 128, 8, 256, "float32", True, 0.0), name="ce_train_alu_bytes"),
        # the 128 output ports of the largest chip, odd sizes, a padded batch
        dict(_ce("ce_train", 333, 128, 10007, "float32", True, 0.1), name="ce_train_ports_odd"),
        # a few samples against a large vocabulary: one gradient step of a fine-tuning loop
        dict(_ce("ce_train", 8, 1024, 50000, "float32", True, 0.0), name="ce_train_few_rows"),
        # an ordinary fp32 training batch
        dict(_ce("ce_train", 2048, 512, 32768, "float32", False, 0.0), name="ce_train_fp32"),
        # the largest: a token batch in bf16
        dict(_ce("ce_train", 4096, 1024, 50000, "bfloat16", True, 0.05), name="ce_train_bf16_large"),
        # scoring one sample
        dict(_ce("ce_score", 1, 1024, 50000, "float32", True, 0.0), name="ce_score_one"),
        # scoring an evaluation set, ragged
        dict(_ce("ce_score", 8191, 520, 32001, "bfloat16", True, 0.2), name="ce_score_bf16_ragged"),
        # the three cell grids of the ALU chip
        dict(_mat("orthogonalize", 3, 62, 62, "float32"), name="orthogonalize_alu_grids"),
        # the filter bank of the largest chip: 32 directions of 63 x 63 taps
        dict(_mat("orthogonalize", 1, 32, 3969, "float32"), name="orthogonalize_filters"),
        # a tall odd-sized bf16 matrix, such as a readout's
        dict(_mat("orthogonalize", 1, 2001, 513, "bfloat16"), name="orthogonalize_tall_bf16"),
        # update of the 256 x 256 chip's three grids
        dict(_mat("muon", 3, 256, 256, "float32"), name="muon_256_grids"),
        # update of the 1024 x 1024 chip's three grids
        dict(_mat("muon", 3, 1024, 1024, "float32"), name="muon_1024_grids"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("ce_train", "ce_train", "ce_score", "orthogonalize", "muon"))
    dtype = rng.choice(("float32", "float32", "bfloat16"))
    if kind.startswith("ce"):
        while True:
            rows, dim, classes = _log(rng, 1, 8192), _log(rng, 8, 1024), _log(rng, 10, 65536)
            if rows * dim * classes <= (2e11 if dtype == "bfloat16" else 4e10) and rows * classes <= 2.6e8:
                return _ce(kind, rows, dim, classes, dtype, rng.random() < 0.7,
                           rng.choice((0.0, 0.0, 0.1, 0.5)))
    while True:
        rows, cols, batch = _log(rng, 8, 1024), _log(rng, 8, 4096), rng.choice((1, 1, 2, 3))
        if rng.random() < 0.5:
            rows, cols = cols, rows
        if batch * min(rows, cols) ** 2 * max(rows, cols) <= 3 * 1024 ** 3:
            return _mat(kind, batch, rows, cols, dtype if kind == "orthogonalize" else "float32")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"].startswith("ce"):
        n, d, v = case["rows"], case["dim"], case["classes"]
        s["features"] = normal(n, d).to(dt)
        s["weight"] = (normal(v, d) * (2.0 / math.sqrt(d))).to(dt)
        s["bias_t"] = (0.5 * normal(v)).to(dt) if case["bias"] else None
        labels = torch.randint(0, v, (n,), generator=g, device="cuda")
        drop = torch.rand(n, generator=g, device="cuda") < case["ignored"]
        s["labels"] = torch.where(drop, torch.full_like(labels, IGNORE), labels).to(torch.int32)
        return s
    b, r, c = case["batch"], case["rows"], case["cols"]
    k = min(8, r, c)
    # a gradient: a few strong directions over noise
    s["grad"] = (normal(b, r, c) + normal(b, r, k) @ normal(b, k, c)).mul_(1e-3).to(dt)
    if case["op"] == "muon":
        s["param"] = 0.1 * normal(b, r, c)
        s["momentum"] = 1e-3 * normal(b, r, c)
    return s


# hyper-parameters of the update cases
LR, BETA, DECAY = 0.02, 0.95, 0.01


def run(state):
    op = state["op"]
    if own:
        ops = _ops()
        if op == "ce_train":
            return ops.linear_softmax_ce_value_and_grad(state["features"], state["weight"], state["labels"],
                                                        bias=state["bias_t"], ignore_index=IGNORE)
        if op == "ce_score":
            return ops.linear_softmax_ce_loss(state["features"], state["weight"], state["labels"],
                                              bias=state["bias_t"], ignore_index=IGNORE, reduction="none")
        if op == "orthogonalize":
            return ops.orthogonalize(state["grad"], coefficients=COEFFS, eps=EPS)
        # the update runs in place; the copies keep the state for the next pass, as the plain
        # form's new tensors do
        p, m = state["param"].clone(), state["momentum"].clone()
        ops.muon_(p, state["grad"], m, LR, beta=BETA, weight_decay=DECAY, coefficients=COEFFS, eps=EPS)
        return p, m
    if op.startswith("ce"):
        return _plain_ce(state, op == "ce_train")
    if op == "orthogonalize":
        return _plain_orthogonalize(state["grad"]).to(state["grad"].dtype)
    m = BETA * state["momentum"] + state["grad"]
    o = _plain_orthogonalize(state["grad"] + BETA * m)
    scale = max(1.0, o.shape[-2] / o.shape[-1]) ** 0.5
    return state["param"] * (1.0 - LR * DECAY) - (LR * scale) * o, m


def _plain_ce(state, train):
    dt = state["features"].dtype
    f, w = state["features"].float(), state["weight"].float()
    labels = state["labels"].long()
    kept = labels != IGNORE
    at = torch.where(kept, labels, torch.zeros_like(labels))
    z = f @ w.T
    if state["bias_t"] is not None:
        z = z + state["bias_t"].float()
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    loss = torch.log(total)[:, 0] + top[:, 0] - z.gather(1, at[:, None])[:, 0]
    loss = torch.where(kept, loss, torch.zeros_like(loss))
    if not train:
        return loss
    count = kept.sum().clamp(min=1)
    p = e / total
    p.scatter_add_(1, at[:, None], torch.full_like(p[:, :1], -1.0))
    p = p * (kept / count)[:, None]
    return (loss.sum() / count, (p @ w).to(dt), (p.T @ f).to(dt),
            None if state["bias_t"] is None else p.sum(dim=0).to(dt))


def _plain_orthogonalize(x):
    # the norm in 64 bits: the iteration magnifies an error of scale about a hundred times
    norm = x.double().square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS
    x = (x.double() / norm).float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1) if tall else x
    a, b, c = COEFFS
    for _ in range(5):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("ce"):
        return _exact_ce(s, case["op"] == "ce_train")
    if case["op"] == "orthogonalize":
        return _exact_orthogonalize(s["grad"].double())
    m = BETA * s["momentum"].double() + s["grad"].double()
    o = _exact_orthogonalize(s["grad"].double() + BETA * m)
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return s["param"].double() * (1.0 - LR * DECAY) - LR * scale * o, m


def _exact_ce(s, train):
    """Row blocks of log-softmax in 64 bits."""
    w = s["weight"].double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device="cuda") if s["bias_t"] is None else s["bias_t"].double()
    labels = s["labels"].long()
    n = labels.numel()
    count = max(1, int((labels != IGNORE).sum()))
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    gf = torch.zeros(n, w.shape[1], dtype=torch.float64, device="cuda")
    gw, gb = torch.zeros_like(w), torch.zeros_like(b)
    step = max(1, (1 << 26) // w.shape[0])
    for i in range(0, n, step):
        rows = torch.nonzero(labels[i:i + step] != IGNORE)[:, 0] + i
        if rows.numel() == 0:
            continue
        f = s["features"][rows].double()
        lp = torch.log_softmax(torch.addmm(b, f, w.t()), dim=-1)
        pick = torch.arange(rows.numel(), device="cuda")
        loss[rows] = -lp[pick, labels[rows]]
        if train:
            dz = lp.exp_()
            dz[pick, labels[rows]] -= 1.0
            dz /= count
            gf[rows] = dz.mm(w)
            gw.addmm_(dz.t(), f)
            gb += dz.sum(0)
    if not train:
        return loss
    return loss.sum() / count, gf, gw, None if s["bias_t"] is None else gb


def _exact_orthogonalize(x):
    """The iteration acts on the singular values alone: U poly(sigma) V^T."""
    a, b, c = COEFFS
    u, sig, vt = torch.linalg.svd(x / (torch.linalg.matrix_norm(x)[..., None, None] + EPS), full_matrices=False)
    for _ in range(5):
        sig = a * sig + b * sig ** 3 + c * sig ** 5
    return (u * sig[..., None, :]) @ vt


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"].startswith("ce"):
        n, d, v = case["rows"], case["dim"], case["classes"]
        inputs = size * (n * d + v * d + (v if case["bias"] else 0)) + 4 * n
        if case["op"] == "ce_score":
            return {"bytes": inputs + 4 * n, "flops": 2 * n * d * v}
        return {"bytes": inputs + size * (n * d + v * d + (v if case["bias"] else 0)) + 4,
                "flops": 6 * n * d * v}
    b, r, c = case["batch"], case["rows"], case["cols"]
    short, long = min(r, c), max(r, c)
    flops = b * 5 * (4 * short * short * long + 2 * short ** 3)
    tensors = 2 if case["op"] == "orthogonalize" else 5   # muon: gradient, parameters and momentum read, two written
    return {"bytes": tensors * size * b * r * c, "flops": flops}
