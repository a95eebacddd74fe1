"""``optimizer="muon"`` of VNNTrainer and VNNTrainStep: whose momentum it is, sub-ROIs, ranks and
the update's own waits."""
import numpy as np
import pytest
import torch

import neurocell_b200 as nc
from neurocell_b200 import ops
from oracle import vnn_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _params(seed):
    rng = np.random.default_rng(seed)
    cell = torch.tensor(rng.normal(0, 0.1, (3, 62, 62)).astype(np.float32), device=DEV)
    filt = torch.tensor((rng.normal(0, 1, (16, 1, 23, 13)) / np.sqrt(299)).astype(np.float32), device=DEV)
    return nc.VNNParams(cell, filt)


def _batch(B, seed):
    x, y, _ = O.alu_batch(np.random.default_rng(seed), B, noise=0.0)
    return torch.tensor(x, device=DEV), torch.tensor(y, device=DEV)


def _trainer(**kw):
    model = nc.VonNeumannNetwork(nc.ChipTopology2D.alu_chip())
    return nc.VNNTrainer(model.apply, lr=0.02, optimizer="muon", **kw)


def _run(tr, p, x, y, steps=2):
    for _ in range(steps):
        p, _ = tr.train_step(p, x, y)
    return p


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_trainer_starts_over_on_other_parameters():
    x, y = _batch(16, 1)
    want = _run(_trainer(), _params(3), x, y)
    tr = _trainer()
    a = _run(tr, _params(2), x, y)
    assert _same(_run(tr, _params(3), x, y), want)
    # tensors that were freed may come back at the same address
    del a
    for _ in range(3):
        assert _same(_run(tr, _params(3), x, y), want)
    # another shape
    topo = nc.ChipTopology2D.alu_chip(kernel_size=(11, 9), directions=4)
    other = nc.init_vnn_params(5, topo, device=DEV)
    tr.apply_fn = nc.VonNeumannNetwork(topo).apply
    _run(tr, other, x, y, steps=1)


def test_momentum_goes_on_through_views_and_may_be_stored():
    x, y = _batch(16, 1)
    tr, p = _trainer(), _params(3)
    want = _run(tr, p, x, y, steps=4)
    # the same storage by other tensor objects
    tr, p = _trainer(), _params(3)
    for _ in range(4):
        _run(tr, nc.VNNParams(*(t.detach().view(t.shape) for t in p)), x, y, steps=1)
    assert _same(p, want)
    # stored and given to another trainer, on copies of the parameters
    tr, p = _trainer(), _params(3)
    _run(tr, p, x, y)
    stored = nc.VNNParams(*(t.clone() for t in tr.momentum))
    tr, q = _trainer(), nc.VNNParams(*(t.clone() for t in p))
    tr.momentum = stored
    assert _same(_run(tr, q, x, y), want)
    # new values in the same tensors
    for t, v in zip(q, _params(3)):
        t.copy_(v)
    tr.momentum = None
    assert _same(_run(tr, q, x, y, steps=4), want)
