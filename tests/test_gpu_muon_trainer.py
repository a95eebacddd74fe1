"""``optimizer="muon"`` of VNNTrainer and VNNTrainStep: whose momentum it is, sub-ROIs, ranks and
the update's own waits."""
import dataclasses

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


@pytest.mark.parametrize("annealed", [False, True])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_a_sub_roi_keeps_the_cells_outside(decay, annealed):
    """A step on all cells, then steps on a sub-ROI: the cells outside the window and their
    momentum keep their bits; inside, the update of the window as matrices of its own, as
    VNNTrainStep takes it."""
    topo = nc.ChipTopology2D.alu_chip()
    spec = nc.compute_adaptive_spatial_mask(nc.init_vnn_params(701, topo, device=DEV), topo)
    assert not spec.is_full_roi
    x, y = _batch(32, 4)
    codd = dict(codd_mode="annealed", state_temperature=0.7) if annealed else {}
    tr, p = _trainer(weight_decay=decay), _params(6)
    p, _ = tr.train_step(p, x, y, **codd)
    st = nc.VNNTrainStep(topo, p, 32, lr=0.02, in_shapes=((8, 1),) * 3, spatial_mask=spec, optimizer="muon",
                         weight_decay=decay, **codd)
    r0, r1, c0, c1 = st.window
    assert r1 - r0 != c1 - c0      # the step's factor sqrt(rows / cols) is the window's own
    inside = torch.zeros(62, 62, dtype=torch.bool, device=DEV)
    inside[r0:r1, c0:c1] = True
    st.momentum[: st.n_cell].copy_(tr.momentum.cell_params[:, r0:r1, c0:c1].reshape(-1))
    st.momentum[st.n_cell:].copy_(tr.momentum.greens_filters.reshape(-1))
    before, mom = p.cell_params.clone(), tr.momentum.cell_params.clone()
    for _ in range(2):
        _, grads = tr.value_and_grad(p, x, y, spatial_mask=spec, **codd)
        assert not grads.cell_params[:, ~inside].any()
        want, m = (t[:, r0:r1, c0:c1].contiguous() for t in (p.cell_params, tr.momentum.cell_params))
        ops.muon_(want, grads.cell_params[:, r0:r1, c0:c1].contiguous(), m, 0.02, weight_decay=decay)
        if annealed:
            tr.train_step_annealed(p, x, y, state_temperature=0.7, mask_spec=spec)
        else:
            tr.train_step_adaptive(p, x, y, spec)
        assert torch.equal(p.cell_params[:, r0:r1, c0:c1], want)
        st.step(x, y)
    assert torch.equal(p.cell_params[:, ~inside], before[:, ~inside])
    assert torch.equal(tr.momentum.cell_params[:, ~inside], mom[:, ~inside])
    assert not torch.equal(p.cell_params, before)
    assert _same(st.params, p)


def test_sub_rois_that_cannot_be_updated_are_refused():
    topo = nc.ChipTopology2D.alu_chip()
    x, y = _batch(4, 4)
    tr, p = _trainer(), _params(6)
    spec = dataclasses.replace(nc.compute_adaptive_spatial_mask(nc.init_vnn_params(701, topo, device=DEV), topo),
                               cropped_topology=None)
    before = p.cell_params.clone()
    with pytest.raises(ValueError, match="topology"):
        tr.train_step_adaptive(p, x, y, spec)
    outer = dataclasses.replace(spec, cropped_topology=dataclasses.replace(topo, out_in_roi=False))
    with pytest.raises(NotImplementedError, match="output ports"):
        tr.train_step_adaptive(p, x, y, outer)
    assert torch.equal(p.cell_params, before)
    # CIRCULAR chips take no mask: all cells are trained
    ring = dataclasses.replace(spec, cropped_topology=dataclasses.replace(topo, padding_mode="CIRCULAR"))
    assert tr._muon_window(ring) is None


@pytest.mark.parametrize("captured", [False, True])
def test_the_updates_waits_are_seen(captured):
    """The update's workspaces have status words of their own; here a host write stands for a wait
    that ran out."""
    x, y = _batch(16, 1)
    st = nc.VNNTrainStep(nc.ChipTopology2D.alu_chip(), _params(3), 16, lr=0.02, in_shapes=((8, 1),) * 3,
                         optimizer="muon")
    if captured:
        st.load_batch(x, y)
        st.capture()
    st.step(x, y)
    assert st.wait_status() == 0
    for ws in (st.ws, *st._muon_ws):
        ws[:4].view(torch.int32).fill_(1)
        assert st.wait_status() == 1
        st.step(x, y)                       # each step clears them
        assert st.wait_status() == 0


def test_an_eager_step_checks_its_waits(monkeypatch):
    x, y = _batch(16, 1)
    st = nc.VNNTrainStep(nc.ChipTopology2D.alu_chip(), _params(3), 16, lr=0.02, in_shapes=((8, 1),) * 3,
                         optimizer="muon")
    monkeypatch.setattr(ops, "CHECK_WAIT_STATUS", True)
    n = ops.STATUS_CHECKS
    st.step(x, y)
    assert ops.STATUS_CHECKS == n + 3         # propagation, cells, filters
    st.capture()
    st.step(x, y)
    real = ops.workspace_status
    monkeypatch.setattr(ops, "workspace_status", lambda ws: int(ws is st._muon_ws[1]) or real(ws))
    assert st.wait_status() == 1
    st.release()
    with pytest.raises(RuntimeError, match="nc_muon_update"):
        st.step(x, y)


@pytest.mark.parametrize("optimizer", ["sgd", "muon"])
@pytest.mark.parametrize("epoch", [False, True])
def test_a_capture_saves_the_parameters_before_its_warm_up(epoch, optimizer, monkeypatch):
    """The warm-up steps run on a stream of their own, which has to wait for the copies: here what
    follows the stream's wait on the current one is held up for about 50 ms."""
    x, y = _batch(16, 1)
    p = _params(3)
    st = nc.VNNTrainStep(nc.ChipTopology2D.alu_chip(), p, 16, lr=0.5, in_shapes=((8, 1),) * 3, optimizer=optimizer)
    st.load_batch(x, y)
    st.step()
    before = st.flat.clone()
    mom = None if st.momentum is None else st.momentum.clone()
    torch.cuda.synchronize()
    real = torch.cuda.Stream.wait_stream

    def wait_stream(self, other):
        real(self, other)
        if self != torch.cuda.current_stream():
            torch.cuda._sleep(100_000_000)

    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda.Stream, "wait_stream", wait_stream)
        if epoch:
            st.capture_epoch(x[None], y[None])
        else:
            st.capture()
    torch.cuda.synchronize()
    assert torch.equal(st.flat, before)
    assert mom is None or torch.equal(st.momentum, mom)


def _step_of(world, monkeypatch, **kw):
    """A step whose ranks all hold the same batch: the exchange's sum is `world` times its gradient."""
    from neurocell_b200 import trainer

    def exchange(flat, group=None):
        flat.mul_(world)
        return world

    monkeypatch.setattr(trainer, "allreduce_mean_", exchange)
    monkeypatch.setattr(torch.distributed, "get_world_size", lambda group=None: world)
    return nc.VNNTrainStep(nc.ChipTopology2D.alu_chip(), _params(3), 16, lr=0.02, in_shapes=((8, 1),) * 3,
                           optimizer="muon", process_group=object(), weight_decay=0.1, **kw)


@pytest.mark.parametrize("world", [2, 8])
def test_ranks_take_the_step_of_the_mean_gradient(world, monkeypatch):
    """Ranks on the same batch step as one does.  Powers of two scale momentum, norm and eps without
    a rounding, so the bits are the same."""
    x, y = _batch(16, 1)
    flats = []
    for n in (1, world):
        st = _step_of(n, monkeypatch)
        for _ in range(3):
            st.step(x, y)
        flats.append((st.flat.clone(), st.momentum / n))
    assert _same(*flats)


def test_the_fused_exchange_is_refused_with_muon(monkeypatch):
    with pytest.raises(NotImplementedError, match="nvlink"):
        _step_of(2, monkeypatch, exchange="nvlink")
