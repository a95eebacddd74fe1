"""The readout loss and the orthogonalised update together, as a training program uses them: a
VNN's output ports read by a linear layer over many classes, gradients of all of it, and the
update of cells, filters and readout; in eager steps, in VNNTrainer and in captured graphs."""
import numpy as np
import pytest
import torch

import neurocell_b200 as nc
from neurocell_b200 import ops
from oracle import vnn_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _check_wait_status(monkeypatch, request):
    """Every call's bounded waits are checked (not inside a capture, which cannot read them)."""
    if "replayed" not in request.node.name and "captured" not in request.node.name:
        monkeypatch.setattr(ops, "CHECK_WAIT_STATUS", True)


DEV = torch.device("cuda:0")


def _chip(B, seed=0):
    rng = np.random.default_rng(seed)
    cell = torch.tensor(rng.normal(0, 0.1, (3, 62, 62)).astype(np.float32), device=DEV)
    filt = torch.tensor((rng.normal(0, 1, (16, 1, 23, 13)) / np.sqrt(299)).astype(np.float32), device=DEV)
    x, y, _ = O.alu_batch(rng, B, noise=0.0)
    return cell, filt, torch.tensor(x, device=DEV), torch.tensor(y, device=DEV)


@pytest.mark.parametrize("B,classes", [(4, 300), (48, 300)])
def test_gradients_reach_the_chip_through_the_readout(B, classes):
    """d loss / d (cells, filters) equals the VNN's own adjoint of the readout's feature
    gradient: a directional difference of the whole loss along a random direction.  Central
    differences with step h leave h^2 / 6 of the third derivative and twice the loss's
    rounding over 2 h; with h = 2^-5 and |direction| = 1 both are below 2e-3 of the slope."""
    cell, filt, x, _ = _chip(B)
    topo = nc.ChipTopology2D.alu_chip()
    g = torch.Generator().manual_seed(1)
    w = torch.randn(classes, 8, generator=g).to(DEV)
    lab = torch.randint(0, classes, (B,), generator=g).to(DEV)

    def loss_of(c, f):
        out = nc.propagate_vnn_2d(nc.VNNParams(c, f), x, topo).reshape(B, -1)
        return ops.linear_softmax_ce_loss(out, w, lab, reduction="sum")

    c, f = cell.clone().requires_grad_(), filt.clone().requires_grad_()
    gc, gf = torch.autograd.grad(loss_of(c, f), (c, f))
    h = 2.0 ** -5
    with torch.no_grad():
        for p, gr in ((0, gc), (1, gf)):
            d = gr / gr.norm()
            up = loss_of(*((cell + h * d, filt) if p == 0 else (cell, filt + h * d)))
            dn = loss_of(*((cell - h * d, filt) if p == 0 else (cell, filt - h * d)))
            slope = float(gr.norm())
            third = 0.05 * slope
            assert abs(float(up - dn) / (2 * h) - slope) <= third


def test_a_step_of_everything_equals_the_formulas():
    B, classes = 40, 513
    cell, filt, x, _ = _chip(B, 3)
    topo = nc.ChipTopology2D.alu_chip()
    g = torch.Generator().manual_seed(2)
    w = (0.3 * torch.randn(classes, 8, generator=g)).to(DEV)
    b = torch.zeros(classes, device=DEV)
    lab = torch.randint(0, classes, (B,), generator=g).to(DEV)
    leaves = [t.clone().requires_grad_() for t in (cell, filt, w, b)]
    out = nc.propagate_vnn_2d(nc.VNNParams(*leaves[:2]), x, topo).reshape(B, -1)
    loss = ops.linear_softmax_ce_loss(out, leaves[2], lab, bias=leaves[3])
    grads = torch.autograd.grad(loss, leaves)
    # the readout's own gradients, from the same features in 64 bits
    f64 = out.detach().double().requires_grad_()
    w64, b64 = w.double().requires_grad_(), b.double().requires_grad_()
    ref = torch.nn.functional.cross_entropy(f64 @ w64.T + b64, lab)
    rw, rb = torch.autograd.grad(ref, (w64, b64))
    assert abs(float(loss) - float(ref)) <= 1e-5 * float(ref)
    assert (grads[2].double() - rw).norm() <= 1e-5 * rw.norm()
    assert (grads[3].double() - rb).norm() <= 1e-5 * rb.norm()
    # the update of every matrix
    for p, gr in zip((cell, filt, w), grads):
        shape = p.shape if p.ndim != 4 else (p.shape[0], -1)
        q, m = p.clone().view(shape), torch.zeros_like(p).view(shape)
        ops.muon_(q, gr.contiguous().view(shape), m, 0.02)
        u = gr.double().view(shape) * 1.95
        o = ops.orthogonalize(u.float()).double()
        step = 0.02 * max(1.0, shape[-2] / q.shape[-1]) ** 0.5
        assert (q.double() - (p.double().view(shape) - step * o)).norm() <= 1e-5 * step * o.norm() + 1e-7 * p.double().norm()


def _muon_reference(params, grads, momentum, lr, beta=0.95):
    for p, g, m in zip(params, grads, momentum):
        shape = p.shape if p.ndim == 3 else (p.shape[0], p.numel() // p.shape[0])
        ops.muon_(p.view(shape), g.contiguous().view(shape), m.view(shape), lr, beta=beta)


def test_trainer_and_captured_step_update_by_muon():
    """VNNTrainer, VNNTrainStep eager and VNNTrainStep replayed from a graph take the same
    steps, bit for bit, and ops.muon_ on the trainer's gradients gives them."""
    cell, filt, x, y = _chip(32, 5)
    topo = nc.ChipTopology2D.alu_chip()
    model = nc.VonNeumannNetwork(topo)

    def params():
        return nc.VNNParams(cell.clone(), filt.clone())

    tr = nc.VNNTrainer(model.apply, lr=0.02, optimizer="muon")
    ref, mom = params(), [torch.zeros_like(cell), torch.zeros_like(filt)]
    p = params()
    for _ in range(3):
        _, grads = tr.value_and_grad(ref, x, y)
        _muon_reference(ref, grads, mom, 0.02)
        p, _ = tr.train_step(p, x, y)
    for a, b in zip(p, ref):
        assert torch.equal(a, b)
    steps = []
    for capture in (False, True):
        st = nc.VNNTrainStep(topo, params(), 32, lr=0.02, in_shapes=((8, 1),) * 3, optimizer="muon")
        st.load_batch(x, y)
        if capture:
            st.capture()
        for _ in range(3):
            st.step()
        steps.append(st.flat.clone())
    torch.cuda.synchronize()
    assert torch.equal(steps[0], steps[1])
    assert torch.equal(steps[0][: cell.numel()], p.cell_params.reshape(-1))
    assert torch.equal(steps[0][cell.numel():], p.greens_filters.reshape(-1))
    assert not torch.equal(p.cell_params, cell)


def test_captured_epoch_with_muon_equals_eager_steps():
    cell, filt, _, _ = _chip(16, 6)
    topo = nc.ChipTopology2D.alu_chip()
    rng = np.random.default_rng(7)
    batches = [O.alu_batch(rng, 16, noise=0.0)[:2] for _ in range(3)]
    xd = torch.tensor(np.stack([b[0].reshape(16, -1) for b in batches]), device=DEV)
    yd = torch.tensor(np.stack([b[1] for b in batches]), device=DEV)

    def runner():
        return nc.VNNTrainStep(topo, nc.VNNParams(cell.clone(), filt.clone()), 16, lr=0.01,
                               in_shapes=((8, 1),) * 3, optimizer="muon", weight_decay=0.1)

    eager, ep = runner(), runner()
    ep.capture_epoch(xd, yd)
    for _ in range(2):
        for i in range(3):
            eager.step(xd[i], yd[i])
        ep.train_epoch()
    torch.cuda.synchronize()
    assert torch.equal(eager.flat, ep.flat) and torch.equal(eager.momentum, ep.momentum)


def test_refusals_of_the_optimizer():
    cell, filt, _, _ = _chip(4)
    topo = nc.ChipTopology2D.alu_chip()
    with pytest.raises(ValueError, match="optimizer"):
        nc.VNNTrainStep(topo, nc.VNNParams(cell, filt), 4, optimizer="adam")
    with pytest.raises(ValueError, match="optimizer"):
        nc.VNNTrainer(lambda p, x: x, optimizer="lion")
