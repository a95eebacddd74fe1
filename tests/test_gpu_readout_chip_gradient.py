"""The chip's gradients through the readout loss: against the chain in 64 bits (the oracle's port on
the CPU) and against differences along random directions that know nothing of the gradient, one for
each cell grid and for the filters."""
import numpy as np
import pytest
import torch

import neurocell_b200 as nc
from neurocell_b200 import ops
from oracle import torch_port as T
from oracle import vnn_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CLASSES = 300
PARITY = 1e-5      # of the chip's outputs and gradients against the oracle (test_gpu_parity.py)


def _case(B):
    rng = np.random.default_rng(B)
    cell = rng.normal(0, 0.1, (3, 62, 62)).astype(np.float32)
    filt = (rng.normal(0, 1, (16, 1, 23, 13)) / np.sqrt(299)).astype(np.float32)
    x, _, _ = O.alu_batch(rng, B, noise=0.0)
    g = torch.Generator().manual_seed(1)
    w, b = torch.randn(CLASSES, 8, generator=g), 0.5 * torch.randn(CLASSES, generator=g)
    lab = torch.randint(0, CLASSES, (B,), generator=g)
    lab[B // 2] = -100
    return cell, filt, x, w, b, lab


def _loss(cell, filt, x, w, b, lab):
    out = nc.propagate_vnn_2d(nc.VNNParams(cell, filt), x, nc.ChipTopology2D.alu_chip()).reshape(x.shape[0], -1)
    return ops.linear_softmax_ce_loss(out, w, lab, bias=b, reduction="sum")


@pytest.mark.parametrize("B", [4, 48])
def test_against_the_chain_in_64_bits(B):
    cell, filt, x, w, b, lab = _case(B)
    tv = T.TorchVNN(O.alu_geometry(), O.Config(), torch.float64)
    leaves = [torch.as_tensor(t).double().requires_grad_() for t in (cell, filt, w, b)]
    out = tv.forward(leaves[0], leaves[1], torch.from_numpy(O.inject_full(x, O.alu_geometry(), np.float64)), None)
    z = out.reshape(B, -1) @ leaves[2].T + leaves[3]
    want = torch.autograd.grad(torch.nn.functional.cross_entropy(z, lab, reduction="sum"), leaves)
    here = [torch.as_tensor(t).to(DEV).requires_grad_() for t in (cell, filt, w, b)]
    got = torch.autograd.grad(_loss(here[0], here[1], torch.tensor(x, device=DEV), here[2], here[3], lab.to(DEV)), here)
    # the adjoint is within the parity bound of its incoming gradient, and that one is off by the
    # outputs' error (the same bound) and the readout's own roundings, which are smaller
    for name, a, e in (("W", got[0][0], want[0][0]), ("B", got[0][1], want[0][1]), ("S", got[0][2], want[0][2]),
                       ("filters", got[1], want[1]), ("readout", got[2], want[2]), ("bias", got[3], want[3])):
        off = float((a.cpu().double() - e).norm() / e.norm())
        assert off <= 3 * PARITY, f"{name}: {off:.3g}"


@pytest.mark.parametrize("B", [4, 48])
def test_against_differences_along_random_directions(B):
    """Central differences D(h): the truncation is h^2 / 6 times a third derivative and higher terms,
    so |D(2h) - D(h)| is about three times it; the loss is off by PARITY of itself at most, which
    leaves that over h."""
    cell, filt, x, w, b, lab = _case(B)
    c, f, x, w, b, lab = (torch.as_tensor(t).to(DEV) for t in (cell, filt, x, w, b, lab))
    leaves = [c.clone().requires_grad_(), f.clone().requires_grad_()]
    loss = _loss(*leaves, x, w, b, lab)
    gc, gf = torch.autograd.grad(loss, leaves)
    gen = torch.Generator().manual_seed(100 + B)
    seen = [False] * 4      # blocks whose loss from the gradient the differences would show
    for _ in range(4):
        for block, h in enumerate((2.0 ** -5, 2.0 ** -8, 2.0 ** -5, 2.0 ** -10)):
            d, target = (torch.zeros_like(c), 0) if block < 3 else (torch.zeros_like(f), 1)
            part = d[block] if block < 3 else d
            part.copy_(torch.randn(part.shape, generator=gen))
            slope = float(((gc, gf)[target].double() * d.double()).sum())

            def at(t):
                p = [c + t * d, f] if target == 0 else [c, f + t * d]
                with torch.no_grad():
                    return float(_loss(*p, x, w, b, lab).double())

            near, far = ((at(t) - at(-t)) / (2 * t) for t in (h, 2 * h))
            tol = abs(far - near) + PARITY * float(loss.detach()) / h
            assert abs(near - slope) <= tol, (block, near, slope, tol)
            seen[block] |= abs(near) > tol
    assert all(seen)
