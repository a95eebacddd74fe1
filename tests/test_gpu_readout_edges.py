"""Edges of the linear readout's loss: what ignored rows get, and long sums."""
import pytest
import torch

from neurocell_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
IGNORE = -100


@pytest.fixture(autouse=True)
def _check_wait_status(monkeypatch):
    monkeypatch.setattr(ops, "CHECK_WAIT_STATUS", True)


def _inputs(rows, dim, classes, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    f = torch.randn(rows, dim, generator=g).to(dtype).to(DEV)
    w = torch.randn(classes, dim, generator=g).to(dtype).to(DEV)
    lab = torch.randint(0, classes, (rows,), generator=g).to(DEV)
    lab[1::2] = IGNORE
    return f, w, lab


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 140])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), "weight"])
def test_ignored_rows_have_no_gradient_whatever_the_others_hold(rows, what, dtype):
    f, w, lab = _inputs(rows, 40, 90, dtype)
    if what == "weight":
        w[3, 5] = float("inf")
    f.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = ops.linear_softmax_ce_loss(f, w, lab, reduction=reduction)
        g = torch.ones_like(loss)
        if what != "weight":
            g.fill_(what)
        (gf,) = torch.autograd.grad(loss, f, g)
        assert (gf[1::2] == 0).all() and gf[0].isnan().any()
    if what == "weight":
        gf = ops.linear_softmax_ce_value_and_grad(f.detach(), w, lab)[1]
        assert (gf[1::2] == 0).all() and gf[0].isnan().any()
