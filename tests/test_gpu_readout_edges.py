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


# Long sums of bfloat16 operands.  Terms of one sign, so that what each addition loses adds up: a
# float32 accumulator that rounds toward zero loses on average half of 2^-24 to 2^-23 of itself per
# addition.  The mean error over many elements shows it; the roundings to nearest of dz and of the
# result (2^-9 at most each) have random signs and leave 2^-9 / sqrt(elements), eight of which are allowed
# beside 2^-14 for the sums.
def _positive(*shape, gen):
    return (torch.rand(*shape, device=DEV, generator=gen) + 0.5).to(torch.bfloat16)


@pytest.mark.parametrize("rows,dim,classes", [(1 << 18, 16, 300), (1 << 18, 200, 600)])
def test_a_weight_gradient_sums_many_rows(rows, dim, classes):
    gen = torch.Generator(DEV).manual_seed(1)
    f = _positive(rows, dim, gen=gen)
    w = (torch.randn(classes, dim, device=DEV, generator=gen) * 1.2 / dim ** 0.5).to(torch.bfloat16)
    lab = torch.zeros(rows, dtype=torch.int32, device=DEV)
    gw = ops.linear_softmax_ce_value_and_grad(f, w, lab, reduction="sum")[2]
    exact = torch.zeros(classes, dim, dtype=torch.float64, device=DEV)
    for a in range(0, rows, 1 << 16):
        fd = f[a:a + (1 << 16)].double()
        p = torch.softmax(fd @ w.double().T, 1)
        p[:, 0] -= 1
        exact += p.T @ fd
    off = ((gw.double() - exact) / exact)[1:]
    assert abs(float(off.mean())) <= 8 * 2.0 ** -9 / off.numel() ** 0.5 + 2.0 ** -14


def test_a_feature_gradient_sums_many_classes():
    rows, dim, classes = 256, 4096, 200_000
    gen = torch.Generator(DEV).manual_seed(2)
    f = (torch.randn(rows, dim, device=DEV, generator=gen) / dim ** 0.5).to(torch.bfloat16)
    w = _positive(classes, dim, gen=gen)
    lab = torch.randint(0, classes, (rows,), device=DEV, generator=gen)
    gf = ops.linear_softmax_ce_value_and_grad(f, w, lab, reduction="sum")[1]
    z = torch.cat([f.double() @ w[a:a + 20_000].double().T for a in range(0, classes, 20_000)], 1)
    p = torch.softmax(z, 1)
    exact = -w[lab].double()
    for a in range(0, classes, 20_000):
        exact += p[:, a:a + 20_000] @ w[a:a + 20_000].double()
    # the sum of p w is about 1 in every element
    off = gf.double() - exact
    assert abs(float(off.mean())) <= 8 * 2.0 ** -9 / off.numel() ** 0.5 + 2.0 ** -14


def test_a_logit_sums_a_long_dim():
    rows, dim, classes = 40, 1 << 17, 300
    gen = torch.Generator(DEV).manual_seed(3)
    f = _positive(rows, dim, gen=gen)
    size = torch.linspace(0, 20, classes, device=DEV)[:, None] / dim
    w = (_positive(classes, dim, gen=gen) * size).to(torch.bfloat16)
    lab = torch.randint(0, 20, (rows,), device=DEV, generator=gen)
    loss = ops.linear_softmax_ce_loss(f, w, lab, reduction="none")
    z = f.double() @ w.double().T
    exact = torch.logsumexp(z, 1) - z.gather(1, lab[:, None])[:, 0]
    assert (loss.double() - exact).abs().max() <= 2.0 ** -14 * float(z.max()) + 2.0 ** -20 * float(exact.max())


@pytest.mark.parametrize("exponent", [112, -112, 90, -90])
@pytest.mark.parametrize("rows", [4, 140])
def test_far_scales_that_meet_in_the_logits(rows, exponent):
    """Features of 2^e and a weight of 2^-e: logits of ordinary size.  Relative to the largest entry of
    each result: sums of `dim`, `rows` or `classes` products as float32 ones, 2^-20 of their size."""
    f, w, lab = _inputs(rows, 40, 90, torch.float32, seed=5)
    f, w = f * 2.0 ** exponent, w * (0.3 * 2.0 ** -exponent)
    loss, gf, gw, _ = ops.linear_softmax_ce_value_and_grad(f, w, lab)
    fd, wd = f.double().requires_grad_(), w.double().requires_grad_()
    want = torch.nn.functional.cross_entropy(fd @ wd.T, lab)
    assert abs(float(loss) - float(want.detach())) <= 2.0 ** -20 * 10
    for got, e in zip((gf, gw), torch.autograd.grad(want, (fd, wd))):
        assert (got.double() - e).abs().max() <= 2.0 ** -18 * e.abs().max()


# A label's logit of 64 and the others 12 below it, all exact: loss log(1 + (classes - 1) exp(-12)).  exp
# and log are off by 2^-20 of the small part.  The sum that holds the label's 1 takes further terms by
# float32 additions, each rounded by at most 2^-24: up to 32 in a tile of 128 classes (four chains, 16 in
# one of 64; 16 a lane in a window of 512 classes), 2 to join the chains, at most 5 tiles or windows or 5
# per lane of 300 classes' blocks, and 5 in a warp's tree: under 48.  The rounding of a log-sum-exp of
# 64.0018 would be 3.3e-6 here, 48 2^-24 is 2.9e-6.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 16, 140])
def test_the_loss_of_a_confident_row(rows, dtype):
    classes = 300
    f = torch.zeros(rows, 24, device=DEV, dtype=dtype)
    f[:, 0] = 8.0
    w = torch.zeros(classes, 24, device=DEV, dtype=dtype)
    w[:, 0] = 6.5
    w[7, 0] = 8.0
    lab = torch.full((rows,), 7, device=DEV)
    loss = ops.linear_softmax_ce_loss(f, w, lab, reduction="none")
    want = torch.log1p((classes - 1) * torch.exp(torch.tensor(-12.0, dtype=torch.float64)))
    assert (loss.double() - want.item()).abs().max() <= 48 * 2.0 ** -24 + 2.0 ** -20 * want.item()


@pytest.mark.parametrize("rows", [4, 140])
def test_the_loss_where_every_class_has_the_lowest_bias(rows):
    f, w, lab = _inputs(rows, 40, 90, torch.float32)
    b = torch.full((90,), torch.finfo(torch.float32).min, device=DEV)
    loss = ops.linear_softmax_ce_loss(f, w, lab, bias=b, reduction="none")
    want = torch.log(torch.tensor(90.0, dtype=torch.float64)).item()
    assert (loss[::2].double() - want).abs().max() <= 2.0 ** -22 * want and (loss[1::2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 140])
def test_gradients_without_a_class_left_are_nan(rows, dtype):
    f, w, lab = _inputs(rows, 40, 90, dtype)
    for low in (torch.finfo(dtype).min, -1e9):
        b = torch.full((90,), low, device=DEV, dtype=dtype)
        loss, gf, gw, gb = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b)
        assert torch.isfinite(loss)
        assert gf[::2].isnan().all() and (gf[1::2] == 0).all() and gw.isnan().all() and gb.isnan().all()
        # one class left, or one far above the others: as ever
        for high in (0.0, 1e9):
            b[7] = high
            one = torch.where(lab == IGNORE, lab, torch.full_like(lab, 7))
            loss, gf, gw, gb = ops.linear_softmax_ce_value_and_grad(f, w, one, bias=b)
            assert float(loss) == 0 and not gf.any() and not gw.any() and not gb.any()
