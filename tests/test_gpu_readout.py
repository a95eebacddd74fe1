"""The linear readout's softmax cross-entropy (ops.linear_softmax_ce_loss) against its
formula in 64 bits: values, gradients, masks, alignment, streams and graphs.

Tolerances, elementwise, from the arithmetic (u = 2^-24, one rounding of a float32):
* a logit is a sum of `dim` products and a bias.  Sum error (dim + 4) u times the sum of the
  products' magnitudes; the tensor-core path also rounds every factor to 22 bits (2^-23
  relative each) and drops the product of the two low parts (2^-24): 2^-21 in all.
* the loss adds the errors of the log-sum-exp and of one logit, and a few roundings.
* a probability inherits twice the logit error as a relative error, and the rounding of exp
  (2 ulp), of the difference and of its scale: 8 u.  Beside bfloat16 inputs the matrix
  products read it rounded to bfloat16: 2^-8.  Beside float32 inputs they read 2^15 dz (dz
  taken relative to the largest g) as two float16 parts.  float16's smallest step is 2^-24,
  so whatever dz's size the low part is off by at most half of that, 2^-25 / 2^15 = 2^-40.
* a gradient is a sum of `rows` (or `classes`) products again; a bfloat16 result is rounded
  once more: 2^-8 relative.
"""
import ctypes

import numpy as np
import pytest
import torch

from neurocell_b200 import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _check_wait_status(monkeypatch, request):
    """Every call's bounded waits are checked (not inside a capture, which cannot read them)."""
    if not any(k in request.node.name for k in ("replayed", "captured", "at_once")):
        monkeypatch.setattr(ops, "CHECK_WAIT_STATUS", True)


U = 2.0 ** -24
DEV = torch.device("cuda:0")
IGNORE = -100


def _case(rows, dim, classes, dtype=torch.float32, seed=0, bias=True, scale=2.0, drop=0.0):
    g = torch.Generator().manual_seed(seed)
    f = torch.randn(rows, dim, generator=g).to(dtype)
    w = (torch.randn(classes, dim, generator=g) * scale / dim ** 0.5).to(dtype)
    b = (0.5 * torch.randn(classes, generator=g)).to(dtype) if bias else None
    lab = torch.randint(0, classes, (rows,), generator=g)
    lab = torch.where(torch.rand(rows, generator=g) < drop, torch.full_like(lab, IGNORE), lab)
    return [None if t is None else t.to(DEV) for t in (f, w, b, lab)]


def _formula(f, w, b, lab, reduction="mean", g_loss=None):
    """Loss and gradients in 64 bits, with the elementwise tolerances of the module's note."""
    bf16 = f.dtype == torch.bfloat16
    kept = lab != IGNORE
    fd, wd = torch.where(kept[:, None], f, torch.zeros_like(f)).double(), w.double()
    bd = torch.zeros(w.shape[0], dtype=torch.float64, device=f.device) if b is None else b.double()
    rows, dim = f.shape
    classes = w.shape[0]
    at = torch.where(kept, lab, torch.zeros_like(lab)).long()
    z = fd @ wd.T + bd
    mag = (fd.abs() @ wd.abs().T + torch.where(torch.isinf(bd), torch.zeros_like(bd), bd.abs())).max(dim=1).values
    ez = ((dim + 4) * U + 2.0 ** -21) * mag                     # error of a row's logits
    lse = torch.logsumexp(z, 1)
    loss = torch.where(kept, lse - z.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    tol_loss = 2 * ez + 8 * U * (lse.abs() + mag + 1)
    count = max(1, int(kept.sum()))
    g = torch.ones(rows, dtype=torch.float64, device=f.device) if g_loss is None else \
        g_loss.double().expand(rows)
    g = torch.where(kept, g, torch.zeros_like(g)) / (count if reduction == "mean" else 1)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    dz = (p - hot) * g[:, None]
    size = (p + hot) * g.abs()[:, None]
    rel = (2 * ez + 8 * U)[:, None] + (2.0 ** -8 if bf16 else 2.0 ** -21)
    e_dz = size * rel + (0.0 if bf16 else 2.0 ** -40 * float(g.abs().max()))
    out = 2.0 ** -8 if bf16 else 2 * U
    grads = []
    for exact, a, e, y, k in ((dz @ wd, size, e_dz, wd, classes), (dz.T @ fd, size.T, e_dz.T, fd, rows)):
        grads.append((exact, e @ y.abs() + ((k + 4) * U) * (a @ y.abs()) + out * exact.abs() + 1e-30))
    gb = dz.sum(0)
    grads.append((gb, e_dz.sum(0) + (rows + 4) * U * size.sum(0) + out * gb.abs() + 1e-30))
    if reduction == "mean":
        loss, tol_loss = loss.sum() / count, (tol_loss * kept).sum() / count + 2 * U * loss.abs().sum() / count
    elif reduction == "sum":
        loss, tol_loss = loss.sum(), (tol_loss * kept).sum() + 2 * U * loss.abs().sum()
    return (loss, tol_loss), grads


def _within(got, exact, tol, what):
    off = (got.double() - exact).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"


def _check(f, w, b, lab, reduction="mean"):
    (loss, tol), grads = _formula(f, w, b, lab, reduction)
    got = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b, reduction=reduction)
    torch.cuda.synchronize()
    _within(got[0], loss, tol, "loss")
    for name, x, (e, t) in zip(("features", "weight", "bias"), got[1:], grads):
        if name == "bias" and b is None:
            assert x is None
            continue
        assert x.dtype == f.dtype
        _within(x, e, t, "gradient of the " + name)


SHAPES = [(1, 1, 1), (1, 8, 2), (2, 3, 31), (4, 64, 257), (5, 100, 33), (8, 1024, 999), (16, 129, 1000),
          (17, 40, 64), (33, 1030, 100), (128, 8, 256), (130, 72, 515), (257, 36, 1025), (300, 200, 90)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,classes", SHAPES)
def test_value_and_gradients(rows, dim, classes, dtype):
    _check(*_case(rows, dim, classes, dtype, seed=rows + dim))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("rows", [3, 200])
def test_reductions_without_bias_and_with_ignored_rows(rows, reduction, dtype):
    _check(*_case(rows, 48, 300, dtype, seed=7, bias=False, drop=0.4), reduction=reduction)


@pytest.mark.parametrize("rows,dim,classes", [(6, 20, 50), (150, 64, 300)])
def test_ignored_rows_may_hold_anything(rows, dim, classes):
    f, w, b, lab = _case(rows, dim, classes, seed=3, drop=0.3)
    lab[0] = IGNORE
    junk = f.clone()
    junk[lab == IGNORE] = float("nan")
    junk[0] = float("inf")
    a = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b)
    c = ops.linear_softmax_ce_value_and_grad(junk, w, lab, bias=b)
    for x, y in zip(a, c):
        assert torch.isfinite(y).all() and torch.equal(x, y)
    assert (a[1][lab == IGNORE] == 0).all()


@pytest.mark.parametrize("rows", [4, 140])
def test_every_row_ignored(rows):
    f, w, b, lab = _case(rows, 16, 40)
    lab.fill_(IGNORE)
    for x in ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b):
        assert (x == 0).all()


@pytest.mark.parametrize("rows", [3, 140])
def test_masked_classes(rows):
    """A bias of -inf, or of the type's lowest value, takes classes out."""
    f, w, b, lab = _case(rows, 32, 300, seed=5)
    for low in (float("-inf"), torch.finfo(torch.float32).min):
        bm = b.clone()
        bm[7:290] = low
        labm = torch.where((lab >= 7) & (lab < 290), torch.zeros_like(lab), lab)
        keep = torch.cat([torch.arange(7), torch.arange(290, 300)]).to(DEV)
        relabel = torch.searchsorted(keep, labm)
        (loss, tol), grads = _formula(f, w[keep], b[keep], relabel)
        got = ops.linear_softmax_ce_value_and_grad(f, w, labm, bias=bm)
        _within(got[0], loss, tol, "loss")
        _within(got[1], *grads[0], "gradient of the features")
        _within(got[2][keep], *grads[1], "gradient of the weight")
        _within(got[3][keep], *grads[2], "gradient of the bias")
        assert (got[2][7:290] == 0).all() and (got[3][7:290] == 0).all()


@pytest.mark.parametrize("rows", [3, 140])
def test_nothing_left_and_bad_labels_read_nan(rows):
    f, w, b, lab = _case(rows, 32, 70, seed=5)
    assert torch.isnan(ops.linear_softmax_ce_loss(f, w, lab, bias=torch.full_like(b, float("-inf"))))
    for bad in (70, 10 ** 6, -1, 2 ** 40):
        l2 = lab.clone()
        l2[1] = bad
        loss = ops.linear_softmax_ce_loss(f, w, l2, bias=b, reduction="none")
        assert torch.isnan(loss[1]) and torch.isfinite(loss[[0, 2]]).all()
        g = ops.linear_softmax_ce_value_and_grad(f, w, l2, bias=b)
        assert torch.isnan(g[0]) and torch.isnan(g[1][1]).all() and torch.isfinite(g[1][0]).all()
        assert torch.isnan(g[2]).all()


def test_large_logits():
    """exp stays in range whatever the logits' size."""
    for rows in (4, 140):
        f, w, b, lab = _case(rows, 24, 260, seed=9, scale=400.0)
        _check(f, w, b, lab)


def test_scales_of_the_inputs():
    """Features and weights far from one, and one outlier."""
    for rows in (4, 140):
        f, w, b, lab = _case(rows, 48, 200, seed=11)
        _check(f * 2.0 ** 40, w * 2.0 ** -40, b, lab)
        _check(f * 2.0 ** -60, w * 2.0 ** 58, b, lab)
        _check(f * 0, w, b, lab)
        w2 = w.clone()
        w2[5, 3] = 200.0
        _check(f, w2, b, lab)


def test_strided_and_misaligned_inputs():
    for rows in (5, 140):
        for dtype in (torch.float32, torch.bfloat16):
            f, w, b, lab = _case(rows, 64, 131, dtype, seed=13)
            want = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b)
            wide = torch.full((rows, 130), 9.0, dtype=dtype, device=DEV)
            wide[:, :128:2] = f
            got = ops.linear_softmax_ce_value_and_grad(wide[:, :128:2], w.t().contiguous().t(),
                                                       lab.repeat_interleave(2)[::2], bias=b)
            for x, y in zip(want, got):
                assert torch.equal(x, y)
            off = [torch.empty(t.numel() + 1, dtype=dtype, device=DEV)[1:].view(t.shape).copy_(t)
                   for t in (f, w, b)]
            (loss, tol), grads = _formula(f, w, b, lab)
            got = ops.linear_softmax_ce_value_and_grad(off[0], off[1], lab, bias=off[2])
            _within(got[0], loss, tol, "loss")
            for x, (e, t) in zip(got[1:], grads):
                _within(x, e, t, "gradient")


def test_autograd_equals_value_and_grad_and_scales():
    for rows in (6, 150):
        f, w, b, lab = _case(rows, 40, 90, seed=17, drop=0.2)
        want = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b)
        leaves = [t.clone().requires_grad_() for t in (f, w, b)]
        loss = ops.linear_softmax_ce_loss(*leaves[:2], lab, bias=leaves[2])
        assert torch.equal(loss.detach(), want[0])
        (4.0 * loss).backward()
        for t, g in zip(leaves, want[1:]):
            assert torch.allclose(t.grad, 4.0 * g, rtol=2 ** -20, atol=1e-9 * float(g.abs().max()))
        # one input alone
        only = w.clone().requires_grad_()
        (gw,) = torch.autograd.grad(ops.linear_softmax_ce_loss(f, only, lab, bias=b), only)
        assert torch.equal(gw, want[2])
        with torch.no_grad():
            assert not ops.linear_softmax_ce_loss(leaves[0], leaves[1], lab).requires_grad


@pytest.mark.parametrize("rows", [5, 140])
def test_gradient_of_each_row_of_none(rows):
    f, w, b, lab = _case(rows, 40, 90, seed=19, drop=0.2)
    g = torch.randn(rows, device=DEV)
    g[2] = 0.0
    g[3] = 1e4
    (_, _), grads = _formula(f, w, b, lab, "none", g)
    leaves = [t.clone().requires_grad_() for t in (f, w, b)]
    loss = ops.linear_softmax_ce_loss(*leaves[:2], lab, bias=leaves[2], reduction="none")
    got = torch.autograd.grad(loss, leaves, g)
    for x, (e, t) in zip(got, grads):
        _within(x, e, t, "gradient")
    # an expanded gradient (stride 0), as sum() gives
    loss = ops.linear_softmax_ce_loss(*leaves[:2], lab, bias=leaves[2], reduction="none")
    got = torch.autograd.grad(loss.sum(), leaves)
    for x, (e, t) in zip(got, _formula(f, w, b, lab, "none")[1]):
        _within(x, e, t, "gradient")


def test_gradients_against_differences():
    """Central differences of the summed loss.  Step h: truncation h^2 / 6 times the third
    derivative, at most the sum of |x|^3 / (6 sqrt 3) over the rows for a logit's slope x;
    rounding: the loss's own tolerance over h."""
    f, w, b, lab = _case(4, 5, 6, seed=23)
    h = 2.0 ** -6
    _, gf, gw, gb = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b, reduction="sum")
    tol_l = float(_formula(f, w, b, lab, "sum")[0][1])
    for t, g, third in ((f, gf, w.double().abs().max() ** 3 * 6), (w, gw, f.double().abs().pow(3).sum()),
                        (b, gb, torch.tensor(4.0))):
        tol = h * h / 6 * float(third) / (6 * 3 ** 0.5) * 2 + 2 * tol_l / (2 * h)
        flat, gr = t.view(-1), g.reshape(-1)
        for i in range(flat.numel()):
            x = float(flat[i])
            flat[i] = x + h
            up = float(ops.linear_softmax_ce_loss(f, w, lab, bias=b, reduction="sum").double())
            flat[i] = x - h
            dn = float(ops.linear_softmax_ce_loss(f, w, lab, bias=b, reduction="sum").double())
            flat[i] = x
            assert abs((up - dn) / (2 * h) - float(gr[i])) <= tol


def test_no_rows():
    f, w, b, lab = _case(0, 16, 40)
    out = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b)
    assert float(out[0]) == 0.0 and out[1].shape == (0, 16)
    assert (out[2] == 0).all() and (out[3] == 0).all()
    assert ops.linear_softmax_ce_loss(f, w, lab, reduction="none").shape == (0,)


def test_same_bits_twice_on_another_stream_and_replayed():
    for rows in (8, 200):
        f, w, b, lab = _case(rows, 72, 700, seed=29, drop=0.1)
        want = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b)
        s.synchronize()
        for x, y in zip(want, again):
            assert torch.equal(x, y)
        # captured, and replayed on other inputs in the same buffers
        fs = f.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.linear_softmax_ce_value_and_grad(fs, w, lab, bias=b)
        fs.copy_(f * 0.5)
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(ops.linear_softmax_ce_value_and_grad(f * 0.5, w, lab, bias=b), out):
            assert torch.equal(x, y)


def test_c_entry_points_refuse_bad_workspaces():
    lib = _lib.load()
    f, w, b, lab = _case(4, 16, 40)
    lab = lab.to(torch.int32)
    d = _lib.NcLinearCe(4, 16, 40, 0, IGNORE, 0)
    n = lib.nc_linear_ce_workspace_bytes(ctypes.byref(d), 0)
    ws = torch.empty(n + 256, dtype=torch.uint8, device=DEV)
    loss, lse = torch.empty((), device=DEV), torch.empty(4, device=DEV)
    P = ops._ptr
    args = (ctypes.byref(d), P(f), P(w), P(b), P(lab), P(loss), P(lse))
    assert lib.nc_linear_ce_forward(*args, P(ws), n - 1, None) == _lib.NC_ERR_WORKSPACE
    assert lib.nc_linear_ce_forward(*args, ctypes.c_void_p(ws.data_ptr() + 4), n, None) == _lib.NC_ERR_WORKSPACE
    assert lib.nc_linear_ce_forward(*args, None, n, None) == _lib.NC_ERR_WORKSPACE
    assert lib.nc_linear_ce_forward(ctypes.byref(d), None, P(w), P(b), P(lab), P(loss), P(lse), P(ws), n,
                                    None) == _lib.NC_ERR_INVALID


def _past_32_bits(rows, dim, classes, dtype):
    """A weight of more than 2^31 elements: the formula by pieces of the classes."""
    gen = torch.Generator(device=DEV).manual_seed(41)
    w = torch.empty(classes, dim, dtype=dtype, device=DEV).normal_(generator=gen).mul_(2.0 / dim ** 0.5)
    f = torch.randn(rows, dim, device=DEV, generator=gen).to(dtype)
    lab = torch.randint(0, classes, (rows,), device=DEV, generator=gen)
    lab[0], lab[1] = classes - 1, 0
    loss, g_f, g_w, _ = ops.linear_softmax_ce_value_and_grad(f, w, lab)
    torch.cuda.synchronize()
    step, fd = 100_000, f.double()
    pieces = [(k, min(classes, k + step)) for k in range(0, classes, step)]
    lse = torch.full((rows,), -float("inf"), dtype=torch.float64, device=DEV)
    mag, at = torch.zeros_like(lse), torch.zeros_like(lse)
    for a, b in pieces:
        y = w[a:b].double()
        z = fd @ y.T
        lse = torch.logaddexp(lse, torch.logsumexp(z, 1))
        mag = torch.maximum(mag, (fd.abs() @ y.abs().T).amax(1))
        here = (lab >= a) & (lab < b)
        at = torch.where(here, z.gather(1, (lab - a).clamp(0, b - a - 1)[:, None])[:, 0], at)
    ez = ((dim + 4) * U + 2.0 ** -21) * mag
    # the statistics join at most `classes` terms, in float32 sums of a few hundred terms joined as a tree
    tol = 2 * ez + 8 * U * (lse.abs() + mag + 1) + 1024 * U
    _within(loss, (lse - at).mean(), tol.mean() + 2 * U * (lse - at).abs().mean(), "loss")
    bf16 = dtype == torch.bfloat16
    rel = 2 * ez + 1032 * U + (2.0 ** -8 if bf16 else 2.0 ** -21)
    out = 2.0 ** -8 if bf16 else 2 * U
    df, t_df, size_f = (torch.zeros(rows, dim, dtype=torch.float64, device=DEV) for _ in range(3))
    for a, b in pieces:
        y = w[a:b].double()
        p = torch.exp(fd @ y.T - lse[:, None])
        hot = torch.zeros_like(p)
        here = ((lab >= a) & (lab < b)).nonzero()[:, 0]
        hot[here, lab[here] - a] = 1.0
        dz, size = (p - hot) / rows, (p + hot) / rows
        e = size * rel[:, None] + (0.0 if bf16 else 2.0 ** -40 / rows)
        df += dz @ y
        t_df += e @ y.abs()
        size_f += size @ y.abs()
        if a in (0, pieces[len(pieces) // 2][0], pieces[-1][0]):
            dw = dz.T @ fd
            t = e.T @ fd.abs() + (rows + 4) * U * (size.T @ fd.abs()) + out * dw.abs() + 1e-30
            _within(g_w[a:b], dw, t, f"gradient of the weight from {a}")
    # a sum over the classes: roundings of a random sign, eight standard deviations of them
    _within(g_f, df, t_df + 8 * classes ** 0.5 * U * size_f + out * df.abs() + 1e-30, "gradient of the features")


@pytest.mark.parametrize("rows,dim,classes,dtype", [(3, 1024, 2_200_001, torch.float32),
                                                    (3, 1024, 2_200_001, torch.bfloat16),
                                                    (20, 520, 4_200_001, torch.bfloat16),
                                                    (20, 520, 4_200_001, torch.float32)])
def test_offsets_past_32_bits(rows, dim, classes, dtype):
    _past_32_bits(rows, dim, classes, dtype)


@pytest.mark.parametrize("rows,dim,classes,dtype", [(1100, 40, 40001, torch.float32),
                                                    (1100, 72, 80001, torch.bfloat16)])
def test_several_pieces_of_the_classes(rows, dim, classes, dtype):
    # more than 160 MB of dz, so the gradients' products go by pieces and add up df
    _check(*_case(rows, dim, classes, dtype, seed=43, drop=0.1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,dim,classes", [(1001, 1010, 18690), (1024, 1024, 18944), (2048, 512, 4100),
                                              (520, 264, 30000)])
def test_products_by_pairs_of_ctas(rows, dim, classes, dtype):
    # enough rounds of 256 x 256 tiles for the value, dz, dw and df to go by pairs (the first two; the
    # others some of them)
    _check(*_case(rows, dim, classes, dtype, seed=45, drop=0.1))


def test_calls_at_once_on_several_streams():
    cases = [_case(8, 1024, 3001, seed=1), _case(200, 72, 700, seed=2), _case(400, 260, 5000, torch.bfloat16, seed=3),
             _case(2, 64, 50_000, torch.bfloat16, seed=4)]
    want = [ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b) for f, w, b, lab in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        for s, (f, w, b, lab) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for x, y in zip(want[i % len(cases)], out):
            assert torch.equal(x, y), i


@pytest.mark.parametrize("rows", [3, 140])
def test_loss_gradients_of_zero_and_nan(rows):
    f, w, b, lab = _case(rows, 24, 70, seed=47)
    for t in (f, w, b):
        t.requires_grad_()
    for bad in (None, 1):
        g = torch.zeros(rows, device=DEV)
        if bad is not None:
            g[bad] = float("nan")
        loss = ops.linear_softmax_ce_loss(f, w, lab, bias=b, reduction="none")
        gf, gw, gb = torch.autograd.grad(loss, (f, w, b), g)
        if bad is None:
            assert not gf.any() and not gw.any() and not gb.any()
        else:      # a NaN is passed on
            assert gf[bad].isnan().all() and gw.isnan().all() and gb.isnan().all()


def test_two_captures_replayed_at_once():
    # each graph holds its own workspace
    graphs, outs, wants = [], [], []
    for seed, (rows, dim, classes) in enumerate(((8, 64, 3001), (200, 72, 700), (200, 72, 700))):
        f, w, b, lab = _case(rows, dim, classes, seed=60 + seed)
        wants.append(ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.linear_softmax_ce_value_and_grad(f, w, lab, bias=b))
        graphs.append((g, torch.cuda.Stream(), (f, w, b, lab)))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s, _ in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for want, out in zip(wants, outs):
        for x, y in zip(want, out):
            assert torch.equal(x, y)
