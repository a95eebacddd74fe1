"""Newton-Schulz orthogonalisation (ops.orthogonalize) and the update by orthogonalised
momentum (ops.muon_) against their formulas in 64 bits.

The tolerance is a bound on the Frobenius norm of the error, computed beside each case from
the iterates in 64 bits.  A step maps every singular value s by f(s) = a s + b s^3 + c s^5,
so an error that enters before a step leaves it at most max |f'| over [0, largest s] times
as large.  A step adds, for each of its three products, 2^-21 (the factors' rounding, see
below) and 4 sqrt(k) 2^-24 (a sum of k terms, four standard deviations of its roundings) of
the magnitude of what it multiplies, and the roundings of its results:
  |b| |A| |X| + 3 |c| |A|^2 |X| + |a| |X|, spectral norms for A, Frobenius for X.
X0 carries the rounding of its scale, 2^-23.  Factors: float32 values, or their two-part
16-bit form, whose rounding is 2^-23 a factor and 2^-24 for the product left out.
"""
import ctypes

import pytest
import torch

from neurocell_b200 import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _check_wait_status(monkeypatch, request):
    """Every call's bounded waits are checked (not inside a capture, which cannot read them)."""
    if not any(k in request.node.name for k in ("replayed", "captured", "at_once")):
        monkeypatch.setattr(ops, "CHECK_WAIT_STATUS", True)


DEV = torch.device("cuda:0")
U = 2.0 ** -24
COEFFS = ops.NEWTON_SCHULZ_COEFFICIENTS


def _formula(x, steps=5, coeffs=COEFFS, eps=1e-7):
    """(batch of) iterates in 64 bits; returns the result and the error bound per matrix."""
    a, b, c = coeffs
    x = x.double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1) if tall else x
    short, long = x.shape[-2:]
    err = 2 * U * torch.linalg.matrix_norm(x)
    for _ in range(steps):
        s = torch.linalg.matrix_norm(x, 2)
        grid = s[..., None] * torch.linspace(0, 1, 1001, dtype=torch.float64, device=x.device)
        slope = (a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().amax(-1)
        unit = 2.0 ** -21 + 4 * long ** 0.5 * U
        unit2 = 2.0 ** -21 + 4 * short ** 0.5 * U
        size = torch.linalg.matrix_norm(x)
        g = s ** 2
        add = (abs(b) * g * size * (unit + unit2) + abs(c) * g ** 2 * size * (2 * unit + 2 * unit2)
               + abs(a) * size * 2 * U)
        err = err * slope + add
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * gram @ gram) @ x
    err = err + 2 * U * torch.linalg.matrix_norm(x)
    return (x.transpose(-2, -1) if tall else x), err


def _matrices(*shape, seed=0, dtype=torch.float32, scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    r, c = shape[-2:]
    k = min(4, r, c)
    x = torch.randn(*shape, generator=g) + torch.randn(*shape[:-1], k, generator=g) @ torch.randn(
        *shape[:-2], k, c, generator=g)
    return (x * scale).to(dtype).to(DEV)


def _check(x, **kw):
    got = ops.orthogonalize(x, **kw)
    torch.cuda.synchronize()
    assert got.dtype == x.dtype and got.shape == x.shape and torch.isfinite(got).all()
    want, tol = _formula(x, **kw)
    if x.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * torch.linalg.matrix_norm(want)
    off = torch.linalg.matrix_norm(got.double() - want)
    assert (off <= tol).all(), f"{(off / tol).max().item():.3g} times the tolerance"


SHAPES = [(1, 1), (1, 7), (9, 1), (5, 5), (8, 33), (62, 62), (16, 299), (299, 16), (32, 3969), (64, 65), (65, 64),
          (96, 96), (127, 130), (128, 128), (130, 200), (200, 131), (256, 256), (257, 64), (513, 300), (300, 1025)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_orthogonalize(rows, cols, dtype):
    _check(_matrices(rows, cols, seed=rows + cols, dtype=dtype))


@pytest.mark.parametrize("shape", [(3, 62, 62), (2, 3, 20, 9), (5, 70, 200), (4, 200, 70), (3, 256, 256), (7, 1, 3)])
def test_batches(shape):
    _check(_matrices(*shape, seed=1))


@pytest.mark.parametrize("rows,cols", [(24, 40), (150, 90)])
def test_steps_and_coefficients(rows, cols):
    x = _matrices(rows, cols, seed=2)
    for steps in (0, 1, 2, 8):
        _check(x, steps=steps)
    got = ops.orthogonalize(x, steps=12, coefficients=(1.875, -1.25, 0.375))
    want, tol = _formula(x, 12, (1.875, -1.25, 0.375))
    assert torch.linalg.matrix_norm(got.double() - want) <= tol
    # the classic coefficients converge to orthonormal rows or columns
    o = got.double()
    gram = o @ o.T if rows < cols else o.T @ o
    assert torch.linalg.matrix_norm(torch.eye(gram.shape[0], device=DEV) - gram, 2) < 0.05


@pytest.mark.parametrize("rows,cols", [(30, 50), (140, 200)])
def test_scales_zero_and_non_finite_matrices(rows, cols):
    for scale in (1e-30, 1e-12, 1e12, 1e30):
        _check(_matrices(rows, cols, seed=3, scale=scale), eps=0.0)
    x = _matrices(4, rows, cols, seed=4)
    want = ops.orthogonalize(x)
    x[1] = 0
    x[2, 3, 4] = float("nan")
    x[3, 0, 0] = float("inf")
    got = ops.orthogonalize(x)
    assert torch.equal(got[0], want[0]) and (got[1] == 0).all()
    assert torch.isnan(got[2]).any() and not torch.isfinite(got[3]).all()


def test_strided_inputs():
    for rows, cols in ((30, 50), (140, 200)):
        x = _matrices(cols, 2 * rows, seed=5)
        want = ops.orthogonalize(x[:, ::2].t().contiguous())
        assert torch.equal(ops.orthogonalize(x[:, ::2].t()), want)
        for dtype in (torch.float32, torch.bfloat16):
            y = _matrices(rows, cols, seed=6, dtype=dtype)
            off = torch.empty(y.numel() + 1, dtype=dtype, device=DEV)[1:].view(y.shape).copy_(y)
            assert torch.equal(ops.orthogonalize(off), ops.orthogonalize(y))


def test_out_may_be_x():
    lib = _lib.load()
    for rows, cols in ((30, 50), (140, 200), (200, 140)):
        x = _matrices(rows, cols, seed=7)
        want = ops.orthogonalize(x)
        d = ops._newton_schulz_desc(x.shape, "float32", 5, COEFFS, 1e-7)
        ws = torch.empty(lib.nc_newton_schulz_workspace_bytes(ctypes.byref(d)), dtype=torch.uint8, device=DEV)
        _lib.check(lib.nc_orthogonalize(ctypes.byref(d), ops._ptr(x), ops._ptr(x), ops._ptr(ws), ws.numel(),
                                        ops._stream(DEV)), "nc_orthogonalize")
        assert torch.equal(x, want)


@pytest.mark.parametrize("shape", [(3, 62, 62), (16, 299), (257, 130), (3, 256, 256)])
@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_muon_steps(shape, nesterov, decay):
    lr, beta = 0.02, 0.9
    p, m = 100 * _matrices(*shape, seed=8), _matrices(*shape, seed=9)
    p64, m64, tol = p.double(), m.double(), 0.0
    scale = max(1.0, shape[-2] / shape[-1]) ** 0.5
    for step in range(2):
        g = _matrices(*shape, seed=10 + step)
        ops.muon_(p, g, m, lr, beta=beta, nesterov=nesterov, weight_decay=decay)
        m64 = beta * m64 + g.double()
        u64 = g.double() + beta * m64 if nesterov else m64
        o, err = _formula(u64)
        # u itself carries three roundings, which the whole iteration magnifies
        slopes = (COEFFS[0] + 0.5) ** 5
        p64 = p64 * (1 - lr * decay) - lr * scale * o
        tol = tol + lr * scale * (err + slopes * 4 * U) + 4 * U * torch.linalg.matrix_norm(p64)
    torch.cuda.synchronize()
    assert (torch.linalg.matrix_norm(p.double() - p64) <= tol).all()
    # each step rounds twice
    assert (torch.linalg.matrix_norm(m.double() - m64) <= 8 * U * torch.linalg.matrix_norm(m64)).all()


def test_same_bits_twice_on_another_stream_and_replayed():
    for shape in ((3, 62, 62), (32, 1000), (140, 260)):
        x = _matrices(*shape, seed=11)
        want = ops.orthogonalize(x)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            again = ops.orthogonalize(x)
        s.synchronize()
        assert torch.equal(want, again)
        p, m, g = _matrices(*shape, seed=12), torch.zeros_like(x), x.clone()
        graph = torch.cuda.CUDAGraph()
        ops.muon_(p.clone(), g, m.clone(), 0.1)
        with torch.cuda.graph(graph):
            ops.muon_(p, g, m, 0.1)
        p2, m2 = p.clone(), m.clone()
        for k in range(2):
            g.copy_(_matrices(*shape, seed=13 + k))
            graph.replay()
            ops.muon_(p2, g, m2, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(p, p2) and torch.equal(m, m2)


def test_empty_batches():
    assert ops.orthogonalize(torch.zeros(0, 4, 5, device=DEV)).shape == (0, 4, 5)
    z = torch.zeros(0, 4, 5, device=DEV)
    ops.muon_(z, z.clone(), z.clone(), 0.1)


def test_refusals():
    x = _matrices(6, 8)
    with pytest.raises(ValueError, match="expected"):
        ops.orthogonalize(x[0])
    with pytest.raises(ValueError, match="expected"):
        ops.orthogonalize(x.double())
    with pytest.raises(ValueError, match="steps"):
        ops.orthogonalize(x, steps=65)
    with pytest.raises(ValueError, match="eps"):
        ops.orthogonalize(x, eps=-1.0)
    with pytest.raises(ValueError, match="contiguous"):
        ops.muon_(x.t(), x.t(), x.t(), 0.1)
    with pytest.raises(ValueError, match="different buffers"):
        ops.muon_(x, x, x.clone(), 0.1)
    with pytest.raises(ValueError, match="float32"):
        ops.muon_(x.bfloat16(), x, x, 0.1)
    with pytest.raises(ValueError, match="shape"):
        ops.muon_(x, x[:5], x.clone(), 0.1)
    lib = _lib.load()
    d = ops._newton_schulz_desc(x.shape, "float32", 5, COEFFS, 1e-7)
    n = lib.nc_newton_schulz_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    assert lib.nc_orthogonalize(ctypes.byref(d), ops._ptr(x), ops._ptr(x), ops._ptr(ws), n - 1,
                                None) == _lib.NC_ERR_WORKSPACE


def test_calls_at_once_on_several_streams():
    xs = [_matrices(140, 260, seed=21), _matrices(3, 62, 62, seed=22), _matrices(700, 300, seed=23),
          _matrices(40, 70, 96, seed=24), _matrices(32, 2000, seed=25)]
    want = [ops.orthogonalize(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(5):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(ops.orthogonalize(x))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(xs)]), i


@pytest.mark.parametrize("batch,rows,cols,dtype", [(36_000, 62, 1000, torch.bfloat16), (64_000, 65, 520, torch.float32)])
def test_offsets_past_32_bits(batch, rows, cols, dtype):
    gen = torch.Generator(device=DEV).manual_seed(31)
    x = torch.empty(batch, rows, cols, dtype=dtype, device=DEV).normal_(generator=gen)
    got = ops.orthogonalize(x)
    torch.cuda.synchronize()
    for k in (0, batch // 2, batch - 1):
        want, tol = _formula(x[k])
        if dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * torch.linalg.matrix_norm(want)
        assert torch.linalg.matrix_norm(got[k].double() - want) <= tol, k


@pytest.mark.parametrize("rows,cols", [(96, 1000), (1000, 96), (100, 576), (70, 2000), (128, 1024), (384, 384), (300, 400), (96, 4000), (200, 1500)])
def test_several_tiles_of_a_cluster(rows, cols):
    # rows past the end leave some warps without work, which then run ahead of the others
    for batch in (1, 5):
        x = _matrices(batch, rows, cols, seed=39)
        want, tol = _formula(x)
        first = ops.orthogonalize(x)
        assert (torch.linalg.matrix_norm(first.double() - want) <= tol).all()
        for _ in range(20):
            assert torch.equal(ops.orthogonalize(x), first)


def test_a_batch_of_several_launches():
    p, g, m = (_matrices(8000, 70, 96, seed=k) for k in (35, 36, 37))
    p2, m2 = p.clone(), m.clone()
    ops.muon_(p, g, m, 0.1)
    for k in range(0, 8000, 3000):      # a launch's worth or less
        part = slice(k, min(8000, k + 3000))
        ops.muon_(p2[part], g[part], m2[part], 0.1)
    torch.cuda.synchronize()
    assert torch.equal(p, p2) and torch.equal(m, m2)


def test_autograd_sees_the_update():
    p = _matrices(6, 8).requires_grad_()
    m = torch.zeros_like(p)
    y = (p * p).sum()
    with torch.no_grad():
        ops.muon_(p, torch.ones_like(p), m, 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("shape", [(24, 40), (130, 200)])
def test_no_eps(shape):
    x = _matrices(2, *shape, seed=33)
    _check(x, eps=0.0)
    x[1] = 0
    got = ops.orthogonalize(x, eps=0.0)
    assert torch.isfinite(got[0]).all() and got[1].isnan().all()


def test_coefficients_that_diverge_show():
    got = ops.orthogonalize(_matrices(130, 200, seed=34), coefficients=(40.0, 0.0, 0.0))
    assert not torch.isfinite(got).all()
