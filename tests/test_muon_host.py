"""Refusals of the orthogonalisation and of the update by orthogonalised momentum on the
host (no GPU)."""
import ctypes

import pytest
import torch

from neurocell_b200 import _lib, ops


def _bytes(batch=1, rows=4, cols=8, dtype=0, steps=5, eps=1e-7):
    d = _lib.NcNewtonSchulz(batch, rows, cols, dtype, steps, 3.4445, -4.775, 2.0315, eps)
    return _lib.load().nc_newton_schulz_workspace_bytes(ctypes.byref(d))


def test_descriptors_are_checked():
    assert _bytes() > 0 and _bytes(batch=0) > 0 and _bytes(dtype=1) > 0
    for bad in (dict(batch=-1), dict(rows=0), dict(cols=0), dict(dtype=2), dict(steps=-1), dict(steps=65),
                dict(eps=-1.0), dict(eps=float("nan")), dict(batch=65536), dict(rows=1 << 16, cols=1 << 15)):
        assert _bytes(**bad) == 0, bad


def test_c_entries_refuse_before_any_device_work():
    lib = _lib.load()
    d = _lib.NcNewtonSchulz(1, 4, 8, 0, 5, 3.4445, -4.775, 2.0315, 1e-7)
    one, two, three = ctypes.c_void_p(256), ctypes.c_void_p(512), ctypes.c_void_p(768)
    r = ctypes.byref(d)
    assert lib.nc_orthogonalize(None, one, two, one, 1 << 20, None) == _lib.NC_ERR_INVALID
    assert lib.nc_orthogonalize(r, None, two, one, 1 << 20, None) == _lib.NC_ERR_INVALID
    assert lib.nc_orthogonalize(r, ctypes.c_void_p(258), two, one, 1 << 20, None) == _lib.NC_ERR_INVALID
    assert lib.nc_orthogonalize(r, one, two, one, 8, None) == _lib.NC_ERR_WORKSPACE
    assert lib.nc_muon_update(r, one, two, two, 0.1, 0.9, 1, 0.0, one, 1 << 20, None) == _lib.NC_ERR_INVALID
    assert lib.nc_muon_update(r, one, two, three, 0.1, 0.9, 1, 0.0, None, 1 << 20, None) == _lib.NC_ERR_WORKSPACE
    d.dtype = 1
    assert lib.nc_muon_update(r, one, two, three, 0.1, 0.9, 1, 0.0, one, 1 << 20, None) == _lib.NC_ERR_INVALID


def test_host_tensors_are_refused():
    x = torch.zeros(4, 5)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.orthogonalize(x)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.muon_(x, x.clone(), x.clone(), 0.1)


def test_sizes_past_the_limits_are_refused():
    assert _bytes(rows=1, cols=1 << 30) > 0 and _bytes(rows=1 << 15, cols=1 << 15) > 0
    assert _bytes(rows=1, cols=(1 << 30) + 1) == 0 and _bytes(rows=2 ** 31 - 1, cols=1) == 0
    for shape, steps in (((2 ** 32 + 1, 4, 4), 5), ((4, 2 ** 32 + 1), 5), ((4, 4), 2 ** 32 + 5), ((4, 4), -2 ** 32)):
        with pytest.raises(ValueError, match="32 bits"):
            ops._newton_schulz_desc(shape, "float32", steps, ops.NEWTON_SCHULZ_COEFFICIENTS, 1e-7)


def test_overlapping_buffers_are_refused():
    lib = _lib.load()
    d = _lib.NcNewtonSchulz(2, 4, 8, 0, 5, 3.4445, -4.775, 2.0315, 1e-7)     # 256 bytes
    r, n = ctypes.byref(d), _bytes(batch=2)
    x, ws, P = 1 << 20, 1 << 22, ctypes.c_void_p
    for out, w in ((x + 4, ws), (x - 252, ws), (x + 512, x), (ws, ws)):
        assert lib.nc_orthogonalize(r, P(x), P(out), P(w), n, None) == _lib.NC_ERR_INVALID, (out, w)
        assert b"overlap" in lib.nc_last_error()
    for p, g, m, w in ((x, x + 252, x + 512, ws), (x, x + 512, x + 252, ws), (x, x + 512, x + 764, ws),
                       (x, x + 512, x + 1024, x + 512)):
        assert lib.nc_muon_update(r, P(p), P(g), P(m), 0.1, 0.9, 1, 0.0, P(w), n, None) == _lib.NC_ERR_INVALID


def test_workspaces_of_large_batches_stay_small():
    # a launch's matrices share it: past a few thousand the batch does not count
    assert _bytes(batch=65535, rows=65, cols=520) == _bytes(batch=8000, rows=65, cols=520) < 2 ** 31
