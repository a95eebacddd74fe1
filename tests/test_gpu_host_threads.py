"""Calls from several host threads at once (ctypes lets go of the interpreter lock)."""
import ctypes
import threading

import pytest
import torch

from neurocell_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _at_once(calls, times):
    """Each of ``calls`` in a thread of its own; returns their statuses other than NC_OK."""
    bad, lib = [], _lib.load()
    start = threading.Barrier(len(calls))

    def work(call):
        start.wait()
        for _ in range(times):
            if call() != _lib.NC_OK:
                bad.append(lib.nc_last_error().decode())
                return

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return bad


def _readout(rows, dim, classes, grad, stream):
    lib = _lib.load()
    g = torch.Generator().manual_seed(dim)
    f, w = torch.randn(rows, dim, generator=g).to(DEV), torch.randn(classes, dim, generator=g).to(DEV)
    lab = torch.zeros(rows, dtype=torch.int32, device=DEV)
    d = _lib.NcLinearCe(rows, dim, classes, 0, -100, 0)
    n = lib.nc_linear_ce_workspace_bytes(ctypes.byref(d), int(grad))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    loss, lse, gf, gw = torch.empty((), device=DEV), torch.empty(rows, device=DEV), torch.empty_like(f), torch.empty_like(w)
    s = ctypes.c_void_p(stream.cuda_stream)
    P = ops._ptr

    def call(keep=(f, w, lab, ws, lse)):
        if grad:
            return lib.nc_linear_ce_value_and_grad(ctypes.byref(d), P(f), P(w), None, P(lab), P(loss), P(lse), P(gf),
                                                   P(gw), None, P(ws), n, s)
        return lib.nc_linear_ce_forward(ctypes.byref(d), P(f), P(w), None, P(lab), P(loss), P(lse), P(ws), n, s)

    call.outputs = [loss, gf, gw] if grad else [loss]
    return call


def _orthogonalize(rows, cols, stream):
    lib = _lib.load()
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(cols)).to(DEV)
    out = torch.empty_like(x)
    d = ops._newton_schulz_desc(x.shape, "float32", 5, ops.NEWTON_SCHULZ_COEFFICIENTS, 1e-7)
    n = lib.nc_newton_schulz_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    s = ctypes.c_void_p(stream.cuda_stream)
    P = ops._ptr

    def call(keep=(x, ws)):
        return lib.nc_orthogonalize(ctypes.byref(d), P(x), P(out), P(ws), n, s)

    call.outputs = [out]
    return call


@pytest.mark.parametrize("kind", ["value", "gradients", "orthogonalize"])
def test_sizes_of_one_kernel_from_two_threads(kind):
    """Two sizes that take one kernel with different amounts of shared memory."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    if kind == "orthogonalize":
        calls = [_orthogonalize(62, 62, streams[0]), _orthogonalize(64, 4000, streams[1])]
    else:
        calls = [_readout(8, dim, 3000, kind == "gradients", s) for dim, s in zip((520, 1024), streams)]
    torch.cuda.synchronize()
    want = []
    for c in calls:
        assert c() == _lib.NC_OK
        torch.cuda.synchronize()
        want.append([t.clone() for t in c.outputs])
    assert _at_once(calls, 4000) == []
    for c, w in zip(calls, want):
        assert all(torch.equal(x, y) for x, y in zip(c.outputs, w))
