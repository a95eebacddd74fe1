"""Refusals of the readout loss on the host (no GPU): sizes, types, devices."""
import ctypes

import pytest
import torch

from neurocell_b200 import _lib, ops


def _bytes(rows=4, dim=8, classes=16, dtype=0, ignore=-100, reduction=0, grad=0):
    d = _lib.NcLinearCe(rows, dim, classes, dtype, ignore, reduction)
    return _lib.load().nc_linear_ce_workspace_bytes(ctypes.byref(d), grad)


def test_descriptors_are_checked():
    assert _bytes() > 0 and _bytes(grad=1) > 0 and _bytes(rows=0) > 0
    for bad in (dict(rows=-1), dict(dim=0), dict(classes=0), dict(dtype=7), dict(reduction=3), dict(ignore=3)):
        assert _bytes(**bad) == 0, bad
    assert _lib.load().nc_linear_ce_workspace_bytes(None, 0) == 0


def test_c_entry_refuses_before_any_device_work():
    lib = _lib.load()
    d = _lib.NcLinearCe(4, 8, 16, 0, -100, 0)
    one = ctypes.c_void_p(256)
    assert lib.nc_linear_ce_forward(None, one, one, one, one, one, one, one, 1 << 20, None) == _lib.NC_ERR_INVALID
    assert lib.nc_linear_ce_forward(ctypes.byref(d), None, one, one, one, one, one, one, 1 << 20,
                                    None) == _lib.NC_ERR_INVALID
    assert lib.nc_linear_ce_forward(ctypes.byref(d), ctypes.c_void_p(258), one, one, one, one, one, one, 1 << 20,
                                    None) == _lib.NC_ERR_INVALID
    assert lib.nc_linear_ce_forward(ctypes.byref(d), one, one, one, one, one, one, one, 0,
                                    None) == _lib.NC_ERR_WORKSPACE
    assert lib.nc_linear_ce_backward(ctypes.byref(d), one, one, one, one, one, None, one, one, one, one, 16,
                                     None) == _lib.NC_ERR_WORKSPACE


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="no CPU path"):
        ops.linear_softmax_ce_loss(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="no CPU path"):
        ops.linear_softmax_ce_value_and_grad(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64))


class _Fake(torch.Tensor):
    """A host tensor that says it is on a GPU, for the checks that come before any launch."""
    is_cuda = True


def _fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Fake)


@pytest.mark.parametrize("change,match", [
    (dict(features=_fake(2, 5)), "expected"),
    (dict(features=_fake(6)), "expected"),
    (dict(labels=_fake(3, dtype=torch.int64)), "labels"),
    (dict(labels=_fake(2)), "int32 or int64"),
    (dict(weight=_fake(4, 3, dtype=torch.bfloat16)), "weight is"),
    (dict(bias=_fake(5)), "bias"),
    (dict(bias=_fake(4, dtype=torch.float64)), "bias is"),
    (dict(features=_fake(2, 3, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(reduction="max"), "reduction"),
])
def test_arguments_are_checked(change, match):
    args = dict(features=_fake(2, 3), weight=_fake(4, 3), labels=_fake(2, dtype=torch.int64), bias=None,
                ignore_index=-100, reduction="mean")
    args.update(change)
    with pytest.raises(ValueError, match=match):
        ops._linear_ce_args(args["features"], args["weight"], args["labels"], args["bias"], args["ignore_index"],
                            args["reduction"])


def test_sizes_past_the_tile_counts_are_refused():
    most = 1 << 24
    assert _bytes(rows=most, dim=1, classes=1) > 0 and _bytes(rows=1, dim=1, classes=most, grad=1) > 0
    for bad in (dict(rows=most + 1), dict(dim=most + 1), dict(classes=2 ** 31 - 1), dict(rows=2 ** 31 - 1),
                dict(rows=most, classes=1 << 21), dict(rows=most, dim=1 << 15), dict(classes=most, dim=1 << 15)):
        for grad in (0, 1):
            assert _bytes(grad=grad, **bad) == 0, bad
    assert b"too large" in _lib.load().nc_last_error()


def test_overlapping_buffers_are_refused():
    lib = _lib.load()
    d = _lib.NcLinearCe(4, 8, 16, 0, -100, 0)
    n = lib.nc_linear_ce_workspace_bytes(ctypes.byref(d), 1)
    step = 1 << 20
    names = ["f", "w", "b", "lab", "loss", "lse", "gl", "gf", "gw", "gb", "ws"]
    assert n < step

    def call(which, **change):
        p = {k: ctypes.c_void_p(step * (i + 1)) for i, k in enumerate(names)}
        p.update({k: ctypes.c_void_p(v) for k, v in change.items()})
        if which == "forward":
            return lib.nc_linear_ce_forward(ctypes.byref(d), p["f"], p["w"], p["b"], p["lab"], p["loss"], p["lse"],
                                            p["ws"], n, None)
        if which == "backward":
            return lib.nc_linear_ce_backward(ctypes.byref(d), p["f"], p["w"], p["b"], p["lab"], p["lse"], p["gl"],
                                             p["gf"], p["gw"], p["gb"], p["ws"], n, None)
        return lib.nc_linear_ce_value_and_grad(ctypes.byref(d), p["f"], p["w"], p["b"], p["lab"], p["loss"],
                                               p["lse"], p["gf"], p["gw"], p["gb"], p["ws"], n, None)

    at = {k: step * (i + 1) for i, k in enumerate(names)}
    for which, change in (("forward", dict(loss=at["lse"] + 12)), ("forward", dict(lse=at["f"] + 124)),
                          ("forward", dict(ws=at["w"])), ("backward", dict(gw=at["w"])),
                          ("backward", dict(gf=at["f"] + 4)), ("backward", dict(gb=at["gw"] + 508)),
                          ("backward", dict(gf=at["gl"])), ("backward", dict(lse=at["ws"] + 8)),
                          ("both", dict(gw=at["w"] - 4)), ("both", dict(loss=at["lab"])),
                          ("both", dict(gf=at["gw"] + 4))):
        assert call(which, **change) == _lib.NC_ERR_INVALID, (which, change)
        assert b"overlap" in lib.nc_last_error()


@pytest.mark.parametrize("ignore", [2 ** 32 - 100, -2 ** 31, 2 ** 31 - 1, -2 ** 40])
def test_ignore_index_has_to_fit(ignore):
    with pytest.raises(ValueError, match="32 bits"):
        ops._linear_ce_args(_fake(2, 3), _fake(4, 3), _fake(2, dtype=torch.int64), None, ignore, "mean")


def test_sizes_past_32_bits_are_refused():
    wide = torch.zeros(1, 1).expand(2 ** 32 + 2, 1).as_subclass(_Fake)
    with pytest.raises(ValueError, match="32 bits"):
        ops._linear_ce_args(_fake(2, 1), wide, _fake(2, dtype=torch.int64), None, -100, "mean")
