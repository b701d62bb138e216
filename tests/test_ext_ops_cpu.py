"""The side API's operators without a GPU: struct layouts as the header declares them, and calls that have to come
back without touching a device (NULL inputs; a context that found no device refuses)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

from nchelp import capi

HEADER = (Path(__file__).resolve().parent.parent / "include" / "nc_ext.h").read_text()
C_TYPES = {"int": ctypes.c_int, "float": ctypes.c_float}


@pytest.mark.parametrize("name,cls", [("nc_ext_rope_opts", capi.RopeOpts), ("nc_ext_policy_opts", capi.PolicyOpts)])
def test_struct_matches_header(name, cls):
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", HEADER).group(1)
    want = []
    for kind, field, count in re.findall(r"(int|float)\s+(\w+)(?:\[(\d+)\])?;", body):
        want.append((field, C_TYPES[kind] * int(count) if count else C_TYPES[kind]))
    assert [(n, ctypes.sizeof(t)) for n, t in cls._fields_] == [(n, ctypes.sizeof(t)) for n, t in want]


def test_flags_match_header():
    for name, value in (("INTERLEAVED", capi.ROPE_INTERLEAVED), ("AXIS_FREQ", capi.ROPE_AXIS_FREQ), ("NO_NORM", capi.ROPE_NO_NORM)):
        assert re.search(rf"NC_EXT_ROPE_{name} = {value}\b", HEADER)


def test_null_inputs_come_back():
    L = capi.load_b200()
    more = ctypes.c_void_p(1)
    assert L.nc_ext_qk_norm_rope(None, None, None, None, None) is None
    assert L.nc_ext_policy_loss(None, None, None, None, None, None, None, ctypes.byref(more)) is None and not more.value
    more = ctypes.c_void_p(1)
    assert L.nc_ext_preference_loss(None, None, None, None, 0.1, 0.0, ctypes.byref(more)) is None and not more.value
    assert L.nc_ext_device_data(None, 1) is None
    assert L.nc_ext_backward_from(None, None) == 4
    assert L.nc_ext_optim_get_state(None, None) == 4 and L.nc_ext_optim_put_state(None, None) == 4
    assert L.nc_ext_adamw8(None, None, 0, capi.OptimOpts()) is None


def test_context_without_a_device_refuses():
    L = capi.load_b200()
    if L.nc_ext_device_count() > 0:
        pytest.skip("a device is visible")
    ctx = L.nc_init(ctypes.byref(capi.Config(0, 1, 0, 0)))
    try:
        for _ in range(2):
            assert L.nc_ext_adamw8(ctx, None, 0, capi.OptimOpts()) is None
            assert not L.nc_ok(ctx)
            L.nc_clear_error(ctx)
    finally:
        L.nc_free_ctx(ctx)
