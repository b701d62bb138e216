"""Floats written through nc_optim_state's pointer reach the next step, also when nc_ext_optim_get_state was called
between taking the pointer and writing."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi, seeded

pytestmark = pytest.mark.gpu
SHAPES = [(300,), (7, 40)]


@pytest.mark.parametrize("make", ["nc_adamw", "nc_adam", "nc_ext_adamw8"])
@pytest.mark.parametrize("slot", [0, 1])
def test_writes_behind_a_state_copy_reach_the_step(make, slot):
    ws = [seeded(i, s) for i, s in enumerate(SHAPES)]
    n = sum(w.size for w in ws)

    def run(copies):
        with Eng("b200") as e:
            ts = [e.param(w) for w in ws]
            o = e.check(getattr(e.L, make)(e.ctx, capi.ptr_array(ts), 2, capi.OptimOpts(1e-2, 0.0, 0.01, 0.9, 0.999, 1e-8)))
            values = e.t(np.zeros((2, n), np.float32), persistent=True)
            got = []
            for k in range(2):
                for t, s in zip(ts, SHAPES):
                    e.L.nc_clear_grad(t)
                    assert e.L.nc_ext_backward_from(t, e.t(seeded(10 + k, s))) == 0, e.err()
                if k:
                    p = ctypes.cast(e.check(e.L.nc_optim_state(o, 1, slot)), ctypes.POINTER(ctypes.c_float))
                    state = np.ctypeslib.as_array(p, (ws[1].size,))
                    for c in range(3):
                        if copies:
                            assert e.L.nc_ext_optim_get_state(o, values) == 0, e.err()
                        state[5 + c] = 2.0 + c
                e.L.nc_optim_step(o)
            assert e.L.nc_ext_optim_get_state(o, values) == 0, e.err()
            got = [e.np(values)] + [e.np(t) for t in ts]
            assert e.ok(), e.err()
            e.L.nc_optim_free(o)
            return got

    want, got = run(False), run(True)
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    at = ws[0].size + 5  # the written floats are there: 0.9 or 0.999 of 2, 3, 4 and a little
    assert np.all(np.abs(got[0][slot, at:at + 3] - np.array([2, 3, 4])) < 1)


@pytest.mark.parametrize("make", ["nc_adamw", "nc_ext_adamw8"])
def test_a_copy_shows_what_was_written(make):
    """What a copy shows between writes, and that the state put back is what the next step starts from."""
    with Eng("b200") as e:
        t = e.param(seeded(1, (256,)))
        o = e.check(getattr(e.L, make)(e.ctx, capi.ptr_array([t]), 1, capi.OptimOpts(1e-2, 0.0, 0.0, 0.9, 0.999, 1e-8)))
        values = e.t(np.zeros((2, 256), np.float32), persistent=True)
        p = ctypes.cast(e.check(e.L.nc_optim_state(o, 0, 0)), ctypes.POINTER(ctypes.c_float))
        for x in (4.0, 8.0):  # the largest of its block is held as it is in 8 bits too
            p[3] = x
            assert e.L.nc_ext_optim_get_state(o, values) == 0
            assert e.np(values)[0, 3] == x
        put = np.zeros((2, 256), np.float32)
        put[0, 9] = 16.0
        assert e.L.nc_ext_optim_put_state(o, e.t(put)) == 0, e.err()
        assert e.L.nc_ext_optim_get_state(o, values) == 0
        assert np.array_equal(e.np(values), put)
        assert e.L.nc_ext_backward_from(t, e.t(np.zeros(256, np.float32))) == 0
        e.L.nc_optim_step(o)
        assert e.L.nc_ext_optim_get_state(o, values) == 0
        assert np.array_equal(e.np(values), put * np.float32(0.9))
        e.L.nc_optim_free(o)
