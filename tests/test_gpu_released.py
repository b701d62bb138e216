"""Tensors whose memory was given back (nc_release_temp, a backward pass that frees its graph, a view of either) are
refused by the operators for tuning and their helpers before anything is launched."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi, seeded

pytestmark = pytest.mark.gpu
FREE_GRAPH, STATE = 1, 5


def refused(e, result, text="released"):
    assert not result and not e.ok() and text in e.err(), e.err()
    e.L.nc_clear_error(e.ctx)


def gone(e, arr, how):
    """a tensor of arr whose memory was given back"""
    t = e.t(arr)
    if how == "view":
        v = e.check(e.L.nc_slice(t, 0, 0, arr.shape[0], 1))
        e.L.nc_release_temp(t)
        return v
    e.L.nc_release_temp(t)
    return t


@pytest.mark.parametrize("how", ["temporary", "view"])
def test_released_inputs(how):
    F, I = np.float32, np.int32
    z, lab, row = seeded(1, (4, 3, 7)), np.zeros((4, 3), I), seeded(2, (4, 3))
    x, w, pos = seeded(3, (2, 3, 4, 8)), seeded(4, (8,)), np.zeros((3, 1), I)
    policy, rope = capi.PolicyOpts(0.2, 0.2, 0.1), capi.RopeOpts(2, 1, (ctypes.c_int * 3)(4), 10000.0, 1e-6, 0)
    with Eng("b200") as e:
        L = e.L
        for k in range(6):
            args = [z, lab, row, row, row, np.ones((4, 3), np.uint8 if k % 2 else I)]
            args = [gone(e, a, how) if i == k else e.t(a) for i, a in enumerate(args)]
            refused(e, L.nc_ext_policy_loss(*args, ctypes.byref(policy), None))
        for k in range(4):
            args = [gone(e, a, how) if i == k else e.t(a) for i, a in enumerate([z, lab, np.zeros(4, F), np.ones((4, 3), I)])]
            refused(e, L.nc_ext_preference_loss(*args, 0.1, 0.0, None))
        for k in range(4):
            args = [gone(e, a, how) if i == k else e.t(a) for i, a in enumerate([x, w, w, pos])]
            refused(e, L.nc_ext_qk_norm_rope(*args, ctypes.byref(rope)))
        p = e.param(w)
        assert L.nc_ext_backward_from(p, gone(e, w, how)) == STATE and "released" in e.err()
        L.nc_clear_error(e.ctx)
        assert e.grad(p) is None
        o = e.check(L.nc_ext_adamw8(e.ctx, capi.ptr_array([p]), 1, capi.OptimOpts(1e-3, 0.0, 0.0, 0.9, 0.999, 1e-8)))
        for call in (L.nc_ext_optim_get_state, L.nc_ext_optim_put_state):
            assert call(o, gone(e, np.zeros((2, 8), F), how)) == STATE and "released" in e.err()
            L.nc_clear_error(e.ctx)
        assert not L.nc_ext_device_data(gone(e, w, how), 0)
        L.nc_optim_free(o)
        assert e.ok(), e.err()


def test_after_a_pass_that_freed_its_graph():
    with Eng("b200") as e:
        x = e.param(seeded(1, (6, 9)))
        z = e.check(e.L.nc_tanh(x))
        o = capi.PolicyOpts(0.2, 0.2, 0.0)
        fixed = [e.t(np.zeros(6, np.int32)), e.t(np.full(6, -2, np.float32)), None, e.t(np.ones(6, np.float32)), None]
        loss = e.check(e.L.nc_ext_policy_loss(z, *fixed, ctypes.byref(o), None))
        assert e.L.nc_backward_ex(loss, FREE_GRAPH, None, 0) == 0, e.err()
        first = e.grad(x)
        refused(e, e.L.nc_ext_policy_loss(z, *fixed, ctypes.byref(o), None))
        again = e.check(e.L.nc_ext_policy_loss(e.check(e.L.nc_tanh(x)), *fixed, ctypes.byref(o), None))
        e.L.nc_clear_grad(x)
        assert e.L.nc_backward(again) == 0 and np.array_equal(e.grad(x), first)
