"""nc_ext_adamw8: what one element of a block of 256 does to the others, and which lists of parameters it takes."""

from __future__ import annotations

import numpy as np
import pytest

from nchelp import Eng, capi
from test_gpu_adamw8 import BLOCK, F, Emulated, give, opts, optimizer, same_bits, state, through_codes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("big", [7e20, -1e21, 3e38])
def test_a_finite_gradient_leaves_its_block_finite(big):
    """The square of a gradient above about 6e20 is beyond fp32: v is held as the largest finite float, so that the
    other 255 elements keep finite moments and weights. A gradient of infinity still makes its block not finite."""
    rng = np.random.default_rng(1)
    n = 3 * BLOCK + 40
    w = rng.standard_normal(n).astype(F)
    top = np.finfo(F).max
    m, v = np.zeros(n, F), np.zeros(n, F)
    with Eng("b200") as e:
        t = e.param(w)
        o = optimizer(e, [t], opts(decay=0.0))
        for k in range(4):
            g = rng.standard_normal(n).astype(F)
            g[BLOCK:BLOCK + 8] = 0
            g[BLOCK + 9] = big
            if k == 0:
                g[-1] = np.inf
            before = e.np(t)
            give(e, [t], [g])
            e.L.nc_optim_step(o)
            got = state(e, o, n)
            with np.errstate(all="ignore"):
                m = F(0.9) * m + (F(1) - F(0.9)) * g
                v = F(0.999) * v + ((F(1) - F(0.999)) * g) * g
            v = np.where(np.isinf(v) & np.isfinite(g), top, v)
            m, v = through_codes(m, v)
            ok = slice(0, 3 * BLOCK)
            assert np.isfinite(got[:, ok]).all(), k
            assert same_bits(got[0][ok], m[ok]) and same_bits(got[1][ok], v[ok]), k
            assert got[1][BLOCK + 9] == top
            assert np.isfinite(e.np(t)[ok]).all()
            assert not np.isfinite(got[0][3 * BLOCK:]).any() and not np.isfinite(got[1][3 * BLOCK:]).any()
            if k == 0:  # the step divides by the moment before it is held: an infinite one moves nothing
                assert e.np(t)[BLOCK + 9] == before[BLOCK + 9]
        e.L.nc_optim_free(o)


def test_a_parameter_is_taken_once():
    """The same parameter twice would be stepped by two blocks at once: refused, and nothing is changed."""
    with Eng("b200") as e:
        a, b = e.param(np.ones(300, F)), e.param(np.ones(5, F))
        give(e, [a, b], [np.full(300, 2, F), np.full(5, 3, F)])
        for ts in ([a, a], [a, b, a]):
            assert not e.L.nc_ext_adamw8(e.ctx, capi.ptr_array(ts), len(ts), opts()) and "twice" in e.err()
            e.L.nc_clear_error(e.ctx)
        assert np.array_equal(e.grad(a), np.full(300, 2, F)) and np.array_equal(e.grad(b), np.full(5, 3, F))
        o = optimizer(e, [a, b])
        e.L.nc_optim_step(o)
        assert e.ok() and (e.np(a) < 1).all() and (e.np(b) < 1).all()
        e.L.nc_optim_free(o)


def test_a_parameter_of_another_context_is_refused():
    with Eng("b200") as e, Eng("b200") as other:
        a, b = e.param(np.ones(300, F)), other.param(np.ones(300, F))
        assert not e.L.nc_ext_adamw8(e.ctx, capi.ptr_array([a, b]), 2, opts()) and "another context" in e.err()
        e.L.nc_clear_error(e.ctx)
        give(other, [b], [np.full(300, 2, F)])
        o = optimizer(other, [b])
        other.L.nc_optim_step(o)
        assert e.ok() and other.ok() and (other.np(b) < 1).all() and e.grad(a) is None
        other.L.nc_optim_free(o)
