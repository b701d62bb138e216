"""Weight gradients of nc_ext_qk_norm_rope over very many rows. Every row's term is the same number c, so an fp32 sum
carried from row to row rounds in one direction: with c = 1 + (2^(k-1) - 1) 2^-23 nearly half a step is lost at every
addition while the sum lies in [2^k, 2^(k+1)), in all about 2^k e / 2 of it (e = 2^-24). Bound: a term is off by 24 e
(the rows' norms are exact powers of two here, less in truth); an fp32 sum has at most 64 + 2 terms, so 66 roundings of
at most e of its own size; what is above that is in 64 bits, with one rounding a block and one of the result. So
(24 + 66 + 2) e, whatever the number of rows.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.mark.parametrize("k", [7, 8, 9, 10])
@pytest.mark.parametrize("T,H,q_heads,D,flags", [
    (80000, 1500, 1000, 2, 0),                       # a lane a row
    (80000, 1500, 1000, 2, capi.ROPE_INTERLEAVED),
    (2500, 1400, 1000, 256, 0),                      # a warp a row, in vectors
    (11000, 1300, 1300, 64, capi.ROPE_INTERLEAVED),  # 8 lanes a row, query heads only
    (90, 20000, 7000, 64, 0),                        # few tokens: heads in runs
], ids=str)
def test_sums_do_not_lose_with_rows(T, H, q_heads, D, flags, k):
    c = 1 + (2 ** (k - 1) - 1) * 2.0 ** -23
    with Eng("b200") as e:
        shape = (1, T, H, D)
        make = lambda f: e.check(e.L.nc_full(e.ctx, f, *capi.shape_arg(shape)))  # noqa: E731
        x, dy = make(1.0), make(c)
        wq, wk = e.param(np.ones(D, np.float32)), e.param(np.ones(D, np.float32))
        o = capi.RopeOpts(q_heads, 1, (ctypes.c_int * 3)(0), 10000.0, 0.0, flags)
        y = e.check(e.L.nc_ext_qk_norm_rope(x, wq, wk, None, ctypes.byref(o)))
        assert e.L.nc_ext_backward_from(y, dy) == 0, e.err()
        for w, heads in ((wq, q_heads), (wk, H - q_heads)):
            want = T * heads * c
            off = abs(e.grad(w).astype(np.float64) - want)
            assert np.all(off <= 92 * E * want), (off.max() / (E * max(want, 1)), heads)
        assert e.ok(), e.err()
