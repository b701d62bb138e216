"""The losses at the borders between their kernels' ways of dealing with rows (lanes, warps, blocks, parts of rows), no
rows at all, and gradients added to what is there, by each way. Bounds as in test_gpu_policy.py."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi
from test_gpu_policy import make, policy, preference, run_policy

pytestmark = pytest.mark.gpu

SIZES = [(70, 4), (70, 5), (33, 8), (33, 9), (9, 16), (9, 17), (65, 32), (65, 33), (40, 64), (40, 65), (7, 128), (7, 129), (9, 255),
         (9, 256), (9, 257), (5, 512), (5, 513), (5, 900), (3, 2048), (3, 2049), (1100, 4099), (1023, 2051), (3, 12289),
         (2, 65535), (7, 65537), (1, 200003), (297, 65536), (400, 80003)]


@pytest.mark.parametrize("N,V", SIZES)
def test_borders(N, V):
    z, act, old, ref, adv = make(N + V, (N,), V)
    mask = (np.random.default_rng(N).random(N) < 0.8).astype(np.int32)
    loss, lp, dz, dl, off, T = policy(z, act, old, ref, adv, mask, 0.2, 0.25, 0.1)
    with Eng("b200") as e:
        tz = e.param(z)
        for k in (1, 2):  # the second pass adds to the first's gradient
            _, tl, more = run_policy(e, z, act, old, ref, adv, mask, tz=tz)
            assert e.L.nc_backward(tl) == 0, e.err()
            assert abs(float(e.np(tl)) - loss) <= dl
            assert np.all(abs(e.np(more) - lp) <= T + abs(lp) * 2.0 ** -24 + 1e-30)
            g = e.grad(tz)
            assert np.all(abs(g - k * dz) <= k * off + k * abs(dz) * 2.0 ** -23)
            assert not g[mask == 0].any()
        assert e.ok(), e.err()


@pytest.mark.parametrize("V", [3, 700, 3000, 70000])
def test_no_rows(V):
    f = np.zeros(0, np.float32)
    with Eng("b200") as e:
        tz, tl, more = run_policy(e, np.zeros((0, V), np.float32), f.astype(np.int32), f, f, f, None)
        assert e.L.nc_backward(tl) == 0, e.err()
        assert float(e.np(tl)) == 0.0 and e.np(more).shape == (0,) and e.grad(tz).shape == (0, V)
        tz = e.param(np.zeros((2, 0, V), np.float32))
        lab = e.t(np.zeros((2, 0), np.int32))
        tl = e.check(e.L.nc_ext_preference_loss(tz, lab, None, None, 0.1, 0.0, None))
        assert e.L.nc_backward(tl) == 0 and abs(float(e.np(tl)) - np.log(2)) < 1e-6 and e.ok(), e.err()


@pytest.mark.parametrize("T,V", [(300, 3), (7, 300), (5, 800), (3, 9000), (2, 70001)])
def test_preference_adds_to_a_gradient(T, V):
    rng = np.random.default_rng(T)
    z = rng.standard_normal((4, T, V)).astype(np.float32)
    lab = rng.integers(0, V, (4, T)).astype(np.int32)
    ref = preference(z, lab, None, None, 0.1, 0)[1].astype(np.float32)
    _, _, dz, _, _, off = preference(z, lab, ref, None, 0.1, 0.0)
    with Eng("b200") as e:
        tz = e.param(z)
        for k in (1, 2):
            tl = e.check(e.L.nc_ext_preference_loss(tz, e.t(lab), e.t(ref), None, 0.1, 0.0, None))
            assert e.L.nc_backward(tl) == 0, e.err()
            assert np.all(abs(e.grad(tz) - k * dz) <= k * off + k * abs(dz) * 2.0 ** -23)


def test_long_answers_keep_their_sums():
    """40000 tokens: an error of 1e-7 in the mean of a token's log probability would show as 4e-3 in a sum. The bound
    takes 4e-9 in the mean and 3e-7 of random error a token (6 standard errors of the sum)."""
    T, V = 40000, 96
    rng = np.random.default_rng(5)
    z = (rng.standard_normal((2, T, V)) * 2).astype(np.float32)
    lab = rng.integers(0, V, (2, T)).astype(np.int32)
    seq = preference(z, lab, None, None, 0.1, 0)[1]
    with Eng("b200") as e:
        more = ctypes.c_void_p()
        e.check(e.L.nc_ext_preference_loss(e.t(z), e.t(lab), None, None, 0.1, 0.0, ctypes.byref(more)))
        got = e.np(more.value)
    bound = 4e-9 * T + 6 * 3e-7 * np.sqrt(T) + 2.0 ** -24 * abs(seq)
    assert np.all(abs(got - seq) <= bound), (got - seq, bound)
