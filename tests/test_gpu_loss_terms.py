"""Terms of the policy and preference losses where a part of the formula is very small, or infinite.

Logits that are equal along a row have log probability -log V, which the kernels form from an exact sum in 64 bits
(the maximum is exact, V is below 2^24): so a row's KL term e^away - away - 1, away = ref - lp, is known to the
precision of its own arithmetic, down to the smallest away that an fp32 ref can be away from it. Bounds: lp is off by
two steps of 64 bits (4e-16 |lp|, at most 1e-14 here), away by 1.1e-14, the term (about away^2 / 2, slope e^away - 1) by
1.1e-14 |e^away - 1| and one rounding to fp32 for the term, kl's product and the loss each: 4 e, e = 2^-24.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
F = np.float32


def kl_term(away):
    """e^away - away - 1 in 64 bits, for any away"""
    if abs(away) < 0.1:
        term, total = away * away / 2, 0.0
        for k in range(3, 20):
            total, term = total + term, term * away / k
        return total
    return np.expm1(away) - away


def policy(e, z, act, old, ref, adv, kl):
    tz = e.param(z)
    loss = e.check(e.L.nc_ext_policy_loss(tz, e.t(act), e.t(old), None if ref is None else e.t(ref), e.t(adv), None,
                                          ctypes.byref(capi.PolicyOpts(0.2, 0.25, kl)), None))
    assert e.L.nc_backward(loss) == 0, e.err()
    return float(e.np(loss)), e.grad(tz)


@pytest.mark.parametrize("V", [1, 2, 61, 1000, 2000, 20000, 70000])  # every way the rows are read
def test_kl_term_of_a_policy_near_its_reference(V):
    lp = -np.log(float(V))
    with Eng("b200") as e:
        for d in (0.0, 1e-7, -1e-7, 1e-6, -3e-6, 1e-5, -1e-4, 1e-3, -1e-3, 0.011, -0.3, 1.0, -1.0, 3.0, -20.0, 20.0):
            ref = F(lp + d)
            away = float(ref) - lp
            for kl in (1.0, 0.02):
                z, one = np.full((1, V), 2.5, F), np.ones(1, F)
                loss, g = policy(e, z, np.zeros(1, np.int32), np.full(1, lp, F), np.full(1, ref, F), 0 * one, kl)
                want = float(F(kl)) * kl_term(away)
                assert loss >= 0
                assert abs(loss - want) <= 4 * E * want + float(F(kl)) * 1.1e-14 * abs(np.expm1(away)) + 1e-30, (d, kl)
                # the gradient -kl (e^away - 1) (1[label] - 1 / V): 8 roundings of fp32 and the approximate power's 4 e
                c = -float(F(kl)) * np.expm1(away)
                hot = np.zeros(V)
                hot[0] = 1
                assert np.all(abs(g[0] - c * (hot - 1 / V)) <= 16 * E * abs(c) * (hot + 1 / V) + 1.2e-14 + 1e-30), (d, kl)
            e.step_end()


def test_kl_term_over_rows_is_their_mean():
    """5000 rows of a policy 1e-4 away from its reference: about 5e-9 a row, none of it lost."""
    V, n = 64, 5000
    lp = -np.log(float(V))
    ref = (lp + 1e-4 * np.random.default_rng(1).standard_normal(n)).astype(F)
    want = float(F(0.1)) * np.mean([kl_term(float(r) - lp) for r in ref])
    with Eng("b200") as e:
        loss, _ = policy(e, np.zeros((n, V), F), np.zeros(n, np.int32), np.full(n, lp, F), ref, np.zeros(n, F), 0.1)
    assert abs(loss - want) <= 8 * E * want


@pytest.mark.parametrize("V", [4, 700, 20000])
def test_kl_term_of_an_impossible_action_is_infinite(V):
    """lp = -inf: e^away - away - 1 is +inf, and so is the loss (its two parts alone would give NaN); with the
    reference's -inf instead, -away is."""
    z = np.zeros((2, V), F)
    z[0, 1] = -np.inf
    with Eng("b200") as e:
        act = np.array([1, 0], np.int32)
        for adv in (0.0, 1.0, -1.0):
            loss, g = policy(e, z, act, np.full(2, -1, F), np.full(2, -1, F), np.full(2, adv, F), 0.1)
            assert loss == np.inf and np.isfinite(g[1]).all()
        loss, g = policy(e, np.zeros((2, V), F), act, np.full(2, -1, F), np.array([-np.inf, -1], F), np.zeros(2, F), 0.1)
        assert loss == np.inf and np.isfinite(g).all()
        loss, g = policy(e, z, act, np.full(2, -1, F), None, np.ones(2, F), 0.0)  # without a KL term: a ratio of 0
        assert np.isfinite(loss) and np.isfinite(g).all() and not g[0].any()


@pytest.mark.parametrize("V", [4, 700, 20000])
def test_preference_of_an_impossible_answer(V):
    """An answer with a token of probability 0: h is infinite, and without smoothing the pair's loss is 0 where the
    impossible answer is the other one (log sigmoid(-h) has weight 0) and infinite where it is the preferred one."""
    T = 3
    for side in (0, 1):
        z = np.random.default_rng(V).standard_normal((4, T, V)).astype(F)
        lab = np.zeros((4, T), np.int32)
        z[2 * side, 1, 0] = -np.inf  # a token of the first pair's preferred answer, or of its other one
        with Eng("b200") as e:
            def run(eps):
                tz = e.param(z)
                loss = e.check(e.L.nc_ext_preference_loss(tz, e.t(lab), None, None, 0.5, eps, None))
                assert e.L.nc_backward(loss) == 0, e.err()
                return float(e.np(loss)), e.grad(tz)

            loss, g = run(0.0)
            lp = z.astype(np.float64) - np.log(np.exp(z.astype(np.float64)).sum(-1, keepdims=True))
            h = 0.5 * (lp[1, :, 0].sum() - lp[3, :, 0].sum())  # the second pair
            if side:
                # lp is off by (8 max|z| + 64 + V / 32) e as everywhere, and T of them make a sum
                unit = (8 * 6 + 64 + V / 32) * E
                assert abs(loss - np.log1p(np.exp(-h)) / 2) <= 2 * T * unit * 0.5 + 4 * E
                assert np.isfinite(g).all() and not g[0].any() and not g[2].any() and g[1].any()
            else:
                assert loss == np.inf and np.isfinite(g[1]).all() and np.isfinite(g[3]).all()
            assert run(0.1)[0] == np.inf
