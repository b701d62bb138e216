"""nc_ext_policy_loss and nc_ext_preference_loss against their formulas in 64 bits.

Tolerances, in units of e = 2^-24 (half an fp32 step, relative). Logits are below Z in size.
  - exp(z - m): z - m is rounded once and multiplied by log2 e (2 e of an exponent below 2 Z log2 e, so 4 Z e of
    the value at most) and the exponential is off by 2 steps (4 e). A sum of V of them adds at most
    V / team + 12 roundings and one rescaling (4 e + 4 Z e) per doubling of the maximum, a few in all; in relation
    to the sum, whose large terms have exponents near 0, (8 Z + 64 + V / 32) e bounds it.
  - so lp is off by T = (8 Z + 64 + V / 32) e, a probability by T + 4 Z e + 8 e.
  - ratio = exp(lp - old) by T + 8 e, a term of the loss by (T + 16 e) (|ratio A| + kl (e^away + 1 + |away|)).
  - a gradient entry by |c| p (T + 4 Z e + 16 e) + |error of c| (p + 1[label]).
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi, seeded

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def stats(z, lab):
    """log probabilities of the labels and all probabilities, in 64 bits"""
    z = z.astype(np.float64)
    m = z.max(-1, keepdims=True)
    ex = np.exp(z - m)
    s = ex.sum(-1, keepdims=True)
    lp = np.take_along_axis(z, lab[..., None].astype(np.int64), -1) - m - np.log(s)
    return lp[..., 0], ex / s


def unit(z):
    fin = np.abs(z[np.isfinite(z)])
    return (8 * (fin.max() if fin.size else 0) + 64 + z.shape[-1] / 32) * E


def policy(z, act, old, ref, adv, mask, lo, hi, kl):
    """loss, lp, dz, and the bounds of the loss's and the gradient's error"""
    w = np.ones(act.shape, bool) if mask is None else mask != 0
    zz = np.where(w[..., None], z, 0).astype(np.float64)
    lab = np.where(w, act, 0)
    lp, p = stats(zz, lab)
    T = unit(zz)
    old, adv = np.where(w, old, 0).astype(np.float64), np.where(w, adv, 0).astype(np.float64)
    r = np.exp(lp - old)
    lo, hi = float(np.float32(1) - np.float32(lo)), float(np.float32(1) + np.float32(hi))
    term = -np.minimum(r * adv, np.clip(r, lo, hi) * adv)
    c = np.where(np.where(adv >= 0, r <= hi, r >= lo), -adv * r, 0.0)
    size = abs(r * adv) + abs(hi * adv)
    if kl:
        kl = float(np.float32(kl))
        away = np.where(w, ref, 0).astype(np.float64) - lp
        term = term + kl * (np.exp(away) - away - 1)
        c = c + kl * (1 - np.exp(away))
        size = size + abs(kl) * (np.exp(away) + 1 + abs(away))
    n = max(1, w.sum())
    c, size = np.where(w, c, 0) / n, np.where(w, size, 0) / n
    hot = np.zeros_like(zz)
    np.put_along_axis(hot, lab[..., None].astype(np.int64), 1, -1)
    dz = c[..., None] * (hot - p)
    off = abs(c)[..., None] * p * (T + 4 * 60 * E) + (size * (T + 32 * E))[..., None] * (p + hot)
    return (np.where(w, term, 0).sum() / n, np.where(w, lp, 0), dz, size.sum() * (T + 32 * E) + 1e-12, off + 1e-30, T)


def make(seed, shape, V, scale=2.0, span=0.3):
    rng = np.random.default_rng(seed)
    z = (rng.standard_normal((*shape, V)) * scale).astype(np.float32)
    act = rng.integers(0, V, shape).astype(np.int32)
    lp, _ = stats(z, act)
    ratio = span * rng.standard_normal(shape)
    for edge in (np.log(0.8), np.log(1.25)):  # 32 and 64 bits may fall on different sides of a border
        ratio = np.where(abs(ratio - edge) < 1e-3, edge + 2e-3, ratio)
    old, ref = (lp - ratio).astype(np.float32), (lp + rng.standard_normal(shape)).astype(np.float32)
    return z, act, old, ref, rng.standard_normal(shape).astype(np.float32)


def run_policy(e, z, act, old, ref, adv, mask, lo=0.2, hi=0.25, kl=0.1, tz=None, want_logp=True):
    tz = e.param(z) if tz is None else tz
    more = ctypes.c_void_p()
    t = lambda v: None if v is None else e.t(v)  # noqa: E731
    loss = e.check(e.L.nc_ext_policy_loss(tz, t(act), t(old), t(ref), t(adv), t(mask),
                                          ctypes.byref(capi.PolicyOpts(lo, hi, kl)), ctypes.byref(more) if want_logp else None))
    return tz, loss, more.value


@pytest.mark.parametrize("shape,V", [((1,), 1), ((1,), 2), ((3,), 5), ((2, 3), 31), ((9,), 96), ((40, 7), 97), ((5,), 1023),
                                     ((5,), 1024), ((5,), 1025), ((2, 4), 4097), ((3,), 50001), ((2,), 131072), ((5000,), 3),
                                     ((70000,), 4)], ids=str)
def test_policy_matches_formula(shape, V):
    z, act, old, ref, adv = make(V, shape, V)
    mask = (np.random.default_rng(1).random(shape) < 0.7).astype(np.int32) * 5
    for m, kl in ((None, 0.1), (mask, 0.0)):
        loss, lp, dz, dl, off, T = policy(z, act, old, ref, adv, m, 0.2, 0.25, kl)
        with Eng("b200") as e:
            tz, tl, more = run_policy(e, z, act, old, ref if kl else None, adv, m, kl=kl)
            assert e.L.nc_backward(tl) == 0, e.err()
            assert abs(float(e.np(tl)) - loss) <= dl
            got = e.np(more)
            assert np.all(abs(got - lp) <= T + abs(lp) * E + 1e-30)
            g = e.grad(tz)
            assert g.shape == z.shape and np.all(abs(g - dz) <= off)
            if m is not None:
                assert not g[m == 0].any() and not got[m == 0].any()
            assert e.ok(), e.err()


@pytest.mark.parametrize("V", [64, 1500])
def test_policy_borders_and_sign(V):
    """Ratios well below, inside and well above the clip range, advantages of both signs and 0: which rows move."""
    rng = np.random.default_rng(2)
    z = rng.standard_normal((9, V)).astype(np.float32)
    act = rng.integers(0, V, 9).astype(np.int32)
    lp, _ = stats(z, act)
    old = (lp - np.log([0.5, 1.0, 1.7] * 3)).astype(np.float32)
    adv = np.repeat([1.0, -1.0, 0.0], 3).astype(np.float32)
    loss, _, dz, dl, off, _ = policy(z, act, old, None, adv, None, 0.2, 0.25, 0)
    with Eng("b200") as e:
        tz, tl, _ = run_policy(e, z, act, old, None, adv, None, kl=0.0)
        e.L.nc_backward(tl)
        g = e.grad(tz)
        assert abs(float(e.np(tl)) - loss) <= dl and np.all(abs(g - dz) <= off)
        assert [bool(g[i].any()) for i in range(9)] == [True, True, False, False, True, True, False, False, False]


@pytest.mark.parametrize("V", [40, 2000])
def test_policy_rows_left_out_hold_anything(V):
    z, act, old, ref, adv = make(3, (6,), V)
    mask = np.array([1, 0, 1, 0, 0, 1], np.int32)
    loss, lp, dz, dl, off, _ = policy(z, act, old, ref, adv, mask, 0.2, 0.25, 0.1)
    z[1], z[3, ::3], z[4] = np.nan, np.inf, -np.inf
    act[1], act[3], old[3], ref[4], adv[1] = -100, 2**31 - 1, np.nan, np.inf, np.nan
    with Eng("b200") as e:
        tz, tl, more = run_policy(e, z, act, old, ref, adv, mask)
        assert e.L.nc_backward(tl) == 0
        assert abs(float(e.np(tl)) - loss) <= dl
        g = e.grad(tz)
        assert np.all(abs(g - dz) <= off) and not g[mask == 0].any()
        assert e.ok(), e.err()
        for m in (np.zeros(6, np.int32),):  # nothing counts
            e.L.nc_clear_grad(tz)
            _, tl, more = run_policy(e, z, act, old, ref, adv, m, tz=tz)
            assert e.L.nc_backward(tl) == 0
            assert float(e.np(tl)) == 0.0 and not e.np(more).any() and not e.grad(tz).any()


@pytest.mark.parametrize("V", [5, 40, 2000, 20000])
@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_policy_nan_in_counted_rows_shows(V, kl):
    """A counted row with a NaN (or +inf) logit, old log probability or advantage: the loss is NaN and so is the
    row's whole gradient; the other rows have theirs."""
    z, act, old, ref, adv = make(13, (6,), V)
    _, _, dz, _, off, _ = policy(z, act, old, ref, adv, None, 0.2, 0.25, kl)
    z[1, V // 2], z[2, V - 1], old[3], adv[4] = np.nan, np.inf, np.nan, np.nan
    with Eng("b200") as e:
        tz, tl, _ = run_policy(e, z, act, old, ref, adv, None, kl=kl)
        assert e.L.nc_backward(tl) == 0
        g = e.grad(tz)
        assert np.isnan(float(e.np(tl))) and np.isnan(g[1:5]).all()
        for i in (0, 5):
            assert np.all(abs(g[i] - dz[i]) <= off[i])
        assert e.ok(), e.err()


@pytest.mark.parametrize("V", [33, 4000])
@pytest.mark.parametrize("low", [-np.inf, np.finfo(np.float32).min])
def test_policy_banned_and_extreme_logits(V, low):
    """Entries of -inf or the lowest float, large logits, a maximum that rises along the row."""
    z, act, old, ref, adv = make(4, (5,), V)
    z[:, V // 2:] = low
    act[:] = np.arange(5) % (V // 2)
    z[1] += 3e4
    z[2, :V // 2] = np.sort(z[2, :V // 2]) * 20
    z[3, :] = low
    z[3, 2], act[3] = -1e30, 2  # one entry carries the row
    lp, _ = stats(z, act)
    old, ref = (lp - 0.1).astype(np.float32), lp.astype(np.float32)
    loss, lp, dz, dl, off, _ = policy(z, act, old, ref, adv, None, 0.2, 0.25, 0.1)
    # row 1: fp32 cannot hold lp - old better than the rounding of old itself, which the reference shares
    with Eng("b200") as e:
        tz, tl, more = run_policy(e, z, act, old, ref, adv, None)
        assert e.L.nc_backward(tl) == 0
        got, g = e.np(more), e.grad(tz)
        assert np.all(np.isfinite(g)) and np.all(abs(got - lp) <= 200 * E * (1 + abs(lp)))
        small = unit(z[[0, 2, 4]][..., :V // 2])
        assert np.all(abs(g - dz) <= off * max(1.0, small / E) + 1e-6 * abs(dz).max())
        assert not g[:, V // 2:].any()


def test_policy_reads_a_slice_of_tokens_and_strides():
    """logits[:, :-1] of [batch, tokens, vocab] is read in place; the storage's last tokens get no gradient.
    A view with strided vocabulary entries is copied."""
    B, T, V = 3, 5, 37
    z, act, old, ref, adv = make(5, (B, T), V)
    loss, _, dz, dl, off, _ = policy(z[:, :-1], act[:, 1:], old[:, 1:], ref[:, 1:], adv[:, 1:], None, 0.2, 0.25, 0.1)
    with Eng("b200") as e:
        tz = e.param(z)
        cut = lambda a: e.L.nc_slice(e.t(a), 1, 1, T - 1, 1)  # noqa: E731
        more = ctypes.c_void_p()
        o = capi.PolicyOpts(0.2, 0.25, 0.1)
        tl = e.check(e.L.nc_ext_policy_loss(e.L.nc_slice(tz, 1, 0, T - 1, 1), cut(act), cut(old), cut(ref), cut(adv), None,
                                            ctypes.byref(o), ctypes.byref(more)))
        assert e.L.nc_backward(tl) == 0, e.err()
        g = e.grad(tz)
        assert abs(float(e.np(tl)) - loss) <= dl
        assert np.all(abs(g[:, :-1] - dz) <= off) and not g[:, -1].any()
        tt = e.param(np.ascontiguousarray(z.transpose(0, 2, 1)))
        loss, _, dz, dl, off, _ = policy(z, act, old, ref, adv, None, 0.2, 0.25, 0.1)
        _, tl, _ = run_policy(e, None, act, old, ref, adv, None, tz=e.L.nc_transpose(tt, 1, 2))
        assert e.L.nc_backward(tl) == 0, e.err()
        assert abs(float(e.np(tl)) - loss) <= dl and np.all(abs(e.grad(tt).transpose(0, 2, 1) - dz) <= off)


@pytest.mark.parametrize("V", [50, 3001])
def test_policy_gradient_scales_accumulates_repeats(V):
    z, act, old, ref, adv = make(6, (20,), V)
    with Eng("b200") as e:
        tz = e.param(z)

        def go(f):
            _, tl, _ = run_policy(e, z, act, old, ref, adv, None, tz=tz, want_logp=False)
            assert e.L.nc_backward(e.check(e.L.nc_scale(tl, f))) == 0
            v = float(e.np(tl))
            g = e.grad(tz)
            e.step_end()
            return v, g

        v, one = go(1.0)
        v2, three = go(2.0)  # on top of the first
        assert v == v2 and np.allclose(three, 3 * one, rtol=1e-6, atol=0)
        e.L.nc_clear_grad(tz)
        assert np.array_equal(go(1.0)[1], one)


def test_policy_gradient_against_differences():
    z, act, old, ref, adv = make(7, (4,), 11)
    f = lambda z: policy(z, act, old, ref, adv, None, 0.2, 0.25, 0.1)[0]  # noqa: E731
    with Eng("b200") as e:
        tz, tl, _ = run_policy(e, z, act, old, ref, adv, None)
        e.L.nc_backward(tl)
        g = e.grad(tz)
    base = z.astype(np.float64)
    for i in range(z.size):
        lo, hi = base.copy(), base.copy()
        lo.flat[i] -= 1e-6
        hi.flat[i] += 1e-6
        assert abs((f(hi) - f(lo)) / 2e-6 - g.flat[i]) < 1e-6


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-abs(x)))


def preference(z, lab, ref, mask, beta, eps):
    S, T, V = z.shape
    w = np.ones((S, T), bool) if mask is None else mask != 0
    zz, lab = np.where(w[..., None], z, 0), np.where(w, lab, 0)
    if T:
        lp, p = stats(zz, lab)
    else:
        lp, p = np.zeros((S, 0)), np.zeros(z.shape)
    seq = np.where(w, lp, 0).sum(1)
    beta, eps = float(np.float32(beta)), float(np.float32(eps))
    gap = seq - (0 if ref is None else ref.astype(np.float64))
    h = beta * (gap[:S // 2] - gap[S // 2:])
    loss = ((1 - eps) * softplus(-h) + eps * softplus(h)).mean()
    c = beta / (S // 2) * (1 / (1 + np.exp(-h)) - (1 - eps))
    c = np.concatenate((c, -c))[:, None] * w
    hot = np.zeros(z.shape)
    if T:
        np.put_along_axis(hot, lab[..., None].astype(np.int64), 1, -1)
    unit_ = unit(zz) if T else E
    dseq = T * unit_ + 1e-30  # every token's lp is off by unit_
    dh = 2 * beta * dseq
    dc = abs(c) * 4 * E + beta / (S // 2) * dh
    off = (abs(c) * (unit_ + 4 * 60 * E))[..., None] * p + dc[..., None] * (p + hot) + 1e-30
    return loss, seq, c[..., None] * (hot - p), dh + 2 * E * loss + 1e-12, dseq, off


@pytest.mark.parametrize("P,T,V,eps", [(1, 1, 1, 0.0), (1, 1, 2, 0.1), (2, 3, 17, 0.0), (5, 33, 96, 0.1), (300, 2, 5, 0.0),
                                       (2, 700, 130, 0.5), (1, 9, 5001, 0.0), (3, 5, 32000, 0.1), (2, 0, 7, 0.0)], ids=str)
def test_preference_matches_formula(P, T, V, eps):
    rng = np.random.default_rng(P + T + V)
    z = (rng.standard_normal((2 * P, T, V)) * 2).astype(np.float32)
    lab = rng.integers(0, V, (2 * P, T)).astype(np.int32)
    mask = (rng.random((2 * P, T)) < 0.7).astype(np.int32)
    if T:
        mask[0] = 0  # an answer with nothing counted
    ref = (preference(z, lab, None, None, 0.1, 0)[1] + rng.standard_normal(2 * P)).astype(np.float32)
    for m, rf in ((None, ref), (mask, None)):
        beta = 0.3 if rf is not None else 0.02
        loss, seq, dz, dl, ds, off = preference(z, lab, rf, m, beta, eps)
        with Eng("b200") as e:
            tz = e.param(z)
            more = ctypes.c_void_p()
            tl = e.check(e.L.nc_ext_preference_loss(tz, e.t(lab), None if rf is None else e.t(rf),
                                                    None if m is None else e.t(m), beta, eps, ctypes.byref(more)))
            assert e.L.nc_backward(tl) == 0, e.err()
            assert abs(float(e.np(tl)) - loss) <= dl
            assert np.all(abs(e.np(more.value) - seq) <= ds + abs(seq) * E)
            g = e.grad(tz)
            assert np.all(abs(g - dz) <= off)
            if m is not None:
                assert not g[m == 0].any()
            assert e.ok(), e.err()


def test_preference_extremes_and_masked_rows():
    """Pairs far apart on either side (no overflow, the gradient saturates) and anything in uncounted rows."""
    P, T, V = 3, 4, 19
    rng = np.random.default_rng(11)
    z = rng.standard_normal((2 * P, T, V)).astype(np.float32)
    lab = rng.integers(0, V, (2 * P, T)).astype(np.int32)
    mask = np.ones((2 * P, T), np.int32)
    mask[:, 2:] = 0
    ref = np.array([-1e5, 1e5, 0, 0, 0, 0], np.float32)
    loss, seq, dz, dl, ds, off = preference(z, lab, ref, mask, 1.0, 0.0)
    z[:, 2:], lab[:, 2:] = np.nan, -1
    with Eng("b200") as e:
        tz = e.param(z)
        tl = e.check(e.L.nc_ext_preference_loss(tz, e.t(lab), e.t(ref), e.t(mask), 1.0, 0.0, None))
        assert e.L.nc_backward(tl) == 0, e.err()
        g = e.grad(tz)
        assert abs(float(e.np(tl)) - loss) <= dl + 4 * E * loss and np.all(abs(g - dz) <= off) and np.isfinite(g).all()
        assert e.ok(), e.err()


def test_preference_gradient_against_differences():
    P, T, V = 2, 3, 6
    rng = np.random.default_rng(12)
    z = rng.standard_normal((2 * P, T, V)).astype(np.float32)
    lab = rng.integers(0, V, (2 * P, T)).astype(np.int32)
    f = lambda z: preference(z, lab, None, None, 0.5, 0.1)[0]  # noqa: E731
    with Eng("b200") as e:
        tz = e.param(z)
        e.L.nc_backward(e.check(e.L.nc_ext_preference_loss(tz, e.t(lab), None, None, 0.5, 0.1, None)))
        g = e.grad(tz)
    base = z.astype(np.float64)
    for i in range(z.size):
        lo, hi = base.copy(), base.copy()
        lo.flat[i] -= 1e-6
        hi.flat[i] += 1e-6
        assert abs((f(hi) - f(lo)) / 2e-6 - g.flat[i]) < 1e-6


def test_labels_out_of_range_are_reported():
    """From a host copy before anything is launched; from a label made on the device at the next synchronisation,
    after which the context goes on."""
    for V in (10, 2000):
        z, act, old, ref, adv = make(13, (4,), V)
        bad = act.copy()
        bad[2] = V
        with Eng("b200") as e:
            o = capi.PolicyOpts(0.2, 0.25, 0.0)
            args = lambda lab: (e.t(z), lab, e.t(old), None, e.t(adv), None, ctypes.byref(o), None)  # noqa: E731
            assert not e.L.nc_ext_policy_loss(*args(e.t(bad))) and "label" in e.err()
            e.L.nc_clear_error(e.ctx)
            made = e.check(e.L.nc_to_dtype(e.t(bad.astype(np.float32)), capi.I32))
            assert e.L.nc_ext_policy_loss(*args(made))
            assert e.L.nc_ext_synchronize(e.ctx) == 4 and "label" in e.err()
            e.L.nc_clear_error(e.ctx)
            assert np.isfinite(e.np(e.check(e.L.nc_ext_policy_loss(*args(e.t(act))))))


def test_refusals():
    z, act, old, ref, adv = make(14, (2, 3), 5)
    mask = np.ones((2, 3), np.int32)
    with Eng("b200") as e:
        def refused(text, code, call):
            before = e.L.nc_ext_launch_count(e.ctx)
            more = ctypes.c_void_p(1)
            assert not call(more) and not more.value
            assert text in e.err() and e.L.nc_status_code(e.ctx) == code, e.err()
            assert e.L.nc_ext_launch_count(e.ctx) == before
            e.L.nc_clear_error(e.ctx)

        def pol(text, code, o=capi.PolicyOpts(0.2, 0.25, 0.1), grad=(), **kw):
            a = dict(z=z, act=act, old=old, ref=ref, adv=adv, mask=mask)
            a.update(kw)
            t = {k: None if v is None else e.param(v) if k in grad else e.t(v) for k, v in a.items()}
            refused(text, code, lambda m: e.L.nc_ext_policy_loss(t["z"], t["act"], t["old"], t["ref"], t["adv"], t["mask"],
                                                                 None if o is None else ctypes.byref(o), ctypes.byref(m)))

        pol("opts", 4, o=None)
        for o in ((-0.1, 0.2, 0), (1.1, 0.2, 0), (np.nan, 0.2, 0), (0.2, -0.1, 0), (0.2, np.inf, 0), (0.2, np.nan, 0)):
            pol("clip", 4, o=capi.PolicyOpts(*o))
        pol("kl_coef", 4, o=capi.PolicyOpts(0.2, 0.2, np.nan))
        pol("KL", 4, ref=None)
        pol("logits must be f32", 2, z=act)
        pol("logits must be [", 1, z=z[0, 0])
        pol("logits must be [", 1, z=z[..., :0])
        pol("labels must be i32", 2, act=old)
        pol("mask must be i32", 2, mask=old)
        pol("old_logp must be f32", 2, old=act)
        pol("ref_logp must be f32", 2, ref=act)
        pol("advantages must be f32", 2, adv=act)
        for k in ("act", "old", "ref", "adv", "mask"):
            pol("leading shape", 1, **{k: {"act": act, "old": old, "ref": ref, "adv": adv, "mask": mask}[k][:, :2]})
            pol("leading shape", 1, **{k: {"act": act, "old": old, "ref": ref, "adv": adv, "mask": mask}[k].ravel()})
        for k in ("old", "ref", "adv"):
            pol("constant", 4, grad=(k,))

        def pref(text, code, beta=0.1, eps=0.0, grad=(), **kw):
            a = dict(z=z, lab=act, ref=old[:, 0], mask=mask)
            a.update(kw)
            t = {k: None if v is None else e.param(v) if k in grad else e.t(v) for k, v in a.items()}
            refused(text, code, lambda m: e.L.nc_ext_preference_loss(t["z"], t["lab"], t["ref"], t["mask"], beta, eps, ctypes.byref(m)))

        for b in (0.0, -1.0, np.nan, np.inf):
            pref("beta", 4, beta=b)
        for s in (-0.1, 0.6, np.nan):
            pref("label_smoothing", 4, eps=s)
        pref("2 pairs", 1, z=z[0], lab=act[0], mask=mask[0])
        pref("2 pairs", 1, z=z[:1], lab=act[:1], mask=mask[:1])
        pref("2 pairs", 1, z=z[:0], lab=act[:0], mask=mask[:0])
        pref("leading shape", 1, lab=act[:, :2])
        pref("ref_logp must be [2 pairs]", 1, ref=old[0])
        pref("constant", 4, grad=("ref",))
        assert e.L.nc_ext_policy_loss(None, None, None, None, None, None, None, None) is None
        assert e.L.nc_ext_preference_loss(None, None, None, None, 0.1, 0.0, None) is None and e.ok()
        # constants may require grad while gradients are off
        e.L.nc_set_grad_enabled(e.ctx, 0)
        tl = e.L.nc_ext_policy_loss(e.param(z), e.t(act), e.param(old), e.t(ref), e.t(adv), e.t(mask.astype(np.uint8)),
                                    ctypes.byref(capi.PolicyOpts(0.2, 0.25, 0.1)), None)
        assert np.isfinite(e.np(tl)) and not e.L.nc_requires_grad(tl)


def test_rows_behind_2_to_the_31_elements():
    """Offsets past 32 bits: the last rows of 2^31 + 70000 logits, with a gradient."""
    import torch

    V, N = 65537, 32770
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 34 GB")
    with Eng("b200") as e:
        e.L.nc_persistent_begin(e.ctx)
        tz = e.check(e.L.nc_zeros(e.ctx, capi.F32, *capi.shape_arg((N, V))))
        e.L.nc_persistent_end(e.ctx)
        e.L.nc_set_requires_grad(tz, 1)
        last = seeded(15, (2, V), 2.0)
        face = type("Face", (), {"__cuda_array_interface__": dict(shape=(N, V), typestr="<f4", data=(e.L.nc_ext_device_data(tz, 1), False), version=2)})
        e.L.nc_ext_synchronize(e.ctx)
        view = torch.as_tensor(face(), device="cuda")
        view[-2:].copy_(torch.from_numpy(last))
        torch.cuda.synchronize()
        mask = np.zeros(N, np.int32)
        mask[-2:] = 1
        act = np.full(N, V - 1, np.int32)
        old = stats(last, act[-2:])[0].astype(np.float32)
        loss, _, dz, dl, off, _ = policy(last, act[-2:], old, None, np.ones(2, np.float32), None, 0.2, 0.25, 0)
        full = np.zeros(N, np.float32)
        full[-2:] = old
        _, tl, _ = run_policy(e, None, act, full, None, np.ones(N, np.float32), mask, kl=0.0, tz=tz, want_logp=False)
        assert e.L.nc_backward(tl) == 0, e.err()
        assert abs(float(e.np(tl)) - loss) <= dl
        g = e.L.nc_grad(tz)
        face = type("Face", (), {"__cuda_array_interface__": dict(shape=(N, V), typestr="<f4", data=(e.L.nc_ext_device_data(g, 0), False), version=2)})
        e.L.nc_ext_synchronize(e.ctx)
        gv = torch.as_tensor(face(), device="cuda")
        assert np.all(abs(gv[-2:].cpu().numpy() - dz) <= off)
        assert int(torch.count_nonzero(gv[:-2])) == 0
        e.L.nc_release(tz)
