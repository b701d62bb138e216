"""nc_ext_qk_norm_rope (query/key head norms with rotary positions) and the two calls beside it,
nc_ext_backward_from and nc_ext_device_data, against the formulas in 64 bits.

Tolerances, in units of e = 2^-24 (half an fp32 step, relative). With u = n w and a pair (a, b):
  - n: at most 13 roundings in the sum of squares (8 in a lane, 5 joining lanes) halve to 6.5 e in its root;
    rsqrtf is off by 2 steps (4 e); with the products by r and w, u is off by less than 13 e.
  - cos and sin: the turn's fraction, below 1/2, is off by 2^-26 turns, that is 1.6 e in the angle, and
    sincospif by 2 steps (4 e): below 6 e of 1.
  - y_a = u_a c - u_b s adds 2 roundings: below 24 e (|u_a| + |u_b|).
  - dx = r (g w - n mean(g w n)): g is off by 8 e of |dy_a| + |dy_b|, the mean by 8 + 13 + 13 + 2 e of the mean of
    absolute values, r and n by 13 e each: below 48 e of r (|g||w| + |n| mean |g w n|).
  - dw sums one term a row (off by 24 e): below (24 + rows) e of the sum of absolute values.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi, seeded

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
INTER, FREQ, NO_NORM = capi.ROPE_INTERLEAVED, capi.ROPE_AXIS_FREQ, capi.ROPE_NO_NORM


def opts(q_heads, sections, flags=0, base=10000.0, eps=1e-6):
    s = list(sections) + [0] * (3 - len(sections))
    return capi.RopeOpts(q_heads, len(sections), (ctypes.c_int * 3)(*s), base, eps, flags)


def pairs(u, flags):
    h = u.shape[-1] // 2
    return (u[..., 0::2], u[..., 1::2]) if flags & INTER else (u[..., :h], u[..., h:])


def join(a, b, flags):
    if flags & INTER:
        return np.stack((a, b), -1).reshape(*a.shape[:-1], -1)
    return np.concatenate((a, b), -1)


def reference(x, wq, wk, pos, o, dy=None):
    """y and, with dy, (dx, dwq, dwk), each with the scale its tolerance multiplies; all in 64 bits."""
    B, T, H, D = x.shape
    x = x.astype(np.float64)
    half, flags = D // 2, o.flags
    angle = np.zeros((B, T, 1, half))
    i = 0
    for a in range(o.n_axes):
        at = np.arange(T, dtype=np.float64) if pos is None else pos[..., a].astype(np.float64)
        for j in range(o.sections[a]):
            p = j / o.sections[a] if flags & FREQ else i / half
            angle[..., 0, i] = at * float(o.base) ** -p
            i += 1
    c, s = np.cos(angle), np.sin(angle)
    w = np.ones((H, D))
    if wq is not None:
        w[:o.q_heads] = wq
    if wk is not None:
        w[o.q_heads:] = wk
    r = 1.0 if flags & NO_NORM else 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + float(o.eps))
    n = x * r
    a, b = pairs(n * w, flags)
    y = join(a * c - b * s, b * c + a * s, flags)
    ys = join(abs(a) + abs(b), abs(a) + abs(b), flags)
    if dy is None:
        return y, ys
    a, b = pairs(dy.astype(np.float64), flags)
    g = join(a * c + b * s, b * c - a * s, flags)
    gs = join(abs(a) + abs(b), abs(a) + abs(b), flags)
    m, ms = (g * w * n).mean(-1, keepdims=True), abs(gs * w * n).mean(-1, keepdims=True)
    if flags & NO_NORM:
        m = ms = 0.0
    dx, dxs = r * (g * w - n * m), r * (gs * abs(w) + abs(n) * ms)
    t, ts = (g * n).sum((0, 1)), (gs * abs(n)).sum((0, 1))
    q = o.q_heads
    return y, ys, (dx, dxs), (t[:q].sum(0), ts[:q].sum(0)), (t[q:].sum(0), ts[q:].sum(0))


def close(got, want, scale, units, what):
    assert got.shape == want.shape, what
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= units * E * scale + 1e-37)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, by up to {np.max(off / (E * scale + 1e-300)):.1f} units"


def inputs(seed, B, T, H, D, A, far):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((B, T, H, D)) * rng.uniform(0.1, 5, (H, 1))).astype(np.float32)
    wq, wk = (rng.uniform(-1.5, 1.5, D).astype(np.float32) for _ in range(2))
    pos = rng.integers(-far - 1, far + 1, (B, T, A)).astype(np.int32)
    return x, wq, wk, pos, rng.standard_normal((B, T, H, D)).astype(np.float32)


CASES = [  # B, T, H, q_heads, D, sections, flags, far
    (1, 1, 1, 1, 2, (1,), 0, 5),
    (1, 1, 1, 0, 2, (0,), INTER, 5),
    (2, 3, 5, 3, 16, (8,), 0, 100),
    (2, 3, 5, 3, 16, (8,), INTER, 100),
    (3, 7, 4, 2, 32, (4, 12), FREQ, 60),
    (1, 37, 6, 4, 128, (16, 24, 24), 0, 1000),
    (1, 37, 6, 6, 128, (16, 24, 24), INTER | FREQ, 1000),
    (2, 5, 3, 1, 72, (18, 18), INTER | FREQ, 37),
    (2, 5, 3, 1, 72, (10, 0, 9), 0, 37),
    (2, 9, 7, 4, 66, (33,), 0, 10),         # one pair per lane step, 33 of 64 places
    (2, 9, 7, 4, 66, (20, 13), INTER, 10),
    (2, 4, 3, 2, 36, (18,), 0, 10),         # vectors of two
    (2, 4, 3, 2, 36, (18,), INTER, 10),
    (1, 2, 2, 1, 250, (125,), 0, 99),
    (1, 2, 2, 1, 256, (64, 64), INTER, 99),
    (16, 1, 12, 8, 64, (32,), 0, 2**31 - 2),  # decoding, positions to the end of i32
    (1, 700, 3, 2, 40, (20,), NO_NORM, 5000),
    (2, 600, 24, 16, 64, (32,), 0, 4000),     # more rows than groups
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_formula(case):
    B, T, H, q, D, sections, flags, far = case
    x, wq, wk, pos, dy = inputs(sum(case[:5]), B, T, H, D, len(sections), far)
    o = opts(q, sections, flags)
    y, ys, dx, dwq, dwk = reference(x, wq, wk, pos, o, dy)
    with Eng("b200") as e:
        tx, tq, tk = e.param(x), e.param(wq), e.param(wk)
        out = e.check(e.L.nc_ext_qk_norm_rope(tx, tq, tk, e.t(pos), ctypes.byref(o)))
        close(e.np(out), y, ys, 24, "y")
        assert e.L.nc_ext_backward_from(out, e.t(dy)) == 0, e.err()
        close(e.grad(tx), *dx, 48, "dx")
        rows = B * T * H
        close(e.grad(tq), *dwq, 24 + rows, "dw of queries")
        close(e.grad(tk), *dwk, 24 + rows, "dw of keys")
        assert e.ok(), e.err()


@pytest.mark.parametrize("layout", ["slice", "heads_first", "odd_offset", "last_strided"])
def test_reads_views_in_place(layout):
    """A slice of a fused projection, [batch, heads, tokens, dim] storage, a view whose rows start off 16 bytes,
    and a view whose last axis is strided; gradients reach the whole storage."""
    B, T, H, D = 2, 5, 4, 24
    o = opts(3, (12,), 0)
    rng = np.random.default_rng(4)
    shape = {"slice": (B, T, H + 3, D), "heads_first": (B, H, T, D), "odd_offset": (B, T, H, D + 3),
             "last_strided": (B, T, D, H)}[layout]
    base = rng.standard_normal(shape).astype(np.float32)
    dy = rng.standard_normal((B, T, H, D)).astype(np.float32)
    wq, wk = seeded(1, (D,)), seeded(2, (D,))
    x = {"slice": lambda a: a[:, :, 2:2 + H], "heads_first": lambda a: a.transpose(0, 2, 1, 3),
         "odd_offset": lambda a: a[..., 1:1 + D], "last_strided": lambda a: a.transpose(0, 1, 3, 2)}[layout]
    y, ys, dx, dwq, _ = reference(x(base), wq, wk, None, o, dy)
    want, scale = np.zeros(shape), np.full(shape, 1e-30)
    x(want)[...], x(scale)[...] = dx
    with Eng("b200") as e:
        tb, tq = e.param(base), e.param(wq)
        v = {"slice": lambda: e.L.nc_slice(tb, 2, 2, H, 1), "heads_first": lambda: e.L.nc_transpose(tb, 1, 2),
             "odd_offset": lambda: e.L.nc_slice(tb, 3, 1, D, 1), "last_strided": lambda: e.L.nc_transpose(tb, 2, 3)}[layout]()
        out = e.check(e.L.nc_ext_qk_norm_rope(v, tq, e.t(wk), None, ctypes.byref(o)))
        close(e.np(out), y, ys, 24, "y")
        assert e.L.nc_ext_backward_from(out, e.t(dy)) == 0, e.err()
        close(e.grad(tb), want, scale, 48, "dx")
        close(e.grad(tq), *dwq, 24 + B * T * H, "dw")


def test_gradient_against_differences():
    """d<y, dy> / d(x, w) by central differences of the 64-bit formula."""
    B, T, H, D = 1, 2, 3, 16
    o = opts(2, (3, 5), FREQ)
    x, wq, wk, pos, dy = inputs(3, B, T, H, D, 2, 50)
    f = lambda x, wq, wk: float((reference(x, wq, wk, pos, o)[0] * dy).sum())  # noqa: E731
    with Eng("b200") as e:
        ts = [e.param(v) for v in (x, wq, wk)]
        out = e.check(e.L.nc_ext_qk_norm_rope(*ts, e.t(pos), ctypes.byref(o)))
        assert e.L.nc_ext_backward_from(out, e.t(dy)) == 0
        grads = [e.grad(t) for t in ts]
    arrs = [v.astype(np.float64) for v in (x, wq, wk)]
    rng = np.random.default_rng(0)
    for k, g in enumerate(grads):
        for i in rng.integers(0, g.size, 12):
            lo, hi = [a.copy() for a in arrs], [a.copy() for a in arrs]
            step = 1e-6
            hi[k].flat[i] += step
            lo[k].flat[i] -= step
            d = (f(*hi) - f(*lo)) / (2 * step)
            # differences: rounding of f (|f| 2^-53 / step) and the third derivative's step^2
            assert abs(d - g.flat[i]) < 2e-5 * max(1.0, np.abs(g).max()), (k, i, d, g.flat[i])


def test_shared_weight_missing_weights_and_zero_rows():
    """One weight for queries and keys, none at all, a row of zeros (eps keeps it finite), and no tokens."""
    B, T, H, D = 2, 3, 4, 32
    o = opts(2, (16,))
    x, w, _, _, dy = inputs(8, B, T, H, D, 1, 3)
    x[0, 1, 2] = 0.0
    y, ys, dx, dwq, dwk = reference(x, w, w, None, o, dy)
    with Eng("b200") as e:
        tx, tw = e.param(x), e.param(w)
        out = e.check(e.L.nc_ext_qk_norm_rope(tx, tw, tw, None, ctypes.byref(o)))
        close(e.np(out), y, ys, 24, "y")
        e.L.nc_ext_backward_from(out, e.t(dy))
        close(e.grad(tx), *dx, 48, "dx")
        close(e.grad(tw), dwq[0] + dwk[0], dwq[1] + dwk[1], 26 + B * T * H, "dw")
        y, ys = reference(x, None, None, None, o)
        close(e.np(e.check(e.L.nc_ext_qk_norm_rope(tx, None, None, None, ctypes.byref(o)))), y, ys, 24, "no weights")
        none, tq = e.param(np.zeros((2, 0, H, D), np.float32)), e.param(w)
        out = e.check(e.L.nc_ext_qk_norm_rope(none, tq, None, None, ctypes.byref(o)))
        assert e.np(out).shape == (2, 0, H, D)
        assert e.L.nc_ext_backward_from(out, e.t(np.zeros((2, 0, H, D), np.float32))) == 0
        assert not e.grad(tq).any()
        assert e.ok(), e.err()


def test_nothing_from_other_rows():
    """NaN and infinity in one head's vector stay in that row and in its gradient."""
    B, T, H, D = 1, 3, 3, 64
    o = opts(2, (32,))
    x, wq, wk, pos, dy = inputs(9, B, T, H, D, 1, 9)
    want, scale = reference(x, wq, wk, pos, o)
    x[0, 1, 1, 7], x[0, 2, 0, 3] = np.nan, np.inf
    with Eng("b200") as e:
        got = e.np(e.check(e.L.nc_ext_qk_norm_rope(e.t(x), e.t(wq), e.t(wk), e.t(pos), ctypes.byref(o))))
    bad = np.zeros((B, T, H), bool)
    bad[0, 1, 1] = bad[0, 2, 0] = True
    assert np.isnan(got[0, 1, 1]).all()
    close(got[~bad], want[~bad], scale[~bad], 24, "other rows")


def test_gradients_accumulate_and_repeat_bit_for_bit():
    """Two passes without clearing add up; after clearing, the same gradient comes back bit for bit."""
    B, T, H, D = 3, 50, 6, 64
    o = opts(4, (32,))
    x, wq, wk, pos, dy = inputs(10, B, T, H, D, 1, 99)
    with Eng("b200") as e:
        ts = [e.param(v) for v in (x, wq, wk)]
        td = e.t(dy, persistent=True)

        def go():
            out = e.check(e.L.nc_ext_qk_norm_rope(*ts, e.t(pos), ctypes.byref(o)))
            assert e.L.nc_ext_backward_from(out, td) == 0, e.err()
            g = [e.grad(t) for t in ts]
            e.step_end()
            return g

        first, second = go(), go()
        for a, b in zip(first, second):
            assert np.array_equal(a + a, b)
        for t in ts:
            e.L.nc_clear_grad(t)
            assert e.grad(t) is None
        for a, b in zip(first, go()):
            assert np.array_equal(a, b)
        assert np.array_equal(e.np(td), dy)  # the given gradient is as it was


def test_backward_from_is_backward_of_the_weighted_sum():
    """The same gradients as backward of sum(y * dy), through ops behind and before the tensor; a leaf takes dy
    itself; strided dy."""
    x, w, dy = seeded(1, (6, 8)), seeded(2, (5, 8)), seeded(3, (6, 5))
    with Eng("b200") as e:
        tx, tw = e.param(x), e.param(w)
        y = lambda: e.check(e.L.nc_tanh(e.check(e.L.nc_linear_fn(tx, tw, None))))  # noqa: E731
        e.backward_with(y(), dy)
        want = [e.grad(t) for t in (tx, tw)]
        for strided in (False, True):
            for t in (tx, tw):
                e.L.nc_clear_grad(t)
            td = e.L.nc_transpose(e.t(np.ascontiguousarray(dy.T)), 0, 1) if strided else e.t(dy)
            assert e.L.nc_ext_backward_from(y(), td) == 0, e.err()
            for t, g in zip((tx, tw), want):
                assert np.array_equal(e.grad(t), g)
        leaf = e.param(x)
        for k in (1, 2):
            assert e.L.nc_ext_backward_from(leaf, e.t(x)) == 0
            assert np.array_equal(e.grad(leaf), k * x)
        out = y()
        td = e.t(dy)
        assert e.L.nc_ext_backward_from(out, td) == 0 and e.L.nc_ext_backward_from(out, td) == 0, e.err()
        assert np.array_equal(e.np(td), dy)


def test_backward_from_the_gradient_of_a_leaf():
    """dy is the gradient buffer of x, which the pass adds to: the pass reads dy as it was."""
    x, w, first = seeded(1, (40, 24)), seeded(2, (24, 24)), seeded(3, (40, 24))
    with Eng("b200") as e:
        tx, tw = e.param(x), e.param(w)
        assert e.L.nc_ext_backward_from(tx, e.t(first)) == 0  # x's gradient is `first`
        y = e.check(e.L.nc_linear_fn(tx, tw, None))
        assert e.L.nc_ext_backward_from(y, e.L.nc_grad(tx)) == 0, e.err()
        x, w, first = (v.astype(np.float64) for v in (x, w, first))
        # sums of 24 and 40 products: at most 40 roundings of the sum of absolute values (3xTF32 drops 2^-21 of each)
        assert np.all(abs(e.grad(tw) - first.T @ x) <= (40 * E + 2.0 ** -20) * (abs(first).T @ abs(x)))
        assert np.all(abs(e.grad(tx) - (first + first @ w)) <= (40 * E + 2.0 ** -20) * (abs(first) + abs(first) @ abs(w)))


def test_backward_from_refuses():
    with Eng("b200") as e:
        p = e.param(seeded(1, (2, 3)))
        y = e.check(e.L.nc_tanh(p))
        for td, text in [(e.t(seeded(2, (3, 2))), "gradient"), (e.t(np.ones((2, 3), np.int32)), "f32")]:
            assert e.L.nc_ext_backward_from(y, td) != 0 and text in e.err()
            e.L.nc_clear_error(e.ctx)
        assert e.L.nc_ext_backward_from(e.t(seeded(2, (2, 3))), e.t(seeded(2, (2, 3)))) == 5 and "grad" in e.err()
        e.L.nc_clear_error(e.ctx)
        assert e.L.nc_ext_backward_from(None, y) != 0 and e.L.nc_ext_backward_from(y, None) != 0
        assert e.ok()


def test_refusals():
    B, T, H, D = 2, 3, 4, 16
    x, w = seeded(1, (B, T, H, D)), seeded(2, (D,))
    pos = np.zeros((B, T, 1), np.int32)
    with Eng("b200") as e:
        def refused(text, code, o=opts(2, (8,)), x=x, wq=w, wk=w, pos=pos):
            t = lambda v: None if v is None else e.t(v)  # noqa: E731
            before = e.L.nc_ext_launch_count(e.ctx)
            assert not e.L.nc_ext_qk_norm_rope(t(x), t(wq), t(wk), t(pos), None if o is None else ctypes.byref(o))
            assert text in e.err() and e.L.nc_status_code(e.ctx) == code, e.err()
            assert e.L.nc_ext_launch_count(e.ctx) == before
            e.L.nc_clear_error(e.ctx)

        refused("opts", 4, o=None)
        refused("x must be", 1, x=x[0])
        refused("f32", 2, x=np.zeros((B, T, H, D), np.int32))
        refused("even", 1, x=seeded(1, (B, T, H, 15)), wq=None, wk=None)
        refused("even", 1, x=seeded(1, (1, 1, 1, 258)), wq=None, wk=None)
        refused("even", 1, x=seeded(1, (1, 1, 1, 0)), wq=None, wk=None)
        refused("q_heads", 4, o=opts(5, (8,)))
        refused("q_heads", 4, o=opts(-1, (8,)))
        refused("n_axes", 4, o=capi.RopeOpts(2, 0, (ctypes.c_int * 3)(), 1e4, 1e-6, 0))
        refused("n_axes", 4, o=capi.RopeOpts(2, 4, (ctypes.c_int * 3)(), 1e4, 1e-6, 0))
        refused("section", 4, o=opts(2, (-1,)))
        refused("dim / 2", 4, o=opts(2, (9,)))
        refused("dim / 2", 4, o=opts(2, (2**31 - 1, 2**31 - 1)), pos=np.zeros((B, T, 2), np.int32))
        for bad in (0.0, -1.0, np.nan, np.inf):
            refused("base", 4, o=opts(2, (8,), base=bad))
        for bad in (-1e-6, np.nan, np.inf):
            refused("eps", 4, o=opts(2, (8,), eps=bad))
        refused("flags", 4, o=opts(2, (8,), flags=8))
        refused("weights", 1, wq=seeded(1, (D + 1,)))
        refused("weights", 1, wk=seeded(1, (1, D)))
        refused("weights", 2, wk=np.ones(D, np.int32))
        refused("positions must be i32", 2, pos=np.zeros((B, T, 1), np.float32))
        refused("positions must be [", 1, pos=np.zeros((B, T, 2), np.int32))
        refused("positions must be [", 1, pos=np.zeros((B, T + 1, 1), np.int32))
        refused("positions must be [", 1, pos=np.zeros((1, T, 1), np.int32))
        refused("positions must be [", 1, pos=np.zeros((T,), np.int32))
        refused("several axes", 4, o=opts(2, (4, 4)), pos=None)
        assert e.L.nc_ext_qk_norm_rope(None, None, None, None, None) is None and e.ok()
        assert e.L.nc_ext_qk_norm_rope(e.t(x), e.t(w), e.t(w), e.t(pos[0]), ctypes.byref(opts(2, (8,))))  # [tokens, axes]


def test_device_data_is_the_tensor():
    import torch

    with Eng("b200") as e:
        def view(t, write):
            p = e.L.nc_ext_device_data(t, write)
            shape = e.shape(t)
            face = type("Face", (), {"__cuda_array_interface__": dict(shape=shape, typestr="<f4", data=(p, False), version=2)})
            return torch.as_tensor(face(), device="cuda")

        a = seeded(1, (3, 700))
        for arr in (a, a[:, :2].copy()):  # with and without a host mirror from birth
            t = e.t(arr)
            e.L.nc_ext_synchronize(e.ctx)
            v = view(t, 1)
            assert np.array_equal(v.cpu().numpy(), arr)
            v.mul_(2)
            torch.cuda.synchronize()
            assert np.array_equal(e.np(t), 2 * arr)
            assert np.array_equal(e.np(e.L.nc_neg(t)), -2 * arr)
        s = e.L.nc_slice(e.t(a), 0, 1, 1, 1)
        e.L.nc_ext_synchronize(e.ctx)
        assert np.array_equal(view(s, 0).cpu().numpy(), a[1:2])
        host = e.t(a)
        p = ctypes.cast(e.L.nc_data_f32(host), ctypes.POINTER(ctypes.c_float))
        p[0] = 7.0  # a host write still to be pushed
        v = view(host, 0)
        e.L.nc_ext_synchronize(e.ctx)
        assert float(v[0, 0]) == 7.0
        assert e.L.nc_ext_device_data(None, 0) is None


def test_device_data_for_writing_computes_what_still_reads_the_tensor():
    import torch

    a = seeded(4, (300, 128))
    with Eng("b200") as e:
        t = e.t(a)
        want = e.np(e.check(e.L.nc_gelu(e.t(a), 0)))
        y = e.check(e.L.nc_gelu(t, 0))  # kept pending until something reads it
        face = type("Face", (), {"__cuda_array_interface__": dict(shape=a.shape, typestr="<f4", data=(e.L.nc_ext_device_data(t, 1), False), version=2)})
        e.L.nc_ext_synchronize(e.ctx)
        torch.as_tensor(face(), device="cuda").zero_()
        torch.cuda.synchronize()
        assert np.array_equal(e.np(y), want)
        assert not e.np(t).any()


def test_inside_attention():
    """Fused projection -> norms and rotation -> the framework's attention, forward and backward, against torch in
    64 bits; the fused attention reads the rotated heads through slices and transposes."""
    import torch

    B, T, H, D = 2, 24, 4, 16
    C = H * D
    o = opts(H, (D // 2,))
    x, w = seeded(1, (B, T, C)), seeded(2, (3 * C, C), 0.2)
    wq, wk = seeded(3, (D,), 0.3) + 1, seeded(4, (D,), 0.3) + 1
    dy = seeded(5, (B, H, T, D))
    tw = [torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in (x, w, wq, wk)]
    qkv = (tw[0] @ tw[1].T).view(B, T, 3 * H, D)
    n = qkv / torch.sqrt((qkv * qkv).mean(-1, keepdim=True) + 1e-6)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    c, s = ang.cos()[None, :, None], ang.sin()[None, :, None]
    rot = lambda u: torch.cat((u[..., :D // 2] * c - u[..., D // 2:] * s, u[..., D // 2:] * c + u[..., :D // 2] * s), -1)  # noqa: E731
    q, k, v = rot(n[:, :, :H] * tw[2]), rot(n[:, :, H:2 * H] * tw[3]), qkv[:, :, 2 * H:]
    q, k, v = (u.transpose(1, 2) for u in (q, k, v))
    mask = torch.ones(T, T).triu(1).bool()
    want = torch.softmax((q @ k.transpose(2, 3) * D ** -0.5).masked_fill(mask, -1e9), -1) @ v
    want.backward(torch.tensor(dy, dtype=torch.float64))
    with Eng("b200") as e:
        L = e.L
        ts = [e.param(a) for a in (x, w, wq, wk)]
        nd, shp = capi.shape_arg((B, T, 3 * H, D))
        qkv = e.check(L.nc_reshape(e.check(L.nc_linear_fn(ts[0], ts[1], None)), nd, shp))
        qk = e.check(L.nc_ext_qk_norm_rope(e.check(L.nc_slice(qkv, 2, 0, 2 * H, 1)), ts[2], ts[3], None, ctypes.byref(o)))
        head = lambda u, at: e.check(L.nc_transpose(e.check(L.nc_slice(u, 2, at, H, 1)), 1, 2))  # noqa: E731
        q, k, v = head(qk, 0), head(qk, H), head(qkv, 2 * H)
        sc = e.check(L.nc_scale(e.check(L.nc_matmul(q, e.check(L.nc_transpose(k, 2, 3)))), D ** -0.5))
        sc = e.check(L.nc_masked_fill(sc, e.t(np.triu(np.ones((T, T), np.int32), 1)), -1e9))
        out = e.check(L.nc_matmul(e.check(L.nc_softmax(sc)), v))
        from nchelp import rel_err
        assert L.nc_ext_backward_from(out, e.t(dy)) == 0, e.err()
        # 3xTF32 products of up to 64 terms and a softmax: well below 1e-4 of the largest value
        assert rel_err(e.np(out), want.detach().numpy()) < 1e-4
        for t, r in zip(ts, tw):
            assert rel_err(e.grad(t), r.grad.numpy()) < 1e-4
