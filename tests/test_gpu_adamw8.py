"""nc_ext_adamw8 (AdamW with 8-bit moments) and the device copies of optimizer state.

The moments are a function of the gradients alone, defined step by step in fp32 (include/nc_ext.h and the kernel's
header): the emulation below rounds each product and sum as numpy's float32 does and has to agree bit for bit. The
weights are compared with the step in 64 bits from the same moments. One step's error, e = 2^-24: w keep is rounded
once with the subtraction (e of w), keep itself once (e of w), and the step, at most lr m' / (sqrt(v') + eps), by rate,
root, its factor, the sum, the division and one product: below 24 e of the step.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
F = np.float32
BLOCK = 256
T_M = ((np.arange(1, 128) - 0.5) ** 2).astype(F)
T_V = ((np.arange(1, 256) - 0.5) ** 4).astype(F)
K_M, K_V = F(1.0 / 127 ** 2), F(1.0 / 255.0 ** 4)


def blocks(a):
    n = -(-a.size // BLOCK) * BLOCK
    b = np.zeros(n, F)
    b[:a.size] = a.ravel()
    return b.reshape(-1, BLOCK)


def through_codes(m, v):
    """what m and v (flat, of one parameter) read as after 8 bits"""
    n = m.size
    m, v = blocks(m), blocks(v)
    with np.errstate(all="ignore"):
        out = []
        for a, steps, full, unit, power in ((np.abs(m), T_M, F(127 ** 2), K_M, 2), (v, T_V, F(255.0 ** 4), K_V, 4)):
            top = a.max(1, keepdims=True)
            top = np.where(top < F(2.0 ** -94), F(0), top)
            share = a * np.where(top > 0, (F(1) / top) * full, F(0))
            c = np.searchsorted(steps, share, side="right").astype(F)
            if power == 4:
                c = np.where((a > 0) & (top > 0), np.maximum(c, F(1)), F(0))
                q = c * c
                val = np.where(c == 255, top, ((top * unit) * q) * q)
            else:
                val = np.where(c == 127, top, (top * unit) * (c * c))
                val = np.where((m < 0) & (c > 0), -val, val)  # code 0 has no sign
            out.append(val.ravel()[:n])
    return out


class Emulated:
    """The moments of each parameter, and the step of its weights in 64 bits."""

    def __init__(self, ws, lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, decay=0.01):
        self.h = tuple(F(x) for x in (lr, b1, b2, eps, decay))
        self.w = [w.astype(np.float64) for w in ws]
        self.m = [np.zeros(w.size, F) for w in ws]
        self.v = [np.zeros(w.size, F) for w in ws]
        self.off = [np.zeros(w.shape) for w in ws]
        self.t = 0

    def step(self, gs, scale=F(1)):
        lr, b1, b2, eps, decay = self.h
        self.t += 1
        bc1, bc2 = F(1) - np.power(b1, F(self.t)), F(1) - np.power(b2, F(self.t))
        for i, g in enumerate(gs):
            if g is None:
                continue
            g = (scale * g.ravel().astype(F)).astype(F)
            m = b1 * self.m[i] + (F(1) - b1) * g
            v = b2 * self.v[i] + ((F(1) - b2) * g) * g
            d = lambda x: np.asarray(x, np.float64)  # noqa: E731
            with np.errstate(invalid="ignore"):
                move = d(lr) * d(m) / d(bc1) / (np.sqrt(d(v) / d(bc2)) + d(eps))
            shape = self.w[i].shape
            self.off[i] += E * (2 * abs(self.w[i]) + 24 * abs(move.reshape(shape))) + 1e-30
            self.w[i] = self.w[i] * d(F(1) - lr * decay) - move.reshape(shape)
            self.m[i], self.v[i] = through_codes(m, v)


def opts(lr=1e-2, decay=0.01, b1=0.9, b2=0.999, eps=1e-8):
    return capi.OptimOpts(lr, 0.0, decay, b1, b2, eps)


def optimizer(e, ts, o=None, make="nc_ext_adamw8"):
    return e.check(getattr(e.L, make)(e.ctx, capi.ptr_array(ts), len(ts), o or opts()))


def give(e, ts, gs):
    """the gradients as a backward pass leaves them; None: the parameter is not reached"""
    for t, g in zip(ts, gs):
        e.L.nc_clear_grad(t)
        if g is not None:
            assert e.L.nc_ext_backward_from(t, e.t(g.astype(F))) == 0, e.err()


def state(e, o, n):
    e.L.nc_persistent_begin(e.ctx)
    t = e.check(e.L.nc_empty(e.ctx, capi.F32, *capi.shape_arg((2, n))))
    e.L.nc_persistent_end(e.ctx)
    assert e.L.nc_ext_optim_get_state(o, t) == 0, e.err()
    got = e.np(t)
    e.L.nc_release(t)
    return got


def same_bits(a, b):
    return np.array_equal(np.ascontiguousarray(a, F).view(np.uint32), np.ascontiguousarray(b, F).view(np.uint32))


def gradients(rng, shapes):
    """rows of very different sizes, zeros, one outlier a block"""
    out = []
    for s in shapes:
        g = rng.standard_normal(s) * np.exp(3 * rng.standard_normal(s)) * 1e-3
        g = np.where(rng.random(s) < 0.1, 0, g)
        out.append(g.astype(F))
    return out


SHAPES = [[(1,)], [(255,), (256,), (257,)], [(2047,), (2048,), (2049,), (3,)], [(0,), (17, 3), (0, 5), (64, 100)],
          [(700, 301), (5,), (4096,)]]


@pytest.mark.parametrize("shapes", SHAPES, ids=str)
def test_moments_bit_for_bit_and_weights(shapes):
    rng = np.random.default_rng(len(shapes))
    ws = [rng.standard_normal(s).astype(F) for s in shapes]
    n = sum(w.size for w in ws)
    em = Emulated(ws)
    with Eng("b200") as e:
        ts = [e.param(w) for w in ws]
        o = optimizer(e, ts)
        for k in range(6):
            gs = gradients(rng, shapes)
            give(e, ts, gs)
            e.L.nc_optim_step(o)
            em.step(gs)
            got = state(e, o, n)
            assert same_bits(got[0], np.concatenate(em.m)), k
            assert same_bits(got[1], np.concatenate(em.v)), k
            e.step_end()
        for t, w, off in zip(ts, em.w, em.off):
            assert np.all(abs(e.np(t) - w) <= off)
        assert e.L.nc_optim_get_step(o) == 6 and e.ok(), e.err()
        e.L.nc_optim_free(o)


def test_absent_gradients_accumulation_and_settings():
    """A parameter without a gradient keeps weights and moments; four micro-batches count as their mean; learning
    rate, options and step count apply from the next step."""
    rng = np.random.default_rng(3)
    shapes = [(300,), (1000,)]
    ws = [rng.standard_normal(s).astype(F) for s in shapes]
    em = Emulated(ws)
    with Eng("b200") as e:
        ts = [e.param(w) for w in ws]
        o = optimizer(e, ts)
        gs = gradients(rng, shapes)
        give(e, ts, gs)
        e.L.nc_optim_step(o)
        em.step(gs)
        only = [gradients(rng, shapes)[0], None]
        give(e, ts, only)
        e.L.nc_optim_step(o)
        em.step(only)
        assert same_bits(state(e, o, 1300), np.stack((np.concatenate(em.m), np.concatenate(em.v))))
        e.L.nc_optim_set_accumulation(o, 4)
        e.L.nc_optim_set_lr(o, 0.5)
        em.h = (F(0.5), *em.h[1:])
        gs = gradients(rng, shapes)
        give(e, ts, gs)
        before = [e.np(t) for t in ts]
        for _ in range(3):
            e.L.nc_optim_step(o)
            assert all(np.array_equal(e.np(t), b) for t, b in zip(ts, before))
        e.L.nc_optim_step(o)
        em.step(gs, F(0.25))
        e.L.nc_optim_set_accumulation(o, 1)
        e.L.nc_optim_set_opts(o, opts(1e-3, 0.2, 0.8, 0.99, 1e-6))
        e.L.nc_optim_set_step(o, 50)
        em.h, em.t = tuple(F(x) for x in (1e-3, 0.8, 0.99, 1e-6, 0.2)), 50
        e.L.nc_optim_step(o)
        em.step(gs)
        got = state(e, o, 1300)
        assert same_bits(got, np.stack((np.concatenate(em.m), np.concatenate(em.v))))
        for t, w, off in zip(ts, em.w, em.off):
            assert np.all(abs(e.np(t) - w) <= off)


def test_state_goes_out_and_comes_back_bit_for_bit():
    """Device copies and the host mirror: what was decoded encodes to the same codes, so a resumed run continues
    exactly as the one that went on."""
    rng = np.random.default_rng(4)
    shapes = [(513,), (40, 70), (7,)]
    n = sum(int(np.prod(s)) for s in shapes)
    ws = [rng.standard_normal(s).astype(F) for s in shapes]
    all_gs = [gradients(rng, shapes) for _ in range(6)]
    with Eng("b200") as e:
        def run(resume):
            ts = [e.param(w) for w in ws]
            o = optimizer(e, ts)
            for k, gs in enumerate(all_gs):
                if k == 3 and resume:
                    old = state(e, o, n)
                    new = optimizer(e, ts)
                    if resume == "device":
                        assert e.L.nc_ext_optim_put_state(new, e.t(old)) == 0, e.err()
                    else:
                        for i in range(len(ts)):
                            for slot in (0, 1):
                                size = ws[i].size * 4
                                src, dst = e.L.nc_optim_state(o, i, slot), e.L.nc_optim_state(new, i, slot)
                                assert src and dst and src != dst
                                ctypes.memmove(dst, src, size)
                    e.L.nc_optim_set_step(new, e.L.nc_optim_get_step(o))
                    e.L.nc_optim_free(o)
                    o = new
                    assert same_bits(state(e, o, n), old)
                give(e, ts, gs)
                e.L.nc_optim_step(o)
                e.step_end()
            got = state(e, o, n), [e.np(t) for t in ts]
            at = 0
            for i, w in enumerate(ws):  # the mirror shows the same values
                for slot in (0, 1):
                    p = ctypes.cast(e.L.nc_optim_state(o, i, slot), ctypes.POINTER(ctypes.c_float))
                    assert same_bits(np.ctypeslib.as_array(p, (w.size,)), got[0][slot, at:at + w.size])
                at += w.size
            e.L.nc_optim_free(o)
            return got

        want = run(None)
        for how in ("device", "host"):
            got = run(how)
            assert same_bits(got[0], want[0]) and all(same_bits(a, b) for a, b in zip(got[1], want[1]))


def test_every_code_survives():
    """Blocks whose values are each code's value, at sizes from 2^-90 to 2^100: decoding returns them unchanged."""
    c = np.arange(-127, 129)
    c[-1] = 5
    d = np.arange(256)
    rows = []
    for s in (F(2.0 ** -90), F(1.7e-7), F(1), F(3.3), F(2.0 ** 100)):
        cm, q = c.astype(F), (d * d).astype(F)
        m = np.where(abs(cm) == 127, np.copysign(s, cm), (s * K_M) * (cm * abs(cm))).astype(F)
        v = np.where(d == 255, s, ((s * K_V) * q) * q).astype(F)
        rows.append((m, v))
    m, v = (np.concatenate([r[k] for r in rows]) for k in (0, 1))
    with Eng("b200") as e:
        t = e.param(np.zeros(m.size, F))
        o = optimizer(e, [t])
        assert e.L.nc_ext_optim_put_state(o, e.t(np.stack((m, v)))) == 0, e.err()
        assert same_bits(state(e, o, m.size) + 0.0, np.stack((m, v)) + 0.0)


def test_small_shares_zeros_and_bad_gradients():
    rng = np.random.default_rng(5)
    n = 4 * BLOCK + 9
    w = rng.standard_normal(n).astype(F)
    g = rng.standard_normal(n).astype(F)
    g[1] = 1e9                    # the rest of block 0 is below the smallest share
    g[BLOCK:2 * BLOCK] = 0        # nothing in block 1
    g[2 * BLOCK:3 * BLOCK] = 1e-20  # v below 2^-94
    g[3 * BLOCK + 3] = np.nan
    g[-1] = np.inf
    em = Emulated([w])
    with Eng("b200") as e:
        t = e.param(w)
        o = optimizer(e, [t])
        give(e, [t], [g])
        e.L.nc_optim_step(o)
        m, v = state(e, o, n)
        got = e.np(t)
        em.step([g])
        ok = slice(0, 3 * BLOCK)
        assert same_bits(m[ok], em.m[0][ok]) and same_bits(v[ok], em.v[0][ok])
        assert np.all(abs(got[ok] - em.w[0][ok]) <= em.off[0][ok])
        assert (v[:BLOCK] > 0).all() and not m[BLOCK:2 * BLOCK].any() and not v[BLOCK:3 * BLOCK].any()
        assert not np.isfinite(m[3 * BLOCK:]).any() and not np.isfinite(v[3 * BLOCK:4 * BLOCK]).any()
        assert np.isfinite(got[ok]).all() and np.isnan(got[3 * BLOCK + 3])
        assert np.isfinite(np.delete(got[3 * BLOCK:4 * BLOCK], 3)).all()  # the step itself is per element


def test_follows_adamw_on_a_problem():
    """Least squares with a few thousand weights: after 60 steps the 8-bit run stands within a few percent of the
    way of the fp32 run (steps are rounded to 1 / 127 of a block's largest root at worst, without a bias)."""
    rng = np.random.default_rng(6)
    w0, goal = rng.standard_normal((2, 3000)).astype(F)
    ends = []
    with Eng("b200") as e:
        for make in ("nc_adamw", "nc_ext_adamw8"):
            t = e.param(w0)
            o = optimizer(e, [t], opts(2e-2, 0.0), make)
            for _ in range(60):
                give(e, [t], [e.np(t) - goal])
                e.L.nc_optim_step(o)
                e.step_end()
            ends.append(e.np(t))
            e.L.nc_optim_free(o)
    way = np.linalg.norm(ends[0] - w0)
    assert np.linalg.norm(ends[1] - ends[0]) < 0.1 * way


def test_state_copies_of_other_optimizers_and_refusals():
    rng = np.random.default_rng(7)
    ws = [rng.standard_normal(s).astype(F) for s in ((5,), (3, 7))]
    gs = [rng.standard_normal(w.shape).astype(F) for w in ws]
    with Eng("b200") as e:
        ts = [e.param(w) for w in ws]
        o = optimizer(e, ts, opts(), "nc_adam")
        give(e, ts, gs)
        e.L.nc_optim_step(o)
        got = state(e, o, 26)
        flat = np.concatenate([(g + F(0.01) * w).ravel() for g, w in zip(gs, ws)])  # Adam's decay is part of the gradient
        assert np.allclose(got[0], 0.1 * flat, rtol=1e-5) and np.allclose(got[1], 0.001 * flat * flat, rtol=1e-4)
        assert e.L.nc_ext_optim_put_state(o, e.t(2 * got)) == 0 and same_bits(state(e, o, 26), 2 * got)
        p = ctypes.cast(e.L.nc_optim_state(o, 1, 1), ctypes.POINTER(ctypes.c_float))
        assert p[0] == 2 * got[1, 5]
        o8 = optimizer(e, ts)
        for t, text, code in ((e.t(np.zeros((2, 25), F)), "expected", 1), (e.t(np.zeros(52, F)), "expected", 1),
                              (e.t(np.zeros((2, 26), np.int32)), "f32", 2),
                              (e.L.nc_transpose(e.t(np.zeros((26, 2), F)), 0, 1), "expected", 1)):
            for call in (e.L.nc_ext_optim_get_state, e.L.nc_ext_optim_put_state):
                for opt in (o, o8):
                    assert call(opt, t) == code and text in e.err()
                    e.L.nc_clear_error(e.ctx)
        sgd = optimizer(e, ts, opts(), "nc_sgd")
        assert e.L.nc_ext_optim_get_state(sgd, e.t(got)) == 5 and "two moments" in e.err()
        e.L.nc_clear_error(e.ctx)
        assert e.L.nc_ext_optim_get_state(None, e.t(got)) == 4 and e.L.nc_ext_optim_put_state(o8, None) == 4
        with Eng("b200") as other:
            assert e.L.nc_ext_optim_put_state(o8, other.t(got)) == 4 and "another context" in e.err()
            e.L.nc_clear_error(e.ctx)
        assert not e.L.nc_ext_adamw8(e.ctx, capi.ptr_array([e.t(ws[0])]), 1, opts()) and "parameter" in e.err()
        e.L.nc_clear_error(e.ctx)
        assert not e.L.nc_ext_adamw8(e.ctx, None, 1, opts()) and not e.L.nc_ext_adamw8(None, None, 0, opts())
        e.L.nc_clear_error(e.ctx)
        empty = optimizer(e, [])
        e.L.nc_optim_step(empty)
        assert e.L.nc_ext_optim_get_state(empty, e.t(np.zeros((2, 0), F))) == 0 and e.ok(), e.err()


@pytest.mark.parametrize("eight", [True, False])
def test_state_over_a_tensor_that_something_pending_reads(eight):
    w = np.random.default_rng(9).standard_normal((3, 200)).astype(F)
    vals = np.random.default_rng(10).standard_normal((2, 600)).astype(F)
    with Eng("b200") as e:
        t = e.param(w)
        o = optimizer(e, [t], make="nc_ext_adamw8" if eight else "nc_adamw")
        tv = e.t(vals)
        want = e.np(e.check(e.L.nc_gelu(e.t(vals), 0)))
        y = e.check(e.L.nc_gelu(tv, 0))
        assert e.L.nc_ext_optim_get_state(o, tv) == 0, e.err()
        assert np.array_equal(e.np(y), want) and not e.np(tv).any()


def test_parameter_of_more_than_2_to_the_31_elements():
    """Offsets past 32 bits: the last elements of one parameter of 2^31 + 777."""
    import torch

    n = 2 ** 31 + 777
    if torch.cuda.get_device_properties(0).total_memory < 80 << 30:
        pytest.skip("needs 40 GB")
    rng = np.random.default_rng(8)
    tail = 777 + 2 * BLOCK
    w, g = rng.standard_normal(tail).astype(F), gradients(rng, [(tail,)])[0]
    em = Emulated([w])
    with Eng("b200") as e:
        t = e.check(e.L.nc_parameter(e.ctx, None, *capi.shape_arg((n,))))
        o = optimizer(e, [t])

        def view(x):
            p = e.L.nc_ext_device_data(x, 1)
            e.L.nc_ext_synchronize(e.ctx)
            face = type("Face", (), {"__cuda_array_interface__": dict(shape=(n,), typestr="<f4", data=(p, False), version=2)})
            return torch.as_tensor(face(), device="cuda")

        view(t)[-tail:].copy_(torch.from_numpy(w))
        torch.cuda.synchronize()
        assert e.L.nc_ext_backward_from(t, t) == 0, e.err()  # a gradient of the whole: the weights
        view(e.L.nc_grad(t)).zero_()[-tail:].copy_(torch.from_numpy(g))
        torch.cuda.synchronize()
        e.L.nc_optim_step(o)
        em.step([g])
        got = view(t)
        assert np.all(abs(got[-tail:].cpu().numpy() - em.w[0]) <= em.off[0])
        assert int(torch.count_nonzero(got[:-tail])) == 0
        e.L.nc_optim_free(o)
        e.L.nc_release(t)
