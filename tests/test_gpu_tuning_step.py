"""One tuning step of a small language model out of the framework's operators, as they are used together: fused
projection, query/key norms with rotary positions, the framework's attention, a linear head, the policy loss or the
preference loss, and AdamW with 8-bit moments; against the same model in torch in 64 bits.

Bounds: every product runs as 3xTF32 or exact fp32 (relative error below 1e-5 of the largest value at these sizes, as
tests/test_gpu_gemm.py holds it to), and the chain has about ten of them one after the other, so losses and gradients
are held to 1e-4 of the largest value. Weights after AdamW's first step from zero moments move by lr sign(g) whatever
the gradient's size: they are compared where |g| is above 1e-3 of the largest, with the same relative bound of lr.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from nchelp import Eng, capi, rel_err, seeded

pytestmark = pytest.mark.gpu
B, T, C, H, V = 4, 12, 64, 4, 50
D = C // H
NAMES = ("emb", "qkv", "proj", "wq", "wk", "head")


def weights():
    shapes = {"emb": (V, C), "qkv": (3 * C, C), "proj": (C, C), "wq": (D,), "wk": (D,), "head": (V, C)}
    w = {n: seeded(i + 1, s, 0.5 if n == "emb" else 0.15) for i, (n, s) in enumerate(shapes.items())}
    w["wq"], w["wk"] = w["wq"] + 1, w["wk"] + 1
    return w


def batch():
    rng = np.random.default_rng(20)
    ids = rng.integers(0, V, (B, T)).astype(np.int32)
    act = rng.integers(0, V, (B, T - 1)).astype(np.int32)
    mask = (np.arange(T - 1)[None] < np.array([[11], [3], [0], [7]])).astype(np.int32)  # one answer is empty
    return ids, act, mask, rng


def torch_model(w):
    import torch

    p = {n: torch.tensor(v, dtype=torch.float64, requires_grad=True) for n, v in w.items()}
    ang = torch.arange(T, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    c, s = ang.cos()[None, :, None], ang.sin()[None, :, None]
    mask = torch.ones(T, T).triu(1).bool()

    def logits(ids):
        x = p["emb"][torch.tensor(ids.astype(np.int64))]
        qkv = (x @ p["qkv"].T).view(B, T, 3 * H, D)
        n = qkv / torch.sqrt((qkv * qkv).mean(-1, keepdim=True) + 1e-6)
        rot = lambda u: torch.cat((u[..., :D // 2] * c - u[..., D // 2:] * s, u[..., D // 2:] * c + u[..., :D // 2] * s), -1)  # noqa: E731
        q, k, v = (u.transpose(1, 2) for u in (rot(n[:, :, :H] * p["wq"]), rot(n[:, :, H:2 * H] * p["wk"]), qkv[:, :, 2 * H:]))
        a = torch.softmax((q @ k.transpose(2, 3) * D ** -0.5).masked_fill(mask, -1e9), -1) @ v
        x = x + a.transpose(1, 2).reshape(B, T, C) @ p["proj"].T
        return x @ p["head"].T

    return p, logits


def engine_logits(e, p, ids, opts):
    L, ck = e.L, e.check
    rs = lambda t, *s: ck(L.nc_reshape(t, *capi.shape_arg(s)))  # noqa: E731
    x = rs(ck(L.nc_index_select(p["emb"], e.t(ids.ravel()))), B, T, C)
    qkv = rs(ck(L.nc_linear_fn(x, p["qkv"], None)), B, T, 3 * H, D)
    qk = ck(L.nc_ext_qk_norm_rope(ck(L.nc_slice(qkv, 2, 0, 2 * H, 1)), p["wq"], p["wk"], None, ctypes.byref(opts)))
    head = lambda u, at: ck(L.nc_transpose(ck(L.nc_slice(u, 2, at, H, 1)), 1, 2))  # noqa: E731
    q, k, v = head(qk, 0), head(qk, H), head(qkv, 2 * H)
    sc = ck(L.nc_scale(ck(L.nc_matmul(q, ck(L.nc_transpose(k, 2, 3)))), D ** -0.5))
    sc = ck(L.nc_masked_fill(sc, e.t(np.triu(np.ones((T, T), np.int32), 1)), -1e9))
    a = ck(L.nc_matmul(ck(L.nc_softmax(sc)), v))
    a = rs(ck(L.nc_contiguous(ck(L.nc_transpose(a, 1, 2)))), B, T, C)
    x = ck(L.nc_add(x, ck(L.nc_linear_fn(a, p["proj"], None))))
    return ck(L.nc_linear_fn(x, p["head"], None))


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_tuning_step(loss):
    import torch

    w = weights()
    ids, act, mask, rng = batch()
    p64, logits64 = torch_model(w)
    z = logits64(ids)[:, :-1]
    lp = torch.log_softmax(z, -1).gather(-1, torch.tensor(act.astype(np.int64))[..., None])[..., 0]
    m = torch.tensor(mask)
    if loss == "policy":
        old = (lp.detach().numpy() + 0.3 * rng.standard_normal((B, T - 1))).astype(np.float32)
        ref = (lp.detach().numpy() + 0.3 * rng.standard_normal((B, T - 1))).astype(np.float32)
        adv = rng.standard_normal((B, T - 1)).astype(np.float32)
        r, A = torch.exp(lp - torch.tensor(old)), torch.tensor(adv).double()
        away = torch.tensor(ref) - lp
        each = -torch.minimum(r * A, r.clamp(0.8, 1.25) * A) + 0.1 * (torch.exp(away) - away - 1)
        want = (each * m).sum() / m.sum()
    else:
        ref = rng.standard_normal(B).astype(np.float32)
        gap = (lp * m).sum(1) - torch.tensor(ref)
        want = -torch.nn.functional.logsigmoid(0.5 * (gap[:2] - gap[2:])).mean()
    want.backward()
    want = float(want.detach())
    lr = 1e-3
    opts = capi.RopeOpts(H, 1, (ctypes.c_int * 3)(D // 2), 10000.0, 1e-6, 0)
    with Eng("b200") as e:
        p = {n: e.param(v) for n, v in w.items()}
        o = e.check(e.L.nc_ext_adamw8(e.ctx, capi.ptr_array([p[n] for n in NAMES]), len(NAMES),
                                      capi.OptimOpts(lr, 0.0, 0.0, 0.9, 0.999, 1e-8)))
        for step in range(3):  # the first step against torch, then the loss has to stay finite and the graph reusable
            z = e.check(e.L.nc_slice(engine_logits(e, p, ids, opts), 1, 0, T - 1, 1))
            if loss == "policy":
                tl = e.check(e.L.nc_ext_policy_loss(z, e.t(act), e.t(old), e.t(ref), e.t(adv), e.t(mask),
                                                    ctypes.byref(capi.PolicyOpts(0.2, 0.25, 0.1)), None))
            else:
                tl = e.check(e.L.nc_ext_preference_loss(z, e.t(act), e.t(ref), e.t(mask), 0.5, 0.0, None))
            e.L.nc_optim_clear_grad(o)
            assert e.L.nc_backward_ex(tl, 1, None, 0) == 0, e.err()
            got = float(e.np(tl))
            if step == 0:
                assert abs(got - want) < 1e-4 * max(1, abs(want))
                for n in NAMES:
                    assert rel_err(e.grad(p[n]), p64[n].grad.numpy()) < 1e-4, n
            e.L.nc_optim_step(o)
            if step == 0:
                for n in NAMES:
                    g = p64[n].grad.numpy()
                    big = np.abs(g) > 1e-3 * np.abs(g).max()
                    step_of = (w[n] - e.np(p[n]))[big]
                    assert np.all(np.abs(step_of - lr * np.sign(g[big])) < 1e-3 * lr + 2.0 ** -23 * np.abs(w[n][big]) + 1e-4 * lr), n
            assert np.isfinite(got)
            e.step_end()
        assert e.ok(), e.err()
        e.L.nc_optim_free(o)


def test_two_contexts_at_once():
    """Two contexts (streams, scratch) with their operators interleaved give what each gives alone, bit for bit."""
    z, act = seeded(1, (300, 777), 2.0), np.random.default_rng(2).integers(0, 777, 300).astype(np.int32)
    old, adv = seeded(3, (300,)) - 6, seeded(4, (300,))
    x, wt = seeded(5, (2, 100, 6, 64)), seeded(6, (64,)) + 1
    ro = capi.RopeOpts(4, 1, (ctypes.c_int * 3)(32), 10000.0, 1e-6, 0)
    po = capi.PolicyOpts(0.2, 0.2, 0.0)

    def start(e):
        tz, tx, tw = e.param(z), e.param(x), e.param(wt)
        tl = e.check(e.L.nc_ext_policy_loss(tz, e.t(act), e.t(old), None, e.t(adv), None, ctypes.byref(po), None))
        y = e.check(e.L.nc_ext_qk_norm_rope(tx, tw, tw, None, ctypes.byref(ro)))
        return tz, tx, tw, tl, y

    def end(e, tz, tx, tw, tl, y):
        e.L.nc_backward(tl)
        e.L.nc_ext_backward_from(y, tx)
        return [e.np(tl), e.grad(tz), e.np(y), e.grad(tx), e.grad(tw)]

    with Eng("b200") as e:
        alone = end(e, *start(e))
    with Eng("b200") as a, Eng("b200") as b:
        sa, sb = start(a), start(b)
        for e, s in ((a, sa), (b, sb)):
            for u, v in zip(end(e, *s), alone):
                assert np.array_equal(u, v)


@pytest.mark.parametrize("rows", [8, 100, 400, 1600, 8 * 200 * 6])
def test_steps_back_to_back_are_steps_one_by_one(rows):
    """Kernels take their places while the one before ends, and each reads what that one wrote (rows of 76800 to 64
    logits: every way the losses run): 25 steps without a pause give the weights and moments of 25 steps with the host
    waiting after every call, bit for bit."""
    x, wt = seeded(1, (8, 200, 6, 64)), seeded(2, (64,)) + 1
    V = x.size // rows
    rng = np.random.default_rng(3)
    act, adv = rng.integers(0, V, rows).astype(np.int32), seeded(4, (rows,))
    old, mask = np.full(rows, -np.log(V), np.float32), (rng.random(rows) < 0.8).astype(np.int32)
    ro, po = capi.RopeOpts(4, 1, (ctypes.c_int * 3)(32), 10000.0, 1e-6, 0), capi.PolicyOpts(0.2, 0.2, 0.0)

    def run(pause):
        with Eng("b200") as e:
            wait = (lambda: e.L.nc_ext_synchronize(e.ctx)) if pause else (lambda: None)
            e.L.nc_persistent_begin(e.ctx)
            fixed = [e.t(v) for v in (act, old, adv, mask)]
            state = e.t(np.zeros((2, x.size + 64), np.float32))
            e.L.nc_persistent_end(e.ctx)
            tx, tw = e.param(x), e.param(wt)
            o = e.check(e.L.nc_ext_adamw8(e.ctx, capi.ptr_array([tx, tw]), 2, capi.OptimOpts(1e-2, 0.0, 0.01, 0.9, 0.999, 1e-8)))
            for _ in range(25):
                y = e.check(e.L.nc_ext_qk_norm_rope(tx, tw, tw, None, ctypes.byref(ro)))
                wait()
                z = e.check(e.L.nc_reshape(y, *capi.shape_arg((rows, V))))
                loss = e.check(e.L.nc_ext_policy_loss(z, fixed[0], fixed[1], None, fixed[2], fixed[3], ctypes.byref(po), None))
                wait()
                e.L.nc_optim_clear_grad(o)
                assert e.L.nc_backward_ex(loss, 1, None, 0) == 0, e.err()
                wait()
                e.L.nc_optim_step(o)
                wait()
                assert e.L.nc_ext_optim_get_state(o, state) == 0, e.err()
                wait()
                e.step_end()
            out = [e.np(t) for t in (tx, tw, state)]
            e.L.nc_optim_free(o)
            return out

    for a, b in zip(run(True), run(False)):
        assert np.isfinite(a).all() and np.array_equal(a, b)
