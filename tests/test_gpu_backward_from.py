"""nc_ext_backward_from with a gradient that an earlier pass left: a retained pass keeps the gradients of intermediate
tensors, and the pass that follows starts those from zero. The given gradient is read as it was and left as it was.

Bounds: a sum of K products has at most K roundings of the sum of absolute values (3xTF32 drops 2^-21 of each product),
and tanh and its slope 1 - y^2 are off by less than 2^-20 of 1.
"""

from __future__ import annotations

import numpy as np
import pytest

from nchelp import Eng, capi, seeded

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
RETAIN = 2
N = 24  # square, so that every gradient of the graph can stand for every other one


def build(e):
    """x and w (leaves), h = x w^T, y = tanh(h) and z = y w^T, after a retained pass from sum(z * G)"""
    tx, tw = e.param(seeded(1, (N, N))), e.param(seeded(2, (N, N), 0.3))
    h = e.check(e.L.nc_linear_fn(tx, tw, None))
    y = e.check(e.L.nc_tanh(h))
    z = e.check(e.L.nc_linear_fn(y, tw, None))
    loss = e.check(e.L.nc_sum(e.check(e.L.nc_mul(z, e.t(seeded(3, (N, N))))), capi.ALL_AXES, 0))
    assert e.L.nc_backward_ex(loss, RETAIN, None, 0) == 0, e.err()
    for t in (tx, tw):
        e.L.nc_clear_grad(t)
    return tx, tw, dict(h=h, y=y, z=z)


def formula(root, dy):
    """gradients of x and w from d root = dy, and the sums of absolute values that their bounds multiply"""
    x, w, dy = seeded(1, (N, N)).astype(np.float64), seeded(2, (N, N), 0.3).astype(np.float64), dy.astype(np.float64)
    y = np.tanh(x @ w.T)
    gw, gws, size = np.zeros((N, N)), np.zeros((N, N)), abs(dy)
    if root == "z":
        gw, gws = dy.T @ y, size.T @ abs(y)
        dy, size = dy @ w, size @ abs(w)
    if root in ("z", "y"):
        dy = dy * (1 - y * y)
    return dy @ w, size @ abs(w), gw + dy.T @ x, gws + size.T @ abs(x)


@pytest.mark.parametrize("kind", ["whole", "view", "pending"])
@pytest.mark.parametrize("root,of", [("y", "y"), ("h", "h"), ("y", "h"), ("z", "h"), ("z", "z"), ("z", "y")])
def test_dy_is_a_gradient_that_a_retained_pass_left(root, of, kind):
    with Eng("b200") as e:
        tx, tw, t = build(e)
        g = e.check(e.L.nc_grad(t[of]))
        left = e.np(g)
        assert left.any()
        dy, value = g, left
        if kind == "view":
            dy, value = e.check(e.L.nc_transpose(g, 0, 1)), left.T
        elif kind == "pending":
            dy, value = e.check(e.L.nc_gelu(g, 0)), e.np(e.check(e.L.nc_gelu(e.t(left), 0)))
        assert e.L.nc_ext_backward_from(t[root], dy) == 0, e.err()
        gx, gxs, gw, gws = formula(root, value)
        unit = 3 * N * E + 2.0 ** -18
        assert np.all(abs(e.grad(tx) - gx) <= unit * gxs) and np.all(abs(e.grad(tw) - gw) <= unit * gws)
        assert np.array_equal(e.np(dy), value)  # as it was
        if kind != "pending":
            assert np.array_equal(e.np(g), left)
        assert e.ok(), e.err()


def test_two_passes_from_the_same_left_gradient():
    with Eng("b200") as e:
        tx, tw, t = build(e)
        g = e.check(e.L.nc_grad(t["y"]))
        left = e.np(g)
        grads = []
        for _ in range(2):
            assert e.L.nc_ext_backward_from(t["z"], g) == 0, e.err()
            grads.append((e.grad(tx), e.grad(tw)))
            for p in (tx, tw):
                e.L.nc_clear_grad(p)
        assert all(np.array_equal(a, b) for a, b in zip(*grads)) and grads[0][0].any()
        assert np.array_equal(e.np(g), left)


@pytest.mark.parametrize("first", [0, 1, 2, 3])
@pytest.mark.parametrize("op", ["tanh", "linear", "layer_norm", "softmax", "rope"])
def test_dy_begins_at_any_element(op, first):
    """A contiguous dy within a larger tensor, off every 16-byte boundary, is read where it is: the gradients are those
    of a dy with memory of its own, but for the order of sums."""
    import ctypes

    B, D = 64, 128
    x, w, dy = seeded(1, (B, D)), seeded(2, (D, D), 0.2), seeded(3, (B, D))
    with Eng("b200") as e:
        tx, tw, tv = e.param(x), e.param(w), e.param(1 + w[0])
        o = capi.RopeOpts(1, 1, (ctypes.c_int * 3)(16), 10000.0, 1e-6, 0)
        run = {"tanh": lambda: e.L.nc_tanh(tx), "linear": lambda: e.L.nc_linear_fn(tx, tw, tv),
               "layer_norm": lambda: e.L.nc_layer_norm(tx, 1, tv, None, 1e-5), "softmax": lambda: e.L.nc_softmax(tx),
               "rope": lambda: e.L.nc_reshape(e.check(e.L.nc_ext_qk_norm_rope(
                   e.check(e.L.nc_reshape(tx, *capi.shape_arg((1, B, 4, 32)))), None, None, None, ctypes.byref(o))),
                   *capi.shape_arg((B, D)))}[op]
        got = []
        for at in (None, first):
            flat = e.t(np.concatenate((np.zeros(at or 0, np.float32), dy.ravel())))
            td = flat if at is None else e.check(e.L.nc_slice(flat, 0, at, B * D, 1))
            td = e.check(e.L.nc_reshape(td, *capi.shape_arg((B, D))))
            assert e.L.nc_ext_backward_from(e.check(run()), td) == 0, e.err()
            got.append([e.grad(t) for t in (tx, tw, tv)])
            for t in (tx, tw, tv):
                e.L.nc_clear_grad(t)
            assert np.array_equal(e.np(td), dy)
        for a, b in zip(*got):
            assert (a is None) == (b is None)
            assert a is None or np.abs(a - b).max() <= 2 * B * E * np.abs(a).max() + 1e-30
        assert got[0][0].any() and e.ok(), e.err()


@pytest.mark.parametrize("cleared", [False, True])
def test_a_left_gradient_of_a_tensor_with_two_consumers(cleared):
    """h feeds two ops, so its new gradient is a sum of two; whether the old one, which is dy, was cleared before."""
    with Eng("b200") as e:
        tx, tw = e.param(seeded(1, (N, N))), e.param(seeded(2, (N, N), 0.3))
        h = e.check(e.L.nc_linear_fn(tx, tw, None))
        z = e.check(e.L.nc_mul(e.check(e.L.nc_tanh(h)), e.check(e.L.nc_sigmoid(h))))
        loss = e.check(e.L.nc_sum(e.check(e.L.nc_mul(z, e.t(seeded(3, (N, N))))), capi.ALL_AXES, 0))
        assert e.L.nc_backward_ex(loss, RETAIN, None, 0) == 0, e.err()
        g = e.check(e.L.nc_grad(h))
        left = e.np(g)
        for t in (tx, tw) + ((h, z) if cleared else ()):
            e.L.nc_clear_grad(t)
        assert e.L.nc_ext_backward_from(z, g) == 0, e.err()
        x, w = seeded(1, (N, N)).astype(np.float64), seeded(2, (N, N), 0.3).astype(np.float64)
        y, s = np.tanh(x @ w.T), 1 / (1 + np.exp(-x @ w.T))
        dh, size = left * ((1 - y * y) * s + y * s * (1 - s)), abs(left)
        unit = 3 * N * E + 2.0 ** -18
        assert np.all(abs(e.grad(tx) - dh @ w) <= unit * (size @ abs(w)))
        assert np.all(abs(e.grad(tw) - dh.T @ x) <= unit * (size.T @ abs(x)))
        assert np.array_equal(e.np(g), left)


def test_a_cleared_gradient_that_a_pass_dropped():
    """nc_backward's own way to the same place: a retained pass, the gradient of h cleared, a pass that does not reach
    h's consumers but drops its gradient, and one that reaches both."""
    with Eng("b200") as e:
        tx = e.param(seeded(1, (N, N)))
        h = e.check(e.L.nc_scale(tx, 0.5))
        y, s = e.check(e.L.nc_tanh(h)), e.check(e.L.nc_sigmoid(h))
        z = e.check(e.L.nc_mul(y, s))
        loss = lambda t: e.check(e.L.nc_sum(t, capi.ALL_AXES, 0))  # noqa: E731
        want = []
        for clear in (False, True):
            assert e.L.nc_backward_ex(loss(z), RETAIN, None, 0) == 0, e.err()
            if clear:
                e.L.nc_clear_grad(h)
            assert e.L.nc_backward(loss(e.check(e.L.nc_scale(h, 2.0)))) == 0, e.err()
            if clear:
                e.L.nc_clear_grad(h)
            e.L.nc_clear_grad(tx)
            assert e.L.nc_backward(loss(z)) == 0, e.err()
            want.append(e.grad(tx))
            e.L.nc_clear_grad(tx)
        assert np.array_equal(*want) and want[0].any()
