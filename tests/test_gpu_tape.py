"""The gated scan and the 8-bit activations through tensors and the autograd tape: views, shapes, errors, and a layer's gradients."""
import numpy as np
import pytest

import sequence_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from rtensors_amd import tensor as T
    b = T.Backend(0)
    yield b
    b.sync()


def dev(be, a):
    from rtensors_amd import tensor as T
    name = {np.float32: "f32", np.float64: "f64", np.bool_: "bool"}[a.dtype.type]
    return T.Tensor.from_buf(be, name, a.reshape(-1), list(a.shape))


def close(got, want, M, S, form, dtype):
    bound = R.scan_bound(form, dtype, M, S)
    assert got.shape == want.shape and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_scan_along_any_axis(be, axis, form):
    rng = np.random.default_rng(axis)
    shape = (5, 70, 33)
    gate, x = 1 / (1 + np.exp(-rng.standard_normal((2,) + shape)))
    lead, rest = shape[:axis + 1], shape[:axis] + shape[axis + 1:]
    state, reset = rng.standard_normal(rest), rng.random(lead) < 0.1
    outer, steps, inner = int(np.prod(shape[:axis])), shape[axis], int(np.prod(shape[axis + 1:]))
    want, M, S = R.scan(form, gate.reshape(outer, steps, inner), x.reshape(outer, steps, inner), state.reshape(outer, inner), reset.reshape(outer, steps))
    h, last = dev(be, x).gated_scan(dev(be, gate), axis, form, dev(be, state), dev(be, reset), want_last=True)
    assert h.shape == list(shape) and last.shape == list(rest)
    close(h.to_numpy().reshape(outer, steps, inner), want, M, S, form, np.float64)
    assert (last.to_numpy().reshape(outer, inner) == h.to_numpy().reshape(outer, steps, inner)[:, -1]).all()


def test_scan_of_views(be):
    """Permuted, sliced and reversed operands give what their copies give."""
    from rtensors_amd.tensor import Slice
    rng = np.random.default_rng(3)
    a, g = rng.standard_normal((40, 6, 50)).astype(np.float32), rng.random((50, 6, 42)).astype(np.float32)
    x = dev(be, a).permute([2, 1, 0])
    gate = dev(be, g).slice(2, Slice.range(1, 41)).slice(0, Slice(49, None, -1))
    r = rng.random((50, 12)) < 0.2
    reset = dev(be, r).slice(1, Slice(0, 12, 2))
    an, gn, rn = a.transpose(2, 1, 0), g[::-1, :, 1:41], r[:, ::2]
    assert x.shape == gate.shape == [50, 6, 40] and reset.shape == [50, 6]
    got = x.gated_scan(gate, 1, "sigmoid", reset=reset).to_numpy()
    want = dev(be, np.ascontiguousarray(an)).gated_scan(dev(be, np.ascontiguousarray(gn)), 1, "sigmoid", reset=dev(be, np.ascontiguousarray(rn))).to_numpy()
    assert got.tobytes() == want.tobytes()
    p = x.pack8().unpack8()
    c, e = R.pack(np.ascontiguousarray(an).reshape(-1))
    assert p.shape == [50, 6, 40] and (p.to_numpy().reshape(-1) == R.restore(c, e, np.float32)).all()


def test_errors(be):
    from rtensors_amd import tensor as T
    z = lambda *s, dt="f32": T.Tensor.zeros(be, dt, list(s))
    x = z(3, 4, 5)
    for call, kind in ((lambda: x.gated_scan(z(3, 4, 5), 3), "InvalidDim"), (lambda: x.gated_scan(z(3, 5, 4), 1), "InvalidShape"),
                       (lambda: x.gated_scan(z(3, 4, 5, dt="f64"), 1), "UnsupportedOperation"), (lambda: x.gated_scan(z(3, 4, 5), 1, state=z(3, 4)), "InvalidShape"),
                       (lambda: x.gated_scan(z(3, 4, 5), 1, reset=z(3, 4)), "UnsupportedOperation"),
                       (lambda: x.gated_scan(z(3, 4, 5), 1, reset=z(3, 5, dt="bool")), "InvalidShape"),
                       (lambda: z(3, 4, dt="i32").gated_scan(z(3, 4, dt="i32"), 0), "UnsupportedOperation"), (lambda: z(3, dt="i32").pack8(), "UnsupportedOperation"),
                       (lambda: x.unary_pack8("relu"), "UnsupportedOperation"), (lambda: z(3, 4).unary_backward_pack8("silu", x.pack8()), "InvalidShape"),
                       (lambda: z(3, 6, 5).matmul_backward_pack8(x.pack8()), "InvalidShape"), (lambda: z(4, 5).matmul_backward_pack8(x.pack8()), "InvalidShape"),
                       (lambda: z(3, 4, 5, dt="f64").unary_backward_pack8("silu", x.pack8()), "UnsupportedOperation"),
                       (lambda: z(3, 4, 5, dt="f64").matmul_backward_pack8(x.pack8()), "UnsupportedOperation")):
        with pytest.raises(T.TensorError) as e:
            call()
        assert e.value.kind == kind, (e.value.kind, str(e.value))


def test_matmul_gradient_of_a_batch(be):
    rng = np.random.default_rng(5)
    x, dy = rng.standard_normal((2, 3, 70, 40)), rng.standard_normal((2, 3, 70, 24))
    got = dev(be, dy).matmul_backward_pack8(dev(be, x).pack8())
    c, e = R.pack(x.reshape(-1))
    xr = R.restore(c, e, np.float64).reshape(x.shape)
    want = np.matmul(np.swapaxes(xr, -1, -2), dy)
    assert got.shape == [2, 3, 40, 24]
    assert (np.abs(got.to_numpy() - want) <= 74 * 2.0 ** -53 * 1.01 * np.matmul(np.swapaxes(np.abs(xr), -1, -2), np.abs(dy))).all()


def layer(rng, tokens, d, f, e, dtype=np.float64):
    ws = [rng.standard_normal(s) / np.sqrt(s[0]) for s in ((d, f), (d, f), (f, e))]
    return [a.astype(dtype) for a in (rng.standard_normal((tokens, d)), *ws, rng.standard_normal((tokens, e)))]


def held(a, packed):
    if not packed:
        return a
    c, e = R.pack(np.ascontiguousarray(a).reshape(-1))
    return R.restore(c, e, a.dtype.type).reshape(a.shape)


def sigmoid(x):
    return 1 / (1 + np.exp(-x))


def by_hand(x, wg, wv, wo, target, reset, packed):
    """Loss and weight gradients from the formulas, with what the tape holds in 8 bits in its place."""
    g, u = x @ wg, x @ wv
    v = u * sigmoid(u)
    h = R.scan("sigmoid", g[None], v[None], None, None if reset is None else reset[None])[0][0].astype(np.float64)
    y = h @ wo
    dy = np.sign(y - target) / float(np.float32(y.size))
    x8, u8, v8, h8 = (held(a, packed) for a in (x, u, v, h))
    (dg, _), (dv, _), _ = R.scan_backward("sigmoid", g[None], v8[None], h8[None], (dy @ wo.T)[None], None, None if reset is None else reset[None])
    dg, dv = dg[0].astype(np.float64), dv[0].astype(np.float64)
    s = sigmoid(u8)
    du = dv * s * (1 + u8 * (1 - s))
    return np.abs(y - target).mean(), [x8.T @ dg, x8.T @ du, h8.T @ dy]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("tokens, d, f, e", [(1, 8, 5, 3), (50, 16, 33, 7), (300, 40, 64, 20), (700, 32, 9, 16)])
def test_layer_gradients(be, tokens, d, f, e, packed):
    """The three gradients of a layer against the formulas in doubles.  Sums of at most a few thousand terms: 1e-10 of the largest element
    is four orders above their rounding, and far below one step of an 8-bit code (1 / 127), which a value on a code's border would move."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(tokens)
    a = layer(rng, tokens, d, f, e)
    reset = rng.random(tokens) < 0.02
    loss, grads, kept = T.gated_layer_step(*[dev(be, t) for t in a], 0.0, reset=dev(be, reset), packed=packed, seed_with_loss=False)
    want_loss, want = by_hand(*a, reset, packed)
    assert abs(loss.to_numpy().reshape(-1)[0] - want_loss) <= 1e-12 * want_loss
    for g, w in zip(grads, want):
        assert np.abs(g.to_numpy() - w).max() <= 1e-10 * np.abs(w).max()
    assert kept > 0


def test_layer_gradients_against_differences(be):
    """Central differences of the loss in doubles, whole activations.  The loss is piecewise linear in y; with no sign change within the
    step the error is eps^2 / 6 times a third derivative of order 1, plus 1e-16 / eps: below 1e-9 for eps = 1e-5."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(17)
    a = layer(rng, 40, 6, 10, 5)
    a[4] = a[4] + np.where(a[4] > 0, 30, -30)               # targets out of reach: no sign changes
    reset = rng.random(40) < 0.1
    step = lambda t: T.gated_layer_step(*[dev(be, q) for q in t], 0.0, reset=dev(be, reset), seed_with_loss=False)
    grads = [g.to_numpy() for g in step(a)[1]]
    for k, g in enumerate(grads):
        for at in rng.choice(g.size, 5, replace=False):
            two = []
            for eps in (1e-5, -1e-5):
                moved = [t.copy() for t in a]
                moved[1 + k].reshape(-1)[at] += eps
                two.append(step(moved)[0].to_numpy().reshape(-1)[0])
            assert abs((two[0] - two[1]) / 2e-5 - g.reshape(-1)[at]) < 1e-7, (k, at)


def test_layer_step_in_f32(be):
    """Packing leaves the forward pass bit for bit as it is and the kept bytes near a quarter of the activations'; the weights move by
    lr times the gradients; a run of steps is the same run again."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(23)
    tokens, d, f, e = 1024, 64, 128, 32
    a = layer(rng, tokens, d, f, e, np.float32)
    out = {}
    for packed in (False, True):
        runs = []
        for _ in range(2):
            t = [dev(be, q) for q in a]
            loss, grads, kept = T.gated_layer_step(*t, 0.1, packed=packed)
            g = [q.to_numpy() for q in grads]
            for k in range(3):
                moved = t[1 + k].to_numpy()
                assert np.isfinite(g[k]).all() and moved.tobytes() == (a[1 + k] - (g[k] * np.float32(0.1)).astype(np.float32)).tobytes()
            for _ in range(3):
                more, _, _ = T.gated_layer_step(*t, 0.1, packed=packed)
            runs.append((loss.to_numpy().tobytes(), [q.tobytes() for q in g], more.to_numpy().tobytes()))
        assert runs[0] == runs[1]
        out[packed] = runs[0][0], kept
    assert out[False][0] == out[True][0]
    # x twice, u, v, h (twice whole: by the scan and by the last matmul) and the gate; weights as the matmuls keep them, the loss map
    whole = 4 * (2 * tokens * d + 5 * tokens * f + 2 * d * f + f * e + tokens * e)
    eight = (2 * tokens * d + 4 * tokens * f) * 33 // 32 + 4 * (tokens * f + 2 * d * f + f * e + tokens * e)
    assert out[False][1] == whole and out[True][1] == eight, (out, whole, eight)


def test_forward_without_gradients(be):
    """Nodes whose operands carry no gradient are not recorded; sigmoid, silu and tanh give the elementwise results."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal(1000).astype(np.float32)
    for op in ("sigmoid", "silu", "tanh"):
        y, p = dev(be, x).unary_pack8(op)
        assert y.to_numpy().tobytes() == dev(be, x).unary(op).to_numpy().tobytes()
        c, e = R.pack(x)
        assert (p.unpack8().to_numpy() == R.restore(c, e, np.float32)).all()
