"""The tape's nodes of sigmoid, silu and tanh and of the gated scan, one at a time: gradients against the formulas in doubles, against
differences, and what the tape keeps."""
import numpy as np
import pytest

import sequence_ref as R
from test_gpu_tape import be, dev, held, sigmoid  # noqa: F401

pytestmark = pytest.mark.gpu


def slope(op, x):
    if op == "tanh":
        e = np.exp(-2 * np.abs(x))
        return 4 * e / (1 + e) ** 2
    s, rest = sigmoid(x), 1 / (1 + np.exp(x))
    return s * rest if op == "sigmoid" else s * (1 + x * rest)


FUNCTION = {"sigmoid": sigmoid, "silu": lambda x: x * sigmoid(x), "tanh": np.tanh}


def unit(y, target):
    """The gradient of a mean L1 loss: the tape divides by the count as an f32 number."""
    return np.sign(y - target) / float(np.float32(y.size))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("op", ["sigmoid", "silu", "tanh"])
def test_activation_gradients(be, op, packed):
    """d(bias) is the slope times the loss's own gradient, in doubles: a dozen roundings of 2^-53 next to 1e-13."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(len(op))
    x, b, t = rng.standard_normal((3, 37, 50)) * 2
    loss, g, kept = T.activation_step(dev(be, x), dev(be, b), dev(be, t), op, 0.0, packed=packed, seed_with_loss=False)
    z = x + b
    y = FUNCTION[op](z)
    assert abs(loss.to_numpy().reshape(-1)[0] - np.abs(y - t).mean()) <= 1e-12
    want = unit(y, t) * slope(op, held(z, packed))
    assert (np.abs(g.to_numpy() - want) <= 1e-13 * np.abs(unit(y, t))).all()
    # the input of op (whole or 8-bit) and the loss's map
    assert kept == (1850 + 58 if packed else 8 * 1850) + 8 * 1850


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("op", ["sigmoid", "silu", "tanh"])
def test_a_bias_of_one_row(be, op, packed):
    """A broadcast bias gets the sum over the rows, and moves by lr times it."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(9)
    x, b, t = rng.standard_normal((64, 40)), rng.standard_normal(40), rng.standard_normal((64, 40))
    tb = dev(be, b)
    _, g, _ = T.activation_step(dev(be, x), tb, dev(be, t), op, 0.5, packed=packed, seed_with_loss=False)
    z = x + b
    want = (unit(FUNCTION[op](z), t) * slope(op, held(z, packed))).sum(axis=0)
    assert g.shape == [40] and np.abs(g.to_numpy() - want).max() <= 1e-14
    assert tb.to_numpy().tobytes() == (b - 0.5 * g.to_numpy()).tobytes()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape, axis", [((70,), 0), ((5, 40), 1), ((60, 9), 0), ((3, 50, 33), 1), ((4, 3, 45), 2), ((2, 300, 64), 1)])
def test_scan_gradients(be, shape, axis, form, with_state, packed):
    """d(bias), d(gate), d(state) from the formulas, whole and packed; sums of a few hundred terms of order 1 / n in doubles."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(len(shape) + axis)
    sizes = int(np.prod(shape[:axis])), shape[axis], int(np.prod(shape[axis + 1:]))
    rest, lead = shape[:axis] + shape[axis + 1:], shape[:axis + 1]
    x, b, t, g = rng.standard_normal((4,) + shape)
    g = sigmoid(g + 1) * np.where(rng.random(shape) < 0.1, -1, 1) if form == "linear" else g
    state, reset = np.asarray(rng.standard_normal(rest)) if with_state else None, rng.random(lead) < 0.05
    loss, grads, kept = T.scan_step(dev(be, x), dev(be, b), dev(be, g), dev(be, t), axis, form, 0.0, state=None if state is None else dev(be, state),
                                    reset=dev(be, reset), packed=packed, seed_with_loss=False)
    g3, z3 = g.reshape(sizes), (x + b).reshape(sizes)
    s2, r2 = None if state is None else state.reshape(sizes[0], sizes[2]), reset.reshape(sizes[:2])
    h = R.scan(form, g3, z3, s2, r2)[0].astype(np.float64)
    assert abs(loss.to_numpy().reshape(-1)[0] - np.abs(h - t.reshape(sizes)).mean()) <= 1e-12
    dy = unit(h, t.reshape(sizes))
    (dg, _), (dz, _), (ds, _) = R.scan_backward(form, g3, held(z3, packed), held(h, packed), dy, s2, r2)
    for got, want, like in zip(grads, (dz, dg, ds), (shape, shape, rest)):
        if got is None:
            assert state is None and want is ds
            continue
        assert got.shape == list(like)
        want = want.astype(np.float64)
        assert np.abs(got.to_numpy().reshape(want.shape) - want).max() <= 1e-11 * np.abs(want).max()
    assert (grads[2] is None) == (state is None)
    n, one = x.size, -(-x.size // 32)
    act = (2 if form == "sigmoid" else 1) * ((n + one) if packed else 8 * n)
    assert kept == act + 8 * n + (0 if state is None else 8 * state.size) + reset.size + 8 * n        # activations, gate, state, reset, the loss's map


@pytest.mark.parametrize("form", ["linear", "sigmoid"])
def test_scan_gradients_against_differences(be, form):
    """As for the layer: the loss is smooth within the step with targets out of reach, and its error is below 1e-7."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(4)
    x, b, t, g = rng.standard_normal((4, 3, 20, 7))
    g = sigmoid(g) if form == "linear" else g
    s, r = rng.standard_normal((3, 7)), rng.random((3, 20)) < 0.1
    a = [b, g, s]
    step = lambda a: T.scan_step(dev(be, x), dev(be, a[0]), dev(be, a[1]), dev(be, t + np.where(t > 0, 40, -40)), 1, form, 0.0, state=dev(be, a[2]), reset=dev(be, r),
                                 seed_with_loss=False)
    grads = [q.to_numpy() for q in step(a)[1]]
    for k in range(3):
        for at in rng.choice(a[k].size, 6, replace=False):
            two = []
            for eps in (1e-5, -1e-5):
                moved = [q.copy() for q in a]
                moved[k].reshape(-1)[at] += eps
                two.append(step(moved)[0].to_numpy().reshape(-1)[0])
            assert abs((two[0] - two[1]) / 2e-5 - grads[k].reshape(-1)[at]) < 1e-7, (k, at)


@pytest.mark.parametrize("packed", [False, True])
def test_nothing_is_kept_without_parameters(be, packed):
    """Operands that carry no gradient leave no node: the same loss, no gradients, and the loss's own map is all that is kept."""
    from rtensors_amd import tensor as T
    rng = np.random.default_rng(2)
    x, b, t, g = rng.standard_normal((4, 30, 20)).astype(np.float32)
    for op in ("sigmoid", "silu", "tanh"):
        with_tape = T.activation_step(dev(be, x), dev(be, b), dev(be, t), op, 0.0, packed=packed)
        loss, grad, kept = T.activation_step(dev(be, x), dev(be, b), dev(be, t), op, 0.0, packed=packed, train=False)
        assert grad is None and kept == 4 * 600 < with_tape[2] and loss.to_numpy().tobytes() == with_tape[0].to_numpy().tobytes()
    for form in ("linear", "sigmoid"):
        with_tape = T.scan_step(dev(be, x), dev(be, b), dev(be, g), dev(be, t), 0, form, 0.0, packed=packed)
        loss, grads, kept = T.scan_step(dev(be, x), dev(be, b), dev(be, g), dev(be, t), 0, form, 0.0, packed=packed, train=False)
        assert grads == [None] * 3 and kept == 4 * 600 < with_tape[2] and loss.to_numpy().tobytes() == with_tape[0].to_numpy().tobytes()


def test_refusals(be):
    from rtensors_amd import tensor as T
    z = lambda *s, dt="f32": T.Tensor.zeros(be, dt, list(s))
    for call, kind in ((lambda: T.activation_step(z(3, 4), z(3, 4), z(3, 4), "relu", 0.1), "UnsupportedOperation"),
                       (lambda: T.scan_step(z(3, 4), z(3, 4), z(4, 3), z(3, 4), 1, "linear", 0.1), "InvalidShape"),
                       (lambda: T.scan_step(z(3, 4), z(3, 4), z(3, 4), z(3, 4), 2, "linear", 0.1), "InvalidDim"),
                       (lambda: T.scan_step(z(3, 4), z(3, 4), z(3, 4), z(3, 4), 1, "linear", 0.1, state=z(4)), "InvalidShape")):
        with pytest.raises(T.TensorError) as e:
            call()
        assert e.value.kind == kind, (e.value.kind, str(e.value))
