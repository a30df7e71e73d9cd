"""The linear scan where parts of it leave the type's range although no state does: sums that a stretch forms from a start of zero, and
products of a stretch's factors.  And the numbers of its launches, where they come round."""
import numpy as np
import pytest

import sequence_ref as R
from test_gpu_scan import TYPES, hip, near, poison, put, run_forward  # noqa: F401

pytestmark = pytest.mark.gpu

# one wave, tiles of two to sixteen waves, many tiles; a lane a column, few columns, short rows that share a tile
SHAPES = [(3, 7, 70), (1, 32, 64), (2, 64, 64), (3, 110, 33), (1, 256, 70), (1, 2500, 64), (2, 1500, 200), (1, 2500, 3), (20, 9000, 1), (6, 9000, 1), (1, 60000, 1),
          (1100, 74, 1), (1300, 100, 3)]


def backward(hip, d, h):
    """dgate, dx, dstate of the linear form."""
    shape = d["gate"].shape
    outs = [poison(hip, h), poison(hip, h), poison(hip, d["state"])]
    hip.gated_scan_backward("linear", put(hip, d["gate"]), None, put(hip, h), put(hip, d["dh"]), outs[0], outs[1], *shape, state=put(hip, d["state"]),
                            dlast=put(hip, d["dlast"]), dstate=outs[2])
    return [hip.dump(o).reshape(s) for o, s in zip(outs, (shape, shape, d["state"].shape))]


def plain_backward(d, h):
    """The plain loop in the type under test."""
    steps, D, carry = h.shape[1], np.zeros_like(h), d["dlast"]
    with np.errstate(over="ignore", under="ignore"):
        for t in range(steps - 1, -1, -1):
            D[:, t] = d["dh"][:, t] + carry
            carry = d["gate"][:, t] * D[:, t]
        before = np.concatenate([d["state"][:, None], h[:, :-1]], axis=1)
        return D * before, D, carry


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("every", [1, 41])
@pytest.mark.parametrize("shape", SHAPES)
def test_sums_from_zero_that_leave_the_range(hip, shape, every, dtype):
    """Gates of 1, a state of -c, and x of +c, +c, -c, -c, ...: the states are -c, 0 and c, every sum of two of them is exact, and two equal
    x one after the other are infinite from a start of zero.  With `every` = 1 each stretch has such pairs, else some."""
    T = TYPES[dtype]
    c = T(0.9) * np.finfo(T).max
    outer, steps, inner = shape
    x = np.zeros(shape, T)
    places = np.arange(1, steps, every)
    x[:, places] = np.where(np.arange(places.size) % 4 < 2, c, -c)[None, :, None]
    state = np.full((outer, inner), -c, T)
    want = (np.cumsum(np.sign(x), axis=1) - 1) * c
    assert np.abs(want).max() <= c
    d = {"gate": np.ones(shape, T), "x": x, "state": state, "dlast": state, "reset": None, "dh": np.ascontiguousarray(x[:, ::-1])}
    h, last = run_forward(hip, "linear", d)
    assert (h == want).all() and (last == want[:, -1]).all()
    small = np.full(shape, T(2) ** -100)                              # h of its own, so that dgate stays in the range
    got, wish = backward(hip, d, small), plain_backward(dict(d), small)
    assert (wish[1] == want[:, ::-1]).all()
    for g, w, name in zip(got, wish, ("dgate", "dx", "dstate")):
        if name == "dgate":
            g, w = g[:, 1:], w[:, 1:]                                 # the state of the first step is -c: out of the range
        assert (g == w).all(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_states_that_sink_and_rise_again(hip, shape, dtype):
    """Gates that are powers of two, no x: 40 small ones and then 40 large ones, so that a state goes far down and comes back exactly, and
    the factors' product over a stretch (2^-200; f64 2^-1600) is far below the smallest number.  All values are exact."""
    T, (down, top) = TYPES[dtype], {"f32": (5, 100), "f64": (40, 900)}[dtype]
    outer, steps, inner = shape
    k = np.arange(steps) % 80
    e = np.where(k < 40, -down, down)
    level = top + np.cumsum(e)
    assert level.min() > np.log2(np.finfo(T).tiny) and level.max() <= top
    sign = np.where(np.arange(outer * inner) % 2, -1.0, 1.0).reshape(outer, inner)
    state = (sign * 2.0 ** top).astype(T)
    gate = np.broadcast_to((2.0 ** e)[None, :, None], shape).astype(T)
    d = {"gate": gate, "x": np.zeros(shape, T), "state": state, "dlast": state, "reset": None, "dh": np.zeros(shape, T)}
    h, last = run_forward(hip, "linear", d)
    want = (sign[:, None] * 2.0 ** level[None, :, None]).astype(T)
    assert (h == want).all() and (last == want[:, -1]).all()
    # backward, the gates in the opposite order; h of 2^-20 keeps dgate in the range where dx is
    d["gate"] = np.ascontiguousarray(gate[:, ::-1])
    small = np.full(shape, T(2) ** -20)
    d["state"] = np.full((outer, inner), T(2) ** -20)
    got, wish = backward(hip, d, small), plain_backward(d, small)
    assert (wish[2] == last).all()
    for g, w, name in zip(got, wish, ("dgate", "dx", "dstate")):
        assert (g == w).all(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_states_of_many_magnitudes(hip, shape, dtype):
    """Gates of either sign that lead the states up and down over most of the range, slowly and fast, with x of the states' size, under the
    bounds of the plain loop."""
    T, most = TYPES[dtype], {"f32": 95, "f64": 900}[dtype]
    outer, steps, inner = shape
    rng = np.random.default_rng(steps)
    t = np.arange(steps + 1)
    level = most * np.sin(t / rng.uniform(5, 9)) * np.cos(t / rng.uniform(60, 90))
    e = np.diff(level)
    gate = (2.0 ** e)[None, :, None] * rng.choice([-0.9, 0.9, 0.5, 1.0], shape)
    x = rng.standard_normal(shape) * (2.0 ** level[1:])[None, :, None]
    d = {"gate": gate.astype(T), "x": x.astype(T), "state": rng.standard_normal((outer, inner)).astype(T) * T(2.0 ** level[0]), "reset": None}
    want, M, S = R.scan("linear", d["gate"], d["x"], d["state"])
    d["dlast"] = d["state"]
    h, last = run_forward(hip, "linear", d)
    near(h, want, R.scan_bound("linear", T, M, S), shape)
    assert last.tobytes() == np.ascontiguousarray(h[:, -1]).tobytes()
    # the same sizes from the last step back
    d["dh"] = np.ascontiguousarray(d["x"][:, ::-1])
    d["gate"] = np.ascontiguousarray(np.concatenate([d["gate"][:, :1], d["gate"][:, 1:][:, ::-1]], axis=1))
    small = np.full(shape, T(2) ** -20)
    d["state"] = np.full((outer, inner), T(2) ** -20)
    got = backward(hip, d, small)
    wish = R.scan_backward("linear", d["gate"], x, small, d["dh"], d["state"], None, d["dlast"])
    for g, (w, bound), name in list(zip(got, wish, ("dgate", "dx", "dstate")))[:2]:
        near(g, w, bound, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("period", [48, 700, 3000])
@pytest.mark.parametrize("shape", SHAPES)
def test_products_beyond_the_range_of_states_that_are_zero(hip, shape, period, dtype):
    """Gates whose product goes far below the range and then far above it, and a state of zero that they leave at zero until a few small x
    come near the end: whatever the products are, nothing comes of them."""
    T, (down, up) = TYPES[dtype], {"f32": (-60, 100), "f64": (-600, 900)}[dtype]
    outer, steps, inner = shape
    e = np.where(np.arange(steps) % period < period // 2, down, up)
    last = max(steps - 3, 0)
    e[last:] = 0
    d = {"gate": np.broadcast_to((2.0 ** e)[None, :, None], shape).astype(T), "x": np.zeros(shape, T), "state": np.zeros((outer, inner), T), "reset": None}
    d["x"][:, last:] = 3
    d["dlast"] = d["state"]
    h, end = run_forward(hip, "linear", d)
    want = np.cumsum(d["x"], axis=1)
    assert (h == want).all() and (end == want[:, -1]).all()
    d["dh"] = np.ascontiguousarray(d["x"][:, ::-1])
    d["gate"] = np.ascontiguousarray(np.concatenate([d["gate"][:, :1], d["gate"][:, 1:][:, ::-1]], axis=1))
    got, wish = backward(hip, d, h), plain_backward(d, h)
    assert (wish[1] == want[:, ::-1]).all()
    for g, w, name in zip(got, wish, ("dgate", "dx", "dstate")):
        assert (g == w).all(), name


def test_more_launches_than_there_are_numbers(hip):
    """The words that tiles hand on carry the launch's number, one of 2^17."""
    rng = np.random.default_rng(1)
    shape = (1, 600, 33)
    n = 600 * 33
    gate, x = (put(hip, rng.random(n).astype(np.float32)) for _ in range(2))
    h, again = poison(hip, np.empty(n, np.float32)), poison(hip, np.empty(n, np.float32))
    hip.gated_scan("linear", gate, x, h, *shape)
    for k in range((1 << 17) + 200):
        hip.gated_scan("linear", gate, x, again, *shape)
        if k % 4096 == 0 or k > 1 << 17:
            assert hip.equal(h, again), k


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_that_are_not_finite_next_to_sums_that_overflow(hip, shape, form, dtype):
    """NaN and infinities in some columns' x, in others the pairs of the first test, in others neither, resets here and there: each column
    has what it has on its own, kinds and places of the values that are not finite as in the plain loop."""
    T = TYPES[dtype]
    c = T(0.9) * np.finfo(T).max
    outer, steps, inner = shape
    rng = np.random.default_rng(inner)
    gate, x, state = np.ones(shape, T), np.zeros(shape, T), np.zeros((outer, inner), T)
    kind = np.arange(outer * inner).reshape(outer, inner) % 4
    pairs = np.zeros(steps, T)
    pairs[1:] = np.where(np.arange(steps - 1) % 4 < 2, c, -c)
    for o in range(outer):
        for i in range(inner):
            if kind[o, i] == 0:
                x[o, :, i], state[o, i] = rng.integers(-5, 6, steps), 7
            elif kind[o, i] == 1:
                x[o, :, i], state[o, i] = rng.integers(-5, 6, steps), 7
                x[o, steps // 3, i] = (np.inf, -np.inf, np.nan)[i % 3]
            elif kind[o, i] == 2:
                x[o, :, i], state[o, i] = pairs, -c
            else:                                     # both: the pairs before, an infinity behind
                x[o, :, i], state[o, i] = pairs, -c
                x[o, steps // 2 :, i] = 0
                x[o, (steps + steps // 2) // 2, i] = np.inf
    reset = np.zeros((outer, steps), bool)
    if form == "sigmoid":                             # forward: averages of x, not sums
        gate[:] = 40
        with np.errstate(all="ignore"):
            x = np.where(np.isfinite(x), np.sign(x), x).astype(T)
    d = {"gate": gate, "x": x, "state": state if form == "linear" else np.sign(state), "reset": reset, "dlast": state}
    with np.errstate(all="ignore"):
        want = R.scan(form, gate, x, d["state"])[0].astype(T)
    h, last = run_forward(hip, form, dict(d, reset=None))
    for k in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(k(h), k(want)), k
    fine = np.isfinite(want)
    assert (h[fine] == want[fine]).all() if form == "linear" else (np.abs(h[fine] - want[fine]) <= 1e-5).all()
    # backward: gates of 1 (the sigmoid form: of 40, a factor of 1 within 2^-57), the columns' x from the last step on
    d["dh"] = np.ascontiguousarray(d["x"][:, ::-1]) if form == "linear" else np.ascontiguousarray(x[:, ::-1])
    small = np.full(shape, T(2) ** -100)
    outs = [poison(hip, small), poison(hip, small), poison(hip, state)]
    hip.gated_scan_backward(form, put(hip, gate), put(hip, small), put(hip, small), put(hip, d["dh"]), outs[0], outs[1], *shape, state=put(hip, state),
                            dlast=put(hip, d["dlast"]), dstate=outs[2])
    dx = hip.dump(outs[1]).reshape(shape)
    if form == "linear":
        plain = plain_backward(dict(d, state=state), small)[1] if np.isfinite(d["dh"]).all() else None
        with np.errstate(all="ignore"):
            D, carry = np.zeros(shape, T), d["dlast"]
            for t in range(steps - 1, -1, -1):
                D[:, t] = d["dh"][:, t] + carry
                carry = D[:, t]
        assert plain is None or (plain == D).all()
        for k in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(k(dx), k(D)), k
        fine = np.isfinite(D)
        assert (dx[fine] == D[fine]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gates_that_are_not_finite(hip, shape, form, dtype):
    """NaN, infinite and zero gates in some columns, none in others: kinds and places of the values that are not finite as in the plain loop,
    the other values within its bounds; forward and backward."""
    T = TYPES[dtype]
    outer, steps, inner = shape
    rng = np.random.default_rng(steps + inner)
    gate, x = rng.uniform(0.5, 1, shape), rng.standard_normal(shape)
    column = np.arange(outer * inner).reshape(outer, inner)
    for k, v in ((1, [np.nan]), (2, [np.inf]), (3, [-np.inf, 0.0]), (4, [np.nan, np.inf, 0.0])):
        for q, value in enumerate(v):
            o, i = np.nonzero(column % 6 == k)
            gate[o, rng.integers(steps // 4, steps, o.size), i] = value
    d = {"gate": gate.astype(T), "x": x.astype(T), "state": rng.standard_normal((outer, inner)).astype(T), "reset": rng.random((outer, steps)) < 2 / (steps + 20)}
    with np.errstate(all="ignore"):
        want, M, S = R.scan(form, d["gate"], d["x"], d["state"], d["reset"])
    h, last = run_forward(hip, form, dict(d, dlast=d["state"]))
    for k in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(k(h), k(want)), k
    fine = np.isfinite(want)
    assert (np.abs(h.astype(want.dtype) - want)[fine] <= R.scan_bound(form, T, M, S)[fine]).all()
    assert last.tobytes() == np.ascontiguousarray(h[:, -1]).tobytes()
    small = np.full(shape, T(0.5))
    outs = [poison(hip, small), poison(hip, small), poison(hip, d["state"])]
    hip.gated_scan_backward(form, put(hip, d["gate"]), put(hip, small), put(hip, small), put(hip, d["x"]), outs[0], outs[1], *shape, state=put(hip, d["state"]),
                            reset=put(hip, d["reset"]), dlast=put(hip, d["state"]), dstate=outs[2])
    with np.errstate(all="ignore"):
        wish = R.scan_backward(form, d["gate"], small, small, d["x"], d["state"], d["reset"], d["state"])
    for out, (w, bound), name in zip(outs[1:], wish[1:], ("dx", "dstate")):
        got = hip.dump(out).reshape(w.shape)
        for k in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(k(got), k(w)), (name, k)
        fine = np.isfinite(w)
        assert (np.abs(got.astype(w.dtype) - w)[fine] <= bound[fine]).all(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("every", [9, 50, 700])
@pytest.mark.parametrize("shape", SHAPES)
def test_zero_gates_among_growing_ones(hip, shape, every, dtype):
    """The product of a stretch with a zero gate in it is 0 however large its other factors are."""
    T, up = TYPES[dtype], {"f32": 3, "f64": 20}[dtype]
    outer, steps, inner = shape
    gate = np.full(shape, T(2) ** up)
    gate[:, 5::every] = 0
    last = max(steps - 3, 0)
    gate[:, last:] = 1
    x = np.zeros(shape, T)
    x[:, last:] = 3
    d = {"gate": gate, "x": x, "state": np.ones((outer, inner), T), "reset": None}
    d["dlast"] = d["state"]
    h, end = run_forward(hip, "linear", d)
    want, p = np.zeros(shape, T), d["state"]
    for t in range(steps):
        p = gate[:, t] * p + x[:, t]
        want[:, t] = p
    assert (h == want).all() and (end == want[:, -1]).all()
    d["dh"] = np.ascontiguousarray(x[:, ::-1])
    d["gate"] = np.ascontiguousarray(np.concatenate([gate[:, :1], gate[:, 1:][:, ::-1]], axis=1))
    got, wish = backward(hip, d, h), plain_backward(d, h)
    assert np.isfinite(wish[1]).all() and (got[1] == wish[1]).all() and (got[2] == wish[2]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first", [np.inf, -np.inf])
@pytest.mark.parametrize("shape", SHAPES + [(1, 9, 3), (9, 33, 2), (13, 25, 1)])
def test_an_infinity_before_pairs_that_overflow(hip, shape, first, dtype):
    """An infinite state stays what it is over x of -c and c in pairs, whose sums from a start of zero are infinities of either sign."""
    T = TYPES[dtype]
    outer, steps, inner = shape
    c = T(0.9) * np.finfo(T).max
    x = np.zeros(shape, T)
    x[:, 1:] = np.where(np.arange(steps - 1) % 4 < 2, c, -c)[None, :, None]
    x[:, 0] = first
    d = {"gate": np.ones(shape, T), "x": x, "state": np.zeros((outer, inner), T), "reset": None, "dh": np.ascontiguousarray(x[:, ::-1])}
    d["dlast"] = d["state"]
    h, last = run_forward(hip, "linear", d)
    assert (h == first).all() and (last == first).all()
    small = np.full(shape, T(2) ** -100)
    got = backward(hip, d, small)
    assert (got[1] == first).all() and (got[2] == first).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", [np.nan, 0.0])
@pytest.mark.parametrize("shape", SHAPES)
def test_nan_and_zero_gates_among_very_small_ones(hip, shape, what, dtype):
    """Nothing is left of a state behind a few gates near the smallest number, but NaN is, and an infinite state is NaN behind a gate of 0;
    also where the gate is a tile's first one."""
    T = TYPES[dtype]
    outer, steps, inner = shape
    gate = np.full(shape, np.finfo(T).tiny)
    starts = np.array([128, 256, 512, 640, 1024, 2048, 0, 8, 16, 32, 64, 4096])
    column = np.arange(outer * inner).reshape(outer, inner)
    first = starts[column % starts.size] % steps
    o, i = np.indices((outer, inner))
    gate[o, first, i] = what
    d = {"gate": gate, "x": np.ones(shape, T), "state": np.full((outer, inner), 1 if np.isnan(what) else np.inf, T), "reset": None}
    d["dlast"], d["dh"] = d["state"], d["x"]
    want = np.arange(steps)[None, :, None] >= first[:, None]
    h, last = run_forward(hip, "linear", d)
    assert np.array_equal(np.isnan(h), want) and np.isnan(last).all()
    got = backward(hip, d, np.ones(shape, T))
    before = np.arange(steps)[None, :, None] < first[:, None]       # the gate of a step is that of the state before it
    assert np.array_equal(np.isnan(got[1]), before) and np.isnan(got[2]).all()
