"""The linear scan where sums that a stretch forms from a start of zero leave the type's range although no state does."""
import numpy as np
import pytest

from test_gpu_scan import TYPES, hip, poison, put, run_forward  # noqa: F401

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
