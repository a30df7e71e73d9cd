"""rt_gated_scan and its backward passes against a plain recurrence in a wider type."""
import itertools

import numpy as np
import pytest

import sequence_ref as R

pytestmark = pytest.mark.gpu

TYPES = {"f32": np.float32, "f64": np.float64}
# (outer, steps, inner): single tokens, lengths around the tile sizes, odd widths, one column, many columns, long axes
SHAPES = [(1, 1, 1), (5, 1, 300), (3, 2, 64), (1, 17, 63), (2, 64, 64), (1, 65, 130), (2, 129, 257), (7, 31, 5), (3, 255, 1), (1, 1000, 1),
          (2, 513, 2), (1, 257, 33), (1, 2050, 96), (1, 5001, 7), (40, 333, 3), (1, 20000, 1), (2, 4099, 65), (300, 5, 19), (1, 1500, 1025)]


@pytest.fixture(scope="module")
def hip():
    from rtensors_amd import hip as H
    b = H.Hip.new(0)
    yield b
    b.sync()


def put(hip, a):
    from rtensors_amd import hip as H
    if a is None:
        return None
    code = {np.float32: H.F32, np.float64: H.F64, np.bool_: H.BOOL, np.int8: H.I8, np.uint8: H.U8}[a.dtype.type]
    return hip.alloc_from_slice(code, a.reshape(-1))


def poison(hip, like, n=None):
    """A buffer of NaN, so that an element that is not written shows."""
    return put(hip, np.full(like.size if n is None else n, np.nan, dtype=like.dtype))


def make(shape, dtype, form, seed, state=True, reset=False, long_memory=True):
    rng = np.random.default_rng(seed)
    outer, steps, inner = shape
    gate = rng.standard_normal(shape) * 1.5 + (2 if long_memory else 0)
    if form == "linear":
        gate = np.where(rng.random(shape) < 0.1, -1, 1) / (1 + np.exp(-gate))
    d = {"gate": gate, "x": rng.standard_normal(shape), "dh": rng.standard_normal(shape), "dlast": rng.standard_normal((outer, inner)),
         "state": rng.standard_normal((outer, inner)) if state else None}
    d = {k: None if v is None else v.astype(dtype) for k, v in d.items()}
    d["reset"] = rng.random((outer, steps)) < (0.2 if steps < 50 else 3 / 200) if reset else None
    return d


def run_forward(hip, form, d, last=True):
    shape = d["gate"].shape
    h = poison(hip, d["gate"])
    out = poison(hip, d["dlast"]) if last else None
    hip.gated_scan(form, put(hip, d["gate"]), put(hip, d["x"]), h, *shape, state=put(hip, d["state"]), reset=put(hip, d["reset"]), last=out)
    return hip.dump(h).reshape(shape), hip.dump(out).reshape(shape[0], shape[2]) if last else None


def near(got, want, bound, what):
    got = got.astype(want.dtype)
    worst = np.max(np.abs(got - want) - bound, initial=-1)
    assert np.isfinite(got).all() and worst <= 0, (what, float(worst), float(np.max(np.abs(got - want) / np.maximum(bound, 1e-300))))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(hip, shape, form, dtype):
    for k, (state, reset) in enumerate(itertools.product((False, True), repeat=2)):
        d = make(shape, TYPES[dtype], form, 10 * k + 1, state, reset)
        want, M, S = R.scan(form, d["gate"], d["x"], d["state"], d["reset"])
        h, last = run_forward(hip, form, d)
        near(h, want, R.scan_bound(form, TYPES[dtype], M, S), (shape, state, reset))
        assert last.tobytes() == np.ascontiguousarray(h[:, -1]).tobytes()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("held", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(hip, shape, held, form, dtype):
    T = TYPES[dtype]
    for k, (state, reset) in enumerate(itertools.product((False, True), repeat=2)):
        d = make(shape, T, form, 10 * k + 5, state, reset)
        dlast = d["dlast"] if k != 1 else None
        h = R.scan(form, d["gate"], d["x"], d["state"], d["reset"])[0].astype(T)
        x = d["x"]
        outs = [poison(hip, x), poison(hip, x), poison(hip, d["dlast"])]
        rest = dict(state=put(hip, d["state"]), reset=put(hip, d["reset"]), dlast=put(hip, dlast), dstate=outs[2])
        if held:
            x8, h8 = R.pack(x.reshape(-1)), R.pack(h.reshape(-1))
            x, h = R.restore(*x8, T).reshape(shape), R.restore(*h8, T).reshape(shape)
            pairs = [tuple(put(hip, a) for a in p) for p in (x8, h8)]
            hip.gated_scan_backward_packed8(form, put(hip, d["gate"]), None if form == "linear" else pairs[0], pairs[1], put(hip, d["dh"]), outs[0], outs[1],
                                            *shape, **rest)
        else:
            hip.gated_scan_backward(form, put(hip, d["gate"]), None if form == "linear" else put(hip, x), put(hip, h), put(hip, d["dh"]), outs[0], outs[1],
                                    *shape, **rest)
        want = R.scan_backward(form, d["gate"], x, h, d["dh"], d["state"], d["reset"], dlast)
        for got, (w, bound), name in zip(outs, want, ("dgate", "dx", "dstate")):
            near(hip.dump(got).reshape(w.shape), w, bound, (name, shape, state, reset, held))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("steps", [9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 96, 127, 128, 129, 255, 256, 257])
def test_lengths_around_those_of_waves_and_tiles(hip, steps, form, dtype):
    test_forward(hip, (2, steps, 70), form, dtype)
    test_backward(hip, (2, steps, 70), False, form, dtype)
    test_backward(hip, (2, steps, 70), True, form, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape", [(4, 20000, 1), (5, 9000, 2), (16, 9000, 1), (17, 3000, 2), (40, 4097, 1), (17, 900, 31)])
def test_few_columns_and_few_or_many_rows(hip, shape, form, dtype):
    test_forward(hip, shape, form, dtype)


@pytest.mark.parametrize("form", ["linear", "sigmoid"])
def test_gradients_against_differences(hip, form):
    """Central differences of sum(h * w) + sum(last * v) in doubles: the step's own error is eps^2 * |third derivative| / 6, with
    eps = 1e-5 below 1e-9 here, and the rounding of the two sums over 2 eps below 1e-9."""
    shape, rng = (2, 70, 9), np.random.default_rng(3)
    d = make(shape, np.float64, form, 2, True, True)

    def value(d):
        h, last = run_forward(hip, form, d)
        return float((h * d["dh"]).sum() + (last * d["dlast"]).sum())

    h, _ = run_forward(hip, form, d)
    outs = {"gate": poison(hip, d["gate"]), "x": poison(hip, d["x"]), "state": poison(hip, d["state"])}
    hip.gated_scan_backward(form, put(hip, d["gate"]), put(hip, d["x"]), put(hip, h), put(hip, d["dh"]), outs["gate"], outs["x"], *shape,
                            state=put(hip, d["state"]), reset=put(hip, d["reset"]), dlast=put(hip, d["dlast"]), dstate=outs["state"])
    for name, buf in outs.items():
        got = hip.dump(buf)
        for at in rng.choice(got.size, 12, replace=False):
            two = []
            for eps in (1e-5, -1e-5):
                moved = dict(d)
                moved[name] = d[name].copy()
                moved[name].reshape(-1)[at] += eps
                two.append(value(moved))
            assert abs((two[0] - two[1]) / 2e-5 - got[at]) < 1e-7, (name, at)


@pytest.mark.parametrize("shape", [(2, 40, 70), (1, 3000, 65), (1, 900, 3), (2, 20000, 1)])
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
def test_nothing_crosses_a_reset(hip, form, shape):
    """Infinities and NaN in front of a reset leave what follows alone, forward; behind it leave what precedes alone, backward."""
    outer, steps, inner = shape
    cut = steps // 2
    d = make(shape, np.float32, form, 4)
    d["reset"] = np.zeros((outer, steps), dtype=bool)
    d["reset"][:, cut] = True
    clean, _ = run_forward(hip, form, d)
    for bad in (np.inf, -np.inf, np.nan):
        e = dict(d, gate=d["gate"].copy(), x=d["x"].copy(), dh=d["dh"].copy(), state=np.full_like(d["state"], bad))
        e["x"][:, cut - 1], e["gate"][:, cut - 3] = bad, bad
        if form == "linear":
            e["gate"][:, cut] = bad                      # the gate of a step that nothing precedes is not used
        h, last = run_forward(hip, form, e)
        near(h[:, cut:], clean[:, cut:].astype(np.float64), 1e-5 * np.abs(clean[:, cut:]) + 1e-5, "after the reset")
        assert not np.isfinite(h[:, cut - 1]).any()
        f = dict(d, dh=d["dh"].copy(), dlast=np.full_like(d["dlast"], bad))
        f["dh"][:, cut] = bad
        outs = [poison(hip, d["x"]), poison(hip, d["x"]), poison(hip, d["dlast"])]
        hip.gated_scan_backward(form, put(hip, d["gate"]), put(hip, d["x"]), put(hip, clean), put(hip, f["dh"]), outs[0], outs[1], *shape,
                                state=put(hip, d["state"]), reset=put(hip, d["reset"]), dlast=put(hip, f["dlast"]), dstate=outs[2])
        got = [hip.dump(o).reshape(outer, -1, inner) for o in outs]
        want = R.scan_backward(form, d["gate"], d["x"], clean, d["dh"], d["state"], d["reset"], None)
        for g, (w, b), name in zip(got, want, ("dgate", "dx", "dstate")):
            w, b = w.reshape(outer, -1, inner), b.reshape(outer, -1, inner)
            near(g[:, :cut] if name != "dstate" else g, w[:, :cut] if name != "dstate" else w, b[:, :cut] if name != "dstate" else b, (name, bad))


@pytest.mark.parametrize("shape", [(1, 2500, 64), (1, 2500, 3), (1, 30000, 1), (2, 700, 200)])
def test_growing_gates(hip, shape):
    """Gates above 1 whose product over a stretch leaves the range while the states stay in it: zeros until late, then small numbers."""
    outer, steps, inner = shape
    d = make(shape, np.float32, "linear", 6, state=False)
    d["gate"][:] = 1.5
    d["x"][:] = 0
    d["x"][:, -20:] = 1
    want, M, S = R.scan("linear", d["gate"], d["x"])
    h, _ = run_forward(hip, "linear", d)
    near(h, want, R.scan_bound("linear", np.float32, M, S), shape)
    d["dh"][:] = 0
    d["dh"][:, :20] = 1
    outs = [poison(hip, d["x"]), poison(hip, d["x"])]
    hip.gated_scan_backward("linear", put(hip, d["gate"]), None, put(hip, h), put(hip, d["dh"]), outs[0], outs[1], *shape)
    (wg, bg), (wx, bx), _ = R.scan_backward("linear", d["gate"], d["x"], h, d["dh"])
    near(hip.dump(outs[1]).reshape(shape), wx, bx, "dx")
    near(hip.dump(outs[0]).reshape(shape), wg, bg, "dgate")


def test_infinite_values_travel_as_in_the_plain_loop(hip):
    """Kinds and places of the values that are not finite, where the plain loop has them."""
    for shape in ((1, 600, 64), (1, 600, 5), (1, 5000, 1)):
        d = make(shape, np.float32, "linear", 8, state=False)
        d["gate"] = np.abs(d["gate"])
        d["x"][0, 100, ::2] = np.inf
        d["gate"][0, 300, :] = 0                           # 0 * inf = NaN from here on
        with np.errstate(all="ignore"):
            want, _, _ = R.scan("linear", d["gate"], d["x"])
        h, _ = run_forward(hip, "linear", d)
        for kind in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(kind(h), kind(want.astype(np.float32))), (shape, kind)


@pytest.mark.parametrize("shape", [(3, 1, 200), (2, 50, 3), (1, 700, 70), (1, 3000, 1)])
def test_in_place_and_equal_bits(hip, shape):
    """h over x or gate, last over state, dx over dh or x, dstate over dlast give the bits of the separate buffers; so does the same
    call again; elements behind the run stay as they were."""
    n = int(np.prod(shape))
    for form in ("linear", "sigmoid"):
        d = make(shape, np.float32, form, 9, True, True)
        h, last = run_forward(hip, form, d)
        for over in ("x", "gate"):
            b = {k: put(hip, d[k]) for k in ("gate", "x", "state", "reset")}
            tail = np.concatenate([d[over].reshape(-1), np.full(7, 123.0, np.float32)])
            b[over] = put(hip, tail)
            hip.gated_scan(form, b["gate"], b["x"], b[over], *shape, state=b["state"], reset=b["reset"], last=b["state"])
            got = hip.dump(b[over])
            assert got[:n].tobytes() == h.tobytes() and (got[n:] == 123.0).all()
            assert hip.dump(b["state"]).tobytes() == last.tobytes()
        plain = None
        for over in (None, "dh", "x"):
            b = {k: put(hip, d[k]) for k in ("gate", "x", "dh", "dlast", "state", "reset")}
            outs = [poison(hip, h), poison(hip, h) if over is None else b[over], poison(hip, last) if over is None else b["dlast"]]
            hip.gated_scan_backward(form, b["gate"], b["x"], put(hip, h), b["dh"], outs[0], outs[1], *shape, state=b["state"], reset=b["reset"],
                                    dlast=b["dlast"], dstate=outs[2])
            got = [hip.dump(o).tobytes() for o in outs]
            plain = plain or got
            assert got == plain, over


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["linear", "sigmoid"])
@pytest.mark.parametrize("shape", [(1100, 74, 1), (3190, 48, 1), (2048, 100, 3), (1025, 9, 31), (2100, 20, 17), (600, 300, 1), (5000, 11, 2), (10000, 37, 5)])
def test_short_rows_that_share_a_tile(hip, shape, form, dtype):
    test_forward(hip, shape, form, dtype)
    test_backward(hip, shape, False, form, dtype)
    test_backward(hip, shape, True, form, dtype)


@pytest.mark.parametrize("shape", [(20, 9000, 1), (6, 9000, 1), (17, 5000, 2), (3, 60, 70), (3, 110, 33), (1100, 74, 1), (1300, 100, 3)])
def test_tiles_of_other_widths(hip, shape):
    """The tests above where rows or steps give tiles of two, four, eight and sixteen waves."""
    test_growing_gates(hip, shape)
    test_in_place_and_equal_bits(hip, shape)
    for form in ("linear", "sigmoid"):
        test_nothing_crosses_a_reset(hip, form, shape)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(62, 3241, 11), (23, 9280, 25), (4, 60664, 21), (30, 20000, 17), (1, 20000, 96), (3, 8000, 64)])
def test_many_equal_calls_give_equal_bits(hip, shape, dtype):
    """Tiles that hand states on meet each other at different moments in every call."""
    n = int(np.prod(shape))
    rng = np.random.default_rng(11)
    T = TYPES[dtype]
    gate, x = (put(hip, rng.random(n).astype(T)) for _ in range(2))
    h, dg, dx, h2, dg2, dx2 = (poison(hip, np.empty(n, T)) for _ in range(6))
    hip.gated_scan("linear", gate, x, h, *shape)
    hip.gated_scan_backward("linear", gate, None, h, x, dg, dx, *shape)
    for k in range(60):
        hip.gated_scan("linear", gate, x, h2, *shape)
        hip.gated_scan_backward("linear", gate, None, h, x, dg2, dx2, *shape)
        assert hip.equal(h, h2) and hip.equal(dg, dg2) and hip.equal(dx, dx2), k


def test_no_steps_and_no_columns(hip):
    from rtensors_amd import hip as H
    st = np.arange(6, dtype=np.float32)
    none = hip.alloc(H.F32, 0)
    last = poison(hip, st)
    hip.gated_scan("linear", none, none, none, 2, 0, 3, state=put(hip, st), last=last)
    assert (hip.dump(last) == st).all()
    hip.gated_scan("sigmoid", none, none, none, 2, 0, 3, last=last)
    assert (hip.dump(last) == 0).all()
    hip.gated_scan_backward("linear", none, None, none, none, none, none, 2, 0, 3, dlast=put(hip, st), dstate=last)
    assert (hip.dump(last) == st).all()
    hip.gated_scan("linear", none, none, none, 0, 5, 3)
    hip.gated_scan("linear", none, none, none, 4, 5, 0)


def test_many_calls_of_many_sizes_in_a_row(hip):
    """Calls share the context's workspace: large after small after large, without a wait between them, each checked at the end."""
    shapes = [(1, 4000, 64), (2, 9, 3), (1, 20000, 1), (1, 4000, 64), (1, 700, 300), (1, 20000, 1), (4, 2048, 128), (1, 4000, 64)]
    todo = []
    for k, shape in enumerate(shapes):
        d = make(shape, np.float32, "sigmoid", 20 + k, True, k % 2 == 0)
        h = poison(hip, d["x"])
        todo.append((shape, d, h, {n: put(hip, d[n]) for n in ("gate", "x", "state", "reset")}))
    for rep in range(3):
        for shape, d, h, b in todo:
            hip.gated_scan("sigmoid", b["gate"], b["x"], h, *shape, state=b["state"], reset=b["reset"])
    for shape, d, h, b in todo:
        want, M, S = R.scan("sigmoid", d["gate"], d["x"], d["state"], d["reset"])
        near(hip.dump(h).reshape(shape), want, R.scan_bound("sigmoid", np.float32, M, S), shape)


def test_two_contexts_at_once(hip):
    """Two contexts on one device, each with its own stream and workspace, calls in turn without a wait."""
    from rtensors_amd import hip as H
    other = H.Hip.new(0)
    shape = (1, 30000, 96)
    d = make(shape, np.float32, "sigmoid", 31)
    want, M, S = R.scan("sigmoid", d["gate"], d["x"], d["state"])
    sides = []
    for be in (hip, other):
        sides.append((be, poison(be, d["x"]), [put(be, d[n]) for n in ("gate", "x", "state")]))
    for _ in range(20):
        for be, h, (g, x, s) in sides:
            be.gated_scan("sigmoid", g, x, h, *shape, state=s)
    for be, h, _ in sides:
        near(be.dump(h).reshape(shape), want, R.scan_bound("sigmoid", np.float32, M, S), "two contexts")
    del sides, h, be
    other.sync()


@pytest.mark.parametrize("inner", [16384, 1])
def test_offsets_beyond_32_bits(hip, inner):
    """More than 2^32 bytes and 2^31 elements: h of gate 0.5 and x 1 is 2 - 2^-t."""
    from rtensors_amd import hip as H
    steps = (1 << 31) // inner + 100
    n = steps * inner
    gate, x, h = (hip.alloc_uninit(H.F32, n) for _ in range(3))
    hip.fill_contiguous(gate, 0.5, 0, n)
    hip.fill_contiguous(x, 1.0, 0, n)
    hip.fill_contiguous(h, -1.0, 0, n)
    hip.gated_scan("linear", gate, x, h, 1, steps, inner)
    for t in (0, 1, 2, steps // 2, steps - 3, steps - 1):
        for i in {0, inner // 2, inner - 1}:
            assert hip.read(h, t * inner + i) == np.float32(2 - 2.0 ** -t), (t, i)
    hip.gated_scan_backward("linear", gate, None, h, x, hip.alloc_uninit(H.F32, n), x, 1, steps, inner)
    for t in (0, steps // 2, steps - 2, steps - 1):
        assert hip.read(x, t * inner + inner - 1) == np.float32(2 - 2.0 ** -(steps - 1 - t)), t


def test_more_columns_than_a_launch_has_lanes():
    """One token over more than 2^31 columns: h = 0.5 * 2 + 1, in place of x, and the new state in place of the old one."""
    from rtensors_amd import hip as H
    be, n = H.Hip.new(0), (1 << 31) + 1000
    gate, x, state = (be.alloc_uninit(H.F32, n) for _ in range(3))
    for b, v in ((gate, 0.5), (x, 1.0), (state, 2.0)):
        be.fill_contiguous(b, v, 0, n)
    places = (0, 12345, (1 << 31) - 1, 1 << 31, n - 1)
    be.gated_scan("linear", gate, x, x, 1, 1, n, state=state, last=state)
    for i in places:
        assert be.read(x, i) == 2 and be.read(state, i) == 2, i
    be.fill_contiguous(state, 4.0, 0, n)
    dgate, dstate = be.alloc_uninit(H.F32, n), be.alloc_uninit(H.F32, n)
    be.gated_scan_backward("linear", gate, None, x, x, dgate, be.alloc_uninit(H.F32, n), 1, 1, n, state=state, dstate=dstate)
    for i in places:
        assert be.read(dgate, i) == 8 and be.read(dstate, i) == 1, i
    be.gated_scan("linear", gate, x, x, 1, 0, n, last=state)                       # no steps and no state: zeros
    for i in places:
        assert be.read(state, i) == 0, i


def test_more_rows_than_a_launch_has_lanes():
    """512 lanes a row and more than 2^22 rows."""
    from rtensors_amd import hip as H
    be, (outer, steps, inner) = H.Hip.new(0), ((1 << 22) + 3, 33, 33)
    n = outer * steps * inner
    gate, x, h = (be.alloc_uninit(H.F32, n) for _ in range(3))
    for b, v in ((gate, 0.5), (x, 1.0), (h, -1.0)):
        be.fill_contiguous(b, v, 0, n)
    rows = (0, 1000, (1 << 22) - 1, 1 << 22, outer - 1)
    be.gated_scan("linear", gate, x, h, outer, steps, inner)
    for o in rows:
        for t in (0, 1, steps - 1):
            for i in (0, inner - 1):
                assert be.read(h, (o * steps + t) * inner + i) == np.float32(2 - 2.0 ** -t), (o, t, i)
    be.gated_scan_backward("linear", gate, None, h, x, be.alloc_uninit(H.F32, n), x, outer, steps, inner)
    for o in rows:
        for t in (0, 1, steps - 1):
            assert be.read(x, (o * steps + t) * inner + inner - 1) == np.float32(2 - 2.0 ** -(steps - 1 - t)), (o, t)
