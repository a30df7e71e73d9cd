"""The 8-bit form of activations (rt_pack8 and the passes that read it) against its definition in plain numpy."""
import numpy as np
import pytest

import sequence_ref as R
from test_gpu_scan import poison, put

pytestmark = pytest.mark.gpu

TYPES = {"f32": np.float32, "f64": np.float64}
SIZES = [1, 3, 4, 31, 32, 33, 255, 1000, 4095, 4096, 4097, 100003]


@pytest.fixture(scope="module")
def hip():
    from rtensors_amd import hip as H
    b = H.Hip.new(0)
    yield b
    b.sync()


def room(hip, n, spare=0):
    from rtensors_amd import hip as H
    return hip.alloc_from_slice(H.I8, np.full(n + spare, 99, np.int8)), hip.alloc_from_slice(H.U8, np.full(-(-n // 32) + spare, 99, np.uint8))


def values(n, dtype, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(n) * np.exp(rng.standard_normal(n) * 3)
    x[::17] = 0
    x[5::23] *= -0.0
    return x.astype(dtype)


def check_pack(hip, x, start=0, spare=5):
    n = x.size - start
    c, e = room(hip, n, spare)
    hip.pack8(put(hip, x), start, n, c, e)
    wc, we = R.pack(x[start:])
    gc, ge = hip.dump(c), hip.dump(e)
    assert (gc[:n] == wc).all() and (ge[:we.size] == we).all()
    assert (gc[n:] == 99).all() and (ge[we.size:] == 99).all()
    y = poison(hip, x, n + spare)
    hip.unpack8(c, e, n, y)
    got, want = hip.dump(y), R.restore(wc, we, x.dtype.type)
    assert np.array_equal(got[:n], want, equal_nan=True) and np.isnan(got[n:]).all()
    return want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", SIZES)
def test_pack_and_restore(hip, n, dtype):
    x = values(n, TYPES[dtype], n)
    back = check_pack(hip, x)
    groups = np.repeat(np.maximum.reduceat(np.abs(x), np.arange(0, n, 32)), 32)[:n]
    assert (np.abs(back - x) <= np.maximum(groups / 126, 2.0 ** -120)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start", [1, 2, 3, 5, 32])
def test_pack_from_any_start(hip, start, dtype):
    check_pack(hip, values(5000 + start, TYPES[dtype], start), start)


def test_borders(hip):
    """Values on and beside the borders of a code, an exponent and the range."""
    rows = []
    for k in (-149, -130, -126, -120, -119, -113, -112, -20, 0, 5, 100, 121):
        for top in (64.0, 127.0, 127.49999, 127.5, 127.50001, 127.99999, 126.5, 100.3):
            with np.errstate(over="ignore", under="ignore"):
                r = np.ldexp(np.concatenate([[top], np.arange(-127.5, 128, 1)[:15] + 0.0, [0.5, -0.5, 1.5, 2.5, 0.49999997, 0.50000006, -1.5], np.arange(9) * 13.7]), k)
                rows.append(np.clip(r, -3.4e38, 3.4e38).astype(np.float32))
    x = np.concatenate(rows)
    assert all(r.size == 32 for r in rows)
    check_pack(hip, x)
    check_pack(hip, x.astype(np.float64))
    check_pack(hip, np.concatenate([np.ldexp(x[:320].astype(np.float64), k) for k in (-900, -400, 7, 20, 300, 800)]))


@pytest.mark.parametrize("dtype", TYPES)
def test_groups_that_are_not_finite(hip, dtype):
    x = values(320, TYPES[dtype], 3)
    x[40], x[100], x[319] = np.nan, np.inf, -np.inf
    back = check_pack(hip, x)
    assert np.isnan(back[32:64]).all() and np.isnan(back[96:128]).all() and np.isnan(back[288:]).all() and np.isfinite(back[:32]).all()
    x = np.full(40, -np.nan, dtype=TYPES[dtype])
    check_pack(hip, x)


def test_nothing_to_pack(hip):
    from rtensors_amd import hip as H
    e = hip.alloc(H.F32, 0)
    c, x = room(hip, 0)
    hip.pack8(e, 0, 0, c, x)
    hip.unpack8(c, x, 0, e)


def slope(op, x):
    """f'(x) and its bound in half steps, in the type of x (wider than the one under test)."""
    with np.errstate(over="ignore"):
        s, r = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
        if op == "sigmoid":
            return s * r, 17 * s * r                      # 8 for each factor, their product
        if op == "silu":
            return s * (1 + x * r), s * (10 * np.abs(1 + x * r) + 10 * np.abs(x * r))
        e = np.exp(-2 * np.abs(x))
        return 4 * e / (1 + e) ** 2, 16 * 4 * e / (1 + e) ** 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("op", ["sigmoid", "silu", "tanh"])
@pytest.mark.parametrize("n", [1, 37, 4099, 70001])
def test_unary_forward_and_backward(hip, n, op, dtype):
    T = TYPES[dtype]
    x = values(n, T, n + 1)
    x[::5] *= 30
    x = np.clip(x, -600, 600).astype(T)
    up = values(n, T, n + 2)
    c, e = room(hip, n)
    y, same, dx = poison(hip, x), poison(hip, x), poison(hip, x)
    hip.pack8_unary(op, put(hip, x), 0, n, y, c, e)
    hip.unary_to(op, put(hip, x), 0, n, same)
    assert hip.dump(y).tobytes() == hip.dump(same).tobytes()
    wc, we = R.pack(x)
    assert (hip.dump(c) == wc).all() and (hip.dump(e) == we).all()
    hip.pack8_unary_backward(op, c, e, put(hip, up), n, dx)
    W, u = R.WIDE[T], R.HALF_STEP[T]
    held = R.restore(wc, we, T).astype(W)
    f, b = slope(op, held)
    got = hip.dump(dx)
    # below the normal range the roundings are absolute ones, of half the smallest number each; silu multiplies those of the sigmoid by
    # 1 + x (1 - s), at most 1 + |x|
    tiny = W(np.finfo(T).smallest_subnormal)
    bound = np.abs(up.astype(W)) * (b + 2 * np.abs(f)) * u * 1.01 + 4 * tiny * (1 + np.abs(up.astype(W)) * (1 + np.abs(held)))
    bad = np.abs(got.astype(W) - up.astype(W) * f) > bound
    assert not bad.any(), (held[bad][:5], up[bad][:5], got[bad][:5])
    # in place: y over x, dx over the upstream gradient
    b1, b2 = put(hip, x), put(hip, up)
    hip.pack8_unary(op, b1, 0, n, b1, c, e)
    hip.pack8_unary_backward(op, c, e, b2, n, b2)
    assert hip.dump(b1).tobytes() == hip.dump(y).tobytes() and hip.dump(b2).tobytes() == got.tobytes()


# (b, m, k, n): single rows and columns, sizes around the tiles, ragged ones, a long axis of rows, batches
MATMULS = [(1, 1, 1, 1), (1, 1, 40, 50), (1, 33, 1, 7), (1, 64, 32, 32), (1, 100, 65, 130), (2, 31, 33, 17), (3, 130, 128, 128), (1, 257, 129, 255),
           (1, 1000, 96, 64), (1, 20000, 40, 24), (1, 5000, 256, 320), (5, 64, 20, 300), (1, 512, 384, 512), (1, 2, 700, 900)]


def matmul_case(b, m, k, n, T, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal(b * m * k) * np.exp(rng.standard_normal(b * m * k))).astype(T)
    dy = (rng.standard_normal((b, m, n)) * np.exp(3 * rng.standard_normal((b, m, n)))).astype(T)
    return R.pack(x), dy


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", MATMULS)
def test_matmul_backward(hip, size, dtype):
    """m products summed in any order: off by at most (m + 4) roundings of the sum of magnitudes."""
    T = TYPES[dtype]
    b, m, k, n = size
    (c, e), dy = matmul_case(*size, T, m)
    out = poison(hip, dy, b * k * n + 3)
    hip.pack8_matmul_backward(put(hip, c), put(hip, e), put(hip, dy), out, b, m, k, n)
    W, u = R.WIDE[T], R.HALF_STEP[T]
    x = R.restore(c, e, T).reshape(b, m, k)
    want = np.matmul(x.transpose(0, 2, 1).astype(W), dy.astype(W))
    mag = np.matmul(np.abs(x).transpose(0, 2, 1).astype(W), np.abs(dy).astype(W))
    got = hip.dump(out)
    assert np.isnan(got[b * k * n:]).all()
    got = got[:b * k * n].reshape(b, k, n)
    assert (np.abs(got.astype(W) - want) <= (m + 4) * u * 1.01 * mag).all(), float(np.max(np.abs(got - want) / (u * mag + 1e-300)))
    again = poison(hip, dy, b * k * n)
    hip.pack8_matmul_backward(put(hip, c), put(hip, e), put(hip, dy), again, b, m, k, n)
    assert hip.dump(again).tobytes() == np.ascontiguousarray(got).tobytes()


def test_matmul_of_no_rows_is_zero(hip):
    from rtensors_amd import hip as H
    out = poison(hip, np.zeros(60, np.float32))
    hip.pack8_matmul_backward(*room(hip, 0), hip.alloc(H.F32, 0), out, 1, 0, 6, 10)
    assert (hip.dump(out) == 0).all()


@pytest.mark.parametrize("size", [(1, 70, 40, 50), (1, 300, 200, 260), (1, 4096, 64, 64)])
def test_matmul_of_values_that_are_not_finite(hip, size):
    """Infinities and NaN of the upstream gradient reach exactly the results that the plain product has them in; so do the groups that
    are not finite."""
    b, m, k, n = size
    (c, e), dy = matmul_case(*size, np.float32, 5)
    dy[0, 3, 5], dy[0, 10, 7], dy[0, 20, 9] = np.inf, -np.inf, np.nan
    dy[0, 30, 11] = np.frombuffer(np.uint32(0x7f800001).tobytes(), np.float32)[0]
    dy[0, 31, 12] = 3.3e38
    c = c.copy()
    c.reshape(m, k)[[3, 10, 31]] = np.where(c.reshape(m, k)[[3, 10, 31]] == 0, 1, c.reshape(m, k)[[3, 10, 31]])
    c.reshape(m, k)[3, 8] = 0                              # 0 * inf
    e = e.copy()
    e[(40 * k) // 32] = 255
    e[31 * k // 32: 32 * k // 32 + 1] = 100
    out = poison(hip, dy, k * n)
    hip.pack8_matmul_backward(put(hip, c), put(hip, e), put(hip, dy), out, b, m, k, n)
    x = R.restore(c, e, np.float32).reshape(m, k).astype(np.float64)
    with np.errstate(all="ignore"):
        # element by element: a library product may skip or reorder what is not finite
        want = np.zeros((k, n))
        for r in range(m):
            want += np.outer(x[r], dy[0, r].astype(np.float64))
    got = hip.dump(out).reshape(k, n)
    for kind in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(kind(got), kind(want)), kind


def test_matmul_over_the_range_of_exponents(hip):
    """Upstream gradients from the smallest normal numbers to the largest: what is lost is below the sum's own rounding."""
    m, k, n = 64, 32, 48
    rng = np.random.default_rng(11)
    x = rng.standard_normal(m * k).astype(np.float32)
    c, e = R.pack(x)
    for scale in (2.0 ** -125, 2.0 ** -100, 2.0 ** -60, 1.0, 2.0 ** 60, 2.0 ** 115):
        dy = (rng.standard_normal((m, n)) * scale).astype(np.float32)
        out = poison(hip, dy, k * n)
        hip.pack8_matmul_backward(put(hip, c), put(hip, e), put(hip, dy), out, 1, m, k, n)
        xr = R.restore(c, e, np.float32).reshape(m, k).astype(np.float64)
        want, mag = xr.T @ dy.astype(np.float64), np.abs(xr).T @ np.abs(dy).astype(np.float64)
        # 2^-126 per product: a part of an element below the normal range may be dropped
        bound = (m + 4) * 2.0 ** -24 * 1.01 * mag + np.abs(xr).T @ np.full((m, n), 2.0 ** -126)
        assert (np.abs(hip.dump(out).reshape(k, n) - want) <= bound).all(), scale


def test_more_elements_than_a_launch_has_lanes():
    """More than 2^33 elements: 3 is 96 steps of 2^-5."""
    from rtensors_amd import hip as H
    be, n = H.Hip.new(0), (1 << 33) + 100
    src, (codes, exps) = be.alloc_uninit(H.F32, n), be.alloc_pack8(n)
    be.fill_contiguous(src, 3.0, 0, n)
    be.fill_contiguous(codes, 0, 0, n)
    be.pack8(src, 0, n, codes, exps)
    places = (0, (1 << 33) - 1, 1 << 33, n - 1)
    for i in places:
        assert be.read(codes, i) == 96 and be.read(exps, i // 32) == 122, i
    be.fill_contiguous(src, -1.0, 0, n)
    be.unpack8(codes, exps, n, src)
    for i in places:
        assert be.read(src, i) == 3, i
