"""The gated linear recurrence and the 8-bit form of activations in plain numpy, in a wider type than the one under test, with the
error bounds the tests hold the kernels to."""
import numpy as np

WIDE = {np.float32: np.float64, np.float64: np.longdouble}
HALF_STEP = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}       # largest relative error of one rounding
GROUP, LOWEST = 32, -119


def factors(form, gate):
    """a (the factor of the state before) and r (the factor of x) in the type of `gate`."""
    if form == "linear":
        return gate, np.ones_like(gate)
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate))


def scan(form, gate, x, state=None, reset=None):
    """h and, for each element, the sums M (of the magnitudes that h is a sum of) and S (each of them times the steps it was carried)."""
    W = WIDE[gate.dtype.type]
    a, r = factors(form, gate.astype(W))
    b = r * x.astype(W)
    outer, steps, inner = gate.shape
    h, M, S = np.zeros((3, outer, steps, inner), dtype=W)
    p = np.zeros((outer, inner), dtype=W) if state is None else state.astype(W)
    m, s = np.abs(p), np.zeros_like(p)
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(steps):
            cut = np.zeros((outer, 1), dtype=bool) if reset is None else reset[:, t, None] != 0
            if t == 0 and state is None:
                cut = np.ones((outer, 1), dtype=bool)
            p = np.where(cut, b[:, t], a[:, t] * p + b[:, t])
            m = np.where(cut, np.abs(b[:, t]), np.abs(a[:, t]) * m + np.abs(b[:, t]))
            s = np.where(cut, m, np.abs(a[:, t]) * s + m)
            h[:, t], M[:, t], S[:, t] = p, m, s
    return h, M, S


# Roundings a step adds to everything it carries: the product and the sum (LINEAR); for SIGMOID also those of the factor -- the
# exponential (4 half steps), 1 + e, the quotient (2), and for 1 - s the product with e.
PER_STEP = {"linear": 2, "sigmoid": 10}
# Roundings that come once: joining stretches that were summed apart (two for each of at most six levels), and the last ones.
ONCE = 16


def scan_bound(form, dtype, M, S):
    return HALF_STEP[dtype] * 1.01 * (PER_STEP[form] * S + ONCE * M)


def scan_backward(form, gate, x, h, dh, state=None, reset=None, dlast=None):
    """dgate, dx, dstate with a bound for each."""
    W, u = WIDE[gate.dtype.type], HALF_STEP[gate.dtype.type]
    a, r = factors(form, gate.astype(W))
    outer, steps, inner = gate.shape
    D, M, S = np.zeros((3, outer, steps, inner), dtype=W)
    carry, m, s = (np.zeros((outer, inner), dtype=W) if dlast is None else dlast.astype(W)), None, None
    m, s = np.abs(carry), np.zeros_like(carry)
    none = np.zeros((outer, steps, 1), dtype=bool) if reset is None else (reset != 0)[:, :, None].copy()
    cut = none.copy()
    if state is None and form == "linear" and steps:
        cut[:, 0] = True
    for t in range(steps - 1, -1, -1):
        d = dh[:, t].astype(W)
        D[:, t], M[:, t] = d + carry, np.abs(d) + m
        S[:, t] = s + M[:, t]
        carry = np.where(none[:, t], 0, a[:, t] * D[:, t])
        m, s = np.where(none[:, t], 0, np.abs(a[:, t]) * M[:, t]), np.where(none[:, t], 0, np.abs(a[:, t]) * S[:, t])
    first = np.zeros((outer, 1, inner), dtype=W) if state is None else state.astype(W)[:, None]
    before = np.concatenate([first, h.astype(W)[:, :-1]], axis=1) if steps else h.astype(W)
    before = np.where(none, 0, before)
    bD = scan_bound(form, gate.dtype.type, M, S)
    # the gradient of the state carries D one step further
    bstate = u * 1.01 * (PER_STEP[form] * (s + m) + ONCE * m)
    if form == "linear":
        before = np.where(cut, 0, before)
        return (D * before, np.abs(before) * (bD + 2 * u * np.abs(D))), (D, bD), (carry, bstate)
    dg = D * (before - x.astype(W)) * (a * r)
    slope = np.abs(before - x.astype(W)) * (a * r)
    # the difference (1), two factors (8 each), three products
    return (dg, slope * (bD + 20 * u * np.abs(D))), (r * D, r * (bD + 9 * u * np.abs(D))), (carry, bstate)


def pack(x):
    """codes, exponent bytes of the 8-bit form of a 1-D float array."""
    n = x.size
    groups = -(-n // GROUP)
    v = np.zeros(groups * GROUP, dtype=np.float64)
    v[:n] = x
    v = v.reshape(groups, GROUP)
    fine = np.isfinite(v).all(axis=1)
    top = np.where(fine, np.abs(np.where(np.isfinite(v), v, 0)).max(axis=1, initial=0), 0)
    e = np.frexp(top)[1].astype(np.int64) - 7
    e = np.maximum(e, -1000)
    e = np.where(np.rint(np.ldexp(top, -e)) > 127, e + 1, e)
    e = np.where(top == 0, LOWEST, np.maximum(e, LOWEST))
    fine &= e <= 127
    codes = np.zeros((groups, GROUP), dtype=np.int8)
    codes[fine] = np.rint(np.ldexp(v[fine], -e[fine, None]))
    return codes.reshape(-1)[:n], np.where(fine, e + 127, 255).astype(np.uint8)


def restore(codes, exps, dtype):
    e = np.repeat(exps.astype(np.int64), GROUP)[:codes.size]
    out = np.ldexp(codes.astype(np.float64), e - 127)
    out[e == 255] = np.nan
    return out.astype(dtype)
