"""Calls of the gated scan and of the 8-bit activation entry points that have to be refused.  The arguments are checked before the
context is looked at, so no device is needed: a call that passes the checks ends at the null context instead."""
import ctypes as C

import numpy as np
import pytest

INVALID, DTYPE, BOUNDS = 1, 2, 3
F32, F64, I32 = 10, 11, 6


@pytest.fixture(scope="module")
def lib():
    from rtensors_amd._ffi import lib
    return lib


class Room:
    """Addresses that never get touched: distinct stretches of one host array."""

    def __init__(self):
        self.a = np.zeros(1 << 16, dtype=np.uint8)
        self.base = (self.a.ctypes.data + 255) & ~255
        self.at = 0

    def take(self, nbytes):
        p = self.base + self.at
        self.at += (nbytes + 63) & ~63
        return p


def said(lib):
    return lib.rt_last_error().decode()


def passes(lib, status):
    """Whether the call got as far as the null context."""
    return status == INVALID and "context" in said(lib)


def scan_call(lib, change=None, drop=(), dtype=F32, form=0, sizes=(2, 5, 3), back=None):
    es = 4 if dtype == F32 else 8
    o, t, i = sizes
    n, cols, g = o * t * i, o * i, -(-o * t * i // 32)
    names = {None: ["gate", "x", "state", "reset", "h", "last"],
             "whole": ["gate", "x", "h", "state", "reset", "dh", "dlast", "dgate", "dx", "dstate"],
             "held": ["gate", "xc", "xe", "hc", "he", "state", "reset", "dh", "dlast", "dgate", "dx", "dstate"]}[back]
    room, ops = Room(), {}
    for k in names:
        length = {"reset": o * t, "state": cols, "last": cols, "dlast": cols, "dstate": cols, "xe": g, "he": g}.get(k, n)
        ops[k] = [room.take(max(length, 1) * (1 if k in ("reset", "xc", "xe", "hc", "he") else es)), length]
    for k in drop:
        ops[k] = [None, 0]
    for k, f in (change or {}).items():
        ops[k] = f(ops)
    args = [v for k in names for v in ops[k]]
    fn = {None: lib.rt_gated_scan, "whole": lib.rt_gated_scan_backward, "held": lib.rt_gated_scan_backward_packed8}[back]
    return fn(None, dtype, form, *args, o, t, i)


@pytest.mark.parametrize("back", [None, "whole", "held"])
@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("dtype", [F32, F64])
def test_plain_calls_pass_the_checks(lib, back, form, dtype):
    assert passes(lib, scan_call(lib, dtype=dtype, form=form, back=back)), said(lib)
    optional = ["state", "reset"] + (["last"] if back is None else ["dlast", "dstate"])
    assert passes(lib, scan_call(lib, drop=optional, dtype=dtype, form=form, back=back)), said(lib)
    if back and form == 0:
        assert passes(lib, scan_call(lib, drop=["x"] if back == "whole" else ["xc", "xe"], back=back)), said(lib)


@pytest.mark.parametrize("back", [None, "whole", "held"])
def test_dtype_form_and_sizes(lib, back):
    assert scan_call(lib, dtype=I32, back=back) == DTYPE
    for form in (-1, 2):
        assert scan_call(lib, form=form, back=back) == INVALID and "form" in said(lib)
    for sizes in ((1 << 41, 1, 1), (1 << 20, 1 << 20, 2), (1 << 40, 0, 1 << 30), (1, (1 << 64) - 1, 1), (1 << 63, 1 << 63, 1 << 63)):
        o, t, i = sizes
        fn = {None: lib.rt_gated_scan, "whole": lib.rt_gated_scan_backward, "held": lib.rt_gated_scan_backward_packed8}[back]
        assert fn(None, F32, 0, *[None, 0] * {None: 6, "whole": 10, "held": 12}[back], o, t, i) == INVALID and "too long" in said(lib)


@pytest.mark.parametrize("back", [None, "whole", "held"])
def test_short_null_and_unaligned_operands(lib, back):
    needed = {None: ["gate", "x", "h"], "whole": ["gate", "x", "h", "dh", "dgate", "dx"], "held": ["gate", "xc", "xe", "hc", "he", "dh", "dgate", "dx"]}[back]
    rest = ["state", "reset"] + (["last"] if back is None else ["dlast", "dstate"])
    for k in needed + rest:
        assert scan_call(lib, {k: lambda o, k=k: [o[k][0], o[k][1] - 1]}, form=1, back=back) == BOUNDS and k.replace("c", "").replace("e", "")[:1] in said(lib), k
    for k in needed:
        assert scan_call(lib, drop=[k], form=1, back=back) == INVALID and "null" in said(lib), k
    for k in needed + rest:
        if k not in ("reset", "xc", "xe", "hc", "he"):
            assert scan_call(lib, {k: lambda o, k=k: [o[k][0] + 2, o[k][1]]}, form=1, back=back) == INVALID and "aligned" in said(lib), k


def test_overlaps_of_the_forward_pass(lib):
    for k in ("x", "gate"):
        assert passes(lib, scan_call(lib, {"h": lambda o, k=k: o[k]}))
        assert scan_call(lib, {"h": lambda o, k=k: [o[k][0] + 4, o[k][1]]}) == INVALID and "overlaps" in said(lib)
    assert passes(lib, scan_call(lib, {"last": lambda o: o["state"]}))
    for out, k in (("h", "state"), ("h", "reset"), ("last", "gate"), ("last", "x"), ("last", "reset"), ("last", "h")):
        assert scan_call(lib, {out: lambda o, k=k, out=out: [o[k][0] & ~3, o[out][1]]}) == INVALID and "overlaps" in said(lib), (out, k)


@pytest.mark.parametrize("back", ["whole", "held"])
def test_overlaps_of_the_backward_pass(lib, back):
    for out, k in [("dx", "dh"), ("dstate", "dlast")] + ([("dx", "x")] if back == "whole" else []):
        assert passes(lib, scan_call(lib, {out: lambda o, k=k: o[k]}, form=1, back=back)), (out, k, said(lib))
    others = ["gate", "state", "reset"] + (["h"] if back == "whole" else ["xc", "xe", "hc", "he"])
    for out in ("dgate", "dx", "dstate"):
        for k in others + [m for m in ("dgate", "dx", "dstate") if m != out]:
            assert scan_call(lib, {out: lambda o, k=k, out=out: [o[k][0] & ~3, o[out][1]]}, form=1, back=back) == INVALID and "overlaps" in said(lib), (out, k)
    for k in ("dh",) + (("x",) if back == "whole" else ()):
        assert scan_call(lib, {"dgate": lambda o, k=k: o[k]}, form=1, back=back) == INVALID, k
        assert scan_call(lib, {"dx": lambda o, k=k: [o[k][0] + 4, o["dx"][1]]}, form=1, back=back) == INVALID, k


def test_pack_refusals(lib):
    r = Room()
    src, codes, exps, dst = r.take(400), r.take(100), r.take(8), r.take(400)
    ok = dict(dtype=F32, src=src, n=100, start=0, len=100, codes=codes, cl=100, exps=exps, el=4, dst=dst, dl=100, op=3)

    def pack(**kw):
        a = dict(ok, **kw)
        return lib.rt_pack8(None, a["dtype"], a["src"], a["n"], a["start"], a["len"], a["codes"], a["cl"], a["exps"], a["el"])

    def unary(**kw):
        a = dict(ok, **kw)
        return lib.rt_pack8_unary(None, a["dtype"], a["op"], a["src"], a["n"], a["start"], a["len"], a["dst"], a["dl"], a["codes"], a["cl"], a["exps"], a["el"])

    def unpack(**kw):
        a = dict(ok, **kw)
        return lib.rt_unpack8(None, a["dtype"], a["codes"], a["cl"], a["exps"], a["el"], a["len"], a["dst"], a["dl"])

    def back(**kw):
        a = dict(ok, **kw)
        return lib.rt_pack8_unary_backward(None, a["dtype"], a["op"], a["codes"], a["cl"], a["exps"], a["el"], a["src"], a["n"], a["len"], a["dst"], a["dl"])

    for f in (pack, unary, unpack, back):
        assert passes(lib, f()), said(lib)
        assert f(dtype=I32) == DTYPE
        assert f(cl=99) == BOUNDS and f(el=3) == BOUNDS and f(codes=None) == INVALID and f(exps=None) == INVALID
        assert f(len=(1 << 40) + 1) == INVALID
    for f in (pack, unary):
        assert f(start=1) == BOUNDS and f(start=(1 << 64) - 1) == BOUNDS and f(src=None) == INVALID and f(src=src + 1) == INVALID
        assert f(codes=src + 396) == INVALID and f(exps=src) == INVALID and f(exps=codes + 3) == INVALID
        assert passes(lib, f(len=0, codes=None, exps=None, src=None, dst=None))
    for f in (unary, unpack, back):
        assert f(dl=99) == BOUNDS and f(dst=None) == INVALID and f(dst=dst + 2) == INVALID
    assert passes(lib, unary(dst=src)) and unary(dst=src + 4) == INVALID and unary(dst=codes - 200 & ~3) == INVALID
    assert unary(src=dst - 0, dst=dst, start=1, n=101) == INVALID            # shifted by the start
    assert passes(lib, back(dst=src)) and back(dst=src + 4) == INVALID and back(n=99) == BOUNDS and back(src=None) == INVALID
    assert unpack(dst=codes) == INVALID and unpack(dst=exps) == INVALID
    for f in (unary, back):
        for op in (1, 0, 5, 31):
            assert f(op=op) == DTYPE, op
        for op in (-1, 77):
            assert f(op=op) == INVALID, op


def test_matmul_refusals(lib):
    r = Room()
    b, m, k, n = 2, 4, 10, 6
    ok = dict(dtype=F32, codes=r.take(80), cl=80, exps=r.take(3), el=3, up=r.take(192), ul=48, dst=r.take(480), dl=120, b=b, m=m, k=k, n=n)

    def call(**kw):
        a = dict(ok, **kw)
        return lib.rt_pack8_matmul_backward(None, a["dtype"], a["codes"], a["cl"], a["exps"], a["el"], a["up"], a["ul"], a["dst"], a["dl"], a["b"], a["m"], a["k"], a["n"])

    assert passes(lib, call()), said(lib)
    assert call(dtype=I32) == DTYPE
    for kw in (dict(cl=79), dict(el=2), dict(ul=47), dict(dl=119)):
        assert call(**kw) == BOUNDS, kw
    for kw in (dict(codes=None), dict(exps=None), dict(up=None), dict(dst=None), dict(up=ok["up"] + 2), dict(dst=ok["dst"] + 1), dict(dst=ok["up"]),
               dict(dst=ok["codes"] + 40), dict(dst=ok["exps"] & ~3), dict(m=1 << 40), dict(b=1 << 33, k=1 << 33), dict(n=(1 << 64) - 1)):
        assert call(**kw) == INVALID, kw
    assert passes(lib, call(n=0, dst=None, up=None)) and passes(lib, call(m=0, codes=None, exps=None, up=None))


def test_python_face_refuses_wrong_dtypes():
    from rtensors_amd import hip as H

    class Bare(H.Hip):
        def __init__(self):
            self._ctx = None

    be = Bare()
    f, d, i, u = (be.borrow(4096 * k, 8, t) for k, t in ((1, H.F32), (2, H.F64), (3, H.I8), (4, H.U8)))
    for call in (lambda: be.gated_scan("linear", f, d, f, 1, 8, 1), lambda: be.gated_scan("linear", f, f, f, 1, 8, 1, reset=u),
                 lambda: be.gated_scan_backward("linear", f, None, f, f, f, d, 1, 8, 1), lambda: be.pack8(f, 0, 8, u, u), lambda: be.unpack8(i, i, 8, f),
                 lambda: be.pack8_unary("silu", f, 0, 8, d, i, u), lambda: be.pack8_unary_backward("silu", i, u, d, 8, f),
                 lambda: be.pack8_matmul_backward(i, u, d, f, 1, 2, 4, 4), lambda: be.gated_scan_backward_packed8("linear", f, None, (u, u), f, f, f, 1, 8, 1)):
        with pytest.raises(H.TensorError) as e:
            call()
        assert e.value.status == 2
    with pytest.raises(KeyError):
        be.gated_scan("cubic", f, f, f, 1, 8, 1)
