"""The gated linear recurrence and the 8-bit activation checkpoints: cases to time, plain forms, 64-bit values.

Kinds of case (sizes in elements; `dtype` is "f32" or "f64"):
  scan        h_t = a_t h_{t-1} + b_t over (outer, steps, inner); returns h and the last state
  scan_grad   its backward pass; returns d(gate), d(x), d(state)
  scan_grad8  the same with x and h held in 8 bits
  pack        an activation held in 8 bits and restored; returns the restored values
  act         y = f(x) with x held in 8 bits, then d(x) from the held form; returns y and d(x)
  wgrad       d(w) = x^T d(y) of a projection y = x w, with x held in 8 bits; returns d(w)
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f64": torch.float64}
GROUP = 32          # elements that share an exponent
LOWEST = -119       # the least exponent a group takes


def listed():
    return [
        # one new token for each of 64 requests: the state of every request moves on by one step
        {"name": "scan token", "kind": "scan", "dtype": "f32", "form": "sigmoid", "outer": 64, "steps": 1, "inner": 2048, "state": True, "reset": False},
        # one row of packed documents of a training batch
        {"name": "scan documents", "kind": "scan", "dtype": "f32", "form": "sigmoid", "outer": 1, "steps": 8192, "inner": 1024, "state": False, "reset": True},
        # one long sequence through a wide layer
        {"name": "scan long", "kind": "scan", "dtype": "f32", "form": "linear", "outer": 1, "steps": 65536, "inner": 4096, "state": True, "reset": False},
        # many separate series of an odd length, time contiguous
        {"name": "scan series f64", "kind": "scan", "dtype": "f64", "form": "linear", "outer": 2048, "steps": 4097, "inner": 1, "state": False, "reset": False},
        # backward pass of a training batch of eight sequences, a gradient of the last state among it
        {"name": "scan grad", "kind": "scan_grad", "dtype": "f32", "form": "sigmoid", "outer": 8, "steps": 2048, "inner": 2048, "state": True, "reset": True},
        # backward pass of one long row of documents of an odd width from checkpoints
        {"name": "scan grad packed", "kind": "scan_grad8", "dtype": "f32", "form": "sigmoid", "outer": 1, "steps": 50000, "inner": 1111, "state": False, "reset": True},
        # the activations of a few tokens, a ragged end
        {"name": "pack small", "kind": "pack", "dtype": "f32", "n": 64 * 1024 + 5},
        # a whole layer's activations
        {"name": "pack large", "kind": "pack", "dtype": "f32", "n": 16384 * 16384},
        # the activation of a wide layer, forward and backward
        {"name": "act silu", "kind": "act", "dtype": "f32", "op": "silu", "n": 8192 * 8192},
        # a small layer in doubles, odd sizes
        {"name": "act tanh f64", "kind": "act", "dtype": "f64", "op": "tanh", "n": 1001 * 2047},
        # weight gradient of a square projection over a batch of 16384 tokens
        {"name": "wgrad square", "kind": "wgrad", "dtype": "f32", "m": 16384, "k": 4096, "n": 4096},
        # weight gradient of a narrow projection over a long axis of tokens
        {"name": "wgrad long", "kind": "wgrad", "dtype": "f32", "m": 65536, "k": 256, "n": 320},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["scan", "scan_grad", "scan_grad8", "pack", "act", "wgrad"])
    c = {"kind": kind, "dtype": "f64" if rng.random() < 0.25 else "f32"}
    wide = c["dtype"] == "f32"
    if kind.startswith("scan"):
        most = (1 << 26) if wide else (1 << 25)
        c["form"] = rng.choice(["linear", "sigmoid"])
        c["inner"] = 1 if rng.random() < 0.2 else _size(rng, 2, 8192)
        c["steps"] = _size(rng, 1, min(100000, most // c["inner"]))
        c["outer"] = _size(rng, 1, max(1, min(4096, most // (c["inner"] * c["steps"]))))
        c["state"] = rng.random() < 0.5
        c["reset"] = rng.random() < 0.5
    elif kind == "pack":
        c["n"] = _size(rng, 1000, (1 << 27) if wide else (1 << 26))
    elif kind == "act":
        c["op"] = rng.choice(["silu", "sigmoid", "tanh"])
        c["n"] = _size(rng, 1000, (1 << 26) if wide else (1 << 25))
    else:
        most = 2.5e11 if wide else 5e10
        c["k"] = _size(rng, 16, 6000)
        c["n"] = _size(rng, 16, 6000)
        c["m"] = _size(rng, 1, max(1, min(100000, int(most / (2 * c["k"] * c["n"])))))
    return c


def _packed(x):
    """The 8-bit form of x: whole codes (int8) and the exponent bytes of its groups of 32."""
    n = x.numel()
    g = -(-n // GROUP)
    v = torch.zeros(g * GROUP, dtype=x.dtype, device=x.device)
    v[:n] = x.reshape(-1)
    v = v.view(g, GROUP)
    top = v.abs().amax(dim=1)
    if x.dtype == torch.float32:
        e = (top.view(torch.int32) >> 23) - 133
    else:
        e = ((top.view(torch.int64) >> 52) - 1029).to(torch.int32)
    e = torch.clamp(e, min=LOWEST)
    e = torch.where(top * _two_to(-e, x.dtype) >= 127.5, e + 1, e)
    codes = torch.round(v * _two_to(-e, x.dtype)[:, None]).to(torch.int8)
    return codes.reshape(-1)[:n].contiguous(), (e + 127).to(torch.uint8)


def _two_to(e, dtype):
    """2^e for whole exponents, built from the bits."""
    if dtype == torch.float32:
        return ((e + 127) << 23).view(torch.float32)
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _restored(codes, exps, dtype):
    n = codes.numel()
    s = _two_to(exps.to(torch.int32) - 127, dtype).repeat_interleave(GROUP)[:n]
    return codes.to(dtype) * s


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _steps_doubled(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, h_{-1} = 0, by doubling the stretch that each position covers."""
    a, b, d = a.clone(), b.clone(), 1
    while d < a.shape[1]:
        b[:, d:] = b[:, d:] + a[:, d:] * b[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return b


def _forward(s):
    a, b = s["gate"], s["x"]
    if s["form"] == "sigmoid":
        b = b / (1 + torch.exp(a))
        a = _sigmoid(a)
    if s["reset"] is not None:
        a = torch.where(s["reset"][:, :, None], torch.zeros((), dtype=a.dtype, device=a.device), a)
    if s["state"] is not None:
        b = b.clone()
        b[:, 0] += a[:, 0] * s["state"]
    return _steps_doubled(a, b)


def _backward(s, x, h):
    """d(gate), d(x), d(state) of the recurrence from d(h) and the gradient of the last state."""
    a = _sigmoid(s["gate"]) if s["form"] == "sigmoid" else s["gate"]
    first = s["state"] if s["state"] is not None else torch.zeros_like(h[:, 0])
    before = torch.cat([first[:, None], h[:, :-1]], dim=1)
    carry = a
    if s["reset"] is not None:
        none = torch.zeros((), dtype=a.dtype, device=a.device)
        carry = torch.where(s["reset"][:, :, None], none, carry)
        before = torch.where(s["reset"][:, :, None], none, before)
    up = s["dh"].clone()
    up[:, -1] += s["dlast"]
    after = torch.cat([carry[:, 1:], torch.zeros_like(carry[:, :1])], dim=1)
    total = _steps_doubled(after.flip(1), up.flip(1)).flip(1)
    dstate = carry[:, 0] * total[:, 0]
    if s["form"] == "linear":
        return total * before, total, dstate
    rest = 1 / (1 + torch.exp(s["gate"]))
    return total * (before - x) * (a * rest), total * rest, dstate


def _derivative(op, x):
    if op == "tanh":
        e = torch.exp(-2 * x.abs())
        return 4 * e / ((1 + e) * (1 + e))
    s, rest = _sigmoid(x), 1 / (1 + torch.exp(x))
    return s * rest if op == "sigmoid" else s * (1 + x * rest)


def _function(op, x):
    if op == "tanh":
        a, b = torch.exp(x), torch.exp(-x)
        return (a - b) / (a + b)
    return _sigmoid(x) if op == "sigmoid" else x * _sigmoid(x)


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    s = {k: v for k, v in case.items() if k != "name"}
    if case["kind"].startswith("scan"):
        shape = (case["outer"], case["steps"], case["inner"])
        # gates as a trained layer has them: most states are kept for tens of steps, some for a few
        gate = normal(*shape)
        s["gate"] = 1.5 * gate + 2 if case["form"] == "sigmoid" else _sigmoid(1.5 * gate + 2)
        s["x"] = normal(*shape)
        s["state"] = normal(shape[0], shape[2]) if case["state"] else None
        s["reset"] = torch.rand(shape[:2], generator=g, device="cuda") < 1 / 300 if case["reset"] else None
        if case["kind"] != "scan":
            h = _forward(s)
            s["dh"], s["dlast"] = normal(*shape), normal(shape[0], shape[2])
            if case["kind"] == "scan_grad8":
                s["x8"], s["h8"] = _packed(s.pop("x")), _packed(h)
            else:
                s["h"] = h
    elif case["kind"] == "wgrad":
        s["x8"] = _packed(normal(case["m"], case["k"]))
        s["dy"] = normal(case["m"], case["n"])
    else:
        # activations: a few directions are much larger than the others
        s["x"] = normal(case["n"])
        s["x"][::97] *= 8
        if case["kind"] == "act":
            s["dy"] = normal(case["n"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    like = torch.empty_like
    # what a program that calls again and again keeps: the room for the results
    if case["kind"] == "scan":
        s["out"] = {"h": like(s["x"]), "last": like(s["x"][:, 0])}
    elif case["kind"].startswith("scan"):
        s["out"] = {"dgate": like(s["gate"]), "dx": like(s["gate"]), "dstate": like(s["dlast"])}
    elif case["kind"] == "wgrad":
        s["out"] = {"dw": torch.empty(case["k"], case["n"], dtype=s["dy"].dtype, device="cuda")}
    else:
        s["out"] = {k: like(s["x"]) for k in (("x",) if case["kind"] == "pack" else ("y", "dx"))}
        s["room8"] = (torch.empty(case["n"], dtype=torch.int8, device="cuda"), torch.empty(-(-case["n"] // GROUP), dtype=torch.uint8, device="cuda"))
    if own:
        torch.cuda.current_stream().synchronize()       # the library's context has a stream of its own: what it borrows is there before its first call
    return s


_backend = None


def _run_own(s):
    """The calls go to the context's own stream, one after the other.  Who reads the outputs on another stream, or gives the memory of a
    state back, waits for the context (`_backend.sync()`) or for the device first, as `Hip.borrow` asks."""
    from rtensors_amd import hip as H
    global _backend
    if _backend is None:
        _backend = H.Hip.new(0)
    code = {torch.float32: H.F32, torch.float64: H.F64, torch.bool: H.BOOL, torch.int8: H.I8, torch.uint8: H.U8}

    def buf(t):
        return None if t is None else _backend.borrow(t.data_ptr(), t.numel(), code[t.dtype])

    o, kind = s["out"], s["kind"]
    if kind == "scan":
        _backend.gated_scan(s["form"], buf(s["gate"]), buf(s["x"]), buf(o["h"]), s["outer"], s["steps"], s["inner"],
                            state=buf(s["state"]), reset=buf(s["reset"]), last=buf(o["last"]))
    elif kind == "scan_grad":
        _backend.gated_scan_backward(s["form"], buf(s["gate"]), buf(s["x"]), buf(s["h"]), buf(s["dh"]), buf(o["dgate"]), buf(o["dx"]),
                                     s["outer"], s["steps"], s["inner"], state=buf(s["state"]), reset=buf(s["reset"]), dlast=buf(s["dlast"]),
                                     dstate=buf(o["dstate"]))
    elif kind == "scan_grad8":
        x8 = (buf(s["x8"][0]), buf(s["x8"][1]))
        h8 = (buf(s["h8"][0]), buf(s["h8"][1]))
        _backend.gated_scan_backward_packed8(s["form"], buf(s["gate"]), x8, h8, buf(s["dh"]), buf(o["dgate"]), buf(o["dx"]),
                                             s["outer"], s["steps"], s["inner"], state=buf(s["state"]), reset=buf(s["reset"]), dlast=buf(s["dlast"]),
                                             dstate=buf(o["dstate"]))
    elif kind == "pack":
        codes, exps = buf(s["room8"][0]), buf(s["room8"][1])
        _backend.pack8(buf(s["x"]), 0, s["n"], codes, exps)
        _backend.unpack8(codes, exps, s["n"], buf(o["x"]))
    elif kind == "act":
        codes, exps = buf(s["room8"][0]), buf(s["room8"][1])
        _backend.pack8_unary(s["op"], buf(s["x"]), 0, s["n"], buf(o["y"]), codes, exps)
        _backend.pack8_unary_backward(s["op"], codes, exps, buf(s["dy"]), s["n"], buf(o["dx"]))
    else:
        _backend.pack8_matmul_backward(buf(s["x8"][0]), buf(s["x8"][1]), buf(s["dy"]), buf(o["dw"]), 1, s["m"], s["k"], s["n"])
    return o


def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind == "scan":
        h = _forward(s)
        return {"h": h, "last": h[:, -1].clone()}
    if kind == "pack":
        return {"x": _restored(*_packed(s["x"]), s["x"].dtype)}
    if kind == "act":
        codes, exps = _packed(s["x"])
        return {"y": _function(s["op"], s["x"]), "dx": s["dy"] * _derivative(s["op"], _restored(codes, exps, s["x"].dtype))}
    if kind == "wgrad":
        x = _restored(*s["x8"], s["dy"].dtype).view(s["m"], s["k"])
        return {"dw": x.t() @ s["dy"]}
    if kind == "scan_grad":
        x, h = s["x"], s["h"]
    else:
        x, h = (_restored(*p, s["gate"].dtype).view(s["gate"].shape) for p in (s["x8"], s["h8"]))
    dgate, dx, dstate = _backward(s, x, h)
    return {"dgate": dgate, "dx": dx, "dstate": dstate}


def work(case):
    s = 4 if case["dtype"] == "f32" else 8
    if case["kind"] == "wgrad":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * (1 + 1 / GROUP) + s * (m * n + k * n), "flops": 2 * m * k * n}
    if case["kind"] == "pack":      # read once, the 8-bit form written and read, the values written
        return {"bytes": case["n"] * (2 * s + 2 * (1 + 1 / GROUP)), "flops": 4 * case["n"]}
    if case["kind"] == "act":
        return {"bytes": case["n"] * (4 * s + 2 * (1 + 1 / GROUP)), "flops": 20 * case["n"]}
    n, cols = case["outer"] * case["steps"] * case["inner"], case["outer"] * case["inner"]
    extra = case["outer"] * case["steps"] * int(case["reset"]) + s * cols * (1 + int(case["state"]))
    sig = case["form"] == "sigmoid"
    if case["kind"] == "scan":
        return {"bytes": 3 * s * n + extra, "flops": (10 if sig else 2) * n}
    extra += s * cols
    if case["kind"] == "scan_grad":
        return {"bytes": (6 if sig else 5) * s * n + extra, "flops": (14 if sig else 3) * n}
    return {"bytes": 4 * s * n + (2 if sig else 1) * n * (1 + 1 / GROUP) + extra, "flops": (16 if sig else 4) * n}


def _exact_values(codes, exps):
    at = torch.arange(codes.numel(), device=codes.device) // GROUP
    return torch.ldexp(codes.double(), (exps.double() - 127)[at])


def _exact_held(x):
    """What the 8-bit form of x stands for, in 64 bits."""
    n = x.numel()
    at = torch.arange(n, device=x.device) // GROUP
    top = torch.zeros(-(-n // GROUP), dtype=torch.float64, device=x.device).scatter_reduce(0, at, x.double().abs(), "amax")
    e = torch.frexp(top)[1].double() - 7
    e = torch.clamp(torch.where(torch.round(top * torch.exp2(-e)) > 127, e + 1, e), min=LOWEST)
    step = torch.exp2(e)[at]
    return torch.round(x.double() / step) * step


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "pack":
        return {"x": _exact_held(s["x"])}
    if kind == "act":
        x, held, op = s["x"].double(), _exact_held(s["x"]), case["op"]
        if op == "tanh":
            return {"y": torch.tanh(x), "dx": s["dy"].double() / torch.cosh(held) ** 2}
        p = torch.sigmoid(held)
        slope = p * torch.sigmoid(-held)
        return {"y": torch.sigmoid(x) * (x if op == "silu" else 1), "dx": s["dy"].double() * (p + held * slope if op == "silu" else slope)}
    if kind == "wgrad":
        x = _exact_values(*s["x8"]).view(case["m"], case["k"])
        return {"dw": x.t().contiguous() @ s["dy"].double()}
    steps, sig = case["steps"], case["form"] == "sigmoid"
    a = torch.sigmoid(s["gate"].double()) if sig else s["gate"].double()
    keep = torch.ones(s["gate"].shape[:2], dtype=torch.float64, device="cuda") if s["reset"] is None else (~s["reset"]).double()
    a = a * keep[:, :, None]
    zero = torch.zeros(case["outer"], case["inner"], dtype=torch.float64, device="cuda")
    state = zero if s["state"] is None else s["state"].double()
    if kind == "scan":
        h = s["x"].double() * (torch.sigmoid(-s["gate"].double()) if sig else 1)
        at = state
        for t in range(steps):
            at = torch.addcmul(h[:, t], a[:, t], at)
            h[:, t] = at
        return {"h": h, "last": at}
    d = s["dh"].double()
    at = s["dlast"].double()
    for t in range(steps - 1, -1, -1):
        at = d[:, t] + at if t == steps - 1 else torch.addcmul(d[:, t], a[:, t + 1], at)
        d[:, t] = at
    dstate = a[:, 0] * d[:, 0]
    h = s["h"].double() if kind == "scan_grad" else _exact_values(*s["h8"]).view(d.shape)
    h = torch.cat([state[:, None], h[:, :-1]], dim=1) * keep[:, :, None]
    if not sig:
        return {"dgate": d * h, "dx": d, "dstate": dstate}
    x = s["x"].double() if kind == "scan_grad" else _exact_values(*s["x8"]).view(d.shape)
    rest = torch.sigmoid(-s["gate"].double())
    return {"dgate": d * (h - x) * torch.sigmoid(s["gate"].double()) * rest, "dx": d * rest, "dstate": dstate}
