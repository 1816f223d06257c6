"""What the row operators and the recurrence of `Fused` are measured on: root-mean-square normalisation with the
residual's addition (its 8-bit output and its gradients too), the gated linear recurrence with its gradients, and the
choice of a token from a row of logits. These are what stands between the matrix products of a recurrent language
model: the recurrence mixes along time, the normalisation stands before and behind it, and the last row's logits are
sampled.

A case is a kind of call, an element type and sizes. `run` computes it with elementary tensor operations, or, where
`own` is set, with the library's calls on the library's arrays.

The definitions, for rows of n elements (s, y, q of the element type T unless said otherwise):

norm        s = x + residual (rounded to T);  r = (sum(s^2) / n + eps)^(-1/2);  y = s r w
norm_q8     the same y, not rounded;  scale = max|y| / 127 (rounded to T);  q = round(y / scale), an 8-bit integer
norm_grad   c = r^2 sum(g w s) / n;  gx = r (g w - s c) + gs;  gw = sum over rows of g s r   (gs: what reaches s by the residual stream)
scan        h_t = a_t h_(t-1) + b_t along one axis, from h0
scan_grad   l_t = g_t + a_(t+1) l_(t+1) from the end;  gb = l;  ga_t = l_t h_(t-1);  gh0 = a_0 l_0
sample      w = exp((x - max x) / temperature), in order of falling x, equal ones by index. Of that order the first top_k
            stay; of these the shortest run from the start whose weights are top_p of the sum or more; of these the ones of
            weight min_p or more. The token is the first of those left whose running sum of weights exceeds u times theirs.
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"SFloat": torch.float32, "DFloat": torch.float64}


def listed():
    return [
        # one token's activations on their way through a block: a row, latency alone
        {"name": "norm 1x4096", "kind": "norm", "type": "SFloat", "rows": 1, "cols": 4096},
        # the activations of a prompt or a training step
        {"name": "norm 8192x4096", "kind": "norm", "type": "SFloat", "rows": 8192, "cols": 4096},
        # the same for a product in 8 bits, with rows of an odd length
        {"name": "norm q8 8192x4095", "kind": "norm_q8", "type": "SFloat", "rows": 8192, "cols": 4095},
        # the gradients of a training step
        {"name": "norm grad 8192x4096", "kind": "norm_grad", "type": "SFloat", "rows": 8192, "cols": 4096},
        # gradients of many short rows (one a head or a group of features), of an odd length, in double precision
        {"name": "norm grad 131072x257", "kind": "norm_grad", "type": "DFloat", "rows": 131072, "cols": 257},
        # a step of 64 sequences that are being generated: one token each, the state carried along
        {"name": "recurrence 64x1x4096", "kind": "scan", "type": "SFloat", "batch": 64, "time": 1, "cols": 4096, "along": "time"},
        # a batch of a training step, channels side by side
        {"name": "recurrence 8x4096x2048", "kind": "scan", "type": "SFloat", "batch": 8, "time": 4096, "cols": 2048, "along": "time"},
        # one long document with few channels, not a whole number of vectors of them
        {"name": "recurrence 1x65536x1000", "kind": "scan", "type": "SFloat", "batch": 1, "time": 65536, "cols": 1000, "along": "time"},
        # time along memory, a filter bank in double precision, odd length
        {"name": "recurrence 4096x4095 rows", "kind": "scan", "type": "DFloat", "batch": 1, "time": 4095, "cols": 4096, "along": "rows"},
        # the gradients of a training step
        {"name": "recurrence grad 8x2048x2048", "kind": "scan_grad", "type": "SFloat", "batch": 8, "time": 2048, "cols": 2048, "along": "time"},
        # the next token of one sequence, from a large vocabulary
        {"name": "sample 1x131072", "kind": "sample", "type": "SFloat", "rows": 1, "cols": 131072, "params": "all"},
        # the next tokens of a batch of requests, each with settings of its own; a vocabulary of an odd size
        {"name": "sample 256x50001", "kind": "sample", "type": "SFloat", "rows": 256, "cols": 50001, "params": "each"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm; half of them whole multiples of 16 where they reach that."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = min(high, max(low, n))
    return n // 16 * 16 if n >= 16 and rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["norm", "norm_q8", "norm_grad", "scan", "scan", "scan_grad", "sample", "sample"])
    kind_type = rng.choice(["SFloat", "SFloat", "DFloat"])
    half = 2 if kind_type == "DFloat" else 1
    if kind.startswith("norm"):
        cols = _spread(rng, 48, 16384)
        rows = _spread(rng, 1, min(131072, 2 ** 25 // half // cols))
        return {"kind": kind, "type": kind_type, "rows": rows, "cols": cols}
    if kind == "sample":
        cols = _spread(rng, 1000, 131072)
        rows = _spread(rng, 1, min(256, 256 * 50001 // half // cols))
        return {"kind": kind, "type": kind_type, "rows": rows, "cols": cols, "params": rng.choice(["none", "top_k", "top_p", "all", "each"])}
    most = (2 ** 26 if kind == "scan" else 2 ** 25) // half
    time = _spread(rng, 1, 65536)
    cols = _spread(rng, 16, min(4096, most // time))
    batch = _spread(rng, 1, max(1, min(64, most // (time * cols))))
    return {"kind": kind, "type": kind_type, "batch": batch, "time": time, "cols": cols, "along": rng.choice(["time", "time", "rows"])}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _axis(case):
    return 1 if case["along"] == "time" else 2


def _normal(gen, shape, dt, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dt) * scale


def _made(case, seed):
    """The inputs as tensors."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]
    kind = case["kind"]
    if kind.startswith("norm"):
        shape = (case["rows"], case["cols"])
        w = 1 + _normal(gen, (case["cols"],), dt, 0.1)
        s = {"x": _normal(gen, shape, dt), "residual": _normal(gen, shape, dt, 3.0), "w": w}
        if kind == "norm_grad":
            # what the forward pass left, and what comes back to its two results
            s = {"s": s["x"] + s["residual"], "w": w, "g": _normal(gen, shape, dt), "gs": _normal(gen, shape, dt)}
        return s
    if kind == "sample":
        rows, cols = case["rows"], case["cols"]
        x = _normal(gen, (rows, cols), dt, 2.5)
        # a few tokens that stand out, and a share that may not be chosen
        x = torch.where(torch.rand((rows, cols), generator=gen, device="cuda") < 20.0 / cols, x + 6, x)
        x = torch.where(torch.rand((rows, cols), generator=gen, device="cuda") < 0.01, torch.full_like(x, -math.inf), x)
        s = {"x": x, "u": torch.rand((rows,), generator=gen, device="cuda", dtype=dt), "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
        if case["params"] in ("top_k", "all"):
            s["top_k"] = 50
        if case["params"] in ("top_p", "all"):
            s["top_p"] = 0.95
        if case["params"] == "all":
            s["temperature"], s["min_p"] = 0.8, 0.02
        if case["params"] == "each":
            pick = torch.randint(0, 4, (rows,), generator=gen, device="cuda")
            r = torch.rand((rows, 4), generator=gen, device="cuda", dtype=dt)
            s["temperature"] = torch.where(pick == 0, torch.zeros_like(r[:, 0]), 0.5 + r[:, 0])  # (0: the most probable token)
            s["top_k"] = torch.where(pick == 1, 1 + (r[:, 1] * 200).int(), torch.zeros_like(pick, dtype=torch.int32))
            s["top_p"] = torch.where(pick >= 2, 0.5 + 0.5 * r[:, 2], torch.ones_like(r[:, 2]))
            s["min_p"] = torch.where(pick == 3, 0.1 * r[:, 3], torch.zeros_like(r[:, 3]))
        return s
    shape = (case["batch"], case["time"], case["cols"]) if case["along"] == "time" else (case["batch"], case["cols"], case["time"])
    # gates that forget over ten to a thousand steps, and one in five hundred that forgets everything (another document begins)
    a = 1 - 10 ** (-1 - 2 * torch.rand(shape, generator=gen, device="cuda", dtype=dt))
    a = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.002, torch.zeros_like(a), a)
    b = _normal(gen, shape, dt) * torch.sqrt(1 - a * a)
    h0 = _normal(gen, (case["batch"], case["cols"]), dt)
    if kind == "scan":
        return {"a": a, "b": b, "h0": h0, "axis": _axis(case)}
    return {"a": a, "h": _scan(a, b, h0, _axis(case)), "h0": h0, "g": _normal(gen, shape, dt), "axis": _axis(case)}


class _Memory:
    """An array's memory for torch; holds the array."""

    def __init__(self, a, typestr):
        self.array = a
        self.__cuda_array_interface__ = {"shape": a.shape, "typestr": typestr, "data": (a._ptr(), False), "version": 2}


_TYPESTR = {"sfloat": "<f4", "dfloat": "<f8", "int32": "<i4", "int8": "|i1"}


def _tensor(a):
    return torch.as_tensor(_Memory(a, _TYPESTR[a.type_name]), device="cuda")


def prepare(case, seed):
    """The same values either way; where the library is called they are in arrays of its pool, as in any program that uses it."""
    made = _made(case, seed)
    if not own:
        return {"case": case, **made}
    import cumo_amd

    held = {torch.float32: cumo_amd.SFloat, torch.float64: cumo_amd.DFloat, torch.int32: cumo_amd.Int32}
    state = {"case": case}
    for name, v in made.items():
        if isinstance(v, torch.Tensor):
            state[name] = held[v.dtype](*v.shape)
            _tensor(state[name]).copy_(v)
        else:
            state[name] = v
    return state


# ---------------------------------------------------------------------------------------------------------------
# the operators in elementary operations
# ---------------------------------------------------------------------------------------------------------------
def _norm(s):
    total = s["x"] + s["residual"]
    r = torch.rsqrt((total * total).mean(-1, keepdim=True) + EPS)
    return {"y": total * r * s["w"], "s": total}


def _norm_q8(s):
    total = s["x"] + s["residual"]
    v = total.double()  # (a value next to the border of two integers falls to one side only in more bits)
    y = v * ((v * v).mean(-1, keepdim=True) + EPS) ** -0.5 * s["w"].double()
    scale = (y.abs().amax(-1, keepdim=True) / 127).to(total.dtype)
    q = torch.where(scale > 0, (y / scale.double()).round().clamp(-127, 127), torch.zeros_like(y))
    return {"value": q.to(total.dtype) * scale, "scale": scale, "s": total}


def _norm_grad(s):
    r = torch.rsqrt((s["s"] * s["s"]).mean(-1, keepdim=True) + EPS)
    gw = s["g"] * s["w"]
    c = r * r * (gw * s["s"]).mean(-1, keepdim=True)
    return {"gx": r * (gw - s["s"] * c) + s["gs"], "gw": (s["g"] * s["s"] * r).sum(0)}


def _scan(a, b, h0, axis):
    """Doubling: after the step of length k every pair (a, b) stands for the 2 k elements that end with it."""
    first = b.narrow(axis, 0, 1) + a.narrow(axis, 0, 1) * h0.unsqueeze(axis)
    n, k = b.shape[axis], 1
    b = torch.cat([first, b.narrow(axis, 1, n - 1)], axis)
    while k < n:
        later = a.narrow(axis, k, n - k)
        b = torch.cat([b.narrow(axis, 0, k), b.narrow(axis, k, n - k) + later * b.narrow(axis, 0, n - k)], axis)
        a = torch.cat([a.narrow(axis, 0, k), later * a.narrow(axis, 0, n - k)], axis)
        k *= 2
    return b


def _scan_grad(s):
    a, h, axis = s["a"], s["h"], s["axis"]
    n = a.shape[axis]
    zero = torch.zeros_like(s["h0"])
    after = torch.cat([a.narrow(axis, 1, n - 1), zero.unsqueeze(axis)], axis)
    gb = _scan(after.flip(axis), s["g"].flip(axis), zero, axis).flip(axis)
    before = torch.cat([s["h0"].unsqueeze(axis), h.narrow(axis, 0, n - 1)], axis)
    return {"ga": gb * before, "gb": gb, "gh0": (a * gb).select(axis, 0)}


def _sample(s):
    rows, n = s["x"].shape
    each = lambda v: v.double().unsqueeze(1) if isinstance(v, torch.Tensor) else torch.full((rows, 1), float(v), dtype=torch.float64, device="cuda")  # noqa: E731
    temperature, top_k, top_p, min_p = (each(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    greedy = temperature <= 0
    top_k = torch.where(greedy, torch.ones_like(top_k), torch.where(top_k <= 0, torch.full_like(top_k, n), top_k))
    x, order = torch.sort(s["x"], dim=1, descending=True, stable=True)
    # in 64 bits: the sums are long, and a token at the border of two falls to one side only so
    z = x.double() / torch.where(greedy, torch.ones_like(temperature), temperature)
    w = torch.exp(z - z[:, :1])
    w = torch.where(torch.arange(n, device="cuda") < top_k, w, torch.zeros_like(w))
    before = w.cumsum(1) - w
    w = torch.where((before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1), w, torch.zeros_like(w))
    w = torch.where(w >= min_p, w, torch.zeros_like(w))
    run = w.cumsum(1)
    at = (run <= each(s["u"]) * run[:, -1:]).sum(1, keepdim=True)
    return order.gather(1, torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)).squeeze(1).int()


def _own(s):
    from cumo_amd import Fused

    kind = s["case"]["kind"]
    if kind == "norm":
        y, total = Fused.rmsnorm(s["x"], s["w"], s["residual"], EPS)
        return {"y": _tensor(y), "s": _tensor(total)}
    if kind == "norm_q8":
        q, scale, total = Fused.rmsnorm_q8(s["x"], s["w"], s["residual"], EPS)
        return {"value": _tensor(Fused.dequantize(q, scale)), "scale": _tensor(scale), "s": _tensor(total)}
    if kind == "norm_grad":
        gx, gw = Fused.rmsnorm_grad(s["g"], s["s"], s["w"], s["gs"], EPS)
        return {"gx": _tensor(gx), "gw": _tensor(gw)}
    if kind == "scan":
        return {"h": _tensor(Fused.recurrence(s["a"], s["b"], s["h0"], axis=s["axis"]))}
    if kind == "scan_grad":
        ga, gb, gh0 = Fused.recurrence_grad(s["g"], s["a"], s["h"], s["h0"], axis=s["axis"])
        return {"ga": _tensor(ga), "gb": _tensor(gb), "gh0": _tensor(gh0)}
    return _tensor(Fused.sample(s["x"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"]))


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "scan":
        return {"h": _scan(s["a"], s["b"], s["h0"], s["axis"])}
    return {"norm": _norm, "norm_q8": _norm_q8, "norm_grad": _norm_grad, "scan_grad": _scan_grad, "sample": _sample}[kind](s)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "SFloat" else 8
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["cols"]
        return {"bytes": n * e + case["rows"] * ((5 if case["params"] == "each" else 1) * e + 4), "flops": 4 * n}
    if kind.startswith("norm"):
        n, cols, rows = case["rows"] * case["cols"], case["cols"], case["rows"]
        if kind == "norm":
            return {"bytes": (4 * n + cols) * e, "flops": 5 * n}
        if kind == "norm_q8":  # (the 8-bit values and their scales; then the values they stand for)
            return {"bytes": (3 * n + cols + rows) * e + n + (n + rows * e + n * e), "flops": 8 * n}
        return {"bytes": (4 * n + 2 * cols) * e, "flops": 11 * n}
    n, state = case["batch"] * case["time"] * case["cols"], case["batch"] * case["cols"]
    if kind == "scan":
        return {"bytes": (3 * n + state) * e, "flops": 2 * n}
    return {"bytes": (5 * n + 2 * state) * e, "flops": 3 * n}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """Rows by norms of vectors, the recurrence one step after the other. None for tokens, which are whole numbers."""
    kind = case["kind"]
    if kind == "sample":
        return None
    m = _made(case, seed)
    if kind in ("norm", "norm_q8"):
        total = (m["x"] + m["residual"])
        d = total.double()
        length = torch.sqrt(torch.linalg.vector_norm(d, dim=1, keepdim=True) ** 2 / case["cols"] + EPS)
        y = torch.div(d, length).mul_(m["w"].double())
        if kind == "norm":
            return {"y": y, "s": d}
        most = torch.linalg.vector_norm(y, math.inf, dim=1, keepdim=True)
        scale = most.div(127).to(total.dtype).double()
        return {"value": torch.floor(y / scale + 0.5) * scale, "scale": scale, "s": d}
    if kind == "norm_grad":
        d, g, w, gs = (m[k].double() for k in ("s", "g", "w", "gs"))
        length = torch.sqrt(torch.linalg.vector_norm(d, dim=1, keepdim=True) ** 2 / case["cols"] + EPS)
        unit = d / length
        back = g * w
        along = torch.linalg.vecdot(back, unit, dim=1).unsqueeze(1) / case["cols"]
        return {"gx": (back - unit * along) / length + gs, "gw": torch.linalg.vecdot(g, unit, dim=0)}
    axis = _axis(case)
    a = m["a"].double().movedim(axis, 0).contiguous()
    state = m["h0"].double()
    if kind == "scan":
        b = m["b"].double().movedim(axis, 0).contiguous()
        for t in range(case["time"]):
            state = torch.addcmul(b[t], a[t], state, out=b[t])
        return {"h": b.movedim(0, axis)}
    h = m["h"].double().movedim(axis, 0).contiguous()
    gb = m["g"].double().movedim(axis, 0).contiguous()
    for t in range(case["time"] - 2, -1, -1):
        torch.addcmul(gb[t], a[t + 1], gb[t + 1], out=gb[t])
    ga = torch.empty_like(gb)
    torch.mul(gb[1:], h[:-1], out=ga[1:])
    torch.mul(gb[0], state, out=ga[0])
    return {"ga": ga.movedim(0, axis), "gb": gb.movedim(0, axis), "gh0": a[0] * gb[0]}
