"""What the mixing layer of a language model with a matrix state is measured on, from the 8-bit rows that `Fused.rmsnorm_q8`
answers to what the layer hands on: the product of 8-bit rows and 8-bit weights, the weights' own way into 8 bits, rotary
positions of queries and keys, and linear attention with a decay for each head, for prompts, for one token at a time and with
its gradients.

A case is a kind of call, an element type and sizes. `run` computes it with elementary tensor operations, or, where
`own` is set, with the library's calls on the library's arrays.

The definitions (element type T; heads: q and g have `heads` of them, k and v `shared` of them, each for heads / shared queries' heads in a row):

quantize        of rows of n: scale = max|x| / 127 (rounded to T);  q = round(x / scale), an 8-bit integer
matmul          y[i, j] = (sum over k of x[i, k] w[j, k]) * xscale[i] * wscale[j] (+ bias[j]), x and w in 8 bits
rotary          for the pairs (u, v) = (x[i], x[i + n]) of a head (halves) or (x[2 i], x[2 i + 1]) (interleaved), i < n, at the
                angle t = position * frequency[i]:  (u cos t - v sin t, v cos t + u sin t) * amplitude;  other elements as they are
attend          S_t = a S_(t-1) + k_t v_t^T;  o_t = scale S_t^T q_t, from S_(-1) = state, for t below the sequence's length; o is 0 behind it
attend_grad     G_t = a G_(t+1) + scale q_t g_t^T, from a G_length = gstate:  gq_t = scale S_t g_t;  gk_t = G_t v_t;  gv_t = G_t^T k_t;  a G_0 for state
"""
import math

import torch

own = False

TYPES = {"SFloat": torch.float32, "DFloat": torch.float64}


def listed():
    return [
        # the activations of one token in 8 bits, on their way into a product
        {"name": "quantize 1x4096", "kind": "quantize", "type": "SFloat", "rows": 1, "cols": 4096},
        # a layer's weights, once when a model is loaded; rows of an odd length
        {"name": "quantize 16384x4095", "kind": "quantize", "type": "SFloat", "rows": 16384, "cols": 4095},
        # a projection for 16 sequences that are being generated: the weights' bytes count
        {"name": "matmul 16x4096x4096", "kind": "matmul", "type": "SFloat", "rows": 16, "inner": 4096, "cols": 4096, "bias": True},
        # the same for a prompt: arithmetic counts; an odd number of tokens
        {"name": "matmul 8191x4096x8192", "kind": "matmul", "type": "SFloat", "rows": 8191, "inner": 4096, "cols": 8192, "bias": False},
        # queries of 64 sequences that are being generated, far into their contexts
        {"name": "rotary 64x1x32x128", "kind": "rotary", "type": "SFloat", "batch": 64, "time": 1, "heads": 32, "dim": 128, "turned": 128, "pairs": "halves", "scaling": "yarn"},
        # queries of a batch of prompts, neighbours in pairs, a part of each head
        {"name": "rotary 4x4096x32x96", "kind": "rotary", "type": "SFloat", "batch": 4, "time": 4096, "heads": 32, "dim": 96, "turned": 64, "pairs": "neighbours", "scaling": "none"},
        # a batch of prompts
        {"name": "attend 8x2048x16x128", "kind": "attend", "type": "SFloat", "batch": 8, "time": 2048, "heads": 16, "shared": 16, "dim": 128, "wide": 128, "order": "time", "ragged": False},
        # one long document, few heads
        {"name": "attend 1x65536x8x64", "kind": "attend", "type": "SFloat", "batch": 1, "time": 65536, "heads": 8, "shared": 8, "dim": 64, "wide": 64, "order": "time", "ragged": False},
        # one token each of 64 sequences that are being generated: the states' bytes count
        {"name": "attend 64x1x16x128", "kind": "attend", "type": "SFloat", "batch": 64, "time": 1, "heads": 16, "shared": 16, "dim": 128, "wide": 128, "order": "time", "ragged": False},
        # prompts of different lengths side by side, heads in front of time, keys shared by heads, odd sizes, in double precision
        {"name": "attend 6x777x12x72x100", "kind": "attend", "type": "DFloat", "batch": 6, "time": 777, "heads": 12, "shared": 4, "dim": 72, "wide": 100, "order": "heads", "ragged": True},
        # the gradients of a training step
        {"name": "attend grad 4x2048x16x128", "kind": "attend_grad", "type": "SFloat", "batch": 4, "time": 2048, "heads": 16, "shared": 16, "dim": 128, "wide": 128, "order": "time", "ragged": False},
        # the same of a few short sequences of different lengths, with shared keys, in double precision
        {"name": "attend grad 3x500x8x64", "kind": "attend_grad", "type": "DFloat", "batch": 3, "time": 500, "heads": 8, "shared": 2, "dim": 64, "wide": 64, "order": "heads", "ragged": True},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm; half of them whole multiples of 16 where they reach that."""
    high = max(low, high)
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = min(high, max(low, n))
    return max(low, n // 16 * 16) if n >= 16 and rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["quantize", "matmul", "matmul", "rotary", "attend", "attend", "attend", "attend_grad", "attend_grad"])
    of_type = rng.choice(["SFloat", "SFloat", "DFloat"])
    half = 2 if of_type == "DFloat" else 1
    if kind == "quantize":
        cols = _spread(rng, 48, 16384)
        return {"kind": kind, "type": of_type, "rows": _spread(rng, 1, 2 ** 26 // half // cols), "cols": cols}
    if kind == "matmul":
        inner, cols = _spread(rng, 64, 16384), _spread(rng, 64, 16384)
        return {"kind": kind, "type": of_type, "rows": _spread(rng, 1, min(8192, 2 ** 37 // (inner * cols))), "inner": inner, "cols": cols, "bias": rng.random() < 0.5}
    if kind == "rotary":
        heads, dim = _spread(rng, 1, 64), 2 * _spread(rng, 8, 128)
        turned = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        batch = _spread(rng, 1, 64)
        time = _spread(rng, 1, min(8192, 2 ** 25 // half // (heads * dim * batch)))
        return {"kind": kind, "type": of_type, "batch": batch, "time": time, "heads": heads, "dim": dim, "turned": turned, "pairs": rng.choice(["halves", "neighbours"]),
                "scaling": rng.choice(["none", "linear", "yarn"])}
    dim, wide = _spread(rng, 16, 256), _spread(rng, 16, 256)
    shared = _spread(rng, 1, 16)
    heads = shared * rng.choice([1, 1, 2, 3, 4])
    most = 2 ** 32 // (2 if kind == "attend_grad" else 1) // (2 * half) // (dim * wide)  # steps of heads of sequences
    time = _spread(rng, 1, min(65536, max(1, most // heads)))
    batch = _spread(rng, 1, max(1, min(64, most // (heads * time), 2 ** 24 // (heads * dim * wide))))
    return {"kind": kind, "type": of_type, "batch": batch, "time": time, "heads": heads, "shared": shared, "dim": dim, "wide": wide,
            "order": rng.choice(["time", "heads"]), "ragged": batch > 1 and rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _normal(gen, shape, dt, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dt) * scale


def _frequencies(case):
    """The angles a step turns, by pair, and the factor on what is turned: a context eight times longer than a model has been trained for."""
    turned, base, factor, trained = case["turned"], 10000.0, 8.0, 4096
    f = base ** (-2.0 * torch.arange(turned // 2, device="cuda", dtype=torch.float64) / turned)
    if case["scaling"] == "none":
        return f, 1.0
    if case["scaling"] == "linear":
        return f / factor, 1.0
    # pairs that turn more than 32 times within the trained length stay, those that turn less than once are slowed, others in between
    at = lambda turns: turned * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), turned - 1)
    part = ((torch.arange(turned // 2, device="cuda", dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - part) + f / factor * part, 0.1 * math.log(factor) + 1


def _lengths(case):
    """From a part of the time to all of it."""
    n, time = case["batch"], case["time"]
    return [time * (k + 1) // n for k in range(n)] if case["ragged"] else [time] * n


def _made(case, seed):
    """The inputs as tensors."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]
    kind = case["kind"]
    if kind == "quantize":
        # rows of different sizes
        return {"x": _normal(gen, (case["rows"], case["cols"]), dt) * torch.exp(_normal(gen, (case["rows"], 1), dt))}
    if kind == "matmul":
        rows, inner, cols = case["rows"], case["inner"], case["cols"]
        bytes_of = lambda n: _normal(gen, (n, inner), torch.float32, 32.0).round().clamp(-127, 127).to(torch.int8)  # noqa: E731
        s = {"x": bytes_of(rows), "xscale": torch.exp(_normal(gen, (rows, 1), dt, 0.3)) / 40, "w": bytes_of(cols), "wscale": torch.exp(_normal(gen, (cols, 1), dt, 0.2)) / 2000}
        return {**s, "bias": _normal(gen, (cols,), dt) if case["bias"] else None}
    if kind == "rotary":
        batch, time = case["batch"], case["time"]
        # each sequence somewhere in a long context
        start = torch.randint(0, 131072, (batch, 1), generator=gen, device="cuda")
        positions = (start + torch.arange(time, device="cuda")).int()
        frequencies, amplitude = _frequencies(case)
        return {"x": _normal(gen, (batch, time, case["heads"], case["dim"]), dt), "positions": positions, "frequencies": frequencies, "amplitude": amplitude}
    batch, time, heads, shared, dim, wide = (case[k] for k in ("batch", "time", "heads", "shared", "dim", "wide"))
    shape = lambda h, d: (batch, time, h, d) if case["order"] == "time" else (batch, h, time, d)  # noqa: E731
    s = {"q": _normal(gen, shape(heads, dim), dt), "k": _normal(gen, shape(shared, dim), dt), "v": _normal(gen, shape(shared, wide), dt)}
    # heads that forget over 8 to 2000 steps
    s["decay"] = 1 - 2.0 ** (-3 - 8 * torch.rand((heads,), generator=gen, device="cuda", dtype=dt))
    s["state"] = _normal(gen, (batch, heads, dim, wide), dt, 2.0)
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[torch.randperm(batch, generator=gen, device="cuda")]
    if kind == "attend_grad":
        s["g"] = _normal(gen, shape(heads, wide), dt)
        s["gstate"] = _normal(gen, (batch, heads, dim, wide), dt, 0.1)
    return s


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

    held = {torch.float32: cumo_amd.SFloat, torch.float64: cumo_amd.DFloat, torch.int32: cumo_amd.Int32, torch.int8: cumo_amd.Int8}
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
def _quantize(s):
    v = s["x"].double()  # (a value next to the border of two integers falls to one side only in more bits)
    scale = (v.abs().amax(-1, keepdim=True) / 127).to(s["x"].dtype)
    q = torch.where(scale > 0, (v / scale.double()).round().clamp(-127, 127), torch.zeros_like(v))
    return {"value": q.to(scale.dtype) * scale, "scale": scale}


def _matmul(s):
    dt = s["xscale"].dtype
    y = (s["x"].to(dt) @ s["w"].to(dt).t()) * s["xscale"] * s["wscale"].t()
    return y if s["bias"] is None else y + s["bias"]


def _rotary(s):
    x, n, halves = s["x"], s["case"]["turned"] // 2, s["case"]["pairs"] == "halves"
    angle = (s["positions"].double().unsqueeze(-1) * s["frequencies"]).unsqueeze(-2)
    cos, sin = ((f(angle) * s["amplitude"]).to(x.dtype) for f in (torch.cos, torch.sin))
    u, v = (x[..., :n], x[..., n:2 * n]) if halves else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    u, v = u * cos - v * sin, v * cos + u * sin
    turned = torch.cat([u, v], -1) if halves else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _powers(a, exponent):
    """a^exponent by head, [heads, ...]; 0 where the exponent is below 0."""
    e = exponent.double()
    p = a.double().reshape(-1, *[1] * e.dim()) ** e.clamp(min=0)
    return torch.where(e < 0, torch.zeros_like(p), p).to(a.dtype)


def _walk(q, k, v, a):
    """o_t = sum over s <= t of a^(t-s) (q_t . k_s) v_s for [batch, heads, time, .], in stretches of 64: within each as a masked
    product, across them by the state before each, which is the stretches' own ones in front of it, each with its decay."""
    b, h, t, d = q.shape
    c = min(64, t)
    n = -(-t // c)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, n * c - t)).reshape(b, h, n, c, x.shape[-1]) for x in (q, k, v))
    i = torch.arange(c, device="cuda")
    within = (q @ k.transpose(-1, -2).contiguous()) * _powers(a, i[:, None] - i).unsqueeze(1)
    o = within @ v
    each = (k * _powers(a, c - 1 - i)[:, None, :, None]).transpose(-1, -2).contiguous() @ v
    m = torch.arange(n, device="cuda")
    before = _powers(a, torch.where(m[:, None] > m, (m[:, None] - 1 - m) * c, torch.full_like(m, -1))) @ each.reshape(b, h, n, -1)
    o = o + (q * _powers(a, i + 1)[:, None, :, None]) @ before.reshape(each.shape)
    return o.reshape(b, h, n * c, -1)[:, :, :t]


def _heads_first(s, names):
    """The arrays as [batch, heads, time, .], a head of k and v for each of q; steps behind a sequence's length are 0."""
    case = s["case"]
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((case["batch"],), case["time"], device="cuda")
    there = torch.arange(case["time"], device="cuda") < lengths[:, None]
    arrays = [s[n] if case["order"] == "heads" else s[n].transpose(1, 2) for n in names]
    arrays = [x.repeat_interleave(case["heads"] // x.shape[1], dim=1) for x in arrays]
    return [torch.where(there[:, None, :, None], x, torch.zeros_like(x)) for x in arrays], lengths


def _ahead(s, lengths, last):
    """Decays by [batch, heads, time, 1]: from the state before the first step to each (last: from each to behind the last step)."""
    t = torch.arange(s["case"]["time"], device="cuda")
    e = lengths[:, None] - 1 - t if last else t + 1 + 0 * lengths[:, None]
    return _powers(s["decay"], e).transpose(0, 1).unsqueeze(-1).contiguous()


def _over_all(s, lengths):
    return _powers(s["decay"], lengths).t()[:, :, None, None]


def _attend(s):
    (q, k, v), lengths = _heads_first(s, ("q", "k", "v"))
    q = q * s["case"]["dim"] ** -0.5
    o = _walk(q, k, v, s["decay"]) + (q * _ahead(s, lengths, False)) @ s["state"]
    state = _over_all(s, lengths) * s["state"] + (k * _ahead(s, lengths, True)).transpose(-1, -2).contiguous() @ v
    return {"o": o.transpose(1, 2), "state": state}


def _attend_grad(s):
    case = s["case"]
    (q, k, v, g), lengths = _heads_first(s, ("q", "k", "v", "g"))
    a, scale = s["decay"], case["dim"] ** -0.5
    q = q * scale
    back = lambda *x: _walk(*(y.flip(2) for y in x), a).flip(2)  # noqa: E731
    flipped = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    first, last = _ahead(s, lengths, False), _ahead(s, lengths, True)
    gq = (_walk(g, v, k, a) + (g * first) @ flipped(s["state"])) * scale
    gk = back(v, g, q) + (v * last) @ flipped(s["gstate"])
    gv = back(k, q, g) + (k * last) @ s["gstate"]
    each = lambda x: x.reshape(case["batch"], case["shared"], -1, *x.shape[2:]).sum(2).transpose(1, 2)  # noqa: E731
    gstate = _over_all(s, lengths) * s["gstate"] + flipped(q * first) @ g
    return {"gq": gq.transpose(1, 2), "gk": each(gk), "gv": each(gv), "gstate": gstate}


def _own(s):
    from cumo_amd import Fused

    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        q, scale = Fused.quantize(s["x"])
        return {"value": _tensor(Fused.dequantize(q, scale)), "scale": _tensor(scale)}
    if kind == "matmul":
        return _tensor(Fused.matmul_q8(s["x"], s["xscale"], s["w"], s["wscale"], s["bias"]))
    if kind == "rotary":
        return _tensor(Fused.rotary(s["x"], s["positions"], s["frequencies"], interleaved=case["pairs"] == "neighbours", amplitude=s["amplitude"]))
    by_time = (lambda x: x) if case["order"] == "time" else (lambda x: x.transpose(0, 2, 1, 3))
    q, k, v = (by_time(s[n]) for n in ("q", "k", "v"))
    if kind == "attend":
        o, state = Fused.linear_attention(q, k, v, s["decay"], s["state"], s["lengths"])
        return {"o": _tensor(o), "state": _tensor(state)}
    got = Fused.linear_attention_grad(by_time(s["g"]), q, k, v, s["decay"], s["state"], s["gstate"], s["lengths"])
    return {name: _tensor(x) for name, x in zip(("gq", "gk", "gv", "gstate"), got)}


def run(s):
    if own:
        return _own(s)
    return {"quantize": _quantize, "matmul": _matmul, "rotary": _rotary, "attend": _attend, "attend_grad": _attend_grad}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "SFloat" else 8
    kind = case["kind"]
    if kind == "quantize":  # (the 8-bit values and their scales; then the values they stand for)
        n = case["rows"] * case["cols"]
        return {"bytes": n * e + n + case["rows"] * e + (n + case["rows"] * e + n * e), "flops": 4 * n}
    if kind == "matmul":
        rows, inner, cols = case["rows"], case["inner"], case["cols"]
        return {"bytes": (rows + cols) * (inner + e) + rows * cols * e + (cols * e if case["bias"] else 0), "flops": 2 * rows * inner * cols}
    if kind == "rotary":
        tokens = case["batch"] * case["time"]
        return {"bytes": 2 * tokens * case["heads"] * case["dim"] * e + tokens * 4 + case["turned"] * 4, "flops": 3 * tokens * case["heads"] * case["turned"]}
    steps = sum(_lengths(case))
    heads, shared, dim, wide = (case[k] for k in ("heads", "shared", "dim", "wide"))
    out, state = case["batch"] * case["time"], case["batch"] * heads * dim * wide
    small = heads * e + (case["batch"] * 4 if case["ragged"] else 0)
    read = steps * (heads * dim + shared * (dim + wide)) * e
    if kind == "attend":
        return {"bytes": read + out * heads * wide * e + 2 * state * e + small, "flops": 4 * steps * heads * dim * wide}
    written = out * (heads * dim + shared * (dim + wide)) * e
    return {"bytes": read + steps * heads * wide * e + written + 3 * state * e + small, "flops": 10 * steps * heads * dim * wide}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """Linear attention one step after the other; products of whole numbers; turns by complex numbers."""
    m = _made(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x = m["x"].double()
        scale = torch.linalg.vector_norm(x, math.inf, dim=1, keepdim=True).div(127).to(m["x"].dtype).double()
        return {"value": torch.floor(x / scale + 0.5) * scale, "scale": scale}
    if kind == "matmul":
        y = torch.mm(m["x"].double() * m["xscale"].double(), (m["w"].double() * m["wscale"].double()).t().contiguous())
        return y if m["bias"] is None else y.add_(m["bias"].double())
    if kind == "rotary":
        x, n = m["x"].double(), case["turned"] // 2
        turn = torch.polar(torch.full((1,), m["amplitude"], device="cuda", dtype=torch.float64), m["positions"].double()[:, :, None, None] * m["frequencies"])
        if case["pairs"] == "halves":
            z = torch.complex(x[..., :n], x[..., n:2 * n]) * turn
            x[..., :n], x[..., n:2 * n] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:2 * n:2], x[..., 1:2 * n:2]) * turn
            x[..., 0:2 * n:2], x[..., 1:2 * n:2] = z.real, z.imag
        return x
    batch, time, heads, shared, dim, wide = (case[k] for k in ("batch", "time", "heads", "shared", "dim", "wide"))
    # [time, batch, heads, .]; each head of k and v beside the heads of q that share it
    order = (1, 0, 2, 3) if case["order"] == "time" else (2, 0, 1, 3)
    by_step = lambda n: m[n].double().permute(order).contiguous()  # noqa: E731
    index = torch.arange(heads, device="cuda") // (heads // shared)
    q, k, v = by_step("q"), by_step("k")[:, :, index], by_step("v")[:, :, index]
    a = m["decay"].double()[:, None, None]
    lengths = m["lengths"] if m["lengths"] is not None else torch.full((batch,), time, device="cuda")
    there = (torch.arange(time, device="cuda")[:, None] < lengths).double()[:, :, None, None, None]
    scale = 1 / math.sqrt(dim)
    grads = kind == "attend_grad"
    g = by_step("g") if grads else None
    state = m["state"].double()
    out = []
    for t in range(time):
        ahead = a * state + k[t].unsqueeze(-1) * v[t].unsqueeze(-2)
        state = torch.lerp(state, ahead, there[t]) if case["ragged"] else ahead
        seen = (state * g[t].unsqueeze(-2)).sum(-1) if grads else (state * q[t].unsqueeze(-1)).sum(-2)
        out.append(seen * there[t].squeeze(-1) * scale)
    if not grads:
        return {"o": torch.stack(out, 1), "state": state}
    gq = torch.stack(out, 1)
    behind = m["gstate"].double()  # what reaches the state that the step leaves
    gk, gv = [], []
    for t in range(time - 1, -1, -1):
        here = behind + scale * q[t].unsqueeze(-1) * g[t].unsqueeze(-2)
        gk.append((here * v[t].unsqueeze(-2)).sum(-1) * there[t].squeeze(-1))
        gv.append((here * k[t].unsqueeze(-1)).sum(-2) * there[t].squeeze(-1))
        behind = torch.lerp(behind, a * here, there[t]) if case["ragged"] else a * here
    each = lambda x: torch.stack(x[::-1], 1).reshape(batch, time, shared, heads // shared, -1).sum(3)  # noqa: E731
    return {"gq": gq, "gk": each(gk), "gv": each(gv), "gstate": behind}
