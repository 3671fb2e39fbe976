"""Cases for the sequence-model operators: root-mean-square norm with the residual's addition, rotary positions, attention
with a sliding window and sinks, and the gated dense layer, each forward (serving) and with its gradients (training).

`run` computes a case in plain torch operations, or, with `own` set, through this framework's graphs.  All arrays are
32-bit floats (the framework's one array type); positions and lengths are whole numbers.
"""
import math

import torch

own = False

# ------------------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # one decoding step of eight sequences: the norm in front of a layer, latency only
        {"name": "norm_token", "op": "norm", "rows": 8, "width": 2048, "residual": True, "train": False},
        # a training step's norm over a width that is no multiple of a wavefront
        {"name": "norm_train_odd", "op": "norm", "rows": 4095, "width": 1000, "residual": False, "train": True},
        # a large training step, with the residual stream added and its gradient joined: bandwidth
        {"name": "norm_train_large", "op": "norm", "rows": 16384, "width": 4096, "residual": True, "train": True},
        # one decoding step: a query row per sequence, far positions of a long context
        {"name": "rotary_token", "op": "rotary", "batch": 32, "tokens": 1, "heads": 32, "dim": 128, "pairs": 64,
         "layout": "half", "far": 1000000, "train": False},
        # training, rotation of part of the head only, neighbouring pairs, odd number of tokens
        {"name": "rotary_train_part", "op": "rotary", "batch": 2, "tokens": 2047, "heads": 16, "dim": 80, "pairs": 20,
         "layout": "interleaved", "far": 0, "train": True},
        # the queries of a long prompt: bandwidth
        {"name": "rotary_prompt", "op": "rotary", "batch": 2, "tokens": 8192, "heads": 32, "dim": 128, "pairs": 64,
         "layout": "half", "far": 4096, "train": False},
        # one decoding step over a long cache: grouped heads, sequences of differing lengths
        {"name": "attention_token", "op": "attention", "batch": 16, "tokens": 1, "keys": 16384, "heads": 32, "groups": 8,
         "dim": 128, "window": 4096, "sinks": 4, "ragged": True, "train": False},
        # a training step on a padded batch of odd length
        {"name": "attention_train", "op": "attention", "batch": 4, "tokens": 1023, "keys": 1023, "heads": 12, "groups": 4,
         "dim": 64, "window": 256, "sinks": 2, "ragged": True, "train": True},
        # a long prompt read in one piece
        {"name": "attention_prompt", "op": "attention", "batch": 1, "tokens": 8192, "keys": 8192, "heads": 16, "groups": 4,
         "dim": 128, "window": 1024, "sinks": 4, "ragged": False, "train": False},
        # one decoding step of four sequences: the weights' bytes
        {"name": "gated_token", "op": "gated", "rows": 4, "width": 1024, "hidden": 4096, "activation": "silu", "train": False},
        # a training step with odd sizes
        {"name": "gated_train_odd", "op": "gated", "rows": 1001, "width": 500, "hidden": 1366, "activation": "gelu", "train": True},
        # a large training step: the matrix units
        {"name": "gated_train_large", "op": "gated", "rows": 8192, "width": 2048, "hidden": 8192, "activation": "silu",
         "train": True},
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "attention", "gated"])
    train = rng.random() < 0.5
    if op == "norm":
        width = _log_between(rng, 32, 8192)
        rows = _log_between(rng, 1, max(1, min(32768, (1 << 26) // width)))
        return {"op": op, "rows": rows, "width": width, "residual": rng.random() < 0.5, "train": train}
    if op == "rotary":
        heads = rng.choice([1, 3, 8, 16, 32])
        dim = rng.choice([32, 48, 64, 80, 96, 128, 256])
        pairs = rng.choice([dim // 2, dim // 4, 8])
        batch = _log_between(rng, 1, 32)
        tokens = 1 if rng.random() < 0.2 else _log_between(rng, 2, max(2, (1 << 26) // (batch * heads * dim)))
        return {"op": op, "batch": batch, "tokens": min(tokens, 16384), "heads": heads, "dim": dim, "pairs": pairs,
                "layout": rng.choice(["half", "interleaved"]), "far": rng.choice([0, 5000, 1000000]), "train": train}
    if op == "attention":
        groups = rng.choice([1, 2, 4, 8])
        heads = groups * rng.choice([1, 2, 3, 4])
        dim = rng.choice([32, 40, 64, 80, 96, 128])
        window = rng.choice([0, 1, 100, 256, 1024, 4096])
        sinks = rng.choice([0, 1, 4, 100])
        if rng.random() < 0.4:  # a decoding step
            batch = _log_between(rng, 1, 32)
            keys = _log_between(rng, 16, max(32, min(32768, (1 << 28) // (batch * groups * dim))))
            return {"op": op, "batch": batch, "tokens": 1, "keys": keys, "heads": heads, "groups": groups, "dim": dim,
                    "window": window, "sinks": sinks, "ragged": rng.random() < 0.7, "train": False}
        batch = rng.choice([1, 2, 4])
        most = int(math.sqrt((1 << 29) / (batch * heads)))
        keys = _log_between(rng, 16, min(8192, most))
        tokens = keys if train or rng.random() < 0.6 else rng.randint(1, keys)  # or a chunk behind what the cache holds
        return {"op": op, "batch": batch, "tokens": tokens, "keys": keys, "heads": heads, "groups": groups, "dim": dim,
                "window": window, "sinks": sinks, "ragged": rng.random() < 0.7, "train": train}
    width = _log_between(rng, 64, 4096)
    hidden = _log_between(rng, 64, 8192)
    rows = _log_between(rng, 1, max(1, min(8192, (1 << 36) // (width * hidden))))
    return {"op": op, "rows": rows, "width": width, "hidden": hidden,
            "activation": rng.choice(["silu", "gelu", "relu", "sigmoid"]), "train": train}


# ----------------------------------------------------------------------------------------------------------- inputs

EPSILON = 1e-6


def _inputs(case, seed):
    """The case's arrays, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 12345)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale

    def whole(low, high, count):
        return torch.randint(low, high + 1, (count,), generator=gen, device="cuda", dtype=torch.int64)

    op = case["op"]
    if op == "norm":
        shape = (case["rows"], case["width"])
        t = {"x": normal(*shape), "weight": 1.0 + 0.1 * normal(case["width"])}
        if case["residual"]:
            t["residual"] = normal(*shape, scale=3.0)
        if case["train"]:
            t["dy"] = normal(*shape, scale=0.1)
            if case["residual"]:
                t["dsum"] = normal(*shape, scale=0.1)
        return t
    if op == "rotary":
        shape = (case["batch"], case["tokens"], case["heads"], case["dim"])
        pairs = case["pairs"]
        table = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        t = {"x": normal(*shape), "frequencies": table.to(torch.float32),
             "positions": whole(case["far"] // 2, case["far"], case["batch"])}
        if case["train"]:
            t["dy"] = normal(*shape, scale=0.1)
        return t
    if op == "attention":
        batch, tokens, keys = case["batch"], case["tokens"], case["keys"]
        q = normal(batch, tokens, case["heads"], case["dim"])
        k = normal(batch, keys, case["groups"], case["dim"])
        v = normal(batch, keys, case["groups"], case["dim"])
        length = whole(tokens if tokens < keys else (keys + 1) // 2, keys, batch)
        if not case["ragged"]:
            length = torch.full_like(length, keys)
        # the queries of a whole sequence start at its beginning, those of a step or a chunk are its last tokens
        start = length - tokens if tokens < keys else torch.zeros_like(length)
        t = {"q": q, "k": k, "v": v, "start": start, "length": length}
        if case["train"]:
            t["dy"] = normal(batch, tokens, case["heads"], case["dim"], scale=0.1)
        return t
    rows, width, hidden = case["rows"], case["width"], case["hidden"]
    t = {"x": normal(rows, width), "w_gate": normal(width, hidden, scale=width ** -0.5),
         "w_up": normal(width, hidden, scale=width ** -0.5)}
    if case["train"]:
        t["dy"] = normal(rows, hidden, scale=0.1)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _Graph(case, t)
    return {"case": case, **t}


def run(state):
    if own:
        return state.step()
    case = state["case"]
    return {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention, "gated": _plain_gated}[case["op"]](case, state)


# ------------------------------------------------------------------------------------------------------ plain forms


def _plain_norm(case, t):
    s = t["x"] + t["residual"] if case["residual"] else t["x"]
    scale = torch.rsqrt((s * s).mean(-1, keepdim=True) + EPSILON)
    unit = s * scale
    out = {"y": unit * t["weight"]}
    if case["residual"]:
        out["sum"] = s
    if case["train"]:
        g = t["dy"] * t["weight"]
        dx = scale * (g - unit * (g * unit).mean(-1, keepdim=True))
        out["dx"] = dx + t["dsum"] if case["residual"] else dx
        out["dweight"] = (t["dy"] * unit).sum(0)
    return out


def _pair(x, pairs, layout):
    """The first and the second member of each rotated pair, and what is left as it is."""
    if layout == "half":
        return x[..., :pairs], x[..., pairs : 2 * pairs], x[..., 2 * pairs :]
    return x[..., 0 : 2 * pairs : 2], x[..., 1 : 2 * pairs : 2], x[..., 2 * pairs :]


def _unpair(a, b, rest, layout):
    if layout == "half":
        return torch.cat((a, b, rest), -1)
    return torch.cat((torch.stack((a, b), -1).flatten(-2), rest), -1)


def _plain_rotary(case, t):
    # the angle of a far position needs more than 24 bits before it is reduced
    at = t["positions"][:, None] + torch.arange(case["tokens"], device="cuda")
    angle = at[:, :, None, None].double() * t["frequencies"].double()
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    a, b, rest = _pair(t["x"], case["pairs"], case["layout"])
    out = {"y": _unpair(a * c - b * s, b * c + a * s, rest, case["layout"])}
    if case["train"]:
        a, b, rest = _pair(t["dy"], case["pairs"], case["layout"])
        out["dx"] = _unpair(a * c + b * s, b * c - a * s, rest, case["layout"])
    return out


def _plain_attention(case, t):
    batch, tokens, heads, dim = t["q"].shape
    keys, groups = t["k"].shape[1:3]
    scale = dim ** -0.5
    # query heads of a group lie together: [batch, groups, heads of the group x tokens, dim]
    q = t["q"].reshape(batch, tokens, groups, heads // groups, dim).permute(0, 2, 3, 1, 4).reshape(batch, groups, -1, dim)
    k, v = t["k"].permute(0, 2, 1, 3).contiguous(), t["v"].permute(0, 2, 1, 3).contiguous()
    at = (t["start"][:, None] + torch.arange(tokens, device="cuda"))[:, None, None, :, None]
    key = torch.arange(keys, device="cuda")
    length = t["length"][:, None, None, None, None]
    seen = (key <= at) & (key < length) & (at < length)
    if case["window"]:
        seen = seen & ((at - key < case["window"]) | (key < case["sinks"]))
    seen = seen.expand(batch, groups, heads // groups, tokens, keys).reshape(batch, groups, -1, keys)
    score = (torch.matmul(q, k.transpose(-1, -2)) * scale).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(score - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)
    y = torch.matmul(p, v)

    def back(z):
        return z.reshape(batch, groups, heads // groups, tokens, dim).permute(0, 3, 1, 2, 4).reshape(batch, tokens, heads, dim)

    out = {"y": back(y)}
    if case["train"]:
        dy = t["dy"].reshape(batch, tokens, groups, heads // groups, dim).permute(0, 2, 3, 1, 4).reshape(batch, groups, -1, dim)
        dv = torch.matmul(p.transpose(-1, -2), dy)
        ds = p * (torch.matmul(dy, v.transpose(-1, -2)) - (dy * y).sum(-1, keepdim=True)) * scale
        out["dq"] = back(torch.matmul(ds, k))
        out["dk"] = torch.matmul(ds.transpose(-1, -2), q).permute(0, 2, 1, 3)
        out["dv"] = dv.permute(0, 2, 1, 3)
    return out


def _activation(name, g):
    """The activation's value and its derivative."""
    if name == "relu":
        return g.clamp_min(0.0), (g > 0.0).to(g.dtype)
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-g))
    if name == "sigmoid":
        return s, s * (1.0 - s)
    return g * s, s * (1.0 + g * (1.0 - s))


def _plain_gated(case, t):
    g, u = torch.matmul(t["x"], t["w_gate"]), torch.matmul(t["x"], t["w_up"])
    a, da = _activation(case["activation"], g)
    out = {"y": a * u}
    if case["train"]:
        dg, du = t["dy"] * u * da, t["dy"] * a
        out["dx"] = torch.matmul(dg, t["w_gate"].t()) + torch.matmul(du, t["w_up"].t())
        out["dw_gate"] = torch.matmul(t["x"].t(), dg)
        out["dw_up"] = torch.matmul(t["x"].t(), du)
    return out


# --------------------------------------------------------------------------------------------- the framework's form

_backend = None


class _Window:
    """A parameter's device memory as an array that torch can look at without a copy."""

    def __init__(self, pointer, shape):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (pointer, False), "version": 2}


class _Graph:
    """A case as a user of the framework holds it: parameters with the inputs' values, a graph, and the parameters
    that the graph writes."""

    def __init__(self, case, t):
        global _backend
        from descent_amd import Environment
        from descent_amd.hip_backend import HipBackend

        if _backend is None:
            _backend = HipBackend()
        self.env = env = Environment(_backend)
        self.inputs, self.outputs, self.seen = {}, {}, {}
        for name, value in t.items():
            p = self.inputs[name] = env.static_parameter(tuple(value.shape), name)
            if value.dtype == torch.int64:
                env.write_parameter(p, value.cpu().numpy().astype("uint32"))
            else:
                env.writer(p).zero_fill()
                env.sync()
                self._look(p).copy_(value)
        torch.cuda.synchronize()
        self.graph = env.build_graph(lambda scope: self._build(case, scope))
        env.prepare(self.graph)

    def _build(self, case, scope):
        def dual(name):
            return scope.parameter(self.inputs[name])

        def value(name):
            return scope.parameter_value(self.inputs[name])

        def whole(name):
            return value(name).to_u32_bits()

        def keep(name, array):
            p = self.outputs[name] = self.env.static_parameter(tuple(array.shape), name)
            scope.write_parameter_value(p, array)

        op, train = case["op"], case["train"]
        if op == "norm":
            total = None
            if case["residual"]:
                y, total = dual("x").add_rms_norm(dual("residual"), dual("weight"), EPSILON)
                keep("sum", total.value())
            else:
                y = dual("x").rms_norm(dual("weight"), EPSILON)
        elif op == "rotary":
            y = dual("x").rotary(value("frequencies"), whole("positions"), layout=case["layout"])
        elif op == "attention":
            y = dual("q").attention(dual("k"), dual("v"), window=case["window"] or None, sinks=case["sinks"],
                                    start=whole("start"), length=whole("length"))
        else:
            y = dual("x").gated_dense(dual("w_gate"), dual("w_up"), activation=case["activation"])
        keep("y", y.value())
        if train:
            y.loss_grad().accumulate(value("dy"))
            if op == "norm" and case["residual"]:
                total.loss_grad().accumulate(value("dsum"))
            wanted = {"norm": ["x", "weight"], "rotary": ["x"], "attention": ["q", "k", "v"], "gated": ["x", "w_gate", "w_up"]}[op]
            grads = {name: dual(name).loss_grad() for name in wanted}
            for name, grad in grads.items():
                keep("d" + name, grad)

    def _look(self, parameter):
        at = _backend.device_ptr(parameter.buffer)
        view = self.seen.get((at, parameter.name))
        if view is None:
            view = self.seen[at, parameter.name] = torch.as_tensor(_Window(at, parameter.shape), device="cuda")
        return view

    def step(self):
        self.env.run(self.graph, 0)
        return {name: self._look(p) for name, p in self.outputs.items()}

    def __del__(self):
        for p in list(self.inputs.values()) + list(self.outputs.values()):
            if p.buffer is not None:
                _backend.free(p.buffer)
                p.buffer = None


# ------------------------------------------------------------------------------------------------------------- work


def _lengths(case):
    """Sequence lengths spread as the inputs' are."""
    tokens, keys = case["tokens"], case["keys"]
    if not case["ragged"]:
        return [keys]
    low = tokens if tokens < keys else (keys + 1) // 2
    return [low + (keys - low) * i // 8 for i in range(9)]


def _mean_seen(case):
    """Of one sequence and head, on the average: query-key pairs that the mask leaves, query rows that are no padding,
    and keys that some query sees."""
    tokens, keys, window, sinks = case["tokens"], case["keys"], case["window"] or case["keys"], case["sinks"]
    lengths = _lengths(case)
    first = [n - tokens if tokens < keys else 0 for n in lengths]
    pairs = sum(min(at + 1, window) + max(0, min(sinks, at + 1 - window)) for n, a in zip(lengths, first) for at in range(a, n))
    reach = sum(n if a < window else n - a - 1 + window + min(sinks, a + 1 - window) for n, a in zip(lengths, first))
    rows = sum(n - a for n, a in zip(lengths, first))
    return pairs / len(lengths), rows / len(lengths), reach / len(lengths)


def work(case):
    op, train = case["op"], case["train"]
    if op == "norm":
        cells = case["rows"] * case["width"]
        arrays = 2 + (2 if case["residual"] else 0)  # x, y, and the residual and the sum
        if train:
            arrays += 2 + (1 if case["residual"] else 0)  # dy, dx, and the sum's gradient
        return {"bytes": 4.0 * (arrays * cells + case["width"] * (2 if train else 1)), "flops": 0.0}
    if op == "rotary":
        cells = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 4.0 * cells * (4 if train else 2), "flops": 0.0}
    if op == "attention":
        pairs, rows, reach = _mean_seen(case)
        each = case["batch"] * case["dim"]
        whole = case["batch"] * case["tokens"] * case["heads"] * case["dim"]  # outputs have a row for padding too
        read = each * (case["heads"] * rows * (2 if train else 1) + 2 * case["groups"] * reach)
        written = whole * (2 if train else 1) + (2 * each * case["groups"] * case["keys"] if train else 0)
        products = 7 if train else 2  # q k and p v; then again q k, dy v, and those of dq, dk, dv
        return {"bytes": 4.0 * (read + written), "flops": 2.0 * products * each * case["heads"] * pairs}
    rows, width, hidden = case["rows"], case["width"], case["hidden"]
    cells = rows * width + 2 * width * hidden + rows * hidden
    return {"bytes": 4.0 * cells * (2 if train else 1), "flops": (12.0 if train else 4.0) * rows * width * hidden}


# ------------------------------------------------------------------------------------------------------------ exact


def exact(case, seed):
    """The definitions in 64 bits; gradients by differentiating them."""
    t = {name: value.double() if value.is_floating_point() else value for name, value in _inputs(case, seed).items()}
    leaves = {"norm": ["x", "weight"], "rotary": ["x"], "attention": ["q", "k", "v"], "gated": ["x", "w_gate", "w_up"]}[case["op"]]
    if case["train"]:
        for name in leaves:
            t[name].requires_grad_(True)
    extra = None
    if case["op"] == "norm":
        s = t["x"] + t["residual"] if case["residual"] else t["x"]
        y = s / torch.sqrt((s.pow(2).sum(-1) / case["width"] + EPSILON)).unsqueeze(-1) * t["weight"]
        extra = s if case["residual"] else None
    elif case["op"] == "rotary":
        pairs, dim = case["pairs"], case["dim"]
        steps = torch.arange(case["tokens"], device="cuda", dtype=torch.float64)
        phase = (t["positions"].double()[:, None] + steps)[..., None] * t["frequencies"]
        turn = torch.polar(torch.ones_like(phase), phase)[:, :, None, :]
        first = torch.arange(pairs, device="cuda") * (1 if case["layout"] == "half" else 2)
        second = first + (pairs if case["layout"] == "half" else 1)
        z = torch.complex(t["x"][..., first], t["x"][..., second]) * turn
        order = torch.cat((first, second, torch.arange(2 * pairs, dim, device="cuda")))
        y = torch.cat((z.real, z.imag, t["x"][..., 2 * pairs :]), -1)[..., torch.argsort(order)]
    elif case["op"] == "attention":
        heads_each = case["heads"] // case["groups"]
        k = t["k"].repeat_interleave(heads_each, 2).permute(0, 2, 3, 1)
        v = t["v"].repeat_interleave(heads_each, 2).permute(0, 2, 1, 3)
        row = t["start"].reshape(-1, 1, 1, 1) + torch.arange(case["tokens"], device="cuda").reshape(1, 1, -1, 1)
        col = torch.arange(case["keys"], device="cuda").reshape(1, 1, 1, -1)
        hidden = (col > row) | (torch.maximum(row, col) >= t["length"].reshape(-1, 1, 1, 1))
        if case["window"]:
            hidden = hidden | ((row >= col + case["window"]) & (col >= case["sinks"]))
        score = torch.matmul(t["q"].permute(0, 2, 1, 3), k) / math.sqrt(case["dim"])
        score = score.masked_fill(hidden, -math.inf)
        blank = hidden.all(-1, keepdim=True)
        weight = torch.softmax(score.masked_fill(blank, 0.0), -1).masked_fill(blank, 0.0)
        y = torch.matmul(weight, v).permute(0, 2, 1, 3)
    else:
        g, u = t["x"] @ t["w_gate"], t["x"] @ t["w_up"]
        if case["activation"] == "gelu":
            a = g * torch.special.ndtr(g)
        else:
            a = {"silu": lambda: g * torch.sigmoid(g), "relu": lambda: torch.relu(g), "sigmoid": lambda: torch.sigmoid(g)}[case["activation"]]()
        y = a * u
    out = {"y": y.detach()}
    if extra is not None:
        out["sum"] = extra.detach()
    if case["train"]:
        through = (y * t["dy"]).sum()
        if extra is not None:
            through = through + (extra * t["dsum"]).sum()
        grads = torch.autograd.grad(through, [t[name] for name in leaves])
        out.update({"d" + name: g for name, g in zip(leaves, grads)})
    return out
