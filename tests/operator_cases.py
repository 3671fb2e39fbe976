"""Shared by the CPU and GPU tests of the sequence-model operators: kernel descriptors with inputs, and how far a
32-bit result may be from the 64-bit definition.

U = 2^-24 is the largest relative error of one 32-bit rounding.  A sum of n products in any order, each step rounded, is
off by at most n U times the sum of the products' magnitudes (to first order); the bounds below count the roundings of
the kernels that way and add nothing for luck.
"""
import numpy as np

from descent_amd.operators import ACTIVATIONS, DUAL_BOTH, DUAL_GATED, DUAL_SUM, OperatorKernel, OperatorSpec, norm_partials
from descent_amd.shape import Shape, View
from oracle import operators as ref

U = 2.0 ** -24


def kernel(spec, arrays, views=None, results=None):
    views = views or [Shape(a.shape).identity_view() for a in arrays]
    k = OperatorKernel(spec, tuple(views), ())
    return OperatorKernel(spec, tuple(views), tuple(results if results is not None else range(len(k.result_shapes()))))


def flat(arrays):
    return [np.ascontiguousarray(a if a.dtype == np.float32 else a.view(np.float32)).reshape(-1) for a in arrays]


def normal(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float32)


# ---- norm ---------------------------------------------------------------------------------------------------------
# (rows, width, residual)
NORMS = [(1, 1, False), (1, 64, True), (3, 5, True), (7, 100, False), (5, 1000, True), (33, 2048, True), (2, 4100, False), (3, 8192, True),
         (600, 33, True), (1030, 260, False), (2, 40000, True), (1, 131075, False)]


def norm_case(rows, width, residual, rng):
    x, w = normal(rng, rows, width), 1.0 + normal(rng, width, scale=0.2)
    arrays = [x, w.astype(np.float32)] + ([normal(rng, rows, width, scale=3.0)] if residual else [])
    return kernel(OperatorSpec("RmsNorm", (int(residual),), (1e-6,)), arrays), arrays


def norm_bounds(k, arrays, want):
    """A thread adds at most max(32, width / 1024) squares, then 6 exchanges and 16 waves; half of that error reaches the
    root; the root, the division, the mean and the three products round once each, the sum before them twice as much
    because it is squared."""
    width = arrays[0].shape[1]
    steps = max(32, width / 1024) + 22
    rel = (steps / 2 + 10) * U
    return [rel * np.abs(want[0]), U * np.abs(want[1]), rel * np.abs(want[2])]


def norm_grad_case(rows, width, residual, rng):
    s, w = normal(rng, rows, width), (1.0 + normal(rng, width, scale=0.2)).astype(np.float32)
    rho = (1.0 / np.sqrt((s.astype(np.float64) ** 2).mean(-1) + 1e-6)).astype(np.float32)
    arrays = [s, rho, w, normal(rng, rows, width, scale=0.5)] + ([normal(rng, rows, width, scale=0.5)] if residual else [])
    return kernel(OperatorSpec("RmsNormGrad", (int(residual), norm_partials(rows))), arrays), arrays


def norm_grad_bounds(k, arrays, want):
    s, rho, w, dy = (a.astype(np.float64) for a in arrays[:4])
    rows, width = s.shape
    steps = max(32, width / 1024) + 22
    size = np.abs(rho[:, None] * dy * w) + np.abs(s) * rho[:, None] ** 3 * np.abs(s * dy * w).mean(-1, keepdims=True)
    add = np.abs(arrays[4].astype(np.float64)) if len(arrays) > 4 else 0.0
    share = np.abs(dy * s * rho[:, None])
    p = k.spec.ints[1]
    return [(steps + 12) * U * size + 2 * U * add, np.stack([(len(share[i::p]) + 4) * U * share[i::p].sum(0) for i in range(p)])]


# ---- rotary -------------------------------------------------------------------------------------------------------
# (batch, tokens, heads, dim, pairs, layout, rank of positions, far, magnitude, inverse)
ROTARIES = [(1, 1, 1, 2, 1, 0, 0, 0, 1.0, 0), (2, 1, 32, 128, 64, 0, 1, 1000000, 1.0, 0), (1, 5, 3, 64, 32, 1, 1, 40, 1.0, 1),
            (2, 7, 4, 80, 20, 1, 2, 100000, 1.25, 0), (2, 7, 4, 80, 20, 0, 2, 4000000000, 0.5, 1), (1, 3, 2, 7, 3, 0, 0, 0, 1.0, 0),
            (1, 3, 2, 7, 3, 1, 1, 9, 1.0, 1), (3, 33, 1, 256, 128, 0, 1, 8000, 1.0, 0),
            (1, 700, 5, 24, 6, 1, 0, 0, 1.0, 0)]


def rotary_case(batch, tokens, heads, dim, pairs, layout, rank, far, magnitude, inverse, rng):
    x = normal(rng, batch, tokens, heads, dim)
    table = (10000.0 ** (-np.arange(max(pairs, 1)) / max(pairs, 1))).astype(np.float32)
    arrays = [x, table]
    if rank:
        shape = (batch,) if rank == 1 else (batch, tokens)
        arrays.append(rng.integers(far // 2, far + 1, shape).astype(np.uint32))
    return kernel(OperatorSpec("Rotary", (layout, inverse, rank), (magnitude,)), arrays), arrays


def rotary_bounds(k, arrays, want):
    """The angle's rounding to 32 bits is off by at most pi 2^-24 radians, the 64-bit reduction before it by less than
    10^-6 of that; sine and cosine by 10^-7 (stated at their polynomials) and three roundings of the products and sum."""
    m, pairs = abs(np.float32(k.spec.floats[0])), arrays[1].shape[0]
    x = np.abs(arrays[0].astype(np.float64))
    first = np.arange(pairs) if k.spec.ints[0] == 0 else 2 * np.arange(pairs)
    second = first + (pairs if k.spec.ints[0] == 0 else 1)
    bound = np.zeros_like(x)
    size = x[..., first] + x[..., second]
    bound[..., first] = bound[..., second] = size * m * (np.pi * U + 1e-7 + 4 * U)
    return [bound]


# ---- attention ----------------------------------------------------------------------------------------------------
# (batch, tokens, keys, heads, groups, dim, window, sinks, places): places "none", "start", "length", "both"
ATTENTIONS = [
    (1, 1, 1, 1, 1, 1, 0, 0, "none"), (2, 5, 5, 2, 1, 16, 0, 0, "none"), (1, 70, 70, 2, 2, 64, 0, 0, "none"),
    (2, 130, 130, 6, 2, 64, 40, 0, "length"), (1, 200, 200, 4, 1, 32, 64, 5, "none"), (2, 65, 129, 3, 3, 48, 33, 70, "both"),
    (1, 100, 100, 2, 1, 128, 1, 0, "none"), (1, 90, 90, 2, 1, 128, 1, 3, "length"), (2, 67, 67, 2, 2, 80, 20, 2, "both"),
    (1, 70, 70, 1, 1, 200, 30, 1, "none"), (1, 66, 66, 2, 1, 256, 0, 0, "length"), (1, 90, 90, 2, 1, 30, 17, 4, "length"),
    (3, 1, 40, 8, 2, 64, 0, 0, "both"), (2, 1, 300, 4, 4, 128, 100, 4, "both"), (1, 1, 2000, 4, 1, 64, 0, 0, "none"),
    (1, 1, 1500, 2, 1, 128, 700, 9, "both"), (2, 3, 600, 4, 2, 40, 290, 20, "both"), (1, 17, 600, 3, 1, 96, 0, 0, "start"),
    (1, 1, 700, 1, 1, 256, 0, 0, "length"), (2, 4, 9, 2, 1, 31, 0, 0, "start"), (1, 300, 300, 1, 1, 64, 100, 130, "none"),
]


def attention_places(batch, tokens, keys, places, rng):
    start = length = None
    if places in ("length", "both"):
        length = rng.integers(0, keys + 1, batch).astype(np.uint32)
        length[0] = keys if batch > 1 else max(1, keys - 3)
        if batch > 1:
            length[-1] = min(length[-1], tokens // 2)  # a short one: rows of padding, or none at all
    if places in ("start", "both"):
        start = np.full(batch, max(0, keys - tokens), np.uint32)
        start[-1] = max(0, (keys - tokens) // 2)
    return start, length


def attention_case(batch, tokens, keys, heads, groups, dim, window, sinks, places, rng, splits=1, results=None):
    q, k, v = normal(rng, batch, tokens, heads, dim), normal(rng, batch, keys, groups, dim), normal(rng, batch, keys, groups, dim)
    start, length = attention_places(batch, tokens, keys, places, rng)
    arrays = [q, k, v] + [a for a in (start, length) if a is not None]
    has = (start is not None) | (length is not None) << 1
    return kernel(OperatorSpec("Attention", (window, sinks if window else 0, int(has), splits), (float(dim) ** -0.5,)), arrays, results=results), arrays


def _pairs(k, arrays, places_at):
    """Per (sequence, head): what the mask leaves, and the operands."""
    ints = k.spec.ints
    q, key = arrays[0].astype(np.float64), arrays[1].astype(np.float64)
    places = arrays[places_at:]
    start = places[0] if ints[2] & 1 else None
    length = places[-1] if ints[2] & 2 else None
    for i, j, g, first, count in ref._each_head(q, key, start, length):
        yield i, j, g, ref.visible(q.shape[1], key.shape[1], ints[0], ints[1], first, count)


def attention_bounds(k, arrays, want):
    """A score sums dim products (dim + 3 roundings with the scale's); an error e of a score is a relative error e of its
    probability, and of the denominator at most the largest; exponentials are good to 2 U and see their argument rounded
    by half of U per unit, which the score's bound covers since |score - top| <= 2 max |score|."""
    scale = abs(k.spec.floats[0])
    q, key, v = (np.abs(a.astype(np.float64)) for a in arrays[:3])
    out, lse = np.zeros(want[0].shape), np.zeros(want[1].shape)
    dim = q.shape[-1]
    for i, j, g, sees in _pairs(k, arrays, 3):
        size = scale * q[i, :, j] @ key[i, :, g].T
        worst = np.where(sees, size, 0.0).max(1, initial=0.0) * (dim + 8) * U
        count = sees.sum(1)
        real = scale * arrays[0][i, :, j].astype(np.float64) @ arrays[1][i, :, g].astype(np.float64).T
        real = np.where(sees, real, -np.inf)
        p = np.where(sees, np.exp(real - np.where(sees.any(1), real.max(1), 0.0)[:, None]), 0.0)
        p = p / np.maximum(p.sum(1), 1e-300)[:, None]
        out[i, :, j] = (p @ v[i, :, g]) * (2 * worst + (2 * count + 20) * U)[:, None]
        lse[i, :, j] = np.where(sees.any(1), worst + (count + 12) * U + 4 * U * np.abs(np.where(np.isfinite(want[1][i, :, j]), want[1][i, :, j], 0.0)), 0.0)
    return [out, lse]


def attention_grad_cases(batch, tokens, keys, heads, groups, dim, window, sinks, places, rng, pieces=0):
    """The gradient kernels (with `pieces` those that share the sinks' rows, too), on the 64-bit forward results rounded to 32."""
    k, arrays = attention_case(batch, tokens, keys, heads, groups, dim, window, sinks, places, rng)
    out, lse = (a.astype(np.float32) for a in ref.evaluate(k, flat(arrays)))
    dout = normal(rng, *out.shape, scale=0.5)
    ints, floats, tail = k.spec.ints[:3], k.spec.floats, arrays[3:]
    delta = (out.astype(np.float64) * dout).sum(-1).astype(np.float32)
    by_query = arrays[:3] + [out, dout, lse] + tail
    by_key = arrays[:3] + [dout, lse, delta] + tail
    cases = [(kernel(OperatorSpec("AttentionGradQuery", ints, floats), by_query), by_query),
             (kernel(OperatorSpec("AttentionGradKeyValue", ints + (0,), floats), by_key), by_key)]
    if pieces:
        far = kernel(OperatorSpec("AttentionGradSinks", ints + (pieces,), floats), by_key)
        some = [normal(rng, *s) for s in far.result_shapes()]
        joined = by_key[:6] + some + tail
        cases += [(far, by_key), (kernel(OperatorSpec("AttentionGradKeyValue", ints + (pieces,), floats), joined), joined)]
    return cases


def attention_grad_bounds(k, arrays, want):
    """As above; a probability is formed against the given denominator (one more score rounding), ds = p (do.v - delta)
    carries p's relative error and the two sums' own, and the last product sums as many terms as there are pairs."""
    scale = abs(k.spec.floats[0])
    by_query = k.spec.name == "AttentionGradQuery"
    q, key, v = (a.astype(np.float64) for a in arrays[:3])
    dout, lse = (arrays[i].astype(np.float64) for i in ((4, 5) if by_query else (3, 4)))
    out = arrays[3].astype(np.float64) if by_query else None
    heads, groups, dim = q.shape[2], key.shape[2], q.shape[3]
    dq, delta, dk, dv = np.zeros(q.shape), np.zeros(lse.shape), np.zeros(key.shape), np.zeros(key.shape)
    joins = not by_query and k.spec.name == "AttentionGradKeyValue" and k.spec.ints[3]
    for i, j, g, sees in _pairs(k, arrays, 8 if joins else 6):
        real = scale * q[i, :, j] @ key[i, :, g].T
        size = scale * np.abs(q[i, :, j]) @ np.abs(key[i, :, g]).T
        row = np.where(np.isfinite(lse[i, :, j]), lse[i, :, j], 0.0)
        p = np.where(sees, np.exp(np.where(sees, real, 0.0) - row[:, None]), 0.0)
        off = (size * (dim + 8) + 4 * np.abs(row)[:, None] + 12) * U
        dov, dov_size = dout[i, :, j] @ v[i, :, g].T, np.abs(dout[i, :, j]) @ np.abs(v[i, :, g]).T
        if by_query:
            own, own_size = (out[i, :, j] * dout[i, :, j]).sum(-1), np.abs(out[i, :, j] * dout[i, :, j]).sum(-1)
        else:
            own = arrays[5].astype(np.float64)[i, :, j]
            own_size = np.abs(own)
        ds = p * np.abs(dov - own[:, None])
        ds_off = ds * off + p * (dim + 4) * U * (dov_size + own_size[:, None])
        count = sees.sum() + 4
        dq[i, :, j] = scale * ((ds_off + ds * (sees.sum(1)[:, None] + 4) * U) @ np.abs(key[i, :, g]))
        delta[i, :, j] = (dim + 4) * U * own_size
        rows = heads // groups * sees.sum(0)[:, None] + 4
        dk[i, :, g] += scale * (ds_off.T @ np.abs(q[i, :, j]) + rows * U * (ds.T @ np.abs(q[i, :, j])))
        dv[i, :, g] += (p * off).T @ np.abs(dout[i, :, j]) + rows * U * (p.T @ np.abs(dout[i, :, j]))
    if k.spec.name == "AttentionGradSinks":  # any piece may hold any of the rows
        sinks = want[0].shape[2]
        return [np.broadcast_to(a[None, :, :sinks], want[0].shape) for a in (dk / scale, dv)]
    if joins:
        sinks, n = arrays[6].shape[2], arrays[6].shape[0] + 2
        dk[:, :sinks] += scale * n * U * np.abs(arrays[6].astype(np.float64)).sum(0)
        dv[:, :sinks] += n * U * np.abs(arrays[7].astype(np.float64)).sum(0)
    return [dq, delta] if by_query else [dk, dv]


def join_case(splits, batch, tokens, heads, dim, rng):
    part = normal(rng, splits, batch, tokens, heads, dim)
    lse = normal(rng, splits, batch, tokens, heads, scale=4.0)
    lse[rng.random(lse.shape) < 0.3] = -np.inf
    lse[:, 0, 0, 0] = -np.inf
    return kernel(OperatorSpec("AttentionJoin"), [part, lse]), [part, lse]


def join_bounds(k, arrays, want):
    part, lse = (a.astype(np.float64) for a in arrays)
    top = np.where(np.isneginf(lse.max(0)), 0.0, lse.max(0))
    w = np.exp(lse - top)
    size = (np.abs(part) * w[..., None]).sum(0) / np.maximum(w.sum(0), 1e-300)[..., None]
    n = part.shape[0]
    arg = np.abs(np.where(np.isfinite(lse), lse - top, 0.0)).max(0) + 4  # the exponent's own rounding, per unit
    return [size * ((2 * n + 8 + 4 * arg) * U)[..., None], (n + 8 + 4 * arg + 4 * np.abs(top)) * U]


# ---- dual product -------------------------------------------------------------------------------------------------
# (mode, rows, columns, k, activation)
DUALS = [(DUAL_GATED, 1, 1, 1, 0), (DUAL_GATED, 1, 4096, 200, 0), (DUAL_GATED, 3, 70, 33, 1), (DUAL_GATED, 8, 129, 260, 2), (DUAL_GATED, 9, 40, 17, 3),
         (DUAL_GATED, 31, 100, 64, 0), (DUAL_GATED, 130, 66, 97, 1), (DUAL_GATED, 257, 700, 32, 2), (DUAL_GATED, 2100, 1030, 40, 0),
         (DUAL_SUM, 1, 1, 1, 0), (DUAL_SUM, 65, 129, 70, 0), (DUAL_SUM, 5, 300, 100, 0), (DUAL_SUM, 2050, 1100, 36, 0), (DUAL_SUM, 300, 700, 100, 0),
         (DUAL_BOTH, 1, 1, 1, 0), (DUAL_BOTH, 70, 129, 35, 0), (DUAL_BOTH, 33, 64, 200, 0), (DUAL_BOTH, 1030, 1100, 36, 0), (DUAL_BOTH, 400, 300, 70, 0)]


def dual_case(mode, rows, columns, k, act, rng, transposed=(), splits=1):
    """`transposed`: operands that are read through a transposing view."""
    left = 2 if mode == DUAL_SUM else 1
    shapes = [(rows, k)] * left + [(k, columns)] * 2
    arrays, views = [], []
    for i, s in enumerate(shapes):
        if i in transposed:
            arrays.append(normal(rng, s[1], s[0]))
            views.append(Shape((s[1], s[0])).identity_view().transposed())
        else:
            arrays.append(normal(rng, *s))
            views.append(Shape(s).identity_view())
    return kernel(OperatorSpec("DualMatMul", (mode, act, splits)), arrays, views), arrays


def dual_bounds(k, arrays, want):
    """Each of the six products of parts is added with one rounding: 6 k of them, each at most U times the sum of the
    products' magnitudes, and the products left out are below 4 U of them together."""
    x = [np.abs(ref.through(v, a).astype(np.float64)) for v, a in zip(k.inputs, flat(arrays))]
    mode, act, _ = k.spec.ints
    n = x[0].shape[1]
    step = (6 * n + 4) * U
    if mode == DUAL_BOTH:
        return [step * (x[0] @ x[1]), step * (x[0] @ x[2])]
    if mode == DUAL_SUM:
        return [2 * step * (x[0] @ x[2] + x[1] @ x[3])]
    eg, eu = step * (x[0] @ x[1]), step * (x[0] @ x[2])
    value, _ = ref.activation(ACTIVATIONS[act], want[1])
    slope = 1.13  # no activation is steeper
    return [slope * eg * (np.abs(want[2]) + eu) + np.abs(value) * eu + 16 * U * (np.abs(want[0]) + U), eg, eu]


def gated_grad_case(count, act, rng):
    arrays = [normal(rng, count[0], count[1], scale=3.0), normal(rng, *count), normal(rng, *count)]
    arrays[0].flat[0] = 100.0
    if arrays[0].size > 1:
        arrays[0].flat[1] = -100.0
    return kernel(OperatorSpec("GatedGrad", (act,)), arrays), arrays


def gated_grad_bounds(k, arrays, want):
    """Logistic function to 4 U, 1 - s to U of one, the error function's complement to 8 U; three products."""
    g, u, dh = (np.abs(a.astype(np.float64)) for a in arrays)
    return [dh * u * (1.0 + g) * 24 * U, dh * (1.0 + g) * 24 * U]


GRAD_COUNTS = [(1, 1), (3, 7), (64, 64), (33, 130)]
