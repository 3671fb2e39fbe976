"""The sequence-model operators' definitions in 64 bits, as plain numpy.  TEST INFRASTRUCTURE ONLY.

`evaluate(kernel, arrays)` computes what an `OperatorKernel` writes, from the kernel's own inputs through its views;
the functions below it are the formulas, and each gradient is written from the formula (tests compare them with
differences of the forward functions).  Masked entries take no part whatever they hold.
"""
from __future__ import annotations

import math

import numpy as np

from descent_amd.operators import ACTIVATIONS, DUAL_BOTH, DUAL_GATED


def through(view, flat):
    """The array that a view reads (no clamping, as operators require)."""
    strides = view.input_shape.strides()
    base = sum(o * s for o, s in zip(view.input_offsets, strides))
    steps = [0 if axis < 0 else strides[axis] * step for axis, step in view.mapping]
    return np.lib.stride_tricks.as_strided(flat[base:], tuple(view.output_shape), [4 * s for s in steps], writeable=False)


def rms_norm(x, weight, residual, epsilon):
    s = x if residual is None else x + residual
    rho = 1.0 / np.sqrt((s * s).mean(-1) + epsilon)
    return s * rho[..., None] * weight, s, rho


def rms_norm_grad(s, rho, weight, dy, ds_in):
    unit = s * rho[..., None]
    g = dy * weight
    ds = rho[..., None] * (g - unit * (g * unit).mean(-1, keepdims=True))
    return ds if ds_in is None else ds + ds_in, dy * unit


def rotary(x, frequencies, positions, layout, magnitude, inverse):
    pairs = frequencies.shape[0]
    b, t, h, _ = x.shape
    if positions is None:
        place = np.broadcast_to(np.arange(t, dtype=np.float64), (b, t))
    elif positions.ndim == 1:
        place = positions[:, None].astype(np.float64) + np.arange(t)
    else:
        place = positions.astype(np.float64)
    angle = (place[..., None] * frequencies.astype(np.float64))[:, :, None, :] * (-1.0 if inverse else 1.0)
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    first = np.arange(pairs) if layout == 0 else 2 * np.arange(pairs)
    second = first + (pairs if layout == 0 else 1)
    y = x.copy()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def visible(tokens, keys, window, sinks, start, length):
    """[tokens, keys] of one sequence."""
    place = (int(start) + np.arange(tokens, dtype=np.int64))[:, None]
    key = np.arange(keys, dtype=np.int64)[None, :]
    sees = (key <= place) & (key < int(length)) & (place < int(length))
    return sees & ((place - key < window) | (key < sinks)) if window else sees


def _each_head(q, k, start, length):
    b, t, h, _ = q.shape
    keys, groups = k.shape[1:3]
    for i in range(b):
        first = int(start[i]) if start is not None else keys - t
        count = min(int(length[i]), keys) if length is not None else keys
        for j in range(h):
            yield i, j, j // (h // groups), first, count


def attention(q, k, v, window, sinks, scale, start=None, length=None):
    b, t, h, d = q.shape
    out, lse = np.zeros_like(q), np.full((b, t, h), -np.inf)
    for i, j, g, first, count in _each_head(q, k, start, length):
        sees = visible(t, k.shape[1], window, sinks, first, count)
        for r in np.nonzero(sees.any(1))[0]:
            at = np.nonzero(sees[r])[0]
            with np.errstate(invalid="ignore"):
                score = k[i, at, g] @ q[i, r, j] * scale
                top = score.max()
                p = np.exp(score - top)
                out[i, r, j] = p @ v[i, at, g] / p.sum()
                lse[i, r, j] = top + math.log(p.sum()) if np.isfinite(p.sum()) else np.nan
    return out, lse


def attention_grad(q, k, v, out, dout, lse, window, sinks, scale, start=None, length=None, pick=None):
    """dq, dk, dv and delta = sum(out * dout).  `pick(sequence, tokens)` limits the pairs that count."""
    b, t, h, d = q.shape
    dq, dk, dv, delta = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v), np.zeros((b, t, h))
    for i, j, g, first, count in _each_head(q, k, start, length):
        sees = visible(t, k.shape[1], window, sinks, first, count)
        if pick is not None:
            sees = sees & pick(i, t)
        for r in np.nonzero(sees.any(1))[0]:
            at = np.nonzero(sees[r])[0]
            with np.errstate(invalid="ignore"):
                p = np.exp(k[i, at, g] @ q[i, r, j] * scale - lse[i, r, j])
                delta[i, r, j] = out[i, r, j] @ dout[i, r, j]
                ds = p * (v[i, at, g] @ dout[i, r, j] - delta[i, r, j]) * scale
                dq[i, r, j] = ds @ k[i, at, g]
                dk[i, at, g] += ds[:, None] * q[i, r, j]
                dv[i, at, g] += p[:, None] * dout[i, r, j]
    return dq, dk, dv, delta


_erf = np.vectorize(math.erf, otypes=[np.float64])
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def activation(name, g):
    """Value and derivative."""
    if name == "relu":
        return np.maximum(g, 0.0), (g > 0.0).astype(np.float64)
    if name == "gelu":
        cdf = 0.5 * _erfc(-g * math.sqrt(0.5))
        return g * cdf, cdf + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    with np.errstate(over="ignore"):
        s = 1.0 / (1.0 + np.exp(-g))
    return (s, s * (1.0 - s)) if name == "sigmoid" else (g * s, s * (1.0 + g * (1.0 - s)))


def append(kernel, rows, start, cache):
    """CacheAppend on the cache's own buffer."""
    rows = through(kernel.inputs[0], rows)
    at = np.ascontiguousarray(through(kernel.inputs[1], start)).view(np.uint32)
    whole = cache[: kernel.shape.element_count()].reshape(tuple(kernel.shape))
    for b in range(rows.shape[0]):
        for t in range(rows.shape[1]):
            if int(at[b]) + t < whole.shape[1]:
                whole[b, int(at[b]) + t] = rows[b, t]


def evaluate(kernel, arrays):
    """The kernel's results, in 64 bits, in the order in which it binds them."""
    spec, ints, floats = kernel.spec, kernel.spec.ints, kernel.spec.floats
    raw = [through(view, a) for view, a in zip(kernel.inputs, arrays)]
    x = [a.astype(np.float64) for a in raw]
    whole = [np.ascontiguousarray(a).view(np.uint32) for a in raw]
    name = spec.name
    if name == "RmsNorm":
        got = rms_norm(x[0], x[1], x[2] if ints[0] else None, float(np.float32(floats[0])))
    elif name == "RmsNormGrad":
        ds, share = rms_norm_grad(x[0], x[1], x[2], x[3], x[4] if ints[0] else None)
        got = ds, np.stack([share[p :: ints[1]].sum(0) for p in range(ints[1])])
    elif name == "Rotary":
        got = (rotary(x[0], raw[1], whole[2] if ints[2] else None, ints[0], float(np.float32(floats[0])), ints[1]),)
    elif name in ("Attention", "AttentionGradQuery", "AttentionGradKeyValue", "AttentionGradSinks"):
        joins = name == "AttentionGradKeyValue" and ints[3] > 0
        places = whole[3 if name == "Attention" else 8 if joins else 6 :]
        start = places[0] if ints[2] & 1 else None
        length = places[-1] if ints[2] & 2 else None
        scale = float(np.float32(floats[0]))
        if name == "Attention":
            out, lse = attention(*x[:3], ints[0], ints[1], scale, start, length)
            if ints[3] > 1:  # the whole answer as the first piece, the others empty: what the join makes of it is the same
                out = np.concatenate([out[None], np.zeros((ints[3] - 1,) + out.shape)])
                lse = np.concatenate([lse[None], np.full((ints[3] - 1,) + lse.shape, -np.inf)])
            got = out, lse
        elif name == "AttentionGradQuery":
            dq, _, _, delta = attention_grad(*x[:6], ints[0], ints[1], scale, start, length)
            got = dq, delta
        else:
            # the output enters through its product with the gradient, which is operand 5
            q, k, v, dout, lse, delta = x[:6]
            square = (dout * dout).sum(-1, keepdims=True)
            out = np.where(square > 0, dout * delta[..., None] / np.where(square > 0, square, 1.0), 0.0)
            if joins or name == "AttentionGradSinks":  # rows at this place or past it belong to the sinks' kernel
                def far(i, t):
                    place = (int(start[i]) if start is not None else k.shape[1] - t) + np.arange(t)
                    return place[:, None] >= np.minimum(np.arange(k.shape[1]) // 64 * 64 + 63, k.shape[1] - 1) + ints[0]

                pick = far if name == "AttentionGradSinks" else lambda i, t: ~far(i, t)
            else:
                pick = None
            _, dk, dv, _ = attention_grad(q, k, v, out, dout, lse, ints[0], ints[1], scale, start, length, pick)
            if name == "AttentionGradSinks":
                sinks = min(ints[1], k.shape[1])
                got = [np.concatenate([a[None, :, :sinks], np.zeros((ints[3] - 1,) + a[:, :sinks].shape)]) for a in (dk / scale, dv)]
            else:
                if joins:
                    sinks = x[6].shape[2]
                    dk[:, :sinks] += x[6].sum(0) * scale
                    dv[:, :sinks] += x[7].sum(0)
                    for i in range(k.shape[0] if length is not None else 0):  # keys past the length get no gradient
                        dk[i, int(length[i]) :] = dv[i, int(length[i]) :] = 0.0
                got = dk, dv
    elif name == "AttentionJoin":
        part, lse = x
        top = lse.max(0)
        safe = np.where(np.isneginf(top), 0.0, top)
        w = np.exp(lse - safe)
        total = w.sum(0)
        out = (part * w[..., None]).sum(0) / np.where(total > 0, total, 1.0)[..., None]
        with np.errstate(divide="ignore"):
            got = out, safe + np.log(total)
    elif name == "DualMatMul":
        if ints[0] == DUAL_GATED:
            g, u = x[0] @ x[1], x[0] @ x[2]
            got = activation(ACTIVATIONS[ints[1]], g)[0] * u, g, u
        elif ints[0] == DUAL_BOTH:
            got = x[0] @ x[1], x[0] @ x[2]
        else:
            got = (x[0] @ x[2] + x[1] @ x[3],)
        if ints[2] > 1:  # the whole sum as the first piece: what is made of the pieces is their sum
            got = [np.concatenate([a[None], np.zeros((ints[2] - 1,) + a.shape)]) for a in got]
    else:
        assert name == "GatedGrad"
        a, slope = activation(ACTIVATIONS[ints[0]], x[0])
        got = x[2] * x[1] * slope, x[2] * a
    return [got[i] for i in kernel.results]
