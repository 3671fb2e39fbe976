"""CPU: the sequence-model operators' definitions against differences, the graphs they make, what is refused, and that
every kernel compiles."""
import ctypes as C
import math

import numpy as np
import pytest

import operator_cases as cases
from descent_amd import Environment, SelfAttention, TransformerBlock, _abi, hip_backend, rotary_frequencies
from descent_amd.operators import DUAL_BOTH, DUAL_GATED, DUAL_SUM, OperatorKernel, OperatorSpec, attention_splits
from descent_amd.shape import Shape, View
from oracle import operators as ref
from oracle.cpu_backend import CpuBackend


def _env():
    return Environment(CpuBackend())


# ------------------------------------------------------------------------------------------------- the definitions


def _differences(f, x, step=1e-6):
    """Gradient of the scalar f at x by central differences."""
    out = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        keep = x[i]
        x[i] = keep + step
        up = f()
        x[i] = keep - step
        down = f()
        x[i] = keep
        out[i] = (up - down) / (2 * step)
    return out


def _close(a, b):
    # central differences of step h are off by h^2 and by the 64-bit roundings over h
    assert np.allclose(a, b, rtol=1e-6, atol=1e-7), np.abs(a - b).max()


def test_norm_definition():
    rng = np.random.default_rng(0)
    x, r, w, dy, ds = (rng.standard_normal(s) for s in ((3, 7), (3, 7), (7,), (3, 7), (3, 7)))

    def loss():
        y, s, _ = ref.rms_norm(x, w, r, 1e-3)
        return (y * dy).sum() + (s * ds).sum()

    _, s, rho = ref.rms_norm(x, w, r, 1e-3)
    dx, share = ref.rms_norm_grad(s, rho, w, dy, ds)
    _close(dx, _differences(loss, x))
    _close(dx, _differences(loss, r))
    _close(share.sum(0), _differences(loss, w))


@pytest.mark.parametrize("layout", [0, 1])
def test_rotary_definition(layout):
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((2, 3, 2, 10)), rng.standard_normal((2, 3, 2, 10))
    table = np.array([1.0, 0.3, 0.01], np.float32)
    start = np.array([4, 1000], np.uint32)
    y = ref.rotary(x, table, start, layout, 1.5, 0)
    assert np.array_equal(y[..., 6:], x[..., 6:])
    # the inverse turns the gradient back
    _close(ref.rotary(dy, table, start, layout, 1.5, 1)[..., :6], _differences(lambda: (ref.rotary(x, table, start, layout, 1.5, 0) * dy).sum(), x)[..., :6])
    _close(ref.rotary(ref.rotary(x, table, start, layout, 1.0, 0), table, start, layout, 1.0, 1), x)
    # scores depend on the distance of two positions only
    q, k = rng.standard_normal((1, 1, 1, 6)), rng.standard_normal((1, 1, 1, 6))
    at = lambda a, p: ref.rotary(a, table, np.array([p], np.uint32), layout, 1.0, 0).ravel()  # noqa: E731
    assert abs(at(q, 9) @ at(k, 4) - at(q, 1009) @ at(k, 1004)) < 1e-9


@pytest.mark.parametrize("window,sinks,places", [(0, 0, "none"), (3, 0, "length"), (2, 2, "both")])
def test_attention_definition(window, sinks, places):
    rng = np.random.default_rng(2)
    q, k, v, do = (rng.standard_normal(s) for s in ((2, 5, 4, 3), (2, 7, 2, 3), (2, 7, 2, 3), (2, 5, 4, 3)))
    start, length = cases.attention_places(2, 5, 7, places, rng)

    def loss():
        return (ref.attention(q, k, v, window, sinks, 0.7, start, length)[0] * do).sum()

    out, lse = ref.attention(q, k, v, window, sinks, 0.7, start, length)
    dq, dk, dv, _ = ref.attention_grad(q, k, v, out, do, lse, window, sinks, 0.7, start, length)
    _close(dq, _differences(loss, q))
    _close(dk, _differences(loss, k))
    _close(dv, _differences(loss, v))
    # against a dense softmax
    for i, j, g, first, count in ref._each_head(q, k, start, length):
        sees = ref.visible(5, 7, window, sinks, first, count)
        s = np.where(sees, 0.7 * q[i, :, j] @ k[i, :, g].T, -1e30)
        p = np.exp(s - s.max(1, keepdims=True)) * sees
        _close(out[i, :, j], p / np.maximum(p.sum(1, keepdims=True), 1e-300) @ v[i, :, g])


@pytest.mark.parametrize("name", ["silu", "gelu", "relu", "sigmoid"])
def test_activation_definitions(name):
    g = np.array([-30.0, -3.0, -0.5, 0.25, 1.0, 4.0, 30.0])
    value, slope = ref.activation(name, g)
    _close(slope, (ref.activation(name, g + 1e-6)[0] - ref.activation(name, g - 1e-6)[0]) / 2e-6)
    want = {"silu": g / (1 + np.exp(-g)), "gelu": g * 0.5 * (1 + ref._erf(g / math.sqrt(2))), "relu": np.maximum(g, 0), "sigmoid": 1 / (1 + np.exp(-g))}[name]
    assert np.allclose(value, want, rtol=1e-12, atol=1e-15)


def test_rotary_tables():
    assert np.allclose(rotary_frequencies(8), 10000.0 ** (-np.arange(4) / 4), rtol=2.0 ** -23)
    assert np.allclose(rotary_frequencies(8, scale=4.0), rotary_frequencies(8) / 4, rtol=2.0 ** -22)
    mixed = rotary_frequencies(64, scale=8.0, original=4096)
    plain = rotary_frequencies(64)
    assert mixed[0] == plain[0] and np.isclose(mixed[-1], plain[-1] / 8, rtol=1e-6) and (np.diff(mixed) < 0).all()
    for bad in ({"dims": 7}, {"dims": 8, "scale": 0.0}, {"dims": 8, "base": -1.0}, {"dims": 8, "slow": 5.0, "fast": 5.0}):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


# -------------------------------------------------------------------------------------------------------- graphs


def _labels(graph):
    return [graph.clusters[c].kernel.label_name().split()[0] for c in graph.clusters_sorted]


def _kernels(graph, name):
    return [graph.clusters[c].kernel for c in graph.clusters_sorted if graph.clusters[c].kernel.label_name().startswith(name + " ")]


def test_results_that_nothing_reads_are_not_written():
    env = _env()
    x, r, w, y = (env.static_parameter(s, n) for n, s in (("x", [4, 6]), ("r", [4, 6]), ("w", [6]), ("y", [4, 6])))
    graph = env.build_graph(lambda s: s.write_parameter_value(y, s.parameter(x).add_rms_norm(s.parameter(r), s.parameter(w))[0].value()))
    assert _labels(graph) == ["RmsNorm"] and _kernels(graph, "RmsNorm")[0].results == (0,)
    q, k = env.static_parameter([1, 5, 2, 4], "q"), env.static_parameter([1, 5, 2, 4], "k")
    o = env.static_parameter([1, 5, 2, 4], "o")
    graph = env.build_graph(lambda s: s.write_parameter_value(o, s.parameter(q).attention(s.parameter(k), s.parameter(k)).value()))
    assert _labels(graph) == ["Attention"] and _kernels(graph, "Attention")[0].results == (0,)


def test_one_result_for_two_parameters_and_a_sum_without_gradient():
    env = _env()
    rng = np.random.default_rng(3)
    data = {n: rng.standard_normal(s).astype(np.float32) for n, s in (("x", (4, 6)), ("r", (4, 6)), ("w", (6,)), ("dy", (4, 6)))}
    p = {n: env.static_parameter_with_data(a.shape, n, a) for n, a in data.items()}
    gx, gr, gw = env.static_parameter([4, 6], "gx"), env.static_parameter([4, 6], "gr"), env.static_parameter([6], "gw")

    def build(s):
        y, _ = s.parameter(p["x"]).add_rms_norm(s.parameter(p["r"]), s.parameter(p["w"]))
        y.loss_grad().accumulate(s.parameter_value(p["dy"]))
        for out, of in ((gx, "x"), (gr, "r"), (gw, "w")):
            s.write_parameter_value(out, s.parameter(p[of]).loss_grad())

    graph = env.build_graph(build)
    assert _kernels(graph, "RmsNormGrad")[0].spec.ints[0] == 0
    env.run(graph, 0)
    d = {n: a.astype(np.float64) for n, a in data.items()}
    _, s, rho = ref.rms_norm(d["x"], d["w"], d["r"], 1e-6)
    want, share = ref.rms_norm_grad(s, rho, d["w"], d["dy"], None)
    assert np.allclose(env.read_parameter(gx), want, atol=1e-5) and np.array_equal(env.read_parameter(gx), env.read_parameter(gr))
    assert np.allclose(env.read_parameter(gw), share.sum(0), atol=1e-5)


def test_views_are_read_in_place_where_the_kernel_can():
    env = _env()
    packed, o = env.static_parameter([2, 5, 8, 4], "packed"), env.static_parameter([2, 5, 4, 4], "o")

    def slices(s):
        a = s.parameter_value(packed)
        q, k, v = a.limit_axis(2, 0, 4), a.limit_axis(2, 4, 6), a.limit_axis(2, 6, 8)
        s.write_parameter_value(o, q.attention(k, v))

    assert _labels(env.build_graph(slices)) == ["Attention"]
    turned = env.static_parameter([2, 4, 5, 4], "turned")
    assert _labels(env.build_graph(lambda s: s.write_parameter_value(o, (lambda a: a.attention(a, a))(s.parameter_value(turned).permute_axes([0, 2, 1, 3]))))) == ["Attention"]
    # the head's elements apart, or repeated past the edge: a copy first
    apart = env.static_parameter([2, 5, 4, 4], "apart")
    graph = env.build_graph(lambda s: s.write_parameter_value(o, (lambda a: a.attention(a, a))(s.parameter_value(apart).permute_axes([0, 1, 3, 2]))))
    assert _labels(graph) == ["PerElement", "Attention"]
    short = env.static_parameter([2, 3, 4, 4], "short")
    graph = env.build_graph(lambda s: s.write_parameter_value(o, (lambda a: a.attention(a, a))(s.parameter_value(short).pad(1, 1, 1))))
    assert _labels(graph) == ["PerElement", "Attention"]
    # a gradient that is a literal
    def literal(s):
        y = s.parameter(apart).attention(s.parameter(apart), s.parameter(apart))
        y.loss_grad().accumulate(s.literal(1.0).value().broadcast(y.shape))
        s.write_parameter_value(o, s.parameter(apart).loss_grad())

    assert "PerElement" in _labels(env.build_graph(literal))


def test_a_block_step_by_step_gives_the_whole():
    env = _env()
    rng = np.random.default_rng(4)
    block = TransformerBlock(env, 24, heads=4, n_hidden=20, groups=2, window=4, sinks=1)
    for p in _trainable(block):
        env.reset_parameter(p, rng)
    data = rng.standard_normal((2, 9, 24)).astype(np.float32)
    x, y = env.static_parameter_with_data(data.shape, "x", data), env.static_parameter(data.shape, "y")
    env.run(env.build_graph(lambda s: s.write_parameter_value(y, block.test(s.parameter(x)).value())), 0)
    whole = env.read_parameter(y)
    cache = block.attention.cache(env, 2, 9)
    xt, yt, start = env.static_parameter([2, 3, 24], "xt"), env.static_parameter([2, 3, 24], "yt"), env.static_parameter([2], "start")
    graph = env.build_graph(lambda s: s.write_parameter_value(yt, block.step(s.parameter_value(xt), cache, s.parameter_value(start).to_u32_bits())))
    for done in (0, 3, 6):
        env.write_parameter(xt, data[:, done : done + 3])
        env.write_parameter(start, np.full(2, done, np.uint32))
        env.run(graph, 0)
        assert np.allclose(env.read_parameter(yt), whole[:, done : done + 3], atol=1e-6)


def _trainable(module):
    from descent_amd import Module

    out = []
    for v in vars(module).values():
        if isinstance(v, Module):
            out += _trainable(v)
        elif getattr(v, "reset_to", None) is not None:
            out.append(v)
    return out


def test_a_blocks_gradients_against_differences():
    """Every parameter's gradient along a random direction."""
    env = _env()
    rng = np.random.default_rng(5)
    block = TransformerBlock(env, 12, heads=2, n_hidden=10, groups=1, window=3, sinks=1, activation="gelu")
    params = _trainable(block)
    for p in params:
        env.reset_parameter(p, rng)
    data, weight = rng.standard_normal((2, 5, 12)), rng.standard_normal((2, 5, 12))
    x, w = env.static_parameter_with_data(data.shape, "x", data), env.static_parameter_with_data(data.shape, "w", weight)
    y = env.static_parameter(data.shape, "y")
    grads = [env.static_parameter(p.shape, "g") for p in params]

    def build(s):
        z = block.train(s.parameter(x))
        s.write_parameter_value(y, z.value())
        z.loss_grad().accumulate(s.parameter_value(w))
        for p, g in zip(params, grads):
            s.write_parameter_value(g, s.parameter(p).loss_grad())

    graph = env.build_graph(build)
    env.run(graph, 0)
    values = [env.read_parameter(p).astype(np.float64) for p in params]
    along = [rng.standard_normal(v.shape) for v in values]
    got = [(env.read_parameter(g) * a).sum() for g, a in zip(grads, along)]
    for p, v, a, g in zip(params, values, along, got):
        ends = []
        for sign in (1.0, -1.0):
            env.write_parameter(p, (v + sign * 1e-2 * a).astype(np.float32))
            env.run(graph, 0)
            ends.append((env.read_parameter(y).astype(np.float64) * weight).sum())
        env.write_parameter(p, v.astype(np.float32))
        # a step of 10^-2 leaves the third derivative's share, 10^-4 of it, and node outputs rounded to 2^-24 over the step
        assert abs((ends[0] - ends[1]) / 2e-2 - g) <= 2e-2 * max(abs(g), 1.0), p.name


# ------------------------------------------------------------------------------------------------------ refusals


def test_arguments_are_checked():
    env = _env()
    q, k, s8 = env.static_parameter([2, 5, 4, 6], "q"), env.static_parameter([2, 5, 2, 6], "k"), env.static_parameter([2, 5, 3, 6], "s8")
    x, w, other, t = (env.static_parameter(s, "p") for s in ([4, 6], [6, 8], [6, 9], [4]))
    bad = [
        lambda s: s.parameter_value(x).rms_norm(s.parameter_value(t)),
        lambda s: s.parameter_value(x).rms_norm(s.parameter_value(env.static_parameter([6], "w")), -1.0),
        lambda s: s.parameter_value(x).add_rms_norm(s.parameter_value(w), s.parameter_value(env.static_parameter([6], "w"))),
        lambda s: s.parameter_value(q).rotary(s.parameter_value(t)),
        lambda s: s.parameter_value(q).rotary(s.parameter_value(env.static_parameter([3], "f")), s.parameter_value(env.static_parameter([3], "p"))),
        lambda s: s.parameter_value(q).rotary(s.parameter_value(env.static_parameter([3], "f")), layout="pairs"),
        lambda s: s.parameter_value(x).rotary(s.parameter_value(t)),
        lambda s: s.parameter_value(q).attention(s.parameter_value(k), s.parameter_value(s8)),
        lambda s: s.parameter_value(q).attention(s.parameter_value(s8), s.parameter_value(s8)),
        lambda s: s.parameter_value(q).attention(s.parameter_value(k), s.parameter_value(k), window=0),
        lambda s: s.parameter_value(q).attention(s.parameter_value(k), s.parameter_value(k), sinks=-1),
        lambda s: s.parameter_value(q).attention(s.parameter_value(k), s.parameter_value(k), scale=float("inf")),
        lambda s: s.parameter_value(q).attention(s.parameter_value(k), s.parameter_value(k), length=s.parameter_value(t)),
        lambda s: (lambda a: a.attention(a.limit_axis(1, 0, 3), a.limit_axis(1, 0, 3)))(s.parameter_value(q)),  # more queries than keys
        lambda s: (lambda a: a.attention(a, a))(s.parameter_value(env.static_parameter([1, 2, 1, 257], "wide"))),
        lambda s: s.parameter_value(x).gated_dense(s.parameter_value(w), s.parameter_value(other)),
        lambda s: s.parameter_value(x).gated_dense(s.parameter_value(w), s.parameter_value(w), "tanh"),
        lambda s: s.parameter_value(q).gated_dense(s.parameter_value(w), s.parameter_value(w)),
        lambda s: s.parameter_value(x).gated_dense(env.scope().parameter_value(w), s.parameter_value(w)),  # another scope
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError) as e:
            env.build_graph(f)
        assert len(str(e.value)) > 15, i
    with pytest.raises(ValueError, match="do not fit"):
        env.build_graph(lambda s: s.parameter_value(env.static_parameter([2, 9, 5], "c")).cache_append(s.parameter_value(env.static_parameter([2, 1, 6], "r")), s.parameter_value(t)))
    with pytest.raises(ValueError, match="start must be"):
        env.build_graph(lambda s: s.parameter_value(env.static_parameter([2, 9, 5], "c")).cache_append(s.parameter_value(env.static_parameter([2, 1, 5], "r")), s.parameter_value(t)))
    cache = SelfAttention(env, 8, 2).cache(env, 2, 4)
    with pytest.raises(ValueError, match="cache holds"):
        env.build_graph(lambda s: cache.append(s, cache.keys, s.parameter_value(q), s.parameter_value(t)))


def _view(shape, offsets=None, mapping=None, out=None):
    v = Shape(shape).identity_view()
    return View(v.input_shape, tuple(offsets or v.input_offsets), tuple(mapping or v.mapping), Shape(out or shape))


def test_malformed_operator_descriptors_are_rejected_with_a_message():
    ident = lambda *s: Shape(s).identity_view()  # noqa: E731
    q, k, f = ident(2, 5, 4, 8), ident(2, 5, 2, 8), ident(4)
    att = lambda ints, inputs, results=(0, 1), scale=1.0: OperatorKernel(OperatorSpec("Attention", ints, (scale,)), inputs, results)  # noqa: E731
    bad = [
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (1e-6,)), (ident(4, 6), ident(5)), (0,)),
        OperatorKernel(OperatorSpec("RmsNorm", (1,), (1e-6,)), (ident(4, 6), ident(6)), (0,)),
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (-1.0,)), (ident(4, 6), ident(6)), (0,)),
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (float("inf"),)), (ident(4, 6), ident(6)), (0,)),
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (1e-6,)), (ident(4, 6), ident(6)), (1,)),
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (1e-6,)), (ident(4, 6), ident(6)), (0, 2, 1)),
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (1e-6,)), (_view((4, 6), (0, 3)), ident(6)), (0,)),  # leaves the array
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (1e-6,)), (ident(6, 4).transposed(), ident(6)), (0,)),
        OperatorKernel(OperatorSpec("RmsNorm", (0,), (1e-6,)), (ident(4, 6), _view((12,), mapping=((0, 2),), out=(6,))), (0,)),
        OperatorKernel(OperatorSpec("RmsNormGrad", (0, 5)), (ident(4, 6), ident(4), ident(6), ident(4, 6)), (0,)),
        OperatorKernel(OperatorSpec("Rotary", (0, 0, 0), (1.0,)), (q, ident(5)), (0,)),
        OperatorKernel(OperatorSpec("Rotary", (2, 0, 0), (1.0,)), (q, f), (0,)),
        OperatorKernel(OperatorSpec("Rotary", (0, 0, 1), (1.0,)), (q, f, ident(3)), (0,)),
        OperatorKernel(OperatorSpec("Rotary", (0, 0, 2), (1.0,)), (q, f, ident(2)), (0,)),
        att((0, 0, 0, 1), (q, ident(2, 5, 3, 8), ident(2, 5, 3, 8))),
        att((-1, 0, 0, 1), (q, k, k)),
        att((0, 0, 0, 65), (q, k, k)),
        att((0, 0, 2, 1), (q, k, k, ident(3))),
        att((0, 0, 1, 1), (q, k, k)),
        att((0, 0, 0, 1), (q, ident(2, 4, 2, 8), ident(2, 4, 2, 8))),
        att((0, 0, 0, 1), (q, k, _view((2, 5, 8, 2), mapping=((0, 1), (1, 1), (3, 1), (2, 1)), out=(2, 5, 2, 8)))),
        att((0, 0, 0, 1), (q, k, k), scale=float("nan")),
        OperatorKernel(OperatorSpec("AttentionGradQuery", (0, 0, 0), (1.0,)), (q, k, k, q, q, ident(2, 5, 3)), (0,)),
        OperatorKernel(OperatorSpec("AttentionGradKeyValue", (0, 0, 0, 0), (1.0,)), (q, k, k, k, ident(2, 5, 4), ident(2, 5, 4)), (0,)),
        OperatorKernel(OperatorSpec("AttentionGradKeyValue", (3, 2, 0, 2), (1.0,)), (q, k, k, q, ident(2, 5, 4), ident(2, 5, 4)), (0,)),
        OperatorKernel(OperatorSpec("AttentionGradKeyValue", (3, 2, 0, 2), (1.0,)), (q, k, k, q, ident(2, 5, 4), ident(2, 5, 4)) + (ident(3, 2, 2, 2, 8),) * 2, (0,)),
        OperatorKernel(OperatorSpec("AttentionGradSinks", (3, 2, 0, 65), (1.0,)), (q, k, k, q, ident(2, 5, 4), ident(2, 5, 4)), (0, 1)),
        OperatorKernel(OperatorSpec("AttentionGradSinks", (0, 2, 0, 2), (1.0,)), (q, k, k, q, ident(2, 5, 4), ident(2, 5, 4)), (0, 1)),
        OperatorKernel(OperatorSpec("AttentionJoin"), (ident(3, 2, 5, 4, 8), ident(2, 2, 5, 4)), (0,)),
        OperatorKernel(OperatorSpec("DualMatMul", (DUAL_GATED, 4, 1)), (ident(3, 4), ident(4, 5), ident(4, 5)), (0,)),
        OperatorKernel(OperatorSpec("DualMatMul", (DUAL_BOTH, 0, 1)), (ident(3, 4), ident(5, 5), ident(5, 5)), (0,)),
        OperatorKernel(OperatorSpec("DualMatMul", (DUAL_SUM, 0, 1)), (ident(3, 4), ident(2, 4), ident(4, 5), ident(4, 5)), (0,)),
        OperatorKernel(OperatorSpec("DualMatMul", (DUAL_BOTH, 0, 1)), (_view((6, 8), mapping=((0, 2), (1, 2)), out=(3, 4)), ident(4, 5), ident(4, 5)), (0,)),
        OperatorKernel(OperatorSpec("CacheAppend", (9,)), (ident(2, 3, 4), ident(3)), (0,)),
        OperatorKernel(OperatorSpec("CacheAppend", (9,)), (ident(2, 4, 3).transposed(), ident(2)), (0,)),
        OperatorKernel(OperatorSpec("GatedGrad", (4,)), (ident(3, 4),) * 3, (0,)),
        OperatorKernel(OperatorSpec("GatedGrad", (0,)), (ident(3, 4), ident(3, 4), ident(4, 3)), (0,)),
    ]
    for i, kernel in enumerate(bad):
        with pytest.raises(hip_backend.DescentHipError) as e:
            hip_backend.codegen_source(kernel)
        assert e.value.status == _abi.ERR_INVALID and len(str(e.value)) > 20, (i, str(e.value))
    # attributes that the Python classes cannot hold
    good = [(att((0, 0, 0, 1), (q, k, k)), 3, 0), (OperatorKernel(OperatorSpec("DualMatMul", (0, 0, 1)), (ident(3, 4), ident(4, 5), ident(4, 5)), (0,)), 0, 3),
            (OperatorKernel(OperatorSpec("RmsNormGrad", (0, 1)), (ident(4, 6), ident(4), ident(6), ident(4, 6)), (0,)), 1, 0)]
    for kernel, at, value in good:
        mk = _abi.MarshalledKernel(kernel)
        mk.desc.op_int[at] = value
        out = C.c_void_p()
        assert hip_backend.lib().dsc_codegen_source(C.byref(mk.desc), C.byref(out)) == _abi.ERR_INVALID


def test_long_arrays_are_addressed_in_64_bits():
    """A cache of 2^33 elements: its offsets do not fit 32 bits, and the descriptor is taken."""
    cache = Shape((64, 1 << 20, 1, 128)).identity_view()
    kernel = OperatorKernel(OperatorSpec("Attention", (0, 0, 0, 16), (1.0,)), (Shape((64, 1, 8, 128)).identity_view(), cache, cache), (0, 1))
    assert "#define AT_K_B (134217728ll)" in hip_backend.codegen_source(kernel)
    assert hip_backend.codegen_compile(kernel) > 0


def test_keys_are_split_for_few_rows_only():
    assert attention_splits(Shape((1, 1, 8, 64)), Shape((1, 16384, 1, 64)), None, 0) == 64
    assert attention_splits(Shape((64, 1, 8, 64)), Shape((64, 16384, 8, 64)), None, 0) == 1
    assert attention_splits(Shape((1, 512, 8, 64)), Shape((1, 16384, 8, 64)), None, 0) == 1
    assert attention_splits(Shape((1, 1, 8, 64)), Shape((1, 200, 8, 64)), None, 0) == 1


# ------------------------------------------------------------------------------------------------------- kernels


def _compiled_kernels():
    rng = np.random.default_rng(6)
    out = []
    for c in cases.NORMS:
        out += [cases.norm_case(*c, rng)[0], cases.norm_grad_case(*c, rng)[0]] if c[1] < 50000 else []
    out += [cases.rotary_case(*c, rng)[0] for c in cases.ROTARIES]
    out += [cases.attention_case(*c, rng)[0] for c in cases.ATTENTIONS]
    for c in cases.ATTENTIONS[:6]:
        out += [k for k, _ in cases.attention_grad_cases(*c, rng, pieces=2 if c[6] and c[7] else 0)]
    out += [cases.dual_case(*c, rng)[0] for c in cases.DUALS if c[1] < 2000]
    out += [cases.gated_grad_case((5, 3), a, rng)[0] for a in range(4)]
    out += [cases.join_case(3, 2, 1, 2, 8, rng)[0]]
    out += [OperatorKernel(OperatorSpec("CacheAppend", (9,)), (Shape((2, 3, w)).identity_view(), Shape((2,)).identity_view()), (0,)) for w in (8, 7)]
    return out


def test_every_kernel_compiles_for_gfx950():
    for kernel in _compiled_kernels():
        source = hip_backend.codegen_source(kernel)
        assert 'extern "C" __global__' in source
        assert hip_backend.codegen_compile(kernel, "gfx950") > 0, kernel


def test_schedules_keep_operators_whole():
    """The planner fuses what surrounds the operators and leaves them alone: one launch each, fused or not."""
    env = _env()
    block = TransformerBlock(env, 48, heads=4, n_hidden=72, groups=2, window=7, sinks=2)
    for p in _trainable(block):
        env.writer(p).zero_fill()
    x, y = env.static_parameter([3, 21, 48], "x"), env.static_parameter([3, 21, 48], "y")
    grads = [env.static_parameter(p.shape, "g") for p in _trainable(block)]

    def build(s):
        z = block.train(s.parameter(x))
        s.write_parameter_value(y, z.value())
        (z * z).set_loss()
        for p, g in zip(_trainable(block), grads):
            s.write_parameter_value(g, s.parameter(p).loss_grad())

    graph = env.build_graph(build)
    count = sum(isinstance(graph.clusters[c].kernel, OperatorKernel) for c in graph.clusters_sorted)
    for fused in (True, False):
        text = hip_backend.check_schedule(graph, fused=fused)
        names = ("RmsNorm", "Rotary", "Attention", "DualMatMul", "GatedGrad")
        assert sum(line.split(": ", 1)[-1].startswith(names) for line in text.splitlines()) == count
