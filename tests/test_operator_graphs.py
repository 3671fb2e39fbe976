"""CPU: graphs of the sequence-model operators in which not every result leads to the loss."""
import numpy as np
import pytest

from descent_amd import Environment, hip_backend
from oracle.cpu_backend import CpuBackend


@pytest.mark.parametrize("rows", [1, 4, 700])
@pytest.mark.parametrize("then", ["directly", "through a layer"])
def test_a_loss_that_takes_the_sum_and_not_the_norm(rows, then):
    """d sum goes to both summands as it is, and the norm's weight gets zeros."""
    env = Environment(CpuBackend())
    rng = np.random.default_rng(1)
    data = {n: rng.standard_normal(s).astype(np.float32) for n, s in (("x", (rows, 6)), ("r", (rows, 6)), ("w", (6,)), ("dsum", (rows, 6)))}
    p = {n: env.static_parameter_with_data(a.shape, n, a) for n, a in data.items()}
    out = {n: env.static_parameter(data[n].shape, "g" + n) for n in "xrw"}

    def build(s, n):
        _, total = s.parameter(p["x"]).add_rms_norm(s.parameter(p["r"]), s.parameter(p["w"]))
        if then != "directly":
            total = total * 2.0
        total.loss_grad().accumulate(s.parameter_value(p["dsum"]))
        s.write_parameter_value(out[n], s.parameter(p[n]).loss_grad())

    for n in "xrw":  # (a graph each: one value cannot become two parameters')
        graph = env.build_graph(lambda s: build(s, n))
        assert not any("RmsNorm" in graph.clusters[c].kernel.label_name() for c in graph.clusters_sorted)
        for fused in (True, False):
            hip_backend.check_schedule(graph, fused=fused)
        env.run(graph, 0)
    want = data["dsum"] * np.float32(1.0 if then == "directly" else 2.0)
    assert np.array_equal(env.read_parameter(out["x"]), want) and np.array_equal(env.read_parameter(out["r"]), want)
    assert np.array_equal(env.read_parameter(out["w"]), np.zeros(6))


def test_a_norm_that_no_loss_takes_beside_one_that_does():
    """Two norms share their weight and the first one's sum feeds the second: the weight's gradient is the second's alone."""
    from oracle import operators as ref

    env = Environment(CpuBackend())
    rng = np.random.default_rng(2)
    data = {n: rng.standard_normal(s).astype(np.float32) for n, s in (("x", (5, 6)), ("r", (5, 6)), ("w", (6,)), ("dy", (5, 6)))}
    p = {n: env.static_parameter_with_data(a.shape, n, a) for n, a in data.items()}
    out = {n: env.static_parameter(data[n].shape, "g" + n) for n in "xrw"}

    def build(s):
        _, total = s.parameter(p["x"]).add_rms_norm(s.parameter(p["r"]), s.parameter(p["w"]))
        y = total.rms_norm(s.parameter(p["w"]))
        y.loss_grad().accumulate(s.parameter_value(p["dy"]))
        for n in "xrw":
            s.write_parameter_value(out[n], s.parameter(p[n]).loss_grad())

    graph = env.build_graph(build)
    env.run(graph, 0)
    d = {n: a.astype(np.float64) for n, a in data.items()}
    _, total, rho = ref.rms_norm(d["x"] + d["r"], d["w"], None, 1e-6)
    want, share = ref.rms_norm_grad(total, rho, d["w"], d["dy"], None)
    assert np.allclose(env.read_parameter(out["x"]), want, atol=1e-5) and np.array_equal(env.read_parameter(out["x"]), env.read_parameter(out["r"]))
    assert np.allclose(env.read_parameter(out["w"]), share.sum(0), atol=1e-5)


def test_places_given_as_numbers():
    """A start, a length or a position may be a number where an array of one would do: it is a whole number then, not the
    bits of a float."""
    env = Environment(CpuBackend())
    rng = np.random.default_rng(3)
    q, k, rows = rng.standard_normal((1, 2, 4, 6)), rng.standard_normal((1, 9, 2, 6)), rng.standard_normal((1, 2, 5))
    p = {n: env.static_parameter_with_data(a.shape, n, a) for n, a in (("q", q), ("k", k), ("rows", rows), ("f", np.array([1.0, 0.1])))}
    place = env.static_parameter([1], "place")
    env.write_parameter(place, np.array([3], np.uint32))
    results = []
    for given in (None, 3, np.int64(3), np.uint32(3)):
        out = [env.static_parameter(s, "out") for s in ([1, 2, 4, 6], [1, 2, 4, 6], [1, 2, 4, 6], [1, 9, 5])]
        cache = env.static_parameter_with_data([1, 9, 5], "cache", np.zeros((1, 9, 5)))

        def build(s):
            at = s.parameter_value(place).to_u32_bits() if given is None else given
            a, b = s.parameter_value(p["q"]), s.parameter_value(p["k"])
            s.write_parameter_value(out[0], a.attention(b, b, start=at, length=at))
            s.write_parameter_value(out[1], s.parameter(p["q"]).attention(s.parameter(p["k"]), s.parameter(p["k"]), start=at).value())
            s.write_parameter_value(out[2], a.rotary(p["f"], at))
            s.write_parameter_value(cache, s.parameter_value(cache).cache_append(p["rows"], at))

        graph = env.build_graph(build)
        hip_backend.check_schedule(graph)
        env.run(graph, 0)
        results.append([env.read_parameter(o) for o in out[:3]] + [env.read_parameter(cache)])
    assert np.abs(results[0][1]).min() > 0 and not results[0][0].any()  # (a length of 3: both tokens are padding)
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert np.array_equal(a, b)
    for bad in (3.0, -1, 1 << 32, True):
        with pytest.raises(ValueError, match="whole number"):
            env.build_graph(lambda s: s.parameter_value(p["q"]).attention(p["k"], p["k"], start=bad))
        with pytest.raises(ValueError, match="whole number"):
            env.build_graph(lambda s: s.parameter_value(p["q"]).rotary(p["f"], bad))
