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
