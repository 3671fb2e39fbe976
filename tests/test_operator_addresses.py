"""CPU: what the operators' kernels read and write stays inside their operands (host_kernel.py)."""
import re

import numpy as np
import pytest

import host_kernel
import operator_cases as cases
from descent_amd import Environment, hip_backend
from descent_amd.operators import OperatorKernel, OperatorSpec, emit
from descent_amd.shape import Shape
from oracle.cpu_backend import CpuBackend


def _grid(kernel):
    """Workgroups of a kernel's launch, from the listing of a schedule that holds nothing else."""
    env = Environment(CpuBackend())
    operands = [env.static_parameter(list(v.output_shape), "p") for v in kernel.inputs]
    results = [env.static_parameter(list(kernel.result_shapes()[i]), "r") for i in kernel.results]

    def build(s):
        got = emit([s.parameter_value(p) for p in operands], kernel.spec, len(results))
        for p, a in zip(results, got):
            s.write_parameter_value(p, a)

    (grid,) = re.findall(r" grid (\d+)x", hip_backend.check_schedule(env.build_graph(build), fused=False))
    return int(grid)


def _kernels():
    rng = np.random.default_rng(3)
    out = []
    for c in [(1, 1, False), (7, 100, True), (33, 2048, True), (600, 33, False), (2, 40000, True)]:
        out += [cases.norm_case(*c, rng), cases.norm_grad_case(*c, rng)]
    out += [cases.rotary_case(*c, rng) for c in cases.ROTARIES[:6]]
    out += [cases.dual_case(*c, rng) for c in cases.DUALS if c[1] < 300]
    # (batch, tokens, keys, heads, groups, dim, window, sinks, places)
    for c in [(2, 1, 40, 4, 2, 16, 0, 0, "both"), (1, 3, 90, 2, 1, 30, 17, 4, "start"), (1, 33, 33, 1, 1, 256, 0, 0, "none"), (1, 70, 100, 3, 1, 48, 20, 5, "length"),
              (2, 65, 65, 2, 2, 112, 9, 70, "length"), (1, 66, 130, 2, 1, 200, 64, 1, "both")]:
        out += [cases.attention_case(*c, rng)] + cases.attention_grad_cases(*c, rng, pieces=3 if c[6] and c[7] else 0)
        out += [cases.attention_case(*c, rng, splits=3)] if c[1] < 17 else []
    return out


def test_operators_stay_inside_their_operands():
    for kernel, arrays in _kernels():
        host_kernel.run(kernel, arrays, _grid(kernel))


def _split_grid(kernel):
    """Workgroups of the attention kernel for more than 64 rows of a key head and heads of up to 128."""
    define = dict(re.findall(r"#define (AT_\w+) \(?(-?\d+)", hip_backend.codegen_source(kernel)))
    assert "AT_FORWARD_SPLIT" in define
    b, t, h, g, waves = (int(define["AT_" + n]) for n in ("B", "T", "H", "G", "WAVES"))
    return b * g * -(-t * (h // g) // (32 * waves))


@pytest.mark.parametrize("dim", [16, 48, 80, 112, 20, 32, 128, 15, 31])
def test_prompt_attention_reads_inside_its_operands(dim):
    """Heads that are no multiple of the 32 elements that a matrix instruction's tile takes end with the query row."""
    kernel, arrays = cases.attention_case(2, 70, 70, 2, 2, dim, 20, 2, "none", np.random.default_rng(1))
    host_kernel.run(kernel, arrays, _split_grid(kernel))


@pytest.mark.parametrize("window", [20, 70])
def test_more_sinks_than_keys(window):
    """A descriptor may ask for any number of sinks: past the last key there are none, and nothing is read there."""
    kernel, arrays = cases.attention_case(1, 90, 90, 2, 2, 32, window, 2, "none", np.random.default_rng(2))
    most = cases.kernel(OperatorSpec("Attention", (window, 0x7FFFFFFF) + kernel.spec.ints[2:], kernel.spec.floats), arrays)
    host_kernel.run(most, arrays, _split_grid(most))
    all_of_them = cases.kernel(OperatorSpec("Attention", (window, 90) + kernel.spec.ints[2:], kernel.spec.floats), arrays)
    assert hip_backend.codegen_source(most) == hip_backend.codegen_source(all_of_them)


def test_rows_of_a_key_head_are_counted_in_32_bits():
    """Up to what a kernel adds to the last of them while it rounds up to tiles."""
    def prompt(tokens):
        q, k = Shape((1, tokens, 2, 4)).identity_view(), Shape((1, (1 << 30) - 1, 1, 4)).identity_view()
        return OperatorKernel(OperatorSpec("Attention", (8, 0, 0, 1), (1.0,)), (q, k, k), (0, 1))

    assert "attention_split" in hip_backend.codegen_source(prompt((1 << 30) - 300))
    with pytest.raises(hip_backend.DescentHipError, match="rows of a key head"):
        hip_backend.codegen_source(prompt((1 << 30) - 1))
