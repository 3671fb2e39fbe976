"""CPU: what the operators' kernels read and write stays inside their operands (host_kernel.py)."""
import re

import numpy as np
import pytest

import host_kernel
import operator_cases as cases
from descent_amd import hip_backend
from descent_amd.operators import OperatorKernel, OperatorSpec
from descent_amd.shape import Shape


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
