"""GPU: elements at the ends of the operators' ranges -- not finite, too large for a shorter type, behind an operand --
reach the results that they take part in, and no others."""
import numpy as np
import pytest

import operator_cases as cases
from descent_amd.shape import Shape, View
from test_gpu_operators import check, launch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [16, 48, 80, 112, 20, 31, 64])
def test_query_rows_end_with_their_head(hip_backend_session, dim):
    """Behind each head of a query, and in the rows of padding, stands NaN: no row that counts takes any of it in."""
    kernel, arrays = cases.attention_case(2, 70, 70, 4, 2, dim, 20, 2, "length", np.random.default_rng(21))
    arrays[3][:] = [70, 60]
    want = check(hip_backend_session, kernel, arrays, cases.attention_bounds)
    q = arrays[0]
    wide = np.full(q.shape[:3] + (dim + 16,), np.nan, np.float32)
    wide[..., :dim] = q
    wide[1, 60:] = np.nan
    dense = Shape(q.shape).identity_view()
    inside = View(Shape(wide.shape), (0, 0, 0, 0), dense.mapping, dense.output_shape)
    strided = cases.kernel(kernel.spec, arrays, [inside] + list(kernel.inputs[1:]))
    padded = [q.copy()] + arrays[1:]
    padded[0][1, 60:] = np.nan
    for k, a in ((strided, [wide] + arrays[1:]), (kernel, padded)):
        for w, g in zip(want, launch(hip_backend_session, k, a)):
            assert np.array_equal(w, g)
