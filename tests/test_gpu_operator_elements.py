"""GPU: elements at the ends of the operators' ranges -- not finite, too large for a shorter type, behind an operand --
reach the results that they take part in, and no others."""
import numpy as np
import pytest

import operator_cases as cases
from descent_amd.operators import ACTIVATIONS, DUAL_BOTH, DUAL_GATED, DUAL_SUM, OperatorKernel, OperatorSpec
from descent_amd.shape import Shape, View
from oracle import operators as ref
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


def _agree(got, want, bounds):
    """NaN exactly where the definition has it, everything else within its bound."""
    for i, (g, w, b) in enumerate(zip(got, want, bounds)):
        assert np.array_equal(np.isnan(g), np.isnan(w)), f"result {i}: {np.isnan(g).sum()} NaN for {np.isnan(w).sum()}"
        rest = ~np.isnan(w)
        low = np.isneginf(w)
        assert np.array_equal(np.isneginf(g), low), f"result {i}"
        rest &= ~low
        off = np.abs(g.astype(np.float64) - np.where(rest, w, 0.0))[rest] - (np.broadcast_to(b, w.shape) + cases.U * np.abs(w))[rest]
        assert off.max(initial=-1.0) <= 0.0, f"result {i}: {off.max()}"


def _clean(arrays):
    return [np.where(np.isfinite(a), a, np.float32(0)) if a.dtype == np.float32 else a for a in arrays]


def _forward(backend, kernel, arrays, splits):
    """The kernel's results and the definition's, with the bounds of the same call without the odd elements."""
    want = ref.evaluate(kernel, cases.flat(arrays))
    bounds = cases.attention_bounds(kernel, _clean(arrays), ref.evaluate(kernel, cases.flat(_clean(arrays))))
    if splits == 1:
        return launch(backend, kernel, arrays), want, bounds
    pieces = cases.kernel(OperatorSpec("Attention", kernel.spec.ints[:3] + (splits,), kernel.spec.floats), arrays)
    part = launch(backend, pieces, arrays)
    # the join's exponentials, sums and quotient, each against the largest value
    largest = [np.abs(_clean(arrays)[2]).max(), 1.0]
    joined = launch(backend, cases.kernel(OperatorSpec("AttentionJoin"), part), part)
    return joined, want, [b + 8 * splits * cases.U * (np.where(np.isfinite(w), np.abs(w), 0.0) + m) for b, w, m in zip(bounds, want, largest)]


# (batch, tokens, keys, heads, groups, dim, splits): a few rows, whole and in pieces; tiles in three parts; wide heads
KERNELS = [(2, 1, 600, 4, 2, 64, 1), (2, 1, 600, 4, 2, 48, 2), (1, 3, 600, 2, 1, 200, 5), (1, 2, 600, 3, 3, 30, 64), (2, 70, 70, 4, 2, 64, 1),
           (1, 80, 90, 2, 1, 48, 1), (1, 90, 90, 2, 2, 80, 1), (1, 70, 80, 1, 1, 31, 1), (1, 70, 70, 2, 1, 200, 1), (2, 80, 90, 2, 2, 160, 1)]


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_queries_that_are_not_finite(hip_backend_session, case, value):
    """Every score of such a row is NaN or infinite, so the row is NaN, and so is its denominator; a row of padding is not."""
    batch, tokens, keys, heads, groups, dim, splits = case
    for window, sinks in ((0, 0), (20, 2), (1, 0)):
        kernel, arrays = cases.attention_case(batch, tokens, keys, heads, groups, dim, window, sinks, "both", np.random.default_rng(22))
        arrays[3][:] = [keys - tokens, 0][:batch]
        arrays[4][:] = [keys, max(1, tokens - 4)][:batch]
        arrays[0][:, :: max(1, tokens // 5), -1, dim // 2] = value  # the first row among them, which may see one key only
        got, want, bounds = _forward(hip_backend_session, kernel, arrays, splits)
        assert np.isnan(want[1]).any() and not np.isnan(want[1]).all()
        _agree(got, want, bounds)


@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_keys_that_are_not_numbers(hip_backend_session, case):
    """A row is NaN if and only if it sees such a key: as one of many, as the only one of a row, of a block of 16 or of a
    piece, as a sink, or its own new key behind a cache."""
    batch, tokens, keys, heads, groups, dim, splits = case
    for window, sinks, at in ((0, 0, 0), (0, 0, keys - tokens), (1, 0, keys - tokens), (1, 0, 16), (7, 3, 1), (0, 0, 16)):
        kernel, arrays = cases.attention_case(batch, tokens, keys, heads, groups, dim, window, sinks, "both", np.random.default_rng(23))
        arrays[3][:] = [16 if at == 16 and tokens < 16 else keys - tokens, 0][:batch]
        arrays[4][:] = [keys, keys - 3][:batch]
        arrays[1][:, at, :, dim - 1] = np.nan
        got, want, bounds = _forward(hip_backend_session, kernel, arrays, splits)
        assert np.isnan(want[0]).any()
        _agree(got, want, bounds)


@pytest.mark.parametrize("case", [c for c in KERNELS if c[1] > 60 or c[6] == 1], ids=str)
def test_gradients_of_rows_that_are_not_numbers(hip_backend_session, case):
    """A row whose query is NaN: its own gradient is NaN, and that of every key that it sees, and no other."""
    batch, tokens, keys, heads, groups, dim, _ = case
    for window, sinks in ((0, 0), (20, 2), (1, 0)):
        (by_query, qa), (by_key, ka) = cases.attention_grad_cases(batch, tokens, keys, heads, groups, dim, window, sinks, "both", np.random.default_rng(24))
        clean = [[a.copy() for a in arrays] for arrays in (qa, ka)]
        start, length = qa[-2:]
        row = next(t for t in range(tokens) if int(start[0]) + t < int(length[0]))
        for arrays, touched in ((qa, (0, 3, 5)), (ka, (0, 4, 5))):
            for i in touched:
                arrays[i][0, row, 0] = np.nan  # the query, and what the forward pass made of it
        for (k, arrays), without in zip(((by_query, qa), (by_key, ka)), clean):
            bounds = cases.attention_grad_bounds(k, without, ref.evaluate(k, cases.flat(without)))
            want = ref.evaluate(k, cases.flat(arrays))
            assert np.isnan(want[0]).any() and np.isnan(want[1]).any()
            _agree(launch(hip_backend_session, k, arrays), want, bounds)


@pytest.mark.parametrize("tokens,keys,dim", [(1, 2000, 64), (70, 70, 48), (66, 66, 136)])
def test_a_graph_passes_what_is_not_a_number_on(hip_backend_session, tokens, keys, dim):
    """Through the public calls, forward and backward: a NaN query reaches its row and the gradients, a NaN key its readers."""
    from descent_amd import Environment

    rng = np.random.default_rng(25)
    env = Environment(hip_backend_session)
    data = {"q": cases.normal(rng, 1, tokens, 4, dim), "k": cases.normal(rng, 1, keys, 2, dim), "v": cases.normal(rng, 1, keys, 2, dim),
            "dy": cases.normal(rng, 1, tokens, 4, dim)}
    data["q"][0, 0, 1, 3] = np.nan
    p = {n: env.static_parameter_with_data(a.shape, n, a) for n, a in data.items()}
    out = {n: env.static_parameter(data[n if n != "y" else "q"].shape, n) for n in ("y", "q", "k", "v")}

    def build(s):
        y = s.parameter(p["q"]).attention(s.parameter(p["k"]), s.parameter(p["v"]))
        y.loss_grad().accumulate(s.parameter_value(p["dy"]))
        s.write_parameter_value(out["y"], y.value())
        for n in "qkv":
            s.write_parameter_value(out[n], s.parameter(p[n]).loss_grad())

    graph = env.build_graph(build)
    env.run(graph, 0)
    got = {n: np.isnan(env.read_parameter(a)) for n, a in out.items()}
    row = np.zeros((1, tokens, 4, dim), bool)
    row[0, 0, 1] = True
    seen = np.zeros((1, keys, 2, dim), bool)
    seen[0, : keys - tokens + 1, 0] = True
    assert np.array_equal(got["y"], row) and np.array_equal(got["q"], row)
    assert np.array_equal(got["k"], seen) and np.array_equal(got["v"], seen)


LARGEST = np.finfo(np.float32).max  # past what rounds to a finite bfloat16


@pytest.mark.parametrize("transposed", [(), (1, 2), (0, 3)], ids=str)
@pytest.mark.parametrize("rows", [4, 40, 300])
@pytest.mark.parametrize("mode", [DUAL_GATED, DUAL_SUM, DUAL_BOTH])
def test_dual_products_of_the_largest_numbers(hip_backend_session, mode, rows, transposed):
    """Elements of the largest magnitude beside small ones and zeros: the products are finite, and as good as all others."""
    kernel, arrays = cases.dual_case(mode, rows, 70, 96, ACTIVATIONS.index("relu"), np.random.default_rng(26), transposed)
    x = [a.T if i in transposed else a for i, a in enumerate(arrays)]
    left = 2 if mode == DUAL_SUM else 1
    for i, a in enumerate(x):
        if i < left:
            a[2, 5], a[1, 9] = LARGEST, -LARGEST
            a[:, 50] *= np.float32(2.0 ** -80)
            a[:, 51] = 0.0
        else:
            a[5], a[9] = a[5] * np.float32(2.0 ** -80), 0.0
            a[50, 7], a[51, 8] = -LARGEST, LARGEST
    check(hip_backend_session, kernel, arrays, cases.dual_bounds)


@pytest.mark.parametrize("mode", [DUAL_GATED, DUAL_SUM, DUAL_BOTH])
def test_dual_products_of_small_numbers(hip_backend_session, mode):
    """Down to 2^-99 all three parts of a number are normal ones of the shorter type, and the bounds are the same."""
    kernel, arrays = cases.dual_case(mode, 40, 70, 96, ACTIVATIONS.index("relu"), np.random.default_rng(27))
    for i, a in enumerate(arrays):
        left = i < (2 if mode == DUAL_SUM else 1)
        a[:] = np.sign(a) * np.maximum(np.abs(a), 0.25) * np.float32(2.0 ** (-97 if left else 60))
    check(hip_backend_session, kernel, arrays, cases.dual_bounds)


@pytest.mark.parametrize("case", KERNELS, ids=str)
def test_attention_to_the_largest_numbers(hip_backend_session, case):
    """A key, a value and a query of the type's lowest value: harmless where the mask hides them or the other factor is 0,
    and weighted like any other where a row sees them."""
    batch, tokens, keys, heads, groups, dim, splits = case
    for window, sinks in ((0, 0), (20, 2), (1, 0)):
        kernel, arrays = cases.attention_case(batch, tokens, keys, heads, groups, dim, window, sinks, "both", np.random.default_rng(28))
        arrays[3][:] = [keys - tokens, 0][:batch]
        arrays[4][:] = [keys, max(1, tokens - 4)][:batch]
        q, k, v = arrays[:3]
        q[..., 0], k[:, [1, keys - tokens], :, 0] = 0.0, -LARGEST
        k[..., dim - 1], q[:, tokens - 1, :, dim - 1] = 0.0, -LARGEST
        v[:, keys - tokens, :, ::3] = -LARGEST
        _agree(*_forward(hip_backend_session, kernel, arrays, splits))


@pytest.mark.parametrize("width", [8196, 16384, 20001, 32768, 32772, 65536])
def test_wide_norms(hip_backend_session, width):
    """Rows around the widths at which a row no longer stays in the registers of its threads."""
    for residual in (False, True):
        rng = np.random.default_rng(29)
        check(hip_backend_session, *cases.norm_case(3, width, residual, rng), cases.norm_bounds)
        check(hip_backend_session, *cases.norm_grad_case(3, width, residual, rng), cases.norm_grad_bounds)


@pytest.mark.parametrize("tokens,dim", [(1, 64), (70, 64), (70, 160)])
def test_a_cache_of_more_than_2_31_elements(hip_backend_session, tokens, dim):
    """The last keys of the last sequence lie past 2^31 elements: appended there, and seen through a window."""
    be, rng = hip_backend_session, np.random.default_rng(30)
    keys, window, tail = (1 << 30) // dim + 128, 40, 128
    q, k, v = (cases.normal(rng, 2, n, 1, dim) for n in (tokens, tail, tail))
    places = [np.full(2, keys - tokens, np.uint32), np.full(2, keys, np.uint32)]
    cache = Shape((2, keys, 1, dim))
    whole = []
    for rows in (k, v):  # only the rows that are seen are ever written; the rest stays as allocated
        h = be.alloc(cache.buffer_size())
        whole.append(h)
        handles = []
        for a in cases.flat([rows.reshape(2, tail, dim), np.full(2, keys - tail, np.uint32)]):
            handles.append(be.alloc(a.nbytes))
            be.write(handles[-1], 0, a)
        kernel = OperatorKernel(OperatorSpec("CacheAppend", (keys,)), (Shape((2, tail, dim)).identity_view(), Shape((2,)).identity_view()), (0,))
        be.launch(kernel, handles + [h], 0)
        last = np.frombuffer(be.read(h, cache.buffer_size() - 4 * tail * dim, 4 * tail * dim), np.float32)
        assert np.array_equal(last, rows[1].ravel())
        for a in handles:
            be.free(a)
    handles = []
    for a in cases.flat([q] + places):
        handles.append(be.alloc(a.nbytes))
        be.write(handles[-1], 0, a)
    views = (Shape(q.shape).identity_view(), cache.identity_view(), cache.identity_view()) + (Shape((2,)).identity_view(),) * 2
    kernel = OperatorKernel(OperatorSpec("Attention", (window, 0, 3, 1), (dim ** -0.5,)), views, (0, 1))
    out = [be.alloc(s.buffer_size()) for s in kernel.result_shapes()]
    be.launch(kernel, [handles[0]] + whole + handles[1:] + out, 0)
    got = [np.frombuffer(be.read(h, 0, s.buffer_size()), np.float32).reshape(tuple(s)) for h, s in zip(out, kernel.result_shapes())]
    for h in handles + whole + out:
        be.free(h)
    arrays = [q, k, v, np.full(2, tail - tokens, np.uint32), np.full(2, tail, np.uint32)]
    small = cases.kernel(kernel.spec, arrays)
    want = ref.evaluate(small, cases.flat(arrays))
    _agree(got, want, cases.attention_bounds(small, arrays, want))


@pytest.mark.parametrize("dim", [48, 64, 136])
def test_sinks_pieces_pass_what_is_not_a_number_on(hip_backend_session, dim):
    """A NaN query past the window reaches the gradients of the sinks and of its window, a row of padding reaches nothing."""
    case = (1, 200, 200, 4, 2, dim, 20, 5, "length")
    (_, _), (whole, ka), (far, fa), (joined, ja) = cases.attention_grad_cases(*case, np.random.default_rng(31), 3)
    clean = [a.copy() for a in ka]
    bounds = cases.attention_grad_bounds(whole, clean, ref.evaluate(whole, cases.flat(clean)))
    length = int(ka[-1][0])
    assert 160 < length < 200
    for arrays in (ka, fa, ja):
        for i in (0, 4, 5):
            arrays[i][0, 150, 1] = np.nan
        for i in (0, 3):
            arrays[i][0, length:] = np.nan
    want = ref.evaluate(whole, cases.flat(ka))
    assert np.isnan(want[0][0, :5, 0]).all() and np.isnan(want[0][0, 131:151, 0]).all() and np.isfinite(want[0][0, 5:131]).all()
    pieces = launch(hip_backend_session, far, fa)
    for p in pieces:
        assert np.isnan(p.sum(0)[0, :, 0]).all() and np.isfinite(p[:, :, :, 1]).all()
    got = launch(hip_backend_session, joined, ja[:6] + pieces + ja[8:])
    _agree(got, want, [2 * b for b in bounds])
