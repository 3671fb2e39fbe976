"""GPU: the sequence-model operators against their definitions in 64 bits, with the bounds of operator_cases.py."""
import numpy as np
import pytest

import operator_cases as cases
from conftest import rel_l2
from descent_amd.operators import ACTIVATIONS, DUAL_BOTH, DUAL_GATED, DUAL_SUM, OperatorKernel, OperatorSpec
from descent_amd.shape import Shape, View
from oracle import operators as ref

pytestmark = pytest.mark.gpu


def launch(backend, kernel, arrays, guard=64):
    """The kernel's results; what lies behind each result's buffer must stay as it was."""
    handles = []
    for a in cases.flat(arrays):
        h = backend.alloc(a.nbytes)
        backend.write(h, 0, a)
        handles.append(h)
    shapes = [kernel.result_shapes()[i] for i in kernel.results]
    outs, mark = [], np.full(guard, 12345.0, np.float32)
    for s in shapes:
        h = backend.alloc(s.buffer_size() + mark.nbytes)
        backend.write(h, 0, np.full(s.element_count() + guard, 12345.0, np.float32))
        outs.append(h)
    backend.launch(kernel, handles + outs, 0)
    got = []
    for s, h in zip(shapes, outs):
        raw = np.frombuffer(backend.read(h, 0, s.buffer_size() + mark.nbytes), np.float32)
        assert np.array_equal(raw[s.element_count() :], mark)
        got.append(raw[: s.element_count()].reshape(tuple(s)).copy())
    for h in handles + outs:
        backend.free(h)
    return got


def check(backend, kernel, arrays, bounds):
    want = ref.evaluate(kernel, cases.flat(arrays))
    got = launch(backend, kernel, arrays)
    for i, (g, w, b) in enumerate(zip(got, want, bounds(kernel, arrays, want))):
        finite = np.isfinite(w)
        assert np.array_equal(g[~finite], w[~finite].astype(np.float32)), f"result {i}"
        over = np.abs(g.astype(np.float64)[finite] - w[finite]) - np.broadcast_to(b, w.shape)[finite] - cases.U * np.abs(w[finite])
        assert over.max(initial=-1.0) <= 0.0, f"result {i}: {over.max()} past its bound at {np.argmax(over)} of {w.shape}"
    return got


@pytest.mark.parametrize("case", cases.NORMS, ids=str)
def test_norm(hip_backend_session, case):
    rng = np.random.default_rng(1)
    kernel, arrays = cases.norm_case(*case, rng)
    got = check(hip_backend_session, kernel, arrays, cases.norm_bounds)
    if case[2]:
        assert np.array_equal(got[1], arrays[0] + arrays[2])
    check(hip_backend_session, *cases.norm_grad_case(*case, rng), cases.norm_grad_bounds)


@pytest.mark.parametrize("case", cases.ROTARIES, ids=str)
def test_rotary(hip_backend_session, case):
    check(hip_backend_session, *cases.rotary_case(*case, np.random.default_rng(2)), cases.rotary_bounds)


@pytest.mark.parametrize("case", cases.ATTENTIONS, ids=str)
def test_attention(hip_backend_session, case):
    check(hip_backend_session, *cases.attention_case(*case, np.random.default_rng(3)), cases.attention_bounds)


@pytest.mark.parametrize("case", [c for c in cases.ATTENTIONS if c[2] <= 300], ids=str)
def test_attention_gradients(hip_backend_session, case):
    for kernel, arrays in cases.attention_grad_cases(*case, np.random.default_rng(4)):
        check(hip_backend_session, kernel, arrays, cases.attention_grad_bounds)


@pytest.mark.parametrize("pieces", [1, 3, 64])
@pytest.mark.parametrize("case", [c for c in cases.ATTENTIONS if c[6] and c[7] and 60 <= c[2] <= 300], ids=str)
def test_attention_gradients_of_sinks(hip_backend_session, case, pieces):
    """The rows past a tile's window, summed in pieces, and the key gradient that takes the pieces."""
    (_, _), (whole, whole_arrays), (far, arrays), (joined, joined_arrays) = cases.attention_grad_cases(*case, np.random.default_rng(18), pieces)
    want = ref.evaluate(far, cases.flat(arrays))
    got = launch(hip_backend_session, far, arrays)
    for g, w, b in zip(got, want, cases.attention_grad_bounds(far, arrays, want)):
        assert (np.abs(g.astype(np.float64).sum(0) - w.sum(0)) <= b[0] + pieces * cases.U * np.abs(w).sum(0)).all()
    check(hip_backend_session, joined, joined_arrays, cases.attention_grad_bounds)
    # together: what the kernel without pieces gives
    tail = joined_arrays[8:]
    both = launch(hip_backend_session, joined, joined_arrays[:6] + got + tail)
    want = ref.evaluate(whole, cases.flat(whole_arrays))
    for g, w, b in zip(both, want, cases.attention_grad_bounds(whole, whole_arrays, want)):
        assert (np.abs(g - w) <= 2 * b + cases.U * np.abs(w)).all()


@pytest.mark.parametrize("splits", [2, 5, 64])
@pytest.mark.parametrize("case", [c for c in cases.ATTENTIONS if c[1] <= 17], ids=str)
def test_attention_in_pieces(hip_backend_session, case, splits):
    """The pieces and their join give what the whole call gives."""
    kernel, arrays = cases.attention_case(*case, np.random.default_rng(5))
    pieces = cases.kernel(OperatorSpec("Attention", kernel.spec.ints[:3] + (splits,), kernel.spec.floats), arrays)
    part = launch(hip_backend_session, pieces, arrays)
    joined = launch(hip_backend_session, cases.kernel(OperatorSpec("AttentionJoin"), part), part)
    want = ref.evaluate(kernel, cases.flat(arrays))
    bound = cases.attention_bounds(kernel, arrays, want)
    more = 8 * splits * cases.U  # the join's exponentials, sums and quotient
    for g, w, b in zip(joined, want, bound):
        finite = np.isfinite(w)
        assert np.array_equal(g[~finite], w[~finite].astype(np.float32))
        slack = b + more * (np.abs(w) + (np.abs(arrays[2]).max() if w.ndim == 4 else 1.0))
        assert (np.abs(g - np.where(finite, w, 0.0))[finite] <= slack[finite]).all()


@pytest.mark.parametrize("shape", [(2, 1, 1, 1, 1), (5, 2, 3, 4, 40), (64, 1, 1, 2, 128)], ids=str)
def test_attention_join(hip_backend_session, shape):
    check(hip_backend_session, *cases.join_case(*shape, np.random.default_rng(6)), cases.join_bounds)


@pytest.mark.parametrize("case", cases.DUALS, ids=str)
def test_dual_product(hip_backend_session, case):
    rng = np.random.default_rng(7)
    check(hip_backend_session, *cases.dual_case(*case, rng), cases.dual_bounds)
    left = 2 if case[0] == DUAL_SUM else 1
    check(hip_backend_session, *cases.dual_case(*case, rng, transposed=range(left)), cases.dual_bounds)
    check(hip_backend_session, *cases.dual_case(*case, rng, transposed=range(left, left + 2)), cases.dual_bounds)
    check(hip_backend_session, *cases.dual_case(*case, rng, transposed=(left,)), cases.dual_bounds)


@pytest.mark.parametrize("splits", [2, 7, 64])
@pytest.mark.parametrize("case", [c for c in cases.DUALS if c[0] != DUAL_GATED and c[1] < 2000], ids=str)
def test_dual_product_in_pieces(hip_backend_session, case, splits):
    """More pieces than steps leave some empty; the sum over the pieces is the product."""
    kernel, arrays = cases.dual_case(*case, np.random.default_rng(17), splits=splits)
    whole = cases.kernel(OperatorSpec("DualMatMul", kernel.spec.ints[:2] + (1,)), arrays)
    want = ref.evaluate(whole, cases.flat(arrays))
    for g, w, b in zip(launch(hip_backend_session, kernel, arrays), want, cases.dual_bounds(whole, arrays, want)):
        assert g.shape[0] == splits
        assert (np.abs(g.astype(np.float64).sum(0) - w) <= b + cases.U * np.abs(w)).all()


@pytest.mark.parametrize("rows", [4, 40, 300])
@pytest.mark.parametrize("mode", [DUAL_GATED, DUAL_SUM, DUAL_BOTH])
def test_dual_product_keeps_all_bits(hip_backend_session, mode, rows):
    """Products and sums that 32 bits hold exactly come out exactly: 12-bit whole numbers (every product of upper and
    middle parts counts), and 24-bit ones times powers of two (so does the lowest part)."""
    rng = np.random.default_rng(8)
    for wide in (False, True):
        kernel, arrays = cases.dual_case(mode, rows, 70, 96, ACTIVATIONS.index("relu"), rng)
        for i, a in enumerate(arrays):
            left = i < (2 if mode == DUAL_SUM else 1)
            a[:] = 0.0
            if left:  # one term per row
                a[np.arange(a.shape[0]), rng.integers(0, a.shape[1], a.shape[0])] = rng.integers(1, 1 << (24 if wide else 12), a.shape[0])
            else:
                a[:] = 2.0 ** rng.integers(-3, 4, a.shape) if wide else rng.integers(1, 1 << 12, a.shape)
        if mode == DUAL_SUM:
            arrays[1][:] = 0.0
        got = launch(hip_backend_session, kernel, arrays)
        want = ref.evaluate(kernel, cases.flat(arrays))
        for i, (g, w) in enumerate(zip(got, want)):
            if mode != DUAL_GATED or i > 0:
                assert np.array_equal(g.astype(np.float64), w)


def test_dual_product_with_elements_that_are_not_finite(hip_backend_session):
    """They reach the results that they take part in and no others."""
    for rows in (4, 200):
        kernel, arrays = cases.dual_case(DUAL_GATED, rows, 130, 70, 0, np.random.default_rng(9))
        clean = launch(hip_backend_session, kernel, arrays)
        arrays[0][2, 5] = np.inf
        arrays[1][7, 100] = np.nan
        got = launch(hip_backend_session, kernel, arrays)
        touched = [np.zeros((rows, 130), bool) for _ in range(3)]
        for t in touched:
            t[2] = True
        touched[0][:, 100] = touched[1][:, 100] = True
        for g, c, t in zip(got, clean, touched):
            assert np.array_equal(g[~t], c[~t])
        assert not np.isfinite(got[1][touched[1]]).any() and not np.isfinite(got[2][2]).any()


@pytest.mark.parametrize("act", range(len(ACTIVATIONS)))
@pytest.mark.parametrize("count", cases.GRAD_COUNTS, ids=str)
def test_gated_gradient(hip_backend_session, count, act):
    check(hip_backend_session, *cases.gated_grad_case(count, act, np.random.default_rng(10)), cases.gated_grad_bounds)


def _slices(arrays, at, rng):
    """The arrays at `at` as slices of larger ones: more heads, more elements per head, tokens behind them; returns the
    arrays and the views."""
    out, views = [], []
    for i, a in enumerate(arrays):
        if i not in at:
            out.append(a)
            views.append(Shape(a.shape).identity_view())
            continue
        b, t, h, d = a.shape
        whole = rng.standard_normal((b, t + 3, h + 2, d + 4)).astype(np.float32)
        whole[:, 2 : 2 + t, 1 : 1 + h, 4:] = a
        v = Shape(whole.shape).identity_view()
        out.append(whole)
        views.append(View(v.input_shape, (0, 2, 1, 4), Shape(a.shape).identity_view().mapping, Shape(a.shape)))
    return out, views


@pytest.mark.parametrize("case", [(2, 70, 70, 4, 2, 64, 20, 2, "both"), (2, 1, 300, 4, 2, 40, 0, 0, "both"), (1, 66, 66, 2, 1, 30, 9, 1, "none")], ids=str)
def test_strided_attention(hip_backend_session, case):
    """Queries, keys and values that are slices of larger arrays, and heads that lie before tokens."""
    rng = np.random.default_rng(11)
    kernel, arrays = cases.attention_case(*case, rng)
    dense = launch(hip_backend_session, kernel, arrays)
    sliced, views = _slices(arrays, (0, 1, 2), rng)
    for g, w in zip(launch(hip_backend_session, OperatorKernel(kernel.spec, tuple(views), kernel.results), sliced), dense):
        assert np.array_equal(g, w)
    turned = [np.ascontiguousarray(a.transpose(0, 2, 1, 3)) for a in arrays[:3]]
    views = [Shape(a.shape).identity_view().permute_axes([0, 2, 1, 3]) for a in turned] + views[3:]
    for g, w in zip(launch(hip_backend_session, OperatorKernel(kernel.spec, tuple(views), kernel.results), turned + arrays[3:]), dense):
        assert np.array_equal(g, w)
    for kernel, arrays in cases.attention_grad_cases(*case, rng):
        at = (0, 1, 2, 3, 4) if kernel.spec.name == "AttentionGradQuery" else (0, 1, 2, 3)
        dense = launch(hip_backend_session, kernel, arrays)
        sliced, views = _slices(arrays, at, rng)
        for g, w in zip(launch(hip_backend_session, OperatorKernel(kernel.spec, tuple(views), kernel.results), sliced), dense):
            assert np.array_equal(g, w)


@pytest.mark.parametrize("case", [(2, 5, 3, 64, 16, 0, 1, 1000, 1.0, 0), (1, 6, 2, 22, 5, 1, 2, 50, 1.0, 1)], ids=str)
def test_strided_rotary_and_norm(hip_backend_session, case):
    rng = np.random.default_rng(12)
    kernel, arrays = cases.rotary_case(*case, rng)
    dense = launch(hip_backend_session, kernel, arrays)
    sliced, views = _slices(arrays, (0,), rng)
    assert np.array_equal(launch(hip_backend_session, OperatorKernel(kernel.spec, tuple(views), kernel.results), sliced)[0], dense[0])
    for make in (cases.norm_case, cases.norm_grad_case):
        kernel, arrays = make(37, 50, True, rng)
        dense = launch(hip_backend_session, kernel, arrays)
        out, views = [], []
        for a in arrays:
            if a.ndim == 1:
                out.append(a)
                views.append(Shape(a.shape).identity_view())
                continue
            whole = rng.standard_normal((a.shape[0] + 1, a.shape[1] + 3)).astype(np.float32)
            whole[1:, 2:-1] = a
            v = Shape(a.shape).identity_view()
            out.append(whole)
            views.append(View(Shape(whole.shape), (1, 2), v.mapping, v.output_shape))
        for g, w in zip(launch(hip_backend_session, OperatorKernel(kernel.spec, tuple(views), kernel.results), out), dense):
            # (rows that are no longer 16-byte aligned are summed in another order)
            assert rel_l2(g, w) <= 64 * cases.U


@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 2, 5, 8), (2, 7, 9, 130), (4, 1, 33, 64)], ids=str)
def test_cache_append(hip_backend_session, shape):
    """Rows replace what the cache holds; those past the capacity are dropped, the others untouched."""
    batch, tokens, capacity, width = shape
    rng = np.random.default_rng(19)
    rows, cache = cases.normal(rng, batch, tokens, width), cases.normal(rng, batch, capacity, width)
    start = rng.integers(0, capacity + 1, batch).astype(np.uint32)
    start[0] = 0xFFFFFFFF if batch > 2 else 0
    whole = rng.standard_normal((batch, tokens, width + 4)).astype(np.float32)
    whole[:, :, 4:] = rows
    dense = Shape(rows.shape).identity_view()
    sliced = View(Shape(whole.shape), (0, 0, 4), dense.mapping, dense.output_shape)
    be = hip_backend_session
    for array, view in ((rows, dense), (whole, sliced)):
        kernel = OperatorKernel(OperatorSpec("CacheAppend", (capacity,)), (view, Shape((batch,)).identity_view()), (0,))
        handles = []
        for a in cases.flat([array, start, cache]):
            handles.append(be.alloc(a.nbytes))
            be.write(handles[-1], 0, a)
        be.launch(kernel, handles, 0)
        got = np.frombuffer(be.read(handles[2], 0, cache.nbytes), np.float32)
        want = cache.reshape(-1).copy()
        ref.append(kernel, *cases.flat([array, start]), want)
        assert np.array_equal(got, want)
        for h in handles:
            be.free(h)


@pytest.mark.parametrize("tokens,keys", [(70, 70), (1, 300), (3, 90)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_masked_elements_take_no_part(hip_backend_session, tokens, keys, value):
    """What a row does not see does not reach it, whatever it holds: keys past the length, outside the window, ahead."""
    rng = np.random.default_rng(13)
    case = (2, tokens, keys, 4, 2, 64, 20, 2, "both")
    kernel, arrays = cases.attention_case(*case, rng)
    start, length = arrays[3:]
    start[:] = [keys - tokens, max(0, keys - tokens - 9)]
    length[:] = [keys, keys - 5]
    bad = 40 if tokens > 3 else keys - tokens - 21  # one that some rows see, or none
    before = launch(hip_backend_session, kernel, arrays)
    arrays[1][:, bad] = arrays[2][:, bad] = value
    arrays[1][1, keys - 5 :] = arrays[2][1, keys - 5 :] = value
    after = launch(hip_backend_session, kernel, arrays)
    for i in range(2):
        clean = ~ref.visible(tokens, keys, 20, 2, start[i], length[i])[:, bad]
        for b, a in zip(before, after):
            assert np.allclose(b[i][clean], a[i][clean], rtol=64 * cases.U, atol=64 * cases.U)
            assert clean.all() or not np.isfinite(a[i][~clean]).all()
    if tokens == 70:
        _masked_gradients(hip_backend_session, case, value)


def _masked_gradients(backend, case, value):
    rng = np.random.default_rng(14)
    (by_query, qa), (by_key, ka) = cases.attention_grad_cases(*case, rng)
    tokens, keys = case[1], case[2]
    start, length = qa[-2:]
    dq = launch(backend, by_query, qa)[0]
    qa[1][0, 40] = qa[2][0, 40] = value
    got = launch(backend, by_query, qa)[0]
    clean = ~ref.visible(tokens, keys, 20, 2, start[0], length[0])[:, 40]
    assert clean.any() and not clean.all()
    assert np.allclose(dq[0][clean], got[0][clean], rtol=256 * cases.U, atol=256 * cases.U)
    assert not np.isfinite(got[0][~clean]).all()
    want = launch(backend, by_key, ka)
    ka[0][0, 40] = ka[3][0, 40] = value  # a query row: the keys that it does not see stay clean
    got = launch(backend, by_key, ka)
    clean = ~ref.visible(tokens, keys, 20, 2, start[0], length[0])[40]
    assert clean.any() and not clean.all()
    for w, g in zip(want, got):
        assert np.allclose(w[0][clean], g[0][clean], rtol=256 * cases.U, atol=256 * cases.U)
        assert not np.isfinite(g[0][~clean]).all()


def _block(env, rng, **kw):
    from descent_amd import TransformerBlock

    block = TransformerBlock(env, 48, heads=4, n_hidden=72, groups=2, window=7, sinks=2, **kw)
    params = trainable(block)
    for p in params:
        env.reset_parameter(p, rng)
    env.write_parameter(block.norm_attention.weight, 1.0 + 0.1 * rng.standard_normal(48))
    return block, params


def trainable(module):
    from descent_amd import Module

    out = []
    for v in vars(module).values():
        if isinstance(v, Module):
            out += trainable(v)
        elif getattr(v, "reset_to", None) is not None:
            out.append(v)
    return out


def _train(env, batch, tokens, steps, fused=None):
    """Steps of a block under Adam on a padded batch; every parameter and the output afterwards."""
    from descent_amd import Adam

    rng = np.random.default_rng(15)
    block, params = _block(env, rng)
    x = env.static_parameter_with_data([batch, tokens, 48], "x", rng.standard_normal((batch, tokens, 48)))
    y = env.static_parameter_with_data([batch, tokens, 48], "y", rng.standard_normal((batch, tokens, 48)))
    length = env.static_parameter([batch], "length")
    env.write_parameter(length, np.array([tokens] + [tokens // 2] * (batch - 1), np.uint32))
    out = env.static_parameter([batch, tokens, 48], "out")
    scope = env.scope()
    z = block.eval(scope.parameter(x), None, scope.parameter_value(length).to_u32_bits())
    scope.write_parameter_value(out, z.value())
    loss = (z - scope.parameter(y)).square().reduce_sum(-1, False).reduce_sum(-1, True)
    loss.set_loss()
    Adam(env, scope, scope.trainable_parameters(), 0.01, 0.9, 0.99, 1e-8)
    graph = scope.build_graph()
    for i in range(steps):
        env.run(graph, i)
    return [env.read_parameter(p) for p in params] + [env.read_parameter(out)]


def test_block_trains_like_the_definitions(hip_backend_session):
    """One step's output, and its parameters after the step, against the same graph computed in 64 bits per node."""
    from descent_amd import Environment
    from oracle.cpu_backend import CpuBackend

    got, want = _train(Environment(hip_backend_session), 3, 21, 1), _train(Environment(CpuBackend()), 3, 21, 1)
    # the first step of Adam moves every element by the learning rate times the gradient's sign: the parameters agree
    # where the gradient is not within rounding of zero, the output everywhere
    for g, w in zip(got[:-1], want[:-1]):
        assert (np.abs(g - w) <= 1e-4).mean() >= 0.999
    assert rel_l2(got[-1], want[-1]) <= 1e-5


@pytest.mark.parametrize("fused", [True, False, "graph-replay"])
def test_block_steps_repeat_bit_for_bit(hip_backend_session, fused):
    """Several steps, launch by launch, fused and replayed as captured graphs: no atomics, so the same bits."""
    from descent_amd import Environment

    first = _train(Environment(hip_backend_session, fused=True), 2, 33, 6)
    again = _train(Environment(hip_backend_session, fused=fused), 2, 33, 6)
    for a, b in zip(first, again):
        assert np.isfinite(a).all()
        if fused is False:
            assert rel_l2(a, b) <= 1e-2  # other kernels sum the matrix products, and Adam divides by small gradients
        else:
            assert np.array_equal(a, b)


def test_block_serves_what_it_computes_whole(hip_backend_session):
    """Token by token and in chunks through the cache, against the whole sequence in one call."""
    from descent_amd import Environment

    env = Environment(hip_backend_session)
    rng = np.random.default_rng(16)
    block, _ = _block(env, rng)
    batch, tokens = 3, 40
    data = rng.standard_normal((batch, tokens, 48)).astype(np.float32)
    x, y = env.static_parameter_with_data(data.shape, "x", data), env.static_parameter(data.shape, "y")
    env.run(env.build_graph(lambda s: s.write_parameter_value(y, block.test(s.parameter(x)).value())), 0)
    whole = env.read_parameter(y)
    cache = block.attention.cache(env, batch, tokens + 2)
    start = env.static_parameter([batch], "start")
    graphs = {}
    for n in (5, 1):
        xt, yt = env.static_parameter([batch, n, 48], "xt"), env.static_parameter([batch, n, 48], "yt")
        graph = env.build_graph(
            lambda s: s.write_parameter_value(yt, block.step(s.parameter_value(xt), cache, s.parameter_value(start).to_u32_bits()))
        )
        graphs[n] = graph, xt, yt
    done = 0
    for n in [5] * 3 + [1] * 20 + [5]:
        graph, xt, yt = graphs[n]
        env.write_parameter(xt, data[:, done : done + n])
        env.write_parameter(start, np.full(batch, done, np.uint32))
        env.run(graph, 0)
        assert rel_l2(env.read_parameter(yt), whole[:, done : done + n]) <= 1e-5
        done += n
    assert done == tokens
    # the last five tokens once more: their slots are written again, the answer is the same
    again = graphs[5][2]
    last = env.read_parameter(again)
    env.run(graphs[5][0], 0)
    assert np.array_equal(env.read_parameter(again), last)
    # past the capacity nothing is written
    keys = env.read_parameter(cache.keys)
    graph, xt, yt = graphs[5]
    env.write_parameter(start, np.full(batch, tokens + 2, np.uint32))
    env.run(graph, 0)
    assert np.array_equal(env.read_parameter(cache.keys), keys)


def test_block_without_device_allocation(hip_backend_session):
    """run_static: intermediates in the library's scratch array, written parameters alternating with a spare buffer."""
    from descent_amd import Environment

    results = []
    for static in (False, True):
        env = Environment(hip_backend_session)
        rng = np.random.default_rng(20)
        block, _ = _block(env, rng)
        data = rng.standard_normal((2, 3, 48)).astype(np.float32)
        x, y = env.static_parameter_with_data(data.shape, "x", data), env.static_parameter(data.shape, "y")
        env.writer(y).zero_fill()
        start = env.static_parameter([2], "start")
        cache = block.attention.cache(env, 2, 20)
        graph = env.build_graph(lambda s: s.write_parameter_value(y, block.step(s.parameter_value(x), cache, s.parameter_value(start).to_u32_bits())))
        for done in (0, 3, 6):
            env.write_parameter(start, np.full(2, done, np.uint32))
            (env.run_static if static else env.run)(graph, 0)
        results.append([env.read_parameter(p) for p in (y, cache.keys, cache.values)])
    for a, b in zip(*results):
        assert np.isfinite(a).all() and np.array_equal(a, b)


def test_two_environments_at_once(hip_backend_session):
    """Two contexts with streams of their own, their runs interleaved."""
    from descent_amd import Environment
    from descent_amd.hip_backend import HipBackend

    other = HipBackend()
    try:
        envs = [Environment(hip_backend_session), Environment(other)]
        got = [_train(e, 2, 33, 3) for e in envs]
        for a, b in zip(*got):
            assert np.array_equal(a, b)
    finally:
        other.close()
