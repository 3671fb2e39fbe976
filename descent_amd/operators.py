"""Operators of sequence models: what each takes, what it leaves, and which views of an operand it reads in place.

An operator is one op node (`Op("Operator", spec)`) and one kernel.  The node stands for the operator's first result;
further results are `Op("Result", i)` nodes whose one argument is the operator's node, and a result that nothing reads
is not computed.  The kernels behind the specs are in csrc/kernels (rms_norm.inc, rotary.inc, attention.inc,
dual_matmul.inc); none of them has a counterpart in the reference, whose sequence model is the unrolled LSTM cell
(src/module.rs:281-363).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Tuple

import numpy as np

from .shape import Shape, View

# kinds, in the order of dsc_kernel_kind from DSC_KERNEL_RMS_NORM on
OPERATORS = (
    "RmsNorm", "RmsNormGrad", "Rotary", "Attention", "AttentionJoin", "AttentionGradQuery", "AttentionGradKeyValue",
    "DualMatMul", "GatedGrad", "AttentionGradSinks", "CacheAppend",
)
ACTIVATIONS = ("silu", "gelu", "relu", "sigmoid")
LAYOUTS = ("half", "interleaved")
DUAL_GATED, DUAL_SUM, DUAL_BOTH = range(3)
MAX_HEAD_DIM = 256


@dataclass(frozen=True)
class OperatorSpec:
    """`ints` and `floats` are the scalar attributes in the order of dsc_kernel_desc.op_int / op_float:

    RmsNorm                ints (has_residual,)                          floats (epsilon,)
    RmsNormGrad            ints (has_sum_grad, partials)
    Rotary                 ints (layout, inverse, positions rank)        floats (magnitude,)
    Attention              ints (window, sinks, 1 start | 2 length, splits)   floats (scale,)
    AttentionJoin          -
    AttentionGradQuery     ints (window, sinks, 1 start | 2 length)      floats (scale,)
    AttentionGradSinks, AttentionGradKeyValue   the same and pieces
    DualMatMul             ints (mode, activation, splits)
    GatedGrad              ints (activation,)
    CacheAppend            ints (capacity,); the node's operand 0 is the cache, taken over in place
    """

    name: str
    ints: Tuple[int, ...] = ()
    floats: Tuple[float, ...] = ()

    def __str__(self):
        return self.name

    def result_shapes(self, shapes: List[Shape]) -> List[Shape]:
        """Shapes of all results, from the operands' shapes."""
        name = self.name
        if name == "RmsNorm":
            rows, n = shapes[0]
            return [Shape((rows, n)), Shape((rows, n)), Shape((rows,))]
        if name == "RmsNormGrad":
            rows, n = shapes[0]
            return [Shape((rows, n)), Shape((self.ints[1], n))]
        if name == "Rotary":
            return [shapes[0]]
        if name == "Attention":
            b, t, h, d = shapes[0]
            splits = self.ints[3]
            if splits == 1:
                return [shapes[0], Shape((b, t, h))]
            return [Shape((splits, b, t, h, d)), Shape((splits, b, t, h))]
        if name == "AttentionJoin":
            return [Shape(shapes[0][1:]), Shape(shapes[1][1:])]
        if name == "AttentionGradQuery":
            return [shapes[0], Shape(shapes[0][:3])]
        if name == "AttentionGradSinks":
            b, keys, groups, dim = shapes[1]
            return [Shape((self.ints[3], b, min(self.ints[1], keys), groups, dim))] * 2
        if name == "AttentionGradKeyValue":
            return [shapes[1], shapes[2]]
        if name == "DualMatMul":
            mode, _, splits = self.ints
            out = Shape(((splits,) if splits > 1 else ()) + (shapes[0][0], shapes[-1][1]))
            return {DUAL_GATED: [out] * 3, DUAL_SUM: [out], DUAL_BOTH: [out] * 2}[mode]
        if name == "CacheAppend":
            return [Shape((shapes[-2][0], self.ints[0], shapes[-2][2]))]
        assert name == "GatedGrad"
        return [shapes[0], shapes[0]]

    def operand_kind(self, arg: int) -> str:
        """How freely an operand may be strided: "rows" (any strides, elements of the last axis side by side), "matrix"
        (elements of one of the two axes side by side) or "dense"."""
        name = self.name
        if name == "DualMatMul":
            return "matrix"
        if name == "Rotary":
            return "rows" if arg == 0 else "dense"
        if name == "CacheAppend":
            return "rows" if arg == 1 else "dense"
        if name == "Attention":
            return "rows" if arg < 3 else "dense"
        if name == "AttentionGradQuery":
            return "rows" if arg < 5 else "dense"
        if name in ("AttentionGradSinks", "AttentionGradKeyValue"):
            return "rows" if arg < 4 else "dense"
        if name in ("RmsNorm", "RmsNormGrad"):
            wide = {"RmsNorm": (0, 2), "RmsNormGrad": (0, 3, 4)}[name]
            return "rows" if arg in wide else "dense"
        return "dense"

    def reads_in_place(self, arg: int, view: View) -> bool:
        """Whether the kernel can read operand `arg` through `view`; if not, the view is copied out first."""
        if any(view.input_needs_clamp(axis) for axis in range(len(view.input_shape))):
            return False
        kind = self.operand_kind(arg)
        if kind == "dense":
            return view.is_contiguous()
        strides = view.input_shape.strides()
        steps = [0 if axis < 0 else strides[axis] * step for axis, step in view.mapping]
        if any(step < 0 for step in steps):
            return False

        def side_by_side(axis):
            return steps[axis] == 1 or view.output_shape[axis] == 1

        return side_by_side(-1) or (kind == "matrix" and side_by_side(-2))


@dataclass(frozen=True)
class OperatorKernel:
    """Kernel descriptor of an operator: the results it writes (indices into `spec.result_shapes`) follow its inputs in
    the binding order."""

    spec: OperatorSpec
    inputs: Tuple[View, ...]
    results: Tuple[int, ...]

    @property
    def shape(self) -> Shape:
        return self.result_shapes()[0]

    def result_shapes(self) -> List[Shape]:
        return self.spec.result_shapes([v.output_shape for v in self.inputs])

    def buffer_count(self):
        return len(self.inputs) + len(self.results)

    def group_count(self):
        return (self.shape.element_count() + 63) // 64

    def label_name(self):
        return f"{self.spec.name} {self.shape!r}"


def emit(arrays, spec: OperatorSpec, count: int):
    """Appends the operator's node with `arrays` as its operands, and nodes for its first `count` results."""
    from .array import Array
    from .graph import Op

    scope = arrays[0].scope
    for a in arrays:
        if a.scope is not scope:
            raise ValueError(f"{spec.name}: operands come from different scopes")
    # each operand goes through a view of its own: where the kernel can read that view it disappears again, where it
    # cannot (padding, a literal) it becomes the copy that the kernel reads
    operands = [a.view(a.shape.identity_view()) for a in arrays]
    shapes = spec.result_shapes([a.shape for a in operands])
    first = scope.ops.new_node(scope.colour, shapes[0], Op("Operator", spec), [a.node_id for a in operands])
    nodes = [first] + [scope.ops.new_node(scope.colour, shapes[i], Op("Result", i), [first]) for i in range(1, count)]
    return [Array(n, scope) for n in nodes]


def rotary_frequencies(dims: int, base: float = 10000.0, scale: float = 1.0, original: int = 0, slow: float = 1.0, fast: float = 32.0) -> np.ndarray:
    """The frequencies that rotate `dims` elements of a head: base^(-2 i / dims), as 32-bit floats.

    `scale` stretches a context to `scale` times the length that a model was trained on.  With `original` 0 every
    frequency is divided by it; with `original` the trained length, a frequency that turns fewer than `slow` times over
    that length is, one that turns more than `fast` times stays as it is, and those between change over linearly in the
    number of turns."""
    if dims < 0 or dims % 2 or base <= 0 or scale <= 0 or original < 0 or not 0 <= slow < fast:
        raise ValueError(f"rotary_frequencies: bad arguments {dims}, {base}, {scale}, {original}, {slow}, {fast}")
    table = float(base) ** (-np.arange(0, dims, 2, dtype=np.float64) / max(dims, 1))
    if original:
        turns = original * table / (2.0 * np.pi)
        kept = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        table = table * (kept + (1.0 - kept) / scale)
    else:
        table = table / scale
    return table.astype(np.float32)


# ------------------------------------------------------------------------------------------- checks of arguments


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def norm_spec(x: Shape, weight: Shape, epsilon: float, residual) -> OperatorSpec:
    _need(len(weight) == 1 and weight[0] == x[-1], f"rms_norm: weight {weight!r} does not fit the last axis of {x!r}")
    _need(residual is None or tuple(residual) == tuple(x), f"rms_norm: residual {residual!r} differs from {x!r}")
    _need(0.0 <= epsilon < float("inf"), f"rms_norm: epsilon must be finite and not negative, got {epsilon}")
    return OperatorSpec("RmsNorm", (int(residual is not None),), (float(epsilon),))


def norm_partials(rows: int) -> int:
    """Rows of partial weight gradients: one per workgroup of the gradient kernel, which then sums its share of the rows
    in registers.  512 workgroups keep two on each of the 256 CUs; fewer rows than that get one each."""
    return min(rows, 512)


def rotary_spec(x: Shape, frequencies: Shape, positions, layout: str, magnitude: float, inverse: bool) -> OperatorSpec:
    _need(len(x) == 4, f"rotary: needs [batch, tokens, heads, dim], got {x!r}")
    _need(len(frequencies) == 1 and 2 * frequencies[0] <= x[3],
          f"rotary: {frequencies!r} frequencies rotate twice as many elements, the heads of {x!r} have {x[3]}")
    _need(layout in LAYOUTS, f"rotary: layout must be one of {LAYOUTS}, got {layout!r}")
    _need(abs(magnitude) < float("inf"), f"rotary: magnitude must be finite, got {magnitude}")
    rank = 0
    if positions is not None:
        rank = len(positions)
        _need(tuple(positions) in ((x[0],), (x[0], x[1])),
              f"rotary: positions must be [{x[0]}] or [{x[0]}, {x[1]}], got {positions!r}")
    return OperatorSpec("Rotary", (LAYOUTS.index(layout), int(inverse), rank), (float(magnitude),))


def attention_ints(q: Shape, k: Shape, v: Shape, window, sinks: int, start, length) -> Tuple[int, int, int]:
    _need(len(q) == len(k) == len(v) == 4, "attention: needs [batch, tokens, heads, dim] queries, keys and values")
    _need(tuple(k) == tuple(v), f"attention: keys {k!r} and values {v!r} differ")
    _need(q[0] == k[0] and q[3] == k[3], f"attention: queries {q!r} and keys {k!r} differ in batch or head size")
    _need(q[2] % k[2] == 0, f"attention: {q[2]} query heads cannot share {k[2]} key heads evenly")
    _need(q[3] <= MAX_HEAD_DIM, f"attention: heads of at most {MAX_HEAD_DIM} elements, got {q[3]}")
    _need(window is None or 1 <= window < 1 << 31, f"attention: window must be at least 1, got {window}")
    _need(0 <= sinks < 1 << 31, f"attention: sinks must not be negative, got {sinks}")
    # (kernels count positions in 32 bits; offsets into the arrays are 64 bits wide)
    _need(k[1] < 1 << 30 and q[1] < 1 << 30, "attention: at most 2^30 tokens and keys")
    for name, a in (("start", start), ("length", length)):
        _need(a is None or tuple(a) == (q[0],), f"attention: {name} must be [{q[0]}]")
    _need(start is not None or q[1] <= k[1], f"attention: {q[1]} queries behind {k[1]} keys need `start`")
    has = (1 if start is not None else 0) | (2 if length is not None else 0)
    return (window or 0, min(sinks, k[1]) if window else 0, has)


def append_spec(cache: Shape, rows: Shape, start: Shape) -> OperatorSpec:
    _need(len(cache) == 3 and len(rows) == 3 and rows[0] == cache[0] and rows[2] == cache[2],
          f"cache_append: rows {rows!r} do not fit the cache {cache!r}")
    _need(tuple(start) == (cache[0],), f"cache_append: start must be [{cache[0]}], got {start!r}")
    return OperatorSpec("CacheAppend", (cache[1],))


def attention_splits(q: Shape, k: Shape, window, sinks: int) -> int:
    """Pieces that the keys of a call with few query rows are cut into.  A workgroup takes 16 rows (the queries of one
    sequence and key head, those of the group's heads side by side) and deals its keys in blocks of 16 to its four waves;
    with fewer than 512 workgroups -- two per CU -- the keys are split until there are as many, at 256 keys a piece or more."""
    batch, tokens, heads, _ = q
    groups = k[2]
    rows = tokens * (heads // groups)
    workgroups = batch * groups * ((rows + 15) // 16)
    if rows > 64:
        return 1
    reach = k[1] if window is None else min(k[1], window + sinks + tokens)
    return max(1, min(512 // workgroups, reach // 256, 64))


def sink_pieces(q: Shape, k: Shape, window, sinks: int) -> int:
    """Pieces of 256 rows that the rows beyond a window's length are cut into for the sinks' gradients (0: no kernel of
    their own, fewer than two pieces)."""
    if not window or not sinks:
        return 0
    rows = max(0, q[1] - window) * (q[2] // k[2])
    return 0 if rows <= 256 else min((rows + 255) // 256, 64)


def dual_matmul_shapes(x: Shape, w_gate: Shape, w_up: Shape, activation: str) -> None:
    _need(len(x) == 2, f"gated_dense: needs [rows, width], got {x!r}")
    _need(len(w_gate) == 2 and tuple(w_gate) == tuple(w_up) and w_gate[0] == x[1],
          f"gated_dense: weights {w_gate!r} and {w_up!r} must both be [{x[1]}, hidden]")
    _need(activation in ACTIVATIONS, f"gated_dense: activation must be one of {ACTIVATIONS}, got {activation!r}")


def dual_matmul_splits(rows: int, columns: int, k: int, mode: int) -> int:
    """Pieces of the k range of a gradient's product.  Where the result is small its tiles (128 rows by 128 columns, or 64
    of each of two products) are too few for 256 CUs: k is then cut into up to 8 pieces of 12 steps of 16 or more, until
    there are 384 workgroups, and a Reduce sums the pieces.  Measured: 1001 x 500 over k 2 x 1366 113 us whole, 27 in 8
    pieces; 500 x 1366 (two results) over k 1001 52 us whole, 31 in 4."""
    tiles = (rows + 127) // 128 * ((columns + 127) // 128 if mode == DUAL_SUM else (columns + 63) // 64)
    steps = (k + 15) // 16 * (2 if mode == DUAL_SUM else 1)
    return max(1, min(384 // tiles, steps // 12, 8))
