"""Layer building blocks; every one lowers to array ops.

Host-side mirror of src/module.rs (Dense :37-90, Conv2D :92-215, MaxPool2D
:217-224, MaxBlurPool2D :226-252, Dropout :254-279).  Images are NHWC, conv
filters are [groups, oc/groups, fh, fw, ic/groups], dense weights [in, out].
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

from .array import Array, DualArray, Parameter
from .operators import rotary_frequencies


@dataclass(frozen=True)
class Initializer:
    """src/parameter.rs:10-26"""

    kind: str  # "zero" | "constant" | "normal" | "uniform"
    scale: float = 0.0

    @staticmethod
    def zero():
        return Initializer("zero")

    @staticmethod
    def constant(value: float):
        """Beside the reference's: every element `value` (the weight of a norm starts at 1)."""
        return Initializer("constant", float(np.float32(value)))

    @staticmethod
    def rand_normal(scale: float):
        return Initializer("normal", float(np.float32(scale)))

    @staticmethod
    def rand_uniform(scale: float):
        return Initializer("uniform", float(np.float32(scale)))

    @staticmethod
    def for_relu(fan_in: int):
        return Initializer.rand_normal(float(np.sqrt(np.float32(2.0) / np.float32(fan_in))))

    @staticmethod
    def for_siren(fan_in: int, is_first_layer: bool):
        scale = np.sqrt(np.float32(6.0) / np.float32(fan_in)) * np.float32(30.0 if is_first_layer else 1.0)
        return Initializer.rand_uniform(float(scale))


@dataclass(frozen=True)
class EvalContext:
    is_training: bool


class Module:
    def eval(self, x: DualArray, ctx: EvalContext) -> DualArray:
        raise NotImplementedError

    def train(self, x: DualArray) -> DualArray:
        return self.eval(x, EvalContext(True))

    def test(self, x: DualArray) -> DualArray:
        return self.eval(x, EvalContext(False))


class Dense(Module):
    def __init__(self, env, n_in: int, n_out: int, w_initializer=None, b_initializer=None):
        self.w = env.trainable_parameter([n_in, n_out], "w", w_initializer or Initializer.for_relu(n_in))
        self.b = env.trainable_parameter([n_out], "b", b_initializer or Initializer.zero())

    def eval(self, x, ctx):
        return x.next_colour().matmul(self.w) + self.b


class Conv2D(Module):
    def __init__(self, env, in_channels, out_channels, filter_w, filter_h, pad=0, stride=(1, 1), groups=1,
                 is_blur=False):
        fic, foc = in_channels // groups, out_channels // groups
        if fic * groups != in_channels or foc * groups != out_channels:
            raise ValueError("channels not divisible by groups")
        shape = [groups, foc, filter_h, filter_w, fic]
        if is_blur:
            # fixed 3x3 binomial filter per channel (src/module.rs:141-167)
            assert [foc, filter_h, filter_w, fic] == [1, 3, 3, 1]
            self.f = env.static_parameter(shape, "f")
            self.b = env.static_parameter([out_channels], "b")
            taps = np.array([1, 2, 1, 2, 4, 2, 1, 2, 1], dtype=np.float32) / np.float32(16.0)
            env.write_parameter(self.f, np.tile(taps, groups))
            env.writer(self.b).zero_fill()
        else:
            self.f = env.trainable_parameter(shape, "f", Initializer.for_relu(filter_h * filter_w * fic))
            self.b = env.trainable_parameter([out_channels], "b", Initializer.zero())
        self.pad = pad
        self.stride = tuple(stride)

    def eval(self, x, ctx):
        return x.next_colour().conv2d(self.f, self.pad, self.stride) + self.b


class MaxPool2D(Module):
    def eval(self, x, ctx):
        return x.next_colour().max_pool2d((2, 2), (2, 2))


class MaxBlurPool2D(Module):
    def __init__(self, env, channels: int):
        self.blur = Conv2D(env, channels, channels, 3, 3, pad=1, stride=(2, 2), groups=channels, is_blur=True)

    def eval(self, x, ctx):
        return self.blur.eval(x.next_colour().max_pool2d((2, 2), (1, 1)), ctx)


class Dropout(Module):
    """Inverted dropout from the counter-based generator; forward and backward
    evaluate the same Rand node so the masks agree (src/module.rs:254-279)."""

    def __init__(self, amount: float):
        self.amount = amount

    def eval(self, x, ctx):
        if not ctx.is_training:
            return x
        scope = x.scope
        scope.next_colour()
        rv = scope.rand(x.shape).value()
        a, da = x.into_inner()
        survivor_scale = float(np.float32(1.0) / (np.float32(1.0) - np.float32(self.amount)))
        b, db = rv.select_gt(self.amount, survivor_scale * a, 0.0).with_empty_grad()
        da.accumulate(rv.select_gt(self.amount, survivor_scale * db, 0.0))
        return DualArray(b, db)


class LSTMCell(Module):
    """Unrolled over the time axis (-2) (src/module.rs:281-363)."""

    class _Weight:
        def __init__(self, env, prefix, n_in, n_out):
            self.input = env.trainable_parameter([n_in, n_out], f"{prefix}_wi", Initializer.rand_normal(0.01))
            self.hidden = env.trainable_parameter([n_out, n_out], f"{prefix}_wh", Initializer.rand_normal(0.01))
            self.bias = env.trainable_parameter([n_out], f"{prefix}_b", Initializer.zero())

        def eval(self, x, hidden):
            y = x.matmul(self.input)
            if hidden is not None:
                y = y + hidden.matmul(self.hidden)
            return y + self.bias

    def __init__(self, env, n_in, n_out):
        self.forget_gate = self._Weight(env, "forget", n_in, n_out)
        self.input_gate = self._Weight(env, "input", n_in, n_out)
        self.output_gate = self._Weight(env, "output", n_in, n_out)
        self.cell_input = self._Weight(env, "cell", n_in, n_out)

    def eval(self, x, ctx):
        steps = x.shape[-2]
        prev_cell = prev_hidden = None
        for i in range(steps):
            xi = x.next_colour().lock_axis(-2, i, False)
            input_gate = self.input_gate.eval(xi, prev_hidden).sigmoid()
            output_gate = self.output_gate.eval(xi, prev_hidden).sigmoid()
            cell_input = self.cell_input.eval(xi, prev_hidden).tanh()
            cell = input_gate * cell_input
            if prev_cell is not None:
                cell = cell + self.forget_gate.eval(xi, prev_hidden).sigmoid() * prev_cell
            prev_hidden = output_gate * cell.tanh()
            prev_cell = cell
        return prev_hidden


class RMSNorm(Module):
    """Root-mean-square norm over the last axis (no counterpart in the reference)."""

    def __init__(self, env, n: int, epsilon: float = 1e-6):
        self.weight = env.trainable_parameter([n], "weight", Initializer.constant(1.0))
        self.epsilon = epsilon

    def eval(self, x, ctx):
        x.scope.next_colour()
        return x.rms_norm(self.weight, self.epsilon)

    def add(self, x, residual):
        """(norm of x + residual, x + residual), for arrays with or without gradients."""
        x.scope.next_colour()
        return x.add_rms_norm(residual, self.weight, self.epsilon)


class GatedFeedForward(Module):
    """activation(x w_gate) * (x w_up), then w_down, on [rows, n] (no counterpart in the reference)."""

    def __init__(self, env, n: int, n_hidden: int, activation: str = "silu"):
        scale = Initializer.rand_normal(float(n) ** -0.5)
        self.w_gate = env.trainable_parameter([n, n_hidden], "w_gate", scale)
        self.w_up = env.trainable_parameter([n, n_hidden], "w_up", scale)
        self.w_down = env.trainable_parameter([n_hidden, n], "w_down", Initializer.rand_normal(float(n_hidden) ** -0.5))
        self.activation = activation

    def eval(self, x, ctx):
        x.scope.next_colour()
        return x.gated_dense(self.w_gate, self.w_up, self.activation).matmul(self.w_down)


class KeyValueCache:
    """Rotated keys and values of `batch` sequences of up to `capacity` tokens, as SelfAttention.step keeps them."""

    def __init__(self, env, batch: int, capacity: int, groups: int, head_dim: int):
        self.shape = [batch, capacity, groups, head_dim]
        self.keys = env.static_parameter(self.shape, "keys")
        self.values = env.static_parameter(self.shape, "values")
        for p in (self.keys, self.values):
            env.writer(p).zero_fill()

    def append(self, scope, parameter: Parameter, new: Array, start: Array) -> Array:
        """Writes new [batch, tokens, groups, dim] behind the `start` tokens that each sequence holds, in place, and
        returns the whole array.  Tokens past the capacity are dropped."""
        batch, capacity, groups, dim = self.shape
        if [new.shape[0], new.shape[2], new.shape[3]] != [batch, groups, dim]:
            raise ValueError(f"cache holds {parameter.shape!r}, got {new.shape!r}")
        old = scope.parameter_value(parameter).reshape([batch, capacity, groups * dim])
        whole = old.cache_append(new.reshape([batch, new.shape[1], groups * dim]), start).reshape(self.shape)
        scope.write_parameter_value(parameter, whole)
        return whole


class SelfAttention(Module):
    """Causal self-attention on [batch, tokens, n] with rotary positions, grouped key heads and, on request, a sliding
    window with sinks (no counterpart in the reference)."""

    def __init__(self, env, n: int, heads: int, groups=None, head_dim=None, window=None, sinks: int = 0, frequencies=None):
        self.heads, self.groups = heads, groups or heads
        self.head_dim = head_dim or n // heads
        self.window, self.sinks = window, sinks
        scale = Initializer.rand_normal(float(n) ** -0.5)
        self.w_query = env.trainable_parameter([n, heads * self.head_dim], "w_query", scale)
        self.w_key = env.trainable_parameter([n, self.groups * self.head_dim], "w_key", scale)
        self.w_value = env.trainable_parameter([n, self.groups * self.head_dim], "w_value", scale)
        self.w_out = env.trainable_parameter([heads * self.head_dim, n], "w_out", Initializer.rand_normal(float(heads * self.head_dim) ** -0.5))
        table = rotary_frequencies(self.head_dim // 2 * 2) if frequencies is None else np.asarray(frequencies, np.float32)
        self.frequencies = env.static_parameter_with_data([len(table)], "frequencies", table)

    def _heads(self, x, start):
        batch, tokens, n = x.shape
        x.scope.next_colour()
        rows = x.reshape([batch * tokens, n])
        q = rows.matmul(self.w_query).reshape([batch, tokens, self.heads, self.head_dim])
        k = rows.matmul(self.w_key).reshape([batch, tokens, self.groups, self.head_dim])
        v = rows.matmul(self.w_value).reshape([batch, tokens, self.groups, self.head_dim])
        return q.rotary(self.frequencies, start), k.rotary(self.frequencies, start), v

    def _out(self, y):
        batch, tokens, heads, dim = y.shape
        rows = y.reshape([batch * tokens, heads * dim]).matmul(self.w_out)
        return rows.reshape([batch, tokens, rows.shape[-1]])

    def eval(self, x, ctx, length=None):
        """`length`: u32 array [batch] of a padded batch's sequence lengths."""
        q, k, v = self._heads(x, None)
        return self._out(q.attention(k, v, self.window, self.sinks, length=length))

    def cache(self, env, batch: int, capacity: int) -> KeyValueCache:
        return KeyValueCache(env, batch, capacity, self.groups, self.head_dim)

    def step(self, x: Array, cache: KeyValueCache, start: Array) -> Array:
        """Serving: x [batch, tokens, n] holds the next tokens (usually one) of sequences that have `start` (u32 [batch])
        tokens in the cache; their keys and values are appended and they attend to all that precede them."""
        q, k, v = self._heads(x, start)
        keys = cache.append(x.scope, cache.keys, k, start)
        values = cache.append(x.scope, cache.values, v, start)
        return self._out(q.attention(keys, values, self.window, self.sinks, start=start))


class TransformerBlock(Module):
    """x + attention(norm(x)), then the same with the gated feed-forward, on [batch, tokens, n] (no counterpart in the
    reference)."""

    def __init__(self, env, n: int, heads: int, n_hidden: int, groups=None, head_dim=None, window=None, sinks: int = 0, activation: str = "silu"):
        self.norm_attention = RMSNorm(env, n)
        self.attention = SelfAttention(env, n, heads, groups, head_dim, window, sinks)
        self.norm_feed_forward = RMSNorm(env, n)
        self.feed_forward = GatedFeedForward(env, n, n_hidden, activation)

    def _feed_forward(self, x, attended, ctx):
        y, total = self.norm_feed_forward.add(attended, x)
        n = y.shape[-1]
        return self.feed_forward.eval(y.reshape([y.shape[0] * y.shape[1], n]), ctx).reshape(y.shape) + total

    def eval(self, x, ctx, length=None):
        return self._feed_forward(x, self.attention.eval(self.norm_attention.eval(x, ctx), ctx, length), ctx)

    def step(self, x: Array, cache: KeyValueCache, start: Array) -> Array:
        ctx = EvalContext(False)
        return self._feed_forward(x, self.attention.step(self.norm_attention.eval(x, ctx), cache, start), ctx)
