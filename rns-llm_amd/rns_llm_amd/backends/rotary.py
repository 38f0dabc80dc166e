"""Rotary positions of queries and keys.

``create_rotary`` settles the frequencies of a model's pairs once; ``rotate`` turns
queries and keys by their positions, forward and, under autograd, backward.  No counterpart in
the reference, which leaves positions to the model.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field
from fractions import Fraction
from typing import Sequence

import torch

from .. import _native
from .kv_cache import _FLOAT_CODES, _has_tangent

_POSITION_CODES = {torch.int32: _native.INT32, torch.int64: _native.INT64}
_MAX_CHECKED = 64
_PI = Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)


@dataclass(frozen=True)
class Rotary:
    """The frequencies of a head's pairs.  ``steps`` int64 ``[rotary_dim / 2]`` on the
    device: turns a position, in 2**-64 of a turn (modulo 2**64); ``frequencies``: the same
    in radians."""

    steps: torch.Tensor
    frequencies: tuple[float, ...]
    rotary_dim: int
    interleaved: bool
    magnitude: float
    device: torch.device
    _struct: object = field(repr=False, compare=False, default=None)
    _ref: int = field(repr=False, compare=False, default=0)
    # arguments that were checked: their types, shapes and strides -> what a call passes on
    _checked: dict = field(repr=False, compare=False, default_factory=dict)


class _Rotate(torch.autograd.Function):
    """The gradient turns back by the same angles, with the same magnitude; a tangent turns with its value."""

    @staticmethod
    def forward(ctx, backend, rotary, back, positions, q, k):
        ctx.backend, ctx.rotary, ctx.back = backend, rotary, back
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.set_materialize_grads(False)
        return backend._rotated(rotary, positions, q, k, back, False)

    @staticmethod
    def backward(ctx, gq, gk):
        positions, = ctx.saved_tensors
        first, second = (gq, gk) if gq is not None else (gk, None)
        if first is None:
            return (None,) * 6
        out = ctx.backend._turned(ctx.rotary, positions, first, second, not ctx.back)  # itself differentiated, it may be
        gq, gk = out if gq is not None else (None, out[0])
        return None, None, None, None, gq, gk

    @staticmethod
    def jvp(ctx, *tangents):
        positions, = ctx.saved_tensors
        return ctx.backend._turned(ctx.rotary, positions, tangents[4], None, ctx.back)


def _disjoint(x: torch.Tensor) -> bool:
    """Whether no two rows or heads of x share memory."""
    rows, heads, dim = x.shape
    inner, outer = sorted(((x.stride(0), rows), (x.stride(1), heads)))
    if rows <= 1 or heads <= 1:
        stride, n = (x.stride(0), rows) if heads <= 1 else (x.stride(1), heads)
        return n <= 1 or stride >= dim
    return inner[0] >= dim and outer[0] >= inner[0] * (inner[1] - 1) + dim


class RotaryOps:
    """The entry points, part of ``HipRNSBackend``."""

    def create_rotary(self, *, device: torch.device, rotary_dim: int, base: float = 10000.0, layout: str = "half",
                      scaling: str | None = None, factor: float = 1.0, original_length: int | None = None,
                      low_turns: float = 1.0, high_turns: float = 32.0, magnitude: float = 1.0,
                      frequencies: Sequence[float] | None = None) -> Rotary:
        """Pair i of ``rotary_dim / 2`` turns by ``base ** (-2 i / rotary_dim)`` radians a
        position.  ``layout``: "half" pairs value i with value i + rotary_dim / 2,
        "interleaved" value 2 i with 2 i + 1.

        For contexts longer than a model was trained on, ``scaling`` by ``factor``:
        "linear" divides every frequency; "base" raises the base so that the slowest pair
        is divided and the fastest stays; "bands" divides pairs that make at most
        ``low_turns`` turns in ``original_length`` tokens, keeps those of ``high_turns`` and
        more, and goes from one to the other linearly in the turns.  ``frequencies`` (radians a
        position) takes the place of all that.  ``magnitude`` multiplies the result."""
        rotary_dim = int(rotary_dim)
        if not 2 <= rotary_dim <= _native.ROTARY_MAX_DIM or rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even, 2 to {_native.ROTARY_MAX_DIM}")
        if layout not in ("half", "interleaved"):
            raise ValueError("layout must be 'half' or 'interleaved'")
        if not math.isfinite(ctypes.c_float(magnitude).value):  # as the library takes it
            raise ValueError("magnitude must be finite in float32")
        if frequencies is not None:
            if scaling is not None:
                raise ValueError("frequencies are given, nothing is left to scale")
            values = [float(f) for f in frequencies]
            if len(values) != rotary_dim // 2 or not all(map(math.isfinite, values)):
                raise ValueError(f"frequencies must be {rotary_dim // 2} finite numbers")
        else:
            try:
                values = self._frequencies(rotary_dim, float(base), scaling, float(factor), original_length, float(low_turns),
                                           float(high_turns))
            except (OverflowError, ZeroDivisionError):
                values = [math.inf]
            if not all(map(math.isfinite, values)):
                raise ValueError(f"base {base} and factor {factor} give frequencies that are not finite")
        turns = [round(Fraction(f) * 2 ** 64 / (2 * _PI)) % 2 ** 64 for f in values]
        steps = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)
        struct = _native.RotaryStruct(steps.data_ptr(), rotary_dim // 2, layout == "interleaved", float(magnitude))
        return Rotary(steps, tuple(values), rotary_dim, layout == "interleaved", float(magnitude), steps.device, struct,
                      ctypes.addressof(struct))

    @staticmethod
    def _frequencies(dim: int, base: float, scaling: str | None, factor: float, original: int | None, low: float,
                     high: float) -> list[float]:
        if not (base > 0 and math.isfinite(base)):
            raise ValueError("base must be positive and finite")
        if scaling not in (None, "linear", "base", "bands"):
            raise ValueError("scaling must be 'linear', 'base' or 'bands'")
        if scaling is None and factor != 1.0:
            raise ValueError("factor goes with scaling")
        if not (factor > 0 and math.isfinite(factor)):
            raise ValueError("factor must be positive and finite")
        if scaling == "base":
            if dim < 4:
                raise ValueError("one pair is the fastest and the slowest: 'base' needs rotary_dim 4 and more")
            base *= factor ** (dim / (dim - 2))
        values = [base ** (-2 * i / dim) for i in range(dim // 2)]
        if scaling == "linear":
            values = [f / factor for f in values]
        elif scaling == "bands":
            if original is None or original < 1 or not 0 <= low < high < math.inf:
                raise ValueError("'bands' needs original_length and 0 <= low_turns < high_turns")
            kept = [min(max((int(original) * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for f in values]
            values = [f * s + f / factor * (1.0 - s) for f, s in zip(values, kept)]
        return values

    def rotate(self, rotary: Rotary, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None, *,
               inplace: bool = False):
        """``q`` ``[rows, heads, head_dim]`` and ``k`` (as many rows, heads of its own) of any
        strides, their first ``rotary_dim`` values turned by ``positions`` (int32 or int64
        ``[rows]``, any value), in float32, rounded once, in one launch -> new tensors
        (or one, without k).  Angles are exact to 2**-32 of a turn up to position 2**32, beyond
        it to 2**-65 of a turn a position.
        ``inplace``: the tensors themselves, which share no value (and lie among each other at one
        row stride alone), are turned and returned, a change that autograd sees like that of any
        operation in place.

        Differentiable in q and k, backward and in forward mode, but for calls in place.  As with any backward pass, one is
        captured into a graph only when no eager pass's graph of the same leaves is alive."""
        if not inplace:
            out = self._turned(rotary, positions, q, k, False)
        elif _has_tangent(q, k) or torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad):
            raise ValueError("a call in place has no gradient: detach q and k, or call it under torch.no_grad()")
        else:
            out = self._rotated(rotary, positions, q, k, False, True)
            # torch has not seen the write, and an operation may have kept what was there
            torch.autograd.graph.increment_version((q,) if k is None else (q, k))
        return out if k is not None else out[0]

    def _turned(self, rotary: Rotary, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None, back: bool):
        """New tensors, with what autograd asks for."""
        if _has_tangent(q, k):  # each by itself, so that one without a tangent gets none
            return tuple(None if x is None else _Rotate.apply(self, rotary, back, positions, x, None)[0] for x in (q, k))
        if torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad):
            return _Rotate.apply(self, rotary, back, positions, q, k)
        return self._rotated(rotary, positions, q, k, back, False)

    def _rotated(self, rotary: Rotary, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None, back: bool, inplace: bool):
        key = (q.dtype, q.shape, q.stride(), q.device, None if k is None else (k.dtype, k.shape, k.stride(), k.device),
               positions.dtype, positions.shape, positions.stride(), positions.device, back, inplace)
        checked = rotary._checked.get(key)
        if checked is None:
            plain = [self._rotary_rows(rotary, x, name, inplace) for x, name in ((q, "q"), (k, "k")) if x is not None]
            if positions.dtype not in _POSITION_CODES or positions.device != rotary.device or positions.ndim != 1:
                raise ValueError(f"positions must be a 1-dimensional int32 or int64 tensor on {rotary.device}")
            if positions.shape[0] != q.shape[0] or (k is not None and (k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
                raise ValueError("positions, q and k must have one number of rows, q and k one head dimension")
            if k is not None and k.dtype != q.dtype:
                raise ValueError("q and k must have one dtype")
            if rotary.device.type != "cuda":
                raise ValueError(f"queries must be on the GPU, they are on {rotary.device}")
            if plain[0] is not q or plain[-1] is not (q if k is None else k) or not positions.is_contiguous():
                return self._rotated(rotary, positions.contiguous(), plain[0], None if k is None else plain[-1], back, inplace)
            checked = self._rotary_call(rotary, positions, q, k, back, inplace)
            if len(rotary._checked) >= _MAX_CHECKED:
                rotary._checked.clear()
            rotary._checked[key] = checked
        _, ref = checked
        if inplace:
            out = (q, k)
        else:
            out = (torch.empty_like(q, memory_format=torch.contiguous_format),
                   None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format))
        self._on_device(rotary.device, self._lib.rnsmx_rotate, rotary._ref, ref, positions.data_ptr(), q.data_ptr(),
                        None if k is None else k.data_ptr(), out[0].data_ptr(), None if k is None else out[1].data_ptr())
        self._stats["rotate_calls"] += 1
        return out

    @staticmethod
    def _rotary_rows(rotary: Rotary, x: torch.Tensor, name: str, inplace: bool) -> torch.Tensor:
        if x.dtype not in _FLOAT_CODES or x.device != rotary.device:
            raise ValueError(f"{name} must be float32, float16 or bfloat16 on {rotary.device}")
        if x.ndim != 3 or x.shape[2] < rotary.rotary_dim or x.shape[2] > _native.ROTARY_MAX_DIM:
            raise ValueError(f"{name} must be [rows, heads, {rotary.rotary_dim} to {_native.ROTARY_MAX_DIM}], got {tuple(x.shape)}")
        if inplace and x.numel() and not (x.stride(2) == 1 and _disjoint(x)):
            raise ValueError(f"{name} is turned in place: its values must lie apart, those of a head in a row")
        return x if x.stride(2) == 1 else x.contiguous()

    def _rotary_call(self, rotary: Rotary, positions, q, k, back: bool, inplace: bool):
        """The checked arguments as the library takes them."""
        strides, heads = [], []
        for x in (q, k):
            heads.append(0 if x is None else int(x.shape[1]))
            strides.append((0, 0) if x is None else x.stride()[:2])
        outs = strides if inplace else [(h * q.shape[2], q.shape[2]) for h in heads]
        rows = _native.RotaryRowsStruct(int(q.shape[0]), *strides[0], *strides[1], *outs[0], *outs[1], *heads, int(q.shape[2]),
                                        _FLOAT_CODES[q.dtype], _POSITION_CODES[positions.dtype], back)
        return rows, ctypes.addressof(rows)
