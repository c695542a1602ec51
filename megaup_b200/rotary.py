"""Rotary positions with several axes on head-parallel BSHD, SBHD and packed THD tensors.

This is the step between a peer-write projection, which delivers ``q`` and ``k``
with the whole sequence and a rank's share of the heads, and the attention
(``window_attention_*``). One launch turns both tensors; slices of a fused
projection may be passed as they are.

Pair ``p`` of a head belongs to one axis (time, height, width, ...) and turns by
``positions[axis, row] * frequency[p]`` radians: ``(x, y) -> (x cos - y sin,
x sin + y cos)``. BF16 in and out; the angle is reduced in 64 bits (positions of
millions keep their fraction of a turn), sine, cosine and the products are FP32,
each element is rounded once. The gradient is the rotation by minus the angle.
Kernel: ``csrc/mup_rotary.cu``.
"""

from __future__ import annotations

import ctypes
import math
import struct
from collections.abc import Sequence
from dataclasses import dataclass, field

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _native
from .attention import (
    _AXES, _check_heads_tensor, _current_stream, _dense_strides, _dispatch_modes, _is_compiled, _is_same, _is_traced,
    _refuse_tangents, _refuse_tracing, _row_strides, _rows_are_loadable, _share_elements, _span, _strides_are_loadable,
)
from .ops import _tensor_signature

_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_POSITIONS_LABEL = {"bshd": "[axes,S] or [axes,B,S]", "sbhd": "[axes,S] or [axes,S,B]", "thd": "[axes,T]"}


@dataclass(frozen=True)
class AxialRotary:
    """Frequencies of every pair, on the device; see ``prepare_axial_rotary``."""

    axis_dims: tuple[int, ...]
    theta: float
    interleaved: bool
    shared_frequencies: bool
    turns: Tensor
    pair_axis: Tensor
    plans: dict = field(default_factory=dict, init=False, repr=False, compare=False)

    def __getstate__(self) -> dict:
        return {**self.__dict__, "plans": {}}  # a copy has its own tables: kept blocks know these ones' addresses

    @property
    def pairs(self) -> int:
        return sum(self.axis_dims) // 2

    @property
    def device(self) -> torch.device:
        return self.turns.device


def prepare_axial_rotary(
    axis_dims: Sequence[int],
    *,
    theta: float = 10000.0,
    interleaved: bool = True,
    shared_frequencies: bool = False,
    device: torch.device | str,
) -> AxialRotary:
    """Frequencies for heads whose first ``sum(axis_dims)`` elements are turned, the
    pairs of axis 0 first, ``axis_dims[a]`` (even) elements for axis ``a``; the
    elements behind them stay as they are. Build once and use for every layer.

    ``interleaved``: pairs are neighbours ``(2p, 2p + 1)``; otherwise ``(p, p +
    sum / 2)``, and ``sum`` must be a multiple of 16. ``shared_frequencies``: pair
    ``p`` of the head turns with ``theta ** (-2p / sum)``; otherwise every axis has
    a row of its own, ``theta ** (-2i / axis_dims[a])`` for its pair ``i``.
    """

    dims = tuple(int(d) for d in axis_dims)
    if not dims or min(dims) <= 0 or any(d % 2 for d in dims):
        raise ValueError(f"axis_dims must be positive even numbers, got {tuple(axis_dims)}")
    total = sum(dims)
    if total > 256:
        raise ValueError(f"at most 256 elements of a head can be turned, got {total}")
    if not interleaved and total % 16:
        raise ValueError(f"rotated halves need sum(axis_dims) to be a multiple of 16, got {total}")
    theta = float(theta)
    if not (0.0 < theta < math.inf):
        raise ValueError(f"theta must be positive and finite, got {theta}")
    exponents = (
        [2 * p / total for p in range(total // 2)]
        if shared_frequencies
        else [2 * i / d for d in dims for i in range(d // 2)]
    )
    turns = [theta**-e / (2.0 * math.pi) for e in exponents]
    axis = [a for a, d in enumerate(dims) for _ in range(d // 2)]
    # one copy to the device
    packed = struct.pack(f"={len(turns)}d{len(axis)}i", *turns, *axis)
    both = torch.frombuffer(bytearray(packed), dtype=torch.uint8).to(device, copy=True)
    return AxialRotary(
        axis_dims=dims,
        theta=theta,
        interleaved=bool(interleaved),
        shared_frequencies=bool(shared_frequencies),
        turns=both[: 8 * len(turns)].view(torch.float64),
        pair_axis=both[8 * len(turns) :].view(torch.int32),
    )


def _check(kind: str, q: Tensor, k: Tensor | None, rotary: AxialRotary, positions: object) -> None:
    _check_heads_tensor(q, "q", kind, None)
    batch_axis, row_axis, _ = _AXES[kind]
    head_dim = q.shape[-1]
    if head_dim % 8 or head_dim > 256 or 2 * rotary.pairs > head_dim:
        raise ValueError(
            f"head_dim must be a multiple of 8 up to 256 and hold the {2 * rotary.pairs} turned elements, got {head_dim}"
        )
    if k is not None:
        _check_heads_tensor(k, "k", kind, q.device)
        if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != head_dim:
            raise ValueError(f"q and k must differ in their heads only, got {tuple(q.shape)} and {tuple(k.shape)}")
    for name, tensor in (("q", q), ("k", k)):
        if tensor is not None and not _strides_are_loadable(tensor):
            raise ValueError(
                f"{name} must have contiguous heads at positive strides of whole 16 bytes, got strides "
                f"{tensor.stride()}; pass {name}.contiguous()"
            )
    if rotary.device != q.device:
        raise ValueError(f"rotary lives on {rotary.device}, q on {q.device}")
    axes, rows = len(rotary.axis_dims), int(q.shape[row_axis])
    shapes = [(axes, rows)]
    if batch_axis is not None:
        shapes.append((axes, *q.shape[:2]))
    if (
        not isinstance(positions, Tensor)
        or positions.dtype not in _POSITION_TYPES
        or positions.device != q.device
        or tuple(positions.shape) not in shapes
    ):
        raise ValueError(
            f"positions must be int32, int64 or float32 {_POSITIONS_LABEL[kind]} on {q.device}, here "
            f"{' or '.join(map(str, shapes))}, got {_tensor_signature(positions)}"
        )


def _check_outputs(out: object, tensors: Sequence[Tensor], spans: Sequence[int]) -> None:
    if not isinstance(out, Sequence) or len(out) != len(tensors):
        raise ValueError(f"out must hold {len(tensors)} tensors")
    out_spans = list(spans)
    for i, (given, x) in enumerate(zip(out, tensors)):
        if given is x:
            continue
        if not isinstance(given, Tensor) or given.shape != x.shape or given.dtype != x.dtype or given.device != x.device:
            raise ValueError(f"out must be BF16 {tuple(x.shape)} on {x.device}, got {_tensor_signature(given)}")
        if not _rows_are_loadable(given):
            raise ValueError(f"out must have contiguous heads at 16-byte aligned strides, got {given.stride()}")
        out_spans[i] = _span(given)
        if _share_elements(given, out_spans[i], x, spans[i]) and not _is_same(given, x):
            raise ValueError("an output may be its own input, and must not overlap it otherwise")
    if len(out) == 2:
        (a, b), (q, k) = out, tensors
        if (
            _share_elements(a, out_spans[0], b, out_spans[1])
            or (b is not k and _share_elements(a, out_spans[0], k, spans[1]))
            or (a is not q and _share_elements(b, out_spans[1], q, spans[0]))
        ):
            raise ValueError("an output must not overlap the other one or its input")


def _block(kind: str, tensors: Sequence[Tensor], rotary: AxialRotary, positions: Tensor) -> bytes:
    """The argument block of a call without its tensors' addresses, the outputs dense."""

    a = _native.MupAxialRotary()
    x = tensors[0]
    batch_axis, row_axis, head_axis = _AXES[kind]
    a.device = x.device.index
    a.batch = 1 if batch_axis is None else x.shape[batch_axis]
    a.rows, a.head_dim = x.shape[row_axis], x.shape[-1]
    a.pairs, a.axes, a.interleaved = rotary.pairs, len(rotary.axis_dims), rotary.interleaved
    n = len(tensors)
    a.heads[:n] = [t.shape[head_axis] for t in tensors]
    a.x_strides[: 3 * n] = [s for t in tensors for s in _row_strides(t.shape, t.stride(), kind)]
    a.y_strides[: 3 * n] = [s for t in tensors for s in _row_strides(t.shape, _dense_strides(t.shape), kind)]
    strides = positions.stride()
    if positions.ndim == 2:
        a.pos_strides[:] = (strides[0], 0, strides[1])
    else:
        a.pos_strides[:] = (strides[0], strides[1 + batch_axis], strides[1 + row_axis])
    a.position_type = _POSITION_TYPES[positions.dtype]
    a.turns, a.pair_axis = rotary.turns.data_ptr(), rotary.pair_axis.data_ptr()
    return bytes(a)


def _turn(
    block: bytes, kind: str, tensors: Sequence[Tensor], outputs: Sequence[Tensor], positions: Tensor, inverse: bool,
    *, dense: bool = True,
) -> None:
    a = _native.MupAxialRotary.from_buffer_copy(block)
    a.q, a.q_out = address, _ = tensors[0].data_ptr(), outputs[0].data_ptr()
    if len(tensors) == 2:
        a.k, a.k_out = other, _ = tensors[1].data_ptr(), outputs[1].data_ptr()
        address |= other
    if address % 16:
        raise ValueError("q and k must be 16-byte aligned, got addresses " + ", ".join(hex(t.data_ptr()) for t in tensors))
    if not dense:
        a.y_strides[: 3 * len(outputs)] = [s for t in outputs for s in _row_strides(t.shape, t.stride(), kind)]
    a.positions, a.inverse = positions.data_ptr(), inverse
    _native.call("mup_axial_rotary_launch", ctypes.byref(a), _current_stream(a.device))


def _fresh(tensors: Sequence[Tensor]) -> list[Tensor]:
    return [torch.empty_like(t, memory_format=torch.contiguous_format) for t in tensors]


class _AxialRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, block, kind, rotary, positions, *tensors):
        outputs = _fresh(tensors)
        _turn(block, kind, tensors, outputs, positions, False)
        ctx.kind, ctx.rotary = kind, rotary
        ctx.save_for_backward(positions)
        return tuple(outputs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        if forward_ad._current_level >= 0:
            _refuse_tangents("the gradient of axial_rotary", *grads)
        # a broadcast or transposed gradient is laid out first
        grads = [g if _rows_are_loadable(g) else g.clone(memory_format=torch.contiguous_format) for g in grads]
        outputs = _fresh(grads)
        block, _ = _plan(ctx.kind, grads, ctx.rotary, positions)
        _turn(block, ctx.kind, grads, outputs, positions, True)
        return (None, None, None, None, *outputs)


_MAX_PLANS = 512


def _plan(
    kind: str, tensors: Sequence[Tensor | None], rotary: AxialRotary, positions: Tensor
) -> tuple[bytes, list[int]]:
    """The checked argument block of a call and its tensors' spans, kept per set of shapes and strides."""

    try:
        q = tensors[0]
        key = (kind, positions.shape, positions.stride(), positions.dtype, positions.device,
               q.shape, q.stride(), q.dtype, q.device)
        if len(tensors) == 2:
            k = tensors[1]
            key += (k.shape, k.stride(), k.dtype, k.device)
        return rotary.plans[key]
    except (KeyError, AttributeError):  # new, not a tensor
        _check(kind, tensors[0], tensors[1] if len(tensors) > 1 else None, rotary, positions)
    if len(rotary.plans) >= _MAX_PLANS:
        rotary.plans.clear()
    plan = rotary.plans[key] = _block(kind, tensors, rotary, positions), [_span(x) for x in tensors]
    return plan


def _rotate(kind: str, q: Tensor, k: Tensor | None, rotary: AxialRotary, positions: Tensor, out: object):
    if _is_compiled():  # see window_attention: run as it is, at a graph break
        return torch.compiler.disable(_rotate)(kind, q, k, rotary, positions, out)
    if not isinstance(rotary, AxialRotary):
        raise TypeError("rotary must be an AxialRotary from prepare_axial_rotary")
    tensors = (q,) if k is None else (q, k)
    block, spans = _plan(kind, tensors, rotary, positions)
    if forward_ad._current_level >= 0:
        _refuse_tangents(f"axial_rotary_{kind}", *tensors, positions, *(out if isinstance(out, Sequence) else ()))
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if out is not None:
            raise ValueError("out cannot be given when a gradient is wanted")
        if _dispatch_modes():
            _refuse_tracing(f"axial_rotary_{kind}", is_a_node=True)
        outputs = _AxialRotary.apply(block, kind, rotary, positions, *tensors)
    else:
        if _dispatch_modes() or _is_traced():
            _refuse_tracing(f"axial_rotary_{kind}", is_a_node=False)
        if out is None:
            outputs = _fresh(tensors)
        else:
            _check_outputs(out, tensors, spans)
            if torch.is_grad_enabled() and any(x.requires_grad for x in out):
                raise ValueError("out cannot be given when a gradient is wanted")
            outputs = out
            increment_version(outputs)  # autograd refuses a graph that had saved them
        _turn(block, kind, tensors, outputs, positions, False, dense=out is None)
    return outputs[0], outputs[1] if k is not None else None


def axial_rotary_bshd(
    q: Tensor,
    k: Tensor | None,
    rotary: AxialRotary,
    positions: Tensor,
    *,
    out: tuple[Tensor, ...] | None = None,
) -> tuple[Tensor, Tensor | None]:
    """Turn ``q [B,S,H,D]`` and, unless ``None``, ``k [B,S,Hkv,D]`` by their positions;
    returns both.

    ``positions`` (int32, int64 or float32 on the device) are ``[axes,S]``, shared
    by the batch, or ``[axes,B,S]``. ``out``: tensors of the same shapes to write;
    each may be its own input and overlaps no input otherwise. Differentiable in ``q`` and ``k``, once and in reverse
    mode; ``positions`` get no gradient.
    """

    return _rotate("bshd", q, k, rotary, positions, out)


def axial_rotary_sbhd(
    q: Tensor,
    k: Tensor | None,
    rotary: AxialRotary,
    positions: Tensor,
    *,
    out: tuple[Tensor, ...] | None = None,
) -> tuple[Tensor, Tensor | None]:
    """Sequence-first variant: ``q [S,B,H,D]``, ``positions [axes,S]`` or ``[axes,S,B]``."""

    return _rotate("sbhd", q, k, rotary, positions, out)


def axial_rotary_thd(
    q: Tensor,
    k: Tensor | None,
    rotary: AxialRotary,
    positions: Tensor,
    *,
    out: tuple[Tensor, ...] | None = None,
) -> tuple[Tensor, Tensor | None]:
    """Packed variant: ``q [T,H,D]``, ``positions [axes,T]``."""

    return _rotate("thd", q, k, rotary, positions, out)
