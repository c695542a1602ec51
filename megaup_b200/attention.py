"""Sliding-window attention with sinks on head-parallel BSHD, SBHD and packed THD tensors.

This is the step between the two exchange GEMMs: a peer-write projection
delivers ``q``, ``k`` and ``v`` with the whole sequence and a rank's share of
the heads, a head-shard pull projection takes the result. No communication and
no runtime is involved.

Row ``i`` of a sequence with ``Lq`` queries and ``Lk`` keys stands at position
``at = i + Lk - Lq`` (new tokens at the end of a cache) and sees key ``j`` when

* ``j < Lk`` and, with ``causal``, ``j <= at``, and
* ``j < sinks`` or ``at - left <= j <= at + right``.

``out = softmax(scale * q k^T) v`` over the visible keys, query head ``h`` using
key/value head ``h // (heads_q // heads_kv)``. A row that sees no key gets 0. A
key that no query row sees and a row that sees no key have no influence and the
gradient 0, whatever they hold; an infinity or NaN in a key or value row that
some query sees may reach the other rows of the same block of queries (backward:
one in a row of the gradient or a query the other keys of a block of keys).

BF16 in and out, FP32 sums, one rounding of the probabilities (and, backward,
of the score gradients) to BF16 for the second product and one of the results.
The gradient is deterministic. Kernels: ``csrc/mup_attn_*.cuh``.
"""

from __future__ import annotations

import array
import ctypes
import math
from collections.abc import Sequence
from dataclasses import dataclass, field
from functools import lru_cache
from itertools import chain
from operator import itemgetter

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _native
from .ops import _INPUT_LABEL, _normalize_cu_seqlens, _tensor_signature
from .runtime import _KERNEL_TIMEOUT_NS

# index of {sequence of the batch, row, head} in a tensor of each layout (None: no such dimension)
_AXES = {"bshd": (0, 1, 2), "sbhd": (1, 0, 2), "thd": (None, 0, 1)}
_MAX_LENGTH = 1 << 29


# --------------------------------------------------------------------------- packed sequences


@dataclass(frozen=True)
class PackedSequences:
    """Boundaries of packed sequences and the row blocks the kernels walk, on the
    device. Built once per step by ``prepare_packed_sequences`` and used for every layer."""

    cu_seqlens_q: tuple[int, ...]
    cu_seqlens_k: tuple[int, ...]
    sequences: Tensor
    q_blocks_256: Tensor
    q_blocks_128: Tensor
    k_blocks_128: Tensor
    longest_q: int
    longest_k: int
    plans: dict = field(default_factory=dict, init=False, repr=False, compare=False)

    def __getstate__(self) -> dict:
        return {**self.__dict__, "plans": {}}  # a copy has its own tables: kept plans know these ones' addresses

    @property
    def num_sequences(self) -> int:
        return len(self.cu_seqlens_q) - 1

    @property
    def device(self) -> torch.device:
        return self.sequences.device


def _blocks(table: list[tuple[int, int, int, int]], lengths: list[int]) -> list[tuple[int, ...]]:
    """(sequence, first row, the sequence's entry of ``table``, 0, 0) of every block of
    128 rows, the last rows first: under a causal mask they have the most keys."""

    blocks = [
        (s, r, *entry, 0, 0) for s, (entry, length) in enumerate(zip(table, lengths)) for r in range(0, length, 128)
    ]
    blocks.sort(key=itemgetter(1), reverse=True)
    return blocks


def prepare_packed_sequences(
    cu_seqlens_q: Tensor | Sequence[int],
    cu_seqlens_k: Tensor | Sequence[int] | None = None,
    *,
    device: torch.device | str,
) -> PackedSequences:
    """Describe packed sequences to ``window_attention_thd``.

    ``cu_seqlens_q`` are the boundaries of the query rows, ``cu_seqlens_k`` those
    of the key rows (default: the same). For the split-sample scheme pass
    ``THDLayout.cu_seqlens_out``. A CUDA tensor is synchronised to the host here.
    """

    cu_q = _normalize_cu_seqlens(cu_seqlens_q)
    cu_k = cu_q if cu_seqlens_k is None else _normalize_cu_seqlens(cu_seqlens_k)
    if len(cu_q) != len(cu_k):
        raise ValueError(f"cu_seqlens_q describes {len(cu_q) - 1} sequences, cu_seqlens_k {len(cu_k) - 1}")
    if max(cu_q[-1], cu_k[-1]) > _MAX_LENGTH:
        raise ValueError(f"at most {_MAX_LENGTH} rows, got {max(cu_q[-1], cu_k[-1])}")
    queries = [b - a for a, b in zip(cu_q, cu_q[1:])]
    keys = [b - a for a, b in zip(cu_k, cu_k[1:])]
    table = [(a, n, b, m) for a, n, b, m in zip(cu_q, queries, cu_k, keys)]

    # one copy to the device; entries of 8 numbers start at multiples of 32 bytes
    q_blocks = _blocks(table, queries)
    parts = {
        "q_blocks_256": [block for block in q_blocks if block[1] % 256 == 0],
        "q_blocks_128": q_blocks,
        "k_blocks_128": (q_blocks if keys == queries else _blocks(table, keys))[::-1],
        "sequences": table,
    }
    flat = array.array("i", chain.from_iterable(chain.from_iterable(parts.values())))
    everything = torch.frombuffer(flat, dtype=torch.int32).to(device, copy=True)
    tables, start = {}, 0
    for name, rows in parts.items():
        width = 4 if name == "sequences" else 8
        tables[name] = everything[start : start + len(rows) * width].view(len(rows), width)
        start += len(rows) * width
    return PackedSequences(
        cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, longest_q=max(queries), longest_k=max(keys), **tables
    )


# --------------------------------------------------------------------------- validation


def _check_heads_tensor(tensor: object, name: str, kind: str, device: torch.device | None) -> None:
    if not isinstance(tensor, Tensor) or tensor.ndim != len(_INPUT_LABEL[kind].split(",")):
        raise ValueError(f"{name} must be {_INPUT_LABEL[kind]}, got {_tensor_signature(tensor)}")
    if tensor.dtype != torch.bfloat16 or not tensor.is_cuda or (device is not None and tensor.device != device):
        raise ValueError(f"{name} must be BF16 on one CUDA device, got {tensor.dtype} on {tensor.device}")
    if min(tensor.shape) <= 0:
        raise ValueError(f"all dimensions of {name} must be positive, got {tuple(tensor.shape)}")


def _strides_are_loadable(tensor: Tensor) -> bool:
    """Contiguous heads at steps of whole 16 bytes: what the kernels' copies need. A
    dimension of size 1 may have any stride."""

    strides = tensor.stride()
    return strides[-1] == 1 and all(
        n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(tensor.shape[:-1], strides[:-1])
    )


def _rows_are_loadable(tensor: Tensor) -> bool:
    return tensor.data_ptr() % 16 == 0 and (tensor.is_contiguous() or _strides_are_loadable(tensor))


def _refuse_tangents(what: str, *tensors: object) -> None:
    """A kernel reads a dual tensor's value and would drop its tangent without a word. (Callers look at
    ``forward_ad._current_level`` first: below 0 there are no dual tensors, and an attribute costs nothing.)"""

    for x in tensors:
        if isinstance(x, Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative, and an argument carries a tangent")


# (bound once: a chain of attributes costs a tenth of a microsecond of a short call's ten)
_is_compiled = torch.compiler.is_dynamo_compiling
_is_traced = torch._C._is_tracing
_dispatch_modes = torch._C._len_torch_dispatch_stack


def _refuse_tracing(what: str, *, is_a_node: bool) -> None:
    """For calls where ``_is_traced() or _dispatch_modes()``: a tracer sees the result's allocation and not the kernel,
    and what it records would return memory that nobody wrote. (``is_a_node``: an autograd function, which
    ``torch.jit.trace`` records as a whole.)"""

    proxies = _dispatch_modes() and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None
    if proxies or (_is_traced() and not is_a_node):
        raise RuntimeError(f"{what} cannot be recorded by make_fx or, without gradients, by torch.jit.trace")


# The handle of a device's current stream. (``torch.cuda.current_stream`` makes an object of it: 1.3 us of a short call's 11.)
_current_stream = torch._C._cuda_getCurrentRawStream


def _dense_strides(shape: Sequence[int]) -> list[int]:
    strides = [1]
    for n in reversed(shape[1:]):
        strides.insert(0, strides[0] * n)
    return strides


def _row_strides(shape: Sequence[int], strides: Sequence[int], kind: str) -> list[int]:
    """{sequence, row, head} strides; a harmless one where the dimension has size 1."""

    return [shape[-1] if axis is None or shape[axis] == 1 else strides[axis] for axis in _AXES[kind]]


def _stride_array(shape: Sequence[int], strides: Sequence[int], kind: str) -> ctypes.Array:
    return (ctypes.c_int64 * 3)(*_row_strides(shape, strides, kind))


def _window_sides(window: object, causal: bool) -> tuple[int, int]:
    """(left, right) with -1 for "no limit"."""

    if window is None or isinstance(window, int):
        left, right = window, 0 if causal else window
    elif isinstance(window, Sequence) and len(window) == 2:
        left, right = window
        if causal and right not in (None, 0):
            raise ValueError(f"a causal window has no right side, got window={tuple(window)}")
    else:
        raise ValueError(f"window must be None, an int or (left, right), got {window!r}")
    for side in (left, right):
        if side is not None and (not isinstance(side, int) or isinstance(side, bool) or side < 0):
            raise ValueError(f"window sides must be non-negative ints or None, got {window!r}")
    return (
        -1 if left is None else min(left, _MAX_LENGTH),
        0 if causal else -1 if right is None else min(right, _MAX_LENGTH),
    )


def _saved_layouts(q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, rest: Tensor) -> tuple:
    """What decides whether a backward pass may go by the forward pass's block. (Sizes as bytes: four microseconds of a
    short call's 120 with all shapes and types, two without.)"""

    return (
        q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype,
        out.is_contiguous(), lse.is_contiguous(), rest.is_contiguous(),
        q.nbytes, k.nbytes, v.nbytes, out.nbytes, lse.nbytes, rest.nbytes,
        q.device, k.device, v.device, out.device, lse.device, rest.device,
    )


class _Plan:
    """The checks and the host arithmetic of a call, kept per set of shapes, strides
    and settings: the argument block without addresses, and the workspace sizes."""

    __slots__ = (
        "kind", "block", "device", "index", "shapes", "saved", "spans", "lse_shape", "forward_bytes", "backward_bytes", "tables",
    )

    def __init__(
        self, kind: str, q: Tensor, k: Tensor, v: Tensor, causal: bool, window: object, sinks: int,
        scale: float | None, sequences: PackedSequences | None, with_lengths: bool,
    ) -> None:
        _check_heads_tensor(q, "q", kind, None)
        _check_heads_tensor(k, "k", kind, q.device)
        _check_heads_tensor(v, "v", kind, q.device)
        if k.shape != v.shape:
            raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
        batch_axis, row_axis, head_axis = _AXES[kind]
        head_dim = int(q.shape[-1])
        if head_dim != k.shape[-1] or head_dim % 8 or head_dim > 128:
            raise ValueError(f"head_dim must be one multiple of 8 up to 128, got {head_dim} and {int(k.shape[-1])}")
        heads, heads_kv = int(q.shape[head_axis]), int(k.shape[head_axis])
        if heads % heads_kv:
            raise ValueError(f"heads of q ({heads}) must be a multiple of those of k and v ({heads_kv})")
        batch = 1 if batch_axis is None else int(q.shape[batch_axis])
        if batch_axis is not None and batch != k.shape[batch_axis]:
            raise ValueError(f"q holds {batch} sequences, k and v {k.shape[batch_axis]}")
        rows, keys = int(q.shape[row_axis]), int(k.shape[row_axis])
        if max(rows, keys) > _MAX_LENGTH:
            raise ValueError(f"at most {_MAX_LENGTH} rows, got {rows} and {keys}")
        for name, tensor in (("q", q), ("k", k), ("v", v)):
            if not _strides_are_loadable(tensor):
                raise ValueError(
                    f"{name} must have contiguous heads at positive strides of whole 16 bytes, got strides "
                    f"{tensor.stride()}; pass {name}.contiguous()"
                )
        if not isinstance(sinks, int) or isinstance(sinks, bool) or sinks < 0:
            raise ValueError(f"sinks must be a non-negative int, got {sinks!r}")
        scale = head_dim**-0.5 if scale is None else scale
        if not 0.0 < scale <= 1e30:
            raise ValueError(f"scale must be positive and finite, got {scale}")
        left, right = _window_sides(window, causal)
        if sequences is not None:
            if sequences.device != q.device:
                raise ValueError(f"sequences live on {sequences.device}, q on {q.device}")
            if sequences.cu_seqlens_q[-1] != rows or sequences.cu_seqlens_k[-1] != keys:
                raise ValueError(
                    f"sequences describe {sequences.cu_seqlens_q[-1]} query and {sequences.cu_seqlens_k[-1]} key "
                    f"rows, got {rows} and {keys}"
                )
        a = _native.MupWindowAttention()
        a.device = q.device.index
        a.batch, a.heads_q, a.heads_kv, a.head_dim, a.seq_q, a.seq_k = batch, heads, heads_kv, head_dim, rows, keys
        a.causal, a.left, a.right, a.sinks, a.scale = causal, left, right, min(sinks, _MAX_LENGTH), scale
        for name, tensor in (("q", q), ("k", k), ("v", v)):
            setattr(a, name + "_strides", _stride_array(tensor.shape, tensor.stride(), kind))
        # results and gradients are dense
        for name, shape in (("out", q.shape), ("dout", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", k.shape)):
            setattr(a, name + "_strides", _stride_array(shape, _dense_strides(shape), kind))
        if sequences is not None:
            a.sequences, a.n_sequences = sequences.sequences.data_ptr(), sequences.num_sequences
            for name in ("q_blocks_256", "q_blocks_128", "k_blocks_128"):
                blocks = getattr(sequences, name)
                setattr(a, name, blocks.data_ptr())
                setattr(a, "n_" + name, len(blocks))
            a.longest_q, a.longest_k = sequences.longest_q, sequences.longest_k
        a.timeout_ns = _KERNEL_TIMEOUT_NS
        a.kv_lengths = 1 if with_lengths else None  # only whether there are any matters here
        forward, backward = ctypes.c_uint64(), ctypes.c_uint64()
        _native.call(
            "mup_window_attention_workspace", ctypes.byref(a), ctypes.byref(forward), ctypes.byref(backward)
        )
        a.kv_lengths = None
        self.kind, self.block = kind, bytes(a)
        # a plan that a backward pass still holds keeps the tables whose addresses it knows
        self.tables = None if sequences is None else (
            sequences.sequences, sequences.q_blocks_256, sequences.q_blocks_128, sequences.k_blocks_128,
        )
        self.lse_shape = (heads, rows) if batch_axis is None else (batch, heads, rows)
        # what a backward pass expects of q, k, v, out, lse and rest
        self.spans = _span(q), _span(k), _span(v)
        lse = q.new_empty(self.lse_shape, dtype=torch.float32, device="meta")
        dense = q.new_empty(q.shape, device="meta")
        self.shapes = q.shape, k.shape, v.shape, q.shape, lse.shape, q.shape
        self.saved = (*_saved_layouts(q, k, v, dense, lse, dense)[:-6], *[q.device] * 6)
        self.device, self.index = q.device, q.device.index
        self.forward_bytes, self.backward_bytes = forward.value, backward.value

    def arguments(self, q: Tensor, k: Tensor, v: Tensor) -> _native.MupWindowAttention:
        a = _native.MupWindowAttention.from_buffer_copy(self.block)
        a.q, a.k, a.v = addresses = q.data_ptr(), k.data_ptr(), v.data_ptr()
        if (addresses[0] | addresses[1] | addresses[2]) % 16:
            raise ValueError(f"q, k and v must be 16-byte aligned, got addresses {[hex(x) for x in addresses]}")
        return a

    def saved_arguments(self, saved: Sequence[Tensor]) -> tuple[_native.MupWindowAttention, list[Tensor]]:
        """The block of a backward pass, and ``q, k, v, out, lse, rest`` as its copies may read them. A hook of saved
        tensors (offloading, checkpointing) may return them with other strides or addresses than the forward pass had."""

        q, k, v, out, lse, rest = saved
        if _saved_layouts(q, k, v, out, lse, rest) == self.saved:
            a = _native.MupWindowAttention.from_buffer_copy(self.block)
            a.q, a.k, a.v = aq, ak, av = q.data_ptr(), k.data_ptr(), v.data_ptr()
            a.out, a.lse, a.out_rest = ao, al, ar = out.data_ptr(), lse.data_ptr(), rest.data_ptr()
            if not (aq | ak | av | ao | al | ar) % 16:
                return a, saved
        tensors = list(saved)
        for i, name in enumerate(("q", "k", "v", "out", "lse", "rest")):
            x, shape, dtype = saved[i], self.shapes[i], torch.float32 if name == "lse" else torch.bfloat16
            if x.shape != shape or x.dtype != dtype or x.device != self.device:
                raise RuntimeError(
                    f"a hook of saved tensors returned {x.dtype} {tuple(x.shape)} on {x.device} for {name}, which was "
                    f"{dtype} {tuple(shape)} on {self.device}"
                )
            if not (_rows_are_loadable(x) if i < 3 else x.is_contiguous() and x.data_ptr() % 16 == 0):
                tensors[i] = x.clone(memory_format=torch.contiguous_format)
        a = self.arguments(*tensors[:3])
        for name, x in zip("qkv", tensors):
            setattr(a, name + "_strides", _stride_array(x.shape, x.stride(), self.kind))
        a.out, a.lse, a.out_rest = (x.data_ptr() for x in tensors[3:])
        return a, tensors

    def launch(self, function: str, a: _native.MupWindowAttention, workspace_bytes: int, q: Tensor) -> None:
        """On the current stream of the device of ``q``."""

        if workspace_bytes:
            # freed with this frame: the allocator hands it out again in stream order
            workspace = q.new_empty(workspace_bytes, dtype=torch.uint8)
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace_bytes
        _native.call(function, ctypes.byref(a), _current_stream(self.index))


_PLANS: dict[object, _Plan] = {}
_MAX_PLANS = 512


def _plan(
    kind: str, q: Tensor, k: Tensor, v: Tensor, causal: bool, window: object, sinks: int, scale: float | None,
    sequences: PackedSequences | None, with_lengths: bool,
) -> _Plan:
    plans = _PLANS if sequences is None else sequences.plans
    # (True and 1.0 are equal to 1 and would find its plan: what is no plain int is checked each time)
    sides = window if window is None or type(window) is int else _window_sides(window, causal)
    try:
        key = (
            kind, q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype,
            q.device, k.device, v.device, causal, sides, sinks, type(sinks), scale, with_lengths,
        )
        return plans[key]
    except (KeyError, TypeError, AttributeError):  # new, not hashable, not a tensor
        plan = _Plan(kind, q, k, v, causal, window, sinks, scale, sequences, with_lengths)
    if len(plans) >= _MAX_PLANS:
        plans.clear()
    plans[key] = plan
    return plan


def _check_kv_lengths(kv_lengths: object, q: Tensor, kind: str) -> None:
    batch = q.shape[_AXES[kind][0]]
    if (
        not isinstance(kv_lengths, Tensor)
        or kv_lengths.dtype != torch.int32
        or kv_lengths.device != q.device
        or kv_lengths.shape != (batch,)
        or not kv_lengths.is_contiguous()
    ):
        raise ValueError(f"kv_lengths must be contiguous int32 [{batch}] on {q.device}, got {_tensor_signature(kv_lengths)}")


def _meet(distance: int, steps: list[tuple[int, int, int]]) -> bool:
    """Whether ``distance`` is a sum of ``stride * t`` with ``low <= t <= high``; ``steps`` are (stride, low, high), the
    largest stride first."""

    if not steps:
        return distance == 0
    (stride, low, high), rest = steps[0], steps[1:]
    # what the other steps can reach leaves a few t, for strides that nest at most two
    least, most = sum(s * l for s, l, _ in rest), sum(s * h for s, _, h in rest)
    first, last = max(low, -((most - distance) // stride)), min(high, (distance - least) // stride)
    return any(_meet(distance - stride * t, rest) for t in range(first, last + 1))


@lru_cache(256)
def _layouts_meet(
    a_shape: Sequence[int], a_strides: Sequence[int], b_shape: Sequence[int], b_strides: Sequence[int], distance: int
) -> bool:
    """Whether tensors of one buffer share an element, the second's first one ``distance`` elements behind the first's.
    Slices with the same strides are compared exactly (interleaved ones are apart), others only where both are dense."""

    if distance == 0:
        return True
    dims = list(zip(a_shape, b_shape, a_strides, b_strides))
    if all(s == t or m == 1 or n == 1 for m, n, s, t in dims):
        # an element of `a` at i and one of `b` at j are the same where the sum of (i - j) * stride is the distance
        return _meet(distance, sorted(((t if m == 1 else s, 1 - n, m - 1) for m, n, s, t in dims), reverse=True))
    if list(a_strides) != _dense_strides(a_shape) or list(b_strides) != _dense_strides(b_shape):
        return False
    return -math.prod(b_shape) < distance < math.prod(a_shape)


def _span(x: Tensor) -> int:
    """Bytes from the first to the last element."""

    return 2 * (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1)


def _share_elements(a: Tensor, a_span: int, b: Tensor, b_span: int) -> bool:
    """Whether two BF16 tensors of as many dimensions are known to share an element."""

    distance = b.data_ptr() - a.data_ptr()
    return -b_span < distance < a_span and _layouts_meet(a.shape, a.stride(), b.shape, b.stride(), distance // 2)


def _is_same(a: Tensor, b: Tensor) -> bool:
    """Element for element the same memory."""

    return a is b or (a.data_ptr() == b.data_ptr() and a.shape == b.shape and (
        a.stride() == b.stride() or all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))
    ))


def _check_out(plan: _Plan, out: object, q: Tensor, k: Tensor, v: Tensor) -> None:
    q_span, k_span, v_span = plan.spans
    span = q_span
    if out is not q:
        if not isinstance(out, Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"out must be BF16 {tuple(q.shape)} on {q.device}, got {_tensor_signature(out)}")
        if not _rows_are_loadable(out):
            raise ValueError(f"out must have contiguous heads at 16-byte aligned strides, got {out.stride()}")
        span = _span(out)
        if _share_elements(out, span, q, q_span) and not _is_same(out, q):
            raise ValueError("out may be q itself, and must not overlap it otherwise")
    if _share_elements(out, span, k, k_span) or _share_elements(out, span, v, v_span):
        raise ValueError("out must not overlap k or v")


def _forward(
    plan: _Plan, q: Tensor, k: Tensor, v: Tensor, out: Tensor | None, need_lse: bool, kv_lengths: Tensor | None,
    rest: Tensor | None = None,
) -> tuple[Tensor, Tensor | None]:
    a = plan.arguments(q, k, v)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        a.out_strides = _stride_array(out.shape, out.stride(), plan.kind)
        increment_version(out)  # autograd refuses a graph that had saved it
    a.out = out.data_ptr()
    lse = None
    if need_lse:
        lse = q.new_empty(plan.lse_shape, dtype=torch.float32)
        a.lse = lse.data_ptr()
    if kv_lengths is not None:
        a.kv_lengths = kv_lengths.data_ptr()
    if rest is not None:
        a.out_rest = rest.data_ptr()
    plan.launch("mup_window_attention_forward", a, plan.forward_bytes, q)
    return out, lse


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan):
        ctx.set_materialize_grads(False)
        # what the result's rounding leaves: the backward pass sums result * gradient per row
        rest = torch.empty_like(q, memory_format=torch.contiguous_format)
        out, lse = _forward(plan, q, k, v, None, True, None, rest)
        ctx.save_for_backward(q, k, v, out, lse, rest)
        ctx.plan = plan
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return None, None, None, None
        if forward_ad._current_level >= 0:
            _refuse_tangents("the gradient of window_attention", dout)
        plan: _Plan = ctx.plan
        a, (q, k, v, *_) = plan.saved_arguments(ctx.saved_tensors)
        if not _rows_are_loadable(dout):  # a broadcast or transposed gradient
            dout = dout.clone(memory_format=torch.contiguous_format)
        elif not dout.is_contiguous():
            a.dout_strides = _stride_array(dout.shape, dout.stride(), plan.kind)
        dq, dk, dv = grads = [torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v)]
        a.dout = dout.data_ptr()
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        plan.launch("mup_window_attention_backward", a, plan.backward_bytes, q)
        return (*grads, None)


def _attend(
    kind: str, q: Tensor, k: Tensor, v: Tensor, causal: bool, window: object, sinks: int, scale: float | None,
    kv_lengths: Tensor | None, sequences: PackedSequences | None, out: Tensor | None, return_lse: bool,
):
    if _is_compiled():
        # torch.compile's tracer mistakes the fields of an argument block: the call runs as it is, at a graph break
        return torch.compiler.disable(_attend)(
            kind, q, k, v, causal, window, sinks, scale, kv_lengths, sequences, out, return_lse
        )
    # plans are kept by these values: no object that can change (a tensor of one number) stands for them
    causal, scale = bool(causal), None if scale is None else float(scale)
    plan = _plan(kind, q, k, v, causal, window, sinks, scale, sequences, kv_lengths is not None)
    if forward_ad._current_level >= 0:
        _refuse_tangents(f"window_attention_{kind}", q, k, v, out)
    if kv_lengths is not None:
        _check_kv_lengths(kv_lengths, q, kind)
    if out is not None:
        _check_out(plan, out, q, k, v)
    if torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad or v.requires_grad or (out is not None and out.requires_grad)
    ):
        if out is not None:
            raise ValueError("out cannot be given when a gradient is wanted")
        if kv_lengths is not None:
            raise ValueError("kv_lengths is for tokens over a cache: there is no gradient through it")
        if _dispatch_modes():
            _refuse_tracing(f"window_attention_{kind}", is_a_node=True)
        result, lse = _WindowAttention.apply(q, k, v, plan)
    else:
        if _dispatch_modes() or _is_traced():
            _refuse_tracing(f"window_attention_{kind}", is_a_node=False)
        result, lse = _forward(plan, q, k, v, out, return_lse, kv_lengths)
    return (result, lse) if return_lse else result


def window_attention_bshd(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    causal: bool = True,
    window: int | tuple[int | None, int | None] | None = None,
    sinks: int = 0,
    scale: float | None = None,
    kv_lengths: Tensor | None = None,
    out: Tensor | None = None,
    return_lse: bool = False,
):
    """Attention of ``q [B,Sq,H,D]`` over ``k, v [B,Sk,Hkv,D]``; returns ``[B,Sq,H,D]``.

    ``window``: keys before the own position that stay visible (causal), the same
    on both sides or ``(left, right)`` (not causal); ``None``: no limit. ``sinks``:
    first keys that stay visible whatever the window. ``scale`` defaults to
    ``D ** -0.5``. ``kv_lengths`` (int32 ``[B]`` on the device): how many rows of
    ``k`` and ``v``, from the first, hold keys of each sequence - a cache that is
    filled to different lengths; the queries are then its last rows. A length
    outside ``[0, Sk]`` counts as the nearer end. Slices of a fused projection may
    be passed as they are; ``D`` is a multiple of 8 up to 128. ``return_lse`` adds
    the FP32 ``[B,H,Sq]`` log-sum-exp of every row (no gradient flows through it).
    ``out`` is written instead of a new tensor; it may be ``q`` itself and overlaps
    no other input. Differentiable in ``q``, ``k`` and ``v``, once and in reverse mode.
    """

    return _attend("bshd", q, k, v, causal, window, sinks, scale, kv_lengths, None, out, return_lse)


def window_attention_sbhd(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    causal: bool = True,
    window: int | tuple[int | None, int | None] | None = None,
    sinks: int = 0,
    scale: float | None = None,
    kv_lengths: Tensor | None = None,
    out: Tensor | None = None,
    return_lse: bool = False,
):
    """Sequence-first variant: ``q [Sq,B,H,D]``, ``k, v [Sk,B,Hkv,D]`` -> ``[Sq,B,H,D]``
    (log-sum-exp ``[B,H,Sq]``)."""

    return _attend("sbhd", q, k, v, causal, window, sinks, scale, kv_lengths, None, out, return_lse)


def window_attention_thd(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    sequences: PackedSequences,
    *,
    causal: bool = True,
    window: int | tuple[int | None, int | None] | None = None,
    sinks: int = 0,
    scale: float | None = None,
    out: Tensor | None = None,
    return_lse: bool = False,
):
    """Packed variant: ``q [Tq,H,D]``, ``k, v [Tk,Hkv,D]`` -> ``[Tq,H,D]`` (log-sum-exp
    ``[H,Tq]``), every sequence of ``sequences`` (``prepare_packed_sequences``) by itself."""

    if not isinstance(sequences, PackedSequences):
        raise TypeError("sequences must be PackedSequences from prepare_packed_sequences")
    return _attend("thd", q, k, v, causal, window, sinks, scale, None, sequences, out, return_lse)
