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
key that no query row sees has no influence, whatever it holds; an infinity or
NaN in a key or value row that some query sees may reach the other rows of the
same block of queries.

BF16 in and out, FP32 sums, one rounding of the probabilities (and, backward,
of the score gradients) to BF16 for the second product and one of the results.
The gradient is deterministic. Kernels: ``csrc/mup_attn_*.cuh``.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence
from dataclasses import dataclass, field

import torch
from torch import Tensor

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

    @property
    def num_sequences(self) -> int:
        return len(self.cu_seqlens_q) - 1

    @property
    def device(self) -> torch.device:
        return self.sequences.device


def _blocks(lengths: list[int], rows: int) -> list[tuple[int, int]]:
    """(sequence, first row) of every block of ``rows`` rows, the last rows first:
    under a causal mask they have the most keys."""

    blocks = [(s, r) for s, length in enumerate(lengths) for r in range(0, length, rows)]
    return sorted(blocks, key=lambda block: -block[1])


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

    def on_device(rows):
        return torch.tensor(rows, dtype=torch.int32).to(device)

    return PackedSequences(
        cu_seqlens_q=cu_q,
        cu_seqlens_k=cu_k,
        sequences=on_device(table),
        q_blocks_256=on_device(_blocks(queries, 256)),
        q_blocks_128=on_device(_blocks(queries, 128)),
        k_blocks_128=on_device(_blocks(keys, 128)[::-1]),
        longest_q=max(queries),
        longest_k=max(keys),
    )


# --------------------------------------------------------------------------- validation


def _check_heads_tensor(tensor: object, name: str, kind: str, device: torch.device | None) -> None:
    if not isinstance(tensor, Tensor) or tensor.ndim != len(_INPUT_LABEL[kind].split(",")):
        raise ValueError(f"{name} must be {_INPUT_LABEL[kind]}, got {_tensor_signature(tensor)}")
    if tensor.dtype != torch.bfloat16 or not tensor.is_cuda or (device is not None and tensor.device != device):
        raise ValueError(f"{name} must be BF16 on one CUDA device, got {tensor.dtype} on {tensor.device}")
    if min(tensor.shape) <= 0:
        raise ValueError(f"all dimensions of {name} must be positive, got {tuple(tensor.shape)}")


def _rows_are_loadable(tensor: Tensor) -> bool:
    """Contiguous heads at 16-byte steps: what the kernels' copies need. A dimension
    of size 1 may have any stride."""

    strides = tensor.stride()
    return (
        strides[-1] == 1
        and tensor.data_ptr() % 16 == 0
        and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(tensor.shape[:-1], strides[:-1]))
    )


def _strides(tensor: Tensor, kind: str) -> tuple[int, int, int]:
    """{sequence, row, head} strides; a harmless one where the dimension has size 1."""

    shape, strides = tensor.shape, tensor.stride()
    dim = -(-int(shape[-1]) // 8) * 8
    return tuple(
        dim if axis is None or shape[axis] == 1 else strides[axis] for axis in _AXES[kind]
    )  # type: ignore[return-value]


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


@dataclass(frozen=True)
class _Options:
    """What a call fixes apart from its tensors."""

    kind: str
    causal: bool
    left: int
    right: int
    sinks: int
    scale: float
    kv_lengths: Tensor | None = field(default=None, compare=False)
    sequences: PackedSequences | None = field(default=None, compare=False)


def _options(
    kind: str, q: Tensor, k: Tensor, v: Tensor, *, causal: bool, window: object, sinks: int, scale: float | None,
    kv_lengths: Tensor | None, sequences: PackedSequences | None,
) -> _Options:
    _check_heads_tensor(q, "q", kind, None)
    _check_heads_tensor(k, "k", kind, q.device)
    _check_heads_tensor(v, "v", kind, q.device)
    if k.shape != v.shape:
        raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    batch_axis, row_axis, _ = _AXES[kind]
    head_dim = int(q.shape[-1])
    if head_dim != k.shape[-1] or head_dim % 8 or head_dim > 128:
        raise ValueError(
            f"head_dim must be one multiple of 8 up to 128, got {head_dim} and {int(k.shape[-1])}"
        )
    if q.shape[-2] % k.shape[-2]:
        raise ValueError(f"heads of q ({q.shape[-2]}) must be a multiple of those of k and v ({k.shape[-2]})")
    if batch_axis is not None and q.shape[batch_axis] != k.shape[batch_axis]:
        raise ValueError(f"q holds {q.shape[batch_axis]} sequences, k and v {k.shape[batch_axis]}")
    if max(q.shape[row_axis], k.shape[row_axis]) > _MAX_LENGTH:
        raise ValueError(f"at most {_MAX_LENGTH} rows, got {q.shape[row_axis]} and {k.shape[row_axis]}")
    for name, tensor in (("q", q), ("k", k), ("v", v)):
        if not _rows_are_loadable(tensor):
            raise ValueError(
                f"{name} must have contiguous heads at 16-byte aligned, positive strides, got strides "
                f"{tensor.stride()} at address {tensor.data_ptr():#x}; pass {name}.contiguous()"
            )
    if not isinstance(sinks, int) or isinstance(sinks, bool) or sinks < 0:
        raise ValueError(f"sinks must be a non-negative int, got {sinks!r}")
    scale = head_dim**-0.5 if scale is None else float(scale)
    if not (0.0 < scale <= 1e30):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    left, right = _window_sides(window, bool(causal))
    if kv_lengths is not None:
        if (
            not isinstance(kv_lengths, Tensor)
            or kv_lengths.dtype != torch.int32
            or kv_lengths.device != q.device
            or tuple(kv_lengths.shape) != (q.shape[batch_axis],)
            or not kv_lengths.is_contiguous()
        ):
            raise ValueError(
                f"kv_lengths must be contiguous int32 [{q.shape[batch_axis]}] on {q.device}, "
                f"got {_tensor_signature(kv_lengths)}"
            )
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            raise ValueError("kv_lengths is for tokens over a cache: there is no gradient through it")
    if kind == "thd":
        if not isinstance(sequences, PackedSequences):
            raise TypeError("sequences must be PackedSequences from prepare_packed_sequences")
        if sequences.device != q.device:
            raise ValueError(f"sequences live on {sequences.device}, q on {q.device}")
        if sequences.cu_seqlens_q[-1] != q.shape[0] or sequences.cu_seqlens_k[-1] != k.shape[0]:
            raise ValueError(
                f"sequences describe {sequences.cu_seqlens_q[-1]} query and {sequences.cu_seqlens_k[-1]} key rows, "
                f"got {q.shape[0]} and {k.shape[0]}"
            )
    return _Options(kind, bool(causal), left, right, min(sinks, _MAX_LENGTH), scale, kv_lengths, sequences)


def _check_out(out: object, q: Tensor, *inputs: Tensor) -> None:
    if out is None:
        return
    if not isinstance(out, Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError(f"out must be BF16 {tuple(q.shape)} on {q.device}, got {_tensor_signature(out)}")
    if not _rows_are_loadable(out):
        raise ValueError(f"out must have contiguous heads at 16-byte aligned strides, got {out.stride()}")


# --------------------------------------------------------------------------- calls of the library


def _arguments(o: _Options, q: Tensor, k: Tensor, v: Tensor) -> _native.MupWindowAttention:
    a = _native.MupWindowAttention()
    batch_axis, row_axis, head_axis = _AXES[o.kind]
    a.device = q.device.index
    a.batch = 1 if batch_axis is None else q.shape[batch_axis]
    a.heads_q, a.heads_kv, a.head_dim = q.shape[head_axis], k.shape[head_axis], q.shape[-1]
    a.seq_q, a.seq_k = q.shape[row_axis], k.shape[row_axis]
    a.causal, a.left, a.right, a.sinks, a.scale = o.causal, o.left, o.right, o.sinks, o.scale
    for name, tensor in (("q", q), ("k", k), ("v", v)):
        _bind(a, name, tensor, o.kind)
    if o.kv_lengths is not None:
        a.kv_lengths = o.kv_lengths.data_ptr()
    if o.sequences is not None:
        s = o.sequences
        a.sequences, a.n_sequences = s.sequences.data_ptr(), s.num_sequences
        for name in ("q_blocks_256", "q_blocks_128", "k_blocks_128"):
            blocks = getattr(s, name)
            setattr(a, name, blocks.data_ptr())
            setattr(a, "n_" + name, len(blocks))
        a.longest_q, a.longest_k = s.longest_q, s.longest_k
    a.timeout_ns = _KERNEL_TIMEOUT_NS
    return a


def _bind(a: _native.MupWindowAttention, name: str, tensor: Tensor, kind: str) -> None:
    setattr(a, name, tensor.data_ptr())
    setattr(a, name + "_strides", (ctypes.c_int64 * 3)(*_strides(tensor, kind)))


def _launch(function: str, a: _native.MupWindowAttention, device: torch.device, which: int) -> None:
    """Give the call its workspace and launch it on the current stream of ``device``."""

    sizes = (ctypes.c_uint64 * 2)()
    address = ctypes.addressof(sizes)
    pointer = ctypes.POINTER(ctypes.c_uint64)
    _native.call(
        "mup_window_attention_workspace", ctypes.byref(a), ctypes.cast(address, pointer),
        ctypes.cast(address + 8, pointer),
    )
    if sizes[which]:
        # freed with this frame: the allocator hands it out again in stream order
        workspace = torch.empty(sizes[which], dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), sizes[which]
    _native.call(function, ctypes.byref(a), torch.cuda.current_stream(device).cuda_stream)


def _lse_shape(o: _Options, q: Tensor) -> tuple[int, ...]:
    batch_axis, row_axis, head_axis = _AXES[o.kind]
    tail = (int(q.shape[head_axis]), int(q.shape[row_axis]))
    return tail if batch_axis is None else (int(q.shape[batch_axis]), *tail)


def _forward(
    o: _Options, q: Tensor, k: Tensor, v: Tensor, out: Tensor | None, need_lse: bool
) -> tuple[Tensor, Tensor | None]:
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(_lse_shape(o, q), dtype=torch.float32, device=q.device) if need_lse else None
    a = _arguments(o, q, k, v)
    _bind(a, "out", out, o.kind)
    a.lse = None if lse is None else lse.data_ptr()
    _launch("mup_window_attention_forward", a, q.device, 0)
    return out, lse


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, options):
        out, lse = _forward(options, q, k, v, None, True)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.options = options
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, lse = ctx.saved_tensors
        o = ctx.options
        if not _rows_are_loadable(dout):
            dout = dout.contiguous()  # a broadcast or transposed gradient
        if dout.data_ptr() % 16:
            dout = dout.clone()
        grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v)]
        a = _arguments(o, q, k, v)
        for name, tensor in zip(("out", "dout", "dq", "dk", "dv"), (out, dout, *grads)):
            _bind(a, name, tensor, o.kind)
        a.lse = lse.data_ptr()
        _launch("mup_window_attention_backward", a, q.device, 1)
        return (*grads, None)


def _attend(kind, q, k, v, *, out, return_lse, **settings):
    o = _options(kind, q, k, v, **settings)
    _check_out(out, q)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if out is not None:
            raise ValueError("out cannot be given when a gradient is wanted")
        result, lse = _WindowAttention.apply(q, k, v, o)
    else:
        result, lse = _forward(o, q, k, v, out, return_lse)
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
    Differentiable in ``q``, ``k`` and ``v``.
    """

    return _attend(
        "bshd", q, k, v, causal=causal, window=window, sinks=sinks, scale=scale, kv_lengths=kv_lengths,
        sequences=None, out=out, return_lse=return_lse,
    )


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

    return _attend(
        "sbhd", q, k, v, causal=causal, window=window, sinks=sinks, scale=scale, kv_lengths=kv_lengths,
        sequences=None, out=out, return_lse=return_lse,
    )


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

    return _attend(
        "thd", q, k, v, causal=causal, window=window, sinks=sinks, scale=scale, kv_lengths=None,
        sequences=sequences, out=out, return_lse=return_lse,
    )
