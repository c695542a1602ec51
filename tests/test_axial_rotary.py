"""Rotary positions with several axes: the arguments they refuse (no GPU needed) and their results against 64 bits."""

from __future__ import annotations

import copy
import ctypes
import math
import pickle

import pytest
import torch

import megaup_b200 as mega_up
from _attention_reference import assert_within, rotate
from megaup_b200 import _native, build

DEVICE = torch.device("cuda", 0)
BF16 = torch.bfloat16


def _frequencies(axis_dims, theta, shared):
    total = sum(axis_dims)
    axis, exponents = [], []
    for a, d in enumerate(axis_dims):
        for i in range(d // 2):
            exponents.append(2 * len(axis) / total if shared else 2 * i / d)
            axis.append(a)
    return torch.tensor(axis), torch.tensor([theta**-e for e in exponents], dtype=torch.float64)


# --------------------------------------------------------------------------- without a GPU


@pytest.mark.parametrize("shared", [False, True])
def test_frequencies(shared) -> None:
    r = mega_up.prepare_axial_rotary([44, 42, 42], theta=256.0, shared_frequencies=shared, device="cpu")
    axis, frequencies = _frequencies([44, 42, 42], 256.0, shared)
    assert r.pairs == 64 and r.pair_axis.tolist() == axis.tolist()
    assert torch.allclose(r.turns, frequencies / (2 * math.pi), rtol=1e-15, atol=0)


@pytest.mark.parametrize(
    "dims,settings",
    [([], {}), ([3], {}), ([0, 4], {}), ([-2], {}), ([256, 2], {}), ([24], dict(interleaved=False)),
     ([64], dict(theta=0.0)), ([64], dict(theta=float("inf"))), ([64], dict(theta=float("nan")))],
    ids=str,
)
def test_prepare_refuses(dims, settings) -> None:
    with pytest.raises(ValueError):
        mega_up.prepare_axial_rotary(dims, device="cpu", **settings)


def _block(**changes) -> _native.MupAxialRotary:
    a = _native.MupAxialRotary()
    a.batch, a.rows, a.head_dim, a.pairs, a.axes, a.interleaved = 1, 4, 64, 32, 1, 1
    a.heads[:] = (2, 1)
    a.q = a.q_out = 4096
    a.k = a.k_out = 8192
    a.x_strides[:] = a.y_strides[:] = (512, 128, 64, 512, 128, 64)
    a.positions = a.turns = a.pair_axis = 4096
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize(
    "changes",
    [dict(head_dim=4), dict(head_dim=68), dict(head_dim=264), dict(pairs=0), dict(pairs=33), dict(interleaved=0, pairs=12),
     dict(batch=0), dict(rows=0), dict(axes=0), dict(heads=(ctypes.c_int32 * 2)(0, 1)), dict(positions=0), dict(turns=0),
     dict(pair_axis=0), dict(position_type=3), dict(k=0),
     dict(q_out=4104), dict(x_strides=(ctypes.c_int64 * 6)(512, 129, 64, 512, 128, 64)),
     dict(y_strides=(ctypes.c_int64 * 6)(512, 128, 64, 512, 128, -64))],
    ids=str,
)
def test_the_library_refuses(changes) -> None:
    build.ensure_built()
    library = _native.lib()
    assert library.mup_axial_rotary_launch(ctypes.byref(_block(**changes)), None) in (-1, -3)
    assert b"axial rotary" in library.mup_last_error()
    assert library.mup_axial_rotary_launch(None, None) == -1


def test_host_tensors_are_refused() -> None:
    r = mega_up.prepare_axial_rotary([64], device="cpu")
    x = torch.zeros(4, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        mega_up.axial_rotary_thd(x, None, r, torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(TypeError):
        mega_up.axial_rotary_thd(x, None, None, torch.zeros(1, 4, dtype=torch.int32))


# --------------------------------------------------------------------------- on the GPU


def _normal(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEVICE)


def _positions(axes, shape, dtype, seed=5, largest=2_000_000):
    generator = torch.Generator().manual_seed(seed)
    x = torch.randint(-largest, largest, (axes, *shape), generator=generator)
    if dtype == torch.float32:
        return (x.float() / 7).to(DEVICE)  # exact in FP32 or not: the kernel and the check see the same value
    return x.to(dtype).to(DEVICE)


CASES = [
    # kind, batch, rows, heads, kv heads, dim, axis dims, interleaved, shared, position type, one row per sequence
    ("bshd", 1, 1, 1, 1, 64, [64], True, False, torch.int64, False),
    ("bshd", 2, 37, 5, 5, 128, [44, 42, 42], True, False, torch.int64, False),
    ("bshd", 3, 20, 6, 2, 128, [44, 42, 42], True, False, torch.int32, True),
    ("sbhd", 3, 20, 6, 2, 128, [32, 48, 48], False, True, torch.int64, True),
    ("sbhd", 2, 129, 3, 1, 96, [20, 30], True, True, torch.float32, False),  # 46 elements stay
    ("thd", 1, 301, 40, 8, 64, [16, 8, 8], False, False, torch.int32, False),  # 32 elements stay
    ("thd", 1, 77, 9, None, 72, [2], True, False, torch.int64, False),
    ("thd", 1, 50, 2, 2, 256, [128, 64, 64], True, False, torch.float32, False),
    ("bshd", 2, 30, 3, 3, 256, [256], False, False, torch.int64, False),
    ("bshd", 2, 30, 3, 3, 248, [100, 100, 48], True, False, torch.int64, True),
    ("bshd", 2, 30, 3, 3, 248, [48, 64], False, True, torch.int64, True),
    ("bshd", 1, 64, 33, 1, 8, [6], True, False, torch.int64, False),
    ("sbhd", 1, 64, 33, 1, 24, [16], False, False, torch.int64, False),
]


def _angles(kind, positions, axis, frequencies):
    """[..., 1, pairs] that broadcasts against the layout."""

    angle = torch.movedim(positions.double().cpu()[axis], 0, -1) * frequencies
    if positions.ndim == 2 and kind != "thd":
        angle = angle[None] if kind == "bshd" else angle[:, None]
    return angle.unsqueeze(-2)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(case) -> None:
    kind, batch, rows, heads, kv_heads, dim, dims, interleaved, shared, dtype, own_rows = case
    lead = {"bshd": (batch, rows), "sbhd": (rows, batch), "thd": (rows,)}[kind]
    q = _normal((*lead, heads, dim), 1).requires_grad_()
    k = None if kv_heads is None else _normal((*lead, kv_heads, dim), 2).requires_grad_()
    positions = _positions(len(dims), lead if own_rows else (rows,), dtype)
    rotary = mega_up.prepare_axial_rotary(dims, theta=5000.0, interleaved=interleaved, shared_frequencies=shared, device=DEVICE)
    call = getattr(mega_up, f"axial_rotary_{kind}")
    angle = _angles(kind, positions, *_frequencies(dims, 5000.0, shared))
    got = call(q, k, rotary, positions)
    assert (got[1] is None) == (k is None)
    for i, x in enumerate((q, k)):
        if x is None:
            continue
        want, error = rotate(x, angle, interleaved=interleaved)
        assert_within(got[i], want, error, "result")
        g = _normal(x.shape, 3 + i)
        (gradient,) = torch.autograd.grad(got[i], x, g, retain_graph=True)
        want, error = rotate(g, -angle, interleaved=interleaved)
        assert_within(gradient, want, error, "gradient")
    with torch.no_grad():  # in place, and the same bits
        copies = [x.detach().clone() for x in (q, k) if x is not None]
        again = call(copies[0], copies[1] if k is not None else None, rotary, positions, out=tuple(copies))
    assert again[0].data_ptr() == copies[0].data_ptr()
    for a, b in zip(got, again):
        assert a is None or torch.equal(a, b)


@pytest.mark.gpu
def test_the_gradient_is_the_slope() -> None:
    """The map is linear: the difference along a direction is exact."""

    x, g = _normal((40, 3, 64), 1).requires_grad_(), _normal((40, 3, 64), 2)
    rotary = mega_up.prepare_axial_rotary([32, 32], device=DEVICE)
    positions = _positions(2, (40,), torch.int64)
    y, _ = mega_up.axial_rotary_thd(x, None, rotary, positions)
    (gradient,) = torch.autograd.grad(y, x, g)
    angle = _angles("thd", positions, *_frequencies([32, 32], 10000.0, False))
    direction = torch.randn(x.shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    moved = x.detach().double().cpu()
    ends = [float((rotate(moved + s * direction, angle, interleaved=True)[0] * g.double().cpu()).sum()) for s in (1.0, -1.0)]
    _, error = rotate(g, -angle, interleaved=True)
    got = float((gradient.double().cpu() * direction).sum())
    assert abs(got - (ends[0] - ends[1]) / 2) <= float((error * direction.abs()).sum()) + 1e-9


@pytest.mark.gpu
def test_infinities_and_untouched_elements() -> None:
    x = _normal((5, 2, 64), 1)
    x[1, 0, 40], x[2, 1, 50], x[3, 0, 63] = float("inf"), float("nan"), -float("inf")
    rotary = mega_up.prepare_axial_rotary([20, 12], device=DEVICE)
    y, _ = mega_up.axial_rotary_thd(x, None, rotary, _positions(2, (5,), torch.int64))
    assert torch.equal(y[..., 32:].view(torch.int16), x[..., 32:].view(torch.int16))
    assert bool(torch.isfinite(y[..., :32]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_slices_of_a_fused_projection(interleaved) -> None:
    fused = _normal((50, 2, 10, 64), 1)
    rotary = mega_up.prepare_axial_rotary([32, 32], interleaved=interleaved, device=DEVICE)
    positions = _positions(2, (50,), torch.int32)
    q, k, v = fused.split((6, 2, 2), dim=2)
    want = mega_up.axial_rotary_sbhd(q.contiguous(), k.contiguous(), rotary, positions)
    got = mega_up.axial_rotary_sbhd(q, k, rotary, positions)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    kept = v.clone()
    mega_up.axial_rotary_sbhd(q, k, rotary, positions, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)
    every_second = mega_up.axial_rotary_sbhd(fused[::2, :, :6], None, rotary, positions[:, ::2])[0]
    assert torch.equal(every_second, mega_up.axial_rotary_sbhd(fused[::2, :, :6].contiguous(), None, rotary, positions[:, ::2].contiguous())[0])


@pytest.mark.gpu
def test_gradients_that_are_broadcast_or_missing() -> None:
    q, k = _normal((1, 9, 2, 64), 1).requires_grad_(), _normal((1, 9, 1, 64), 2).requires_grad_()
    rotary = mega_up.prepare_axial_rotary([64], device=DEVICE)
    positions = torch.arange(9, device=DEVICE)[None]
    a, b = mega_up.axial_rotary_bshd(q, k, rotary, positions)
    want = torch.autograd.grad(a, q, torch.ones_like(a), retain_graph=True)[0]
    got = torch.autograd.grad(a, q, torch.ones((), dtype=BF16, device=DEVICE).expand_as(a), retain_graph=True)[0]
    assert torch.equal(want, got)
    gq, gk = torch.autograd.grad(a, (q, k), torch.ones_like(a), allow_unused=True)
    assert torch.equal(gq, want) and (gk is None or not bool(gk.any()))


@pytest.mark.gpu
def test_another_stream_and_a_captured_graph() -> None:
    q, k = _normal((1, 300, 4, 128), 1), _normal((1, 300, 1, 128), 2)
    rotary = mega_up.prepare_axial_rotary([44, 42, 42], device=DEVICE)
    positions = _positions(3, (300,), torch.int64)
    want = mega_up.axial_rotary_bshd(q, k, rotary, positions)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = mega_up.axial_rotary_bshd(q, k, rotary, positions)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = mega_up.axial_rotary_bshd(q, k, rotary, positions)
    positions.add_(3)
    q.copy_(_normal(q.shape, 7))
    want = mega_up.axial_rotary_bshd(q, k, rotary, positions)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_offsets_behind_32_bits() -> None:
    stride = (1 << 31) // 2 + 64
    store = torch.empty(3 * stride, dtype=BF16, device=DEVICE)
    x = store.as_strided((3, 10, 2, 64), (stride, 128, 64, 1))
    x.copy_(_normal((1, 10, 2, 64), 1).expand_as(x))
    rotary = mega_up.prepare_axial_rotary([64], device=DEVICE)
    y, _ = mega_up.axial_rotary_bshd(x, None, rotary, torch.arange(10, device=DEVICE)[None])
    assert torch.equal(y[0], y[2]) and torch.equal(y[0], y[1])
    mega_up.axial_rotary_bshd(x, None, rotary, torch.arange(10, device=DEVICE)[None], out=(x,))
    assert torch.equal(x, y)


@pytest.mark.gpu
def test_refusals() -> None:
    q, k = _normal((2, 10, 4, 64), 1), _normal((2, 10, 2, 64), 2)
    rotary = mega_up.prepare_axial_rotary([32, 32], device=DEVICE)
    positions = _positions(2, (10,), torch.int64)
    call = mega_up.axial_rotary_bshd
    call(q, k, rotary, positions)
    for arguments in (
        (q, k[:1], rotary, positions), (q, k[..., :56], rotary, positions), (q[..., :56], None, rotary, positions),
        (q.float(), None, rotary, positions), (q[0], None, rotary, positions), (q, k, rotary, positions[:1]),
        (q, k, rotary, positions[:, :9]), (q, k, rotary, positions.double()), (q, k, rotary, positions.cpu()),
        (q, k, rotary, None), (q[:, :0], None, rotary, positions), (q[..., ::2], None, rotary, positions),
        (q[:, :, :1].expand(-1, -1, 4, -1), None, rotary, positions),
        (q, k, mega_up.prepare_axial_rotary([32, 32], device="cpu"), positions), (q, 3, rotary, positions),
    ):
        with pytest.raises(ValueError):
            call(*arguments)
    shifted = torch.empty(q.numel() + 8, dtype=BF16, device=DEVICE)[1 : 1 + q.numel()].view(q.shape)
    with pytest.raises(ValueError, match="aligned"):
        call(shifted, None, rotary, positions)
    for out in ((q,), (k, q), (q, k.float()), q):
        with pytest.raises(ValueError):
            call(q, k, rotary, positions, out=out)
    leaf = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        call(leaf, k, rotary, positions, out=(torch.empty_like(q), torch.empty_like(k)))


def test_copies_keep_no_plan() -> None:
    """Plans know the addresses of the tables: a copy, which has tables of its own, must not use them."""

    rotary = mega_up.prepare_axial_rotary([8, 4, 4], device="cpu")
    rotary.plans["some call"] = object()
    for other in (copy.copy(rotary), copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary))):
        assert other.plans == {} and other.axis_dims == (8, 4, 4) and other.pairs == 8
        assert torch.equal(other.turns, rotary.turns) and torch.equal(other.pair_axis, rotary.pair_axis)
        assert other.turns.data_ptr() % 8 == 0
    assert rotary.plans


@pytest.mark.gpu
def test_a_copy_outlives_its_original() -> None:
    rotary = mega_up.prepare_axial_rotary([32, 16, 16], device=DEVICE)
    q = torch.randn(30, 2, 64, device=DEVICE).to(BF16)
    positions = torch.arange(90, device=DEVICE).view(3, 30)
    want, _ = mega_up.axial_rotary_thd(q, None, rotary, positions)
    other = copy.deepcopy(rotary)
    rotary.turns.zero_()  # no turn at all where it is used by mistake
    assert torch.equal(mega_up.axial_rotary_thd(q, None, other, positions)[0], want)
    loss = (q.float().requires_grad_() * 2).to(BF16)
    saved = loss.square().sum()
    with torch.no_grad():
        mega_up.axial_rotary_thd(loss, None, other, positions, out=(loss,))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
