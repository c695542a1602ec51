"""Tables and addresses that the C entries of the attention and the rotary positions refuse before anything is launched
(no GPU needed: every call here fails)."""

from __future__ import annotations

import ctypes

import pytest

from megaup_b200 import _native, build


@pytest.fixture(scope="module")
def library() -> ctypes.CDLL:
    build.ensure_built()
    return _native.lib()


def _packed(**changes) -> _native.MupWindowAttention:
    """Three sequences that every other check accepts; 4096 stands for an aligned address, and nothing reads it."""

    a = _native.MupWindowAttention()
    a.device = 63  # not there: a call that no check stops ends with the driver's error
    a.batch, a.heads_q, a.heads_kv, a.head_dim, a.seq_q, a.seq_k = 1, 4, 2, 64, 400, 500
    a.causal, a.left, a.right, a.sinks, a.scale = 1, 50, 0, 4, 0.125
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, name, 4096)
        setattr(a, name + "_strides", (ctypes.c_int64 * 3)(64, 256, 64))
    a.lse = 4096
    for name in ("sequences", "q_blocks_256", "q_blocks_128", "k_blocks_128", "workspace"):
        setattr(a, name, 4096)
    a.workspace_bytes = 1 << 30
    a.n_sequences, a.n_q_blocks_256, a.n_q_blocks_128, a.n_k_blocks_128, a.longest_q, a.longest_k = 3, 3, 4, 5, 300, 400
    for name, value in changes.items():
        setattr(a, name, value)
    return a


BOTH = ("mup_window_attention_forward", "mup_window_attention_backward")


@pytest.mark.parametrize(
    "changes",
    [
        dict(q_blocks_256=0), dict(q_blocks_128=0), dict(k_blocks_128=0), dict(q_blocks_256=4112), dict(q_blocks_128=4104),
        dict(k_blocks_128=4112), dict(sequences=4104), dict(n_q_blocks_256=1, n_q_blocks_128=2),
        dict(n_q_blocks_256=2, n_q_blocks_128=2), dict(lse=4098),
    ],
    ids=str,
)
def test_packed_tables(library, changes) -> None:
    for name in BOTH:
        assert getattr(library, name)(ctypes.byref(_packed(**changes)), None) == -1, (name, changes)
        assert b"window attention" in library.mup_last_error()


def test_a_gradient_needs_the_key_blocks(library) -> None:
    for changes in (dict(n_k_blocks_128=0, k_blocks_128=0), dict(n_k_blocks_128=3)):
        assert library.mup_window_attention_backward(ctypes.byref(_packed(**changes)), None) == -1
        assert b"k_blocks_128" in library.mup_last_error()
        # the forward pass does not read them
        assert library.mup_window_attention_forward(ctypes.byref(_packed(**changes)), None) == -2


def test_the_workspace_is_aligned(library) -> None:
    for changes in (dict(workspace=4104), dict(workspace=0), dict(workspace_bytes=64)):
        assert library.mup_window_attention_backward(ctypes.byref(_packed(**changes)), None) in (-1, -2), changes
    dense = dict(sequences=0, seq_q=1, seq_k=1 << 20, left=-1, sinks=0)
    for changes in (dict(workspace=4104), dict(workspace=0), dict(workspace_bytes=64), dict(kv_lengths=4097)):
        assert library.mup_window_attention_forward(ctypes.byref(_packed(**dense, **changes)), None) == -1, changes
    assert library.mup_window_attention_backward(ctypes.byref(_packed(workspace=4104)), None) == -1
    assert b"aligned" in library.mup_last_error()


def test_a_call_that_nothing_stops_reaches_the_driver(library) -> None:
    for name in BOTH:
        assert getattr(library, name)(ctypes.byref(_packed()), None) == -2


@pytest.mark.parametrize(
    "changes", [dict(positions=4100), dict(positions=4098, position_type=0), dict(turns=4100), dict(pair_axis=4098)], ids=str
)
def test_rotary_tables(library, changes) -> None:
    a = _native.MupAxialRotary()
    a.device, a.batch, a.rows, a.head_dim, a.pairs, a.axes, a.interleaved = 63, 1, 4, 64, 32, 1, 1
    a.heads[:] = (2, 0)
    a.q = a.q_out = a.positions = a.turns = a.pair_axis = 4096
    a.x_strides[:] = a.y_strides[:] = (512, 128, 64, 512, 128, 64)
    a.position_type = 1
    assert library.mup_axial_rotary_launch(ctypes.byref(a), None) == -2
    for name, value in changes.items():
        setattr(a, name, value)
    assert library.mup_axial_rotary_launch(ctypes.byref(a), None) == -1
    assert b"aligned" in library.mup_last_error()
