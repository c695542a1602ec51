"""Sliding-window attention with sinks: the arguments it refuses (no GPU needed) and its results against 64 bits."""

from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch

import megaup_b200 as mega_up
from _attention_reference import HALF_BF16, assert_within, attention, visible
from megaup_b200 import _native, attention as module, build

DEVICE = torch.device("cuda", 0)
BF16 = torch.bfloat16

# --------------------------------------------------------------------------- without a GPU


@pytest.fixture(scope="module")
def library() -> ctypes.CDLL:
    build.ensure_built()
    return _native.lib()


def _block(**changes) -> _native.MupWindowAttention:
    """A call that every check accepts; nothing behind the addresses is touched before they fail."""

    a = _native.MupWindowAttention()
    a.batch, a.heads_q, a.heads_kv, a.head_dim, a.seq_q, a.seq_k = 2, 4, 2, 64, 100, 300
    a.causal, a.left, a.right, a.sinks, a.scale = 1, 50, 0, 4, 0.125
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, name, 4096)
        setattr(a, name + "_strides", (ctypes.c_int64 * 3)(300 * 256, 256, 64))
    a.lse = 4096
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize(
    "changes",
    [
        dict(head_dim=0), dict(head_dim=12), dict(head_dim=136), dict(heads_q=3), dict(heads_kv=0), dict(batch=0),
        dict(seq_q=0), dict(seq_k=0), dict(seq_k=(1 << 29) + 1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0),
        dict(scale=float("nan")), dict(scale=float("inf")), dict(q=0), dict(k=4104), dict(v=4098), dict(out=0),
        dict(q_strides=(ctypes.c_int64 * 3)(0, 256, 64)), dict(k_strides=(ctypes.c_int64 * 3)(1024, 257, 64)),
        dict(v_strides=(ctypes.c_int64 * 3)(1024, 256, -64)),
        dict(sequences=4096), dict(sequences=4096, batch=1, n_sequences=1, longest_q=101),
    ],
    ids=str,
)
def test_the_library_refuses(library, changes) -> None:
    for name in ("mup_window_attention_forward", "mup_window_attention_backward"):
        assert getattr(library, name)(ctypes.byref(_block(**changes)), None) in (-1, -3), changes
        assert b"window attention" in library.mup_last_error()


def test_the_library_refuses_a_gradient_it_cannot_compute(library) -> None:
    assert library.mup_window_attention_backward(ctypes.byref(_block(kv_lengths=4096)), None) == -3
    assert library.mup_window_attention_backward(ctypes.byref(_block(lse=0)), None) == -1
    assert library.mup_window_attention_backward(ctypes.byref(_block(dq=4097)), None) == -1
    assert library.mup_window_attention_forward(None, None) == -1
    assert library.mup_window_attention_workspace(None, None, None) == -1


def test_workspace_sizes(library) -> None:
    forward, backward = ctypes.c_uint64(), ctypes.c_uint64()

    def sizes(**changes):
        code = library.mup_window_attention_workspace(
            ctypes.byref(_block(**changes)), ctypes.byref(forward), ctypes.byref(backward)
        )
        assert code == 0
        return forward.value, backward.value

    # enough row blocks for the GPU: nothing to join; the backward pass keeps two floats per row
    assert sizes(batch=64, seq_q=4096, seq_k=4096, heads_q=4, sinks=0) == (0, 2 * 64 * 4 * 4096 * 4)
    few, _ = sizes(batch=1, seq_q=1, seq_k=1 << 20, left=-1, sinks=0)
    assert few > 0 and few % (4 * (64 + 1)) == 0


def test_the_workspace_is_bounded(library) -> None:
    """Sequences of very different lengths are cut for the longest one: that may not cost memory for every short one."""

    forward, backward = ctypes.c_uint64(), ctypes.c_uint64()
    sequences, longest = 4000, 1 << 20
    rows = sequences + longest
    for sinks, left, longest_q in ((4, 127, longest), (4, 127, 1), (0, -1, 1), (300, 1023, 16)):
        a = _block(
            batch=1, seq_q=rows if longest_q > 16 else longest_q * sequences, seq_k=rows, left=left, sinks=sinks,
            sequences=4096, n_sequences=sequences, n_q_blocks_256=sequences, n_q_blocks_128=2 * sequences + 8192,
            n_k_blocks_128=sequences + 8192, longest_q=longest_q, longest_k=longest,
        )
        assert library.mup_window_attention_workspace(ctypes.byref(a), ctypes.byref(forward), ctypes.byref(backward)) == 0
        per_row = 4 * 2 * 4 * a.seq_q
        assert forward.value <= 1 << 28 and backward.value - per_row <= 1 << 28, (sinks, left, longest_q)


def test_window_sides() -> None:
    assert module._window_sides(None, True) == (-1, 0)
    assert module._window_sides(None, False) == (-1, -1)
    assert module._window_sides(7, True) == (7, 0)
    assert module._window_sides(7, False) == (7, 7)
    assert module._window_sides((3, None), False) == (3, -1)
    assert module._window_sides((3, 0), True) == (3, 0)
    assert module._window_sides([1 << 40, 2], False) == (1 << 29, 2)
    for window, causal in ((-1, True), ((1, 2), True), ((1, 2, 3), False), ("x", False), (1.5, True), (True, False),
                           ((None, True), False)):
        with pytest.raises(ValueError):
            module._window_sides(window, causal)


def test_packed_sequences_on_the_host() -> None:
    s = mega_up.prepare_packed_sequences([0, 300, 300, 301], [0, 0, 5, 140], device="cpu")
    assert s.sequences.tolist() == [[0, 300, 0, 0], [300, 0, 0, 5], [300, 1, 5, 135]]
    table = s.sequences.tolist()

    def blocks(*pairs):
        return [[sequence, row, *table[sequence], 0, 0] for sequence, row in pairs]

    assert s.q_blocks_256.tolist() == blocks((0, 256), (0, 0), (2, 0))
    assert s.q_blocks_128.tolist() == blocks((0, 256), (0, 128), (0, 0), (2, 0))
    assert sorted(s.k_blocks_128.tolist()) == blocks((1, 0), (2, 0), (2, 128))
    assert (s.longest_q, s.longest_k, s.num_sequences) == (300, 135, 3)
    layout = mega_up.prepare_packed_sequences(torch.tensor([0, 4], dtype=torch.int32), device="cpu")
    assert layout.cu_seqlens_k == (0, 4)
    for bad in (([1, 2],), ([0, 2, 1],), ([0],), ([0, 0],), ([0, 4], [0, 2, 4])):
        with pytest.raises(ValueError):
            mega_up.prepare_packed_sequences(*bad, device="cpu")


def test_host_tensors_are_refused() -> None:
    x = torch.zeros(1, 4, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        mega_up.window_attention_bshd(x, x, x)
    with pytest.raises(ValueError):
        mega_up.window_attention_bshd(x, 3, x)
    with pytest.raises(TypeError):
        mega_up.window_attention_thd(x[0], x[0], x[0], [0, 4])


# --------------------------------------------------------------------------- on the GPU


def _normal(shape, seed, factor=1.0):
    generator = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=generator) * factor).to(BF16).to(DEVICE)


def _rows(x, kind, b):
    """[rows, heads, dim] of sequence ``b``."""

    return x[b] if kind == "bshd" else x[:, b]


def _shape(kind, batch, rows, heads, dim):
    return (batch, rows, heads, dim) if kind == "bshd" else (rows, batch, heads, dim)


def _window(causal, left, right):
    return left if causal else (left, right)


CASES = [
    # kind, batch, queries, keys, heads, kv heads, dim, causal, left, right, sinks
    ("bshd", 1, 1, 1, 1, 1, 64, True, None, 0, 0),
    ("bshd", 2, 1, 1, 4, 2, 128, False, 0, 0, 0),
    ("sbhd", 2, 127, 127, 2, 2, 64, True, None, 0, 0),
    ("bshd", 1, 128, 128, 2, 1, 128, True, 0, 0, 0),
    ("bshd", 1, 129, 257, 3, 1, 128, True, 64, 0, 1),
    ("sbhd", 3, 255, 255, 4, 4, 64, False, 17, 40, 0),
    ("bshd", 1, 257, 129, 2, 2, 128, True, None, 0, 0),  # the first 128 rows see nothing
    ("bshd", 1, 300, 40, 2, 1, 64, False, 10, 10, 0),  # rows at negative positions see nothing
    ("bshd", 1, 300, 40, 2, 1, 64, False, 10, 10, 3),  # ... but the sinks
    ("bshd", 1, 384, 384, 8, 1, 128, True, 100, 0, 200),  # a sink tile that is cut
    ("bshd", 2, 200, 650, 6, 3, 96, True, 128, 0, 4),
    ("sbhd", 1, 513, 513, 2, 2, 40, False, None, 0, 0),
    ("bshd", 1, 513, 513, 2, 2, 8, False, 0, None, 130),
    ("bshd", 1, 90, 1000, 5, 5, 128, False, None, None, 0),
    ("bshd", 1, 640, 640, 2, 1, 72, True, 127, 0, 1000),  # more sinks than keys
    ("bshd", 1, 1000, 1000, 4, 2, 128, True, 1 << 40, 0, 0),
    ("sbhd", 2, 700, 700, 2, 1, 120, False, 130, 5, 129),
    ("bshd", 2, 1, 300, 128, 1, 64, True, None, 0, 0),  # a group as large as a tile
    ("sbhd", 1, 3, 400, 48, 2, 128, True, 150, 0, 9),  # 24 heads of a group, packed by eight
    ("bshd", 1, 20, 2500, 6, 2, 128, False, 700, 0, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("factor", [1.0, 6.0], ids=["flat", "peaked"])
def test_forward_and_backward(case, factor) -> None:
    kind, batch, queries, keys, heads, kv_heads, dim, causal, left, right, sinks = case
    q = _normal(_shape(kind, batch, queries, heads, dim), 1, factor).requires_grad_()
    k = _normal(_shape(kind, batch, keys, kv_heads, dim), 2).requires_grad_()
    v = _normal(_shape(kind, batch, keys, kv_heads, dim), 3).requires_grad_()
    dout = _normal(_shape(kind, batch, queries, heads, dim), 4)
    call = getattr(mega_up, f"window_attention_{kind}")
    out, lse = call(q, k, v, causal=causal, window=_window(causal, left, right), sinks=sinks, return_lse=True)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    again = torch.autograd.grad(call(q, k, v, causal=causal, window=_window(causal, left, right), sinks=sinks), (q, k, v), dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "two runs differ"
    with torch.no_grad():
        plain = call(q, k, v, causal=causal, window=_window(causal, left, right), sinks=sinks)
    assert torch.equal(plain, out)
    seen = visible(queries, keys, causal=causal, left=left, right=right, sinks=sinks)
    for b in range(batch):
        e = attention(*(_rows(x, kind, b) for x in (q, k, v)), seen, dout=_rows(dout, kind, b))
        assert_within(_rows(out, kind, b), e.out, e.out_error, "out")
        assert_within(lse[b], e.lse, e.lse_error, "lse")
        for name, got, want, error in zip(("dq", "dk", "dv"), grads, (e.dq, e.dk, e.dv), (e.dq_error, e.dk_error, e.dv_error)):
            assert_within(_rows(got, kind, b), want, error, name)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (5, 5, 64), (12, 4, 128), (16, 1, 80), (1, 1, 128)], ids=str)
@pytest.mark.parametrize("queries", [1, 2, 9, 33])
@pytest.mark.parametrize("kind", ["bshd", "sbhd"])
def test_tokens_over_a_cache(kind, queries, heads, kv_heads, dim) -> None:
    """Every length from nothing to the whole cache; what lies behind a length, and between the sinks and the
    window of the whole call, is NaN."""

    capacity, left, sinks = 700, 100, 5
    lengths = [0, 1, queries, 64, 128, 129, 640, capacity, capacity + 50, -3]
    batch = len(lengths)
    q = _normal(_shape(kind, batch, queries, heads, dim), 1)
    k = _normal(_shape(kind, batch, capacity, kv_heads, dim), 2)
    v = _normal(_shape(kind, batch, capacity, kv_heads, dim), 3)
    for b, n in enumerate(lengths):
        n = min(max(n, 0), capacity)
        for x in (k, v):
            rows = _rows(x, kind, b)
            rows[n:] = float("nan")
            rows[sinks : max(sinks, n - queries - left)] = float("nan")
    out = torch.full(_shape(kind, batch, queries, heads, dim), 7.0, dtype=BF16, device=DEVICE)
    call = getattr(mega_up, f"window_attention_{kind}")
    device_lengths = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    got, lse = call(q, k, v, window=left, sinks=sinks, kv_lengths=device_lengths, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    for b, n in enumerate(lengths):
        n = min(max(n, 0), capacity)
        seen = visible(queries, n, causal=True, left=left, right=0, sinks=sinks)
        e = attention(_rows(q, kind, b), _rows(k, kind, b)[:n], _rows(v, kind, b)[:n], seen)
        assert_within(_rows(out, kind, b), e.out, e.out_error, f"out of length {n}")
        assert_within(lse[b], e.lse, e.lse_error, f"lse of length {n}")


def _packed(lengths_q, lengths_k, heads, kv_heads, dim, *, seed=0, factor=1.0):
    q = _normal((sum(lengths_q), heads, dim), seed + 1, factor)
    k = _normal((sum(lengths_k), kv_heads, dim), seed + 2)
    v = _normal((sum(lengths_k), kv_heads, dim), seed + 3)
    dout = _normal((sum(lengths_q), heads, dim), seed + 4)
    cu = lambda n: [0] + torch.tensor(n).cumsum(0).tolist()  # noqa: E731
    return q, k, v, dout, mega_up.prepare_packed_sequences(cu(lengths_q), cu(lengths_k), device=DEVICE)


@pytest.mark.gpu
@pytest.mark.parametrize(
    "lengths_q,lengths_k,heads,kv_heads,dim,causal,left,right,sinks",
    [
        ([1, 0, 128, 129, 300, 5], [1, 7, 128, 129, 300, 5], 4, 2, 128, True, 60, 0, 3),
        ([100, 28, 1, 500], [100, 0, 400, 130], 3, 3, 64, False, 100, 20, 140),
        ([1, 1, 1, 1], [900, 1, 0, 257], 8, 1, 128, True, None, 0, 0),
        ([2, 1, 3], [900, 100, 257], 10, 2, 96, True, 300, 0, 1),
        ([640], [640], 2, 1, 64, False, None, None, 0),
        ([31, 7], [31, 7], 8, 2, 64, True, 4, 0, 2),
    ],
    ids=str,
)
def test_packed_sequences(lengths_q, lengths_k, heads, kv_heads, dim, causal, left, right, sinks) -> None:
    q, k, v, dout, sequences = _packed(lengths_q, lengths_k, heads, kv_heads, dim)
    for x in (q, k, v):
        x.requires_grad_()
    out, lse = mega_up.window_attention_thd(
        q, k, v, sequences, causal=causal, window=_window(causal, left, right), sinks=sinks, return_lse=True
    )
    grads = torch.autograd.grad(out, (q, k, v), dout)
    a = c = 0
    for n, m in zip(lengths_q, lengths_k):
        qs, ks = slice(a, a + n), slice(c, c + m)
        seen = visible(n, m, causal=causal, left=left, right=right, sinks=sinks)
        e = attention(q[qs], k[ks], v[ks], seen, dout=dout[qs])
        assert_within(out[qs], e.out, e.out_error, "out")
        assert_within(lse[:, qs], e.lse, e.lse_error, "lse")
        assert_within(grads[0][qs], e.dq, e.dq_error, "dq")
        assert_within(grads[1][ks], e.dk, e.dk_error, "dk")
        assert_within(grads[2][ks], e.dv, e.dv_error, "dv")
        a, c = a + n, c + m


@pytest.mark.gpu
@pytest.mark.parametrize("sinks", [4, 200])
def test_one_long_sequence_among_many_short_ones(sinks) -> None:
    lengths = [1 + i % 3 for i in range(300)] + [1500] + [1 + i % 5 for i in range(200)]
    q, k, v, dout, sequences = _packed(lengths, lengths, 4, 2, 64, seed=11)
    for x in (q, k, v):
        x.requires_grad_()
    out = mega_up.window_attention_thd(q, k, v, sequences, window=60, sinks=sinks)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    a = 0
    for n in lengths:
        rows = slice(a, a + n)
        e = attention(q[rows], k[rows], v[rows], visible(n, n, causal=True, left=60, right=0, sinks=sinks), dout=dout[rows])
        assert_within(out[rows], e.out, e.out_error, "out")
        for got, want, error in zip(grads, (e.dq, e.dk, e.dv), (e.dq_error, e.dk_error, e.dv_error)):
            assert_within(got[rows], want, error, "gradient")
        a += n


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks,capacity", [(None, 0, 9000), (300, 4, 9000), (None, 0, 700)])
def test_a_captured_token_over_a_growing_cache(window, sinks, capacity) -> None:
    """One graph, replayed while the cache fills: the lengths and the new rows are read at every replay."""

    batch, heads, kv_heads, dim = 3, 8, 2, 128
    q = _normal((batch, 1, heads, dim), 1)
    k, v = (torch.full((batch, capacity, kv_heads, dim), float("nan"), dtype=BF16, device=DEVICE) for _ in range(2))
    lengths = torch.tensor([capacity - 400, 5, 300], dtype=torch.int32, device=DEVICE)
    rows = [_normal((batch, capacity, kv_heads, dim), s) for s in (2, 3)]
    for b, n in enumerate(lengths.tolist()):
        k[b, :n], v[b, :n] = rows[0][b, :n], rows[1][b, :n]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = mega_up.window_attention_bshd(q, k, v, window=window, sinks=sinks, kv_lengths=lengths)
    for step in range(3):
        for b, n in enumerate(lengths.tolist()):
            k[b, n : n + 130], v[b, n : n + 130] = rows[0][b, n : n + 130], rows[1][b, n : n + 130]
        lengths.add_(130)
        q.copy_(_normal(q.shape, 20 + step))
        graph.replay()
        torch.cuda.synchronize()
        for b, n in enumerate(lengths.tolist()):
            e = attention(q[b], k[b, :n], v[b, :n], visible(1, n, causal=True, left=window, right=0, sinks=sinks))
            assert_within(out[b], e.out, e.out_error, f"step {step}, length {n}")


@pytest.mark.gpu
def test_two_streams_at_once_and_out_in_place_of_q() -> None:
    calls = []
    for s, (queries, keys) in enumerate(((1, 5000), (200, 5000), (2000, 2000), (7, 640))):
        q, k, v = _normal((1, queries, 4, 128), s), _normal((1, keys, 2, 128), 10 + s), _normal((1, keys, 2, 128), 20 + s)
        calls.append((q, k, v, mega_up.window_attention_bshd(q, k, v, window=1000, sinks=2)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    results = [[] for _ in calls]
    for _ in range(10):
        for (q, k, v, _), stream, kept in zip(calls, streams, results):
            with torch.cuda.stream(stream):
                kept.append(mega_up.window_attention_bshd(q, k, v, window=1000, sinks=2))
    torch.cuda.synchronize()
    for (q, k, v, want), kept in zip(calls, results):
        assert all(torch.equal(want, x) for x in kept)
        own = q.clone()
        assert torch.equal(mega_up.window_attention_bshd(own, k, v, window=1000, sinks=2, out=own), want)


@pytest.mark.gpu
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), torch.finfo(BF16).min])
def test_a_sequence_keeps_to_itself(poison) -> None:
    lengths = [130, 200, 70, 300]
    q, k, v, dout, sequences = _packed(lengths, lengths, 4, 2, 128, seed=7)
    settings = dict(window=50, sinks=2)

    def run():
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = mega_up.window_attention_thd(*leaves, sequences, **settings)
        return (out, *torch.autograd.grad(out, leaves, dout))

    before = [x.detach().clone() for x in run()]
    for x in (q, k, v, dout):
        x[130:330] = poison
    after = run()
    for a, b in zip(before, after):
        assert torch.equal(a[:130], b[:130]) and torch.equal(a[330:], b[330:])


@pytest.mark.gpu
def test_unseen_keys_may_hold_anything() -> None:
    q, k, v = (_normal((1, 300, 2, 64), s) for s in (1, 2, 3))
    k = torch.cat((_normal((1, 700, 2, 64), 5), k), 1)
    v = torch.cat((_normal((1, 700, 2, 64), 6), v), 1)
    want = mega_up.window_attention_bshd(q, k, v, window=90, sinks=6)
    for x in (k, v):
        x[:, 6:610] = float("nan")  # before the first row's window
    assert torch.equal(mega_up.window_attention_bshd(q, k, v, window=90, sinks=6), want)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["k", "v", "both"])
@pytest.mark.parametrize("causal, queries, dim", [(True, 300, 64), (True, 100, 128), (False, 77, 128)])
def test_unseen_keys_have_no_gradient_whatever_they_hold(causal, queries, dim, where) -> None:
    q, dout = _normal((1, queries, 4, dim), 1), _normal((1, queries, 4, dim), 2)
    k, v = _normal((1, 1000, 2, dim), 3), _normal((1, 1000, 2, dim), 4)
    low = 1000 - queries - 90  # the first key of the first row's window

    def run():
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = mega_up.window_attention_bshd(*leaves, causal=causal, window=90, sinks=6)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    want = run()
    for x in {"k": (k,), "v": (v,), "both": (k, v)}[where]:
        x[:, 6:low] = float("nan")
    for a, b in zip(want, run()):
        assert torch.equal(a, b)
    assert not want[2][:, 6:low].any() and not want[3][:, 6:low].any()


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("settings, blind", [
    (dict(window=50, sinks=3), 130), (dict(), 130), (dict(causal=False, window=(40, 20)), 110),
])
def test_rows_that_see_nothing_have_no_gradient_whatever_they_hold(settings, blind, packed) -> None:
    queries, keys = 300, 170  # the first rows stand before the first key
    rows = 2 * queries if packed else queries
    q, dout = _normal((rows, 4, 64), 1), _normal((rows, 4, 64), 2)
    k, v = _normal((rows // queries * keys, 2, 64), 3), _normal((rows // queries * keys, 2, 64), 4)
    sequences = mega_up.prepare_packed_sequences([0, queries, 2 * queries], [0, keys, 2 * keys], device=DEVICE) if packed else None

    def run():
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        if packed:
            out = mega_up.window_attention_thd(*leaves, sequences, **settings)
        else:
            out = mega_up.window_attention_bshd(*(x[None] for x in leaves), **settings)[0]
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    want = run()
    for start in range(0, rows, queries):
        assert not want[0][start : start + blind].any() and not want[1][start : start + blind].any()
        assert want[0][start + blind].any() and want[1][start + blind].any()
        q[start : start + blind] = float("nan")
        dout[start : start + blind] = float("inf")
    for a, b in zip(want, run()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_slices_of_a_fused_projection_and_out() -> None:
    heads, kv_heads, dim, rows = 4, 2, 64, 333
    fused = _normal((rows, 2, heads + 2 * kv_heads, dim), 1)
    q, k, v = fused.split((heads, kv_heads, kv_heads), dim=2)
    want = mega_up.window_attention_sbhd(q.contiguous(), k.contiguous(), v.contiguous(), window=40)
    assert torch.equal(mega_up.window_attention_sbhd(q, k, v, window=40), want)
    room = torch.full((rows + 2, 2, heads + 3, dim), 5.0, dtype=BF16, device=DEVICE)
    out = room[1:-1, :, 1 : 1 + heads]
    assert mega_up.window_attention_sbhd(q, k, v, window=40, out=out) is out
    assert torch.equal(out, want)
    room[1:-1, :, 1 : 1 + heads] = 5.0
    assert bool((room == 5.0).all()), "something outside of out was written"


@pytest.mark.gpu
def test_gradients_that_are_broadcast_or_transposed() -> None:
    q, k, v = (_normal((2, 150, 2, 64), s).requires_grad_() for s in (1, 2, 3))
    out = mega_up.window_attention_bshd(q, k, v, window=30)
    ones = torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)
    for a, b in zip(ones, torch.autograd.grad(out.float().sum(), (q, k, v), retain_graph=True)):
        assert torch.equal(a, b)
    for a, b in zip(ones, torch.autograd.grad(out, (q, k, v), torch.ones((), dtype=BF16, device=DEVICE).expand_as(out), retain_graph=True)):
        assert torch.equal(a, b)
    dout = _normal((2, 150, 2, 64), 9)
    strided = torch.empty(2, 2, 150, 64, dtype=BF16, device=DEVICE).transpose(1, 2).copy_(dout)
    assert not strided.is_contiguous()
    for a, b in zip(torch.autograd.grad(out, (q, k, v), dout, retain_graph=True), torch.autograd.grad(out, (q, k, v), strided)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_the_gradient_is_the_slope() -> None:
    """Along a direction, the central difference of the 64-bit loss against the kernel's gradient."""

    queries, keys, heads, kv_heads, dim = 140, 200, 4, 2, 64
    q, k, v = _normal((queries, heads, dim), 1), _normal((keys, kv_heads, dim), 2), _normal((keys, kv_heads, dim), 3)
    dout = _normal((queries, heads, dim), 4)
    seen = visible(queries, keys, causal=True, left=70, right=0, sinks=3)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = mega_up.window_attention_bshd(*(x[None] for x in leaves), window=70, sinks=3)
    grads = torch.autograd.grad(out, leaves, dout[None])
    e = attention(q, k, v, seen, dout=dout)
    errors = (e.dq_error, e.dk_error, e.dv_error)
    h = 2.0**-10
    for i, x in enumerate((q, k, v)):
        direction = torch.randn(x.shape, generator=torch.Generator().manual_seed(20 + i), dtype=torch.float64)

        def loss(step):
            moved = [y.double().cpu() for y in (q, k, v)]
            moved[i] = moved[i] + step * direction
            return float((attention(*moved, seen).out * dout.double().cpu()).sum())

        slope = (loss(h) - loss(-h)) / (2 * h)
        curve = abs(loss(2 * h) - loss(-2 * h) - 2 * (loss(h) - loss(-h))) / (4 * h)  # the difference's own error
        allowed = float((errors[i] * direction.abs()).sum()) + curve + 1e-9 * abs(slope)
        got = float((grads[i].double().cpu() * direction).sum())
        assert abs(got - slope) <= allowed, (i, got, slope, allowed)


@pytest.mark.gpu
def test_another_stream_and_a_captured_graph() -> None:
    q, k, v = (_normal((1, 400, 2, 128), s).requires_grad_() for s in (1, 2, 3))
    dout = _normal((1, 400, 2, 128), 4)

    def step():
        out = mega_up.window_attention_bshd(q, k, v, window=100, sinks=2)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))

    want = [x.clone() for x in step()]
    token = _normal((1, 1, 2, 128), 5)
    want_token = mega_up.window_attention_bshd(token, k.detach(), v.detach())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [x.clone() for x in step()]
        got_token = mega_up.window_attention_bshd(token, k.detach(), v.detach())
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(want_token, got_token)
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graphs, captured = [], []
    for _ in range(2):  # two graphs of one call: each has its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.append((*step(), mega_up.window_attention_bshd(token, k.detach(), v.detach())))
        graphs.append(graph)
    for x in (q, k, v):
        x.data.copy_(_normal(x.shape, 11))
    want = [x.clone() for x in (*step(), mega_up.window_attention_bshd(token, k.detach(), v.detach()))]
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in captured:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_offsets_behind_32_bits() -> None:
    """A cache of more than 2^31 elements: the last sequence and the last rows."""

    rows, kv_heads, dim = 2100, 2, 128
    stride = (1 << 31) // 4 + 4096
    store = torch.empty(5 * stride, dtype=BF16, device=DEVICE)
    k = store.as_strided((5, rows, kv_heads, dim), (stride, kv_heads * dim, dim, 1))
    v = store.as_strided((5, rows, kv_heads, dim), (stride, kv_heads * dim, dim, 1), rows * kv_heads * dim)
    k.copy_(_normal((1, rows, kv_heads, dim), 1).expand_as(k))
    v.copy_(_normal((1, rows, kv_heads, dim), 2).expand_as(v))
    q = _normal((1, 3, 8, dim), 3).expand(5, -1, -1, -1).contiguous()
    out = mega_up.window_attention_bshd(q, k, v, window=1000, sinks=4)
    for b in range(1, 5):
        assert torch.equal(out[b], out[0])
    e = attention(q[4], k[4], v[4], visible(3, rows, causal=True, left=1000, right=0, sinks=4))
    assert_within(out[4], e.out, e.out_error, "out")


@pytest.mark.gpu
def test_refusals() -> None:
    q, k = _normal((2, 40, 4, 64), 1), _normal((2, 50, 2, 64), 2)
    call = mega_up.window_attention_bshd
    bad = [
        (q, k, k[:, :40]), (q, k[:1], k[:1]), (q[..., :32], k, k), (q[:, :, :3], k, k), (q.float(), k, k), (q, k.cpu(), k),
        (q[0], k, k), (q[:, :0], k, k), (q, k[:, :0], k[:, :0]), (q.transpose(2, 3).contiguous().transpose(2, 3), k, k),
        (q[:, :1].expand(-1, 40, -1, -1), k, k), (q[..., :60], k[..., :60], k[..., :60]),
        (_normal((2, 40, 4, 136), 1), _normal((2, 40, 4, 136), 1), _normal((2, 40, 4, 136), 1)),
    ]
    for arguments in bad:
        with pytest.raises(ValueError):
            call(*arguments)
    shifted = torch.empty(q.numel() + 8, dtype=BF16, device=DEVICE)[1 : 1 + q.numel()].view(q.shape)
    with pytest.raises(ValueError, match="aligned"):
        call(shifted, k, k)
    for settings in (
        dict(window=-1), dict(window=(1, 1)), dict(sinks=-1), dict(sinks=1.0), dict(sinks=True), dict(scale=0.0),
        dict(scale=float("nan")), dict(scale=-1.0), dict(kv_lengths=torch.zeros(2, device=DEVICE)),
        dict(kv_lengths=torch.zeros(3, dtype=torch.int32, device=DEVICE)), dict(kv_lengths=torch.zeros(2, dtype=torch.int32)),
        dict(out=torch.empty_like(k)), dict(out=q.float()), dict(out=q.transpose(2, 3).contiguous().transpose(2, 3)),
    ):
        with pytest.raises(ValueError):
            call(q, k, k, **settings)
    call(q, k, k, sinks=1)
    with pytest.raises(ValueError):
        call(q, k, k, sinks=True)  # also after the same call with 1
    leaf = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        call(leaf, k, k, out=torch.empty_like(q))
    with pytest.raises(ValueError, match="gradient"):
        call(leaf, k, k, kv_lengths=torch.full((2,), 50, dtype=torch.int32, device=DEVICE))
    out = call(leaf, k, k)
    (gradient,) = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError):
        gradient.sum().backward()
    sequences = mega_up.prepare_packed_sequences([0, 40], [0, 50], device=DEVICE)
    mega_up.window_attention_thd(q[0], k[0], k[0], sequences)
    with pytest.raises(ValueError):
        mega_up.window_attention_thd(q[0], k[0, :49], k[0, :49], sequences)
    with pytest.raises(ValueError):
        mega_up.window_attention_thd(q[0], k[0], k[0], mega_up.prepare_packed_sequences([0, 40], [0, 50], device="cpu"))


@pytest.mark.gpu
def test_scale_is_used() -> None:
    q, k, v = _normal((1, 100, 2, 64), 1), _normal((1, 100, 2, 64), 2), _normal((1, 100, 2, 64), 3)
    out = mega_up.window_attention_bshd(q, k, v, scale=0.5)
    e = attention(q[0], k[0], v[0], visible(100, 100, causal=True, left=None, right=0, sinks=0), scale=0.5)
    assert_within(out[0], e.out, e.out_error, "out")
    assert e.out_error.max() < 32 * HALF_BF16


def test_copies_of_packed_sequences_keep_no_plan() -> None:
    """Plans know the addresses of the tables: a copy, which has tables of its own, must not use them."""

    sequences = mega_up.prepare_packed_sequences([0, 5, 300], device="cpu")
    sequences.plans["some call"] = object()
    for other in (copy.copy(sequences), copy.deepcopy(sequences), pickle.loads(pickle.dumps(sequences))):
        assert other.plans == {} and other.cu_seqlens_q == (0, 5, 300) and other.longest_k == 295
        assert torch.equal(other.q_blocks_128, sequences.q_blocks_128) and other.q_blocks_128.data_ptr() % 16 == 0
    assert sequences.plans


@pytest.mark.gpu
def test_a_copied_description_outlives_its_original() -> None:
    lengths = [130, 300]
    q, k, v, _, sequences = _packed(lengths, lengths, 4, 2, 64, seed=3)
    want = mega_up.window_attention_thd(q, k, v, sequences, window=40)
    other = copy.deepcopy(sequences)
    for table in (sequences.sequences, sequences.q_blocks_256, sequences.q_blocks_128, sequences.k_blocks_128):
        table.zero_()  # blocks without rows or keys: harmless where they are used by mistake
    assert torch.equal(mega_up.window_attention_thd(q, k, v, other, window=40), want)


@pytest.mark.gpu
def test_a_scale_that_changes_in_place() -> None:
    q, k, v = (_normal((1, 50, 2, 64), s) for s in (1, 2, 3))
    scale, causal = torch.tensor(0.125), torch.tensor(True)
    for value, flag in ((0.125, True), (0.5, True), (0.5, False)):
        scale.fill_(value), causal.fill_(flag)
        want = mega_up.window_attention_bshd(q, k, v, scale=value, causal=flag)
        assert torch.equal(mega_up.window_attention_bshd(q, k, v, scale=scale, causal=causal), want)


@pytest.mark.gpu
def test_a_result_written_over_a_saved_tensor() -> None:
    x, k, v = (_normal((1, 20, 2, 64), s) for s in (1, 2, 3))
    q = x.requires_grad_() * 2
    loss = q.square().sum()
    with torch.no_grad():
        mega_up.window_attention_bshd(q, k, v, out=q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
