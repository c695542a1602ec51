"""A whole attention layer as a user runs it: peer-write projection -> rotary positions -> window attention ->
head-shard pull projection, on one GPU with an emulated UP group. Every step is checked against 64 bits on the very
tensors it was given."""

from __future__ import annotations

import pytest
import torch

import _gpu_harness as h
import megaup_b200 as mega_up
from _attention_reference import HALF_BF16, assert_within, attention, rotate, visible
from test_axial_rotary import _angles, _frequencies

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _normal(shape, seed, factor=1.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * factor
    return x.to(BF16).to(h.DEVICE)


def _assert_linear(got, x, weight, bias, what):
    x, weight = x.double().cpu(), weight.double().cpu()
    want = x @ weight.T + (0.0 if bias is None else bias.double().cpu())
    # FP32 sums of K products over K / 16 steps, one rounding
    error = 2.0**-23 * (x.shape[-1] / 16 + 2) * (x.abs() @ weight.abs().T) + HALF_BF16 * want.abs() + 2.0**-20
    assert_within(got, want, error, what)


@pytest.mark.parametrize("kind", ["bshd", "sbhd"])
def test_a_layer_with_grouped_heads(kind) -> None:
    """One fused QKV projection; q and k are turned in place, in the slices of its result."""

    up, batch, local, heads, kv_heads, dim, width = 2, 2, 70, 8, 2, 128, 512
    own, own_kv, rows = heads // up, kv_heads // up, up * 70
    shape = (batch, local, 4, width // 4) if kind == "bshd" else (local, batch, 4, width // 4)
    xs = [_normal(shape, r) for r in range(up)]
    w_qkv = _normal(((heads + 2 * kv_heads) * dim, width), 10, width**-0.5)
    w_out, bias = _normal((width, heads * dim), 11, (heads * dim) ** -0.5), _normal((width,), 12, 0.02)
    runtimes = mega_up.initialize_emulated_group(up, hidden=(heads + 2 * kv_heads) * dim, max_rows=batch * local, device=h.DEVICE)
    sizes = dict(batch=batch, sequence=local, validate_group=False)
    project = [
        getattr(mega_up, f"prepare_peer_write_gemm_{kind}")(w_qkv, rt, heads=width // dim, head_dim=dim, **sizes)
        for rt in runtimes
    ]
    back = [
        getattr(mega_up, f"prepare_headshard_pull_gemm_{kind}")(w_out, rt, heads=heads, head_dim=dim, bias=bias, **sizes)
        for rt in runtimes
    ]
    fused = mega_up.emulated_peer_write(project, xs)
    axes = [44, 42, 42]
    rotary = mega_up.prepare_axial_rotary(axes, device=h.DEVICE)
    at = torch.arange(rows, device=h.DEVICE)
    positions = torch.stack((at // 35, at % 35 // 7, at % 7))
    angle = _angles(kind, positions, *_frequencies(axes, 10000.0, False))
    seen = visible(rows, rows, causal=True, left=50, right=0, sinks=3)
    seq_axis = 1 if kind == "bshd" else 0
    x_all = torch.cat(xs, seq_axis).flatten(-2)
    attended = []
    for r in range(up):
        # the rank's columns: its q heads, then its k, then its v heads
        columns = slice(r * (own + 2 * own_kv) * dim, (r + 1) * (own + 2 * own_kv) * dim)
        _assert_linear(fused[r].flatten(-2), x_all, w_qkv[columns], None, "projection")
        q, k, v = fused[r].split((own, own_kv, own_kv), dim=-2)
        before = q.clone(), k.clone()
        turned = getattr(mega_up, f"axial_rotary_{kind}")(q, k, rotary, positions, out=(q, k))
        for got, x in zip(turned, before):
            want, error = rotate(x, angle, interleaved=True)
            assert_within(got, want, error, "rotary")
        out = getattr(mega_up, f"window_attention_{kind}")(*turned, v, window=50, sinks=3)
        for b in range(batch):
            e = attention(*(x[b] if kind == "bshd" else x[:, b] for x in (q, k, v)), seen)
            assert_within(out[b] if kind == "bshd" else out[:, b], e.out, e.out_error, "attention")
        attended.append(out)
    result = mega_up.emulated_pull(back, attended)
    torch.cuda.synchronize()
    runtimes[0].check_status()
    whole = torch.cat(attended, -2).flatten(-2)
    for r in range(up):
        part = whole.narrow(seq_axis, r * local, local)
        _assert_linear(result[r].flatten(-2), part, w_out, bias, "output projection")


def test_a_packed_video_layer() -> None:
    """Three projections, clips split evenly over the group, both directions, packed rows."""

    up, heads, dim, width = 2, 4, 64, 256
    own = heads // up
    cu = (0, 40, 41, 150)  # local tokens of every clip
    local = cu[-1]
    xs = [_normal((local, width // dim, dim), r) for r in range(up)]
    weights = [_normal((heads * dim, width), 20 + i, width**-0.5) for i in range(3)]
    w_out = _normal((width, heads * dim), 24, (heads * dim) ** -0.5)
    runtimes = mega_up.initialize_emulated_group(up, hidden=heads * dim, max_rows=local, device=h.DEVICE)
    layouts = [mega_up.prepare_thd_layout(cu, rt) for rt in runtimes]
    qkv = []
    for w in weights:
        prepared = [
            mega_up.prepare_peer_write_gemm_thd(w, rt, heads=width // dim, head_dim=dim, layout=lay, validate_group=False)
            for rt, lay in zip(runtimes, layouts)
        ]
        qkv.append([x.clone() for x in mega_up.emulated_peer_write(prepared, xs)])
    sequences = mega_up.prepare_packed_sequences(layouts[0].cu_seqlens_out, device=h.DEVICE)
    rotary = mega_up.prepare_axial_rotary([16, 24, 24], interleaved=False, device=h.DEVICE)
    at = torch.cat([torch.arange(b - a) for a, b in zip(sequences.cu_seqlens_q, sequences.cu_seqlens_q[1:])]).to(h.DEVICE)
    positions = torch.stack((at // 12, at % 12 // 4, at % 4))
    angle = _angles("thd", positions, *_frequencies([16, 24, 24], 10000.0, False))
    attended = []
    for r in range(up):
        q, k, v = (x[r] for x in qkv)
        turned = mega_up.axial_rotary_thd(q, k, rotary, positions)
        for got, x in zip(turned, (q, k)):
            want, error = rotate(x, angle, interleaved=False)
            assert_within(got, want, error, "rotary")
        out = mega_up.window_attention_thd(*turned, v, sequences, causal=False, window=(30, 20), sinks=12)
        for a, b in zip(sequences.cu_seqlens_q, sequences.cu_seqlens_q[1:]):
            seen = visible(b - a, b - a, causal=False, left=30, right=20, sinks=12)
            e = attention(turned[0][a:b], turned[1][a:b], v[a:b], seen)
            assert_within(out[a:b], e.out, e.out_error, "attention")
        attended.append(out)
    back = [
        mega_up.prepare_headshard_pull_gemm_thd(w_out, rt, heads=heads, head_dim=dim, layout=lay, validate_group=False)
        for rt, lay in zip(runtimes, layouts)
    ]
    result = mega_up.emulated_pull(back, attended)
    torch.cuda.synchronize()
    runtimes[0].check_status()
    whole = torch.cat(attended, -2).flatten(-2)
    for r in range(up):
        # local row j of sample [a, b) on rank r stands at row UP*a + r*(b - a) + j - a
        rows = torch.cat([torch.arange(up * a + r * (b - a), up * a + (r + 1) * (b - a)) for a, b in zip(cu, cu[1:])])
        _assert_linear(result[r].flatten(-2), whole[rows.to(h.DEVICE)], w_out, None, "output projection")
