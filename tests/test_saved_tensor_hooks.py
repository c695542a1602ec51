"""Hooks of saved tensors may return what the forward pass saved with other strides, at other addresses: the backward
pass of the window attention goes by the tensors that it gets."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import megaup_b200 as mega_up
from _stubbed_launch import stub_launches

DEVICE = torch.device("cuda", 0)
BF16 = torch.bfloat16


def _contiguous(x):
    return x.clone(memory_format=torch.contiguous_format)


def _spread(x):
    """Rows that are no longer next to each other, still copied as they are."""

    return torch.empty(*x.shape[:-1], x.shape[-1] + 8, dtype=x.dtype, device=x.device)[..., : x.shape[-1]].copy_(x)


def _reversed_axes(x):
    """Strides that no copy of the kernels can follow."""

    return x.permute(*reversed(range(x.ndim))).contiguous().permute(*reversed(range(x.ndim)))


def _unaligned(x):
    return torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape).copy_(x)


UNPACK = [_contiguous, _spread, _reversed_axes, _unaligned]


def _fused(rows, device):
    generator = torch.Generator().manual_seed(rows)
    fused = torch.randn(2, rows, 8, 64, generator=generator).to(BF16).to(device)
    return [x.detach().requires_grad_() for x in fused.split((4, 2, 2), dim=2)]


@pytest.mark.parametrize("unpack", UNPACK)
def test_the_block_describes_what_the_hooks_return(monkeypatch, unpack) -> None:
    launches = stub_launches(monkeypatch)
    q, k, v = _fused(40, "cpu")
    returned = []

    def unpacked(x):
        returned.append(unpack(x))
        return returned[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpacked):
        out = mega_up.window_attention_bshd(q, k, v, window=7)
    out.sum().backward()
    (_, forward), (name, backward) = launches
    assert name == "mup_window_attention_backward" and list(forward.q_strides) == [40 * 8 * 64, 8 * 64, 64]
    for x, label in zip(returned, ("q", "k", "v", "out", "lse", "out_rest")):
        address = getattr(backward, label)
        assert address % 16 == 0
        if label in ("out", "lse", "out_rest"):
            assert address == x.data_ptr() or not x.is_contiguous() or x.data_ptr() % 16
            continue
        kept = address == x.data_ptr()
        assert kept == (unpack in (_contiguous, _spread))
        want = x.stride() if kept else torch.empty(x.shape, device="meta").stride()
        assert tuple(getattr(backward, label + "_strides")) == tuple(want[:3])


def test_without_hooks_the_block_is_the_forward_pass_s(monkeypatch) -> None:
    launches = stub_launches(monkeypatch)
    q, k, v = _fused(40, "cpu")
    mega_up.window_attention_bshd(q, k, v, window=7).sum().backward()
    (_, forward), (_, backward) = launches
    for name, x in (("q", q), ("k", k), ("v", v)):
        assert getattr(backward, name) == getattr(forward, name) == x.data_ptr()
        assert list(getattr(backward, name + "_strides")) == list(getattr(forward, name + "_strides"))


@pytest.mark.parametrize("unpack", [lambda x: x[..., :1], lambda x: x.float().half(), lambda x: x.to("meta")])
def test_other_tensors_are_refused(monkeypatch, unpack) -> None:
    launches = stub_launches(monkeypatch)
    q, k, v = _fused(40, "cpu")
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
        out = mega_up.window_attention_bshd(q, k, v)
    with pytest.raises(RuntimeError, match="hook of saved tensors"):
        out.sum().backward()
    assert len(launches) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("unpack", UNPACK)
@pytest.mark.parametrize("kind", ["bshd", "thd"])
def test_the_gradients_do_not_change(kind, unpack) -> None:
    q, k, v = _fused(300, DEVICE)
    sequences = mega_up.prepare_packed_sequences([0, 120, 600], device=DEVICE)

    def run():
        if kind == "bshd":
            out = mega_up.window_attention_bshd(q, k, v, window=90, sinks=3)
        else:
            out = mega_up.window_attention_thd(*(x.flatten(0, 1) for x in (q, k, v)), sequences, window=90, sinks=3)
        return out

    dout = torch.randn(600, 4, 64, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEVICE)
    out = run()
    want = torch.autograd.grad(out, (q, k, v), dout.view(out.shape))
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
        out = run()
    for a, b in zip(want, torch.autograd.grad(out, (q, k, v), dout.view(out.shape))):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_tensor_that_was_left_on_the_host_is_refused() -> None:
    q, k, v = _fused(40, DEVICE)
    for place in range(6):
        count = iter(range(6))
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x.cpu() if next(count) == place else x):
            out = mega_up.window_attention_bshd(q, k, v)
        with pytest.raises(RuntimeError, match="hook of saved tensors"):
            out.sum().backward()


@pytest.mark.gpu
def test_offloading_and_checkpointing() -> None:
    q, k, v = _fused(300, DEVICE)
    out = mega_up.window_attention_bshd(q, k, v, window=90)
    want = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    with torch.autograd.graph.save_on_cpu():
        out = mega_up.window_attention_bshd(q, k, v, window=90)
    for a, b in zip(want, torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
        assert torch.equal(a, b)
    out = checkpoint(lambda *x: mega_up.window_attention_bshd(*x, window=90), q, k, v, use_reentrant=False)
    for a, b in zip(want, torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
        assert torch.equal(a, b)
