"""Tracers do not see the kernels: the calls that they would record without them are refused."""

from __future__ import annotations

import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import megaup_b200 as mega_up
from _stubbed_launch import stub_launches

BF16 = torch.bfloat16


def _operator(name):
    rotary, positions = mega_up.prepare_axial_rotary([64], device="cpu"), torch.zeros(1, 8)
    if name == "attention":
        return lambda x: mega_up.window_attention_bshd(x, x, x)
    return lambda x: mega_up.axial_rotary_bshd(x, None, rotary, positions)[0]


@pytest.mark.parametrize("name", ["attention", "rotary"])
def test_tracing(monkeypatch, name) -> None:
    launches = stub_launches(monkeypatch)
    call, x = _operator(name), torch.zeros(1, 8, 2, 64, dtype=BF16)
    leaf = x.clone().requires_grad_()
    for argument in (x, leaf):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(call)(argument)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(call, (x,), check_trace=False)
        traced = torch.jit.trace(call, (leaf,), check_trace=False)  # a node of its own
    before = len(launches)
    traced(leaf)
    assert len(launches) == before + 1
    call(x)
    assert len(launches) == before + 2


@pytest.mark.parametrize("gradient", [False, True])
@pytest.mark.parametrize("name", ["attention", "rotary"])
def test_torch_compile_runs_the_call_as_it_is(monkeypatch, name, gradient) -> None:
    """At a graph break: every run launches once, with the addresses of its own tensors."""

    launches = stub_launches(monkeypatch)
    torch._dynamo.reset()
    call = _operator(name)
    compiled = torch.compile(lambda x: call(x) + 1, backend="eager")
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        for _ in range(4):
            x = torch.zeros(1, 8, 2, 64, dtype=BF16, requires_grad=gradient)
            launches.clear()
            out = compiled(x)
            assert [block.q for _, block in launches] == [x.data_ptr()]
            if gradient:
                dout = torch.zeros_like(out)
                out.backward(dout)
                (_, backward) = launches[1]
                assert len(launches) == 2 and (backward.dout if name == "attention" else backward.q) == dout.data_ptr()
    torch._dynamo.reset()


@pytest.mark.gpu
def test_torch_compile_on_the_gpu() -> None:
    device = torch.device("cuda", 0)
    rotary = mega_up.prepare_axial_rotary([32, 32], device=device)
    positions = torch.arange(80, device=device).view(2, 40)
    leaf = torch.randn(1, 40, 4, 64, device=device).to(BF16).requires_grad_()

    def step(x):
        q, _ = mega_up.axial_rotary_bshd(x * 2, None, rotary, positions)
        return mega_up.window_attention_bshd(q, q, x, window=9) + 1

    torch._dynamo.reset()
    compiled = torch.compile(step, backend="eager")
    for _ in range(3):
        with torch.no_grad():
            leaf.normal_()
        want, got = step(leaf), compiled(leaf)
        assert torch.equal(want, got)
        dout = torch.randn_like(want)
        assert torch.equal(*(torch.autograd.grad(out, leaf, dout)[0] for out in (want, got)))
        with torch.no_grad():
            assert torch.equal(compiled(leaf), want)
    torch._dynamo.reset()
