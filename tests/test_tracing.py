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
