"""Neither operator has a forward-mode derivative: a tangent is refused, never dropped."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import megaup_b200 as mega_up
from _stubbed_launch import stub_launches

BF16 = torch.bfloat16


def _calls():
    x = torch.zeros(1, 8, 2, 64, dtype=BF16)
    rotary = mega_up.prepare_axial_rotary([64], device="cpu")
    positions = torch.zeros(1, 8)
    yield "attention", x, lambda q, k, v: mega_up.window_attention_bshd(q, k, v)
    yield "rotary", x, lambda q, k, v: mega_up.axial_rotary_bshd(q, k, rotary, positions)[0]


@pytest.mark.parametrize("operator", [0, 1], ids=["attention", "rotary"])
def test_a_tangent_is_refused(monkeypatch, operator) -> None:
    launches = stub_launches(monkeypatch)
    name, x, call = list(_calls())[operator]
    places = 3 if name == "attention" else 2
    call(x, x, x)
    with forward_ad.dual_level():
        call(x, x, x)  # an open level alone changes nothing
        for place in range(places):
            for leaf in (False, True):
                tensors = [x.clone().requires_grad_(leaf) for _ in range(3)]
                tensors[place] = forward_ad.make_dual(tensors[place], torch.ones_like(x))
                for grad in (torch.enable_grad(), torch.no_grad()):
                    with grad, pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*tensors)
    call(x, x, x)
    assert len(launches) == 3


@pytest.mark.parametrize("operator", [0, 1], ids=["attention", "rotary"])
def test_a_tangent_of_the_gradient_is_refused(monkeypatch, operator) -> None:
    stub_launches(monkeypatch)
    _, x, call = list(_calls())[operator]
    leaf = x.clone().requires_grad_()
    out = call(leaf, x, x)
    torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True)
    with forward_ad.dual_level():
        torch.autograd.grad(out, leaf, torch.ones_like(out), retain_graph=True)
        dual = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, leaf, dual)


def test_tangents_of_the_other_arguments(monkeypatch) -> None:
    stub_launches(monkeypatch)
    x = torch.zeros(1, 8, 2, 64, dtype=BF16)
    rotary = mega_up.prepare_axial_rotary([64], device="cpu")
    with forward_ad.dual_level():
        positions = forward_ad.make_dual(torch.zeros(1, 8), torch.ones(1, 8))
        with pytest.raises(NotImplementedError):
            mega_up.axial_rotary_bshd(x, None, rotary, positions)
        out = forward_ad.make_dual(x.clone(), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            mega_up.window_attention_bshd(x, x, x, out=out)
        with pytest.raises(NotImplementedError):
            mega_up.axial_rotary_bshd(x, None, rotary, torch.zeros(1, 8), out=(out,))
        # a refused `out` of another kind is refused as such
        with pytest.raises(ValueError):
            mega_up.axial_rotary_bshd(x, None, rotary, torch.zeros(1, 8), out=x)
