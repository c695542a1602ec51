"""What a call of the window attention accepts does not depend on the calls before it."""

from __future__ import annotations

import enum

import numpy as np
import pytest
import torch

import megaup_b200 as mega_up
from _stubbed_launch import stub_launches
from megaup_b200 import attention

BF16 = torch.bfloat16


class Width(enum.IntEnum):
    FIVE = 5


@pytest.mark.parametrize(
    "accepted, causal, refused",
    [
        (1, True, [True, 1.0, np.int64(1), (True, 0), (1.0, None), "1"]),
        (0, True, [False, 0.0, (False, 0), (0, False)]),
        ((1, 0), False, [(True, 0), (1, False), (1.0, 0), [True, 0], (1, 0.0), np.array([1, 0])]),
        (5, False, [5.0, (5.0, 5), (5, np.int32(5))]),
        (None, False, [(None, None, None), float("inf"), ()]),
    ],
    ids=str,
)
def test_windows(monkeypatch, accepted, causal, refused) -> None:
    stub_launches(monkeypatch)
    x = torch.zeros(1, 8, 2, 64, dtype=BF16)
    for when in ("first", "after the same call with what it equals"):
        for window in refused:
            with pytest.raises(ValueError):
                mega_up.window_attention_bshd(x, x, x, causal=causal, window=window)
        mega_up.window_attention_bshd(x, x, x, causal=causal, window=accepted)


@pytest.mark.parametrize("window", [[3, 4], (3, 4), [None, 2], Width.FIVE, [7, None]], ids=str)
def test_forms_of_a_window_keep_their_plan(monkeypatch, window) -> None:
    launches = stub_launches(monkeypatch)
    x = torch.zeros(1, 8, 2, 64, dtype=BF16)
    for _ in range(3):
        mega_up.window_attention_bshd(x, x, x, causal=False, window=window)
    left, right = window if isinstance(window, (list, tuple)) else (window, window)
    want = tuple(-1 if side is None else side for side in (left, right))
    assert [(a.left, a.right) for _, a in launches] == [want] * 3
    assert len(attention._PLANS) == 1


def test_a_list_that_changes(monkeypatch) -> None:
    launches = stub_launches(monkeypatch)
    x = torch.zeros(1, 8, 2, 64, dtype=BF16)
    window = [3, 4]
    mega_up.window_attention_bshd(x, x, x, causal=False, window=window)
    window[0] = 6
    mega_up.window_attention_bshd(x, x, x, causal=False, window=window)
    assert [(a.left, a.right) for _, a in launches] == [(3, 4), (6, 4)]


def test_other_settings(monkeypatch) -> None:
    stub_launches(monkeypatch)
    x = torch.zeros(1, 8, 2, 64, dtype=BF16)
    mega_up.window_attention_bshd(x, x, x, sinks=1, scale=1.0)
    for settings in (dict(sinks=True), dict(sinks=1.0), dict(sinks=[1]), dict(sinks=np.int64(1))):
        with pytest.raises(ValueError):
            mega_up.window_attention_bshd(x, x, x, scale=1.0, **settings)
