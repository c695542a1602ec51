"""The attention's and the rotary positions' host side on the CPU: tensors of the host pass for the device's, and a
launch records its argument block in place of a kernel."""

from __future__ import annotations

import ctypes

import pytest

from megaup_b200 import _native, attention, build, rotary


def stub_launches(monkeypatch: pytest.MonkeyPatch) -> list[tuple[str, ctypes.Structure]]:
    """From here to the test's end; returns the launches, (entry point, argument block), as they are made."""

    build.ensure_built()
    library, launches = _native.lib(), []

    def call(function: str, block, *rest) -> None:
        if function == "mup_window_attention_workspace":  # host arithmetic
            assert getattr(library, function)(block, *rest) == 0, library.mup_last_error()
        else:
            launches.append((function, block._obj))

    for name in ("MupWindowAttention", "MupAxialRotary"):
        base = getattr(_native, name)

        class Block(base):
            def __setattr__(self, name: str, value: object) -> None:
                # a tensor of the host has no device index
                super().__setattr__(name, 0 if name == "device" and value is None else value)

        monkeypatch.setattr(_native, name, Block)
    monkeypatch.setattr(_native, "call", call)
    monkeypatch.setattr(attention, "_PLANS", {})
    for module in (attention, rotary):
        monkeypatch.setattr(module, "_check_heads_tensor", lambda *_: None)
        monkeypatch.setattr(module, "_current_stream", lambda _: 0)
    return launches
