"""The word in which kernels that are given none report a wait that ran out: read without a launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

import megaup_b200 as mega_up
from megaup_b200 import _native, build

DEVICE = torch.device("cuda", 0)
BF16 = torch.bfloat16


def test_arguments_and_a_device_that_was_never_used() -> None:
    build.ensure_built()
    library, word = _native.lib(), ctypes.c_uint32(7)
    assert library.mup_device_status(63, ctypes.byref(word), None) == 0 and word.value == 0
    for device in (-1, 64):
        assert library.mup_device_status(device, ctypes.byref(word), None) == -1
    assert library.mup_device_status(0, None, None) == -1
    mega_up.check_status(63)
    for device in ("cpu", torch.device("cpu")):
        with pytest.raises(ValueError, match="CUDA"):
            mega_up.check_status(device)


@pytest.mark.parametrize("device", [5, "cuda:5", torch.device("cuda", 5)], ids=str)
def test_a_failure_is_raised(monkeypatch, device) -> None:
    asked = []

    def call(function, index, word, device_ptr):
        asked.append((function, index, device_ptr))
        word._obj.value = 2 << 24 | 9

    monkeypatch.setattr(_native, "call", call)
    with pytest.raises(RuntimeError, match=r"cuda:5.*filled shared-memory stage \(detail 9\)"):
        mega_up.check_status(device)
    assert asked == [("mup_device_status", 5, None)]


def _run_out(address: int) -> None:
    """A flag that nobody raises; the kernel reports in the word at `address` and ends."""

    flags = [torch.zeros(8, dtype=torch.int32, device=DEVICE) for _ in range(2)]
    _native.call(
        "mup_flag_barrier", _native.pointer_array([f.data_ptr() for f in flags]), 2, 0, 1, address, 5_000_000,
        torch.cuda.current_stream(DEVICE).cuda_stream,
    )
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_wait_that_ran_out_is_seen_without_another_launch() -> None:
    word, address = ctypes.c_uint32(), ctypes.c_void_p()
    _native.call("mup_device_status", 0, ctypes.byref(word), ctypes.byref(address))
    assert word.value == 0 and address.value
    mega_up.check_status()
    _run_out(address.value)
    with pytest.raises(RuntimeError, match="slot hand-off flag"):
        mega_up.check_status(DEVICE)
    mega_up.check_status("cuda")  # raised once
    # the attention reports in the same word, and the runtime looks at it
    x = torch.randn(1, 40, 2, 64, device=DEVICE).to(BF16)
    want = mega_up.window_attention_bshd(x, x, x)
    again = ctypes.c_void_p()
    _native.call("mup_device_status", 0, ctypes.byref(word), ctypes.byref(again))
    assert again.value == address.value
    _run_out(address.value)
    with pytest.raises(_native.NativeError, match="DEVICE_STATUS"):
        mega_up.window_attention_bshd(x, x, x)
    assert torch.equal(mega_up.window_attention_bshd(x, x, x), want)
    runtimes = mega_up.initialize_emulated_group(2, hidden=512, max_rows=64, device=DEVICE)
    _run_out(address.value)
    with pytest.raises(RuntimeError, match="slot hand-off flag"):
        runtimes[0].check_status()
    runtimes[0].check_status()
