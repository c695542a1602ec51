"""Waits of the attention kernels that run out, in a kernel of their own (bounded_wait_probe.cu): nothing makes a wait of
the attention itself run out. Every lane of a warp leaves with the same result, and the cause is reported."""

from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from megaup_b200 import build

DEVICE = torch.device("cuda", 0)
MILLISECOND = 1_000_000


@pytest.fixture(scope="module")
def probe_library(tmp_path_factory):
    target = tmp_path_factory.mktemp("probe") / "bounded_wait_probe.so"
    source = build.PACKAGE_DIR.parent / "tests" / "bounded_wait_probe.cu"
    command = [build.find_nvcc(), *build.NVCC_FLAGS, "-I", str(build.CSRC), "-o", str(target), str(source)]
    result = subprocess.run(command, capture_output=True, text=True)
    assert result.returncode == 0, result.stderr
    library = ctypes.CDLL(str(target))
    library.bounded_wait_probe.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_uint64] * 3 + [ctypes.c_int] * 2
    library.products_probe.argtypes = [ctypes.c_void_p, ctypes.c_int]
    return library


def test_the_probe_builds(probe_library) -> None:
    assert probe_library.bounded_wait_probe(None, None, None, 3_000_000_000, 0, 0, 0, 0) == -1
    assert probe_library.products_probe(None, 0) == -1


@pytest.fixture
def probe(probe_library):
    def run(*, limit, others=None, delay=0, completes=True, drains=False):
        outcome = torch.full((128,), 9, dtype=torch.int32, device=DEVICE)
        elapsed = torch.zeros(2, dtype=torch.int64, device=DEVICE)
        status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        torch.cuda.synchronize()
        code = probe_library.bounded_wait_probe(
            outcome.data_ptr(), elapsed.data_ptr(), status.data_ptr(), limit, limit if others is None else others,
            delay, completes, drains,
        )
        assert code == 0
        return outcome.view(4, 32).tolist(), elapsed.tolist(), int(status)

    return run


@pytest.mark.gpu
def test_a_phase_that_ends_in_time(probe) -> None:
    outcome, elapsed, status = probe(limit=1000 * MILLISECOND, delay=MILLISECOND // 5)
    assert outcome == [[1] * 32] * 4 and status == 0 and elapsed[0] < 500 * MILLISECOND


@pytest.mark.gpu
def test_a_phase_that_never_ends(probe) -> None:
    outcome, elapsed, status = probe(limit=2 * MILLISECOND, completes=False, drains=True)
    assert outcome == [[0] * 32] * 4 and status == 2 << 24
    assert 2 * MILLISECOND <= elapsed[0] < 500 * MILLISECOND
    assert 200 * MILLISECOND <= elapsed[1] < 1000 * MILLISECOND  # a drain gives up as well


@pytest.mark.gpu
def test_the_others_leave_with_the_first(probe) -> None:
    outcome, elapsed, status = probe(limit=2 * MILLISECOND, others=20_000 * MILLISECOND, completes=False)
    assert outcome == [[0] * 32] * 4 and status == 2 << 24 and elapsed[0] < 1000 * MILLISECOND


@pytest.mark.gpu
def test_a_phase_that_ends_at_the_limit(probe) -> None:
    """Either result, but one for the whole warp."""

    seen = set()
    for limit in (1, 3000, 30_000, 100_000):
        for step in range(200):
            outcome, _, status = probe(limit=limit, delay=limit * (50 + step) // 100)
            for lanes in outcome:
                assert len(set(lanes)) == 1, (limit, step, lanes)
                seen.add(lanes[0])
            assert (status != 0) == any(lanes[0] == 0 for lanes in outcome)
    assert seen == {0, 1}


@pytest.mark.gpu
@pytest.mark.parametrize("repeats", [1, 500])
def test_products_in_flight_end_in_the_drain(probe_library, repeats) -> None:
    sums = torch.zeros(128, 128, device=DEVICE)
    torch.cuda.synchronize()
    assert probe_library.products_probe(sums.data_ptr(), repeats) == 0
    assert bool((sums == 64.0).all())
