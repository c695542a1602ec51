"""An output may take the place of its own input; one that is known to overlap another input is refused (CTAs would read
what others have written), slices of one buffer that only interleave are not."""

from __future__ import annotations

import random

import pytest
import torch

import megaup_b200 as mega_up
from _stubbed_launch import stub_launches
from megaup_b200.attention import _is_same, _share_elements, _span

BF16 = torch.bfloat16


def _elements(x) -> set[int]:
    every = torch.arange(x.untyped_storage().nbytes() // 2)
    return set(every.as_strided(x.shape, x.stride(), x.storage_offset()).flatten().tolist())


def test_slices_of_one_buffer_against_their_elements() -> None:
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(2000):
        batch, rows, heads = rng.randint(1, 3), rng.randint(1, 5), rng.randint(2, 6)
        buffer = torch.zeros(batch, rows, heads, 8, dtype=BF16)

        def part(n):
            low = rng.randrange(n)
            return slice(low, rng.randint(low + 1, n))

        a, b = (buffer[part(batch), part(rows), part(heads)] for _ in range(2))
        want = bool(_elements(a) & _elements(b))
        assert _share_elements(a, _span(a), b, _span(b)) == want, (a.shape, a.stride(), b.shape, b.stride())
        seen[want] += 1
        # steps of two: other strides, never refused where they are apart
        a = a[:, ::2]
        if _share_elements(a, _span(a), b, _span(b)):
            assert _elements(a) & _elements(b)
        if _is_same(a, b):
            assert _elements(a) == _elements(b)
    assert min(seen.values()) > 200


def test_attention(monkeypatch) -> None:
    launches = stub_launches(monkeypatch)
    call = mega_up.window_attention_bshd
    q, k, v = (torch.zeros(1, 8, 2, 64, dtype=BF16) for _ in range(3))
    more = torch.zeros(1, 12, 2, 64, dtype=BF16)
    for out, arguments in (
        (k, (q, k, v)), (v, (q, k, v)), (k.view_as(k), (q, k, v)), (q, (q, q, v)), (q, (q, k, q)),
        (more[:, 2:10], (q, more[:, 4:], v)), (more[:, 4:], (q, k, more[:, :8])), (more[:, 1:9], (more[:, :8], k, v)),
        (q.view(1, 2, 8, 64).transpose(1, 2), (q, k, v)),  # q's memory in another order
    ):
        with pytest.raises(ValueError, match="overlap"):
            call(*arguments, out=out)
    fused = torch.zeros(2, 9, 10, 64, dtype=BF16)
    fq, fk, fv, spare = fused.split((4, 1, 1, 4), dim=2)
    token = torch.zeros(2, 1, 4, 64, dtype=BF16)
    good = [
        (q, (q, k, v)), (q.view_as(q), (q, k, v)), (torch.empty_like(q), (q, k, v)), (more[:, 4:], (more[:, 4:], k, v)),
        (fq, (fq, fk, fv)), (spare, (fq, fk, fv)), (fused[..., :4, :], (fq, fk, fv)), (token, (token, fk, fv)),
        (more[:, :4], (more[:, 4:8], more[:, 8:], more[:, 8:])),
    ]
    for out, arguments in good:
        assert call(*arguments, out=out) is out
    with pytest.raises(ValueError, match="overlap"):
        call(fq, fk, fv, out=fused[:, :, 1:5])
    assert len(launches) == len(good)


def test_rotary(monkeypatch) -> None:
    launches = stub_launches(monkeypatch)
    rotary, positions = mega_up.prepare_axial_rotary([64], device="cpu"), torch.zeros(1, 8)
    q, k, other = (torch.zeros(1, 8, 2, 64, dtype=BF16) for _ in range(3))
    more = torch.zeros(1, 12, 2, 64, dtype=BF16)
    call = mega_up.axial_rotary_bshd
    for out in ((k, q), (k, other), (other, q), (other, other), (q, q), (q, q.view_as(q)), (more[:, :8], more[:, 4:])):
        with pytest.raises(ValueError, match="overlap"):
            call(q, k, rotary, positions, out=out)
    with pytest.raises(ValueError, match="overlap"):
        call(q, q, rotary, positions, out=(q, q))  # one memory would be turned twice
    with pytest.raises(ValueError, match="overlap"):
        call(more[:, :8], None, rotary, positions, out=(more[:, 1:9],))
    fused = torch.zeros(1, 8, 6, 64, dtype=BF16)
    fq, fk, spare = fused.split((2, 2, 2), dim=2)
    good = [((q, k), (q, k)), ((q, k), (q, other)), ((q, k), (other, k)), ((fq, fk), (fq, fk)), ((fq, fk), (spare, fk)),
            ((fq, fk), (fused[:, :, :2], fused[:, :, 2:4])), ((q, q), (other, k))]
    for tensors, out in good:
        got = call(*tensors, rotary, positions, out=out)
        assert got[0] is out[0] and got[1] is out[1]
    assert len(launches) == len(good)


def test_an_output_of_a_graph_of_autograd(monkeypatch) -> None:
    """Its gradient would go to what it held before."""

    launches = stub_launches(monkeypatch)
    rotary, positions = mega_up.prepare_axial_rotary([64], device="cpu"), torch.zeros(1, 8)
    q, k = torch.zeros(1, 8, 2, 64, dtype=BF16), torch.zeros(1, 8, 2, 64, dtype=BF16)
    leaf = torch.zeros(1, 8, 2, 64, dtype=BF16, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="gradient"):
            mega_up.window_attention_bshd(q, k, k, out=out)
        for outs in ((out, k), (q, out)):
            with pytest.raises(ValueError, match="gradient"):
                mega_up.axial_rotary_bshd(q, k, rotary, positions, out=outs)
        assert not launches
        with torch.no_grad():
            mega_up.window_attention_bshd(q, k, k, out=out)
            mega_up.axial_rotary_bshd(q, k, rotary, positions, out=(out, k))
        launches.clear()
