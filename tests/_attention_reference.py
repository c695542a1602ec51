"""Sliding-window attention with sinks and rotary positions in 64 bits, dense and
per sequence, with the rounding errors the kernels may make: every bound below is
the arithmetic of their stated roundings (a rounding to BF16 is off by at most
2^-8 of the value, one to FP32 by 2^-24)."""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

HALF_BF16 = 2.0**-8


def visible(queries: int, keys: int, *, causal: bool, left: int | None, right: int | None, sinks: int) -> torch.Tensor:
    """[queries, keys]: which key a row sees."""

    at = torch.arange(queries)[:, None] + keys - queries
    j = torch.arange(keys)[None, :]
    window = torch.ones(queries, keys, dtype=torch.bool)
    if left is not None:
        window &= j >= at - left
    if causal:
        window &= j <= at
    elif right is not None:
        window &= j <= at + right
    seen = window | (j < sinks)
    return seen & (j <= at) if causal else seen


@dataclass
class Expected:
    out: torch.Tensor
    lse: torch.Tensor
    dq: torch.Tensor | None
    dk: torch.Tensor | None
    dv: torch.Tensor | None
    # largest error of each element
    out_error: torch.Tensor
    lse_error: torch.Tensor
    dq_error: torch.Tensor | None
    dk_error: torch.Tensor | None
    dv_error: torch.Tensor | None


def attention(q, k, v, seen, *, scale=None, dout=None) -> Expected:
    """``q [Sq,H,D]``, ``k, v [Sk,Hkv,D]`` of one sequence, ``seen [Sq,Sk]``."""

    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    seen = seen.cpu()
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim**-0.5 if scale is None else scale
    kh, vh = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    hide = ~seen[None]
    # rows that nobody sees may hold anything
    used = seen.any(0)
    kh, vh = torch.where(used[:, None, None], kh, 0.0), torch.where(used[:, None, None], vh, 0.0)
    s = torch.einsum("ihd,jhd->hij", q, kh) * scale
    s = s.masked_fill(hide, -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:-1], -math.inf, dtype=s.dtype)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    out = torch.einsum("hij,jhd->ihd", p, vh)
    # A score is a sum of dim products kept in FP32 over dim / 16 steps, scaled and shifted (a few FP32 roundings of
    # its size); the exponential adds 2^-22. The error of an exponent is the relative error of a weight.
    size = (torch.einsum("ihd,jhd->hij", q.abs(), kh.abs()) * scale).masked_fill(hide, 0.0)
    size = size.amax(-1, keepdim=True) if size.shape[-1] else size.new_zeros(*size.shape[:-1], 1)
    weight_error = 2.0**-23 * (dim / 16 + 6) * (size + 1.0) + 2.0**-21  # [h, i, 1]
    row_error = weight_error.squeeze(-1).T[..., None]  # [i, h, 1]
    # weights round to BF16 once (and their FP32 sum does not: the quotient keeps the weights' error), the result once
    total = torch.einsum("hij,jhd->ihd", p, vh.abs())
    out_error = (HALF_BF16 + 3 * row_error) * total * (1 + HALF_BF16) + HALF_BF16 * out.abs() + 2.0**-130
    lse_error = 2 * weight_error.squeeze(-1) + 2.0**-22 * lse.abs().nan_to_num(0.0, 0.0, 0.0)
    if dout is None:
        return Expected(out, lse, None, None, None, out_error, lse_error, None, None, None)
    g = dout.detach().double().cpu()
    dp = torch.einsum("ihd,jhd->hij", g, vh)
    delta = (g * out).sum(-1).T[..., None]
    ds = p * (dp - delta)
    fold = lambda x: x.view(x.shape[0], k.shape[1], group, dim).sum(2)  # noqa: E731
    dv = fold(torch.einsum("hij,ihd->jhd", p, g))
    dq = torch.einsum("hij,jhd->ihd", ds, kh) * scale
    dk = fold(torch.einsum("hij,ihd->jhd", ds, q)) * scale
    # P: its relative error and one rounding. dS: that of P, the FP32 sums dP and delta, delta's use of the rounded
    # result, and one rounding.
    fp32_sum = 2.0**-23 * (dim / 16 + 4)
    dp_size = torch.einsum("ihd,jhd->hij", g.abs(), vh.abs())
    delta_error = ((g.abs() * out_error).sum(-1) + fp32_sum * (g.abs() * out.abs()).sum(-1)).T[..., None]
    ds_error = p * (fp32_sum * dp_size + delta_error) + (3 * weight_error + HALF_BF16) * ds.abs()
    ds_error = ds_error * (1 + HALF_BF16)
    long = 2.0**-20  # FP32 sums over the rows of a block of keys or queries
    dv_error = fold(torch.einsum("hij,ihd->jhd", p * (HALF_BF16 + 3 * weight_error + long), g.abs()))
    dq_error = torch.einsum("hij,jhd->ihd", ds_error + long * ds.abs(), kh.abs()) * scale
    dk_error = fold(torch.einsum("hij,ihd->jhd", ds_error + long * ds.abs(), q.abs())) * scale
    finish = lambda e, x: e * (1 + HALF_BF16) + HALF_BF16 * x.abs() + 2.0**-130  # noqa: E731
    return Expected(
        out, lse, dq, dk, dv, out_error, lse_error, finish(dq_error, dq), finish(dk_error, dk), finish(dv_error, dv)
    )


def assert_within(got: torch.Tensor, want: torch.Tensor, error: torch.Tensor, what: str) -> None:
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs())
    assert not torch.isnan(off).any(), f"{what}: NaN"
    worst = (off / error.clamp_min(1e-300)).max() if off.numel() else torch.tensor(0.0)
    assert worst <= 1.0, f"{what}: an element is {worst:.2f} times its error bound off"


def rotate(x, angle, *, interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., D]`` turned by ``angle`` (64 bits, [..., pairs], broadcast over heads); the result and its error."""

    x = x.detach().double().cpu()
    pairs = angle.shape[-1]
    y, error = x.clone(), torch.zeros_like(x)
    first, second = (
        (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved
        else (slice(0, pairs), slice(pairs, 2 * pairs))
    )
    a, b = x[..., first], x[..., second]
    y[..., first] = a * torch.cos(angle) - b * torch.sin(angle)
    y[..., second] = a * torch.sin(angle) + b * torch.cos(angle)
    # sine and cosine: 2^-22 with the FP32 fraction of a turn (2^-25 turns = 2^-22.3 radians); two products and a sum
    size = (a.abs() + b.abs()) * 2.0**-20
    error[..., first] = size + HALF_BF16 * y[..., first].abs()
    error[..., second] = size + HALF_BF16 * y[..., second].abs()
    return y, error
