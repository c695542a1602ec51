"""What is measured of the operators between the two exchange GEMMs: rotary positions with several axes, and
sliding-window attention with sinks, on the head-parallel tensors that a peer-write projection delivers and a
head-shard pull takes back.

A case is a dict of plain values; ``prepare`` makes its inputs from a seed, ``run`` makes one pass (``own`` chooses
the framework's kernels or the plain torch form), ``exact`` is the definition in 64 bits and ``work`` what a pass
cannot do without.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
BF16 = torch.bfloat16

# --------------------------------------------------------------------------- cases


def _rotary(name=None, **more):
    case = dict(op="rotary", layout="bshd", batch=1, rows=1, heads=1, kv_heads=1, head_dim=128, axes="44,42,42",
                interleaved=True, shared=False, theta=10000.0, frame=64, width=8, first=0, fused=False, train=False)
    case.update(more)
    return {"name": name, **case} if name else case


def _attention(name=None, **more):
    case = dict(op="attention", layout="bshd", batch=1, q_len=1, k_len=1, heads=1, kv_heads=1, head_dim=128,
                causal=True, left=-1, right=0, sinks=0, lengths=False, shortest=0, pack=0, fused=False, train=False)
    case.update(more)
    return {"name": name, **case} if name else case


def listed():
    return [
        # one new token of eight sequences: latency
        _rotary("rotary 8 single tokens", layout="sbhd", batch=8, rows=1, heads=8, kv_heads=1, axes="32,48,48",
                interleaved=False, shared=True, theta=500000.0, first=65000, fused=True),
        # a Wan2.1-14B-shaped video of 8 x 4096 tokens on one of eight ranks: 5 of 40 heads
        _rotary("rotary video u8", rows=32768, heads=5, kv_heads=5, frame=1560, width=52),
        # the same on one of two ranks (20 heads), with its gradient
        _rotary("rotary video u2 train", rows=8192, heads=20, kv_heads=20, frame=1560, width=52, train=True),
        # grouped heads as slices of a fused QKV projection, packed rows, rotated halves, far positions
        _rotary("rotary gqa packed", layout="thd", rows=65536, heads=8, kv_heads=2, axes="32,48,48",
                interleaved=False, shared=True, theta=500000.0, frame=400, width=20, first=1000000, fused=True),
        # one new token of one sequence, four heads of one group, a short window: latency
        _attention("attn one token", q_len=1, k_len=4096, heads=4, kv_heads=1, left=1023, sinks=4),
        # one new token of 16 sequences of their own lengths in a cache of 65 536 rows, nothing left out: bandwidth
        _attention("attn 16 tokens long cache", batch=16, q_len=1, k_len=65536, heads=8, kv_heads=1, lengths=True,
                   shortest=8192),
        # a chunk of new tokens after a long prompt: few rows, a long axis
        _attention("attn chunk", batch=1, q_len=200, k_len=32968, heads=4, kv_heads=1, left=16383, sinks=64),
        # video tokens that see their neighbours on both sides and the first frame
        _attention("attn video u8", q_len=32768, k_len=32768, heads=5, kv_heads=5, causal=False, left=4096, right=4096,
                   sinks=1560),
        # packed prompts of 512 to 4096 tokens, eight heads of one group, q, k and v slices of one projection
        _attention("attn packed prompts", layout="thd", batch=0, q_len=32768, k_len=32768, shortest=512, pack=5,
                   heads=8, kv_heads=1, left=1023, sinks=4, fused=True),
        # a training step of grouped heads, sequence first
        _attention("attn train gqa u8", layout="sbhd", q_len=65536, k_len=65536, heads=4, kv_heads=1, left=4095,
                   sinks=4, train=True),
        # the same operator with 64-wide heads, an odd length and a batch
        _attention("attn train 64 wide", batch=2, q_len=4097, k_len=4097, heads=4, kv_heads=4, head_dim=64, left=511,
                   sinks=1, train=True),
        # packed video clips, both directions, with the gradient
        _attention("attn train packed", layout="thd", batch=0, q_len=16384, k_len=16384, shortest=512, pack=9, heads=5,
                   kv_heads=5, causal=False, left=1024, right=1024, sinks=256, train=True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    head_dim = rng.choice((64, 128, 128))
    if rng.random() < 0.3:
        axes = {64: ("16,24,24", "24,20,20", "64"), 128: ("44,42,42", "32,48,48", "16,56,56")}[head_dim]
        kv_heads = rng.choice((1, 2, 5))
        heads = kv_heads * rng.choice((1, 2, 4))
        layout = rng.choice(("bshd", "sbhd", "thd"))
        batch = 1 if layout == "thd" else rng.choice((1, 1, 2, 3, 8))
        width = rng.randint(8, 90)
        return _rotary(layout=layout, batch=batch, rows=_log_uniform(rng, 1, 40000) // batch + 1, heads=heads,
                       kv_heads=kv_heads, head_dim=head_dim, axes=rng.choice(axes), interleaved=rng.random() < 0.5,
                       shared=rng.random() < 0.5, theta=rng.choice((10000.0, 256.0, 500000.0)), width=width,
                       frame=width * rng.randint(4, 60), first=rng.choice((0, rng.randint(1, 1000000))),
                       fused=rng.random() < 0.3, train=rng.random() < 0.4)
    kv_heads = rng.choice((1, 1, 2, 5))
    heads = kv_heads * rng.choice((1, 2, 4, 8) if kv_heads < 5 else (1,))
    sinks = rng.choice((0, 1, 4, rng.randint(5, 700)))
    left = rng.choice((-1, _log_uniform(rng, 1, 5000), _log_uniform(rng, 64, 5000)))
    kind = rng.random()
    if kind < 0.35:  # tokens over a cache
        batch = rng.choice((1, 2, 7, 16))
        q_len = rng.choice((1, 1, 2, rng.randint(3, 300)))
        k_len = q_len + _log_uniform(rng, 8, 262144 // batch)
        return _attention(layout=rng.choice(("bshd", "sbhd")), batch=batch, q_len=q_len, k_len=k_len, heads=heads,
                          kv_heads=kv_heads, head_dim=head_dim, left=left, sinks=sinks, lengths=rng.random() < 0.5,
                          shortest=min(k_len, q_len + rng.randint(0, 64)))
    train = kind > 0.65
    causal = rng.random() < 0.6
    rows = _log_uniform(rng, 100, min(20000, 80000 // heads))
    left = min(left, 4096) if left >= 0 else (-1 if rows < 9000 else 4096)
    right = 0 if causal else rng.choice((left, 0, -1 if rows < 9000 else left))
    layout = rng.choice(("bshd", "sbhd", "thd"))
    batch = 0 if layout == "thd" else rng.choice((1, 1, 2, 3))
    rows = rows if layout == "thd" else max(1, rows // batch)
    return _attention(layout=layout, batch=batch, q_len=rows, k_len=rows, heads=heads, kv_heads=kv_heads,
                      head_dim=head_dim, causal=causal, left=left, right=right, sinks=sinks,
                      shortest=rng.randint(1, 500), pack=rng.randint(1, 1 << 20), fused=not train and rng.random() < 0.4,
                      train=train)


# --------------------------------------------------------------------------- what a case says about its sequences


def _sequences(case):
    """[(first query row, queries, first key row, keys)] over rows that run through all sequences."""
    q_len, k_len = case["q_len"], case["k_len"]
    if case["layout"] == "thd":
        rng, cuts = random.Random(case["pack"]), [0]
        while cuts[-1] < q_len:
            cuts.append(min(q_len, cuts[-1] + rng.randint(case["shortest"], 4096)))
        return [(a, b - a, a, b - a) for a, b in zip(cuts, cuts[1:])]
    keys = [k_len] * case["batch"]
    if case["lengths"]:
        rng = random.Random(case["k_len"])
        keys = [rng.randint(max(case["shortest"], q_len), k_len) for _ in keys]
    return [(b * q_len, q_len, b * k_len, n) for b, n in enumerate(keys)]


def _spans(case, queries, keys):
    """Per query of a sequence: the end of the sinks it sees, and the first and last key of its window."""
    at = np.arange(queries, dtype=np.int64) + keys - queries
    low = np.maximum(at - case["left"], 0) if case["left"] >= 0 else np.zeros_like(at)
    high = at if case["causal"] else (at + case["right"] if case["right"] >= 0 else np.full_like(at, keys - 1))
    high = np.minimum(high, keys - 1)
    sink = np.full_like(at, min(case["sinks"], keys))
    if case["causal"]:
        sink = np.clip(at + 1, 0, sink)
    return sink, low, high


def work(case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        values = case["batch"] * case["rows"] * (heads + kv_heads) * dim
        passes = 2 if case["train"] else 1
        axes = len(case["axes"].split(","))
        return {"bytes": passes * (4 * values + 8 * axes * case["rows"]), "flops": passes * 3 * values}
    pairs = seen = rows = 0
    for _, queries, _, keys in _sequences(case):
        sink, low, high = _spans(case, queries, keys)
        inside = np.maximum(high - np.maximum(low, sink) + 1, 0)
        pairs += int((sink + inside).sum())
        touched = np.zeros(keys + 1, dtype=np.int64)
        some = high >= low
        np.add.at(touched, low[some], 1)
        np.add.at(touched, high[some] + 1, -1)
        touched = np.cumsum(touched)[:keys] > 0
        touched[: int(sink.max(initial=0))] = True
        seen += int(touched.sum())
        rows += queries
    q_bytes, kv_bytes = 2 * rows * heads * dim, 2 * seen * kv_heads * dim
    total = 2 * q_bytes + 2 * kv_bytes  # q and the output, k and v
    flops = 4 * dim * heads * pairs
    if case["train"]:  # the output's gradient, and the gradients of q, k and v
        total += 2 * q_bytes + 2 * kv_bytes
        flops += 10 * dim * heads * pairs
    return {"bytes": total, "flops": flops}


# --------------------------------------------------------------------------- inputs


def _normal(shape, generator):
    return torch.randn(shape, generator=generator, device=DEVICE, dtype=torch.float32).to(BF16)


def _shape(case, length, heads, batch=None):
    batch = case["batch"] if batch is None else batch
    lead = {"bshd": (batch, length), "sbhd": (length, batch), "thd": (length,)}[case["layout"]]
    return (*lead, heads, case["head_dim"])


def _positions(case):
    """[axes, rows] of a video: the frame, the line and the column of every token."""
    at = torch.arange(case["rows"], device=DEVICE, dtype=torch.int64)
    frame, width = case["frame"], case["width"]
    grid = (case["first"] + at // frame, at % frame // width, at % width)
    return torch.stack(grid[: len(case["axes"].split(","))])


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    heads, kv_heads, train = case["heads"], case["kv_heads"], case["train"]
    state = {"case": case}
    if case["op"] == "rotary":
        if case["fused"]:  # slices of one projection's output, which also holds the values
            both = _normal(_shape(case, case["rows"], heads + 2 * kv_heads), generator)
            state["q"], state["k"] = both[..., :heads, :], both[..., heads : heads + kv_heads, :]
        else:
            state["q"] = _normal(_shape(case, case["rows"], heads), generator)
            state["k"] = _normal(_shape(case, case["rows"], kv_heads), generator)
        if train:
            state["dq"] = _normal(state["q"].shape, generator)
            state["dk"] = _normal(state["k"].shape, generator)
        state["positions"] = _positions(case)
        axes = [int(v) for v in case["axes"].split(",")]
        if own:
            import megaup_b200

            state["rotary"] = megaup_b200.prepare_axial_rotary(
                axes, theta=case["theta"], interleaved=case["interleaved"], shared_frequencies=case["shared"],
                device=DEVICE,
            )
        else:
            state["axis"], state["frequency"] = _frequencies(case)
    else:
        if case["fused"]:
            rows = _normal(_shape(case, case["q_len"], heads + 2 * kv_heads), generator)
            state["q"], state["k"], state["v"] = rows.split((heads, kv_heads, kv_heads), dim=-2)
        else:
            state["q"] = _normal(_shape(case, case["q_len"], heads), generator)
            state["k"] = _normal(_shape(case, case["k_len"], kv_heads), generator)
            state["v"] = _normal(_shape(case, case["k_len"], kv_heads), generator)
        if train:
            state["dout"] = _normal(state["q"].shape, generator)
        sequences = _sequences(case)
        if case["lengths"]:
            state["kv_lengths"] = torch.tensor([s[3] for s in sequences], dtype=torch.int32, device=DEVICE)
        if not own:
            state["plan"] = _plain_plan(case, sequences)
        elif case["layout"] == "thd":
            import megaup_b200

            state["sequences"] = megaup_b200.prepare_packed_sequences(
                [0] + [s[0] + s[1] for s in sequences], device=DEVICE
            )
    if train and own:
        for name in ("q", "k", "v"):
            if name in state:
                state[name].requires_grad_()
    return state


# --------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        return _run_rotary(case, state) if own else _plain_rotary(case, state)
    return _run_attention(case, state) if own else _plain_attention(case, state)


def _run_rotary(case, state):
    import megaup_b200

    call = getattr(megaup_b200, "axial_rotary_" + case["layout"])
    q, k = call(state["q"], state["k"], state["rotary"], state["positions"])
    if not case["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _run_attention(case, state):
    import megaup_b200

    call = getattr(megaup_b200, "window_attention_" + case["layout"])
    left, right = (None if v < 0 else v for v in (case["left"], case["right"]))
    more = {"window": left if case["causal"] else (left, right), "sinks": case["sinks"], "causal": case["causal"]}
    if case["layout"] == "thd":
        more["sequences"] = state["sequences"]
    elif case["lengths"]:
        more["kv_lengths"] = state["kv_lengths"]
    out = call(state["q"], state["k"], state["v"], **more)
    if not case["train"]:
        return {"out": out}
    leaves = (state["q"], state["k"], state["v"])
    dq, dk, dv = torch.autograd.grad(out, leaves, state["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


# --------------------------------------------------------------------------- plain forms


def _frequencies(case):
    """The axis and the frequency (64 bits) of every pair."""
    axes = [int(v) for v in case["axes"].split(",")]
    pairs = np.array([n // 2 for n in axes])
    axis = np.repeat(np.arange(len(axes)), pairs)
    if case["shared"]:  # one row of frequencies, cut into the axes
        step = 2.0 * np.arange(sum(pairs)) / sum(axes)
    else:  # every axis has a row of its own
        inside = np.arange(sum(pairs)) - np.repeat(np.cumsum(pairs) - pairs, pairs)
        step = 2.0 * inside / np.repeat(np.array(axes), pairs)
    frequency = np.power(np.float64(case["theta"]), -step)
    return torch.from_numpy(axis).to(DEVICE), torch.from_numpy(frequency).to(DEVICE)


def _turned(case, x, cos, sin):
    """x, its pairs turned, in 32 bits and rounded once; cos and sin are laid out to multiply [..., heads, pairs]."""
    turned = sum(int(v) for v in case["axes"].split(","))
    rest = x[..., turned:]
    x = x[..., :turned].float()
    if case["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = x[..., : turned // 2], x[..., turned // 2 :]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y.to(BF16), rest), dim=-1)


def _plain_rotary(case, state):
    angle = state["positions"][state["axis"]].double().T * state["frequency"]  # [rows, pairs]; far positions: 64 bits
    lead = {"bshd": (1, case["rows"], 1), "sbhd": (case["rows"], 1, 1), "thd": (case["rows"], 1)}[case["layout"]]
    cos, sin = (f(angle).float().view(*lead, -1) for f in (torch.cos, torch.sin))
    out = {name: _turned(case, state[name], cos, sin) for name in ("q", "k")}
    if case["train"]:
        out.update({name: _turned(case, state[name], cos, -sin) for name in ("dq", "dk")})
    return out


def _plain_plan(case, sequences):
    """The rows of q, and the keys they could see, in blocks of equal size: one matrix product for all of them."""
    longest = max(s[3] for s in sequences)
    block = min(1024 if longest > 2048 else 256, max(s[1] for s in sequences))
    reach = longest if min(case["left"], 0 if case["causal"] else case["right"]) < 0 else block + case["left"] + case["right"]
    reach = min(reach, longest)
    first, last, low, start, queries, keys, key0 = [], [], [], [], [], [], []
    for q0, nq, k0, nk in sequences:
        for r in range(0, nq, block):
            at = r + nk - nq
            first.append(q0 + r)
            last.append(q0 + nq)
            start.append(at)
            low.append(min(max(0, at - case["left"] if case["left"] >= 0 else 0), max(0, nk - reach)))
            keys.append(nk)
            key0.append(k0)
    as_tensor = lambda v: torch.tensor(v, dtype=torch.int64, device=DEVICE)[:, None]  # noqa: E731
    return {"block": block, "reach": reach, "sinks": min(case["sinks"], longest), "first": as_tensor(first),
            "last": as_tensor(last), "low": as_tensor(low), "start": as_tensor(start), "keys": as_tensor(keys),
            "key0": as_tensor(key0)}


def _rows_of(case, x):
    """[rows of all sequences, heads, dim], a batch's sequences one after another."""
    if case["layout"] == "sbhd":
        x = x.transpose(0, 1)
    return x.reshape(-1, *x.shape[-2:])


def _in_layout(case, rows, length):
    if case["layout"] == "thd":
        return rows
    x = rows.view(case["batch"], length, *rows.shape[-2:])
    return x.transpose(0, 1).contiguous() if case["layout"] == "sbhd" else x


def _plain_attention(case, state):
    plan, group, dim = state["plan"], case["heads"] // case["kv_heads"], case["head_dim"]
    scale = dim**-0.5
    q, k, v = (_rows_of(case, state[name]) for name in ("q", "k", "v"))
    step = torch.arange(plan["block"], device=DEVICE)
    row = plan["first"] + step
    real = row < plan["last"]
    row = torch.where(real, row, 0)
    at = (plan["start"] + step)[:, :, None]
    # first the sinks, then the window's keys without those that are sinks
    near = plan["low"] + torch.arange(plan["reach"], device=DEVICE)
    sink = torch.arange(plan["sinks"], device=DEVICE).expand(near.shape[0], -1)
    key = torch.cat((sink, near), dim=1)
    is_sink = torch.arange(key.shape[1], device=DEVICE) < plan["sinks"]
    j = key[:, None, :]
    inside = j >= case["sinks"]
    if case["left"] >= 0:
        inside = inside & (j >= at - case["left"])
    if not case["causal"] and case["right"] >= 0:
        inside = inside & (j <= at + case["right"])
    seen = (inside | is_sink) & (j < plan["keys"][:, :, None])
    if case["causal"]:
        seen = seen & (j <= at)
    seen = (seen & real[:, :, None])[:, None, None]  # [blocks, 1, 1, block, keys]
    key = torch.where(key < plan["keys"], key + plan["key0"], 0)

    def heads_first(x, index):  # [blocks, kv heads, group, rows, dim], in 32 bits
        x = x[index].float()
        return x.view(*x.shape[:2], case["kv_heads"], -1, dim).permute(0, 2, 3, 1, 4)

    def to_rows(x):  # [blocks, kv heads, group, rows, dim] of real rows -> [rows, heads, dim]
        x = x.permute(0, 3, 1, 2, 4).reshape(*row.shape, case["heads"], dim)
        return torch.zeros_like(q, dtype=torch.float32).index_put_((row[real],), x[real])

    qb, kb, vb = heads_first(q, row), heads_first(k, key), heads_first(v, key)
    score = torch.where(seen, (qb @ kb.transpose(-1, -2)) * scale, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = weight.sum(dim=-1, keepdim=True)
    weight = weight / torch.where(total == 0, 1.0, total)
    out = weight @ vb
    result = {"out": _in_layout(case, to_rows(out).to(BF16), case["q_len"])}
    if not case["train"]:
        return result
    dout = heads_first(_rows_of(case, state["dout"]), row) * real[:, None, None, :, None]
    dv = (weight.transpose(-1, -2) @ dout).sum(dim=2)
    dscore = dout @ vb.transpose(-1, -2)
    dscore = weight * (dscore - (dout * out).sum(dim=-1, keepdim=True)) * scale
    del weight
    dq = dscore @ kb
    dk = (dscore.transpose(-1, -2) @ qb).sum(dim=2)

    def to_keys(x):  # a key's gradient is the sum over the blocks that see it
        x = x.transpose(1, 2).reshape(-1, case["kv_heads"], dim)
        return torch.zeros_like(k, dtype=torch.float32).index_add_(0, key.reshape(-1), x)

    result["dq"] = _in_layout(case, to_rows(dq).to(BF16), case["q_len"])
    result["dk"] = _in_layout(case, to_keys(dk).to(BF16), case["k_len"])
    result["dv"] = _in_layout(case, to_keys(dv).to(BF16), case["k_len"])
    return result


# --------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    return _exact_attention(case, state)


def _exact_rotary(case, state):
    axes = [int(v) for v in case["axes"].split(",")]
    turned, pair, columns = sum(axes), 0, []
    for axis, width in enumerate(axes):
        for inside in range(width // 2):
            exponent = 2 * pair / turned if case["shared"] else 2 * inside / width
            columns.append(state["positions"][axis].double() * case["theta"] ** -exponent)
            pair += 1
    angle = torch.stack(columns, dim=-1)  # [rows, pairs]
    if case["layout"] == "bshd":
        angle = angle[None]
    elif case["layout"] == "sbhd":
        angle = angle[:, None]
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(-2)

    def rotated(x, turn):
        y = x.double().clone()
        first, second = (slice(0, turned, 2), slice(1, turned, 2)) if case["interleaved"] else (
            slice(0, turned // 2), slice(turned // 2, turned))
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {name: rotated(state[name], turn) for name in ("q", "k")}
    if case["train"]:
        out.update({name: rotated(state[name], turn.conj()) for name in ("dq", "dk")})
    return out


def _exact_attention(case, state):
    group, dim = case["heads"] // case["kv_heads"], case["head_dim"]
    names = ("q", "k", "v", "dout") if case["train"] else ("q", "k", "v")
    rows = {name: _rows_of(case, state[name].detach()) for name in names}
    out = torch.zeros(rows["q"].shape, dtype=torch.float64, device=DEVICE)
    grads = {name: torch.zeros(rows[name].shape, dtype=torch.float64, device=DEVICE) for name in names[:3]}
    chunk = 512
    for q0, queries, k0, keys in _sequences(case):
        sink, low, high = (torch.from_numpy(v).to(DEVICE) for v in _spans(case, queries, keys))
        for r in range(0, queries, chunk):
            end = min(queries, r + chunk)
            a, b, s = int(low[r]), int(high[end - 1]) + 1, int(sink[end - 1])
            a, b = max(a, s), max(b, s, a)
            j = torch.cat((torch.arange(s, device=DEVICE), torch.arange(a, b, device=DEVICE)))
            if not j.numel():
                continue
            hidden = ~((j < sink[r:end, None]) | ((j >= low[r:end, None]) & (j <= high[r:end, None])))
            for h in range(case["kv_heads"]):
                kk, vv = rows["k"][k0 + j, h].double(), rows["v"][k0 + j, h].double()
                own_heads = slice(h * group, (h + 1) * group)
                qq = rows["q"][q0 + r : q0 + end, own_heads].double()
                logits = torch.einsum("rgd,jd->grj", qq, kk) * dim**-0.5
                p = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1).nan_to_num(0.0)
                o = torch.einsum("grj,jd->rgd", p, vv)
                out[q0 + r : q0 + end, own_heads] = o
                if not case["train"]:
                    continue
                g = rows["dout"][q0 + r : q0 + end, own_heads].double()
                dp = torch.einsum("rgd,jd->grj", g, vv) - (g * o).sum(-1).T[..., None]
                ds = p * dp * dim**-0.5
                grads["q"][q0 + r : q0 + end, own_heads] = torch.einsum("grj,jd->rgd", ds, kk)
                grads["k"][:, h].index_add_(0, k0 + j, torch.einsum("grj,rgd->jd", ds, qq))
                grads["v"][:, h].index_add_(0, k0 + j, torch.einsum("grj,rgd->jd", p, g))
    result = {"out": _in_layout(case, out, case["q_len"])}
    if case["train"]:
        for name, length in (("q", case["q_len"]), ("k", case["k_len"]), ("v", case["k_len"])):
            result["d" + name] = _in_layout(case, grads[name], length)
    return result
