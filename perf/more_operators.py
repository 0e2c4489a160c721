"""Workloads of the long-context serving operators: attention for a batch that shares a long prefix, attention
that adds up the weight each cached key receives, and eviction from a cache by that weight.

Each operator has a plain form in elementary torch operations (``own = False``) and the calls of
``basalt_b200.operators`` (``own = True``) on the same inputs.

Definitions. A sequence has ``length`` keys in its row of the cache; query i of its n tokens stands at position
``length - n + i`` and sees key j when ``j <= position`` and (``window`` is 0, or ``position - j < window``, or
``j < sinks``). A query that sees nothing gives zeros.

- shared: every query sees the ``prefix`` keys of one common row besides the keys of its own row.
- weights: each key j < length of a key head gets ``decay * previous + sum of the weights`` that the sequence's
  queries and the head's query heads gave it; places behind the length stay as they were.
- evict: of a longer sequence ``keep`` keys stay in each key head: the first ``sinks``, the last ``recent`` and of
  the others those of the largest mass (ties: lowest place). They move in order to the first places of another
  cache, their masses with them; the masses behind them become zero.

A 4-bit cache holds 32 consecutive channels of one head of one token as a group: a code of 4 bits stands for
``low + code * step``, both bf16. Codes of a head are kept as [8][groups][4] nibbles, low nibble first: channel
``32 g + 4 h + j`` is nibble j of the 16 bits at [h][g].
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    """The cases, each with what it stands for in use."""
    return [
        # A few short chats behind one system prompt, the engine's float32 heads (latency).
        {"name": "shared-small", "op": "shared", "seqs": 4, "new": 1, "prefix": 500, "low": 1, "high": 60,
         "slots": 64, "heads": 8, "kv_heads": 8, "dim": 64, "dtype": "f32", "prefix_storage": "u4",
         "storage": "u4"},
        # A decode step of 32 sequences behind a prompt of 2048 tokens, all in float32.
        {"name": "shared-f32", "op": "shared", "seqs": 32, "new": 1, "prefix": 2048, "low": 33, "high": 512,
         "slots": 512, "heads": 8, "kv_heads": 8, "dim": 64, "dtype": "f32", "prefix_storage": "f32",
         "storage": "f32"},
        # A decode step of 64 sequences behind a document of 8000 tokens, grouped heads, answers of odd lengths.
        {"name": "shared-step", "op": "shared", "seqs": 64, "new": 1, "prefix": 8001, "low": 20, "high": 1000,
         "slots": 1024, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "prefix_storage": "bf16",
         "storage": "bf16"},
        # Four drafted tokens of 24 sequences are checked at once behind a prefix held in 4 bits.
        {"name": "shared-drafts", "op": "shared", "seqs": 24, "new": 4, "prefix": 16384, "low": 50, "high": 700,
         "slots": 704, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "prefix_storage": "u4",
         "storage": "u4"},
        # 256 samples of one very long prompt: the products over the prefix count.
        {"name": "shared-large", "op": "shared", "seqs": 256, "new": 1, "prefix": 32768, "low": 1, "high": 256,
         "slots": 256, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "prefix_storage": "bf16",
         "storage": "bf16"},
        # A single short conversation, one token at a time (latency).
        {"name": "weights-one-short", "op": "weights", "storage": "u4", "seqs": 1, "new": 1, "low": 100,
         "high": 100, "slots": 128, "heads": 8, "kv_heads": 8, "dim": 64, "dtype": "f32", "window": 0,
         "sinks": 0, "decay": 1.0},
        # A batched decode step of ragged sequences over a bf16 cache; old weight fades.
        {"name": "weights-batch", "op": "weights", "storage": "bf16", "seqs": 64, "new": 1, "low": 500,
         "high": 8192, "slots": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "window": 0,
         "sinks": 0, "decay": 0.95},
        # The last 16 tokens of eight prompts vote on what of them stays.
        {"name": "weights-vote", "op": "weights", "storage": "u4", "seqs": 8, "new": 16, "low": 1000,
         "high": 16384, "slots": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "window": 0,
         "sinks": 0, "decay": 0.0},
        # One very long document: the work has to be split over the keys.
        {"name": "weights-one-long", "op": "weights", "storage": "u4", "seqs": 1, "new": 1, "low": 131000,
         "high": 131000, "slots": 131072, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "window": 0,
         "sinks": 0, "decay": 1.0},
        # A few short conversations pass their budget (latency).
        {"name": "evict-small", "op": "evict", "storage": "u4", "seqs": 4, "low": 200, "high": 300, "slots": 320,
         "kv_heads": 8, "dim": 64, "keep": 256, "recent": 32, "sinks": 4, "to_slots": 320},
        # Ragged prompts shrink to a budget of 1024 keys as they move from the prompts' cache to the sequences'.
        {"name": "evict-prompts", "op": "evict", "storage": "bf16", "seqs": 32, "low": 900, "high": 8192,
         "slots": 8192, "kv_heads": 8, "dim": 128, "keep": 1024, "recent": 64, "sinks": 4, "to_slots": 1280},
        # One very long document shrinks to an eighth.
        {"name": "evict-one-long", "op": "evict", "storage": "bf16", "seqs": 1, "low": 131000, "high": 131000,
         "slots": 131072, "kv_heads": 8, "dim": 128, "keep": 16384, "recent": 1024, "sinks": 4,
         "to_slots": 20000},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    op = rng.choice(["shared", "shared", "weights", "weights", "evict"])
    dim = rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    if op == "evict":
        high = _spread(rng, 2, 100000)
        seqs = _spread(rng, 1, max(1, min(64, (1 << 26) // (high * kv_heads * dim))))
        keep = _spread(rng, 1, min(high, 20000))
        recent = rng.randrange(0, min(keep, 1000) + 1)
        return {"op": op, "storage": rng.choice(["u4", "bf16", "f32"]), "seqs": seqs, "low": max(1, high // 8),
                "high": high, "slots": high + rng.randrange(0, 40), "kv_heads": kv_heads, "dim": dim,
                "keep": keep, "recent": recent, "sinks": rng.randrange(0, min(keep - recent, 16) + 1),
                "to_slots": keep + rng.randrange(0, 300)}
    dtype = rng.choice(["f32", "bf16"])
    storage = rng.choice(["u4", "u4", dtype])
    case = {"op": op, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "storage": storage,
            "heads": kv_heads * rng.choice([1, 1, 2, 3, 4, 8]),
            "new": rng.choice([1, 1, rng.randrange(2, 17)]) if storage == "u4" else 1}
    if op == "shared":
        prefix = _spread(rng, 1, 60000)
        # The scores of all queries, and the rows' own keys.
        most = (1 << 25) // (prefix * case["heads"] * case["new"])
        seqs = _spread(rng, 1, max(1, min(256, most)))
        high = _spread(rng, max(1, case["new"]), max(case["new"], min(4000, (1 << 25) // (seqs * kv_heads * dim))))
        return {**case, "seqs": seqs, "prefix": prefix, "prefix_storage": rng.choice([storage, dtype, "u4"]),
                "low": rng.choice([case["new"] if case["new"] > 1 else 0, max(case["new"], high // 8)]),
                "high": high, "slots": high + rng.randrange(0, 40)}
    high = _spread(rng, max(2, case["new"]), 60000)
    seqs = _spread(rng, 1, max(1, min(256, (1 << 25) // (high * max(case["heads"] * case["new"], kv_heads * dim // 2)))))
    window = rng.choice([0, 0, _spread(rng, 1, 5000)])
    return {**case, "seqs": seqs, "low": max(case["new"], high // 8), "high": high,
            "slots": high + rng.randrange(0, 40), "window": window,
            "sinks": rng.randrange(0, 40) if window else 0, "decay": rng.choice([0.0, 1.0, 0.9])}


def _lengths(case):
    """The sequences' lengths: spread over [low, high] by the golden ratio, the first the longest."""
    span = case["high"] - case["low"]
    return [case["high"] - int(span * ((i * 0.6180339887498949) % 1.0)) for i in range(case["seqs"])]


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


# ---- the 4-bit cache in plain form -----------------------------------------------------------
def _quantise(x):
    """[..., dim] float32 -> codes uint8 [..., dim / 2] and (step, low) bf16 [..., dim / 32, 2]."""
    x = x.unflatten(-1, (-1, 32))
    low = x.amin(-1).to(torch.bfloat16)
    step = ((x.amax(-1) - low.float()) / 15.0).to(torch.bfloat16)
    code = ((x - low.float()[..., None]) / step.float().clamp(min=1e-30)[..., None]).round().clamp(0, 15)
    code = code.to(torch.uint8).unflatten(-1, (8, 4)).transpose(-3, -2)  # [..., 8, groups, 4]
    return (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-3), torch.stack([step, low], -1)


def _stands_for(codes, scale):
    """The float32 values of codes [..., dim / 2] with (step, low) [..., dim / 32, 2]."""
    groups = scale.shape[-2]
    pair = codes.unflatten(-1, (8, groups, 2))
    code = torch.stack([pair & 15, pair >> 4], -1).flatten(-2)           # [..., 8, groups, 4]
    code = code.transpose(-3, -2).flatten(-2).to(torch.float32)          # [..., groups, 32]
    scale = scale.to(torch.float32)
    return (scale[..., 1:] + code * scale[..., :1]).flatten(-2)


def _values(cache):
    """The float32 keys and values of a cache (k, v, k_scale, v_scale)."""
    k, v, k_scale, v_scale = cache
    if k_scale is None:
        return k.float(), v.float()
    return _stands_for(k, k_scale), _stands_for(v, v_scale)


# ---- inputs ----------------------------------------------------------------------------------
def _cache(normal, storage, rows, kv_heads, slots, dim, shift):
    k, v = normal(rows, kv_heads, slots, dim) + shift[:, None], normal(rows, kv_heads, slots, dim)
    if storage == "u4":
        (k, k_scale), (v, v_scale) = _quantise(k), _quantise(v)
        return k, v, k_scale, v_scale
    return k.to(_type(storage)), v.to(_type(storage)), None, None


def prepare(case, seed):
    """What a serving program holds before the call: caches, lengths, masses, this step's queries."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    seqs, kvh, dim, slots = case["seqs"], case["kv_heads"], case["dim"], case["slots"]
    state = {"case": case, "lengths": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")}
    # Keys have channels that lie far from zero, as they do in trained models.
    shift = 2.0 * normal(kvh, dim) * (torch.rand(kvh, dim, generator=g, device="cuda") < 0.1)
    state["cache"] = _cache(normal, case["storage"], seqs, kvh, slots, dim, shift)
    if case["op"] != "evict":
        new = case["new"]
        state["q"] = normal(seqs * new, case["heads"], dim).to(_type(case["dtype"]))
        state["starts"] = torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device="cuda")
    if case["op"] == "shared":
        state["prefix"] = _cache(normal, case["prefix_storage"], 1, kvh, case["prefix"], dim, shift)
    else:
        # Most keys gather little weight over a run, a few much.
        state["before"] = torch.rand(seqs, kvh, slots, generator=g, device="cuda") ** 8
    if case["op"] == "weights":
        state["mass"] = torch.zeros_like(state["before"])
    if case["op"] == "evict":
        room = case["to_slots"]
        state["to"] = tuple(None if x is None else torch.zeros((seqs, kvh, room) + x.shape[3:], dtype=x.dtype,
                                                               device="cuda") for x in state["cache"])
        state["mass"] = torch.zeros((seqs, kvh, room), device="cuda")
        state["read"] = torch.arange(0, seqs * case["keep"] + 1, case["keep"], dtype=torch.int32, device="cuda")
        state["all"] = torch.full((seqs,), case["keep"], dtype=torch.int32, device="cuda")
    if own:
        # The handles that a program keeps over its buffers.
        from basalt_b200 import operators
        state["handles"] = {x: operators.KvCache(*state[x]) for x in ("cache", "prefix", "to") if x in state}
    return state


# ---- one pass --------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _calls(state)
    if op == "shared":
        return _shared(state)
    if op == "weights":
        return _weighted(state)
    return _evict(state)


def _calls(state):
    """The calls of the framework's user."""
    from basalt_b200 import operators

    case, handles = state["case"], state["handles"]
    if case["op"] == "evict":
        lengths, kept = operators.kv_evict(handles["cache"], state["before"], state["lengths"], case["keep"],
                                           recent=case["recent"], sinks=case["sinks"], to=handles["to"],
                                           to_mass=state["mass"])
        if case["storage"] == "u4":
            moved = operators.kv_read(handles["to"], state["all"], starts=state["read"],
                                      tokens=case["seqs"] * case["keep"])
        else:
            moved = state["to"][:2]
        return (lengths, kept, state["mass"], *moved)
    starts = state["starts"] if case["new"] > 1 else None
    if case["op"] == "shared":
        return operators.attention_shared(handles["cache"], state["q"], state["lengths"], handles["prefix"],
                                          case["prefix"], starts=starts)
    out = operators.attention_weights(handles["cache"], state["q"], state["lengths"], state["mass"],
                                      previous=state["before"], decay=case["decay"], starts=starts,
                                      window=case["window"], sinks=case["sinks"])
    return out, state["mass"]


def _softmax(scores):
    """Weights of the scores above -inf; a row that has none has weights of zero."""
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / total.masked_fill(total == 0, 1.0)


def _queries(state):
    """float32 queries [seqs, kv_heads, group * new, dim], heads of a group first."""
    case = state["case"]
    q = state["q"].float().reshape(case["seqs"], case["new"], case["kv_heads"], -1, case["dim"])
    return q.permute(0, 2, 3, 1, 4).flatten(2, 3)


def _result(out, state):
    """[seqs, kv_heads, group * new, dim] as [tokens, heads, dim] of the queries' type."""
    case = state["case"]
    out = out.unflatten(2, (-1, case["new"])).permute(0, 3, 1, 2, 4)
    return out.reshape(-1, case["heads"], case["dim"]).to(state["q"].dtype)


def _hidden(state, window, sinks):
    """Which places of its row a query does not see: [seqs, 1, group * new, slots]."""
    case = state["case"]
    n, group = case["new"], case["heads"] // case["kv_heads"]
    key = torch.arange(case["slots"], device="cuda")
    position = (state["lengths"].long()[:, None] - n + torch.arange(n, device="cuda"))[..., None]
    seen = key <= position
    if window:
        seen &= (position - key < window) | (key < sinks)
    return ~seen.repeat(1, group, 1)[:, None]


def _shared(state):
    case = state["case"]
    k, v = _values(state["cache"])
    pk, pv = _values(state["prefix"])
    q = _queries(state) / math.sqrt(case["dim"])
    mine = (q @ k.transpose(-1, -2)).masked_fill(_hidden(state, 0, 0), -math.inf)
    rows = q.transpose(0, 1).flatten(1, 2)                                # [kv_heads, all queries, dim]
    common = (rows @ pk[0].transpose(-1, -2)).unflatten(1, (case["seqs"], -1)).transpose(0, 1)
    p = _softmax(torch.cat([common, mine], -1))
    common, mine = p.split([case["prefix"], case["slots"]], -1)
    out = (common.transpose(0, 1).flatten(1, 2) @ pv[0]).unflatten(1, (case["seqs"], -1)).transpose(0, 1)
    return _result(out + mine @ v, state)


def _weighted(state):
    case = state["case"]
    k, v = _values(state["cache"])
    scores = _queries(state) @ k.transpose(-1, -2) / math.sqrt(case["dim"])
    p = _softmax(scores.masked_fill(_hidden(state, case["window"], case["sinks"]), -math.inf))
    inside = (torch.arange(case["slots"], device="cuda") < state["lengths"][:, None])[:, None]
    state["mass"].copy_(torch.where(inside, case["decay"] * state["before"] + p.sum(2), state["mass"]))
    return _result(p @ v, state), state["mass"]


def _evict(state):
    case = state["case"]
    seqs, keep, room = case["seqs"], case["keep"], case["to_slots"]
    length = state["lengths"].long()[:, None, None]
    key = torch.arange(case["slots"], device="cuda")
    worth = state["before"].masked_fill((key < case["sinks"]) | (key >= length - case["recent"]), math.inf)
    worth = worth.masked_fill(key >= length, -math.inf)
    order = torch.sort(worth, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.where(order < length, order, case["slots"]).sort(-1).values
    there = kept < length
    place = kept.clamp(max=case["slots"] - 1)
    state["mass"].zero_()
    state["mass"][..., :keep] = state["before"].gather(2, place).masked_fill(~there, 0.0)
    row, head = torch.arange(seqs, device="cuda")[:, None, None], torch.arange(case["kv_heads"], device="cuda")[:, None]
    moved = [x[row, head, place] for x in _values(state["cache"])]
    moved = [x.masked_fill(~there[..., None], 0.0) for x in moved]
    if case["storage"] == "u4":
        moved = [x.transpose(1, 2).reshape(seqs * keep, case["kv_heads"], case["dim"]) for x in moved]
    else:
        state["to"][0][:, :, :keep], state["to"][1][:, :, :keep] = moved
        moved = state["to"][:2]
    lengths = state["lengths"].clamp(max=keep)
    return (lengths, torch.where(there, kept, -1).to(torch.int32), state["mass"], *moved)


# ---- what a pass cannot do without -----------------------------------------------------------
def _bytes(storage):
    return {"u4": 0.625, "bf16": 2, "f32": 4}[storage]


def work(case):
    kvh, dim = case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        every, kept = sum(_lengths(case)), sum(min(case["keep"], n) for n in _lengths(case))
        # Masses; what stays, read and written, with its masses and places.
        return {"bytes": int(kvh * (4 * every + kept * (4 * dim * _bytes(case["storage"]) + 8))),
                "flops": kvh * every}
    new, window, sinks = case["new"], case.get("window", 0), case.get("sinks", 0)

    def sees(position):
        """Keys of its own row that a query at `position` sees."""
        n = position + 1
        return n if not window or n <= window + sinks else window + sinks

    lengths = _lengths(case)
    pairs = sum(sees(i) for n in lengths for i in range(n - new, n))
    keys = sum(min(n, sees(n - 1) + new - 1) for n in lengths)
    tokens = new * case["seqs"]
    size = tokens * case["heads"] * dim * 2 * (4 if case["dtype"] == "f32" else 2)
    size += 2 * keys * kvh * dim * _bytes(case["storage"])
    if case["op"] == "shared":
        size += 2 * case["prefix"] * kvh * dim * _bytes(case["prefix_storage"])
        pairs += tokens * case["prefix"]
    else:
        size += sum(lengths) * kvh * (8 if case["decay"] else 4)
    return {"bytes": int(size), "flops": 4 * pairs * case["heads"] * dim}


# ---- the definition in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    """What `run` returns, from the definitions alone, in 64 bits."""
    state = prepare(case, seed)
    kvh, dim = case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        return _exact_evict(case, state)
    group, new = case["heads"] // kvh, case["new"]
    out = torch.zeros((case["seqs"], new, case["heads"], dim), dtype=torch.float64, device="cuda")
    mass = state["mass"].double() if case["op"] == "weights" else None
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    for h in range(kvh):
        if case["op"] == "shared":
            first_k, first_v = _exact_head(state["prefix"], 0, h)
        for s, length in enumerate(_lengths(case)):
            keys, values = (x[:length] for x in _exact_head(state["cache"], s, h))
            q = state["q"][s * new:(s + 1) * new, h * group:(h + 1) * group].double()
            i = torch.arange(length - new, length, device="cuda")[:, None, None]
            j = torch.arange(length, device="cuda")
            unseen = (j > i) | ((i - j >= window) & (j >= sinks) if window else torch.zeros_like(j > i))
            score = torch.einsum("nhc,jc->nhj", q, keys) * dim ** -0.5
            score = torch.where(unseen, -math.inf, score)
            if case["op"] == "shared":
                score = torch.cat([torch.einsum("nhc,jc->nhj", q, first_k) * dim ** -0.5, score], -1)
                values = torch.cat([first_v, values])
            p = torch.softmax(score, -1)
            out[s, :, h * group:(h + 1) * group] = torch.einsum("nhj,jc->nhc", p, values)
            if mass is not None:
                mass[s, h, :length] = case["decay"] * state["before"][s, h, :length].double() + p.sum((0, 1))
    out = out.reshape(-1, case["heads"], dim).cpu().numpy()
    return out if mass is None else (out, mass.cpu().numpy())


def _exact_head(cache, row, head):
    """The keys and values [slots, dim] of one head of a cache's row, in 64 bits."""
    k, v, k_scale, v_scale = cache
    if k_scale is None:
        return k[row, head].double(), v[row, head].double()
    c = torch.arange(2 * k.shape[-1], device="cuda")
    group, half, nibble = c // 32, c % 32 // 4, c % 4
    found = []
    for codes, scale in ((k, k_scale), (v, v_scale)):
        byte = codes[row, head][:, (half * scale.shape[-2] + group) * 2 + nibble // 2].to(torch.int64)
        pair = scale[row, head].double()[:, group]
        found.append(pair[..., 1] + torch.where(nibble % 2 == 1, byte // 16, byte % 16) * pair[..., 0])
    return found


def _exact_evict(case, state):
    """Nothing is computed but the places: they, the masses and the values go by a sort on the host."""
    kvh, keep, dim = case["kv_heads"], case["keep"], case["dim"]
    before = state["before"].cpu().numpy()
    mass = np.zeros((case["seqs"], kvh, case["to_slots"]))
    shape = (case["seqs"], keep, kvh, dim) if case["storage"] == "u4" else (case["seqs"], kvh, case["to_slots"], dim)
    moved = np.zeros((2,) + shape)
    for s, length in enumerate(_lengths(case)):
        for h in range(kvh):
            places = range(length)
            if length > keep:
                some = range(case["sinks"], length - case["recent"])
                best = sorted(some, key=lambda j: (-before[s, h, j], j))
                best = best[:keep - case["sinks"] - case["recent"]]
                places = sorted({*range(case["sinks"]), *best, *range(length - case["recent"], length)})
            places = list(places)
            mass[s, h, :len(places)] = before[s, h, places]
            for which, x in enumerate(_exact_head(state["cache"], s, h)):
                x = x[places].cpu().numpy()
                if case["storage"] == "u4":
                    moved[which, s, :len(places), h] = x
                else:
                    moved[which, s, h, :len(places)] = x
    if case["storage"] == "u4":
        moved = moved.reshape(2, -1, kvh, dim)
    return None, None, mass, moved[0], moved[1]
