"""Workloads of the serving operators: a cache of keys and values held in 4 bits, the attention that
reads it, attention with a sliding window and a few first tokens that stay visible, and drawing
tokens from filtered distributions.

Each operator has a plain form in elementary torch operations (``own = False``) and the calls of
``basalt_b200.operators`` (``own = True``) on the same inputs.

Definitions shared by all attention cases: a sequence has ``length`` cached keys after its own
tokens were stored, query i of its n tokens stands at position ``length - n + i`` and sees key j
when ``j <= position`` and (``window`` is 0, or ``position - j < window``, or ``j < sinks``).

The 4-bit cache holds 32 consecutive channels of one head of one token as a group: ``low`` is the
group's minimum rounded down to bf16, ``step`` is ``(maximum - low) / 15`` rounded up to bf16, and a
channel's code is ``(x - low) / step`` rounded to the nearest even whole number. It stands for
``low + code * step``. Codes of a head are kept as [8][groups][4] nibbles, low nibble first: channel
``32 g + 4 h + j`` is nibble j of the 16 bits at [h][g].
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

# Log-weights below this (2^-40 of the likeliest token) are never drawn.
CUT = -40.0 * math.log(2.0)


def listed():
    """The cases, each with what it stands for in use."""
    return [
        # One decode step of 32 sequences: each stores one token's keys and values (latency).
        {"name": "store-step", "op": "store", "seqs": 32, "new": 1, "low": 33, "high": 128,
         "slots": 128, "kv_heads": 8, "dim": 64, "dtype": "f32"},
        # A batch of 256 prompts of 256 tokens moves into the cache and is read back.
        {"name": "store-prompts", "op": "store", "seqs": 256, "new": 256, "low": 256, "high": 256,
         "slots": 512, "kv_heads": 8, "dim": 64, "dtype": "f32"},
        # A single short conversation, one token at a time (latency).
        {"name": "cached-one-short", "op": "cached", "storage": "u4", "seqs": 1, "new": 1,
         "low": 100, "high": 100, "slots": 128, "heads": 8, "kv_heads": 8, "dim": 64,
         "dtype": "f32", "window": 0, "sinks": 0},
        # The batched decode step of 256 sequences, lengths spread as they are in mid-run.
        {"name": "cached-batch", "op": "cached", "storage": "u4", "seqs": 256, "new": 1,
         "low": 257, "high": 512, "slots": 512, "heads": 8, "kv_heads": 8, "dim": 64,
         "dtype": "f32", "window": 0, "sinks": 0},
        # One very long document, grouped heads: the work has to be split over the keys.
        {"name": "cached-one-long", "op": "cached", "storage": "u4", "seqs": 1, "new": 1,
         "low": 131000, "high": 131000, "slots": 131072, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "window": 0, "sinks": 0},
        # Four drafted tokens of each sequence are checked at once, ragged lengths.
        {"name": "cached-drafts", "op": "cached", "storage": "u4", "seqs": 24, "new": 4,
         "low": 900, "high": 16384, "slots": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "window": 0, "sinks": 0},
        # A decode step that sees the last 2048 tokens and the first 4 of an unquantised cache.
        {"name": "window-step", "op": "cached", "storage": "bf16", "seqs": 64, "new": 1,
         "low": 500, "high": 8192, "slots": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "window": 2048, "sinks": 4},
        # One long prompt through a windowed layer.
        {"name": "window-prompt", "op": "packed", "seqs": 1, "low": 8192, "high": 8192,
         "heads": 16, "kv_heads": 4, "dim": 128, "dtype": "bf16", "window": 1024, "sinks": 4},
        # A batch of short ragged prompts in fp32, one token the shortest.
        {"name": "window-ragged", "op": "packed", "seqs": 24, "low": 1, "high": 700,
         "heads": 8, "kv_heads": 8, "dim": 64, "dtype": "f32", "window": 256, "sinks": 4},
        # A small batch over a small vocabulary, the usual filters (latency).
        {"name": "sample-small", "op": "sample", "rows": 32, "vocabulary": 4096, "dtype": "f32",
         "temperature": 0.8, "top_k": 40, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # Many rows drawn from their whole distribution.
        {"name": "sample-many", "op": "sample", "rows": 2048, "vocabulary": 8192, "dtype": "f32",
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False},
        # A large vocabulary in bf16; each request has its own settings.
        {"name": "sample-large", "op": "sample", "rows": 64, "vocabulary": 131072, "dtype": "bf16",
         "temperature": 0.9, "top_k": 200, "top_p": 0.95, "min_p": 0.02, "mixed": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    op = rng.choice(["store", "cached", "cached", "packed", "sample"])
    if op == "sample":
        vocabulary = _spread(rng, 50, 150000)
        return {"op": op, "rows": _spread(rng, 1, max(1, min(2048, (1 << 23) // vocabulary))),
                "vocabulary": vocabulary, "dtype": rng.choice(["f32", "bf16"]),
                "temperature": round(rng.uniform(0.2, 1.5), 3),
                "top_k": rng.choice([0, _spread(rng, 1, 1000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]),
                "mixed": rng.random() < 0.4}
    dim = rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    dtype = rng.choice(["f32", "bf16"])
    case = {"op": op, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if op == "store":
        high = _spread(rng, 2, 2000)
        new = rng.choice([1, _spread(rng, 1, high)])
        seqs = _spread(rng, 1, max(1, min(256, (1 << 23) // (high * kv_heads * dim))))
        return {**case, "seqs": seqs, "new": new, "low": new, "high": high,
                "slots": high + rng.randrange(0, 60)}
    case["heads"] = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    case["window"] = rng.choice([0, _spread(rng, 1, 3000)])
    case["sinks"] = rng.randrange(0, 40) if case["window"] else 0
    if op == "packed":
        case["heads"] = kv_heads * rng.choice([1, 2])
        high = _spread(rng, 2, 4000)
        seqs = _spread(rng, 1, max(1, min(32, 6000 // high)))
        case["window"] = case["window"] or 512
        return {**case, "seqs": seqs, "low": max(1, high // 8), "high": high}
    high = _spread(rng, 2, 60000)
    seqs = _spread(rng, 1, max(1, min(256, (1 << 26) // (high * kv_heads * dim))))
    storage = rng.choice(["u4", "u4", "u4", dtype])
    new = rng.choice([1, 1, rng.randrange(2, 9)]) if storage == "u4" else 1
    return {**case, "storage": storage, "seqs": seqs, "new": min(new, high),
            "low": max(min(new, high), high // 8), "high": high, "slots": high + rng.randrange(0, 40)}


def _lengths(case):
    """The sequences' lengths: spread over [low, high] by the golden ratio, the first the longest."""
    span = case["high"] - case["low"]
    return [case["high"] - int(span * ((i * 0.6180339887498949) % 1.0)) for i in range(case["seqs"])]


def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


# ---- the 4-bit cache in plain form -----------------------------------------------------------
def _bf16_up(x):
    """Non-negative doubles rounded up to bf16, as float32."""
    f = x.to(torch.float32)
    f = torch.where(f.double() < x, torch.nextafter(f, torch.full_like(f, math.inf)), f)
    bits = f.view(torch.int32)
    up = torch.where((bits & 0xFFFF) != 0, (bits & -65536) + 65536, bits)
    return up.view(torch.float32)


def _bf16_down(x):
    """float32 rounded down to bf16, as float32."""
    bits = x.view(torch.int32)
    cut = bits & -65536
    return torch.where((bits < 0) & ((bits & 0xFFFF) != 0), cut + 65536, cut).view(torch.float32)


def _quantise(x):
    """[..., dim] -> codes uint8 [..., dim / 2] and (step, low) bf16 [..., dim / 32, 2]."""
    groups = x.shape[-1] // 32
    x = x.to(torch.float32).unflatten(-1, (groups, 32))
    low = _bf16_down(x.amin(-1))
    step = _bf16_up((x.amax(-1).double() - low.double()) / 15.0)
    d = torch.where(step == 0, 1.0, step.double())
    code = ((x.double() - low.double()[..., None]) / d[..., None]).round().clamp(0, 15)
    code = code.to(torch.uint8).unflatten(-1, (8, 4)).transpose(-3, -2)  # [..., 8, groups, 4]
    code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code.flatten(-3), torch.stack([step, low], -1).to(torch.bfloat16)


def _stands_for(codes, scale):
    """The float32 values of codes [..., dim / 2] with (step, low) [..., dim / 32, 2]."""
    groups = scale.shape[-2]
    pair = codes.unflatten(-1, (8, groups, 2))
    code = torch.stack([pair & 15, pair >> 4], -1).flatten(-2)           # [..., 8, groups, 4]
    code = code.transpose(-3, -2).flatten(-2).to(torch.float32)          # [..., groups, 32]
    scale = scale.to(torch.float32)
    return (scale[..., 1:] + code * scale[..., :1]).flatten(-2)


# ---- inputs ----------------------------------------------------------------------------------
def prepare(case, seed):
    """What a serving program holds before the call: caches, lengths, this step's tensors."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    state = {"case": case}
    if case["op"] == "sample":
        rows, V = case["rows"], case["vocabulary"]
        state["logits"] = (3.0 * normal(rows, V)).to(_type(case["dtype"]))
        state["uniforms"] = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)

        def setting(value, dtype, *others):
            if not case["mixed"]:
                return value
            t = torch.full((rows,), value, dtype=dtype, device="cuda")
            pick = torch.randint(0, 4, (rows,), generator=g, device="cuda")
            return torch.where(pick == 1, others[0], torch.where(pick == 2, others[1], t)).to(dtype)

        state["temperature"] = setting(case["temperature"], torch.float32, 0.0, 1.0)
        state["top_k"] = setting(case["top_k"], torch.int32, 0, 1)
        state["top_p"] = setting(case["top_p"], torch.float32, 1.0, 0.5)
        state["min_p"] = setting(case["min_p"], torch.float32, 0.0, 0.1)
        return state
    lengths = _lengths(case)
    kvh, dim, dtype = case["kv_heads"], case["dim"], _type(case["dtype"])
    counts = lengths if case["op"] == "packed" else [case["new"]] * case["seqs"]
    tokens = sum(counts)
    starts = np.concatenate([[0], np.cumsum(counts)])
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    # Keys have channels that lie far from zero, as they do in trained models.
    shift = 2.0 * normal(kvh, dim) * (torch.rand(kvh, dim, generator=g, device="cuda") < 0.1)
    if case["op"] == "packed":
        # Queries, keys and values are slices of one fused projection.
        width = (case["heads"] + 2 * kvh) * dim
        fused = normal(tokens, width).to(dtype)
        split = [case["heads"] * dim, kvh * dim, kvh * dim]
        q, k, v = (x.unflatten(-1, (-1, dim)) for x in fused.split(split, -1))
        k += shift.to(dtype)
        return {**state, "q": q, "k": k, "v": v}
    rows, slots = case["seqs"], case["slots"]
    if case["op"] == "store":
        state["k"] = (normal(tokens, kvh, dim) + shift).to(dtype)
        state["v"] = normal(tokens, kvh, dim).to(dtype)
        k_codes = torch.zeros((rows, kvh, slots, dim // 2), dtype=torch.uint8, device="cuda")
        k_scale = torch.zeros((rows, kvh, slots, dim // 32, 2), dtype=torch.bfloat16, device="cuda")
        v_codes, v_scale = k_codes.clone(), k_scale.clone()
    else:
        state["q"] = normal(tokens, case["heads"], dim).to(dtype)
        k = normal(rows, kvh, slots, dim) + shift[:, None]
        v = normal(rows, kvh, slots, dim)
        if case["storage"] == "u4":
            (k_codes, k_scale), (v_codes, v_scale) = _quantise(k), _quantise(v)
        else:
            k_codes, v_codes = (x.to(_type(case["storage"])) for x in (k, v))
            k_scale = v_scale = None
    state.update(k_codes=k_codes, v_codes=v_codes, k_scale=k_scale, v_scale=v_scale)
    if own:
        # The handle that a program keeps over its buffers.
        from basalt_b200 import operators
        state["cache"] = operators.KvCache(k_codes, v_codes, k_scale, v_scale)
    return state


# ---- one pass --------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _calls(state)
    if case["op"] == "store":
        return _store(state)
    if case["op"] == "cached":
        return _cached(state)
    if case["op"] == "packed":
        return _packed(state)
    return _sample(state)


def _calls(state):
    """The calls of the framework's user."""
    from basalt_b200 import operators

    case = state["case"]
    if case["op"] == "store":
        operators.kv_append(state["cache"], state["k"], state["v"], state["lengths"],
                            starts=state["starts"])
        return operators.kv_read(state["cache"], state["lengths"], starts=state["starts"],
                                 tokens=state["k"].shape[0], dtype=state["k"].dtype)
    if case["op"] == "cached":
        starts = state["starts"] if case["new"] > 1 else None
        return operators.attention_cached(state["cache"], state["q"], state["lengths"],
                                          starts=starts, window=case["window"],
                                          sinks=case["sinks"])
    if case["op"] == "packed":
        return operators.attention_packed(state["q"], state["k"], state["v"], state["starts"],
                                          window=case["window"], sinks=case["sinks"])
    return operators.sample_tokens(state["logits"], state["uniforms"],
                                   temperature=state["temperature"], top_k=state["top_k"],
                                   top_p=state["top_p"], min_p=state["min_p"])


def _store(state):
    """The new tokens' codes go into their slots; the values they stand for are read back."""
    case = state["case"]
    n = case["new"]
    row = torch.arange(case["seqs"], device="cuda").repeat_interleave(n)
    slot = (state["lengths"].long()[:, None] - n + torch.arange(n, device="cuda")).flatten()
    for x, codes, scale in ((state["k"], state["k_codes"], state["k_scale"]),
                            (state["v"], state["v_codes"], state["v_scale"])):
        c, s = _quantise(x)
        codes[row, :, slot] = c
        scale[row, :, slot] = s
    return tuple(_stands_for(codes[row, :, slot], scale[row, :, slot]).to(state["k"].dtype)
                 for codes, scale in ((state["k_codes"], state["k_scale"]),
                                      (state["v_codes"], state["v_scale"])))


def _visible(position, key, window, sinks):
    seen = key <= position
    if window:
        seen &= (position - key < window) | (key < sinks)
    return seen


def _weights(scores, seen):
    """Softmax over the visible keys; a row that sees none has weights of zero."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / total.masked_fill(total == 0, 1.0)


def _cached(state):
    case = state["case"]
    n, kvh, dim = case["new"], case["kv_heads"], case["dim"]
    if case["storage"] == "u4":
        k = _stands_for(state["k_codes"], state["k_scale"])
        v = _stands_for(state["v_codes"], state["v_scale"])
    else:
        k, v = state["k_codes"].float(), state["v_codes"].float()
    q = state["q"].float().reshape(case["seqs"], n, kvh, -1, dim).permute(0, 2, 3, 1, 4)
    group = q.shape[2]
    scores = (q.flatten(2, 3) @ k.transpose(-1, -2)) / math.sqrt(dim)
    position = state["lengths"].long()[:, None] - n + torch.arange(n, device="cuda")
    seen = _visible(position[..., None], torch.arange(case["slots"], device="cuda"),
                    case["window"], case["sinks"])                     # [seqs, n, slots]
    p = _weights(scores.unflatten(2, (group, n)), seen[:, None, None]).flatten(2, 3)
    out = (p @ v).unflatten(2, (group, n)).permute(0, 3, 1, 2, 4)
    return out.reshape(case["seqs"] * n, case["heads"], dim).to(state["q"].dtype)


def _packed(state):
    case = state["case"]
    kvh, dim = case["kv_heads"], case["dim"]
    starts = state["starts"].long()
    tokens = state["q"].shape[0]
    at = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts, at, right=True) - 1
    position = at - starts[seq]
    q = state["q"].float().unflatten(1, (kvh, -1)).permute(1, 2, 0, 3)  # [kv, group, tokens, dim]
    k, v = (state[x].float().transpose(0, 1)[:, None] for x in ("k", "v"))
    seen = _visible(position[:, None], position[None], case["window"], case["sinks"])
    seen &= seq[:, None] == seq[None]
    p = _weights((q @ k.transpose(-1, -2)) / math.sqrt(dim), seen)
    return (p @ v).permute(2, 0, 1, 3).flatten(1, 2).to(state["q"].dtype)


def _column(value, rows):
    if not isinstance(value, torch.Tensor):
        value = torch.full((rows,), value, dtype=torch.float32, device="cuda")
    return value.double()[:, None]


def _sample(state):
    """In order: temperature, the top_k largest, the smallest set of the largest that holds top_p of
    what is left, weights of at least min_p of the largest; then the first token, by index, at which
    the running sum passes uniform * total. Ties are kept lowest index first. A temperature of zero
    takes the first of the largest."""
    x = state["logits"].double()
    rows, V = x.shape
    t, k, p, least = (_column(state[n], rows) for n in ("temperature", "top_k", "top_p", "min_p"))
    top = x.amax(-1, keepdim=True)
    greedy = t <= 0
    z = (x - top) / torch.where(greedy, 1.0, t)
    w = torch.where(z >= CUT, torch.exp(z), 0.0)
    _, order = torch.sort(x, dim=-1, descending=True, stable=True)
    s = w.gather(-1, order)
    rank = torch.arange(V, device="cuda")
    kept = (k <= 0) | (rank < k)
    s = torch.where(kept, s, 0.0)
    running = s.cumsum(-1)
    before = running.roll(1, -1)
    before[:, 0] = 0.0
    kept = (p >= 1) | (before < p * running[:, -1:]) | (rank == 0)
    kept &= s >= least.clamp(max=1.0)
    w = torch.zeros_like(w).scatter(-1, order, torch.where(kept, s, 0.0))
    running = w.cumsum(-1)
    token = (running <= state["uniforms"][:, None] * running[:, -1:]).sum(-1)
    return torch.where(greedy[:, 0], order[:, 0], token).to(torch.int32)


# ---- what a pass cannot do without -----------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocabulary"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * 12,
                "flops": 4 * n}
    kvh, dim = case["kv_heads"], case["dim"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "store":
        values = 2 * case["seqs"] * case["new"] * kvh * dim
        # The inputs, the codes and scales they become, and the values read back.
        return {"bytes": int(values * (2 * size + 0.625)), "flops": 6 * values}
    window, sinks = case["window"], case["sinks"]

    def sees(position):
        """Keys that a query at `position` sees."""
        n = position + 1
        return n if not window or n <= window + sinks else window + sinks

    keys = pairs = tokens = 0
    for n in _lengths(case):
        new = n if case["op"] == "packed" else case["new"]
        tokens += new
        pairs += sum(sees(i) for i in range(n - new, n))
        keys += n if case["op"] == "packed" else min(n, sees(n - 1) + new - 1)
    per_value = 0.625 if case.get("storage") == "u4" else size
    return {"bytes": int(2 * keys * kvh * dim * per_value + 2 * tokens * case["heads"] * dim * size),
            "flops": 4 * pairs * case["heads"] * dim}


# ---- the definition in 64 bits ---------------------------------------------------------------
def exact(case, seed):
    """What `run` returns, from the definitions alone, in 64 bits."""
    state = prepare(case, seed)
    if case["op"] == "sample":
        return None  # whole numbers, which have no error
    if case["op"] == "store":
        return tuple(_exact_group(state[x]).cpu().numpy() for x in ("k", "v"))
    dim, kvh, heads = case["dim"], case["kv_heads"], case["heads"]
    window, sinks = case["window"], case["sinks"]
    out = np.zeros((state["q"].shape[0], heads, dim))
    starts = state["starts"].cpu().tolist()
    for s, length in enumerate(_lengths(case)):
        first, last = starts[s], starts[s + 1]
        if case["op"] == "packed":
            keys, values = (state[x][first:last].double() for x in ("k", "v"))
        else:
            keys, values = (_exact_row(state, x, s)[:, :length].transpose(0, 1) for x in "kv")
        i = torch.arange(length - (last - first), length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        hidden = (j > i) | ((i - j >= window) & (j >= sinks) if window else torch.zeros_like(j > i))
        for h in range(heads):
            score = state["q"][first:last, h].double() @ keys[:, h * kvh // heads].T * dim ** -0.5
            score[hidden] = -math.inf
            p = torch.softmax(score, -1)
            out[first:last, h] = (p @ values[:, h * kvh // heads]).cpu().numpy()
    return out


def _exact_row(state, which, row):
    """The values [kv_heads, slots, dim] of one cache row."""
    codes, scale = state[which + "_codes"][row], state[which + "_scale"]
    if scale is None:
        return codes.double()
    groups = scale.shape[-2]
    c = torch.arange(32 * groups, device="cuda")
    group, half, nibble = c // 32, c % 32 // 4, c % 4
    byte = codes[..., (half * groups + group) * 2 + nibble // 2].to(torch.int64)
    code = torch.where(nibble % 2 == 1, byte // 16, byte % 16).double()
    pair = scale[row][..., group, :].double()
    return pair[..., 1] + code * pair[..., 0]


def _exact_group(x):
    """Each value after 4 bits: the nearest of the 16 that its group can hold."""
    x = x.double()
    parts = x.reshape(*x.shape[:-1], -1, 32)

    def to_bf16(y, up):
        exponent = torch.floor(torch.log2(y.abs().clamp(min=1e-300)))
        # log2 may round up to a power of two that is not reached
        exponent = torch.where(torch.exp2(exponent) > y.abs(), exponent - 1, exponent)
        unit = torch.exp2(exponent - 7)
        return (torch.ceil(y / unit) if up else torch.floor(y / unit)) * unit

    low = to_bf16(parts.min(-1, keepdim=True).values, False)
    step = to_bf16((parts.max(-1, keepdim=True).values - low) / 15, True)
    code = torch.round((parts - low) / torch.where(step > 0, step, 1.0))
    return (low + code * step).reshape(x.shape)
