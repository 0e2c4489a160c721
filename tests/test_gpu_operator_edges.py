"""The serving operators on the GPU at the edges of their arguments, against plain 64-bit formulas.

Tolerances are those of test_gpu_operators.py's bound(): a score of d products is off by at most
(d + 8) 2^-23 sum|q k| scale, a weight by twice that and 2^-21, a sum of n weights by (n + 16) 2^-23,
each in units of the largest value that the query sees; bf16 adds 2^-8 of that and of the output.
"""
import math

import numpy as np
import pytest

import operator_reference as ref
from test_gpu_operators import bound, host, ints, ops, tensor, torch_  # noqa: F401 (ops: a fixture)

pytestmark = pytest.mark.gpu


def attend(q, k, v, first=0, window=0, sinks=0, scale=None):
    """One sequence by the formula alone, NaN and infinities as 64-bit arithmetic has them; and the
    bound's sizes: per query and head the largest sum |q k| scale, per output the largest finite
    |v| that the query sees."""
    n, H, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, size, most = np.zeros((n, H, d)), np.zeros((n, H)), np.zeros((n, H, d))
    with np.errstate(all="ignore"):
        for i in range(n):
            if first + i < 0:
                continue
            seen = ref.visible(first + i, k.shape[0], window, sinks)
            for h in range(H):
                kk, vv = k[seen, h * k.shape[1] // H], v[seen, h * k.shape[1] // H]
                s = kk @ q[i, h] * scale
                p = np.exp(s - s.max())
                out[i, h] = p @ vv / p.sum()
                sizes = np.abs(kk) @ np.abs(q[i, h]) * abs(scale)
                size[i, h] = sizes[np.isfinite(sizes)].max(initial=0.0)
                most[i, h] = np.where(np.isfinite(vv), np.abs(vv), 0).max(0)
    return out, size, most


def check(got, want, size, most, d, n, dtype):
    """NaN and infinities where the formula has them, elsewhere numbers within the bound."""
    tol = bound(size, d, n, most, np.where(np.isfinite(want), want, 0), dtype)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    whole = np.isinf(want)
    assert np.array_equal(got[whole], want[whole])
    ok = np.isfinite(want)
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok]), np.abs(got[ok] - want[ok]).max()


def prompt(rng, T, heads, kv_heads, dim, dtype):
    return [tensor(rng.standard_normal((T, h, dim)).astype(np.float32), dtype)
            for h in (heads, kv_heads, kv_heads)]


# ---- packed prompts ----------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("which", [0, 1, 2], ids="qkv")
@pytest.mark.parametrize("dtype,bits", [("f32", 0x7fffffff), ("f32", -1), ("f32", 0x7f800001),
                                        ("f32", 0x7fc00000), ("bf16", 0x7fff), ("bf16", -1)])
def test_any_nan_of_a_prompt_reaches_the_queries_that_see_it(ops, dtype, bits, which, dim):
    """Whatever its bits, in tiles of keys that all of a tile's queries see and in others."""
    torch = torch_()
    x = prompt(np.random.default_rng(dim + which), 200, 2, 2, dim, dtype)
    x[which].view(torch.int32 if dtype == "f32" else torch.int16)[20, 1, 3] = bits
    got = host(ops.attention_packed(*x, ints([0, 200])))
    want, size, most = attend(*[host(t) for t in x])
    assert np.isnan(want).any() and np.isfinite(want[:, 0]).all()
    check(got, want, size, most, dim, 200, dtype)


def test_a_nan_group_of_a_4_bit_cache_stays_one_in_a_prompt(ops):
    """Values read back from the cache go into a prompt's attention, as an engine's do."""
    rng = np.random.default_rng(21)
    q, k, v = prompt(rng, 150, 2, 2, 64, "f32")
    k[30, 0, 40], v[20, 1, 5] = float("nan"), float("inf")
    cache, starts = ops.KvCache.allocate(1, 2, 150, 64), ints([0, 150])
    ops.kv_append(cache, k, v, ints([150]), starts=starts)
    k, v = ops.kv_read(cache, ints([150]), starts=starts, tokens=150)
    want, size, most = attend(host(q), host(k), host(v))
    assert np.isnan(want[30:, 0]).all() and np.isnan(want[20:, 1, :32]).all()
    check(host(ops.attention_packed(q, k, v, starts)), want, size, most, 64, 150, "f32")
    # and the cached form of the last query sees the same
    got = host(ops.attention_cached(cache, q[149:], ints([150])))
    check(got, want[149:], size[149:], most[149:], 64, 150, "f32")


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("which,value", [(1, math.inf), (1, -math.inf), (2, math.inf), (2, -math.inf),
                                         (1, -3.4025e38), (2, 3.4028e38)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_visible_infinities_count_as_the_formula_has_them(ops, dtype, which, value, dim, window, sinks):
    """A key of -inf weighs nothing, one of +inf leaves NaN, an infinite value an infinity: in tiles
    that all queries see as in others. The last two values are floats that the parts of tf32, and
    bf16, round to infinity."""
    rng = np.random.default_rng(dim)
    x = prompt(rng, 200, 2, 2, dim, dtype)
    x[0][:, :, 3] = x[0][:, :, 3].abs() * 0.1 + 0.5       # the sign of the score
    x[which][20, 1, 3] = value
    got = host(ops.attention_packed(*x, ints([0, 200]), window=window, sinks=sinks))
    xh = [host(t) for t in x]
    want, size, most = attend(*xh, 0, window, sinks)
    if which == 1:   # the largest score decides the bound, not the one that weighs nothing
        size = attend(xh[0], np.where(np.abs(xh[1]) > 1e38, 0, xh[1]), xh[2], 0, window, sinks)[1]
    check(got, want, size, most, dim, 200, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,scale", [(2, 2, None), (6, 2, -0.2), (5, 1, 0.5)])
def test_rows_that_are_computed_again_are_as_good(ops, dtype, dim, heads, kv_heads, scale):
    """A value that is not finite has its neighbours' rows computed by another kernel: to the bounds
    that all rows have."""
    rng = np.random.default_rng(dim + heads)
    q, k, v = prompt(rng, 230, heads, kv_heads, dim, dtype)
    k[150, kv_heads - 1], v[150, kv_heads - 1] = math.nan, math.inf
    starts = [0, 30, 230]
    got = host(ops.attention_packed(q, k, v, ints(starts), window=50, sinks=2, scale=scale))
    for a, b in zip(starts, starts[1:]):
        want, size, most = attend(*[host(t)[a:b] for t in (q, k, v)], 0, 50, 2, scale)
        check(got[a:b], want, size, most, dim, 200, dtype)


@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 4)])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.2, 3.0, 1e-40])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompts_at_any_scale(ops, dtype, dim, scale, window, sinks):
    """Zero gives the mean of the visible values, a negative one turns the order around. Aligned
    tensors, so that bf16 takes the tensor-core kernel, and heads that share keys."""
    rng = np.random.default_rng(dim + window)
    q, k, v = prompt(rng, 500, 6, 2, dim, dtype)
    starts = [0, 99, 99, 500]
    got = host(ops.attention_packed(q, k, v, ints(starts), window=window, sinks=sinks, scale=scale))
    for a, b in zip(starts, starts[1:]):
        want, size, most = attend(*[host(t)[a:b] for t in (q, k, v)], 0, window, sinks, scale)
        check(got[a:b], want, size, most, dim, 500, dtype)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("group", [1, 3, 20])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("storage", ["u4", "f32", "bf16"])
def test_cached_attention_at_any_scale(ops, storage, dtype, group, scale):
    rng = np.random.default_rng(group)
    k, v = (tensor(rng.standard_normal((60, 2, 64)).astype(np.float32)) for _ in range(2))
    cache, starts = ops.KvCache.allocate(1, 2, 64, 64, storage), ints([0, 60])
    ops.kv_append(cache, k, v, ints([60]), starts=starts)
    k, v = (host(t) for t in ops.kv_read(cache, ints([60]), starts=starts, tokens=60))
    q = tensor(rng.standard_normal((1, 2 * group, 64)).astype(np.float32), dtype)
    want, size, most = attend(host(q), k, v, 59, 0, 0, scale)
    check(host(ops.attention_cached(cache, q, ints([60]), scale=scale)), want, size, most, 64, 60, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts,lengths,window", [([300, 301], [5000, 700], 0),
                                                   ([1, 2, 150], [9000, 40, 8000], 0),
                                                   ([300, 301], [5000, 700], 1000)])
def test_chunks_of_prompts_over_a_long_cache(ops, dtype, counts, lengths, window):
    torch = torch_()
    rng = np.random.default_rng(sum(counts))
    S, slots, heads, kv_heads, dim = len(counts), 20000, 8, 2, 64
    cache = ops.KvCache.allocate(S, kv_heads, slots, dim)
    stored = np.concatenate([[0], np.cumsum(lengths)])
    x = [tensor(rng.standard_normal((stored[-1], kv_heads, dim)).astype(np.float32)) for _ in range(2)]
    ops.kv_append(cache, *x, ints(lengths), starts=ints(stored))
    k, v = (t.double() for t in ops.kv_read(cache, ints(lengths), starts=ints(stored),
                                            tokens=int(stored[-1])))
    q = tensor(rng.standard_normal((sum(counts), heads, dim)).astype(np.float32), dtype)
    starts = np.concatenate([[0], np.cumsum(counts)])
    got = ops.attention_cached(cache, q, ints(lengths), starts=ints(starts), window=window).double()
    for s, n in enumerate(counts):
        a, L = starts[s], lengths[s]
        kk, vv = (t[stored[s]:stored[s] + L].repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        qq = q[a:a + n].double()
        score = torch.einsum("nhd,khd->nhk", qq, kk) / math.sqrt(dim)
        size = torch.einsum("nhd,khd->nhk", qq.abs(), kk.abs()).amax(-1) / math.sqrt(dim)
        at, key = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")
        seen = (key <= at) & ((at - key < window) | (window == 0))
        p = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), -1)
        want = torch.einsum("nhk,khd->nhd", p, vv)
        tol = bound(host(size), dim, L, host(vv).__abs__().max(), host(want), dtype)
        assert np.all(np.abs(host(got[a:a + n]) - host(want)) <= tol)


@pytest.mark.parametrize("storage,heads,kv_heads,tokens", [("u4", 2, 2, 1), ("u4", 8, 2, 1), ("u4", 8, 2, 5),
                                                           ("bf16", 8, 2, 1), ("f32", 8, 2, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cached_outputs_may_take_the_queries_place(ops, dtype, storage, heads, kv_heads, tokens):
    torch = torch_()
    rng = np.random.default_rng(heads)
    k, v = (tensor(rng.standard_normal((3 * 900, kv_heads, 64)).astype(np.float32)) for _ in range(2))
    cache = ops.KvCache.allocate(3, kv_heads, 900, 64, storage)
    ops.kv_append(cache, k, v, ints([900] * 3), starts=ints([0, 900, 1800, 2700]))
    q = tensor(rng.standard_normal((3 * tokens, heads, 64)).astype(np.float32), dtype)
    lengths, starts = ints([900, 17, 300]), ints(np.arange(4) * tokens) if tokens > 1 else None
    want = ops.attention_cached(cache, q, lengths, starts=starts)
    assert ops.attention_cached(cache, q, lengths, starts=starts, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_packed_outputs_stay_out_of_what_is_read(ops, dtype):
    """Rows may be computed twice, from queries that have to be there still."""
    from basalt_b200 import IllegalArgumentException

    torch = torch_()
    rng = np.random.default_rng(4)
    wide = tensor(rng.standard_normal((200, 8, 64)).astype(np.float32), dtype)
    q, k, v, out = (wide[:, a:b] for a, b in ((0, 2), (2, 4), (4, 6), (6, 8)))
    v[100, 1, 3] = math.inf
    starts = ints([0, 200])
    want = ops.attention_packed(q, k, v, starts, window=50)
    assert torch.isfinite(want[:100]).all() and not torch.isfinite(want[100:150, 1, 3]).any()
    for bad in (q, k, v, wide[:, 1:3]):
        before = wide.clone()
        with pytest.raises(IllegalArgumentException, match="overlap"):
            ops.attention_packed(q, k, v, starts, window=50, out=bad)
        assert torch.equal(wide.nan_to_num(), before.nan_to_num())
    ops.attention_packed(q, k, v, starts, window=50, out=out)
    assert torch.equal(out, want)


def test_counts_beyond_32_bits_keep_their_meaning(ops):
    torch = torch_()
    rng = np.random.default_rng(9)
    q, k, v = prompt(rng, 40, 2, 2, 64, "f32")
    starts = ints([0, 40])
    whole = ops.attention_packed(q, k, v, starts)
    assert torch.equal(ops.attention_packed(q, k, v, starts, window=2 ** 32 + 5), whole)
    cache = ops.KvCache.allocate(1, 2, 40, 64)
    ops.kv_append(cache, k, v, ints([40]), starts=starts)
    whole = ops.attention_cached(cache, q[39:], ints([40]))
    assert torch.equal(ops.attention_cached(cache, q[39:], ints([40]), window=2 ** 32 + 5), whole)
    logits = tensor(rng.standard_normal((50, 300)).astype(np.float32))
    u = tensor(rng.random(50))
    assert torch.equal(ops.sample_tokens(logits, u, top_k=2 ** 32 + 1), ops.sample_tokens(logits, u))


@pytest.mark.parametrize("where", ["hidden", "light", "early"])
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 20, 2.0 ** 40, 2.0 ** 60])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(2, 2, 4), (6, 2, 1), (8, 2, 4), (16, 2, 3), (2, 2, 1),
                                                   (24, 2, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_values_without_weight_leave_the_others_theirs(ops, dtype, heads, kv_heads, tokens, ratio,
                                                             where):
    """Values far above the others at a key that only the last token sees, at one whose score is far
    below the others', or in a first block of keys of which that holds. The bound counts every value
    by its weight: v below is the sum of weight |v|, to which the products of weight and step add
    n 2^-24 of it (they are held to 2^-39 of a power of two that is at most 2^13 times the largest of
    them, and multiply codes of up to 15)."""
    rng = np.random.default_rng(heads + tokens)
    L, dim = 150, 64
    k = rng.standard_normal((L, kv_heads, dim)).astype(np.float32)
    v = rng.standard_normal((L, kv_heads, dim)).astype(np.float32)
    q = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    keys = {"hidden": [L - 1], "light": [0, 50, 120], "early": list(range(16))}[where]
    v[keys] *= np.float32(ratio)
    if where != "hidden":
        q[..., 0], k[:, :, 0] = 12.0, 0.0
        k[keys, :, 0] = -45.0 * math.log2(ratio) / 40       # weights of about 2^-1.3 / ratio^2.4
    cache, starts = ops.KvCache.allocate(1, kv_heads, L + 10, dim), ints([0, L])
    ops.kv_append(cache, tensor(k), tensor(v), ints([L]), starts=starts)
    k, v = (host(t) for t in ops.kv_read(cache, ints([L]), starts=starts, tokens=L))
    q = tensor(q, dtype)
    got = host(ops.attention_cached(cache, q, ints([L]),
                                    starts=ints([0, tokens]) if tokens > 1 else None))
    qh = host(q)
    want, size, _ = attend(qh, k, v, L - tokens)
    for i in range(tokens):
        n = L - tokens + i + 1
        for h in range(heads):
            kk, vv = (x[:n, h * kv_heads // heads] for x in (k, v))
            s = kk @ qh[i, h] / 8
            p = np.exp(s - s.max())
            weighed = (p / p.sum()) @ np.abs(vv).max(1)
            if where == "hidden" and i < tokens - 1:
                assert weighed < 4
            # the scores that matter decide their error
            most = (np.abs(kk) @ np.abs(qh[i, h]) / 8)[p > 1e-3].max()
            tol = bound(np.array([most]), dim, n, weighed, want[i, h], dtype) + n * 2.0 ** -24 * weighed
            assert np.all(np.abs(got[i, h] - want[i, h]) <= tol), (i, h, np.abs(got[i, h] - want[i, h]).max(),
                                                                   tol.min())


def test_a_cache_keeps_few_sizes(ops):
    torch = torch_()
    cache = ops.KvCache.allocate(1, 1, 2000, 32)
    q = torch.zeros((1, 1, 32), device="cuda")
    for window in range(1, 1001):
        ops.attention_cached(cache, q, ints([0]), window=window)
    assert len(cache._sizes) <= 256


@pytest.mark.parametrize("form", ["object", "pointer"])
def test_streams_are_given_as_objects_or_pointers(ops, form):
    """Every call on a stream that waits for nothing of the current one but what it needs."""
    from basalt_b200 import IllegalArgumentException

    torch = torch_()
    rng = np.random.default_rng(6)
    x = prompt(rng, 70, 2, 2, 64, "f32")
    starts, n, one = ints([0, 70]), ints([70]), x[0][69:]
    logits, u = tensor(rng.standard_normal((5, 100)).astype(np.float32)), tensor(rng.random(5))

    def calls(**on):
        cache = ops.KvCache.allocate(1, 2, 70, 64)
        torch.cuda.synchronize()
        ops.kv_append(cache, x[1], x[2], n, starts=starts, **on)
        return (*ops.kv_read(cache, n, starts=starts, tokens=70, **on),
                ops.attention_cached(cache, one, n, **on), ops.attention_packed(*x, starts, **on),
                ops.sample_tokens(logits, u, **on))

    stream = torch.cuda.Stream()
    want = calls()
    got = calls(stream=stream if form == "object" else stream.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    class Elsewhere:
        device, cuda_stream = torch.device("cuda", 7), stream.cuda_stream

    with pytest.raises(IllegalArgumentException, match="stream is on cuda:7"):
        calls(stream=Elsewhere())


@pytest.mark.parametrize("which,value", [(0, math.inf), (0, -math.inf), (1, math.inf), (1, -math.inf),
                                         (0, -3.4025e38), (1, 3.4028e38), (0, math.nan), (1, math.nan)])
@pytest.mark.parametrize("group,dim,window", [(1, 64, 0), (3, 32, 0), (20, 128, 60)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_infinities_of_a_cache_count_as_the_formula_has_them(ops, storage, dtype, group, dim, window,
                                                             which, value):
    """Seen by the first two sequences (one of them split over its keys), not by the others. The finite
    ones are floats that bf16 terms round to infinity."""
    rng = np.random.default_rng(dim + which)
    S, slots, kv_heads = 4, 3000, 2
    lengths = [3000, 1500, 1400, 0]
    x = rng.standard_normal((2, S, slots, kv_heads, dim)).astype(np.float32)
    place = 1480 if window else 1400
    if window:
        lengths[0] = 1500
    x[which, :, place, 1, 3] = value
    cache, starts = ops.KvCache.allocate(S, kv_heads, slots, dim, storage), ints(np.arange(S + 1) * slots)
    ops.kv_append(cache, *(tensor(t.reshape(-1, kv_heads, dim)) for t in x), ints([slots] * S), starts=starts)
    q = rng.standard_normal((S, kv_heads * group, dim)).astype(np.float32)
    q[..., 3] = 0.5 + 0.1 * np.abs(q[..., 3])
    q = tensor(q, dtype)
    got = host(ops.attention_cached(cache, q, ints(lengths), window=window, sinks=2))
    kv = [host(t).reshape(S, slots, kv_heads, dim) for t in (cache.k.transpose(1, 2), cache.v.transpose(1, 2))]
    for s, n in enumerate(lengths):
        if n == 0:
            assert (got[s] == 0).all()
            continue
        k, v = (t[s, :n] for t in kv)
        qs = host(q)[s:s + 1]
        want, size, most = attend(qs, k, v, n - 1, window, 2)
        size = attend(qs, np.where(np.abs(k) < 1e38, k, 0), v, n - 1, window, 2)[1]
        check(got[s:s + 1], want, size, most, dim, n, dtype)
        if s == 2:
            assert np.isfinite(got[s]).all()


@pytest.mark.parametrize("group,kv_heads,counts", [(5, 1, [40, 3, 1, 290]), (12, 2, [65, 130]),
                                                   (300, 1, [5, 1, 3]), (70, 2, [9, 4])])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_heads_to_a_key_head(ops, dtype, dim, group, kv_heads, counts):
    """Groups that are no powers of two, and tokens whose heads span several tiles of rows: in prompts,
    and as several new tokens over a 4-bit cache."""
    rng = np.random.default_rng(group + dim)
    starts = np.concatenate([[0], np.cumsum(counts)])
    q, k, v = prompt(rng, starts[-1], group * kv_heads, kv_heads, dim, dtype)
    got = host(ops.attention_packed(q, k, v, ints(starts), window=29, sinks=2, scale=0.2))
    for a, b in zip(starts, starts[1:]):
        want, size, most = attend(*[host(t)[a:b] for t in (q, k, v)], 0, 29, 2, 0.2)
        check(got[a:b], want, size, np.full_like(most, most.max()), dim, b - a, dtype)
    S, slots = len(counts), 400
    cache = ops.KvCache.allocate(S, kv_heads, slots, dim)
    ops.kv_append(cache, k, v, ints(counts), starts=ints(starts))
    k, v = (host(t) for t in ops.kv_read(cache, ints(counts), starts=ints(starts), tokens=int(starts[-1])))
    got = host(ops.attention_cached(cache, q, ints(counts), starts=ints(starts), window=29, sinks=2,
                                    scale=0.2))
    for a, b in zip(starts, starts[1:]):
        want, size, most = attend(host(q)[a:b], k[a:b], v[a:b], 0, 29, 2, 0.2)
        check(got[a:b], want, size, np.full_like(most, most.max()), dim, b - a, dtype)


@pytest.mark.parametrize("which,value,again", [(0, math.nan, 0), (1, math.nan, 0), (2, math.nan, 1), (1, -math.inf, 4),
                                               (2, math.inf, 4)])
def test_only_infinities_have_rows_computed_again(ops, which, value, again):
    """The workspace holds a flag for each of the four CTAs of 64 rows: a NaN leaves what it should, but
    for a value in a tile that some of a CTA's rows do not see."""
    torch = torch_()
    x = prompt(np.random.default_rng(8), 200, 1, 1, 64, "f32")
    x[which][0, 0, 3] = value
    size = torch.full((4,), 7, dtype=torch.int32, device="cuda")
    ops.attention_packed(*x, ints([0, 200]), workspace=size)
    assert size.tolist().count(1) == again and size.tolist().count(0) == 4 - again
