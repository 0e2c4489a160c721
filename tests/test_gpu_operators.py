"""The serving operators on the GPU against plain 64-bit implementations.

Tolerances. A value read from a 4-bit cache is low + code * step rounded once to float32 (and once
more to bf16). Attention in float32: a score of d products has an error of at most
(d + 8) 2^-23 sum|q k| scale (float32 sums and products split in parts good to 2^-22), the weights'
relative error is twice that plus the exponential's 2^-21, and a sum over n weights adds n 2^-24 on
either side of the quotient, so an output is off by at most max|v| times their sum. bf16 adds the
weights' own rounding to bf16 (2^-8 of max|v|) and the output's (2^-8 of it).
"""
import math

import numpy as np
import pytest

import operator_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(runtime):
    from basalt_b200 import operators

    return operators


def torch_():
    import torch

    return torch


def tensor(x, dtype=None):
    torch = torch_()
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(getattr(torch, {"f32": "float32", "bf16": "bfloat16"}[dtype]))


def ints(x):
    return tensor(np.asarray(x, np.int32))


def host(t):
    return t.detach().to(torch_().float64).cpu().numpy()


def rounded(x, dtype):
    x = np.asarray(x, np.float32)
    return ref.bf16_bits(x) if dtype == "bf16" else x


def bound(size, d, n, vmax, out, dtype):
    s = (d + 8) * 2.0 ** -23 * size[..., None]
    tol = vmax * (2.2 * s + 2.0 ** -21 + (n + 16) * 2.0 ** -23)
    if dtype == "bf16":
        tol = tol + 2.0 ** -8 * vmax + 2.0 ** -8 * np.abs(out)
    return tol


# ---- the cache -------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,heads", [(32, 1), (64, 3), (128, 2)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("storage", ["u4", "bf16", "f32"])
def test_store_and_read(ops, dim, heads, dtype, storage):
    torch = torch_()
    rng = np.random.default_rng(dim + heads)
    counts, lengths, rows = [5, 0, 1, 9], [7, 3, 1, 20], [2, 0, 4, 1]
    starts = np.concatenate([[0], np.cumsum(counts)])
    T = starts[-1] + 2                                  # two tokens behind the last sequence
    fused = rng.standard_normal((T, 2 * heads * dim + 4)).astype(np.float32) * 3 + 1
    fused[3, :32] = 0.25                                # a group of equal values
    fused[4, :32] = -1e-3 * np.arange(32)
    fused = tensor(fused, dtype)
    k = fused[:, :heads * dim].unflatten(-1, (heads, dim))
    v = fused[:, heads * dim:2 * heads * dim].unflatten(-1, (heads, dim))
    cache = ops.KvCache.allocate(5, heads, 20, dim, storage)
    before = cache.k.clone()
    args = dict(starts=ints(starts), rows=ints(rows))
    ops.kv_append(cache, k, v, ints(lengths), **args)
    got = [torch.full((T, heads, dim), 7.5, dtype=k.dtype, device="cuda") for _ in range(2)]
    ops.kv_read(cache, ints(lengths), out=got, **args)
    touched = np.zeros((5, 20), bool)
    for x, out, codes, scale in ((k, got[0], cache.k, cache.k_scale),
                                 (v, got[1], cache.v, cache.v_scale)):
        x, out = host(x), host(out)
        assert np.all(out[starts[-1]:] == 7.5)
        for s, n in enumerate(counts):
            for i in range(n):
                t, slot = starts[s] + i, lengths[s] - n + i
                touched[rows[s], slot] = True
                if storage == "u4":
                    c, step, low, values = ref.quantise(x[t])
                    assert np.array_equal(codes[rows[s], :, slot].cpu().numpy(), c)
                    assert np.array_equal(host(scale[rows[s], :, slot]), np.stack([step, low], -1))
                    want = rounded(values.astype(np.float32), dtype)
                else:
                    want = rounded(rounded(x[t], storage), dtype)
                assert np.array_equal(out[t], want.astype(np.float64)), (s, i)
    changed = (cache.k != before).flatten(3).any(-1).any(1).cpu().numpy()
    assert not (changed & ~touched).any()


def test_borders_of_codes_round_as_the_double_quotient(ops):
    """Values on and next to the middle between two codes."""
    rng = np.random.default_rng(5)
    x = np.zeros((64, 1, 32), np.float32)
    for t in range(64):
        low, step = np.float32(rng.integers(-8, 8)) / 4, np.float32(2.0 ** rng.integers(-6, 3))
        x[t, 0] = low + step * (rng.integers(0, 15, 32) + 0.5).astype(np.float32)
        x[t, 0, 0], x[t, 0, 1] = low, low + 15 * step
        x[t, 0, 8:16] = np.nextafter(x[t, 0, 8:16], np.float32(100))
        x[t, 0, 16:24] = np.nextafter(x[t, 0, 16:24], np.float32(-100))
    cache = ops.KvCache.allocate(64, 1, 1, 32)
    ones = ints(np.ones(64))
    ops.kv_append(cache, tensor(x), tensor(x), ones)
    codes, _, _, values = ref.quantise(x)
    assert np.array_equal(cache.k[:, :, 0].cpu().numpy(), codes)
    assert np.array_equal(host(ops.kv_read(cache, ones)[0]), values.astype(np.float32))


def test_extreme_values_and_places_outside_the_cache(ops):
    torch = torch_()
    x = np.ones((6, 1, 64), np.float32)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 0] = np.nan, np.inf, -np.inf
    x[3, 0, :32] = np.linspace(-3e38, 3e38, 32)
    x[4, 0, :32] = np.linspace(1e-39, 3e-39, 32)
    cache = ops.KvCache.allocate(6, 1, 4, 64)
    lengths, rows = ints([1, 4, 2, 3, 1, 5]), ints([0, 1, 2, 3, 4, 5])   # the last: slot 4 of 4
    ops.kv_append(cache, tensor(x), tensor(x), lengths, rows=rows)
    k = host(ops.kv_read(cache, lengths, rows=rows)[0])
    assert np.isnan(k[0, 0, :32]).all() and (k[0, 0, 32:] == 1).all()
    assert (k[1, 0, :32] == 1).all() and np.isnan(k[1, 0, 32:]).all()
    assert np.isnan(k[2, 0, :32]).all()
    step = 6e38 / 15 * (1 + 2.0 ** -7)
    assert np.abs(k[3, 0, :32] - x[3, 0, :32]).max() <= step / 2 * (1 + 2.0 ** -6)
    assert np.isfinite(k[4]).all() and np.abs(k[4, 0, :32] - x[4, 0, :32]).max() < 2e-40
    assert (k[5] == 0).all()                                              # read as zeros
    ops.kv_append(cache, tensor(x), tensor(x), ints([0] * 6), rows=ints([-1, 9, 0, 0, 0, 0]))
    assert np.array_equal(host(ops.kv_read(cache, lengths, rows=rows)[0])[3:], k[3:])


# ---- attention over a cache ------------------------------------------------------------------
def filled_cache(ops, rng, rows, heads, slots, dim, storage):
    """A cache with every slot stored, and the float64 values it stands for."""
    x = [(rng.standard_normal((rows * slots, heads, dim)) + rng.standard_normal((heads, dim)))
         .astype(np.float32) for _ in range(2)]
    cache = ops.KvCache.allocate(rows, heads, slots, dim, storage)
    starts = ints(np.arange(rows + 1) * slots)
    ops.kv_append(cache, tensor(x[0]), tensor(x[1]), ints([slots] * rows), starts=starts)
    values = ops.kv_read(cache, ints([slots] * rows), starts=starts, tokens=rows * slots)
    return cache, [host(t).reshape(rows, slots, heads, dim) for t in values]


CACHED = [
    # heads, kv_heads, dim, lengths, window, sinks
    (1, 1, 32, [1, 2, 31, 33], 0, 0),
    (8, 8, 64, [1, 63, 64, 65, 200, 0], 0, 0),
    (8, 2, 128, [129, 5, 257], 0, 0),
    (16, 1, 64, [300, 17], 0, 0),
    (24, 2, 32, [90, 1], 0, 0),
    (6, 3, 64, [400, 100, 37], 32, 4),
    (4, 4, 128, [513, 130, 8], 100, 0),
    (8, 2, 64, [700, 3], 1, 1),
    (4, 2, 64, [1000], 64, 200),
    (4, 2, 64, [250, 249], 5000, 3),
]


@pytest.mark.parametrize("heads,kv_heads,dim,lengths,window,sinks", CACHED)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("storage", ["u4", "f32", "bf16"])
def test_one_token_over_a_cache(ops, storage, dtype, heads, kv_heads, dim, lengths, window, sinks):
    rng = np.random.default_rng(sum(lengths) + dim)
    slots, S = max(lengths) + 3, len(lengths)
    cache, (k, v) = filled_cache(ops, rng, S, kv_heads, slots, dim, storage)
    rows = rng.permutation(S)
    wide = tensor(rng.standard_normal((S, heads * dim + 8)).astype(np.float32), dtype)
    q = wide[:, :heads * dim].unflatten(-1, (heads, dim))
    got = host(ops.attention_cached(cache, q, ints(lengths), rows=ints(rows), window=window,
                                    sinks=sinks))
    check_cached(q, got, k, v, rows, lengths, [1] * S, window, sinks, dtype)


def check_cached(q, got, k, v, rows, lengths, counts, window, sinks, dtype, scale=None):
    qh, at, d = host(q), 0, q.shape[2]
    for s, n in enumerate(counts):
        L = lengths[s]
        want, size = ref.attend(qh[at:at + n], k[rows[s], :max(L, 0)], v[rows[s], :max(L, 0)], L - n,
                                window, sinks, scale or 1 / math.sqrt(d))
        vmax = np.abs(v[rows[s], :max(L, 1)]).max()
        tol = bound(size, d, L, vmax, want, dtype)
        diff = np.abs(got[at:at + n] - want)
        assert np.all(diff <= tol), (s, float(diff.max()), float(tol.min()))
        at += n


@pytest.mark.parametrize("heads,kv_heads,dim,lengths,counts,window,sinks", [
    (8, 8, 64, [40, 5, 100, 9], [4, 5, 1, 0], 0, 0),
    (8, 2, 128, [300, 70], [7, 33], 0, 0),
    (4, 1, 32, [129, 64, 3], [64, 64, 3], 0, 0),
    (8, 2, 64, [500, 3, 90], [9, 3, 40], 20, 3),
    (12, 4, 64, [200, 2], [5, 4], 3, 0),       # more tokens than the length: they see nothing
    (64, 2, 64, [77, 20], [3, 2], 50, 1),
])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_several_tokens_over_a_4_bit_cache(ops, dtype, heads, kv_heads, dim, lengths, counts, window,
                                           sinks):
    torch = torch_()
    rng = np.random.default_rng(sum(lengths))
    S, T = len(lengths), sum(counts)
    cache, (k, v) = filled_cache(ops, rng, S, kv_heads, max(lengths) + 1, dim, "u4")
    q = tensor(rng.standard_normal((T + 3, heads, dim)).astype(np.float32), dtype)
    out = torch.full_like(q, 3.25)
    starts = np.concatenate([[0], np.cumsum(counts)])
    ops.attention_cached(cache, q, ints(lengths), starts=ints(starts), window=window, sinks=sinks,
                         out=out, scale=0.3)
    got = host(out)
    assert np.all(got[T:] == 3.25)
    check_cached(q, got, k, v, np.arange(S), lengths, counts, window, sinks, dtype, 0.3)


@pytest.mark.parametrize("storage", ["u4", "f32", "bf16"])
def test_what_is_not_visible_takes_no_part(ops, storage):
    """NaN and infinities in slots behind the length, before the window and between it and the
    sinks; rows outside the cache; lengths of zero."""
    torch = torch_()
    rng = np.random.default_rng(3)
    x = rng.standard_normal((3 * 200, 2, 64)).astype(np.float32)
    bad = x.reshape(3, 200, 2, 64).copy()
    bad[:, 150:] = np.nan
    bad[:, 4:100] = np.inf
    bad = bad.reshape(x.shape)
    starts, full = ints([0, 200, 400, 600]), ints([200] * 3)
    q = tensor(rng.standard_normal((3, 8, 64)).astype(np.float32))
    outs = []
    for values in (x, bad):
        cache = ops.KvCache.allocate(3, 2, 200, 64, storage)
        ops.kv_append(cache, tensor(values), tensor(values), full, starts=starts)
        outs.append(ops.attention_cached(cache, q, ints([150, 0, 149]), rows=ints([1, 2, 0]),
                                         window=49, sinks=4))
    # 150 - 49 = 101 is the first key of the window of the first row, 100 that of the last
    assert torch.equal(outs[0], outs[1])
    assert (outs[0][1] == 0).all() and torch.isfinite(outs[0]).all()
    out = ops.attention_cached(cache, q, ints([5, 5, 5]), rows=ints([-1, 3, 77]))
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (66, 0), (66, 3)])
def test_later_values_of_another_size_stay_out_of_earlier_rows(ops, dtype, window, sinks):
    """Steps that grow or shrink from block to block of keys, some of which only a tile's later, or
    only its earlier, tokens see."""
    rng = np.random.default_rng(window + sinks)
    counts, lengths, heads, dim = [24, 24, 5], [70, 134, 33], 2, 64
    x = rng.standard_normal((3 * 140, heads, dim)).astype(np.float32)
    sizes = (2.0 ** rng.integers(-6, 7, (3, 20))).astype(np.float32)
    sizes[0, :9], sizes[0, 9:] = 1, 64                   # the first sequence: from key 63 on
    values = x * np.repeat(sizes, 7, 1).reshape(-1, 1, 1)
    cache = ops.KvCache.allocate(3, heads, 140, dim)
    full, at = ints([140] * 3), ints([0, 140, 280, 420])
    ops.kv_append(cache, tensor(x), tensor(values), full, starts=at)
    k, v = (host(t).reshape(3, 140, heads, dim) for t in ops.kv_read(cache, full, starts=at, tokens=420))
    q = tensor(rng.standard_normal((sum(counts), heads, dim)).astype(np.float32), dtype)
    starts = np.concatenate([[0], np.cumsum(counts)])
    got = host(ops.attention_cached(cache, q, ints(lengths), starts=ints(starts), window=window,
                                    sinks=sinks))
    # The bounds hold for each query by itself: max|v| over the keys that it sees.
    qh = host(q)
    for s, n in enumerate(counts):
        for i in range(n):
            position, t = lengths[s] - n + i, starts[s] + i
            seen = ref.visible(position, lengths[s], window, sinks)
            want, size = ref.attend(qh[t:t + 1], k[s, :lengths[s]], v[s, :lengths[s]], position, window,
                                    sinks, 1 / 8)
            tol = bound(size, dim, lengths[s], np.abs(v[s, :lengths[s]][seen]).max(), want, dtype)
            assert np.all(np.abs(got[t] - want[0]) <= tol[0]), (s, i)


@pytest.mark.parametrize("heads,dim,lengths,window,sinks", [
    (3, 64, [700, 5, 0, 130], 64, 9), (2, 128, [5000], 0, 0), (2, 128, [9000, 40], 3000, 50),
    (5, 32, [3333, 64, 63], 1000, 7), (1, 64, [33], 31, 1), (2, 32, [20000], 0, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 40, 2.0 ** -60])
def test_one_query_a_key_head_over_4_bits(ops, dtype, heads, dim, lengths, window, sinks, size):
    """Every key head with one query, values of different sizes from block to block, and queries and
    values far from one."""
    rng = np.random.default_rng(dim + sum(lengths))
    S, slots = len(lengths), max(lengths) + 5
    k = rng.standard_normal((S * slots, heads, dim)).astype(np.float32)
    v = rng.standard_normal((S * slots, heads, dim)).astype(np.float32)
    v *= (2.0 ** rng.integers(-8, 9, (S * slots, 1, 1)) * size).astype(np.float32)
    cache = ops.KvCache.allocate(S, heads, slots, dim)
    starts, full = ints(np.arange(S + 1) * slots), ints([slots] * S)
    ops.kv_append(cache, tensor(k), tensor(v), full, starts=starts)
    k, v = (host(t).reshape(S, slots, heads, dim)
            for t in ops.kv_read(cache, full, starts=starts, tokens=S * slots))
    q = tensor((rng.standard_normal((S, heads, dim)) / size).astype(np.float32), dtype)
    scale = size / math.sqrt(dim)
    got = host(ops.attention_cached(cache, q, ints(lengths), window=window, sinks=sinks, scale=scale))
    check_cached(q, got, k, v, np.arange(S), lengths, [1] * S, window, sinks, dtype, scale)


def test_one_query_a_key_head_and_values_that_are_not_finite(ops):
    """Unseen ones take no part; a seen one reaches the 32 channels that it shares a scale with."""
    torch = torch_()
    rng = np.random.default_rng(14)
    for dim in (32, 64, 128):
        x = rng.standard_normal((2 * 300, 2, dim)).astype(np.float32)
        bad = x.reshape(2, 300, 2, dim).copy()
        bad[:, 250:], bad[:, 3:150] = np.nan, -np.inf
        starts, full, lengths = ints([0, 300, 600]), ints([300] * 2), ints([250, 249])
        q = tensor(rng.standard_normal((2, 2, dim)).astype(np.float32))
        outs = []
        for values in (x, bad.reshape(x.shape)):
            cache = ops.KvCache.allocate(2, 2, 300, dim)
            ops.kv_append(cache, tensor(values), tensor(values), full, starts=starts)
            outs.append(ops.attention_cached(cache, q, lengths, window=99, sinks=3))
        assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()
        values = x.copy()
        values[200, 1, 5] = np.nan
        cache = ops.KvCache.allocate(2, 2, 300, dim)
        ops.kv_append(cache, tensor(x), tensor(values), full, starts=starts)
        out = ops.attention_cached(cache, q, lengths)
        assert torch.isnan(out[0, 1, :32]).all()
        assert torch.isfinite(out[0, 1, 32:]).all() and torch.isfinite(out[0, 0]).all()
        assert torch.isfinite(out[1]).all()


def test_a_long_4_bit_cache(ops):
    """Work split over the keys: one sequence of 40 000 keys, and offsets past 2^31 bytes."""
    torch = torch_()
    rng = np.random.default_rng(11)
    cache, (k, v) = filled_cache(ops, rng, 1, 2, 40000, 128, "u4")
    q = tensor(rng.standard_normal((1, 8, 128)).astype(np.float32), "bf16")
    got = host(ops.attention_cached(cache, q, ints([40000])))
    check_cached(q, got, k, v, [0], [40000], [1], 0, 0, "bf16")
    wide = ops.KvCache.allocate(3, 1, 17_000_000, 128)
    assert wide.k.numel() > 2 ** 31
    n = 300
    x = tensor(rng.standard_normal((n, 1, 128)).astype(np.float32))
    length, row, start = ints([17_000_000]), ints([2]), ints([0, n])
    ops.kv_append(wide, x, x, length, starts=start, rows=row)
    values = host(ops.kv_read(wide, length, starts=start, rows=row, tokens=n)[0])
    q = tensor(rng.standard_normal((1, 4, 128)).astype(np.float32))
    got = host(ops.attention_cached(wide, q, length, rows=row, window=n))
    check_cached(q, got, values[None], values[None], [0], [n], [1], 0, 0, "f32")
    del wide
    torch.cuda.empty_cache()


# ---- attention over packed sequences ---------------------------------------------------------
PACKED = [
    (1, 1, 32, [1, 2, 3], 0, 0),
    (4, 4, 64, [1, 64, 65, 0, 127], 0, 0),
    (8, 2, 128, [130, 257, 1], 0, 0),
    (6, 3, 64, [300, 5], 37, 4),
    (4, 1, 128, [500, 129], 128, 1),
    (2, 2, 32, [200], 1, 0),
    (2, 1, 64, [700], 64, 130),
    (8, 4, 128, [1025], 300, 4),
]


@pytest.mark.parametrize("heads,kv_heads,dim,lengths,window,sinks", PACKED)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_packed_prompts(ops, dtype, heads, kv_heads, dim, lengths, window, sinks):
    torch = torch_()
    rng = np.random.default_rng(sum(lengths) + heads)
    starts, T = np.concatenate([[0], np.cumsum(lengths)]), sum(lengths)
    fused = tensor(rng.standard_normal((T + 2, (heads + 2 * kv_heads) * dim)).astype(np.float32), dtype)
    q, k, v = (x.unflatten(-1, (-1, dim)) for x in
               fused.split([heads * dim, kv_heads * dim, kv_heads * dim], -1))
    out = torch.full((T + 2, heads, dim), 1.5, dtype=q.dtype, device="cuda")
    ops.attention_packed(q, k, v, ints(starts), window=window, sinks=sinks, out=out)
    got, qh, kh, vh = host(out), host(q), host(k), host(v)
    assert np.all(got[T:] == 1.5)
    for s, n in enumerate(lengths):
        a, b = starts[s], starts[s + 1]
        if n == 0:
            continue
        want, size = ref.attend(qh[a:b], kh[a:b], vh[a:b], 0, window, sinks, 1 / math.sqrt(dim))
        tol = bound(size, dim, n, np.abs(vh[a:b]).max(), want, dtype)
        diff = np.abs(got[a:b] - want)
        assert np.all(diff <= tol), (s, float(diff.max()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_packed_tensors_of_any_alignment(ops, dtype, dim):
    rng = np.random.default_rng(dim)
    starts = [0, 150, 150, 201]
    wide = tensor(rng.standard_normal((201, 6 * dim + 3)).astype(np.float32), dtype)
    q, k, v = (wide[:, 1 + a * dim:1 + b * dim].unflatten(-1, (-1, dim)) for a, b in
               ((0, 4), (4, 5), (5, 6)))
    got = host(ops.attention_packed(q, k, v, ints(starts), window=70, sinks=3, scale=-0.2))
    qh, kh, vh = host(q), host(k), host(v)
    for a, b in ((0, 150), (150, 201)):
        want, size = ref.attend(qh[a:b], kh[a:b], vh[a:b], 0, 70, 3, -0.2)
        tol = bound(size, dim, b - a, np.abs(vh[a:b]).max(), want, dtype)
        assert np.all(np.abs(got[a:b] - want) <= tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_packed_values_that_are_not_finite_reach_only_those_that_see_them(ops, dtype, dim, value):
    rng = np.random.default_rng(2)
    T = 300
    x = [tensor(rng.standard_normal((T, 2, dim)).astype(np.float32), dtype) for _ in range(3)]
    clean = host(ops.attention_packed(*x, ints([0, 100, T]), window=50, sinks=2))
    x[1][180, 1], x[2][180, 1] = value, value       # position 80 of the second sequence
    got = host(ops.attention_packed(*x, ints([0, 100, T]), window=50, sinks=2))
    sees = (np.arange(T) >= 180) & (np.arange(T) < 230)
    assert np.array_equal(got[:, 0], clean[:, 0])
    tol = 2.0 ** -7 * np.abs(clean).max()            # the same numbers, in whatever order
    assert np.abs(got[~sees, 1] - clean[~sees, 1]).max() <= tol
    assert not np.isfinite(got[sees, 1]).any()


# ---- drawing tokens --------------------------------------------------------------------------
def check_draws(ops, x, u, dtype="f32", **p):
    rows, V = x.shape
    t = tensor(np.asarray(x, np.float32), dtype)
    given = {k: (v if np.isscalar(v) else tensor(np.asarray(v, np.int32 if k == "top_k" else np.float32)))
             for k, v in p.items()}
    got = ops.sample_tokens(t, tensor(np.asarray(u, np.float64)), **given).cpu().numpy()
    xs = host(t)
    for r in range(rows):
        one = {k: (np.float32(v) if k != "top_k" else v) if np.isscalar(v)
               else np.asarray(v, np.float32)[r] for k, v in
               {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **p}.items()}
        one["top_k"] = int(one["top_k"])
        want, margin = ref.draw_token(xs[r], u[r], **one)
        # weights are whole units of 2^-42: a running sum is off by at most V / 2 of them
        assert got[r] == want or margin <= V * 2.0 ** -42, (r, got[r], want, margin, one)
    return got


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4096, 8191, 20000, 131072, 300001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_draws_follow_the_reference(ops, V, dtype):
    rng = np.random.default_rng(V)
    rows = 24
    x = rng.standard_normal((rows, V)) * 3
    check_draws(ops, x, rng.random(rows), dtype)
    check_draws(ops, x, rng.random(rows), dtype, temperature=0.7, top_k=40, top_p=0.9)
    check_draws(ops, x, rng.random(rows), dtype, top_p=0.6, min_p=0.05)
    check_draws(ops, x, rng.random(rows), dtype, temperature=rng.choice([0.0, 0.5, 1.0, 2.0, 50.0], rows),
                top_k=rng.choice([0, 1, 2, 50, V, 5 * V], rows),
                top_p=rng.choice([0.0, 0.3, 0.95, 1.0, 2.0], rows),
                min_p=rng.choice([0.0, 0.01, 0.5, 1.0, 3.0], rows))


def test_draws_with_ties(ops):
    rng = np.random.default_rng(1)
    x = np.round(rng.standard_normal((40, 500)) * 2)           # few distinct logits
    for p in ({}, {"top_k": 17}, {"top_k": 100, "top_p": 0.5}, {"top_p": 0.5}, {"min_p": 0.3},
              {"top_k": 3, "min_p": 1.0}):
        check_draws(ops, x, rng.random(40), **p)
    flat = np.full((16, 64), 2.5)
    got = check_draws(ops, flat, (np.arange(16) + 0.5) / 16, top_k=16)
    assert np.array_equal(got, np.arange(16))                  # ties are kept lowest index first
    check_draws(ops, flat, np.arange(16) / 16.0, top_p=0.25)
    flat[:, 5], flat[:, 6] = 0.0, -0.0                         # the same logit
    check_draws(ops, flat * 0, rng.random(16), top_k=7)


@pytest.mark.parametrize("V", [3000, 8191, 20000, 131072])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_draws_from_many_candidates(ops, V, dtype):
    """top_k around what the lists and the CTAs' threads hold, and ties that overflow them."""
    rng = np.random.default_rng(V + 1)
    rows = 10
    top_k = [255, 257, 400, 512, 513, 700, 1000, 1024, 1025, 2500]
    x = rng.standard_normal((rows, V)) * 2
    check_draws(ops, x, rng.random(rows), dtype, top_k=top_k)
    check_draws(ops, x, rng.random(rows), dtype, top_k=top_k, top_p=0.9, min_p=0.003)
    check_draws(ops, np.sort(x, 1)[:, ::-1], rng.random(rows), dtype, top_k=top_k, top_p=0.99)
    few = np.round(x)                                          # thousands of tokens a value
    check_draws(ops, few, rng.random(rows), dtype, top_k=top_k, top_p=0.97)
    check_draws(ops, few, rng.random(rows), dtype, top_k=20, top_p=0.5, min_p=0.2)


def test_draws_at_the_edges(ops):
    inf, nan = np.inf, np.nan
    x = np.full((8, 70), -inf)
    x[1, 69] = 3.0
    x[2, :3] = [nan, 1.0, nan]
    x[3, [4, 9]] = inf
    x[4] = nan
    x[5] = -3e38
    x[6, 10:20] = np.linspace(-1e-30, 1e-30, 10)
    x[7] = np.linspace(0, 69, 70)
    for u in (0.0, 0.5, 1 - 2.0 ** -53, 1.0, -1.0, 7.0):
        got = check_draws(ops, x, [u] * 8)
        assert list(got[:3]) == [-1, 69, 1] and got[4] == -1 and got[3] in (4, 9)
        check_draws(ops, x, [u] * 8, temperature=1e-30)
        check_draws(ops, x, [u] * 8, temperature=np.float32(np.inf))
        check_draws(ops, x, [u] * 8, temperature=0.0)
        check_draws(ops, x, [u] * 8, temperature=2.5, top_k=5, top_p=0.99, min_p=1e-9)
    # an edge of the weights next to zero, where floats are dense
    y = np.concatenate([[40 * math.log(2)], np.geomspace(1e-38, 1e-3, 60), -np.geomspace(1e-38, 1e-3, 60)])
    check_draws(ops, np.stack([y] * 4), [0.0, 1e-13, 0.5, 1 - 2.0 ** -53])
    check_draws(ops, np.stack([y] * 4), [0.0, 1e-13, 0.5, 1 - 2.0 ** -53], min_p=2.0 ** -40)


def test_draws_from_rows_of_a_wider_tensor(ops):
    torch = torch_()
    rng = np.random.default_rng(9)
    wide = tensor(rng.standard_normal((6, 1003)).astype(np.float32))
    u = tensor(rng.random(6))
    out = torch.full((6,), -7, dtype=torch.int32, device="cuda")
    ops.sample_tokens(wide[:, 1:1000], u, top_k=30, out=out)
    want = [ref.draw_token(host(wide)[r, 1:1000], host(u)[r], 1.0, 30, 1.0, 0.0)[0] for r in range(6)]
    assert out.tolist() == want


# ---- together --------------------------------------------------------------------------------
def test_a_prompt_and_decode_steps_together(ops):
    """Prompts through windowed attention, their keys and values into a 4-bit cache, then steps of
    append, attention, a head and a draw: every step against 64 bits on the same cache."""
    torch = torch_()
    rng = np.random.default_rng(21)
    H, KV, d, V, window, sinks = 4, 2, 64, 600, 24, 2
    prompts = [30, 1, 77]
    S, T, slots = 3, sum(prompts), 100
    starts = np.concatenate([[0], np.cumsum(prompts)])
    qkv = [tensor(rng.standard_normal((T, n, d)).astype(np.float32)) for n in (H, KV, KV)]
    cache = ops.KvCache.allocate(S, KV, slots, d)
    lengths = ints(prompts)
    ops.kv_append(cache, qkv[1], qkv[2], lengths, starts=ints(starts))
    kept = ops.kv_read(cache, lengths, starts=ints(starts), tokens=T)
    a = host(ops.attention_packed(qkv[0], *kept, ints(starts), window=window, sinks=sinks))
    b = host(ops.attention_cached(cache, qkv[0], lengths, starts=ints(starts), window=window, sinks=sinks))
    seen = [host(x) for x in kept]
    for s in range(S):
        i, j = starts[s], starts[s + 1]
        want, size = ref.attend(host(qkv[0])[i:j], seen[0][i:j], seen[1][i:j], 0, window, sinks, 1 / 8)
        tol = bound(size, d, prompts[s], np.abs(seen[1]).max(), want, "f32")
        assert np.all(np.abs(a[i:j] - want) <= tol) and np.all(np.abs(b[i:j] - want) <= tol)
    head = tensor((rng.standard_normal((H * d, V)) * 0.3).astype(np.float32))
    history = [[list(seen[x][starts[s]:starts[s + 1]]) for s in range(S)] for x in range(2)]
    for step in range(6):
        lengths += 1
        q, k, v = (tensor(rng.standard_normal((S, n, d)).astype(np.float32)) for n in (H, KV, KV))
        ops.kv_append(cache, k, v, lengths)
        out = ops.attention_cached(cache, q, lengths, window=window, sinks=sinks)
        now = [host(x) for x in ops.kv_read(cache, lengths)]
        for s in range(S):
            for x in range(2):
                history[x][s].append(now[x][s])
            K, W = np.stack(history[0][s]), np.stack(history[1][s])
            want, size = ref.attend(host(q)[s:s + 1], K, W, len(K) - 1, window, sinks, 1 / 8)
            assert np.all(np.abs(host(out)[s:s + 1] - want) <= bound(size, d, len(K), np.abs(W).max(), want, "f32"))
        logits = out.flatten(1) @ head
        check_draws(ops, logits.cpu().numpy(), rng.random(S), temperature=0.9, top_k=50, top_p=0.9, min_p=0.01)


def test_captured_steps_and_other_streams(ops):
    """A step captured into a graph and replayed on new inputs, on a side stream, gives what eager
    calls give; two streams at once give what each gives alone."""
    torch = torch_()
    rng = np.random.default_rng(4)
    S, H, KV, d, slots, V = 5, 8, 2, 64, 300, 1000
    cache, _ = filled_cache(ops, rng, S, KV, slots, d, "u4")
    q, k, v = (tensor(rng.standard_normal((S, n, d)).astype(np.float32)) for n in (H, KV, KV))
    lengths, u = ints([300, 4, 150, 77, 1]), tensor(rng.random(S))
    head = tensor(rng.standard_normal((H * d, V)).astype(np.float32))

    def step():
        ops.kv_append(cache, k, v, lengths)
        out = ops.attention_cached(cache, q, lengths)
        return out, ops.sample_tokens(out.flatten(1) @ head, u, top_k=100, top_p=0.8)

    step()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.synchronize()
    for change in range(3):
        q.copy_(tensor(rng.standard_normal((S, H, d)).astype(np.float32)))
        lengths.copy_(ints(rng.integers(1, slots, S)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        want = step()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = [ops.attention_cached(cache, q, lengths, window=w) for w in (0, 40)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = [[], []]
    for i in range(20):
        for w, (s, out) in enumerate(zip(streams, both)):
            with torch.cuda.stream(s):
                out.append(ops.attention_cached(cache, q, lengths, window=(0, 40)[w]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, one[w]) for w in range(2) for o in both[w])


def test_captured_prompts_and_draws(ops):
    """Packed attention and draws with per-row settings, captured together, on changed inputs."""
    torch = torch_()
    rng = np.random.default_rng(8)
    T, H, KV, d, V = 200, 4, 2, 64, 3000
    calls = []
    for dtype in ("f32", "bf16"):
        q, k, v = (tensor(rng.standard_normal((T, n, d)).astype(np.float32), dtype) for n in (H, KV, KV))
        starts, u = ints([0, 150, 150, 190]), tensor(rng.random(12))
        x = tensor(rng.standard_normal((12, V)).astype(np.float32), dtype)
        warm = tensor(rng.random(12).astype(np.float32) + 0.5)
        few, most, least = ints(rng.integers(0, 60, 12)), warm - 0.4, warm * 0.01
        calls.append((q, k, v, starts, u, x, warm, few, most, least))

    def step():
        return [(ops.attention_packed(q, k, v, starts, window=40, sinks=2)[:190],
                 ops.sample_tokens(x, u, warm, few, most, least))
                for q, k, v, starts, u, x, warm, few, most, least in calls]

    step()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for change in range(3):
        for q, k, v, starts, u, x, warm, few, most, least in calls:
            for t in (q, k, v, x):
                t.copy_(tensor(rng.standard_normal(t.shape).astype(np.float32)))
            if change == 1:
                v[rng.integers(0, 190), 0, 3] = float("nan")
            u.copy_(tensor(rng.random(12)))
            few.copy_(ints(rng.integers(0, 60, 12)))
            starts.copy_(ints([0, 20 + change, 100, 190]))
        graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in pair] for pair in held]
        for pair, (a, b) in zip(got, step()):
            assert torch.equal(pair[0].nan_to_num(7.0), a.nan_to_num(7.0)) and torch.equal(pair[1], b)


def test_prompts_and_draws_on_two_streams_at_once(ops):
    torch = torch_()
    rng = np.random.default_rng(15)
    T, H, KV, d = 1500, 8, 2, 128
    starts = ints([0, 700, T])
    u, x = tensor(rng.random(300)), tensor(rng.standard_normal((300, 20000)).astype(np.float32))
    sets = [[tensor(rng.standard_normal((T, n, d)).astype(np.float32), dtype) for n in (H, KV, KV)]
            for dtype in ("bf16", "bf16", "f32")]

    def step(i):
        return (ops.attention_packed(*sets[i], starts, window=(0, 300, 100)[i], sinks=2),
                ops.sample_tokens(x, u, top_k=(0, 50, 900)[i], top_p=(0.9, 1.0, 0.8)[i]))

    want = [step(i) for i in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[] for _ in range(3)]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(3) for g in got[i] for a, b in zip(g, want[i]))


def test_memory_belongs_to_the_given_stream(ops):
    """What a call on a stream of its own allocates may be used again in that stream's order only."""
    torch = torch_()
    rng = np.random.default_rng(12)
    cache, _ = filled_cache(ops, rng, 2, 2, 4000, 64, "u4")
    q, lengths = tensor(rng.standard_normal((2, 8, 64)).astype(np.float32)), ints([4000, 3999])
    want = ops.attention_cached(cache, q, lengths)
    u, x = tensor(rng.random(2)), tensor(rng.standard_normal((2, 50)).astype(np.float32))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    s = side.cuda_stream
    outs = [ops.attention_cached(cache, q, lengths, stream=s), ops.sample_tokens(x, u, stream=s),
            *ops.kv_read(cache, lengths, stream=s),
            ops.attention_packed(q, q, q, ints([0, 2]), stream=s)]
    segments = torch.cuda.memory_snapshot()
    for t in outs:
        at = t.data_ptr()
        owner = [g["stream"] for g in segments if g["address"] <= at < g["address"] + g["total_size"]]
        assert owner == [s]
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    zero = ops.attention_cached(cache, q, lengths, stream=0)        # the legacy default stream
    torch.cuda.synchronize()
    assert torch.equal(zero, want)


def test_what_lies_outside_the_tokens_belongs_to_no_sequence(ops):
    """starts below 0 and behind the last token: the sequences' parts between are what counts."""
    torch = torch_()
    rng = np.random.default_rng(13)
    T, KV, d = 40, 2, 64
    q, k, v = (tensor(rng.standard_normal((T, n, d)).astype(np.float32)) for n in (4, KV, KV))
    lengths = ints([9, 60])
    results = []
    for starts in ([0, 7, T], [-5, 7, T + 300]):
        cache = ops.KvCache.allocate(2, KV, 64, d)
        starts = ints(starts)
        ops.kv_append(cache, k, v, lengths, starts=starts)
        results.append([cache.k, cache.v_scale, *ops.kv_read(cache, lengths, starts=starts, tokens=T),
                        ops.attention_cached(cache, q, lengths, starts=starts),
                        ops.attention_packed(q, k, v, starts, window=6, sinks=1),
                        ops.attention_packed(*(x.bfloat16() for x in (q, k, v)), starts)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_the_same_call_twice_gives_the_same_bits(ops):
    torch = torch_()
    rng = np.random.default_rng(6)
    cache, _ = filled_cache(ops, rng, 2, 2, 3000, 128, "u4")
    q = tensor(rng.standard_normal((2, 8, 128)).astype(np.float32))
    a, b = (ops.attention_cached(cache, q, ints([3000, 1234])) for _ in range(2))
    assert torch.equal(a, b)
    x = [tensor(rng.standard_normal((600, 4, 128)).astype(np.float32), "bf16") for _ in range(3)]
    a, b = (ops.attention_packed(*x, ints([0, 600]), window=200, sinks=4) for _ in range(2))
    assert torch.equal(a, b)


def test_workspaces_are_checked(ops):
    torch = torch_()
    from basalt_b200 import BasaltShapeException, IllegalArgumentException

    x = torch.zeros((40, 2, 64), device="cuda")
    with pytest.raises(BasaltShapeException, match="workspace"):
        ops.attention_packed(x, x, x, ints([0, 40]), workspace=torch.empty(1, device="cuda"))
    with pytest.raises(IllegalArgumentException, match="contiguous"):
        ops.attention_packed(x, x, x, ints([0, 40]), workspace=torch.empty(1, device="cuda").expand(1 << 20))
    with pytest.raises(IllegalArgumentException, match="starts"):
        ops.attention_packed(x, x, x, None)
