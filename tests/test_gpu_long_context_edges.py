"""Long-context operators where their pieces meet: masses in a place of their own, two host threads, tokens that
see nothing, arguments that are tensors, tiles that move two scales at once, and errors by the outputs' norm."""
import threading

import numpy as np
import pytest

from test_gpu_long_context import filled, kept_places, raw, softmax
from test_gpu_operators import host, ints, tensor, torch_

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(runtime):
    from basalt_b200 import operators

    return operators


def norm_error(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("own", [False, True])
def test_maxima_and_values_that_grow_in_the_same_tile(ops, dim, own):
    """4-bit keys whose scores grow by about 2^12 from each tile of 64 to the next, and values by 2^3 at the same
    keys: what was summed before is scaled for both (a factor that is lost leaves 2^-3 of the output and more). In
    every third tile only one of them grows. Outputs are rounded to bf16: 2^-8 of each entry at most, and so of a
    row's norm. Weights and values in fp16 add 2^-11 each, scores of up to 320 (base 2) that are good to 2^-20 another
    3e-4; all are well within a second 2^-8."""
    torch = torch_()
    rng = np.random.default_rng(dim)
    kv_heads, heads, tiles, tokens = 2, 16, 40, 20
    n = 64 * tiles
    k, v = rng.standard_normal((2, n, kv_heads, dim)).astype(np.float32) * np.float32([[[[0.1]]], [[[1.0]]]])
    tile = np.arange(n) // 64
    scores, values = np.cumsum(np.arange(tiles) % 3 != 1), np.cumsum(np.arange(tiles) % 3 != 2)
    k[..., 0] = 8.0 * scores[tile, None] * (dim / 64) ** 0.5
    v *= (2.0 ** (3.0 * values[tile]))[:, None, None].astype(np.float32)
    cache, starts = ops.KvCache.allocate(1, kv_heads, n, dim), ints([0, n])
    ops.kv_append(cache, tensor(k), tensor(v), ints([n]), starts=starts)
    k, v = (host(t) for t in ops.kv_read(cache, ints([n]), starts=starts, tokens=n))
    q = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    q[..., 0] = 8.0
    q = tensor(q, "bf16")
    qh = host(q)
    # Rows end in every part of the keys: the later ones see all the growth, the first ones little of it.
    ends = [n - tokens] if own else [n, 64 * 9, 64 * 20 + 5, 64, 130]
    for end in ends:
        if own:
            mass = torch.zeros((1, kv_heads, n), device="cuda")
            got = host(ops.attention_weights(cache, q, ints([n]), mass, starts=ints([0, tokens])))
            assert np.allclose(host(mass).sum(-1), tokens * heads // kv_heads, rtol=1e-4)
        else:
            empty = ops.KvCache.allocate(tokens, kv_heads, 4, dim)
            got = host(ops.attention_shared(empty, q, ints([0] * tokens), cache, end))
        for i in range(tokens):
            stop = end + i + 1 if own else end
            for h in range(heads):
                at = h * kv_heads // heads
                want = softmax(k[:stop, at] @ qh[i, h] * dim ** -0.5) @ v[:stop, at]
                assert norm_error(got[i, h], want) <= 2 * 2.0 ** -8, (end, i, h)


@pytest.mark.parametrize("storage,dim", [("u4", 32), ("u4", 128), ("bf16", 64), ("f32", 128)])
@pytest.mark.parametrize("slots,keep,recent,sinks", [(90, 40, 7, 5), (90, 40, 0, 0), (9000, 4500, 900, 3)])
def test_evicting_in_place_with_masses_elsewhere(ops, storage, dim, slots, keep, recent, sinks):
    """The masses of every kept key arrive, of those too that stay in their slots; `mass` is left as it was."""
    torch = torch_()
    rng = np.random.default_rng(slots + keep)
    lengths, rows = [slots, keep + 1, keep, keep - 1, 1, 0], [3, 0, 6, 2, 5, 1]
    cache, _, _ = filled(ops, rng, 7, 2, slots, dim, storage)
    before = raw(cache)
    m = (rng.random((7, 2, slots)) ** 3).astype(np.float32)
    m[3, 1] = np.sort(m[3, 1])[::-1]      # the first keys stay where they are
    mass, to_mass = tensor(m), torch.full((7, 2, slots), 9.0, device="cuda")
    new, kept = ops.kv_evict(cache, mass, ints(lengths), keep, recent, sinks, rows=ints(rows), to_mass=to_mass)
    assert new.tolist() == [min(n, keep) for n in lengths]
    assert np.array_equal(mass.cpu().numpy(), m)
    want, kept = np.full_like(m, 9.0), kept.cpu().numpy()
    for s, (row, n) in enumerate(zip(rows, lengths)):
        want[row] = 0.0
        for h in range(2):
            places = kept_places(m[row, h], n, keep, recent, sinks)
            assert kept[s, h, :len(places)].tolist() == places
            want[row, h, :len(places)] = m[row, h, places]
            for x, y in zip(raw(cache), before):
                moved = y[row, h][torch.tensor(places, device="cuda", dtype=torch.long)]
                assert torch.equal(x[row, h, :len(places)].view(torch.uint8), moved.view(torch.uint8))
    assert np.array_equal(to_mass.cpu().numpy(), want)


@pytest.mark.parametrize("slots", [(8192, 5000), (30000, 20000)])
def test_evictions_of_two_threads(ops, slots):
    """Two host threads, each with a stream and a cache of its own, whose rows need different room in shared memory."""
    torch = torch_()
    failed = []

    def serve(n, results):
        try:
            g = torch.Generator(device="cuda").manual_seed(n)
            stream = torch.cuda.Stream()
            cache = ops.KvCache.allocate(1, 1, n, 32)
            to, to_mass = ops.KvCache.allocate(1, 1, 64, 32), torch.zeros((1, 1, 64), device="cuda")
            mass = torch.rand((1, 1, n), generator=g, device="cuda")
            lengths, kept = ints([n]), torch.empty((1, 1, 64), dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            for _ in range(4000):
                ops.kv_evict(cache, mass, lengths, 64, 8, 4, to=to, to_mass=to_mass, kept=kept, stream=stream)
            stream.synchronize()
            results[n] = kept[0, 0].tolist()
            assert results[n] == kept_places(mass[0, 0].cpu().numpy(), n, 64, 8, 4)
        except Exception as e:  # noqa: BLE001 - the thread's failure is the test's
            failed.append(e)

    results = {}
    threads = [threading.Thread(target=serve, args=(n, results)) for n in slots]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert len(results) == 2


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("slots", [300, 2100])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_tokens_that_see_nothing_give_zeros_whatever_they_hold(ops, dim, slots, bad):
    """Tokens before the row's first key and behind its last slot, in tiles of which other tokens see keys."""
    torch = torch_()
    rng = np.random.default_rng(dim)
    cache, _, _ = filled(ops, rng, 3, 2, slots, dim, "u4")
    lengths, n = [3, slots + 20, 100], 40
    q = torch.randn((3 * n, 8, dim), device="cuda").bfloat16()
    blind = np.zeros(3 * n, bool)
    blind[:n - 3] = blind[2 * n - 20:2 * n] = True
    q[torch.from_numpy(np.flatnonzero(blind)[::2]).cuda()] = bad
    mass = torch.zeros((3, 2, slots), device="cuda")
    out = host(ops.attention_weights(cache, q, ints(lengths), mass, starts=ints(np.arange(4) * n)))
    assert np.all(out[blind] == 0)
    assert np.isfinite(out).all() and np.all(np.abs(out[~blind]).max((1, 2)) > 0)
    # Every token that sees keys gives each key head four times a weight of one in all.
    got = host(mass)
    assert np.allclose(got.sum(-1), np.array([[3], [20], [40]]) * 4, rtol=1e-4)


def test_rows_without_tokens_fade_where_a_kernel_before_says(ops):
    """`rows` and `lengths` are written on the stream right before the call."""
    torch = torch_()
    cache = ops.KvCache.allocate(64, 2, 700, 64)
    q, starts = torch.zeros((0, 4, 64), device="cuda"), torch.zeros(33, dtype=torch.int32, device="cuda")
    rows, lengths = (torch.empty(32, dtype=torch.int32, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    mass = torch.rand((64, 2, 700), generator=g, device="cuda")
    for _ in range(50):
        want, order = mass.clone(), torch.randperm(64, generator=g, device="cuda")[:32]
        n = torch.randint(0, 701, (32,), generator=g, device="cuda")
        faded = torch.arange(700, device="cuda") < n[:, None, None]
        want[order] = torch.where(faded, want[order] * 0.5, want[order])
        rows.zero_()
        lengths.zero_()
        torch.cuda._sleep(20000)
        rows.copy_(order)
        lengths.copy_(n)
        ops.attention_weights(cache, q, lengths, mass, decay=0.5, starts=starts, rows=rows)
        assert torch.equal(mass, want)


def test_a_row_of_nearly_2_31_slots(ops):
    """Places and strides near the end of 32 bits: eviction into such a row and within it, weights of all its keys."""
    torch = torch_()
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 125 << 30:
        pytest.skip("needs 125 GB of free memory")
    n = 2 ** 31 - 65537
    row = ops.KvCache.allocate(1, 1, n, 32)
    mass = torch.full((1, 1, n), 9.0, device="cuda")

    def others(low, high, but=0):   # all masses but the last `but` lie in [low, high]
        rest = mass[0, 0, :n - but]
        return low <= float(rest.min()) and float(rest.max()) <= high

    # 1000 keys move into it: masses behind them become zero up to the last.
    few = ops.KvCache.allocate(1, 1, 1000, 32)
    new, kept = ops.kv_evict(few, torch.ones((1, 1, 1000), device="cuda"), ints([1000]), 600000, to=row, to_mass=mass)
    assert new.tolist() == [1000] and (mass[0, 0, :1000] == 1).all()
    mass[0, 0, :1000] = 0.0
    assert others(0.0, 0.0)
    del kept
    # All keys but the last are alike; that one weighs about as much as the others together.
    row.k_scale[0, 0, n - 1, 0, 1] = 3.796875
    row.v_scale[0, 0, n - 1, 0, 1] = 1.0
    q, e = torch.ones((1, 1, 32), device="cuda"), float(np.exp(32 * 3.796875 * 32 ** -0.5))
    for starts in (None, ints([0, 1])):
        mass.fill_(9.0)
        out = host(ops.attention_weights(row, q, ints([n]), mass, decay=0.0, starts=starts))
        last, rest = e / (e + n - 1), 1.0 / (e + n - 1)
        assert np.allclose(out, last, rtol=1e-4, atol=0)
        assert abs(float(mass[0, 0, n - 1]) / last - 1) < 1e-4 and others(rest * (1 - 1e-4), rest * (1 + 1e-4), 1)
    # In place, ties: the last five go.
    mass.fill_(0.5)
    new, kept = ops.kv_evict(row, mass, ints([n]), n - 5)
    assert new.tolist() == [n - 5] and (mass[0, 0, n - 5:] == 0).all() and others(0.5, 0.5, 5)
    for at in range(0, n - 5, 1 << 27):
        some = kept[0, 0, at:at + (1 << 27)]
        assert torch.equal(some, torch.arange(at, at + some.shape[0], dtype=torch.int32, device="cuda"))
    del row, mass, kept
    torch.cuda.empty_cache()


def test_arguments_that_are_tensors_count_as_they_are_now(ops):
    """A scale, window or number of sinks in a tensor that is filled anew between calls."""
    torch = torch_()
    rng = np.random.default_rng(2)
    cache, _, _ = filled(ops, rng, 2, 2, 3000, 64, "bf16")
    common, _, _ = filled(ops, rng, 1, 2, 60, 64, "bf16")
    q = torch.randn((2, 4, 64), device="cuda").bfloat16()
    lengths, scale, window, sinks = ints([3000, 2999]), torch.tensor(0.25), torch.tensor(3), torch.tensor(2)

    def calls(scale, window, sinks):
        mass = torch.zeros((2, 2, 3000), device="cuda")
        weighed = ops.attention_weights(cache, q, lengths, mass, scale=scale, window=window, sinks=sinks)
        return (ops.attention_shared(cache, q, lengths, common, 60, scale=scale), weighed, mass,
                ops.attention_cached(cache, q, lengths, scale=scale, window=window, sinks=sinks))

    for s, w, n in ((0.25, 3, 2), (0.0625, 3000, 0), (1.0, 700, 41)):
        scale.fill_(s)
        window.fill_(w)
        sinks.fill_(n)
        for x, y in zip(calls(scale, window, sinks), calls(s, w, n)):
            assert torch.equal(x, y)


def test_lengths_must_be_a_vector(ops):
    from basalt_b200.text_engine import IllegalArgumentException

    torch = torch_()
    cache = ops.KvCache.allocate(1, 2, 20, 64)
    q, mass = torch.zeros((1, 4, 64), device="cuda"), torch.zeros((1, 2, 20), device="cuda")
    one = torch.tensor(5, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.attention_cached(cache, q, one), lambda: ops.attention_shared(cache, q, one, cache, 3),
                 lambda: ops.attention_weights(cache, q, one, mass), lambda: ops.kv_evict(cache, mass, one, 3),
                 lambda: ops.kv_append(cache, q[:, :2], q[:, :2], one), lambda: ops.kv_read(cache, one, tokens=1)):
        with pytest.raises(IllegalArgumentException, match="lengths"):
            call()
    for call in (lambda: ops.attention_cached(cache, q, None), lambda: ops.attention_shared(cache, q, None, cache, 3),
                 lambda: ops.attention_weights(cache, q, None, mass), lambda: ops.kv_evict(cache, mass, None, 3)):
        with pytest.raises(IllegalArgumentException):
            call()


@pytest.mark.parametrize("slots", [8192, 8193, 16385, 32769, 40961, 98305])
@pytest.mark.parametrize("kv_heads,count", [(1, 1), (13, 1), (3, 11), (5, 13)])
def test_evictions_of_few_and_many_heads(ops, slots, kv_heads, count):
    """The clusters of few heads with long rows, and the CTAs that many heads leave one another, around every border."""
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(slots + kv_heads)
    keep, recent, sinks = 700, 50, 3
    cache = ops.KvCache.allocate(count, kv_heads, slots, 32)
    to, to_mass = ops.KvCache.allocate(count, kv_heads, keep, 32), torch.empty((count, kv_heads, keep), device="cuda")
    mass = torch.rand((count, kv_heads, slots), generator=g, device="cuda")
    mass[:, :, ::3] = 0.75     # ties, some of which stay
    lengths = torch.randint(slots // 2, slots + 1, (count,), generator=g, device="cuda", dtype=torch.int32)
    lengths[0] = slots
    new, kept = ops.kv_evict(cache, mass, lengths, keep, recent, sinks, to=to, to_mass=to_mass)
    n = lengths.long()[:, None, None]
    j = torch.arange(slots, device="cuda")
    worth = mass.masked_fill((j < sinks) | (j >= n - recent), float("inf")).masked_fill(j >= n, -float("inf"))
    want = torch.sort(worth, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    assert (new == keep).all() and torch.equal(kept.long(), want)
    assert torch.equal(to_mass, mass.gather(2, want))


# ---- errors by the outputs' norm ---------------------------------------------------------------------
# Rounding x to bf16 moves it by up to 2^-8 of the power of two below it, uniformly: 2^-8 / sqrt 3 of x in the root mean
# square, or less. Weights in 8 bits do the same to each term of a sum of values without a common part, and so to the
# sum's norm. 11 bits (weights times values or steps, and values of 4-bit codes) are 2^-11 / sqrt 3 each. Independent
# errors add up by squares. A single row of 64 entries and more stays within twice its share.
ROUNDED, FP16 = 2.0 ** -8 / 3 ** 0.5, 2.0 ** -11 / 3 ** 0.5
BITS = {8: (2 * ROUNDED ** 2) ** 0.5, 11: (ROUNDED ** 2 + 2 * FP16 ** 2) ** 0.5, 16: ROUNDED * (1 + 2.0 ** -8)}


def check_norms(got, want, limit):
    """All rows together, and each of them."""
    off, size = np.linalg.norm(got - want, axis=-1), np.linalg.norm(want, axis=-1)
    assert np.linalg.norm(off) <= limit * np.linalg.norm(size), np.linalg.norm(off) / np.linalg.norm(size)
    assert np.all(off <= 2 * limit * size), (off / size).max()


@pytest.mark.parametrize("dim,prefix", [(64, 5001), (128, 9000), (128, 40003)])
@pytest.mark.parametrize("storage,rows,bits", [
    ("bf16", 4, 16), ("bf16", 8, 16), ("bf16", 200, 8), ("bf16", 700, 8),   # on tcgen05 weights are bf16
    ("u4", 4, 11), ("u4", 24, 11), ("u4", 200, 11), ("u4", 700, 11)])
def test_bf16_outputs_behind_a_prefix_by_their_norm(ops, storage, rows, bits, dim, prefix):
    """`rows` queries of each of two key heads behind one long prefix."""
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(prefix + rows)
    heads = 8 if rows >= 8 else 4
    count = 2 * rows // heads
    common = ops.KvCache.allocate(1, 2, prefix, dim, storage)
    x = torch.randn((2, prefix, 2, dim), generator=g, device="cuda")
    x[0] += 2 * torch.randn((1, 2, dim), generator=g, device="cuda") * (torch.rand((1, 2, dim), generator=g, device="cuda") < 0.1)
    starts = ints([0, prefix])
    ops.kv_append(common, x[0], x[1], ints([prefix]), starts=starts)
    k, v = (t.double() for t in ops.kv_read(common, ints([prefix]), starts=starts, tokens=prefix))
    own = ops.KvCache.allocate(count, 2, 4, dim, storage)
    q = torch.randn((count, heads, dim), generator=g, device="cuda").bfloat16()
    got = host(ops.attention_shared(own, q, ints([0] * count), common, prefix))
    score = torch.einsum("shgd,jhd->shgj", q.double().unflatten(1, (2, -1)), k) * dim ** -0.5
    want = torch.einsum("shgj,jhd->shgd", torch.softmax(score, -1), v).flatten(1, 2)
    check_norms(got, host(want), BITS[bits])


@pytest.mark.parametrize("storage,dim,heads,tokens,bits", [
    ("u4", 128, 8, 1, 11), ("u4", 64, 8, 1, 11), ("u4", 128, 2, 1, 16), ("u4", 128, 8, 16, 11), ("u4", 64, 16, 40, 11),
    ("bf16", 128, 8, 1, 16), ("bf16", 64, 2, 1, 16)])
def test_bf16_outputs_and_masses_of_weights_by_their_norm(ops, storage, dim, heads, tokens, bits):
    """The last tokens of long rows, of two key heads. Masses are float32: a score is good to 2^-20 of the sum of its
    products' sizes, and the exponential and the sums to 2^-20 of a weight."""
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(dim + heads + tokens)
    n, rows = 6007, 3
    cache = ops.KvCache.allocate(rows, 2, n, dim, storage)
    x = torch.randn((2, rows * n, 2, dim), generator=g, device="cuda")
    starts, lengths = ints(np.arange(rows + 1) * n), ints([n] * rows)
    if storage == "u4":
        ops.kv_append(cache, x[0], x[1], lengths, starts=starts)
        k, v = (t.double().unflatten(0, (rows, n)) for t in ops.kv_read(cache, lengths, starts=starts, tokens=rows * n))
    else:
        for t, y in zip((cache.k, cache.v), x):
            t.copy_(y.unflatten(0, (rows, n)).transpose(1, 2))
        k, v = (t.double().transpose(1, 2) for t in (cache.k, cache.v))
    q = torch.randn((rows * tokens, heads, dim), generator=g, device="cuda").bfloat16()
    mass = torch.zeros((rows, 2, n), device="cuda")
    got = host(ops.attention_weights(cache, q, lengths, mass, decay=0.0,
                                     starts=None if tokens == 1 else ints(np.arange(rows + 1) * tokens)))
    qh = q.double().unflatten(0, (rows, tokens)).unflatten(2, (2, -1))      # [rows, tokens, 2, group, dim]
    score = torch.einsum("stgad,sjgd->stgaj", qh, k) * dim ** -0.5
    size = float(torch.einsum("stgad,sjgd->stgaj", qh.abs(), k.abs()).max()) * dim ** -0.5
    hidden = torch.arange(n, device="cuda") > torch.arange(n - tokens, n, device="cuda")[:, None]
    p = torch.softmax(score.masked_fill(hidden[:, None, None], -np.inf), -1)
    want = torch.einsum("stgaj,sjgd->stgad", p, v).flatten(0, 1).flatten(1, 2)
    check_norms(got, host(want), BITS[bits])
    check_norms(host(mass), host(p.sum((1, 3))), 2.0 ** -20 * (size + 1))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("small,large", [(-16, 0), (-30, 0), (-60, 0), (-6, 4), (-6, 9), (-12, 20)])
def test_small_entries_beside_large_ones(ops, dim, own, small, large):
    """4-bit keys and values of which some are 2^small of the usual size, and some keys 2^large with scores that leave
    them no weight, in every tile of 64. A score may be off by 2^-12 (base 2) by what the large keys' fp16 leaves the
    small ones, which moves a weight by 2^-12 ln 2; outputs otherwise as above."""
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(dim)
    n, kv_heads, heads, tokens = 2600, 2, 16, 24
    x = torch.randn((2, n, kv_heads, dim), generator=g, device="cuda")
    x[:, 5::32] *= 2.0 ** small
    x[1, 6::64] *= 2.0 ** small
    if large:
        x[0, 9::64] = -2.0 ** large * x[0, 9::64].abs()
    cache, starts = ops.KvCache.allocate(1, kv_heads, n, dim), ints([0, n])
    ops.kv_append(cache, x[0], x[1], ints([n]), starts=starts)
    k, v = (t.double() for t in ops.kv_read(cache, ints([n]), starts=starts, tokens=n))
    q = torch.randn((tokens, heads, dim), generator=g, device="cuda")
    q = (q.abs() if large else q).bfloat16()
    if own:
        mass = torch.zeros((1, kv_heads, n), device="cuda")
        got = host(ops.attention_weights(cache, q, ints([n]), mass, starts=ints([0, tokens]), decay=0.0))
    else:
        empty = ops.KvCache.allocate(tokens, kv_heads, 4, dim)
        got = host(ops.attention_shared(empty, q, ints([0] * tokens), cache, n))
    score = torch.einsum("sgad,jgd->sgaj", q.double().unflatten(1, (2, -1)), k) * dim ** -0.5
    if own:
        hidden = torch.arange(n, device="cuda") > torch.arange(n - tokens, n, device="cuda")[:, None]
        score.masked_fill_(hidden[:, None, None], -np.inf)
    p = torch.softmax(score, -1)
    moved = 2.0 ** -12 * np.log(2)
    check_norms(got, host(torch.einsum("sgaj,jgd->sgad", p, v).flatten(1, 2)), BITS[11] + moved)
    if own:
        check_norms(host(mass)[0], host(p.sum((0, 2))), moved)


def test_a_small_entry_does_not_slow_a_call(ops):
    """One token a tile with a key and a value 2^-30 of the others' leaves the time of a call as it is, within a factor of
    three (rows that are added up plainly take a hundred times as long)."""
    torch = torch_()
    cache, own = ops.KvCache.allocate(1, 8, 8192, 128), ops.KvCache.allocate(96, 8, 4, 128)
    x = torch.randn((2, 8192, 8, 128), device="cuda")
    q, lengths = torch.randn((96, 32, 128), device="cuda").bfloat16(), ints([0] * 96)
    mass = torch.zeros((1, 8, 8192), device="cuda")
    times = []
    for factor in (1.0, 2.0 ** -30):
        x[:, ::64] *= factor
        ops.kv_append(cache, x[0], x[1], ints([8192]), starts=ints([0, 8192]))
        for call in (lambda: ops.attention_shared(own, q, lengths, cache, 8192),
                     lambda: ops.attention_weights(cache, q, ints([8192]), mass, starts=ints([0, 96]), decay=0.0)):
            call()
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            e[0].record()
            for _ in range(20):
                call()
            e[1].record()
            torch.cuda.synchronize()
            times.append(e[0].elapsed_time(e[1]))
    assert times[2] <= 3 * times[0] and times[3] <= 3 * times[1], times
