"""Attention behind a shared prefix, attention that adds up weights, and eviction, against plain 64-bit
implementations.

Tolerances. Outputs as for attention over a cache: a score of d products is off by at most
(d + 8) 2^-23 sum|q k| scale, a weight by twice that of itself and the exponential's 2^-21, a sum over n
weights adds n 2^-24 on either side of the quotient, and an output is off by at most max|v| times their sum;
bf16 outputs add their weights' 2^-8 of max|v|, what bf16 values of 4-bit codes add on the tensor cores
(2^-8 of max|v| again, and 2^-11 of a score for keys in fp16), and their own 2^-8. A mass is a sum of
weights (float32 for every type): it is off by the weights' relative error times their sum, and by 2^-23 of
the old mass, which is multiplied and added.
"""
import numpy as np
import pytest

import operator_reference as ref
from test_gpu_operators import bound, host, ints, tensor, torch_

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(runtime):
    from basalt_b200 import operators

    return operators


def filled(ops, rng, rows, kv_heads, slots, dim, storage):
    """A cache whose every slot is stored, and the values [rows, slots, kv_heads, dim] it stands for."""
    cache = ops.KvCache.allocate(rows, kv_heads, slots, dim, storage)
    starts, lengths = ints(np.arange(rows + 1) * slots), ints([slots] * rows)
    x = rng.standard_normal((2, rows * slots, kv_heads, dim)).astype(np.float32)
    x[0] += 2.0 * rng.standard_normal((1, kv_heads, dim)) * (rng.random((1, kv_heads, dim)) < 0.1)
    ops.kv_append(cache, tensor(x[0]), tensor(x[1]), lengths, starts=starts)
    k, v = ops.kv_read(cache, lengths, starts=starts, tokens=rows * slots)
    return cache, *(host(t).reshape(rows, slots, kv_heads, dim) for t in (k, v))


def spoil(cache, row, slot):
    """NaN in every value of a row's slots from `slot` on."""
    for t in (cache.k, cache.v) if cache.k_scale is None else (cache.k_scale, cache.v_scale):
        t[row, :, slot:] = float("nan")


def queries(rng, tokens, heads, dim, dtype):
    """Queries as a slice of a wider tensor, and what they are in 64 bits."""
    wide = tensor(rng.standard_normal((tokens, heads * dim + 64)).astype(np.float32), dtype)
    q = wide[:, 32:32 + heads * dim].unflatten(-1, (heads, dim))
    return q, host(q)


def softmax(score):
    p = np.exp(score - score.max())
    return p / p.sum()


# ---- a shared prefix -----------------------------------------------------------------------------
def shared_reference(q, keys, values, own_k, own_v, first, scale):
    """q [n, H, d] of one sequence, its own keys [m, KV, d] from position `first`; out and sizes."""
    n, H, d = q.shape
    out, size = np.zeros((n, H, d)), np.zeros((n, H))
    for i in range(n):
        m = min(max(first + i + 1, 0), own_k.shape[0]) if first + i < own_k.shape[0] else 0
        for h in range(H):
            at = h * keys.shape[1] // H
            k = np.concatenate([keys[:, at], own_k[:m, at]])
            v = np.concatenate([values[:, at], own_v[:m, at]])
            if len(k):
                out[i, h] = softmax(k @ q[i, h] * scale) @ v
                size[i, h] = (np.abs(k) @ np.abs(q[i, h])).max() * abs(scale)
    return out, size


def shared_bound(size, d, n, vmax, out, dtype, prefix_storage):
    tol = bound(size, d, n, vmax, out, dtype)
    if dtype == "bf16" and prefix_storage == "u4":
        tol = tol + vmax * (2.0 ** -8 + 2.2 * 2.0 ** -11 * size[..., None])
    return tol


def check_shared(ops, rng, storage, prefix_storage, dtype, dim, heads, kv_heads, prefix, lengths, counts=None,
                 slots=None, scale=None, ahead=0):
    slots = slots or max(lengths) + 5
    count = len(lengths)
    own, own_k, own_v = filled(ops, rng, count + 1, kv_heads, slots, dim, storage)
    common, keys, values = filled(ops, rng, 3, kv_heads, prefix + 9, dim, prefix_storage)
    spoil(common, 1, prefix)
    rows = rng.permutation(count + 1)[:count]
    for s, n in enumerate(lengths):
        spoil(own, rows[s], max(n, 0))
    starts = None if counts is None else ahead + np.concatenate([[0], np.cumsum(counts)])
    counts = counts or [1] * count
    tokens = count if starts is None else int(starts[-1]) + 2
    q, q64 = queries(rng, tokens, heads, dim, dtype)
    out = torch_().full((tokens, heads, dim), 7.5, dtype=q.dtype, device="cuda")
    got = ops.attention_shared(own, q, ints(lengths), common, prefix, prefix_row=1, rows=ints(rows),
                               starts=None if starts is None else ints(starts), scale=scale, out=out)
    assert got is out
    got = host(got)
    vmax = max(np.abs(values[1]).max(), np.abs(own_v).max())
    for s, n in enumerate(lengths):
        at = s if starts is None else int(starts[s])
        mine = q64[at:at + counts[s]]
        want, size = shared_reference(mine, keys[1, :prefix], values[1, :prefix], own_k[rows[s], :max(n, 0)],
                                      own_v[rows[s], :max(n, 0)], n - counts[s],
                                      dim ** -0.5 if scale is None else scale)
        tol = shared_bound(size, dim, prefix + max(n, 0), vmax, want, dtype, prefix_storage)
        assert np.all(np.abs(got[at:at + counts[s]] - want) <= tol), (s, np.abs(got[at:at + counts[s]] - want).max())
    if starts is not None:
        assert np.all(got[:ahead] == 7.5) and np.all(got[int(starts[-1]):] == 7.5)


@pytest.mark.parametrize("prefix", [0, 1, 15, 64, 200, 1000])
@pytest.mark.parametrize("storage,prefix_storage,dtype", [
    ("u4", "u4", "f32"), ("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("u4", "u4", "bf16"),
    ("bf16", "u4", "bf16"), ("u4", "f32", "bf16"), ("f32", "bf16", "f32")])
def test_shared_prefix(ops, storage, prefix_storage, dtype, prefix):
    rng = np.random.default_rng(prefix + len(storage))
    check_shared(ops, rng, storage, prefix_storage, dtype, 64, 4, 2, prefix, [3, 1, 0, 40, 17])


@pytest.mark.parametrize("dim,heads,kv_heads,count", [(32, 3, 3, 7), (32, 8, 1, 40), (64, 12, 3, 33), (128, 8, 8, 70),
                                                      (128, 16, 2, 50), (64, 5, 5, 1), (128, 24, 4, 150)])
@pytest.mark.parametrize("storage,dtype", [("u4", "bf16"), ("bf16", "bf16"), ("u4", "f32"), ("f32", "f32")])
def test_shared_prefix_of_many_queries(ops, dim, heads, kv_heads, count, storage, dtype):
    rng = np.random.default_rng(dim + count)
    check_shared(ops, rng, storage, storage, dtype, dim, heads, kv_heads, 333, list(rng.integers(0, 30, count)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("prefix_storage", ["u4", "bf16", "f32"])
def test_shared_prefix_with_several_tokens(ops, dtype, prefix_storage):
    rng = np.random.default_rng(3)
    check_shared(ops, rng, "u4", prefix_storage, dtype, 64, 6, 2, 130, [9, 5, 0, 33, 2], counts=[4, 0, 3, 33, 7],
                 ahead=3)   # a sequence without tokens, one whose tokens have no keys, one longer than its row
    check_shared(ops, rng, "u4", prefix_storage, dtype, 128, 8, 2, 700, [300, 41], counts=[90, 41])


@pytest.mark.parametrize("prefix_storage", ["u4", "bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
def test_shared_prefix_scales(ops, prefix_storage, scale):
    rng = np.random.default_rng(4)
    for dtype in ("bf16", "f32"):
        check_shared(ops, rng, "u4", prefix_storage, dtype, 64, 8, 2, 150, list(rng.integers(0, 9, 40)), scale=scale)


@pytest.mark.parametrize("storage,dtype", [("u4", "bf16"), ("bf16", "bf16"), ("u4", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("dim,heads,kv_heads,count,prefix", [
    (64, 8, 2, 70, 5001), (128, 32, 8, 150, 4159), (128, 4, 4, 300, 9000), (64, 16, 1, 37, 40003), (128, 40, 8, 24, 2048)])
def test_long_prefixes(ops, storage, dtype, dim, heads, kv_heads, count, prefix):
    """Many tiles of keys a CTA, against 64 bits on the GPU."""
    torch = torch_()
    rng = np.random.default_rng(prefix)
    g = torch.Generator(device="cuda").manual_seed(prefix)
    common = ops.KvCache.allocate(1, kv_heads, prefix + 3, dim, storage)
    x = torch.randn((2, prefix, kv_heads, dim), generator=g, device="cuda")
    x[0] += 3 * torch.randn((1, kv_heads, dim), generator=g, device="cuda").clamp(min=1)
    x[0, prefix // 2] *= 4                       # a key that moves many a maximum
    x[1, prefix // 3:] *= 30                     # values that grow on the way
    ops.kv_append(common, x[0], x[1], ints([prefix]), starts=ints([0, prefix]))
    k, v = (t.double().transpose(0, 1) for t in ops.kv_read(common, ints([prefix]), starts=ints([0, prefix]), tokens=prefix))
    spoil(common, 0, prefix)
    own, own_k, own_v = filled(ops, rng, count, kv_heads, 4, dim, storage)
    q = torch.randn((count, heads, dim), generator=g, device="cuda").to(getattr(torch, {"f32": "float32", "bf16": "bfloat16"}[dtype]))
    lengths = rng.integers(0, 5, count)
    got = host(ops.attention_shared(own, q, ints(lengths), common, prefix))
    own_k, own_v = (torch.from_numpy(t).cuda() for t in (own_k, own_v))      # [count, slots, kv_heads, dim]
    group, scale = heads // kv_heads, dim ** -0.5
    hidden = torch.arange(4, device="cuda") >= ints(lengths)[:, None]
    for h in range(kv_heads):
        qh = q[:, h * group:(h + 1) * group].double()                        # [count, group, dim]
        score = torch.cat([qh @ k[h].T, torch.einsum("sgd,sjd->sgj", qh, own_k[:, :, h])
                           .masked_fill(hidden[:, None], -np.inf)], -1) * scale
        p = torch.softmax(score, -1)
        want = p[..., :prefix] @ v[h] + torch.einsum("sgj,sjd->sgd", p[..., prefix:], own_v[:, :, h])
        size = (qh.abs() @ k[h].abs().T).amax(-1).cpu().numpy() * scale
        spread = float(max(v[h].abs().max(), own_v.abs().max()))
        want = want.cpu().numpy()
        tol = shared_bound(size, dim, prefix + 4, spread, want, dtype, storage)
        off = np.abs(got[:, h * group:(h + 1) * group] - want)
        assert np.all(off <= tol), (off / tol).max()


@pytest.mark.parametrize("storage", ["f32", "bf16", "u4"])
def test_float32_sums_over_a_long_prefix(ops, storage):
    """n = 20 000 keys in float32. A running sum is rounded once for 16 keys, 2^-24 of itself; such errors add up as
    random ones do over the n / 16 roundings of all splits together, to sqrt(1250) 2^-24 = 2.1e-6. Scores of up to
    16 are off by 2^-22 of themselves, which every key's weight carries on its own: 16 ln 2 2^-22 / 2 = 1.3e-6. Sums
    that are cut instead of rounded were 1.2e-5 off."""
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(1)
    n, kv_heads, dim, heads = 20000, 3, 128, 9
    common = ops.KvCache.allocate(1, kv_heads, n, dim, storage)
    x = torch.randn((2, n, kv_heads, dim), generator=g, device="cuda")
    x[0] += 2 * torch.randn((1, kv_heads, dim), generator=g, device="cuda") * (torch.rand((1, kv_heads, dim), generator=g, device="cuda") < 0.1)
    ops.kv_append(common, x[0], x[1], ints([n]), starts=ints([0, n]))
    k, v = (t.double() for t in ops.kv_read(common, ints([n]), starts=ints([0, n]), tokens=n))
    own = ops.KvCache.allocate(14, kv_heads, 4, dim, "u4")
    q = torch.randn((14, heads, dim), generator=g, device="cuda")
    got = ops.attention_shared(own, q, ints([0] * 14), common, n).double()
    qh = q.double().unflatten(1, (kv_heads, -1))
    want = torch.einsum("shgj,jhd->shgd", torch.softmax(torch.einsum("shgd,jhd->shgj", qh, k) * dim ** -0.5, -1), v)
    off = (got - want.flatten(1, 2)).norm() / want.norm()
    assert off <= 2.1e-6 + 1.3e-6, off


def test_a_prefix_in_the_same_cache_and_out_over_q(ops):
    torch = torch_()
    rng = np.random.default_rng(5)
    cache, k, v = filled(ops, rng, 4, 2, 90, 64, "bf16")
    q, q64 = queries(rng, 3, 4, 64, "bf16")
    q = q.contiguous()
    lengths, rows = [5, 1, 30], [1, 3, 0]
    got = ops.attention_shared(cache, q, ints(lengths), cache, 77, prefix_row=2, rows=ints(rows), out=q)
    assert got is q
    for s in range(3):
        want, size = shared_reference(q64[s:s + 1], k[2, :77], v[2, :77], k[rows[s], :lengths[s]],
                                      v[rows[s], :lengths[s]], lengths[s] - 1, 0.125)
        assert np.all(np.abs(host(got)[s] - want[0]) <= bound(size, 64, 110, np.abs(v).max(), want, "bf16")[0])
    # rows outside the cache have no keys of their own
    q, q64 = queries(rng, 2, 4, 64, "f32")
    got = host(ops.attention_shared(cache, q, ints([5, 5]), cache, 9, rows=ints([-1, 4])))
    for s in range(2):
        want, size = shared_reference(q64[s:s + 1], k[0, :9], v[0, :9], k[0, :0], v[0, :0], -1, 0.125)
        assert np.all(np.abs(got[s] - want[0]) <= bound(size, 64, 9, np.abs(v).max(), want, "f32")[0])
    # no keys at all: zeros
    got = ops.attention_shared(cache, q, ints([0, 0]), cache, 0)
    assert torch.equal(got, torch.zeros_like(got))


@pytest.mark.parametrize("storage,dtype", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("heads,count", [(2, 3), (8, 40)])
def test_values_of_a_prefix_that_are_not_finite(ops, storage, dtype, heads, count):
    """They count as in the formula: a NaN makes every output NaN, a key whose score is -infinity takes no
    part, an infinite value makes its channel infinite."""
    torch = torch_()
    rng = np.random.default_rng(6)
    dim, prefix = 64, 200
    own, _, _ = filled(ops, rng, count, 2, 8, dim, storage)
    common, keys, values = filled(ops, rng, 1, 2, prefix, dim, storage)
    common.k[0, 0, 70] = 0.0
    common.k[0, 0, 70, 0] = -float("inf")      # score -inf where q[0] > 0
    common.v[0, 1, 199, 5] = float("inf")
    q = torch.rand((count, heads, dim), device="cuda").to(getattr(torch, {"f32": "float32", "bf16": "bfloat16"}[dtype])) + 0.1
    got = host(ops.attention_shared(own, q, ints([8] * count), common, prefix))
    assert np.isfinite(got[:, :heads // 2]).all()
    late = got[:, heads // 2:]
    assert np.all(late[..., 5] == np.inf) and np.isfinite(np.delete(late, 5, -1)).all()
    common.k[0, 1, 3, 9] = float("nan")
    got = host(ops.attention_shared(own, q, ints([8] * count), common, prefix))
    assert np.isfinite(got[:, :heads // 2]).all() and np.isnan(got[:, heads // 2:]).all()


# ---- weights ---------------------------------------------------------------------------------------
def check_weights(ops, rng, storage, dtype, dim, heads, kv_heads, lengths, counts=None, window=0, sinks=0,
                  decay=1.0, slots=None, rows=None, in_place=True, scale=None):
    count, slots = len(lengths), slots or max(lengths) + 3
    cache, k, v = filled(ops, rng, count + 2, kv_heads, slots, dim, storage)
    rows = list(rng.permutation(count + 2)[:count]) if rows is None else rows
    starts = None if counts is None else 1 + np.concatenate([[0], np.cumsum(counts)])
    counts = counts or [1] * count
    tokens = count if starts is None else int(starts[-1]) + 2
    q, q64 = queries(rng, tokens, heads, dim, dtype)
    before = (rng.random((count + 2, kv_heads, slots)) ** 4 * 5).astype(np.float32)
    mass = tensor(before)
    previous = None
    if not in_place:
        previous, mass = mass, torch_().full_like(mass, -3.0)
        if decay == 0:
            previous.fill_(float("nan"))
    kept = host(mass)
    out = ops.attention_weights(cache, q, ints(lengths), mass, previous=previous, decay=decay, rows=ints(rows),
                                starts=None if starts is None else ints(starts), window=window, sinks=sinks,
                                scale=scale)
    plain = ops.attention_cached(cache, q, ints(lengths), rows=ints(rows), window=window, sinks=sinks,
                                 starts=None if starts is None else ints(starts), scale=scale)
    got, out, plain = host(mass), host(out), host(plain)
    scale = dim ** -0.5 if scale is None else scale
    added, tol, end = np.zeros_like(before, np.float64), np.zeros_like(before, np.float64), {}
    for s, n in enumerate(lengths):
        first, row = (s if starts is None else int(starts[s])), rows[s]
        inside = 0 <= row < count + 2
        kk, vv = (x[row] if inside else x[0, :0] for x in (k, v))
        want, size = ref.attend(q64[first:first + counts[s]], kk[:max(0, min(n, slots))], vv[:max(0, min(n, slots))],
                                n - counts[s], window, sinks, scale)
        for i in range(counts[s]):
            if n - counts[s] + i >= slots:     # a token outside the cache sees nothing
                want[i], size[i] = 0, 0
        t = bound(size, dim, n, np.abs(v).max(), want, dtype)
        assert np.all(np.abs(out[first:first + counts[s]] - want) <= t), s
        assert np.all(np.abs(plain[first:first + counts[s]] - want) <= t), s
        if not inside:
            continue
        end[row] = max(end.get(row, 0), min(max(n, 0), slots))
        for i in range(counts[s]):
            position = n - counts[s] + i
            if position < 0 or position >= slots:
                continue
            seen = ref.visible(position, slots, window, sinks)
            for h in range(heads):
                at = h * kv_heads // heads
                p = np.zeros(slots)
                p[seen] = softmax(k[row, seen, at] @ q64[first + i, h] * scale)
                added[row, at] += p
                tol[row, at] += p * (2.2 * (dim + 8) * 2.0 ** -23 * size[i, h] + 2.0 ** -20 + (n + 16) * 2.0 ** -23)
    want = kept.copy()
    for row, n in end.items():
        old = before[row, :, :n] * float(np.float32(decay)) if decay else 0.0
        want[row, :, :n] = old + added[row, :, :n]
        tol[row, :, :n] += 2.0 ** -22 * want[row, :, :n]
    assert np.all(np.abs(got - want) <= tol), np.nanmax(np.abs(got - want) - tol)


@pytest.mark.parametrize("storage,dtype", [("u4", "f32"), ("u4", "bf16"), ("bf16", "bf16"), ("f32", "f32"),
                                           ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("dim,heads,kv_heads", [(32, 2, 2), (64, 8, 2), (128, 4, 4), (64, 12, 1), (128, 24, 2)])
def test_weights(ops, storage, dtype, dim, heads, kv_heads):
    rng = np.random.default_rng(dim + heads)
    check_weights(ops, rng, storage, dtype, dim, heads, kv_heads, [1, 40, 0, 17, 300])
    check_weights(ops, rng, storage, dtype, dim, heads, kv_heads, [33, 150], window=20, sinks=3, decay=0.5)


@pytest.mark.parametrize("storage", ["bf16", "f32"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_weights_of_small_groups(ops, storage, dtype, dim):
    """One to four queries a key head, which float32 and bf16 caches take in kernels of their own."""
    rng = np.random.default_rng(dim)
    for heads in (2, 4, 6, 8):
        check_weights(ops, rng, storage, dtype, dim, heads, 2, [200, 1, 0, 77], window=0 if heads < 6 else 50, sinks=7,
                      decay=0.3)
        check_shared(ops, rng, storage, storage, dtype, dim, heads, 2, 40, [190, 0, 1, 33])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 2), (6, 1)])
def test_weights_of_several_tokens(ops, dtype, heads, kv_heads):
    rng = np.random.default_rng(heads)
    for dim in (32, 64, 128):
        check_weights(ops, rng, "u4", dtype, dim, heads, kv_heads, [20, 5, 0, 41, 2], counts=[4, 0, 2, 41, 7],
                      decay=0.0, in_place=False)
        check_weights(ops, rng, "u4", dtype, dim, heads, kv_heads, [60, 90, 33], counts=[8, 17, 1], window=13,
                      sinks=5, decay=0.9)


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 2), (128, 16, 2), (64, 3, 1), (128, 8, 1)])
def test_weights_of_many_tokens(ops, dim, heads, kv_heads):
    """Query rows by the dozen: votes of prompts' last tokens, and tokens beside sequences of few or none."""
    rng = np.random.default_rng(dim + heads)
    for slots in (None, 2100):   # with many slots on the tensor cores' large tiles, if there are rows enough
        check_weights(ops, rng, "u4", "bf16", dim, heads, kv_heads, [1500, 700, 64, 40], counts=[16, 16, 16, 40],
                      decay=0.5, slots=slots)
        check_weights(ops, rng, "u4", "bf16", dim, heads, kv_heads, [130, 90, 5, 0, 260], counts=[130, 3, 9, 0, 100],
                      decay=0.0, in_place=False, slots=slots)
        check_weights(ops, rng, "u4", "bf16", dim, heads, kv_heads, [90, 200], counts=[60, 60], scale=-0.25, rows=[3, 3],
                      slots=slots)
        check_weights(ops, rng, "u4", "bf16", dim, heads, kv_heads, [90, 200], counts=[60, 60], rows=[-1, 4], slots=slots)
    check_weights(ops, rng, "u4", "bf16", dim, heads, kv_heads, [300, 301, 200], counts=[40, 50, 40], slots=280)
    check_weights(ops, rng, "u4", "bf16", dim, heads, kv_heads, [2070, 2099], counts=[64, 70], slots=2060)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("slots", [200, 2048])
def test_weights_of_tokens_that_see_nan_or_not(ops, dtype, dim, slots):
    """A value that is NaN reaches the tokens that see its key, a key that is NaN their weights too."""
    torch = torch_()
    rng = np.random.default_rng(15)
    cache, _, _ = filled(ops, rng, 2, 2, slots, dim, "u4")
    cache.v_scale[0, 0, 150, 1, 0] = float("nan")       # tokens from position 150 on, channels 32 to 63
    cache.k_scale[0, 1, 160, 0, 1] = float("nan")       # tokens from position 160 on
    q, _ = queries(rng, 60, 16, dim, dtype)
    mass = torch.zeros((2, 2, slots), device="cuda")
    out = host(ops.attention_weights(cache, q, ints([190, 120]), mass, starts=ints([0, 50, 60]), decay=0.0))
    got = host(mass)
    position = np.arange(140, 190)
    first, second = out[:50, :8], out[:50, 8:]
    assert np.isnan(first[position >= 150][..., 32:64]).all() and np.isfinite(np.delete(first, range(32, 64), -1)).all()
    assert np.isfinite(first[position < 150]).all()
    assert np.isnan(second[position >= 160]).all() and np.isfinite(second[position < 160]).all()
    assert np.isfinite(out[50:]).all() and np.isfinite(got[0, 0]).all() and np.isfinite(got[1]).all()
    assert np.isnan(got[0, 1, :190]).all()
    assert np.allclose(got[0, 0, :190].sum(), 50 * 8, rtol=1e-4)


def test_weights_of_long_rows_are_split(ops):
    rng = np.random.default_rng(8)
    check_weights(ops, rng, "u4", "bf16", 128, 8, 2, [9001], decay=0.25, in_place=False)
    check_weights(ops, rng, "u4", "f32", 64, 2, 2, [5000, 2047, 1])
    check_weights(ops, rng, "bf16", "bf16", 64, 8, 1, [4097, 1025], window=2000, sinks=17)
    check_weights(ops, rng, "f32", "f32", 32, 1, 1, [3000])


@pytest.mark.parametrize("heads,counts", [(8, None), (40, None), (8, [3] * 30), (8, [17] * 28 + [0, 40])])
def test_weights_of_many_long_rows(ops, heads, counts):
    """So many keys in all that a CTA adds up several chunks of them: some whole, some ragged, some behind the end."""
    rng = np.random.default_rng(heads)
    lengths = [4600, 1, 511, 512, 513, 0, 1024, 1025, 1536, 1537, 2600, 4097] + [40] * 17 + [2048]
    if counts is not None:
        lengths = [max(n, k) for n, k in zip(lengths, counts)]
    check_weights(ops, rng, "u4", "f32", 32, heads, 8, lengths, counts=counts, decay=0.5, slots=4600)
    check_weights(ops, rng, "u4", "f32", 32, heads, 8, lengths, counts=counts, decay=0.0, in_place=False, window=700,
                  sinks=5, slots=4600)


def test_weights_with_rows_named_twice_outside_and_too_long(ops):
    rng = np.random.default_rng(9)
    for storage in ("u4", "bf16"):
        check_weights(ops, rng, storage, "f32", 64, 4, 2, [30, 12, 25, 30, 7], rows=[2, 0, 2, 7, -1])
        check_weights(ops, rng, storage, "f32", 64, 4, 2, [40, 39, 41], slots=40)
        check_weights(ops, rng, storage, "bf16", 64, 4, 2, [30, 12], scale=-0.3)
        check_weights(ops, rng, storage, "bf16", 64, 4, 2, [30, 12], scale=0.0)


def test_weights_beside_infinities_and_nan(ops):
    """A key of score -infinity weighs nothing; a NaN key makes the weights of the queries that see it NaN;
    what lies behind the length, or outside the window, is not looked at."""
    torch = torch_()
    rng = np.random.default_rng(10)
    for storage, dtype in (("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")):
        cache, _, _ = filled(ops, rng, 3, 2, 64, 64, storage)
        cache.k[0, 0, 9] = 0.0
        cache.k[0, 0, 9, 0] = -float("inf")
        cache.k[1, 1, 20, 3] = float("nan")
        spoil(cache, 0, 50)
        spoil(cache, 2, 10)
        q = torch.rand((3, 4, 64), device="cuda").to(getattr(torch, {"f32": "float32", "bf16": "bfloat16"}[dtype])) + 0.1
        mass = torch.full((3, 2, 64), 2.0, device="cuda")
        ops.attention_weights(cache, q, ints([50, 40, 10]), mass, decay=0.0)
        got = host(mass)
        assert got[0, 0, 9] == 0 and np.isfinite(got[0]).all()
        assert np.allclose(got[0, :, :50].sum(-1), 2.0, atol=1e-4) and np.all(got[0, :, 50:] == 2)
        assert np.isfinite(got[1, 0]).all() and np.isnan(got[1, 1, :40]).all() and np.all(got[1, :, 40:] == 2)
        assert np.allclose(got[2, :, :10].sum(-1), 2.0, atol=1e-4) and np.all(got[2, :, 10:] == 2)
        ops.attention_weights(cache, q, ints([50, 40, 10]), mass, decay=0.0, window=15)
        got = host(mass)
        assert np.isfinite(got).all() and np.all(got[1, 1, :25] == 0)
        assert np.allclose(got[1, :, 25:40].sum(-1), 2.0, atol=1e-4)


# ---- eviction --------------------------------------------------------------------------------------
def kept_places(mass, length, keep, recent, sinks):
    if length <= keep:
        return list(range(max(length, 0)))
    m = np.where(np.isnan(mass), -np.inf, mass)
    middle = range(sinks, length - recent)
    rank = [(np.isnan(mass[j]), -m[j], j) for j in middle]
    best = [j for _, _, j in sorted(rank)[:keep - sinks - recent]]
    return sorted([*range(sinks), *best, *range(length - recent, length)])


def raw_parts(cache):
    return [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


def raw(cache):
    return [t.clone() for t in raw_parts(cache)]


def check_evict(ops, rng, storage, dim, kv_heads, slots, lengths, keep, recent=0, sinks=0, rows=None, to=None,
                to_rows=None, mass=None):
    torch = torch_()
    count, n_rows = len(lengths), len(lengths) + 1
    cache, _, _ = filled(ops, rng, n_rows, kv_heads, slots, dim, storage)
    before = raw(cache)
    m = (rng.random((n_rows, kv_heads, slots)) ** 3).astype(np.float32) if mass is None else mass(n_rows, kv_heads, slots)
    masses = tensor(m)
    use = list(range(count)) if rows is None else rows
    given = None if rows is None else ints(rows)
    target = None
    if to is not None:
        target = ops.KvCache.allocate(n_rows, kv_heads, to, dim, storage)
        old = raw(target)
        to_mass = torch.full((n_rows, kv_heads, to), 9.0, device="cuda")
        new, kept = ops.kv_evict(cache, masses, ints(lengths), keep, recent, sinks, rows=given, to=target,
                                 to_mass=to_mass, to_rows=None if to_rows is None else ints(to_rows))
        dest = list(range(count)) if to_rows is None else to_rows
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(raw(cache), before))
        assert torch.equal(masses.view(torch.int32), tensor(m).view(torch.int32))
    else:
        old = [t.clone() for t in before]
        new, kept = ops.kv_evict(cache, masses, ints(lengths), keep, recent, sinks, rows=given)
        target, to_mass, dest = cache, masses, use
        to = slots
    want_kept = np.full((count, kv_heads, keep), -1)
    want_new = np.zeros(count, int)
    want_mass = np.full((n_rows, kv_heads, to), 9.0, np.float32) if target is not cache else m.copy()
    want = [t.clone() for t in old]
    for s, length in enumerate(lengths):
        there = 0 <= dest[s] < n_rows and dest[s] not in dest[:s]
        length = min(max(length, 0), slots) if there and 0 <= use[s] < n_rows else 0
        want_new[s] = min(length, keep)
        if not there:
            continue
        for h in range(kv_heads):
            places = kept_places(m[use[s], h], length, keep, recent, sinks) if length else []
            want_kept[s, h, :len(places)] = places
            want_mass[dest[s], h, :len(places)] = m[use[s], h, places] if places else []
            want_mass[dest[s], h, len(places):] = 0
            for x, y in zip(want, before):
                if places:
                    x[dest[s], h, :len(places)] = y[use[s], h, torch.tensor(places, device="cuda")]
    assert np.array_equal(new.cpu().numpy(), want_new)
    assert np.array_equal(kept.cpu().numpy(), want_kept)
    assert np.array_equal(to_mass.cpu().numpy(), want_mass, equal_nan=True)
    for x, y in zip(raw(target), want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("storage", ["u4", "bf16", "f32"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("to", [None, 57])
def test_evict(ops, storage, dim, to):
    rng = np.random.default_rng(dim)
    check_evict(ops, rng, storage, dim, 3, 200, [200, 51, 50, 49, 0, 1, 130], 50, 8, 4, to=to)
    check_evict(ops, rng, storage, dim, 1, 90, [80, 90, 33], 33, 0, 0, rows=[2, 0, 3], to=to)
    check_evict(ops, rng, storage, dim, 2, 90, [80, 90, 33], 20, 16, 4, to=to)       # nothing by mass
    check_evict(ops, rng, storage, dim, 2, 40, [40, 7], 1, 0, 1, to=to)
    check_evict(ops, rng, storage, dim, 2, 40, [40, 7], 1, 0, 0, to=to)


@pytest.mark.parametrize("to", [None, 5000])
@pytest.mark.parametrize("slots,keep", [(4096, 4095), (4097, 1), (9000, 4500), (20000, 3001)])
def test_evict_long_rows(ops, to, slots, keep):
    rng = np.random.default_rng(slots)
    check_evict(ops, rng, "u4", 32, 2, slots, [slots, slots - 1], keep, min(keep // 3, 900), min(keep // 2, 3), to=to)
    check_evict(ops, rng, "bf16", 64, 1, slots, [slots], keep, 0, 0, to=to)


@pytest.mark.parametrize("to", [None, 300])
def test_evict_ties_signs_and_nan(ops, to):
    rng = np.random.default_rng(11)

    def few(*shape):
        return rng.choice(np.float32([0.0, -0.0, 1.0, 0.5, -2.0]), shape)

    def odd(*shape):
        m = rng.standard_normal(shape).astype(np.float32)
        m[rng.random(shape) < 0.3] = np.nan
        m[rng.random(shape) < 0.1] = np.inf
        m[rng.random(shape) < 0.1] = -np.inf
        m[rng.random(shape) < 0.1] = 1e-42
        return m

    def close(*shape):   # masses that differ in their last bits
        return (np.float32(1.0) + rng.integers(0, 4, shape).astype(np.float32) * np.float32(2.0 ** -23))

    for mass in (few, odd, close, lambda *shape: np.ones(shape, np.float32), lambda *shape: np.full(shape, np.nan, np.float32)):
        check_evict(ops, rng, "u4", 32, 2, 5000, [5000, 4999, 299], 300, 20, 4, to=to, mass=mass)


def test_evict_rows_named_twice_and_outside(ops):
    rng = np.random.default_rng(12)
    check_evict(ops, rng, "bf16", 64, 2, 60, [60, 50, 40, 30], 20, 4, 2, rows=[1, 1, -1, 5])
    check_evict(ops, rng, "bf16", 64, 2, 60, [60, 50, 40, 30], 20, 4, 2, rows=[1, 1, 0, 0], to=33, to_rows=[2, 3, 2, 0])
    check_evict(ops, rng, "u4", 64, 2, 60, [60, 50, 40, 99], 20, 4, 2, rows=[1, 7, 0, 3], to=33, to_rows=[9, 3, -1, 0])


# ---- large entries ---------------------------------------------------------------------------------
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 19, 2.0 ** 24, 2.0 ** 40, 2.0 ** 60])
@pytest.mark.parametrize("where", ["hidden", "light", "early"])
@pytest.mark.parametrize("dim", [64, 128])
def test_large_values_without_weight_leave_the_others_theirs(ops, dim, where, ratio):
    """Values far above the others at a key that only the last tokens see, at keys whose scores are far below the
    others', or in a first block of keys of which that holds, in front of many queries over 4 bits. Values count by
    their weight: `weighed` is the largest sum of weight |v| of a channel of the query's."""
    rng = np.random.default_rng(int(np.log2(ratio)) + dim)
    L, kv_heads, heads, tokens = 2100 if where == "hidden" else 700, 2, 16, 20
    k = rng.standard_normal((L, kv_heads, dim)).astype(np.float32)
    v = rng.standard_normal((L, kv_heads, dim)).astype(np.float32)
    q = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    keys = {"hidden": [L - 1], "light": [0, 50, 320], "early": list(range(64))}[where]
    v[keys] *= np.float32(ratio)
    if where != "hidden":
        q[..., 0], k[:, :, 0] = 12.0, 0.0
        k[keys, :, 0] = -45.0 * np.log2(ratio) / 40 * (dim / 64) ** 0.5   # weights of about 2^-1.3 / ratio^2.4
    cache, starts = ops.KvCache.allocate(1, kv_heads, L + 10, dim), ints([0, L])
    ops.kv_append(cache, tensor(k), tensor(v), ints([L]), starts=starts)
    k, v = (host(t) for t in ops.kv_read(cache, ints([L]), starts=starts, tokens=L))
    q = tensor(q, "bf16")
    qh = host(q)
    if where == "hidden":
        mass = torch_().zeros((1, kv_heads, L + 10), device="cuda")
        got = host(ops.attention_weights(cache, q, ints([L]), mass, starts=ints([0, tokens]), decay=0.0))
        added = np.zeros((kv_heads, L))
    else:
        own = ops.KvCache.allocate(tokens, kv_heads, 4, dim)
        got = host(ops.attention_shared(own, q, ints([0] * tokens), cache, L))
    for i in range(tokens):
        n = L - tokens + i + 1 if where == "hidden" else L
        for h in range(heads):
            kk, vv = (x[:n, h * kv_heads // heads] for x in (k, v))
            p = softmax(kk @ qh[i, h] * dim ** -0.5)
            weighed = (p @ np.abs(vv)).max()
            size = np.array([(np.abs(kk) @ np.abs(qh[i, h]) * dim ** -0.5)[p > 1e-3 * p.max()].max()])
            want = p @ vv
            tol = shared_bound(size, dim, n, weighed, want, "bf16", "u4")
            assert np.all(np.abs(got[i, h] - want) <= tol), (i, h, (np.abs(got[i, h] - want) / tol).max())
            if where == "hidden":
                added[h * kv_heads // heads, :n] += p
    if where == "hidden":
        assert np.abs(host(mass)[0, :, :L] - added).max() <= 1e-4 * added.max()


@pytest.mark.parametrize("ratio", [2.0 ** -30, 2.0 ** -16, 2.0 ** -8, 2.0 ** 8, 2.0 ** 30])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_of_very_different_sizes(ops, dim, ratio):
    """Keys far above or below the others of their tile, of scores that do not matter or do."""
    torch = torch_()
    rng = np.random.default_rng(dim)
    n, kv_heads, heads, count = 500, 2, 16, 20
    x = rng.standard_normal((2, n, kv_heads, dim)).astype(np.float32)
    x[0, ::37] *= np.float32(ratio)
    x[0, ::37] = -np.abs(x[0, ::37])                       # and far below the others' scores where they are large
    common = ops.KvCache.allocate(1, kv_heads, n, dim)
    ops.kv_append(common, tensor(x[0]), tensor(x[1]), ints([n]), starts=ints([0, n]))
    k, v = (host(t) for t in ops.kv_read(common, ints([n]), starts=ints([0, n]), tokens=n))
    own = ops.KvCache.allocate(count, kv_heads, 4, dim)
    q = torch.from_numpy(np.abs(rng.standard_normal((count, heads, dim))).astype(np.float32)).cuda().bfloat16()
    got, qh = host(ops.attention_shared(own, q, ints([0] * count), common, n)), host(q)
    for i in range(count):
        for h in range(heads):
            kk, vv = k[:, h * kv_heads // heads], v[:, h * kv_heads // heads]
            p = softmax(kk @ qh[i, h] * dim ** -0.5)
            size = np.array([(np.abs(kk) @ np.abs(qh[i, h]) * dim ** -0.5)[p > 1e-3 * p.max()].max()])
            tol = shared_bound(size, dim, n, np.abs(vv).max(), p @ vv, "bf16", "u4")
            assert np.all(np.abs(got[i, h] - p @ vv) <= tol), (i, h, (np.abs(got[i, h] - p @ vv) / tol).max())


# ---- places --------------------------------------------------------------------------------------
@pytest.mark.parametrize("storage", ["u4", "bf16"])
def test_queries_at_odd_places(ops, storage):
    """bf16 queries that 16-byte accesses cannot read give what aligned ones give, within the two kernels' errors."""
    torch = torch_()
    rng = np.random.default_rng(16)
    common, _, v = filled(ops, rng, 1, 2, 700, 64, storage)
    cache, _, _ = filled(ops, rng, 50, 2, 9, 64, "u4")
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn((50, 8 * 64 + 3), generator=g, device="cuda").bfloat16()
    lengths = ints(rng.integers(0, 10, 50))
    for at in (0, 1, 2):
        odd = wide[:, at:at + 512].unflatten(-1, (8, 64))
        straight = odd.contiguous()
        a = host(ops.attention_shared(cache, odd, lengths, common, 700))
        b = host(ops.attention_shared(cache, straight, lengths, common, 700))
        assert np.abs(a - b).max() <= 4 * 2.0 ** -8 * np.abs(v).max()
    long, _, lv = filled(ops, rng, 2, 2, 2100, 64, "u4")
    wide = torch.randn((40, 8 * 64 + 3), generator=g, device="cuda").bfloat16()
    masses = [torch.zeros((2, 2, 2100), device="cuda") for _ in range(2)]
    for q, mass in zip((wide[:, 1:513].unflatten(-1, (8, 64)), wide[:, 1:513].unflatten(-1, (8, 64)).contiguous()), masses):
        ops.attention_weights(long, q, ints([2100, 1500]), mass, starts=ints([0, 20, 40]), decay=0.0)
    assert torch.allclose(*masses, rtol=1e-4, atol=1e-7)


def test_rows_without_tokens_fade(ops):
    torch = torch_()
    cache = ops.KvCache.allocate(3, 2, 50, 64)
    for decay in (0.0, 0.25):
        mass = torch.ones((3, 2, 50), device="cuda")
        q = torch.zeros((0, 4, 64), device="cuda")
        out = ops.attention_weights(cache, q, ints([30, 50]), mass, starts=ints([0, 0, 0]), rows=ints([2, 0]), decay=decay)
        assert out.shape == (0, 4, 64)
        got = host(mass)
        assert (got[1] == 1).all() and (got[0] == decay).all() and (got[2, :, :30] == decay).all() and (got[2, :, 30:] == 1).all()
    # no sequence at all
    ops.attention_weights(cache, q, ints([]), mass, starts=ints([0]))
    ops.attention_shared(cache, q, ints([]), cache, 7, starts=ints([0]))
    n, kept = ops.kv_evict(cache, mass, ints([]), 5)
    assert n.shape == (0,) and kept.shape == (0, 2, 5)
    with pytest.raises(Exception, match="keep"):
        ops.kv_evict(cache, mass, ints([3]), 51)
    with pytest.raises(Exception, match="keep"):
        ops.kv_evict(cache, mass, ints([3]), 2 ** 33)


@pytest.mark.parametrize("storage,dtype", [("bf16", "bf16"), ("u4", "bf16"), ("f32", "f32")])
def test_rows_far_into_a_cache(ops, storage, dtype):
    """Entries behind the 2^32nd: the last row of a cache is what the same row of a small cache is."""
    torch = torch_()
    rng = np.random.default_rng(17)
    slots, kv_heads, dim, heads = 65000, 4, 128, 16
    rows = {"f32": 140, "bf16": 140, "u4": 280}[storage]     # 4.7 to 9.3 thousand million entries
    far = ops.KvCache.allocate(rows, kv_heads, slots, dim, storage)
    near = ops.KvCache.allocate(2, kv_heads, slots, dim, storage)
    g = torch.Generator(device="cuda").manual_seed(5)
    for t in (near.k, near.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda") if storage == "u4" else torch.randn(t.shape, generator=g, device="cuda"))
    if storage == "u4":
        for t in (near.k_scale, near.v_scale):
            t.copy_(torch.rand(t.shape, generator=g, device="cuda") - torch.tensor([0.0, 4.0], device="cuda"))
    for x, y in zip(raw_parts(far), raw_parts(near)):
        x[rows - 1].copy_(y[1])
    q = torch.randn((20, heads, dim), generator=g, device="cuda").to(getattr(torch, {"f32": "float32", "bf16": "bfloat16"}[dtype]))
    lengths, some = ints([64999]), q[:1]
    masses = [torch.rand((r, kv_heads, slots), generator=g, device="cuda") for r in (2, rows)]
    masses[1][rows - 1].copy_(masses[0][1])
    results = []
    for cache, row, mass in ((near, 1, masses[0]), (far, rows - 1, masses[1])):
        a = ops.attention_weights(cache, some, lengths, mass, rows=ints([row]), decay=0.5)
        own = ops.KvCache.allocate(20, kv_heads, 8, dim, "u4")
        b = ops.attention_shared(own, q, ints([0] * 20), cache, 64999, prefix_row=row)
        c = ops.attention_shared(cache, some, lengths, near, 100, rows=ints([row]))
        n, kept = ops.kv_evict(cache, mass, lengths, 3000, 100, 4, rows=ints([row]))
        results.append([a, b, c, mass[row].clone(), n, kept] + [t[row, :, :3000].clone() for t in raw_parts(cache)])
    for x, y in zip(*results):
        assert torch.equal(x.view(torch.uint8) if x.is_floating_point() else x, y.view(torch.uint8) if y.is_floating_point() else y)


# ---- together --------------------------------------------------------------------------------------
@pytest.mark.parametrize("storage,dtype", [("u4", "bf16"), ("u4", "f32"), ("bf16", "bf16"), ("f32", "f32")])
def test_a_server_with_a_budget(ops, storage, dtype):
    """Prompts whose last queries vote are evicted into a small cache; decode steps behind a shared prefix
    append, attend, gather weight, and evict in place. Every step against 64 bits on what the cache holds."""
    torch = torch_()
    rng = np.random.default_rng(13)
    heads, kv_heads, dim, budget, slack = 4, 2, 64, 48, 6
    lengths = [150, 90, 31]
    prompts, _, _ = filled(ops, rng, 3, kv_heads, 150, dim, storage)
    system, sys_k, sys_v = filled(ops, rng, 1, kv_heads, 80, dim, storage)
    votes = torch.zeros((3, kv_heads, 150), device="cuda")
    q, _ = queries(rng, 3, heads, dim, dtype)
    ops.attention_weights(prompts, q, ints(lengths), votes, decay=0.0)
    cache = ops.KvCache.allocate(3, kv_heads, budget + slack, dim, storage)
    mass = torch.full((3, kv_heads, budget + slack), float("nan"), device="cuda")
    at, kept = ops.kv_evict(prompts, votes, ints(lengths), budget, 8, 4, to=cache, to_mass=mass)
    assert at.tolist() == [48, 48, 31]
    for step in range(2 * slack):
        at = at + 1
        new = torch.from_numpy(rng.standard_normal((2, 3, kv_heads, dim)).astype(np.float32)).cuda().to(q.dtype)
        ops.kv_append(cache, new[0], new[1], at)
        q, q64 = queries(rng, 3, heads, dim, dtype)
        n = at.tolist()
        k, v = (host(t).reshape(3, -1, kv_heads, dim) for t in ops.kv_read(
            cache, ints([budget + slack] * 3), starts=ints(np.arange(4) * (budget + slack)), tokens=3 * (budget + slack)))
        old = host(mass)
        own = host(ops.attention_weights(cache, q, at, mass))
        out = host(ops.attention_shared(cache, q, at, system, 80))
        gained = host(mass) - old
        for s in range(3):
            want, size = ref.attend(q64[s:s + 1], k[s, :n[s]], v[s, :n[s]], n[s] - 1, 0, 0, 0.125)
            assert np.all(np.abs(own[s] - want[0]) <= bound(size, dim, n[s], np.abs(v).max(), want, dtype)[0])
            want, size = shared_reference(q64[s:s + 1], sys_k[0], sys_v[0], k[s, :n[s]], v[s, :n[s]], n[s] - 1, 0.125)
            vmax = max(np.abs(v).max(), np.abs(sys_v).max())
            assert np.all(np.abs(out[s] - want[0]) <= shared_bound(size, dim, 80 + n[s], vmax, want, dtype, storage)[0])
            assert np.allclose(gained[s, :, :n[s]].sum(-1), heads // kv_heads, atol=1e-3)
            assert np.all(old[s, :, n[s] - 1] == 0) and np.all(host(mass)[s, :, n[s]:] == 0)
        if max(n) == budget + slack:
            at, kept = ops.kv_evict(cache, mass, at, budget, 8, 4)
            assert at.tolist() == [min(x, budget) for x in n]


def test_captured_and_on_other_streams(ops):
    """A decode step captured once and replayed with new inputs equals the calls; calls on a side stream too."""
    torch = torch_()
    rng = np.random.default_rng(14)
    cache, _, _ = filled(ops, rng, 8, 2, 2000, 64, "u4")
    system, _, _ = filled(ops, rng, 1, 2, 500, 64, "bf16")
    to = ops.KvCache.allocate(8, 2, 300, 64, "u4")
    q = torch.randn((8, 8, 64), device="cuda").bfloat16()
    lengths = ints(rng.integers(500, 2000, 8))
    mass, to_mass = torch.rand((8, 2, 2000), device="cuda"), torch.zeros((8, 2, 300), device="cuda")

    def step(stream=None):
        new = torch.zeros_like(mass) if stream is None else None
        if new is None:
            with torch.cuda.stream(stream):
                new = torch.zeros_like(mass)
        a = ops.attention_shared(cache, q, lengths, system, 500, stream=stream)
        b = ops.attention_weights(cache, q, lengths, new, previous=mass, decay=0.5, stream=stream)
        n, kept = ops.kv_evict(cache, new, lengths, 250, 20, 4, to=to, to_mass=to_mass, stream=stream)
        return a, b, new, n, kept, to_mass.clone() if stream is None else to_mass

    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        lengths.copy_(torch.randint(200, 2000, (8,), generator=g, device="cuda", dtype=torch.int32))
        graph.replay()
        want = [t.clone() for t in held]
        again = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, again))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        third = step(side)
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, third))
