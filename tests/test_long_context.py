"""Shared prefixes, weights and eviction without a GPU: refusals, found from the host's arguments alone."""
import ctypes

import pytest

from basalt_b200 import _lib
from test_operators import batch, cache, spec

FAR = 1 << 40


def shared(c=None, s=None, a=None, p=None, row=0, length=10, q=256, q_stride=256, out=FAR, ws=None, n=0):
    return _lib.load().bst_attention_shared(0, None, c or cache(), s or batch(), a or spec(), p or cache(), row,
                                            length, q, q_stride, out, 256, ws, n)


def weights(c=None, s=None, a=None, q=256, out=FAR, previous=2 * FAR, decay=1.0, mass=3 * FAR, ws=None, n=0):
    return _lib.load().bst_attention_weights(0, None, c or cache(), s or batch(), a or spec(), q, 256, out, 256,
                                             previous, decay, mass, ws, n)


def evict(c=None, s=None, mass=2 * FAR, keep=8, recent=2, sinks=1, to=None, to_rows=None, to_mass=3 * FAR,
          lengths=4 * FAR, kept=5 * FAR):
    return _lib.load().bst_kv_evict(0, None, c or cache(), s or batch(), mass, keep, recent, sinks, to, to_rows,
                                    to_mass, lengths, kept)


@pytest.mark.parametrize("change,status", [
    ({"storage": 7}, _lib.BST_INVALID), ({"head_dim": 48}, _lib.BST_UNSUPPORTED),
    ({"rows": 0}, _lib.BST_SHAPE), ({"k": None}, _lib.BST_INVALID), ({"v_scale": 260}, _lib.BST_INVALID)])
def test_caches_are_checked(change, status):
    assert shared(c=cache(**change)) == status
    assert shared(p=cache(**change)) == status
    assert "prefix" in _lib.last_error()
    assert weights(c=cache(**change)) == status
    assert evict(c=cache(**change)) == status
    assert evict(to=cache(**change)) == status
    assert "to:" in _lib.last_error()


@pytest.mark.parametrize("change,status", [
    ({"count": -1}, _lib.BST_SHAPE), ({"lengths": None}, _lib.BST_INVALID), ({"tokens": 3}, _lib.BST_SHAPE),
    ({"lengths": 258}, _lib.BST_INVALID)])
def test_batches_are_checked(change, status):
    assert shared(s=batch(**change)) == status
    assert weights(s=batch(**change)) == status
    assert evict(s=batch(**change)) == status


def test_prefixes_are_checked():
    assert shared() == _lib.BST_SHAPE and "workspace" in _lib.last_error()
    for bad in (dict(row=-1), dict(row=2), dict(length=-1), dict(length=17)):
        assert shared(**bad) == _lib.BST_SHAPE and "row" in _lib.last_error()
    assert shared(p=cache(kv_heads=1)) == _lib.BST_SHAPE
    assert shared(p=cache(head_dim=32)) == _lib.BST_SHAPE
    assert shared(a=spec(window=5)) == _lib.BST_UNSUPPORTED
    assert shared(a=spec(sinks=5)) == _lib.BST_UNSUPPORTED
    assert shared(c=cache(storage=_lib.DTYPE_BF16), s=batch(starts=256)) == _lib.BST_UNSUPPORTED
    assert shared(out=None) == _lib.BST_INVALID
    assert shared(out=260) == _lib.BST_INVALID and "overlap" in _lib.last_error()
    assert shared(out=256) == _lib.BST_SHAPE     # q itself
    assert shared(q_stride=255) == _lib.BST_SHAPE
    lib = _lib.load()
    assert lib.bst_attention_shared(0, None, cache(), batch(), spec(), None, 0, 1, 256, 256, FAR, 256, None,
                                    0) == _lib.BST_INVALID
    assert lib.bst_attention_shared_workspace(cache(), batch(), spec(), cache(), 0, 1, None) == _lib.BST_INVALID


def test_masses_are_checked():
    assert weights() == _lib.BST_SHAPE and "workspace" in _lib.last_error()
    for bad in (dict(decay=float("nan")), dict(decay=float("inf")), dict(decay=-0.5), dict(mass=None),
                dict(previous=None), dict(mass=FAR + 2), dict(previous=FAR + 1),
                dict(previous=3 * FAR + 4),           # neither mass itself nor apart from it
                dict(mass=FAR), dict(mass=256), dict(previous=FAR), dict(out=260)):
        assert weights(**bad) == _lib.BST_INVALID, bad
    assert weights(previous=None, decay=0.0) == _lib.BST_SHAPE
    assert weights(previous=3 * FAR) == _lib.BST_SHAPE
    assert weights(s=batch(count=0, tokens=0), mass=None) == _lib.BST_OK
    # more CTAs than a launch has
    assert weights(c=cache(rows=1, kv_heads=4096, slots=1 << 30), a=spec(heads=4096, kv_heads=4096),
                   s=batch(count=1, tokens=1), previous=None, decay=0.0,
                   mass=1 << 62, q=1 << 61, out=1 << 60) == _lib.BST_SHAPE


def test_the_workspace_of_weights_holds_the_scores():
    size = ctypes.c_int64(0)
    c = cache(rows=64, kv_heads=8, slots=8190, head_dim=128, storage=_lib.DTYPE_BF16)
    a = spec(heads=32, kv_heads=8, head_dim=128, dtype=_lib.DTYPE_BF16)
    assert _lib.load().bst_attention_weights_workspace(c, batch(count=64, tokens=64), a, size) == _lib.BST_OK
    assert 64 * 32 * 8192 * 4 <= size.value <= 64 * 32 * 8192 * 4 + (8 << 20)


def test_evictions_are_checked():
    other = cache(k=1 << 44, v=1 << 45, k_scale=1 << 46, v_scale=1 << 47)
    for bad, status in ((dict(keep=0), _lib.BST_SHAPE), (dict(keep=17), _lib.BST_SHAPE),
                        (dict(recent=-1), _lib.BST_SHAPE), (dict(sinks=-1), _lib.BST_SHAPE),
                        (dict(recent=6, sinks=3), _lib.BST_SHAPE), (dict(recent=2 ** 31 - 1, sinks=2), _lib.BST_SHAPE),
                        (dict(mass=None), _lib.BST_INVALID), (dict(to_mass=None), _lib.BST_INVALID),
                        (dict(lengths=None), _lib.BST_INVALID), (dict(kept=None), _lib.BST_INVALID),
                        (dict(kept=5 * FAR + 2), _lib.BST_INVALID), (dict(to_rows=256), _lib.BST_INVALID),
                        (dict(s=batch(starts=256)), _lib.BST_INVALID),
                        (dict(to=cache()), _lib.BST_INVALID),                       # the cache's own memory
                        (dict(to=cache(k=1 << 44, v=1 << 45, k_scale=1 << 46, v_scale=256)), _lib.BST_INVALID),
                        (dict(to_mass=2 * FAR + 4), _lib.BST_INVALID),
                        (dict(to=other, to_mass=2 * FAR), _lib.BST_INVALID),        # in place, but the keys are not
                        (dict(to=other, to_mass=1 << 44), _lib.BST_INVALID),
                        (dict(lengths=256), _lib.BST_INVALID),                      # the lengths that are read
                        (dict(kept=2 * FAR), _lib.BST_INVALID), (dict(kept=4 * FAR), _lib.BST_INVALID),
                        (dict(to=cache(kv_heads=1)), _lib.BST_SHAPE), (dict(to=cache(head_dim=32)), _lib.BST_SHAPE),
                        (dict(to=cache(storage=_lib.DTYPE_BF16)), _lib.BST_SHAPE),
                        (dict(to=cache(k=1 << 44, v=1 << 45, k_scale=1 << 46, v_scale=1 << 47, slots=7)), _lib.BST_SHAPE)):
        assert evict(**bad) == status, bad
        assert "kv_evict" in _lib.last_error()
    assert evict(s=batch(count=0, tokens=0)) == _lib.BST_OK
