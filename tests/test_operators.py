"""The serving operators without a GPU: their refusals, found from the host's arguments alone, and
the 64-bit reference's own properties."""
import ctypes

import numpy as np
import pytest

from basalt_b200 import _lib
import operator_reference as ref


def cache(**change):
    c = _lib.KvCacheStruct()
    c.storage, c.rows, c.kv_heads, c.slots, c.head_dim = _lib.DTYPE_U4, 2, 2, 16, 64
    c.k = c.v = c.k_scale = c.v_scale = 256
    for name, value in change.items():
        setattr(c, name, value)
    return c


def batch(**change):
    s = _lib.SequencesStruct()
    s.count, s.tokens, s.lengths = 2, 2, 256
    for name, value in change.items():
        setattr(s, name, value)
    return s


def spec(**change):
    a = _lib.AttentionSpecStruct()
    a.heads, a.kv_heads, a.head_dim, a.dtype, a.scale = 4, 2, 64, _lib.DTYPE_F32, 0.125
    for name, value in change.items():
        setattr(a, name, value)
    return a


def cached(c=None, s=None, a=None, q=256, q_stride=256, out=256, out_stride=256, ws=None, n=0):
    return _lib.load().bst_attention_cached(0, None, c or cache(), s or batch(), a or spec(), q,
                                            q_stride, out, out_stride, ws, n)


def packed(s=None, a=None, q=256, k=256, v=256, out=256, q_stride=256, k_stride=128):
    s = s or batch(starts=256, lengths=None)
    return _lib.load().bst_attention_packed(0, None, s, a or spec(), q, q_stride, k, k_stride, v,
                                            128, out, 256, None, 0)


@pytest.mark.parametrize("change,status", [
    ({"storage": 7}, _lib.BST_INVALID), ({"head_dim": 48}, _lib.BST_UNSUPPORTED),
    ({"rows": 0}, _lib.BST_SHAPE), ({"slots": -1}, _lib.BST_SHAPE), ({"k": None}, _lib.BST_INVALID),
    ({"k_scale": None}, _lib.BST_INVALID), ({"v": 264}, _lib.BST_INVALID)])
def test_caches_are_checked(change, status):
    lib = _lib.load()
    assert lib.bst_kv_append(0, None, cache(**change), batch(), 256, 128, 256, 128,
                             _lib.DTYPE_F32) == status
    assert "kv_append" in _lib.last_error()
    assert lib.bst_kv_read(0, None, cache(**change), batch(), 256, 128, 256, 128,
                           _lib.DTYPE_F32) == status
    assert cached(c=cache(**change)) == status


@pytest.mark.parametrize("change,status", [
    ({"count": -1}, _lib.BST_SHAPE), ({"tokens": -1}, _lib.BST_SHAPE),
    ({"lengths": None}, _lib.BST_INVALID), ({"tokens": 3}, _lib.BST_SHAPE)])
def test_batches_are_checked(change, status):
    assert _lib.load().bst_kv_append(0, None, cache(), batch(**change), 256, 128, 256, 128,
                                     _lib.DTYPE_F32) == status
    assert cached(s=batch(**change)) == status


@pytest.mark.parametrize("change,status", [
    ({"heads": 3}, _lib.BST_SHAPE), ({"kv_heads": 0}, _lib.BST_SHAPE),
    ({"dtype": _lib.DTYPE_U4}, _lib.BST_INVALID), ({"window": -1}, _lib.BST_INVALID),
    ({"sinks": -1}, _lib.BST_INVALID), ({"scale": float("nan")}, _lib.BST_INVALID),
    ({"head_dim": 80}, _lib.BST_UNSUPPORTED), ({"reserved": 1}, _lib.BST_INVALID)])
def test_attention_specs_are_checked(change, status):
    assert cached(a=spec(**change)) == status
    assert packed(a=spec(**change)) == status


def test_attention_arguments_are_checked():
    assert cached(a=spec(kv_heads=4)) == _lib.BST_SHAPE            # not the cache's
    assert cached(q=None) == _lib.BST_INVALID
    assert cached(q_stride=255) == _lib.BST_SHAPE
    assert cached(out=258) == _lib.BST_INVALID
    assert cached(c=cache(storage=_lib.DTYPE_F32), s=batch(starts=256)) == _lib.BST_UNSUPPORTED
    assert packed(s=batch(lengths=None)) == _lib.BST_INVALID       # no starts
    assert packed(s=batch(starts=256)) == _lib.BST_INVALID         # lengths given
    assert packed(k=None) == _lib.BST_INVALID
    assert packed(k_stride=127) == _lib.BST_SHAPE
    many = 1 << 29
    assert packed(s=batch(starts=256, lengths=None, tokens=many)) == _lib.BST_SHAPE
    assert cached(s=batch(count=many, tokens=many)) == _lib.BST_SHAPE
    size = ctypes.c_int64(0)
    assert _lib.load().bst_attention_cached_workspace(cache(), batch(), spec(),
                                                      None) == _lib.BST_INVALID
    assert _lib.load().bst_attention_cached_workspace(cache(), batch(), spec(), size) == 0
    if size.value:
        assert cached(ws=None) == _lib.BST_SHAPE
        assert cached(ws=256, n=size.value - 1) == _lib.BST_SHAPE


@pytest.mark.parametrize("name", ["rows", "starts", "lengths"])
def test_index_arrays_are_aligned(name):
    s = batch(**{name: 258})
    assert _lib.load().bst_kv_append(0, None, cache(), s, 256, 128, 256, 128,
                                     _lib.DTYPE_F32) == _lib.BST_INVALID
    assert cached(s=s) == _lib.BST_INVALID
    if name == "starts":
        assert packed(s=batch(starts=257, lengths=None)) == _lib.BST_INVALID


@pytest.mark.parametrize("name", ["temperatures", "top_ps", "min_ps", "top_ks"])
def test_per_row_settings_are_aligned(name):
    p = _lib.SamplingStruct()
    setattr(p, name, 257)
    assert _lib.load().bst_sample_tokens(0, None, 256, _lib.DTYPE_F32, 2, 10, 10, p, 256,
                                         256) == _lib.BST_INVALID
    assert "aligned" in _lib.last_error()


def test_slots_are_counted_in_32_bits():
    for slots in (2 ** 31 - 1, 2 ** 31 - 65536):
        assert cached(c=cache(slots=slots)) == _lib.BST_SHAPE
        assert _lib.load().bst_kv_read(0, None, cache(slots=slots), batch(), 256, 128, 256, 128,
                                       _lib.DTYPE_F32) == _lib.BST_SHAPE


def test_empty_batches_are_no_work():
    assert cached(s=batch(count=0, tokens=0, lengths=None), q=None, out=None) == _lib.BST_OK
    assert packed(s=batch(count=0, tokens=0, starts=256, lengths=None), q=None) == _lib.BST_OK


@pytest.mark.parametrize("change,status", [
    ({"dtype": 5}, _lib.BST_INVALID), ({"rows": -1}, _lib.BST_SHAPE),
    ({"rows": (1 << 27) + 1}, _lib.BST_SHAPE), ({"vocabulary": 0}, _lib.BST_SHAPE),
    ({"vocabulary": (1 << 20) + 1, "stride": 1 << 21}, _lib.BST_SHAPE), ({"stride": 9}, _lib.BST_SHAPE),
    ({"logits": None}, _lib.BST_INVALID), ({"logits": 258}, _lib.BST_INVALID),
    ({"uniforms": 260}, _lib.BST_INVALID), ({"tokens": None}, _lib.BST_INVALID),
    ({"sampling": None}, _lib.BST_INVALID)])
def test_sampling_arguments_are_checked(change, status):
    p = dict(logits=256, dtype=_lib.DTYPE_F32, rows=2, vocabulary=10, stride=10,
             sampling=_lib.SamplingStruct(), uniforms=256, tokens=256)
    p.update(change)
    assert _lib.load().bst_sample_tokens(0, None, p["logits"], p["dtype"], p["rows"],
                                         p["vocabulary"], p["stride"], p["sampling"],
                                         p["uniforms"], p["tokens"]) == status


def test_python_refusals_name_the_argument():
    import torch

    from basalt_b200 import IllegalArgumentException, operators

    k = torch.zeros((1, 2, 8, 64))
    with pytest.raises(IllegalArgumentException, match="k is on cpu|expected"):
        operators.sample_tokens(torch.zeros((2, 4)), torch.zeros(2, dtype=torch.float64))
    with pytest.raises(IllegalArgumentException, match="scales"):
        operators.KvCache(k.to(torch.uint8), k.to(torch.uint8))
    with pytest.raises(IllegalArgumentException):
        operators.KvCache(k, k[:, :1])


def test_reference_codes_stay_in_range_and_half_a_step_away():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 3, 64)).astype(np.float32) * 10.0 ** rng.integers(-6, 6, (50, 3, 1))
    codes, step, low, values = ref.quantise(x)
    half = np.repeat(step, 32, -1) / 2
    # the quotient is rounded in double: half a step and a few units of 2^-52 of the group's size
    size = np.repeat(np.abs(low) + 16 * step, 32, -1)
    assert np.all(np.abs(values - x) <= half + size * 2.0 ** -50)
    assert codes.shape == (50, 3, 32)


def test_reference_draw_known_answers():
    x = [1.0, 3.0, 3.0, -np.inf, np.nan]
    assert ref.draw_token(x, 0.9, 0.0, 0, 1.0, 0.0)[0] == 1        # greedy: the first largest
    assert ref.draw_token(x, 0.0, 1.0, 0, 1.0, 0.0)[0] == 0
    assert ref.draw_token(x, 0.99, 1.0, 0, 1.0, 0.0)[0] == 2
    assert ref.draw_token(x, 0.99, 1.0, 1, 1.0, 0.0)[0] == 1       # ties: lowest index
    assert ref.draw_token([-np.inf] * 3, 0.5, 1.0, 0, 1.0, 0.0)[0] == -1


def test_specs_with_a_window_or_a_4_bit_cache():
    from basalt_b200 import ModelSpec

    def create(spec):
        s, h = spec.struct(), ctypes.c_uint64(0)
        return _lib.load().bst_engine_create(s, 10 ** 6, ctypes.byref(h))

    decoder = ("padded_decoder", 10, 8, 64, 1, 2, 32)
    assert create(ModelSpec(*decoder, attention_window=-1)) == _lib.BST_INVALID
    assert create(ModelSpec(*decoder, attention_sinks=-1)) == _lib.BST_INVALID
    assert create(ModelSpec(*decoder, weight_dtype="u4")) == _lib.BST_INVALID
    assert create(ModelSpec("last_token", 5, 3, attention_window=2)) == _lib.BST_INVALID
    assert create(ModelSpec("last_token", 5, 3, kv_dtype="u4")) == _lib.BST_INVALID
    # accepted specs get as far as the device, which does not exist
    assert create(ModelSpec(*decoder, kv_dtype="u4", attention_window=3,
                            attention_sinks=1)) == _lib.BST_UNSUPPORTED
