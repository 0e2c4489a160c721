"""The serving operators at the edges of their arguments, as far as the host decides."""
import ctypes

import pytest

from basalt_b200 import _lib
from test_operators import batch, cache, spec


def workspace(count, tokens, slots, heads, kv_heads, head_dim, starts=True, window=0,
              dtype=_lib.DTYPE_BF16):
    size = ctypes.c_int64(-1)
    c = cache(rows=count, kv_heads=kv_heads, slots=slots, head_dim=head_dim)
    s = batch(count=count, tokens=tokens, starts=256 if starts else None)
    a = spec(heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, window=window)
    assert _lib.load().bst_attention_cached_workspace(c, s, a, size) == _lib.BST_OK
    return size.value


@pytest.mark.parametrize("count,tokens,slots,most", [
    (2, 8192, 131072, 0),            # later chunks of prompts: their tiles fill the card
    (2, 65536, 1 << 20, 0),
    (256, 1024, 131072, 128 << 20),  # a few drafted tokens of many sequences
    (4096, 4096, 1 << 20, 128 << 20),
    (3, 40, 1 << 20, 128 << 20)])
def test_the_workspace_of_many_tokens_stays_small(count, tokens, slots, most):
    assert workspace(count, tokens, slots, 32, 8, 128) <= most
    assert workspace(count, tokens, slots, 32, 8, 128, dtype=_lib.DTYPE_F32) <= most


def test_few_tokens_over_long_caches_are_split():
    row = 32 * 130 * 4                                        # bytes of a token's split, 32 heads
    assert workspace(24, 96, 16384, 32, 8, 128) == 4 * 96 * row
    assert workspace(256, 256, 131072, 32, 8, 128, starts=False) >= 16 * 256 * row
    assert workspace(1, 1, 131072, 32, 8, 128, starts=False) == 148 * 2 // 8 * row


def test_outputs_do_not_overlap_what_is_read():
    """Tokens of 4 heads of 64 float32 (1024 bytes), keys and values of 2 heads (512 bytes)."""
    lib, at = _lib.load(), 1 << 20

    def packed(out, out_stride=256, q=at, q_stride=256, k=at + (1 << 16), v=at + (2 << 16), stride=128,
               tokens=2):
        # far pointers pass the check and stop at the workspace, which is missing
        return lib.bst_attention_packed(0, None, batch(tokens=tokens, starts=256, lengths=None), spec(), q,
                                        q_stride, k, stride, v, stride, out, out_stride, None, 0)

    def cached(out, out_stride=256, q_stride=256):
        return lib.bst_attention_cached(0, None, cache(rows=2, slots=1 << 20), batch(), spec(), at,
                                        q_stride, out, out_stride, None, 0)

    assert packed(at + (3 << 16)) == _lib.BST_SHAPE
    assert packed(at + 2048) == _lib.BST_SHAPE                         # right behind q
    for out in (at, at + 4, at + 2044, at - 2044, at + (1 << 16), at + (1 << 16) + 1020, at + (2 << 16)):
        assert packed(out) == _lib.BST_INVALID
        assert "overlap" in _lib.last_error()
    # slices of one tensor: q at 0, keys at 256, values at 384, outputs at 512 of 768 elements
    slices = dict(q_stride=768, k=at + 1024, v=at + 1536, stride=768, out_stride=768)
    assert packed(at + 2048, **slices) == _lib.BST_SHAPE
    for out in (at + 2044, at + 2052, at, at + 1536, at - 1020):
        assert packed(out, **slices) == _lib.BST_INVALID
    assert packed(at + 2048, **{**slices, "out_stride": 769}) == _lib.BST_INVALID
    assert packed(at + 2048, tokens=1, **{**slices, "out_stride": 769}) == _lib.BST_SHAPE
    assert cached(at) == cached(at + 2048) == _lib.BST_SHAPE           # q itself; behind it
    assert cached(at + 4) == cached(at, 260) == cached(at + 1024) == _lib.BST_INVALID


@pytest.mark.parametrize("given,want", [(2 ** 32 + 5, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (7, 7), (0, 0),
                                        (-2 ** 32 + 5, -2 ** 31), (-1, -1)])
def test_counts_beyond_32_bits_keep_their_meaning(given, want):
    """A window or a top_k wider than anything, not what its lower 32 bits say."""
    import torch

    from basalt_b200 import ModelSpec, operators

    operators._torch()
    a = operators._spec(torch.zeros((1, 2, 64)), 1, given, given, None)
    assert (a.window, a.sinks) == (want, want)
    assert operators._setting(torch.device("cpu"), 1, "top_k", given, "torch.int32") == (want, None)
    s = ModelSpec("padded_decoder", 10, 8, 64, 1, 2, 32, attention_window=given,
                  attention_sinks=given).struct()
    assert (s.attention_window, s.attention_sinks) == (want, want)
