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
