"""Calls of the cache rows' largest sizes, without a GPU."""
from __future__ import annotations

import pytest

import hotarubi_amd as hb


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_largest_calls(dim):
    """tokens * heads and heads up to what is documented."""
    lib, at = hb.lib(), 1 << 20

    def reply(fn, tokens, heads, page=64):
        desc = hb.KV_ROWS_DESC.pack(at, 1, heads, page, dim, at, at, heads * dim, dim, heads * dim,
                                    dim, at, hb.HB_TYPE_F16, tokens)
        assert fn(None, desc) == hb.HB_EINVAL
        return hb.last_error()

    for fn, most in ((lib.hb_kv8_append, 1 << 28), (lib.hb_kv8_read, 1 << 28),
                     (lib.hb_kv_append, 1 << 31), (lib.hb_kv_read, 1 << 31)):
        for heads in (1, 8, 4095, 1 << 20, (1 << 23) + 1, (1 << 24) - 1):
            tokens = (most - 1) // heads
            assert "null context" in reply(fn, tokens, heads, 32), (heads, tokens)
            assert f"{tokens + 1} tokens of {heads} heads in one call" in \
                reply(fn, tokens + 1, heads, 32), (heads, tokens)
        assert "1 tokens of 16777216 heads in one call" in reply(fn, 1, 1 << 24, 32)
