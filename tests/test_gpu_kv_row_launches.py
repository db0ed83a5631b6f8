"""Cache rows of more workgroups than a launch holds (2^24 of 256 threads), on an
MI355X: the rows past the first launch's land where they should, runs across the
launches' border stay runs."""
from __future__ import annotations

import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, ints, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu


def test_mxfp4_rows_of_several_launches(gpu):
    """2^25 tokens of 8 heads of 256, 8 tokens of a head a workgroup: three
    launches.  All rows are one row (they lie on each other) and most slots none."""
    say("MXFP4 rows, several launches")
    heads, tokens, dim = 8, 1 << 25, 256
    border = ((1 << 24) - 1) // heads * 8
    assert 2 * border < tokens
    row = torch.randn((1, heads, dim), device=DEV).to(torch.bfloat16)
    slots = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    named = [0, 5, border - 1, border, border + 1, 2 * border - 1, 2 * border, tokens - 1]
    slots[named] = ints(list(range(len(named))))
    cache, want = (torch.zeros(hb.kv_cache_shape(2, heads, 32, dim), dtype=torch.uint8, device=DEV)
                   for _ in range(2))
    rows, few = row.expand(tokens, heads, dim), row.expand(len(named), heads, dim)
    hb.kv_append(k=rows, v=rows, slots=slots, cache=cache, ctx=gpu)
    hb.kv_append(k=few, v=few, slots=ints(list(range(len(named)))), cache=want, ctx=gpu)
    assert bool(want.any()) and torch.equal(cache, want)


def test_8_bit_rows_of_several_launches(gpu):
    """255 tokens of 2^20 + 1 heads of 256 out of the cache, 16 tokens of a head a
    workgroup: two launches.  The heads are all alike, and so are the rows that
    they are read into, which lie on each other."""
    say("8-bit rows, several launches")
    heads, tokens, dim = (1 << 20) + 1, 255, 256
    assert -(-tokens // 16) * heads >= 1 << 24 and tokens * heads < 1 << 28
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = [torch.randn((32, 1, dim), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2)]
    slots = torch.arange(32, dtype=torch.int32, device=DEV)
    outs = []
    for n in (heads, 1):
        cache = torch.zeros(hb.kv8_cache_shape(1, n, 32, dim), dtype=torch.uint8, device=DEV)
        k, v = (y.expand(32, n, dim) for y in x)
        hb.kv8_append(k=k, v=v, slots=slots, cache=cache, ctx=gpu)
        out = [torch.full((tokens, 1, dim), 7.0, dtype=torch.bfloat16, device=DEV)
               for _ in range(2)]
        hb.kv8_read(k=out[0].expand(tokens, n, dim), v=out[1].expand(tokens, n, dim),
                    slots=slots.repeat(8)[:tokens].flip(0).contiguous(), cache=cache, ctx=gpu)
        outs.append(out)
        del cache
    assert bool(outs[1][0].any()) and all(torch.equal(a, b) for a, b in zip(*outs))
