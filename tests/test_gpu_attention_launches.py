"""Attention of more workgroups than a launch holds (2^24 of 256 threads) is
refused, on an MI355X: nothing is written."""
from __future__ import annotations

import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [4, 8])
@pytest.mark.parametrize("batch,heads,dtype", [(65536, 256, torch.bfloat16),
                                               (65537, 256, torch.bfloat16),
                                               ((1 << 24) + 16, 1, torch.float32)])
def test_calls_of_too_many_workgroups(gpu, fmt, batch, heads, dtype):
    """A token of one key a request, a workgroup a request and K/V head; the rows
    lie on each other, which no call that goes ahead would find in order."""
    say("attention of too many workgroups", fmt, batch, heads)
    shape = (hb.kv_cache_shape if fmt == 4 else hb.kv8_cache_shape)(1, heads, 32, 64)
    cache = torch.zeros(shape, dtype=torch.uint8, device=DEV)
    q = torch.ones((1, 1, 64), dtype=dtype, device=DEV).expand(batch, heads, 64)
    out = torch.full((1, 1, 64), 7.0, dtype=dtype, device=DEV)
    kw = dict(q=q, out=out.expand(batch, heads, 64), cache=cache,
              table=torch.zeros((batch, 1), dtype=torch.int32, device=DEV),
              cu=torch.arange(batch + 1, dtype=torch.int32, device=DEV),
              kv_lens=torch.ones(batch, dtype=torch.int32, device=DEV), max_new=1, max_kv=1,
              scale=1.0, ctx=gpu)
    with pytest.raises(hb.HbError, match="attention launch"):
        (hb.kv_attention if fmt == 4 else hb.kv8_attention)(**kw)
    assert bool((out == 7).all())
