"""Drafts over the 8-bit cache on an MI355X: tokens that are written and then
dropped.  The reference is test_gpu_kv8's; no tolerance, stored values are whole
codes times a power of two."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, TYPES, ints, say
from test_gpu_kv8 import Reference, rows_of
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_taken_back(gpu, dtype, dim):
    """A request whose length is taken back within a block (drafts that were not
    accepted) goes on with the scale that the dropped tokens brought; its earlier
    tokens stay as they were rounded to it.  At a block's first token the block
    begins anew."""
    say("tokens taken back", dtype, dim)
    rng = np.random.default_rng(dim)
    cache = torch.zeros(hb.kv8_cache_shape(2, 3, 64, dim), dtype=torch.uint8, device=DEV)
    ref = Reference(2, 3, 64, dim)
    length = 0
    # (tokens, of this size, of which so many stay)
    for new, size, stay in ((9, 1.0, 9), (4, 3.0**6, 1), (5, 1.0, 5), (3, 3.0**9, 0), (1, 1.0, 1),
                            (30, 0.01, 16), (8, 50.0, 0), (40, 1e-3, 40)):
        slots = np.arange(length, length + new)
        k, v = (rows_of(rng, (new, 3, dim), dtype) * size for _ in range(2))
        hb.kv8_append(k=k, v=v, slots=ints(slots), cache=cache, ctx=gpu)
        ref.append(k.double().cpu().numpy(), v.double().cpu().numpy(), slots)
        length += stay
        ref.check(cache, np.arange(length), gpu)
    assert length == 72
