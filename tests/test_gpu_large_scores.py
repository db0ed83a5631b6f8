"""Attention over both caches on an MI355X with scores far past what a softmax
tells apart: the largest takes all, whatever its size, on every way."""
from __future__ import annotations

import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, TYPES, ints, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

#: requests of as many keys and new tokens, query heads (on one K/V head), the way
SIZES = {"splits": (1, 64, 1, 4, "splits"), "splits, joined": (2, 6000, 3, 4, "splits"),
         "rows": (60, 96, 64, 4, "rows"), "prompt": (60, 600, 256, 4, "prompt")}


def make(gpu, fmt, way, dtype, size):
    """A key of ones whose value is `size`, all others their negatives: a row's
    scores are plus and minus one number of 24 bits, which no product with log2 e
    holds exactly.  The call, its arguments and the sign of each row's number."""
    requests, keys, new, heads, kind = SIZES[way]
    page, columns = 96, -(-keys // 96)
    sign = torch.where(torch.arange(keys, device=DEV) == keys // 2, 1.0, -1.0)[:, None, None]
    k, v = (sign.expand(keys, 1, 64).to(dtype).contiguous() * x for x in (1, size))
    cache = torch.zeros((hb.kv_cache_shape if fmt == 4 else hb.kv8_cache_shape)(columns, 1, page, 64),
                        dtype=torch.uint8, device=DEV)
    (hb.kv_append if fmt == 4 else hb.kv8_append)(
        k=k, v=v, slots=torch.arange(keys, dtype=torch.int32, device=DEV), cache=cache, ctx=gpu)
    tokens = requests * new
    gen = torch.Generator(device=DEV).manual_seed(keys)
    q = torch.randn((tokens, heads, 64), generator=gen, device=DEV).to(dtype)
    q[q.double().sum(-1).abs() < 0.1] = 1.5
    table = torch.arange(columns, dtype=torch.int32, device=DEV).expand(requests, columns)
    kw = dict(q=q, out=torch.empty_like(q), cache=cache, table=table.contiguous(),
              kv_lens=ints([keys] * requests), cu=ints([i * new for i in range(requests + 1)]),
              prefix=ints([keys] * requests), max_new=new, max_kv=keys)
    tell = hb.kv_attention_way if fmt == 4 else hb.kv8_attention_way
    assert tell(scale=1.0, **kw)[0] == kind
    attention = hb.kv_attention if fmt == 4 else hb.kv8_attention
    return attention, kw, torch.sign(q.double().sum(-1, keepdim=True)).expand(q.shape)


def check(gpu, attention, kw, want, scales, size):
    for scale in scales:
        for side in (1, -1):
            kw["out"].fill_(7.0)
            attention(scale=side * scale, ctx=gpu, **kw)
            # (a value over its own sum; on one side of as many equal weights as there
            # are other keys)
            off = (kw["out"].double() / size - side * want).abs().max().item()
            assert off <= 2.0**-11, (scale, side, off)


@pytest.mark.parametrize("fmt", [4, 8])
@pytest.mark.parametrize("way,dtype", [(w, t) for w in SIZES for t in TYPES
                                       if (w, t) != ("prompt", F32)])
def test_the_largest_score_takes_all(gpu, fmt, way, dtype):
    say("large scores", fmt, way, dtype)
    scales = (2.0**14 / 3, 2.0**22 / 3, 2.0**30 / 3, 2.0**60 / 3, 2.0**100 / 3)
    check(gpu, *make(gpu, fmt, way, dtype, 1), scales, 1)


@pytest.mark.parametrize("fmt", [4, 8])
@pytest.mark.parametrize("way,dtype", [(w, t) for w in SIZES for t in (BF16, F32)
                                       if (w, t) != ("prompt", F32)])
def test_large_scores_over_large_values(gpu, fmt, way, dtype):
    """Values whose weighted sums would pass fp32, under scores of up to 2^29."""
    say("large scores over large values", fmt, way, dtype)
    size = 2.0**126
    check(gpu, *make(gpu, fmt, way, dtype, size), (2.0**14 / 3, 2.0**19 / 3, 2.0**25 / 3), size)
