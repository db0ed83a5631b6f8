"""Large queries on small keys over the 8-bit cache on an MI355X: a query times a
bare code passes fp32, a query times the key does not.  References and
tolerances are test_gpu_kv8's."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv import DEV, TYPES, say
from test_gpu_kv8 import build, check, ramp
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

#: requests, query heads, K/V heads
SIZES = {"splits": (ramp(2, 300, 90, 40), 16, 16), "rows": (ramp(4, 300, 256), 32, 32),
         "splits, joined": (ramp(12, 3000, 3, 70), 8, 1), "prompt": (ramp(16, 500, 300, 30), 16, 2)}
CASES = [(way, dtype) for way in SIZES for dtype in TYPES if (way, dtype) != ("prompt", F32)]


def make(way, dtype, dim, key_byte):
    requests, hq, hk = SIZES[way]
    s = build(torch.Generator(device=DEV).manual_seed(dim), requests, 64, hk, dim, dtype, hq)
    s["cache"][..., 64 * dim] = key_byte
    return s


def scaled(s, by):
    return dict(s, q=(s["q"].double() * by).to(s["q"].dtype))


@pytest.mark.parametrize("way,dtype", [c for c in CASES if c[1] is not F16])
@pytest.mark.parametrize("dim", [64, 256])
def test_large_queries_on_small_keys(gpu, way, dtype, dim):
    """Queries of 2^121 on keys of 2^-109 and less: bare codes times the query
    would pass fp32."""
    say("large queries", way, dtype, dim)
    s = scaled(make(way, dtype, dim, 10), 2.0**121)
    check(gpu, s, scale=2.0**-12 / dim, way=way.split(",")[0])
    check(gpu, s, scale=-(2.0**-12) / dim, cap=2.0, window=100, sinks=3)


@pytest.mark.parametrize("way,dtype", [c for c in CASES if c[1] is BF16])
def test_large_queries_on_keys_of_bytes_that_prompts_open(gpu, way, dtype):
    """The same with scales that prompts open, and large ones."""
    say("large queries, opened", way, dtype)
    for byte, size in ((64, 2.0**121), (96, 2.0**121), (190, 2.0**40)):
        s = scaled(make(way, dtype, 64, byte), size)
        check(gpu, s, scale=2.0 ** (127 - byte) / size / 4096)
