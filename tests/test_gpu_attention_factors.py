"""Attention on an MI355X where what multiplies a query, a key or their product
is at an end of its range: every score fits fp32, though the parts of its
product, the scale times log2 e or scale / softcap do not.  Against the plain
64-bit implementations and tolerances of test_gpu_kv8 and test_gpu_kv."""
from __future__ import annotations

import math

import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, TYPES, ints, say
from test_gpu_kv import build as build4, check as check4
from test_gpu_kv8 import check, ramp
from test_gpu_kv8_large_queries import CASES, make, scaled
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

LARGEST = 1.6 * 2.0**127  # times log2 e past fp32


@pytest.mark.parametrize("way,dtype", CASES)
@pytest.mark.parametrize("byte,scale", [(246, 512.0), (246, LARGEST), (130, LARGEST),
                                        (130, -LARGEST), (127, 2.0**127)])
def test_zero_queries_under_large_factors(gpu, way, dtype, byte, scale):
    """Scores of 0, whatever they are multiplied by."""
    say("zero queries", way, dtype, byte, scale)
    s = scaled(make(way, dtype, 64, byte), 0.0)
    check(gpu, s, scale=scale)
    check(gpu, s, scale=scale, cap=5.0, window=50, sinks=4)


@pytest.mark.parametrize("way,dtype", CASES)
def test_largest_scale(gpu, way, dtype):
    """Scores of a few units from products of 2^-125."""
    say("largest scale", way, dtype)
    s = scaled(make(way, dtype, 64, 10), 2.0**-19)
    check(gpu, s, scale=LARGEST)
    check(gpu, s, scale=LARGEST, cap=3.0)


@pytest.mark.parametrize("way,dtype", CASES)
@pytest.mark.parametrize("scale", [2.0**-30, 2.0**-40, 2.0**-126, 2.0**-149])
def test_small_factors_and_hidden_keys(gpu, way, dtype, scale):
    """Factors below what fp32 has: every visible key weighs the same, hidden
    ones nothing."""
    say("small factors", way, dtype, scale)
    s = make(way, dtype, 64, 10)
    check(gpu, s, scale=scale)
    check(gpu, s, scale=-scale, window=50, sinks=4)
    check(gpu, s, scale=scale, window=50, cap=2.0**40)


@pytest.mark.parametrize("way,dtype", CASES)
def test_half_queries_between_the_ends(gpu, way, dtype):
    """Scale and scale byte each past where their product is taken in one."""
    say("between the ends", way, dtype)
    for byte in (10, 96, 97, 157, 158, 246):
        s = make(way, dtype, 64, byte)
        check(gpu, s, scale=2.0 ** (127 - byte) / 5000)
        check(gpu, s, scale=2.0 ** (127 - byte) / 5000, cap=4.0)


def pair(fmt, dtype, new, page=64):
    """A request of `page` keys, whose first is x and whose others are -x, their
    values 1 and -1 (whole codes of both formats), and `new` rows of x."""
    shape = (page, 1, 64)
    sign = torch.where(torch.arange(page, device=DEV) == 0, 1.0, -1.0)[:, None, None]
    rows = (sign * torch.ones(shape, device=DEV)).to(dtype).contiguous()
    cache = torch.zeros((hb.kv_cache_shape if fmt == 4 else hb.kv8_cache_shape)(1, 1, page, 64),
                        dtype=torch.uint8, device=DEV)
    (hb.kv_append if fmt == 4 else hb.kv8_append)(
        k=rows, v=rows, slots=torch.arange(page, dtype=torch.int32, device=DEV), cache=cache)
    q = torch.ones((new, 1, 64), device=DEV).to(dtype)
    out = torch.full_like(q, 7.0)
    # (a prefix of all keys: every row sees them)
    kw = dict(q=q, out=out, cache=cache, table=ints([[0]]), cu=ints([0, new]),
              kv_lens=ints([page]), prefix=ints([page]), max_new=new, max_kv=page)
    return (hb.kv_attention if fmt == 4 else hb.kv8_attention), kw


@pytest.mark.parametrize("fmt", [4, 8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 64])
def test_caps_far_from_the_scale(gpu, fmt, dtype, new):
    """scale / softcap past fp32 either way."""
    say("caps far from the scale", fmt, dtype, new)
    attention, kw = pair(fmt, dtype, new)
    mean = (1 - 63) / 64
    near = dict(rtol=2.0**-7, atol=0)
    # scores of +-2^36 under a cap of 2^50: the largest takes all
    big = dict(kw, q=kw["q"] * 2.0**10 if dtype is F16 else kw["q"] * 2.0**120)
    scale = 2.0**20 if dtype is F16 else 2.0**-90
    attention(ctx=gpu, scale=scale, softcap=2.0**50, **big)
    assert bool((kw["out"] == 1).all())
    attention(ctx=gpu, scale=-scale, softcap=2.0**50, **big)
    torch.testing.assert_close(kw["out"], torch.full_like(kw["out"], -1.0), **near)
    # scores of 0 and of nothing but a sign
    zero = dict(kw, q=kw["q"] * 0)
    for scale, cap in ((2.0**100, 2.0**-50), (2.0**127, 0.5), (2.0**-149, 2.0**60)):
        attention(ctx=gpu, scale=scale, softcap=cap, **zero)
        torch.testing.assert_close(kw["out"], torch.full_like(kw["out"], mean), **near)
    # +-32 once capped: e^-64 for the others, and a weight p that is no power of two,
    # so p (1 / p), whose quotient and product are rounded by 2^-24 each
    attention(ctx=gpu, scale=2.0**100, softcap=2.0**5, **kw)
    assert bool(((kw["out"].double() - 1).abs() <= 2.0**-23 + 63 * math.exp(-64)).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("new", [1, 64])
def test_scores_that_only_their_cap_makes_small(gpu, dtype, new):
    """scale / softcap below fp32's smallest: tanh's argument is a number all the
    same, and scores of 2^26 and -2^26 differ."""
    say("small caps' arguments", dtype, new)
    for fmt in (4, 8):
        attention, kw = pair(fmt, dtype, new)
        # q.k is +-2^126
        attention(ctx=gpu, scale=2.0**-100, softcap=2.0**55, **dict(kw, q=kw["q"] * 2.0**120))
        assert bool((kw["out"] == 1).all()), fmt


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests,hq,hk", [(ramp(2, 300, 90, 40), 16, 16), (ramp(4, 300, 256), 32, 32),
                                            (ramp(16, 500, 300, 30), 16, 2)])
def test_largest_scale_over_the_mxfp4_cache(gpu, dtype, requests, hq, hk):
    say("largest scale, MXFP4", dtype, hq)
    s = build4(torch.Generator(device=DEV).manual_seed(3), requests, 64, hk, 64, dtype, hq)
    check4(gpu, scaled(s, 0.0), scale=LARGEST)
    check4(gpu, scaled(s, 0.0), scale=-LARGEST, window=50)
    s["cache"][..., 32 * 64:33 * 64] = 20  # keys of 2^-107 and less
    check4(gpu, scaled(s, 2.0**-19), scale=LARGEST)
