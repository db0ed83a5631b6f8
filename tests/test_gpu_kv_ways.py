"""Attention over the paged cache on every way of dividing its work, for every
type and head size that takes it: ordinary rows, scales of every kind, missing
pages, strides without alignment, bounds that are too small, and lengths that
make no sense.  Each test asserts the way its sizes are meant for, so that a
new line between the ways leaves none of them untested."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, HALF, TINY, build, ints, make_cache, say
from test_gpu_kv_edges import compare, memory_given_back, reference, set_scale  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def ramp(count, kv, new, prefix=0):
    """(keys, new tokens, prefix) of `count` requests, no two alike, the first
    of kv keys and new tokens."""
    return [(kv - i * kv // (2 * count), max(1, new - i * new // (2 * count)), max(0, prefix - i))
            for i in range(count)]


#: sizes, the way, 16-row tiles of a wave, splits (True: more than one)
SIZES = {
    "rows": (ramp(4, 300, 256), 32, 32, "rows", 1, False),
    "rows, two tiles": (ramp(24, 130, 60), 32, 8, "rows", 2, False),
    "rows, two tiles, D 128 in f16": (ramp(64, 170, 60), 16, 4, "rows", 2, False),
    "splits": (ramp(2, 300, 90, 40), 16, 16, "splits", 1, False),
    "splits, two tiles": (ramp(6, 340, 300), 8, 1, "splits", 2, False),
    "splits, joined": (ramp(12, 3000, 3, 70), 8, 1, "splits", 1, True),
    "splits, joined, two tiles": (ramp(3, 3000, 130), 8, 1, "splits", 2, True),
    "shares": (ramp(24, 12000, 2), 8, 2, "shares", 1, True),
    "shares, two tiles": (ramp(24, 12000, 6), 8, 2, "shares", 2, True),
    "prompt": (ramp(16, 500, 300, 30), 16, 2, "prompt", None, False),
}


def cases():
    for name in SIZES:
        for dim in (64, 128, 256):
            for dtype in TYPES:
                if "two tiles" in name and dim == 256:
                    continue
                if name == "rows, two tiles" and (dim, dtype) == (128, F16):
                    continue
                if name.endswith("D 128 in f16") and (dim, dtype) != (128, F16):
                    continue
                if name == "prompt" and dtype is F32:
                    continue
                yield pytest.param(name, dim, dtype, id=f"{name}-{dim}-{str(dtype)[6:]}")


def make(name, dim, dtype):
    requests, hq, hk = SIZES[name][:3]
    gen = torch.Generator(device=DEV).manual_seed(dim + len(name))
    if max(kv for kv, _, _ in requests) < 4000:
        return build(gen, requests, 64, hk, dim, dtype, hq)
    # long requests share their pages: a small cache
    cols = max(kv for kv, _, _ in requests) // 64 + 1
    cu = np.concatenate([[0], np.cumsum([n for _, n, _ in requests])])
    return dict(q=torch.randn((int(cu[-1]), hq, dim), generator=gen, device=DEV).to(dtype),
                cache=make_cache(gen, 96, hk, 64, dim),
                table=torch.randint(0, 96, (len(requests), cols), generator=gen, device=DEV,
                                    dtype=torch.int32),
                cu=ints(cu), kv_lens=ints([kv for kv, _, _ in requests]), prefix=None,
                max_new=max(n for _, n, _ in requests), max_kv=max(kv for kv, _, _ in requests))


def assert_way(name, s, window=0, cap=0.0):
    _, _, _, way, tiles, joined = SIZES[name]
    got = hb.kv_attention_way(q=s["q"], out=s["q"], cache=s["cache"], table=s["table"], cu=s["cu"],
                              kv_lens=s["kv_lens"], max_new=s["max_new"], max_kv=s["max_kv"],
                              scale=0.1, prefix=s["prefix"], window=window, softcap=cap)
    if tiles is None:
        tiles = 2 if s["q"].shape[-1] == 64 else 1
    assert (got[0], got[1], got[2] > 1) == (way, tiles, joined), got
    assert (got[3] > 0) == (joined or way == "prompt")


@pytest.mark.parametrize("name,dim,dtype", cases())
def test_rows_strides_and_missing_pages(gpu, name, dim, dtype):
    say("way", name, dim, dtype)
    s = make(name, dim, dtype)
    assert_way(name, s)
    compare(gpu, s)
    # q, out and table in wider tensors, aligned to their elements alone
    tokens, hq = s["q"].shape[:2]
    wide = torch.zeros((tokens, hq, dim + 3), dtype=dtype, device=DEV)
    wide[..., 3:] = s["q"]
    table = torch.zeros((s["table"].shape[0], s["table"].shape[1] + 5), dtype=torch.int32,
                        device=DEV)
    table[:, 2:-3] = s["table"]
    out = torch.full((hq, tokens, dim + 1), 7.0, dtype=dtype, device=DEV).transpose(0, 1)
    compare(gpu, dict(s, q=wide[..., 3:], table=table[:, 2:-3]), out=out[..., 1:])
    assert bool((out[..., 0] == 7).all())
    # entries that name no page, in the first, a middle and the last column
    table, last = s["table"].clone(), (int(s["kv_lens"][0]) - 1) // 64
    table[0, 0], table[0, last // 2], table[-1, 1] = -1, s["cache"].shape[0], -2**31
    table[1, last // 3] = 2**31 - 1
    compare(gpu, dict(s, table=table))


@pytest.mark.parametrize("name,dim,dtype", cases())
def test_scales_of_every_kind(gpu, name, dim, dtype):
    """V far outside f16's range and past what sums of weights hold, K outside
    f16's, tokens that are NaN, and any bytes past the requests' ends."""
    say("way, scales", name, dim, dtype)
    s = make(name, dim, dtype)
    for b in range(s["table"].shape[0]):  # past the end, where that page is the request's own
        total = int(s["kv_lens"][b])
        if total < 4000 and total % 64:
            s["cache"][s["table"][b, total // 64].long(), :, total % 64 // 32 + 1:] = 0xFF
    base = s["cache"].clone()
    lens = s["kv_lens"].tolist()
    for which, changes in ((3, [(0, 5, 90), (0, lens[0] - 40, 150)]), (3, [(1, 3, 252)]),
                           (3, [(0, lens[0] // 2, 240), (1, lens[1] // 3, 20)]),
                           (2, [(0, 7, 100), (1, 9, 60), (1, lens[1] // 2, 1)]),
                           (2, [(0, lens[0] - 2, 255)]), (3, [(1, lens[1] // 2, 254)])):
        s["cache"].copy_(base)
        for b, token, value in changes:
            set_scale(s, b, token, which, value)
        assert_way(name, s)
        compare(gpu, s)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompts_with_masks_caps_and_bounds_too_small(gpu, dtype, dim):
    """Windows, prefixes, caps of both kinds, and a max_kv that lays out fewer
    records than the requests have."""
    say("prompt, masks", dtype, dim)
    s = make("prompt", dim, dtype)
    for kw in (dict(window=70), dict(cap=5.0), dict(cap=500.0), dict(window=200, cap=30.0)):
        assert_way("prompt", s, **kw)
        compare(gpu, s, **kw)
    for most in (300, 400, 499):
        t = dict(s, max_kv=most)
        assert_way("prompt", t)
        compare(gpu, t)
    t = dict(s, max_new=250)  # the first requests' rows from 250 on stay as they are
    assert_way("prompt", t)
    compare(gpu, t)
    t = dict(s, prefix=None)
    assert_way("prompt", t, window=100)
    compare(gpu, t, window=100)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_beside_single_tokens(gpu, dtype, dim):
    """A step of prompts and decodes: requests of a token or two on the way
    that the prompts' rows choose."""
    say("mixed", dtype, dim)
    gen = torch.Generator(device=DEV).manual_seed(dim)
    requests = [(900, 1, 0), (700, 400, 0), (1, 1, 0), (0, 0, 0), (1500, 2, 40), (300, 300, 0),
                (40, 1, 0), (650, 330, 90)] * 2
    s = build(gen, requests, 64, 2, dim, dtype, 16)
    want = "rows" if dtype is F32 else "prompt"
    got = hb.kv_attention_way(q=s["q"], out=s["q"], cache=s["cache"], table=s["table"], cu=s["cu"],
                              kv_lens=s["kv_lens"], max_new=400, max_kv=1500, scale=0.1,
                              prefix=s["prefix"])
    assert got[0] == want, got
    compare(gpu, s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_shares_with_windows_and_bounds_too_small(gpu, dtype, dim):
    say("shares, masks", dtype, dim)
    s = make("shares", dim, dtype)
    for kw in (dict(window=11500), dict(cap=30.0)):
        assert_way("shares", s, **kw)
        compare(gpu, s, **kw)
    t = dict(s, max_kv=11000)
    assert_way("shares", t)
    compare(gpu, t)
    t = dict(s, prefix=ints([100 * b for b in range(24)]))
    compare(gpu, t, window=500)


@pytest.mark.parametrize("name,dim,dtype", cases())
def test_lengths_without_sense_stay_inside(gpu, name, dim, dtype):
    """Whatever cu and kv_lens hold: no byte around out is written, nor a row
    that belongs to no request, and the rows of requests that make sense come
    out as they would by themselves."""
    say("way, no sense", name, dim, dtype)
    s = make(name, dim, dtype)
    assert_way(name, s)
    tokens, hq = s["q"].shape[:2]
    batch = s["table"].shape[0]
    kw = dict(q=s["q"], cache=s["cache"], table=s["table"], max_new=s["max_new"],
              max_kv=s["max_kv"], scale=0.1, prefix=s["prefix"], ctx=gpu)
    want, tol, _ = reference(s, 0.1, 0, 0.0)
    tol += HALF[dtype] * want.abs() + TINY[dtype]
    cu0, lens0, most = s["cu"].tolist(), s["kv_lens"].tolist(), 2**31 - 1
    others, last = batch - 1, cu0[batch - 1]
    for cu, lens, good in (
            # the last request as it is, the others none: starts past the
            # tensors, below 0, and after their ends
            ([most] * others + cu0[-2:], [most] * others + lens0[-1:], (last, tokens)),
            ([-most - 1] * others + cu0[-2:], [-7] * others + lens0[-1:], (last, tokens)),
            ([-1 - i for i in range(others)] + cu0[-2:], lens0, (last, tokens)),
            ([tokens + others - i for i in range(others)] + cu0[-2:], lens0, (last, tokens)),
            # the first as it is, the second without an end and of more keys
            # than its table holds
            (cu0[:2] + [most] * others, lens0[:1] + [most] * others, (0, cu0[1]))):
        room = torch.full((tokens + 256, hq, dim), 7.0, dtype=s["q"].dtype, device=DEV)
        out = room[128:128 + tokens]
        hb.kv_attention(out=out, cu=ints(cu), kv_lens=ints(lens), **kw)
        mine = torch.zeros(tokens, dtype=torch.bool, device=DEV)
        for c, d in zip(cu, cu[1:]):
            if 0 <= c < d and c < tokens:
                mine[c:min(d, c + s["max_new"])] = True
        assert bool((room[:128] == 7).all()) and bool((room[128 + tokens:] == 7).all())
        assert bool((out[~mine] == 7).all())
        rows = slice(*good)
        assert bool(((out[rows].double() - want[rows]).abs() <= tol[rows]).all())
