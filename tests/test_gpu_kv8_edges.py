"""Edges of serving on the 8-bit cache on an MI355X: subnormal queries, caches
past 4 GiB, padded batches, calls on two streams at once, and contexts that take
calls of different sizes in turn.  Tolerances are test_gpu_kv8's."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, TYPES, ints, say
from test_gpu_kv8 import WAYS, build, call, check, ramp, reference
from test_gpu_kv_edges import memory_given_back  # noqa: F401
from test_gpu_logprobs import check as check_logprobs

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("name,dtype", [(name, dtype) for name in ("splits", "rows", "prompt")
                                        for dtype in TYPES if (name, dtype) != ("prompt", F32)])
def test_tiny_queries(gpu, dtype, name):
    """Queries that the type holds as subnormals enter the products as they are."""
    say("tiny queries", dtype, name)
    requests, hq, hk, way = WAYS[name]
    s = build(torch.Generator(device=DEV).manual_seed(1), requests, 64, hk, 64, dtype, hq)
    small = {F32: 2.0**-128, BF16: 2.0**-128, F16: 2.0**-18}[dtype]
    s["q"] = (s["q"].double() * small).to(dtype)
    assert s["q"].abs().max() < torch.finfo(dtype).smallest_normal * 16
    check(gpu, s, scale=min(2.0**126, 0.002 / small), way=way)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_caches_past_four_gib(gpu, dtype):
    """Rows, copies and attention at byte offsets past 2^32."""
    say("large cache", dtype)
    heads, dim, page = 8, 128, 32
    pages = (1 << 32) // (heads * (64 * dim + 16)) + 300
    cache = torch.empty(hb.kv8_cache_shape(pages, heads, page, dim), dtype=torch.uint8, device=DEV)
    assert cache.numel() > 2**32
    near, far = cache[:40], cache[-40:]
    near.fill_(0)
    far.fill_(0)
    gen = torch.Generator(device=DEV).manual_seed(4)
    tokens, ids = 500, np.random.default_rng(1).permutation(40)[:16]
    k, v = (torch.randn((tokens, heads, dim), generator=gen, device=DEV).to(dtype)
            for _ in range(2))
    at = np.arange(tokens)
    outs = []
    for first in (0, pages - 40):
        table = first + ids
        hb.kv8_append(k=k, v=v, slots=ints(table[at // page] * page + at % page), cache=cache,
                      ctx=gpu)
        q = torch.randn((3, 32, dim), generator=torch.Generator(device=DEV).manual_seed(5),
                        device=DEV).to(dtype)
        out, gk, gv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        hb.kv8_attention(q=q, out=out, cache=cache, table=ints(table[None]), cu=ints([0, 3]),
                         kv_lens=ints([tokens]), max_new=3, max_kv=tokens, scale=0.1, ctx=gpu)
        hb.kv8_read(k=gk, v=gv, slots=ints(table[at // page] * page + at % page), cache=cache,
                    ctx=gpu)
        outs.append((out, gk, gv))
    assert torch.equal(near, far)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    near.fill_(0)
    hb.kv_copy(cache=cache, pairs=ints([[pages - 40 + i, i] for i in range(40)]), ctx=gpu)
    assert torch.equal(near, far) and near.any()


def test_padded_batches(gpu):
    """Rows behind the last request's, requests without tokens between others,
    and rows of slots that are none."""
    say("padded batches")
    requests = [(0, 0, 0), (70, 3, 0), (40, 0, 0), (33, 1, 0), (0, 0, 0)]
    for dtype in TYPES:
        s = build(torch.Generator(device=DEV).manual_seed(3), requests, 32, 2, 64, dtype, 4)
        s["q"] = torch.cat([s["q"], torch.full((6, 4, 64), float("nan"), device=DEV, dtype=dtype)])
        out = torch.full_like(s["q"], 7.0)
        call(s, out, gpu, 0.001)
        want, _, mine = reference(s, 0.001, 0, 0, 0.0)
        assert mine.tolist() == [True] * 4 + [False] * 6
        assert (out[4:] == 7).all() and (out[:4].double() - want[:4]).abs().max() < 0.1
    cache = torch.full(hb.kv8_cache_shape(2, 1, 32, 64), 3, dtype=torch.uint8, device=DEV)
    rows = torch.randn((5, 1, 64), device=DEV)
    hb.kv8_append(k=rows, v=rows, slots=ints([-1] * 5), cache=cache, ctx=gpu)
    hb.kv8_append(k=rows[:0], v=rows[:0], slots=ints([]), cache=cache, ctx=gpu)
    assert (cache == 3).all()


def test_two_streams_at_once():
    """Calls without a context on two streams do not share a workspace."""
    say("two streams")
    gens = [torch.Generator(device=DEV).manual_seed(i) for i in range(2)]
    sets = [build(g, ramp(12, 3000, 3, 70), 64, 1, 128, BF16, 8) for g in gens]
    logits = [torch.randn((4, 90001), generator=g, device=DEV) for g in gens]
    outs = [torch.empty_like(s["q"]) for s in sets]
    ids = [torch.empty((4, 10), dtype=torch.int32, device=DEV) for _ in gens]
    best = [torch.empty((4, 10), device=DEV) for _ in gens]
    kw = []
    for s, out in zip(sets, outs):
        a = {n: s[n] for n in ("q", "cache", "table", "cu", "kv_lens", "max_new", "max_kv",
                               "prefix")}
        kw.append(dict(a, out=out, scale=0.001, sync=False))

    def work(i):
        hb.kv8_attention(**kw[i])
        hb.token_logprobs(logits=logits[i], top_ids=ids[i], top_logprobs=best[i], sync=False)

    want = []
    for i in range(2):
        work(i)
        torch.cuda.synchronize()
        want.append([x.clone() for x in (outs[i], ids[i], best[i])])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                work(i)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip((outs[i], ids[i], best[i]), want[i]))


def test_calls_of_different_sizes_in_turn():
    """A context's workspace grows and is shared by all calls on its stream, one
    after another: attention's partial results, a compaction's marks, parts of
    rows of logits."""
    say("calls in turn")
    ctx = hb.Context(0)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    try:
        gen = torch.Generator(device=DEV).manual_seed(7)
        small = build(gen, ramp(3, 900, 2), 32, 1, 64, F32, 4)
        large = build(gen, ramp(24, 12000, 6), 64, 2, 128, BF16, 8)
        for s in (small, large, small):
            check(ctx, s)
            check_logprobs(ctx, torch.randn((3, 70001), generator=gen, device=DEV), [1, -1, 9], 20)
            pages = 9000
            table = torch.randperm(pages, generator=gen, device=DEV)[:2000].view(50, 40)
            out, free = torch.empty((50, 40), dtype=torch.int32, device=DEV), ints([0] * pages)
            pairs, status, count = ints(np.zeros((pages // 2, 2))), ints([0, 0]), ints([0])
            hb.kv_compact(table=table.to(torch.int32), lens=ints([40 * 32] * 50), pages=pages,
                          page_size=32, table_out=out, free_pages=free, free_count=count,
                          pairs=pairs, status=status, ctx=ctx, sync=False)
            assert sorted(out.flatten().tolist()) == list(range(2000))
            moved = {int(a): int(b) for a, b in pairs.tolist() if a >= 0}
            assert all(moved.get(p, p) == n for p, n in zip(table.flatten().tolist(),
                                                            out.flatten().tolist()))
            assert int(count) == pages - 2000 and status.tolist() == [2000, len(moved)]
    finally:
        ctx.close()


def test_two_runs_of_a_block_leave_others_alone(gpu):
    """A call that brings a block several runs, its slots backwards or twice over:
    what the block holds is not said, but the call ends and no other block's bytes
    change."""
    say("two runs of a block")
    gen = torch.Generator(device=DEV).manual_seed(1)
    for slots in ([70, 69, 68, 67, 66], [64] * 40, [65, 66, 64, 65, 95, 94],
                  list(range(95, 63, -1)) * 20):
        cache = torch.full(hb.kv8_cache_shape(3, 4, 64, 128), 11, dtype=torch.uint8, device=DEV)
        k, v = (torch.randn((len(slots), 4, 128), generator=gen, device=DEV) for _ in range(2))
        hb.kv8_append(k=k, v=v, slots=ints(slots), cache=cache, ctx=gpu)
        assert (cache[1, :, 0] != 11).any()
        cache[1, :, 0] = 11
        assert (cache == 11).all()
