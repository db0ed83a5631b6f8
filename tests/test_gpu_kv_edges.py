"""The serving operators on an MI355X where their arguments are unusual: values
that are not finite, sizes at the ends of their range, against plain 64-bit
implementations."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, HALF, TINY, TYPES, build, rope_reference, say

pytestmark = pytest.mark.gpu


def same(a, b):
    """torch.equal, with no tensors in a failure's message."""
    return bool(torch.equal(a, b))


# ------------------------------------------------------------------ rope --

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 32, False), (64, 32, True), (96, 48, False),
                                                 (128, 0, False), (30, 14, False), (30, 14, True),
                                                 (64, 64, False)])
def test_rotation_of_infinities_and_nans(gpu, dtype, dim, rot, interleaved):
    """What is not finite stays with its own pair, and past `rot` with its own
    element: the rest of the head comes out as for any other row."""
    say("rope, not finite", dtype, dim, rot, interleaved)
    gen = torch.Generator(device=DEV).manual_seed(dim + rot)
    odd = [math.inf, -math.inf, math.nan]
    x = torch.randn((3 * dim, 2, dim), generator=gen, device=DEV).to(dtype)
    for i in range(3 * dim):  # each element of the head once with each of them
        x[i, 0, i % dim] = odd[i // dim]
        x[i, 1, (i + dim // 2) % dim] = odd[i // dim]
    x[0, :, -1] = -0.0
    half = rot // 2
    pos = torch.randint(1, 5000, (1, 3 * dim), generator=gen, device=DEV, dtype=torch.int32)
    freq = 10000.0 ** -(torch.arange(half, device=DEV, dtype=torch.float64) / max(1, half))
    gamma = 1 + 0.3 * torch.randn((dim,), generator=gen, device=DEV)
    for g in (None, gamma):
        out = torch.empty_like(x)
        hb.norm_rope(q=x, positions=pos, inv_freq=freq, q_out=out, gamma_q=g, eps=1e-5,
                     interleaved=interleaved, ctx=gpu)
        want, size = rope_reference(x, g, pos, freq, (half,), interleaved, 1e-5)
        assert same(out.isnan(), want.isnan())
        assert same(torch.where(out.isinf(), out, 0).double(),
                           torch.where(want.isinf(), want, 0))
        fine = want.isfinite()
        tol = HALF[dtype] * want.abs() + (dim + 16) * 2.0**-24 * size + TINY[dtype]
        assert ((out.double() - want).abs() <= tol)[fine].all()
        if g is None:  # not turned: as they went in, bit for bit where they are numbers
            tail, there = x[..., rot:], ~x[..., rot:].isnan()
            assert same(out[..., rot:][there], tail[there])
            assert same(torch.signbit(out[..., rot:][there]), torch.signbit(tail[there]))


# --------------------------------------------------------------- streams --

def attend(s, out, **kw):
    hb.kv_attention(q=s["q"], out=out, cache=s["cache"], table=s["table"], cu=s["cu"],
                    kv_lens=s["kv_lens"], max_new=s["max_new"], max_kv=s["max_kv"], scale=0.1,
                    prefix=s["prefix"], **kw)


def test_calls_without_a_context_run_on_torchs_current_stream(gpu):
    """After torch work that is still under way on the current stream, and
    before what follows there, on the default stream and on another, with
    workspaces of their own."""
    say("no context")
    gen = torch.Generator(device=DEV).manual_seed(1)
    s = build(gen, [(9000, 1, 0), (7000, 2, 0)], 64, 2, 128, torch.bfloat16, 8)
    want = torch.empty_like(s["q"])
    attend(s, want, ctx=gpu)
    k, v = (torch.randn((50, 2, 64), generator=gen, device=DEV) for _ in range(2))
    slots = torch.arange(50, device=DEV, dtype=torch.int32)
    busy = torch.randn((4096, 4096), device=DEV)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.current_stream()):
        late = dict(s, q=torch.zeros_like(s["q"]))
        out, gk, gv = torch.zeros_like(want), torch.zeros_like(k), torch.zeros_like(v)
        lk, lv = torch.zeros_like(k), torch.zeros_like(v)
        cache = torch.zeros(hb.kv_cache_shape(2, 2, 32, 64), dtype=torch.uint8, device=DEV)
        other = torch.zeros_like(cache)
        hb.kv_append(k=k, v=v, slots=slots, cache=other, ctx=gpu)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            x = busy
            for _ in range(5):
                x = x @ busy * 1e-4
            late["q"].copy_(s["q"])
            lk.copy_(k)
            lv.copy_(v)
            attend(late, out, sync=False)
            hb.kv_append(k=lk, v=lv, slots=slots, cache=cache, sync=False)
            hb.kv_read(k=gk, v=gv, slots=slots, cache=cache, sync=False)
            got, got_k = out.clone(), gk.clone()
            out.zero_()
            late["q"].zero_()
        stream.synchronize()
        assert same(got, want) and same(cache, other) and bool(got_k.any())


def test_calls_without_a_context_from_two_threads(gpu):
    say("no context, two threads")
    gen = torch.Generator(device=DEV).manual_seed(2)
    s = build(gen, [(9000, 1, 0)], 64, 2, 128, torch.bfloat16, 8)
    want = torch.empty_like(s["q"])
    attend(s, want, ctx=gpu)
    torch.cuda.synchronize()
    outs = [torch.zeros_like(want) for _ in range(2)]

    def work(out):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                attend(s, out, sync=False)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(out,)) for out in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(same(out, want) for out in outs)
