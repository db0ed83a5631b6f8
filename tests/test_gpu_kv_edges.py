"""The serving operators on an MI355X where their arguments are unusual: values
that are not finite, sizes at the ends of their range, against plain 64-bit
implementations."""
from __future__ import annotations

import functools
import gc
import math
import threading

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, HALF, TINY, TYPES, build, rope_reference, run_plan, say
from test_gpu_kv import record_map as make_record_map

pytestmark = pytest.mark.gpu
record_map = functools.lru_cache(make_record_map)


@pytest.fixture(scope="module", autouse=True)
def memory_given_back():
    """Nothing stays in torch's allocator: tests of batched layers elsewhere
    want tensors made one after another to lie at equal distances."""
    yield
    record_map.cache_clear()
    gc.collect()
    torch.cuda.empty_cache()


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


# ------------------------------------------------------------------ plan --

def test_lengths_past_31_bits_are_refused(gpu):
    """A request whose keys would pass 2^31 - 1 is refused like one whose pages
    pass the table; the one beside it goes on."""
    say("plan, lengths past 31 bits")
    most, page, columns = 2**31 - 1, 1 << 20, 2060
    for lens, new, fine in (([most - 3, 5], [3, 2], 1), ([most - 3, 5], [4, 2], 0),
                            ([most, 5], [1, 2], 0), ([most, 5], [0, 2], 1)):
        table = np.full((2, columns), -1)
        table[0, :2048], table[1, 0] = 1, 3
        got = run_plan(gpu, lens, new, [8, 9], 2, table, page, 6)
        _, cu, kv, slots, positions, status = [g.tolist() for g in got]
        assert cu == [0, new[0], new[0] + 2] and status == [0, 1 - fine]
        assert kv == [lens[0] + (new[0] if fine else 0), 7]
        assert slots[new[0]:new[0] + 2] == [3 * page + 5, 3 * page + 6]
        assert (slots[0] >= 0) == (fine == 1) or new[0] == 0
        assert positions[new[0] + 2:] == [-1] * (4 - new[0])


# ------------------------------------------------------------ cache rows --

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_read_gives_any_stored_byte(gpu, dtype, dim):
    """Every element under every scale: its value rounded to the tensors' type,
    infinite where that does not hold it, NaN under 255."""
    say("read, any byte", dtype, dim)
    cache = torch.zeros(hb.kv_cache_shape(8, 1, 32, dim), dtype=torch.uint8, device=DEV)
    at = record_map(dim)
    col = torch.arange(dim, device=DEV)
    code = col % 16
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    grid = torch.cat([grid, -grid])[code]
    want = torch.empty((256, 1, dim), dtype=torch.float64, device=DEV)
    for byte in range(256):
        record = cache[byte // 32, 0, 0]
        for codes, scales in ((at[0], at[2]), (at[1], at[3])):
            record[scales[byte % 32]] = byte
            pair = (code[::2] | code[1::2] << 4).to(torch.uint8)
            record[codes[byte % 32, ::2]] = pair
        want[byte, 0] = grid * (math.nan if byte == 255 else 2.0**(byte - 127))
    k, v = (torch.full((256, 1, dim), 3.0, dtype=dtype, device=DEV) for _ in range(2))
    hb.kv_read(k=k, v=v, slots=torch.arange(256, dtype=torch.int32, device=DEV), cache=cache,
               ctx=gpu)
    for got in (k, v):
        assert same(got.isnan(), want.isnan())
        assert same(got.nan_to_num(9, math.inf, -math.inf),
                    want.to(dtype).nan_to_num(9, math.inf, -math.inf))


# ------------------------------------------------------------- attention --

def reference(s, scale, window, cap):
    """fp64 rows, their tolerance and which are computed, as test_gpu_kv's, but
    with what weights too small for f16 lose (2^-32 of the largest weight each)
    by the columns' own values, scale bytes of 253 and more as NaN, and caps
    above 64 off by the score's own roundings instead of the cap's."""
    q, cache, table = s["q"], s["cache"], s["table"]
    tokens, hq, d = q.shape
    group, half = hq // cache.shape[1], q.dtype is not torch.float32
    at, col = record_map(d), torch.arange(d, device=DEV) % 2 * 4
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    grid = torch.cat([grid, -grid])

    def rows(rec, codes, scales):
        e = rec[:, scales].double()
        x = grid[(rec[:, codes].int() >> col) & 15] * torch.exp2(e - 127)
        return torch.where(e >= 253, math.nan, x).reshape(-1, d)

    out = torch.zeros((tokens, hq, d), dtype=torch.float64, device=DEV)
    tol, there = torch.zeros_like(out), torch.zeros(tokens, dtype=torch.bool, device=DEV)
    cu, lens = s["cu"].tolist(), s["kv_lens"].tolist()
    for b, total in enumerate(lens):
        new = cu[b + 1] - cu[b]
        n = min(new, s["max_new"])
        mine = slice(cu[b], cu[b] + n)
        there[mine] = True
        if n == 0 or total == 0:
            continue
        key = torch.arange(total, device=DEV)
        pos = total - new + torch.arange(n, device=DEV)[:, None]
        see = (key <= pos) & (pos - key < window if window else key >= 0)
        if s["prefix"] is not None:
            see = see | (key < s["prefix"][b])
        pages = table[b, :-(-total // (32 * cache.shape[2]))].long()
        ok = (pages >= 0) & (pages < cache.shape[0])
        see = see & ok.repeat_interleave(32 * cache.shape[2])[:total]
        pages = torch.where(ok, pages, 0)
        for h in range(cache.shape[1]):
            rec = cache[pages, h].reshape(-1, 34 * d)
            k, v = rows(rec, at[0], at[2])[:total], rows(rec, at[1], at[3])[:total]
            dead = k.isnan().any(-1) | v.isnan().any(-1)
            k, v = torch.nan_to_num(k), torch.nan_to_num(v)
            heads = slice(h * group, (h + 1) * group)
            x = q[mine, heads].double().reshape(n * group, d)
            sees = see.repeat_interleave(group, 0)
            y = x @ k.T * scale
            ds = (d + 8) * 2.0**-24 * (x.abs() @ k.abs().T * abs(scale))
            if cap:
                y = cap * torch.tanh(y / cap)
                ds = ds + (cap * 2.0**-21 if cap <= 64 else 2.0**-21 * y.abs())
            y = torch.where(dead, math.nan, y).masked_fill(~sees, -math.inf)
            top = torch.nan_to_num(y, nan=-math.inf).amax(-1, keepdim=True)
            p = torch.exp(y - torch.where(top.isinf(), 0, top))
            p = p / torch.where(sees.any(-1, keepdim=True), p.sum(-1, keepdim=True), 1)
            out[mine, heads] = (p @ v).view(n, group, d)
            ds = torch.where(sees, ds, 0).amax(-1, keepdim=True)
            off = p @ v.abs() * (2 * ds + (2.0**-11 if half else 0) + total * 2.0**-23 + 2.0**-21)
            tol[mine, heads] = (off + 2.0**-32 * (sees.double() @ v.abs())).view(n, group, d)
    return out, tol, there


def compare(gpu, s, scale=None, window=0, cap=0.0, out=None):
    """The call's rows against the reference, twice: the same bits."""
    q, d = s["q"], s["q"].shape[-1]
    scale = d ** -0.5 if scale is None else scale
    want, tol, mine = reference(s, scale, window, cap)
    first, out = torch.full_like(q, 7.0), torch.empty_like(q) if out is None else out
    out.fill_(7.0)
    for to in (first, out):
        hb.kv_attention(q=q, out=to, cache=s["cache"], table=s["table"], cu=s["cu"],
                        kv_lens=s["kv_lens"], max_new=s["max_new"], max_kv=s["max_kv"],
                        scale=scale, prefix=s["prefix"], window=window, softcap=cap, ctx=gpu)
    assert same(first.nan_to_num(9, math.inf, -math.inf), out.nan_to_num(9, math.inf, -math.inf))
    assert bool((out[~mine] == 7).all())
    got, want, tol = out[mine].double(), want[mine], tol[mine]
    assert same(got.isnan(), want.isnan())
    tol = tol + HALF[q.dtype] * want.abs() + TINY[q.dtype]
    most = torch.finfo(q.dtype).max  # what rounds past it is an infinity
    over = want.abs() - tol > most * (1 + HALF[q.dtype])
    assert (got[over] == torch.sign(want[over]) * math.inf).all()
    there = ~want.isnan() & (want.abs() + tol < most)
    worst = ((got - want).abs() / tol)[there].max().item() if there.any() else 0.0
    assert worst <= 1, f"{worst} of the tolerance"


def attend(s, out, **kw):
    hb.kv_attention(q=s["q"], out=out, cache=s["cache"], table=s["table"], cu=s["cu"],
                    kv_lens=s["kv_lens"], max_new=s["max_new"], max_kv=s["max_kv"], scale=0.1,
                    prefix=s["prefix"], **kw)


# a row of a request, 70 to 90, 200 (requests, K/V heads; a query head each): which way
# of dividing the work these take differs by type and head size
ROWS = {"one": ([(300, 1, 0), (270, 1, 10)], 2), "rows": ([(300, 90, 0), (270, 70, 10)], 16),
        "prompt": ([(300, 200, 0), (270, 200, 10)] * 4, 40)}


def set_scale(s, b, token, which, value, block=None):
    """Scale bytes of K (2) or V (3) of a request's token, of all heads."""
    at = record_map(s["q"].shape[-1])[which, token % 32, ::32]
    at = at if block is None else at[block:block + 1]
    page, group = token // 32 // s["cache"].shape[2], token // 32 % s["cache"].shape[2]
    s["cache"][s["table"][b, page].long(), :, group, at] = value


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", list(ROWS))
def test_scales_past_the_types_range(gpu, dtype, dim, rows):
    """Scale bytes of 253 and 254, whose products pass bf16 and fp32, make the
    rows that see their token NaN and no others."""
    say("scales past the range", dtype, dim, rows)
    gen = torch.Generator(device=DEV).manual_seed(dim)
    requests, hk = ROWS[rows]
    s = build(gen, requests, 32, hk, dim, dtype, hk)
    for which in (2, 3):
        for b, token, value in ((0, 299 if rows == "one" else 230, 253), (1, 20, 254)):
            t = dict(s, cache=s["cache"].clone())
            set_scale(t, b, token, which, value, block=dim // 32 - 1)
            compare(gpu, t)
            compare(gpu, t, window=64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", list(ROWS))
def test_values_of_any_size(gpu, dtype, dim, rows):
    """V from the smallest scale to the largest that is stored (252), alone and
    among ordinary tokens, in whole rows and in one block of 32 columns."""
    say("values of any size", dtype, dim, rows)
    gen = torch.Generator(device=DEV).manual_seed(dim)
    requests, hk = ROWS[rows]
    s = build(gen, requests, 32, hk, dim, dtype, hk)
    for changes in ([(0, 3, 252)], [(0, 3, 206), (0, 4, 200)], [(0, 40, 230), (1, 250, 252)],
                    [(0, 3, 180), (0, 70, 240), (0, 71, 252)], [(1, 33, 30)]):
        for block in (None, 1):
            t = dict(s, cache=s["cache"].clone())
            for b, token, value in changes:
                set_scale(t, b, token, 3, value, block)
            compare(gpu, t)
    for b, (keys, _, _) in enumerate(requests):  # every token alike, and rising
        for t in range(keys):
            set_scale(s, b, t, 3, 252)
    compare(gpu, s)
    compare(gpu, s, scale=3.0)
    for b, (keys, _, _) in enumerate(requests):
        for t in range(keys):
            set_scale(s, b, t, 3, 100 + 152 * t // keys)
    compare(gpu, s)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_key_gives_its_value(gpu, dtype):
    """One key, scale byte by scale byte: the row is the stored value, rounded."""
    say("one key", dtype)
    gen = torch.Generator(device=DEV).manual_seed(1)
    requests = [(1, 1, 0)] * 253
    s = build(gen, requests, 32, 2, 64, dtype, 4)
    for b in range(253):
        set_scale(s, b, 0, 3, b)
    compare(gpu, s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", list(ROWS))
def test_subnormal_queries(gpu, dtype, dim, rows):
    """Queries that are subnormal in a 16-bit type, and those of 2^-110 in fp32
    (below that the third bf16 part is subnormal and loses bits), on keys as
    large as they are small, give the scores of their products."""
    say("subnormal queries", dtype, dim, rows)
    gen = torch.Generator(device=DEV).manual_seed(dim)
    requests, hk = ROWS[rows]
    s = build(gen, requests, 32, hk, dim, dtype, hk)
    small, scale = {torch.float16: (2.0**-17, 138), torch.bfloat16: (2.0**-128, 250),
                    torch.float32: (2.0**-108, 230)}[dtype]
    s["q"] = (s["q"].float() * small).to(dtype)
    if dtype is torch.float32:
        s["q"] += torch.copysign(torch.full_like(s["q"], 2.0**-110), s["q"])
    else:
        assert (s["q"].abs() < torch.finfo(dtype).smallest_normal).any()
    s["cache"][..., 32 * dim:33 * dim] = scale
    compare(gpu, s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", list(ROWS))
def test_caps_of_any_size(gpu, dtype, dim, rows):
    """A cap far above the scores leaves them as they are, one far below makes
    them alike; scores of ordinary size throughout."""
    say("caps", dtype, dim, rows)
    gen = torch.Generator(device=DEV).manual_seed(dim)
    requests, hk = ROWS[rows]
    s = build(gen, requests, 32, hk, dim, dtype, hk)
    for cap in (1e-38, 1e-20, 1e-3, 5.0, 64.0, 65.0, 1000.0, 1e5, 1e7, 1e15, 1e19, 1e30, 3e38):
        compare(gpu, s, cap=cap)
    compare(gpu, s, cap=1e5, scale=-1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_do_not_depend_on_their_alignment(gpu, dtype, dim):
    """The same bits in and out of rows aligned to 16 bytes, to 8 and to their
    elements alone, in calls of few rows and of many."""
    say("alignment", dtype, dim)
    gen = torch.Generator(device=DEV).manual_seed(dim)
    for requests, hq, hk in ([[(300, 3, 0), (90, 1, 0)], 8, 2], [[(500, 300, 0)] * 16, 16, 2]):
        s = build(gen, requests, 64, hk, dim, dtype, hq)
        tokens, outs = s["q"].shape[0], []
        for pad in (0, 4, 1):
            q, out = (torch.full((tokens, hq, dim + pad), 7.0, dtype=dtype, device=DEV)
                      for _ in range(2))
            q[..., pad:] = s["q"]
            attend(dict(s, q=q[..., pad:]), out[..., pad:], ctx=gpu)
            assert bool((out[..., :pad] == 7).all())
            outs.append(out[..., pad:])
        assert same(outs[0], outs[1]) and same(outs[0], outs[2])


# --------------------------------------------------------------- streams --

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
