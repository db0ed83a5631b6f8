"""The 8-bit cache's rows and its attention on an MI355X against plain 64-bit
implementations, at the sizes, masks and contents where they can go wrong, on
every way of dividing attention's work.

Tolerances.  Rows: none, the stored values are whole codes times a power of
two.  Attention, of a row with weights p and A = sum p |v|: the output's
rounding; 2 ds A for scores off by ds (the products' sum over dim terms and the
few operations after it, dim + 8 roundings of 2^-24, and of fp32 queries 2^-133
an element, where bf16 ends); the weights' own rounding (2^-11 A in f16 for the
16-bit types, none for fp32) or 2^-32 of the largest value a key; 2^-24 A a
term, twice, for the sums over the keys; 2^-21 A for exponentials and the
division; caps 2^-21 of the cap on a score."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, HALF, TINY, TYPES, ints, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ------------------------------------------------------------------ rows --

def on_grid(y):
    """float64 on the E4M3 grid, nearest even, past 448 that."""
    a = np.minimum(np.abs(y), 448.0)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0**-6))) - 3)
    return np.copysign(np.rint(a / step) * step, y)


class Reference:
    """A cache in float64: values and exponents (-127: zeros only) of blocks."""

    def __init__(self, pages, heads, page, dim):
        self.size = pages * page
        self.values = np.zeros((2, self.size, heads, dim))
        self.exponent = np.full((2, self.size // 32, heads), -127)

    def append(self, k, v, slots):
        x = np.stack([k, v])  # [2][tokens][heads][dim]
        bad = ~np.isfinite(x).all((0, 3))
        x = np.where(bad[..., None], 0.0, x)
        i = 0
        while i < len(slots):
            s = int(slots[i])
            if not 0 <= s < self.size:
                i += 1
                continue
            n = 1
            while i + n < len(slots) and slots[i + n] == s + n and (s + n) % 32:
                n += 1
            block, t0 = s // 32, s % 32
            top = np.abs(x[:, i:i + n]).max((1, 3))
            need = np.full(top.shape, -127)
            some = top > 0
            need[some] = np.ceil(np.log2(top[some] / 448)).astype(int)
            # (log2 near a power of two)
            need[some] += top[some] > 448 * 2.0 ** need[some]
            need[some] -= top[some] <= 448 * 2.0 ** (need[some] - 1)
            need[some] = np.clip(need[some], -117, 119)
            had = self.exponent[:, block] if t0 else np.full(top.shape, -127)
            e = np.maximum(need, had)
            unit = 2.0 ** e[:, None, :, None].astype(float)
            old = self.values[:, block * 32:block * 32 + t0]
            old[:] = np.where(np.isnan(old), old, on_grid(old / unit) * unit)
            new = on_grid(x[:, i:i + n] / unit) * unit
            new[0][bad[i:i + n]] = np.nan
            self.values[:, s:s + n] = new
            self.exponent[:, block] = e
            i += n

    def check(self, cache, slots, gpu):
        """The stored values and scales of slots' tokens and blocks."""
        inside = (slots >= 0) & (slots < self.size)
        at = np.where(inside, slots, 0)
        want = np.where(inside[:, None, None], self.values[:, at], 0.0)
        heads, dim = want.shape[2:]
        for dtype in TYPES:
            got = [torch.full((len(slots), heads, dim), 3.0, dtype=dtype, device=DEV)
                   for _ in range(2)]
            hb.kv8_read(k=got[0], v=got[1], slots=ints(slots), cache=cache, ctx=gpu)
            for g, w in zip(got, want):
                w = torch.from_numpy(w).to(DEV).to(dtype)
                assert torch.equal(g.isnan(), w.isnan())
                assert torch.equal(torch.nan_to_num(g, 9), torch.nan_to_num(w, 9)), dtype
        groups = cache.shape[2]
        for block in sorted(set(at[inside] // 32)):
            byte = cache[block // groups, :, block % groups, 64 * dim:64 * dim + 2].cpu().numpy()
            e = self.exponent[:, block].T
            assert (byte == np.where(e == -127, 0, e + 127)).all()


def rows_of(rng, shape, dtype, spread=1.0):
    x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[1:]))
    return torch.from_numpy(x).to(DEV).to(dtype)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,page", [(1, 32), (3, 96), (5, 64)])
def test_rows_of_steps(gpu, dim, dtype, heads, page):
    """Prompts, then tokens one by one and a few at a time, of larger values each
    time: earlier tokens are rounded again."""
    say("rows8", dim, dtype, heads, page)
    rng = np.random.default_rng(dim + heads)
    pages = 12
    cache = torch.full(hb.kv8_cache_shape(pages, heads, page, dim), 0x5A, dtype=torch.uint8,
                       device=DEV)
    ref = Reference(pages, heads, page, dim)
    order = rng.permutation(pages)
    lens = [0, 0, 0]
    used = [order[:4], order[4:8], order[8:]]
    for step, new in enumerate([(40, 7, 65), (1, 1, 1), (1, 3, 0), (2, 1, 31), (1, 1, 1)]):
        slots = [-1]
        for b, n in enumerate(new):
            at = np.arange(lens[b], lens[b] + n)
            slots += list(used[b][at // page] * page + at % page) + [-1] * (step % 2)
            lens[b] += n
        slots = np.array(slots)
        k, v = (rows_of(rng, (len(slots), heads, dim), dtype) * 3.0**step for _ in range(2))
        hb.kv8_append(k=k, v=v, slots=ints(slots), cache=cache, ctx=gpu)
        ref.append(k.double().cpu().numpy(), v.double().cpu().numpy(), slots)
        live = np.concatenate([used[b][np.arange(n) // page] * page + np.arange(n) % page
                               for b, n in enumerate(lens)])
        ref.check(cache, live, gpu)


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_odd_values(gpu, dim, dtype):
    say("odd rows8", dim, dtype)
    rng = np.random.default_rng(dim)
    pages, heads, page = 6, 2, 64
    cache = torch.zeros(hb.kv8_cache_shape(pages, heads, page, dim), dtype=torch.uint8, device=DEV)
    ref = Reference(pages, heads, page, dim)
    most = torch.finfo(dtype).max
    for kind in range(6):
        slots = np.concatenate([np.arange(kind * 64, kind * 64 + 50), [-5, 6 * 64, 2**31 - 1]])
        k, v = (rows_of(rng, (53, heads, dim), dtype) for _ in range(2))
        if kind == 0:  # zeros, of both signs, and a block of nothing else
            k[:32] = 0
            v[:40] = -0.0
        elif kind == 1:  # not finite: keys of NaN, no values, no scale
            k[3, 0, 5], v[7, 1, 9], k[33:, 1, 0] = math.nan, math.inf, -math.inf
        elif kind == 2:  # up to the largest
            k[:], v[10:20] = k.sign() * most, most
        elif kind == 3:  # down to the smallest
            k *= torch.finfo(dtype).tiny
            v[:] = torch.finfo(dtype).smallest_normal * 2.0**-4
        elif kind == 4:  # whole codes, ties between them, and just past 448 units
            k[:] = torch.tensor([448, 449, 17, 18, 19, 1.0625, 2.0**-9 * 1.5, 464] * (dim // 8))
            v[:] = 1.0 + torch.arange(dim) / 64
        k, v = k.contiguous(), v.contiguous()
        # in two calls: the second begins within a block
        for part in (slice(0, 21), slice(21, 53)):
            hb.kv8_append(k=k[part], v=v[part], slots=ints(slots[part]), cache=cache, ctx=gpu)
            ref.append(k[part].double().cpu().numpy(), v[part].double().cpu().numpy(), slots[part])
        ref.check(cache, slots, gpu)


def test_rows_begin_blocks_anew_and_leave_others_alone(gpu):
    """A page that another request used: its first token begins each block anew;
    bytes of blocks that no slot names are not touched, nor those of tokens past
    a run."""
    say("rows8 anew")
    rng = np.random.default_rng(3)
    cache = torch.full(hb.kv8_cache_shape(3, 2, 64, 64), 0xFF, dtype=torch.uint8, device=DEV)
    ref = Reference(3, 2, 64, 64)
    slots = np.concatenate([np.arange(64, 64 + 5), np.arange(0, 32)])
    k, v = (rows_of(rng, (len(slots), 2, 64), F32) * 1e-3 for _ in range(2))
    before = cache.clone()
    hb.kv8_append(k=k, v=v, slots=ints(slots), cache=cache, ctx=gpu)
    ref.append(k.double().cpu().numpy(), v.double().cpu().numpy(), slots)
    ref.check(cache, slots, gpu)
    assert torch.equal(cache[2], before[2]) and torch.equal(cache[:2, :, 1], before[:2, :, 1])
    assert (cache[1, :, 0] != 0xFF).sum().item() <= 2 * (5 * 2 * 64 + 2)


def test_runs_of_many_requests_in_one_window(gpu):
    """More tokens and heads than workgroups: many runs a workgroup, whose rows
    stand between one another's."""
    say("many runs8")
    rng = np.random.default_rng(4)
    heads, dim, page, requests = 8, 64, 32, 900
    cache = torch.zeros(hb.kv8_cache_shape(requests, heads, page, dim), dtype=torch.uint8,
                        device=DEV)
    ref = Reference(requests, heads, page, dim)
    lens = np.zeros(requests, int)
    for _ in range(3):
        new = rng.integers(0, 6, requests)
        slots = np.concatenate([b * page + lens[b] + np.arange(n) for b, n in enumerate(new)])
        k, v = (rows_of(rng, (len(slots), heads, dim), BF16, 2.0) for _ in range(2))
        hb.kv8_append(k=k, v=v, slots=ints(slots), cache=cache, ctx=gpu)
        ref.append(k.double().cpu().numpy(), v.double().cpu().numpy(), slots)
        lens += new
    live = np.concatenate([b * page + np.arange(n) for b, n in enumerate(lens)])
    ref.check(cache, live, gpu)


@pytest.mark.parametrize("dtype", TYPES)
def test_row_strides(gpu, dtype):
    say("rows8 strides", dtype)
    gen = torch.Generator(device=DEV).manual_seed(5)
    raw = torch.randn((40 * 5 * 131 + 1,), generator=gen, device=DEV).to(dtype)[1:]
    k, v = raw.view(40, 5, 131)[:, :2, 1:129], raw.view(40, 5, 131)[:, 3:, 3:131]
    slots = torch.arange(3, 43, device=DEV, dtype=torch.int32)
    a, b = (torch.zeros(hb.kv8_cache_shape(2, 2, 32, 128), dtype=torch.uint8, device=DEV)
            for _ in range(2))
    hb.kv8_append(k=k, v=v, slots=slots, cache=a, ctx=gpu)
    hb.kv8_append(k=k.contiguous(), v=v.contiguous(), slots=slots, cache=b, ctx=gpu)
    assert torch.equal(a, b)
    gk = torch.empty((2, 40, 129), dtype=dtype, device=DEV).transpose(0, 1)[..., 1:]
    gv, wk, wv = (torch.empty_like(k.contiguous()) for _ in range(3))
    hb.kv8_read(k=gk, v=gv, slots=slots, cache=a, ctx=gpu)
    hb.kv8_read(k=wk, v=wv, slots=slots, cache=a, ctx=gpu)
    assert torch.equal(gk, wk) and torch.equal(gv, wv)
    assert (wk - k).abs().max() <= k.abs().max() / 16


# ------------------------------------------------------------- attention --

def offsets(dim):
    """Byte offsets in a record of K and V codes [32][dim]."""
    t, col = np.arange(32)[:, None], np.arange(dim)
    w = t // 16 * (dim // 4) + col % (dim // 4)
    k = w // 16 * 1024 + col // (dim // 4) * 256 + t % 16 * 16 + w % 16
    w = col % (dim // 16) * 8 + t % 4 + t // 16 * 4
    v = 32 * dim + w // 16 * 1024 + t % 16 // 4 * 256 + col // (dim // 16) * 16 + w % 16
    return torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV)


def decode(cache, page_ids, head, dim):
    """K, V fp64 [len(page_ids) * page][dim], and which a page has."""
    ok = (page_ids >= 0) & (page_ids < cache.shape[0])
    rec = cache[torch.where(ok, page_ids, 0).long(), head].reshape(-1, 64 * dim + 16)
    out = []
    for i, at in enumerate(offsets(dim)):
        code = rec[:, at].long()
        exp, man = code >> 3 & 15, (code & 7).double()
        x = torch.where(exp > 0, torch.exp2(exp.double() - 7) * (1 + man / 8), man * 2.0**-9)
        x = torch.where(code % 128 == 127, math.nan, torch.where(code > 127, -x, x))
        x = x * torch.exp2(rec[:, 64 * dim + i, None, None].double() - 127)
        out.append(x.reshape(-1, dim))
    return out[0], out[1], ok.repeat_interleave(cache.shape[2] * 32)


def reference(s, scale, window, sinks, cap):
    """fp64 output, the tolerance without its rounding, and the rows that are."""
    q, cache, table = s["q"], s["cache"], s["table"]
    tokens, hq, d = q.shape
    hk, page = cache.shape[1], cache.shape[2] * 32
    group, out = hq // hk, torch.zeros((tokens, hq, d), dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    mine = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    half = q.dtype is not F32
    cu, lens = s["cu"].tolist(), s["kv_lens"].tolist()
    for b in range(table.shape[0]):
        n, total = cu[b + 1] - cu[b], lens[b]
        rows = slice(cu[b], cu[b] + min(n, s["max_new"]))
        mine[rows] = True
        if n <= 0 or total <= 0:
            continue
        i = torch.arange(min(n, s["max_new"]), device=DEV)[:, None]
        pos, key = total - n + i, torch.arange(total, device=DEV)
        see = key <= pos
        if window:
            see = see & ((pos - key < window) | (key < sinks))
        if s["prefix"] is not None:
            see = see | (key < int(s["prefix"][b]))
        for h in range(hk):
            k, v, ok = decode(cache, table[b, :-(-total // page)], h, d)
            k, v, ok = k[:total], v[:total], ok[:total]
            dead = k.isnan().any(-1)
            k = torch.nan_to_num(k)
            for g in range(h * group, (h + 1) * group):
                x = q[rows, g].double()
                sc = x @ k.T.contiguous() * scale
                ds = (d + 8) * 2.0**-24 * (x.abs() @ k.abs().T.contiguous() * abs(scale))
                if not half:  # bf16 parts end at its last step, 2^-133: that much of an element
                    ds = ds + 2.0**-133 * k.abs().sum(-1) * abs(scale)
                if cap:
                    sc = cap * torch.tanh(sc / cap)
                    ds = ds + cap * 2.0**-21
                sc = torch.where(dead, math.nan, sc).masked_fill(~(see & ok), -math.inf)
                top = torch.nan_to_num(sc, nan=-math.inf).amax(-1, keepdim=True)
                p = torch.exp(sc - torch.where(top.isinf(), 0, top))
                total_p = p.sum(-1, keepdim=True)
                p = torch.where(total_p == 0, 0, p / total_p)
                seen = torch.where((see & ok)[..., None].any(0), v, 0.0)
                out[rows, g] = p @ seen
                size = torch.nan_to_num(p) @ seen.abs()
                ds = torch.where(see & ok, ds, 0).amax(-1, keepdim=True)
                tol[rows, g] = size * (2 * ds + (2.0**-11 if half else 0) + total * 2.0**-23 +
                                       2.0**-21) + total * 2.0**-32 * seen.abs().amax()
    return out, tol, mine


def build(gen, requests, page, heads, dim, dtype, hq, spare=2, lo=118, hi=124):
    """requests: (keys, new, prefix).  Past a request's keys its pages hold any
    byte, NaN codes among them."""
    used = [-(-k // page) for k, _, _ in requests]
    shape = hb.kv8_cache_shape(sum(used) + spare, heads, page, dim)
    cache = torch.randint(0, 254, shape, generator=gen, device=DEV, dtype=torch.int32)
    cache = (cache + (cache >= 127)).to(torch.uint8)  # all codes but the NaNs
    cache[..., 64 * dim:] = torch.randint(lo, hi, cache[..., 64 * dim:].shape, generator=gen,
                                          device=DEV, dtype=torch.int32).to(torch.uint8)
    perm = torch.randperm(shape[0], generator=gen, device=DEV).tolist()
    table = np.full((len(requests), max(used + [1]) + 1), -1, np.int64)
    at = 0
    k_at, v_at = offsets(dim)
    for b, n in enumerate(used):
        table[b, :n] = perm[at:at + n]
        at += n
        tail = requests[b][0] % page
        if n and tail:
            rec = cache[perm[at - 1]]  # [heads][groups][record]
            rec[:, tail // 32 + 1:] = 0xFF
            if tail % 32:
                rec[:, tail // 32, k_at[tail % 32:].flatten()] = 0xFF
                rec[:, tail // 32, v_at[tail % 32:].flatten()] = 0x7F
    cache[perm[at:]] = 0xFF
    cu = np.concatenate([[0], np.cumsum([n for _, n, _ in requests])])
    q = torch.randn((int(cu[-1]), hq, dim), generator=gen, device=DEV).to(dtype)
    return dict(q=q, cache=cache, table=ints(table), cu=ints(cu),
                kv_lens=ints([k for k, _, _ in requests]),
                prefix=ints([p for _, _, p in requests]) if any(p for _, _, p in requests) else None,
                max_new=max(n for _, n, _ in requests), max_kv=max(k for k, _, _ in requests))


def call(s, out, gpu, scale, window=0, sinks=0, cap=0.0, fn=None):
    kw = dict(q=s["q"], out=out, cache=s["cache"], table=s["table"], cu=s["cu"],
              kv_lens=s["kv_lens"], max_new=s["max_new"], max_kv=s["max_kv"], scale=scale,
              prefix=s["prefix"], window=window, sinks=sinks, softcap=cap)
    return hb.kv8_attention_way(**kw) if fn else hb.kv8_attention(ctx=gpu, **kw)


def check(gpu, s, scale=None, window=0, sinks=0, cap=0.0, way=None):
    q, d = s["q"], s["q"].shape[-1]
    scale = (d ** -0.5) / 100 if scale is None else scale
    out = torch.full_like(q, 7.0)
    if way is not None:
        assert call(s, out, gpu, scale, window, sinks, cap, True)[0] == way
    call(s, out, gpu, scale, window, sinks, cap)
    want, tol, mine = reference(s, scale, window, sinks, cap)
    got = out.double()
    assert torch.equal(got[mine].isnan(), want[mine].isnan())
    tol = tol + HALF[q.dtype] * want.abs() + TINY[q.dtype]
    most = torch.finfo(q.dtype).max  # what rounds past it is an infinity
    there = mine[:, None, None] & ~want.isnan() & (want.abs() + tol < most)
    over = mine[:, None, None] & (want.abs() - tol > most * (1 + HALF[q.dtype]))
    assert (got[over] == torch.sign(want[over]) * math.inf).all()
    worst = ((got - want).abs() / tol)[there].max().item() if there.any() else 0.0
    assert worst <= 1, f"{worst} of the tolerance"
    assert (out[~mine] == 7.0).all()
    again = torch.full_like(q, 5.0)
    call(s, again, gpu, scale, window, sinks, cap)
    assert torch.equal(torch.nan_to_num(again[mine]), torch.nan_to_num(out[mine]))
    return out


def ramp(count, kv, new, prefix=0):
    return [(kv - i * kv // (2 * count), max(1, new - i * new // (2 * count)), max(0, prefix - i))
            for i in range(count)]


#: requests, query heads, K/V heads, the way that their sizes are meant for
WAYS = {
    "rows": (ramp(4, 300, 256), 32, 32, "rows"),
    "rows, two tiles": (ramp(24, 130, 60), 32, 8, "rows"),
    "splits": (ramp(2, 300, 90, 40), 16, 16, "splits"),
    "splits, joined": (ramp(12, 3000, 3, 70), 8, 1, "splits"),
    "splits, joined, two tiles": (ramp(3, 3000, 130), 8, 1, "splits"),
    "shares": (ramp(24, 12000, 2), 8, 2, "shares"),
    "shares, two tiles": (ramp(24, 12000, 6), 8, 2, "shares"),
    "prompt": (ramp(16, 500, 300, 30), 16, 2, "prompt"),
}


@pytest.mark.parametrize("name,dim,dtype", [
    pytest.param(name, dim, dtype, id=f"{name}-{dim}-{str(dtype)[6:]}")
    for name in WAYS for dim in (64, 128, 256) for dtype in TYPES
    if (name, dtype) != ("prompt", F32) and ("two tiles" not in name or dim < 256)])
def test_attention_on_every_way(gpu, name, dim, dtype):
    requests, hq, hk, way = WAYS[name]
    say("attention8", name, dim, dtype)
    s = build(torch.Generator(device=DEV).manual_seed(dim), requests, 64, hk, dim, dtype, hq)
    if name == "rows, two tiles":  # (some types take these in splits)
        way = None
    check(gpu, s, way=way)
    check(gpu, s, window=77, sinks=40, cap=20.0)


MASKS = [dict(), dict(window=1), dict(window=33, sinks=1), dict(window=100, sinks=4),
         dict(window=64, sinks=64), dict(window=5, sinks=4096), dict(cap=3.0), dict(cap=300.0)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("prefix", [0, 50])
def test_attention_masks_and_lengths(gpu, dim, dtype, prefix):
    """Lengths of nothing, one and around a block's and a page's ends; rows that
    see no key; windows with first tokens that stay visible."""
    say("attention8 masks", dim, dtype, prefix)
    requests = [(0, 0, 0), (1, 1, 0), (0, 2, 0), (31, 1, prefix), (32, 5, prefix), (33, 33, 0),
                (3, 7, 0), (64, 1, 0), (65, 2, prefix), (200, 40, prefix), (129, 1, 1), (500, 3, 0)]
    s = build(torch.Generator(device=DEV).manual_seed(dim + prefix), requests, 32, 2, dim, dtype, 6)
    for mask in MASKS:
        check(gpu, s, **mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lo,hi", [(10, 12), (60, 62), (0, 1), (112, 136), (127, 128), (133, 140),
                                   (150, 220), (244, 247)])
def test_attention_of_scales_of_every_size(gpu, dtype, lo, hi):
    """Values far outside what f16 holds, blocks of zeros (scale byte 0), and
    values whose weighted sums would pass fp32."""
    say("attention8 scales", dtype, lo, hi)
    gen = torch.Generator(device=DEV).manual_seed(lo)
    for requests, hq, hk in (([(300, 3, 0), (77, 1, 0)], 4, 2), (ramp(16, 500, 300, 30), 16, 2)):
        s = build(gen, requests, 64, hk, 64, dtype, hq, lo=lo, hi=hi)
        if lo == 0:  # every second record
            codes = s["cache"].view(-1, 64 * 64 + 16)
            codes[::2, :64 * 64] &= 0x80
            codes[1::2, 64 * 64:] = 120
        # scores of one size whatever the keys'
        scale = 2.0 ** (127 - min(max(lo, 1), 246)) / 4096
        scale = min(max(scale, 2.0**-126), 2.0**100)
        check(gpu, s, scale=scale)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_nan_keys_and_missing_pages(gpu, dim, dtype):
    say("attention8 nan", dim, dtype)
    for requests, hq, hk in (([(150, 2, 0), (90, 40, 10)], 4, 2), (ramp(16, 500, 300, 30), 16, 2)):
        s = build(torch.Generator(device=DEV).manual_seed(dim), requests, 32, hk, dim, dtype, hq)
        k_at, v_at = offsets(dim)
        page = int(s["table"][0, 2])  # keys 64 .. 95
        s["cache"][page, 1, 0, k_at[7]] = 0xFF
        s["cache"][page, 1, 0, v_at[7]] = 0
        table = s["table"].clone()
        table[1, 1], table[1, 2] = -1, s["cache"].shape[0] + 5
        s["table"] = table
        out = check(gpu, s)
        if dtype is not F32 or hq == 4:
            assert out.isnan().any() and not out[:, :hq // hk].isnan().any()
        check(gpu, s, window=20, sinks=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides_and_small_bounds(gpu, dtype):
    """Strided, unaligned q and out, and a max_kv that is too small."""
    say("attention8 strides", dtype)
    for requests, hq, hk in (([(300, 3, 0), (77, 30, 5)], 4, 2), (ramp(16, 500, 300, 30), 16, 2)):
        s = build(torch.Generator(device=DEV).manual_seed(9), requests, 64, hk, 128, dtype, hq)
        plain = check(gpu, s)
        wide = torch.empty((s["q"].shape[0], hq, 131), dtype=dtype, device=DEV)[..., 1:129]
        wide.copy_(s["q"])
        out = torch.empty((hq, s["q"].shape[0], 130), dtype=dtype, device=DEV)
        out = out.transpose(0, 1)[..., 2:]
        call(dict(s, q=wide), out, gpu, 128 ** -0.5 / 100)
        assert torch.equal(out, plain)
        check(gpu, dict(s, max_kv=40))


def test_attention_of_an_odd_plan(gpu):
    """cu and kv_lens that make no sense leave other memory alone: rows outside
    the tensors, lengths past the table, negative ones."""
    say("attention8 odd plan")
    s = build(torch.Generator(device=DEV).manual_seed(2), [(100, 4, 0)] * 4, 32, 2, 64, BF16, 4)
    guard = torch.full((20, 4, 64), 7.0, dtype=BF16, device=DEV)
    for cu, lens in (([0, 4, 900, 12, 16], [100, -7, 2**31 - 1, 100]),
                     ([-5, 3, 3, 2**31 - 1, 1], [2**31 - 1] * 4), ([16, 12, 8, 4, 0], [0] * 4)):
        out = guard[2:18]
        call(dict(s, cu=ints(cu), kv_lens=ints(lens)), out, gpu, 0.001)
        assert (guard[:2] == 7).all() and (guard[18:] == 7).all()


def test_attention_on_another_stream_and_in_a_graph(gpu):
    """Without a context on torch's current stream; captured once sizes are known
    and replayed between eager calls, every replay the eager result's bits."""
    say("attention8 graph")
    s = build(torch.Generator(device=DEV).manual_seed(6), ramp(12, 3000, 3, 70), 64, 1, 128, BF16,
              8)
    want = torch.empty_like(s["q"])
    call(s, want, gpu, 0.001)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = torch.empty_like(want)
        call(s, out, None, 0.001)
        k, v = (torch.randn((70, 1, 128), device=DEV) for _ in range(2))
        cache = torch.zeros(hb.kv8_cache_shape(3, 1, 64, 128), dtype=torch.uint8, device=DEV)
        slots = torch.arange(70, dtype=torch.int32, device=DEV)
        hb.kv8_append(k=k, v=v, slots=slots, cache=cache)
        other = cache.clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            hb.kv8_append(k=k, v=v, slots=slots, cache=other, ctx=None, sync=False)
            kw = dict(s, out=out)
            kw.pop("max_new"), kw.pop("max_kv")
            hb.kv8_attention(max_new=s["max_new"], max_kv=s["max_kv"], scale=0.001, sync=False,
                             **kw)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    for _ in range(3):
        out.zero_()
        other.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, cache)
        torch.randn((1 << 20,), device=DEV).sum()
