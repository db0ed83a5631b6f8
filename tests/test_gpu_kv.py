"""The serving operators on an MI355X against plain 64-bit implementations:
step plans, norm and rotation, cache rows, and attention over the paged MXFP4
cache, at the sizes, masks and contents where they can go wrong.

Tolerances.  A rounding to type t is off by at most eps(t) / 2 of the value.
Norm and rotation: the output's rounding, and 32-bit arithmetic over dim + 16
roundings of the pair's magnitude.  Attention, of a row with weights p and
A = sum p |v|: the output's rounding; 2 ds A for scores off by ds (the
products' sum over dim terms and the few operations after it); the weights'
own rounding (2^-11 A in f16 for the 16-bit types, none for fp32); 2^-24 A a
term for the sums over the keys; 2^-21 A for exponentials and the division."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import hotarubi_amd as hb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}
TYPES = list(HALF)
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)


def say(*what):
    print(*what, flush=True)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ plan --

def plan_reference(lens, new, free, count, table, page, size):
    table = table.copy()
    cu, kv, taken, wanted, refused = [0], [], 0, 0, 0
    slots, positions = np.full(size, -1, np.int64), np.full(size, -1, np.int64)
    count = max(0, min(count, len(free)))
    for b in range(len(lens)):
        have, more = max(0, lens[b]), max(0, new[b])
        old, pages = -(-have // page), -(-(have + more) // page)
        fits = pages <= table.shape[1] and cu[-1] + more <= size
        need = pages - old if fits else 0
        ok = fits and (need == 0 or wanted + need <= count)
        if ok:
            for i in range(need):
                table[b, old + i] = free[count - 1 - wanted - i]
            taken += need
        refused += not ok
        wanted += need
        for i in range(more):
            at = cu[-1] + i
            if at < size:
                positions[at] = have + i
                if ok and table[b, (have + i) // page] >= 0:
                    slots[at] = table[b, (have + i) // page] * page + (have + i) % page
        cu.append(cu[-1] + more)
        kv.append(have + more if ok else have)
    return table, cu, kv, slots, positions, [taken, refused]


def run_plan(gpu, lens, new, free, count, table, page, size):
    t, out = ints(table), [ints([7] * n) for n in (len(lens) + 1, len(lens), size, size, 2)]
    hb.kv_plan(lens=ints(lens), new_tokens=ints(new), free_pages=ints(free),
               free_count=ints([count]), table=t, page_size=page, cu=out[0], kv_lens=out[1],
               slots=out[2], positions=out[3], status=out[4], ctx=gpu)
    return [t] + out


@pytest.mark.parametrize("batch,page,most,slack,pages", [
    (1, 32, 1, 0, 0), (1, 32, 200, 3, 0), (64, 64, 1, 5, 0), (257, 32, 40, 0, -5),
    (1024, 128, 3, 100, 0), (1025, 32, 70, -200, 0), (2500, 96, 30, 7, -100), (40, 32, 3000, 0, 0)])
def test_plan(gpu, batch, page, most, slack, pages):
    say("plan", batch, page, most, slack, pages)
    rng = np.random.default_rng(batch + page)
    lens = rng.integers(0, 500, batch)
    new = np.where(rng.random(batch) < 0.2, 0, rng.integers(1, most + 1, batch))
    cols = int((lens + new).max()) // page + 1
    if batch > 300:
        cols -= 2  # some requests pass the table's columns
    have = -(-lens // page)
    need = int((-(-(lens + new) // page) - have).sum())
    free = rng.permutation(need + 1 + int(have.sum())).astype(np.int64)
    table = np.full((batch, cols), -1, np.int64)
    for b in range(batch):
        table[b, :have[b]] = rng.integers(0, 10000, min(have[b], cols))
    count = max(0, need + pages)
    size = max(1, int(new.sum()) + slack)
    got = run_plan(gpu, lens, new, free, count, table, page, size)
    want = plan_reference(lens, new, free, count, table, page, size)
    for name, g, w in zip(("table", "cu", "kv_lens", "slots", "positions", "status"), got, want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w)), name


def test_plan_of_nothing_and_of_bad_numbers(gpu):
    say("plan of nothing")
    got = run_plan(gpu, [], [], [1, 2], 2, np.zeros((0, 4)), 32, 3)
    assert [g.tolist() for g in got[1:]] == [[0], [], [-1] * 3, [-1] * 3, [0, 0]]
    got = run_plan(gpu, [5], [0], [], 0, np.array([[3]]), 32, 0)
    assert got[1].tolist() == [0, 0] and got[2].tolist() == [5] and got[5].tolist() == [0, 0]
    # negative lengths count as 0, a free count past the stack as its size, a
    # table entry of -1 gives no slot
    lens, new = [-4, 10, 3], [3, -2, 2]
    table = np.array([[-1, -1], [4, -1], [-1, -1]])
    got = run_plan(gpu, lens, new, [8], 100, table, 32, 6)
    want = plan_reference(lens, new, [8], 100, table, 32, 6)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w))


def test_plan_with_a_strided_table(gpu):
    say("plan, strided table")
    wide = ints(np.full((3, 9), 55))
    table = wide[:, 2:6]
    table[:] = -1
    out = [ints([0] * n) for n in (4, 3, 40, 40, 2)]
    hb.kv_plan(lens=ints([0, 0, 0]), new_tokens=ints([33, 1, 2]), free_pages=ints(list(range(9))),
               free_count=ints([9]), table=table, page_size=32, cu=out[0], kv_lens=out[1],
               slots=out[2], positions=out[3], status=out[4], ctx=gpu)
    assert table.tolist() == [[8, 7, -1, -1], [6, -1, -1, -1], [5, -1, -1, -1]]
    assert (wide[:, :2] == 55).all() and (wide[:, 6:] == 55).all()


# ------------------------------------------------------------------ rope --

def rope_reference(x, gamma, positions, inv_freq, sections, interleaved, eps):
    y = x.double()
    if gamma is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * gamma.double()
    half = inv_freq.shape[0]
    axis = [i for i, n in enumerate(sections) for _ in range(n)]
    angle = positions.double()[axis].T * inv_freq if half else positions.new_zeros((x.shape[0], 0))
    c, s = angle.double().cos()[:, None], angle.double().sin()[:, None]
    out, size = y.clone(), y.abs()
    a = y[..., 0:2 * half:2] if interleaved else y[..., :half]
    b = y[..., 1:2 * half:2] if interleaved else y[..., half:2 * half]
    at, bt = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else \
        (slice(0, half), slice(half, 2 * half))
    out[..., at], out[..., bt] = a * c - b * s, b * c + a * s
    size[..., at] = size[..., bt] = a.abs() + b.abs()
    return out, size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hq,hk,dim,rot,axes,interleaved", [
    (1, 1, 1, 64, 64, 1, False), (16, 15, 5, 64, 64, 1, False), (16, 15, 5, 64, 32, 1, True),
    (5, 3, 1, 96, 96, 1, False), (7, 12, 12, 96, 48, 2, True), (33, 32, 8, 128, 128, 3, False),
    (3, 8, 4, 256, 128, 3, True), (9, 2, 1, 512, 512, 1, False), (4, 3, 2, 2, 2, 1, False),
    (5, 2, 2, 30, 14, 1, False), (5, 2, 2, 30, 14, 1, True), (6, 4, 0, 128, 0, 1, False),
    (5000, 3, 1, 64, 64, 1, False)])
def test_norm_rope(gpu, dtype, tokens, hq, hk, dim, rot, axes, interleaved):
    say("norm_rope", dtype, tokens, hq, hk, dim, rot, axes, interleaved)
    gen = torch.Generator(device=DEV).manual_seed(tokens + dim)
    x = torch.randn((tokens, hq + 2 * hk, dim), generator=gen, device=DEV).to(dtype)
    half = rot // 2
    sections = {1: (half,), 2: (half // 3, half - half // 3),
                3: (half // 4, half // 4, half - 2 * (half // 4))}[axes]
    pos = torch.randint(-5, 1 << 20, (axes, tokens), generator=gen, device=DEV, dtype=torch.int32)
    pos[:, 0] = 0
    freq = 100000.0 ** -(torch.arange(half, device=DEV, dtype=torch.float64) / max(1, half))
    gamma = 1 + 0.3 * torch.randn((2, dim), generator=gen, device=DEV)
    q, k = x[:, :hq], x[:, hq:hq + hk]
    for norm in (True, False):
        gq, gk = (gamma[0], gamma[1]) if norm else (None, None)
        oq, ok = torch.empty((tokens, hq, dim), dtype=dtype, device=DEV), None
        if hk:
            ok = torch.empty((tokens, hk, dim), dtype=dtype, device=DEV)
        hb.norm_rope(q=q, k=k if hk else None, positions=pos, inv_freq=freq, q_out=oq, k_out=ok,
                     gamma_q=gq, gamma_k=gk, eps=1e-5, sections=sections, interleaved=interleaved,
                     ctx=gpu)
        for got, src, g in ((oq, q, gq), (ok, k, gk)):
            if got is None:
                continue
            want, size = rope_reference(src, g, pos, freq, sections, interleaved, 1e-5)
            tol = HALF[dtype] * want.abs() + (dim + 16) * 2.0**-24 * size + TINY[dtype]
            assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_rope_strides_and_in_place(gpu, dtype):
    say("norm_rope strides", dtype)
    gen = torch.Generator(device=DEV).manual_seed(3)
    raw = torch.randn((11 * 7 * 67 + 1,), generator=gen, device=DEV).to(dtype)
    q = raw[1:].view(11, 7, 67)[:, 1:5, 2:66]  # no alignment of any kind
    k = raw[1:].view(11, 7, 67)[:, 5:, 3:67]
    pos = torch.arange(22, device=DEV, dtype=torch.int32).view(11, 2).T[:1]
    pos = pos.contiguous()
    freq = 10.0 ** -torch.arange(32, device=DEV, dtype=torch.float64)
    gamma = torch.ones(64, device=DEV)
    want = [rope_reference(x, gamma, pos, freq, (32,), False, 1e-6) for x in (q, k)]
    hq, hk = (torch.empty((4, 11, 64), dtype=dtype, device=DEV).transpose(0, 1),
              torch.empty((2, 11, 64), dtype=dtype, device=DEV).transpose(0, 1))
    kw = dict(positions=pos[0], inv_freq=freq, gamma_q=gamma, gamma_k=gamma, ctx=gpu)
    hb.norm_rope(q=q, k=k, q_out=hq, k_out=hk, **kw)
    hb.norm_rope(q=q, k=k, q_out=q, k_out=k, **kw)
    for outs in ((hq, hk), (q, k)):
        for got, (w, size) in zip(outs, want):
            tol = HALF[dtype] * w.abs() + 80 * 2.0**-24 * size + TINY[dtype]
            assert ((got.double() - w).abs() <= tol).all()


# ------------------------------------------------------------ cache rows --

def encode_reference(x):
    """fp64 [t][h][d] -> stored values, fp64; NaN rows as the caller marks them."""
    t, h, d = x.shape
    y = x.reshape(t, h, d // 32, 32)
    top = np.abs(y).max(-1, keepdims=True)
    e = np.where(top > 0, np.floor(np.log2(np.where(top > 0, top, 1))), 0)
    e = np.where(top > 0, np.where(np.exp2(e) > top, e - 1, e), e)
    e = np.where((top > 0) & (np.exp2(e + 1) <= top), e + 1, e) - 2 * (top > 0)
    unit = np.exp2(np.clip(e, -126, 125))
    m = np.minimum(np.abs(y) / unit, 6)
    hi = np.clip(np.searchsorted(GRID, m), 1, 7)
    lo = hi - 1
    up = (m - GRID[lo] > GRID[hi] - m) | ((m - GRID[lo] == GRID[hi] - m) & (hi % 2 == 0))
    return (np.copysign(np.where(up, GRID[hi], GRID[lo]), y) * unit).reshape(t, h, d)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 64, 32), (64, 8, 128, 64),
                                                   (700, 5, 64, 96), (33, 2, 256, 128),
                                                   (129, 3, 128, 32)])
def test_append_and_read(gpu, dtype, tokens, heads, dim, page):
    say("append", dtype, tokens, heads, dim, page)
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    pages = -(-tokens // page) + 2
    k, v = (torch.randn((tokens, heads, dim), generator=gen, device=DEV) * torch.exp(
        2 * torch.randn((tokens, heads, 1), generator=gen, device=DEV)) for _ in range(2))
    # values on and next to the grid's borders, in blocks of maximum 4..6
    edge = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 0, -.25, -5, 4, 7.99], device=DEV)
    k[0, 0, :32] = edge[torch.arange(32, device=DEV) % 12]
    v[0, 0, :32] = torch.nextafter(k[0, 0, :32], torch.full((32,), 9.0, device=DEV))
    v[0, 0, 32:] = 0
    if tokens > 20:
        k[3] *= 2.0**-140 if dtype is torch.float32 else 2.0**-20  # subnormal rows
        k[4] *= 2.0**119 if dtype is torch.float32 else 2.0**7
        k[5, 0, 1], v[6, 0, dim - 1], k[7, heads - 1, 0] = math.inf, -math.inf, math.nan
    k, v = k.to(dtype), v.to(dtype)
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:tokens].to(torch.int32)
    if tokens > 20:
        slots[10:13] = ints([-1, pages * page, -2**31])
    cache = torch.full(hb.kv_cache_shape(pages, heads, page, dim), 0x77, dtype=torch.uint8,
                       device=DEV)
    hb.kv_append(k=k, v=v, slots=slots, cache=cache, ctx=gpu)
    inside = (slots >= 0) & (slots < pages * page)
    bad = ~(k.isfinite().all(-1) & v.isfinite().all(-1)).cpu().numpy()
    wk, wv = (encode_reference(np.where(bad[..., None], 0, x.double().cpu().numpy()))
              for x in (k, v))
    wk[bad] = np.nan
    out = inside.cpu().numpy()
    wk[~out], wv[~out] = 0, 0
    for to in TYPES:
        gk, gv = (torch.full((tokens, heads, dim), 3.0, dtype=to, device=DEV) for _ in range(2))
        hb.kv_read(k=gk, v=gv, slots=slots, cache=cache, ctx=gpu)
        for got, want in ((gk, wk), (gv, wv)):
            want = torch.from_numpy(want).to(DEV).to(to)  # rounds where `to` is narrower
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(torch.nan_to_num(got, 9), torch.nan_to_num(want, 9))
    # only the slots' bytes were written: 17 dim / 16 bytes a token and head
    changed = (cache != 0x77).sum().item()
    assert changed <= int(inside.sum()) * heads * 17 * dim // 16


@pytest.mark.parametrize("dtype", TYPES)
def test_append_strides(gpu, dtype):
    say("append strides", dtype)
    gen = torch.Generator(device=DEV).manual_seed(5)
    raw = torch.randn((40 * 5 * 131 + 1,), generator=gen, device=DEV).to(dtype)[1:]
    k, v = raw.view(40, 5, 131)[:, :2, 1:129], raw.view(40, 5, 131)[:, 3:, 3:131]
    slots = torch.arange(40, device=DEV, dtype=torch.int32)
    a, b = (torch.zeros(hb.kv_cache_shape(2, 2, 32, 128), dtype=torch.uint8, device=DEV)
            for _ in range(2))
    hb.kv_append(k=k, v=v, slots=slots, cache=a, ctx=gpu)
    hb.kv_append(k=k.contiguous(), v=v.contiguous(), slots=slots, cache=b, ctx=gpu)
    assert torch.equal(a, b)
    gk = torch.empty((2, 40, 129), dtype=dtype, device=DEV).transpose(0, 1)[..., 1:]
    gv = torch.empty_like(k.contiguous())
    hb.kv_read(k=gk, v=gv, slots=slots, cache=a, ctx=gpu)
    want = torch.from_numpy(encode_reference(k.double().cpu().numpy())).to(DEV).to(dtype)
    assert torch.equal(gk, want)


# ------------------------------------------------------------- attention --

def record_map(dim):
    """Byte offsets in a record: K and V codes [32][dim], K and V scales [32][dim]."""
    at = np.zeros((4, 32, dim), np.int64)
    for t in range(32):
        n, tile, g, j = t % 16, t // 16, t % 16 // 4, t % 4 + 4 * (t // 16)
        for col in range(dim):
            w = tile * (dim // 8) + col % (dim // 4) // 2
            at[0, t, col] = w // 16 * 1024 + col // (dim // 4) * 256 + n * 16 + w % 16
            w = j * (dim // 32) + col % (dim // 16) // 2
            at[1, t, col] = 16 * dim + w // 16 * 1024 + g * 256 + col // (dim // 16) * 16 + w % 16
            at[2, t, col] = 32 * dim + col // 32 * 32 + n * 2 + tile
            at[3, t, col] = 33 * dim + col // 32 * 32 + g * 8 + j
    return torch.from_numpy(at).to(DEV)


def decode_reference(cache, page_ids, head, dim):
    """K, V fp64 [len(page_ids) * page][dim]; a page id outside the cache gives zeros."""
    at = record_map(dim)
    ok = (page_ids >= 0) & (page_ids < cache.shape[0])
    rec = cache[torch.where(ok, page_ids, 0).long(), head].reshape(-1, 34 * dim)
    col = torch.arange(dim, device=DEV) % 2 * 4
    grid = torch.tensor(np.concatenate([GRID, -GRID]), device=DEV)
    out = []
    for codes, scales in ((at[0], at[2]), (at[1], at[3])):
        code = (rec[:, codes].int() >> col) & 15
        e = rec[:, scales].double()
        x = grid[code] * torch.where(e == 255, math.nan, torch.exp2(e - 127))
        out.append(x.reshape(-1, dim))
    return out[0], out[1], ok.repeat_interleave(cache.shape[2] * 32)


def attention_reference(q, cache, table, cu, kv_lens, scale, prefix, window, cap, max_new):
    """fp64 output, and the row's tolerance without the output's rounding."""
    tokens, hq, d = q.shape
    hk, page = cache.shape[1], cache.shape[2] * 32
    group, out = hq // hk, torch.zeros((tokens, hq, d), dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    mine = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    half = q.dtype is not torch.float32
    for b in range(table.shape[0]):
        n, total = int(cu[b + 1] - cu[b]), int(kv_lens[b])
        rows = slice(int(cu[b]), int(cu[b]) + min(n, max_new))
        mine[rows] = True
        if n == 0 or total == 0:
            continue
        i = torch.arange(min(n, max_new), device=DEV)[:, None]
        pos, key = total - n + i, torch.arange(total, device=DEV)
        see = key <= pos
        if window:
            see = see & (pos - key < window)
        if prefix is not None:
            see = see | (key < int(prefix[b]))
        for h in range(hk):
            k, v, ok = decode_reference(cache, table[b, :-(-total // page)], h, d)
            k, v, ok = k[:total], v[:total], ok[:total]
            dead = k.isnan().any(-1) | v.isnan().any(-1)
            for g in range(h * group, (h + 1) * group):
                x = q[rows, g].double()
                s = x @ torch.nan_to_num(k).T * scale
                ds = (d + 8) * 2.0**-24 * (x.abs() @ torch.nan_to_num(k).abs().T * abs(scale))
                if cap:
                    s = cap * torch.tanh(s / cap)
                    ds = ds + cap * 2.0**-21
                s = torch.where(dead, math.nan, s).masked_fill(~(see & ok), -math.inf)
                top = torch.nan_to_num(s, nan=-math.inf).amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(top.isinf(), 0, top))
                total_p = p.sum(-1, keepdim=True)
                p = torch.where(total_p == 0, 0, p / total_p)
                vv = torch.nan_to_num(v)
                out[rows, g] = p @ vv
                size = p @ vv.abs()
                ds = torch.where(see & ok, ds, 0).amax(-1, keepdim=True)
                tol[rows, g] = size * (2 * ds + (2.0**-11 if half else 0) + total * 2.0**-23 +
                                       2.0**-21) + total * 2.0**-32 * vv.abs().amax()
    return out, tol, mine


def make_cache(gen, pages, heads, page, dim, lo=122, hi=128):
    cache = torch.randint(0, 256, hb.kv_cache_shape(pages, heads, page, dim), generator=gen,
                          device=DEV, dtype=torch.int32).to(torch.uint8)
    cache[..., 32 * dim:] = torch.randint(lo, hi, cache[..., 32 * dim:].shape, generator=gen,
                                          device=DEV, dtype=torch.int32).to(torch.uint8)
    return cache


def build(gen, requests, page, heads, dim, dtype, hq, spare=2, **kw):
    """requests: (keys, new, prefix)."""
    used = [-(-k // page) for k, _, _ in requests]
    cache = make_cache(gen, sum(used) + spare, heads, page, dim, **kw)
    perm = torch.randperm(cache.shape[0], generator=gen, device=DEV).tolist()
    table = np.full((len(requests), max(used + [1]) + 1), -1, np.int64)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = perm[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum([n for _, n, _ in requests])])
    q = torch.randn((int(cu[-1]), hq, dim), generator=gen, device=DEV).to(dtype)
    return dict(q=q, cache=cache, table=ints(table), cu=ints(cu),
                kv_lens=ints([k for k, _, _ in requests]),
                prefix=ints([p for _, _, p in requests]) if any(p for _, _, p in requests) else None,
                max_new=max(n for _, n, _ in requests), max_kv=max(k for k, _, _ in requests))


def check(gpu, s, scale=None, window=0, cap=0.0, out=None, same=True):
    q, d = s["q"], s["q"].shape[-1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.full_like(q, 7.0) if out is None else out
    kw = dict(q=q, cache=s["cache"], table=s["table"], cu=s["cu"], kv_lens=s["kv_lens"],
              max_new=s["max_new"], max_kv=s["max_kv"], scale=scale, prefix=s["prefix"],
              window=window, softcap=cap, ctx=gpu)
    hb.kv_attention(out=out, **kw)
    want, tol, mine = attention_reference(q, s["cache"], s["table"], s["cu"], s["kv_lens"], scale,
                                          s["prefix"], window, cap, s["max_new"])
    got = out.double()
    assert torch.equal(got[mine].isnan(), want[mine].isnan())
    tol = tol + HALF[q.dtype] * want.abs() + TINY[q.dtype]
    most = torch.finfo(q.dtype).max  # what rounds past it is an infinity
    over = mine[:, None, None] & (want.abs() - tol > most * (1 + HALF[q.dtype]))
    assert (got[over] == torch.sign(want[over]) * math.inf).all()
    there = mine[:, None, None] & ~want.isnan() & (want.abs() + tol < most)
    worst = ((got - want).abs() / tol)[there].max().item() if there.any() else 0.0
    assert worst <= 1, f"{worst} of the tolerance"
    assert (out[~mine] == 7.0).all() or not same
    again = torch.full_like(q, 5.0)
    hb.kv_attention(out=again, **kw)
    assert torch.equal(torch.nan_to_num(again[mine]), torch.nan_to_num(out[mine]))
    return out


CASES = {
    "one key": ([(1, 1, 0)], {}),
    "one token": ([(191, 1, 0)], {}),
    "decode": ([(33, 1, 0), (1, 1, 0), (500, 1, 0), (32, 1, 0), (129, 1, 0)], {}),
    "few": ([(70, 3, 0), (9, 9, 0), (300, 5, 0), (64, 1, 0)], {}),
    "chunk": ([(191, 50, 141), (180, 50, 140), (50, 50, 0)], {}),
    "prompt": ([(300, 300, 0), (517, 190, 37)], {}),
    "window": ([(400, 130, 0), (90, 90, 0), (1000, 3, 0)], dict(window=64)),
    "window of one": ([(77, 20, 0)], dict(window=1)),
    "window and prefix": ([(700, 40, 100), (700, 40, 33)], dict(window=33)),
    "capped": ([(200, 20, 0), (999, 1, 0)], dict(cap=3.0, scale=0.5)),
    "negative scale": ([(100, 7, 0)], dict(scale=-0.3)),
    "scale of zero": ([(100, 7, 0)], dict(scale=0.0)),
    "empty requests": ([(0, 0, 0), (60, 4, 0), (90, 0, 0), (0, 0, 0), (5, 5, 0)], {}),
    # rows before their request's first key, and requests without any
    "no keys": ([(3, 8, 0), (0, 4, 0), (40, 2, 0)], {}),
    "no keys, many rows": ([(70, 200, 0), (0, 100, 0)], {}),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(15, 5, 64, 32), (4, 4, 128, 96), (32, 1, 128, 64),
                                   (8, 2, 256, 128)])
@pytest.mark.parametrize("case", list(CASES))
def test_attention(gpu, dtype, heads, case):
    say("attention", dtype, heads, case)
    hq, hk, dim, page = heads
    requests, kw = CASES[case]
    gen = torch.Generator(device=DEV).manual_seed(len(case) + dim)
    check(gpu, build(gen, requests, page, hk, dim, dtype, hq), **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_many_rows(gpu, dtype, dim):
    """Every way of dividing the work: enough rows for the prompt kernel, for
    waves with rows of their own, for two tiles a wave."""
    gen = torch.Generator(device=DEV).manual_seed(dim)
    for requests, hq, hk in ([[(260, 200, 70)] * 24, 12, 12], [[(900, 128, 0), (300, 128, 0)] * 8, 16, 4],
                             [[(2100, 1100, 0), (1300, 1000, 50)], 24, 8]):
        if dtype is torch.float32 and dim == 256:
            requests = requests[:8]
        say("many rows", dtype, dim, len(requests), hq, hk)
        check(gpu, build(gen, requests, 64, hk, dim, dtype, hq))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_ragged_long_requests(gpu, dtype):
    """Shares over requests of very different lengths, and waves of more than
    128 records; the requests share their pages, so the cache is small."""
    say("ragged", dtype)
    gen = torch.Generator(device=DEV).manual_seed(9)
    heads, dim, page = 8, 64, 64
    cache = make_cache(gen, 64, heads, page, dim)
    lens = [17000 + 13 * b for b in range(60)] + [1, 40, 0, 3000]
    cols = max(lens) // page + 1
    table = torch.randint(0, 64, (64, cols), generator=gen, device=DEV, dtype=torch.int32)
    q = torch.randn((64, 16, dim), generator=gen, device=DEV).to(dtype)
    check(gpu, dict(q=q, cache=cache, table=table, cu=ints(list(range(65))), kv_lens=ints(lens),
                    prefix=None, max_new=1, max_kv=max(lens)))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_one_long_request(gpu, dtype):
    say("long", dtype)
    gen = torch.Generator(device=DEV).manual_seed(4)
    check(gpu, build(gen, [(30011, 2, 0)], 128, 2, 128, dtype, 8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 200])
def test_attention_bad_pages(gpu, dtype, rows):
    """Table entries that name no page hide their keys; what lies past a
    request's end is not looked at."""
    say("bad pages", dtype, rows)
    gen = torch.Generator(device=DEV).manual_seed(rows)
    hk = 32 if rows > 1 else 2
    s = build(gen, [(400, rows, 0), (330, rows, 100)] * (4 if rows > 1 else 1), 32, hk, 128, dtype,
              hk)
    s["table"][0, 3], s["table"][0, 5] = -1, s["cache"].shape[0]
    s["table"][1, 0], s["table"][1, 9] = 2**31 - 1, -2**31
    check(gpu, s)
    s["table"][0, :] = -1  # nothing left
    out = check(gpu, s)
    assert (out[:rows] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_unusual_bytes(gpu, dtype, rows, dim):
    """Scales over the whole range, NaN tokens, and anything at all past the
    request's end."""
    say("unusual bytes", dtype, rows, dim)
    gen = torch.Generator(device=DEV).manual_seed(dim + rows)
    hk = 40 if rows > 1 else 2
    base = build(gen, [(300, rows, 0), (270, rows, 10)] * (2 if rows > 1 else 1), 32, hk, dim, dtype,
                 hk)
    table = base["table"].long()

    def scales(t, b, value, which):  # of token t of request b
        off = record_map(dim)[which, t % 32].unique()
        base["cache"][table[b, t // 32], :, 0, off] = value

    for b, keys in ((0, 300), (1, 270)):  # the last page's unused tokens
        for t in range(keys % 32, 32):
            off = record_map(dim)[:, t].reshape(-1).unique()
            base["cache"][table[b, keys // 32], :, 0, off] = 0xFF
    check(gpu, base)
    # V far outside f16's range, up and down, next to ordinary tokens
    for t, value in ((5, 150), (6, 90), (7, 20), (40, 141), (41, 103)):
        scales(t, 0, value, 3)
    check(gpu, base)
    for t, value in ((8, 100), (9, 60), (10, 1)):
        scales(t, 0, value, 2)
    check(gpu, base)
    # NaN tokens: one that only late rows see, one in V alone
    scales(299 if rows == 1 else 250, 0, 255, 2)
    scales(20, 1, 255, 3)
    check(gpu, base)
    check(gpu, base, window=64)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides(gpu, dtype):
    say("attention strides", dtype)
    gen = torch.Generator(device=DEV).manual_seed(2)
    for requests, hq, hk in ([[(90, 3, 0), (40, 2, 0)], 4, 2], [[(300, 256, 0)] * 4, 32, 32]):
        s = build(gen, requests, 32, hk, 64, dtype, hq)
        plain = check(gpu, s)
        tokens = s["q"].shape[0]
        wide = torch.zeros((tokens, hq, 67), dtype=dtype, device=DEV)
        wide[..., 3:] = s["q"]
        table = torch.zeros((len(requests), s["table"].shape[1] + 5), dtype=torch.int32, device=DEV)
        table[:, 2:-3] = s["table"]
        out = torch.full((hq, tokens, 65), 7.0, dtype=dtype, device=DEV).transpose(0, 1)[..., 1:]
        t = dict(s, q=wide[..., 3:], table=table[:, 2:-3])
        check(gpu, t, out=out)
        assert torch.equal(out, plain)


def test_attention_past_32_bits_of_cache(gpu):
    """Pages whose bytes start past 4 GiB, against the same pages in a small cache."""
    say("past 4 GiB")
    gen = torch.Generator(device=DEV).manual_seed(8)
    s = build(gen, [(500, 3, 0), (200, 100, 0)], 128, 4, 256, torch.bfloat16, 8)
    small = check(gpu, s)
    n, pages = s["cache"].shape[0], 4 * 2**30 // (4 * 4 * 34 * 256) + 50
    big = torch.zeros(hb.kv_cache_shape(pages, 4, 128, 256), dtype=torch.uint8, device=DEV)
    big[pages - n:] = s["cache"]
    out = torch.empty_like(small)
    table = torch.where(s["table"] >= 0, s["table"] + (pages - n), s["table"]).to(torch.int32)
    kw = dict(cu=s["cu"], kv_lens=s["kv_lens"], max_new=100, max_kv=500, scale=256 ** -0.5, ctx=gpu)
    hb.kv_attention(q=s["q"], out=out, cache=big, table=table, **kw)
    assert torch.equal(out, small)
    # rows written and read back there
    slots = ints([pages * 128 - 1, pages * 128 - 200])
    k, v = (torch.randn((2, 4, 256), generator=gen, device=DEV) for _ in range(2))
    gk, gv = torch.empty_like(k), torch.empty_like(v)
    hb.kv_append(k=k, v=v, slots=slots, cache=big, ctx=gpu)
    hb.kv_read(k=gk, v=gv, slots=slots, cache=big, ctx=gpu)
    assert torch.equal(gk.cpu(), torch.from_numpy(encode_reference(k.double().cpu().numpy())).float())


def test_rows_and_requests_past_the_bounds_are_not_computed(gpu):
    say("bounds")
    gen = torch.Generator(device=DEV).manual_seed(6)
    s = build(gen, [(60, 9, 0), (50, 4, 0)], 32, 2, 64, torch.bfloat16, 4)
    s["max_new"] = 5  # rows 5 .. 8 of the first request stay as they are
    check(gpu, s)
    s["max_kv"] = 1  # only a hint of the work
    check(gpu, s)
    q = s["q"]
    out = torch.full_like(q, 7.0)
    for cu, kv in (([0, 2**31 - 1, 5], [60, 50]), ([-3, 4, 13], [60, 2**31 - 1]),
                   ([9, 3, 1], [-7, 50])):  # nonsense stays inside the tensors
        hb.kv_attention(q=q, out=out, cache=s["cache"], table=s["table"], cu=ints(cu),
                        kv_lens=ints(kv), max_new=9, max_kv=60, scale=0.1, ctx=gpu)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_past_max_kv_are_seen_by_prompts(gpu, dtype, dim):
    """max_kv is too small: what it lays out does not hold every record."""
    say("prompt past max_kv", dtype, dim)
    gen = torch.Generator(device=DEV).manual_seed(dim + 1)
    s = build(gen, [(700, 128, 0), (190, 128, 20)] * 4, 64, 4, dim, dtype, 16)
    for most in (1, 200, 699):
        check(gpu, dict(s, max_kv=most))
        check(gpu, dict(s, max_kv=most), window=100)


@pytest.mark.parametrize("dtype", TYPES)
def test_keys_past_max_kv_are_seen_by_ragged_requests(gpu, dtype):
    say("ragged past max_kv", dtype)
    gen = torch.Generator(device=DEV).manual_seed(12)
    heads, dim, page = 8, 64, 64
    cache = make_cache(gen, 64, heads, page, dim)
    lens = [3000 + 701 * (b % 7) for b in range(64)]
    table = torch.randint(0, 64, (64, max(lens) // page + 1), generator=gen, device=DEV,
                          dtype=torch.int32)
    q = torch.randn((64, 16, dim), generator=gen, device=DEV).to(dtype)
    for most in (1, 2000):
        check(gpu, dict(q=q, cache=cache, table=table, cu=ints(list(range(65))),
                        kv_lens=ints(lens), prefix=None, max_new=1, max_kv=most))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_with_window_prefix_and_missing_pages(gpu, dtype, dim):
    """The records a prompt looks at are two ranges, with pages missing in both."""
    say("prompt, two ranges", dtype, dim)
    gen = torch.Generator(device=DEV).manual_seed(dim + 2)
    s = build(gen, [(1100, 260, 200), (900, 200, 40), (300, 300, 0)] * 3, 32, 4, dim, dtype, 16)
    check(gpu, s, window=100)
    s["table"][0, 1], s["table"][0, 30], s["table"][1, 0] = -1, s["cache"].shape[0], -7
    s["table"][2, 8:] = -1
    check(gpu, s, window=100)
    check(gpu, s, window=500, cap=2.0)


# ------------------------------------------------------------ as a step --

def step(ctx, st, sync=False):
    hb.kv_plan(lens=st["lens"], new_tokens=st["new"], free_pages=st["free"], free_count=st["count"],
               table=st["table"], page_size=32, cu=st["cu"], kv_lens=st["kv"], slots=st["slots"],
               positions=st["pos"], status=st["status"], ctx=ctx, sync=sync)
    q, k, v = st["qkv"][:, :6], st["qkv"][:, 6:8], st["qkv"][:, 8:]
    hb.norm_rope(q=q, k=k, positions=st["pos"], inv_freq=st["freq"], q_out=st["q"], k_out=st["k"],
                 gamma_q=st["gamma"], gamma_k=st["gamma"], ctx=ctx, sync=sync)
    hb.kv_append(k=st["k"], v=v, slots=st["slots"], cache=st["cache"], ctx=ctx, sync=sync)
    hb.kv_attention(q=st["q"], out=st["out"], cache=st["cache"], table=st["table"], cu=st["cu"],
                    kv_lens=st["kv"], max_new=st["max_new"], max_kv=400, scale=0.125, ctx=ctx,
                    sync=sync)


def step_state(seed, new):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n, b = sum(new), len(new)
    return dict(lens=ints([0] * b), new=ints(new), free=ints(list(range(40))), count=ints([40]),
                table=ints(np.full((b, 13), -1)), cu=ints([0] * (b + 1)), kv=ints([0] * b),
                slots=ints([0] * n), pos=ints([0] * n), status=ints([0, 0]), max_new=max(new),
                qkv=torch.randn((n, 10, 64), generator=gen, device=DEV).bfloat16(),
                freq=10000.0 ** -(torch.arange(32, device=DEV, dtype=torch.float64) / 32),
                gamma=torch.ones(64, device=DEV),
                q=torch.empty((n, 6, 64), dtype=torch.bfloat16, device=DEV),
                k=torch.empty((n, 2, 64), dtype=torch.bfloat16, device=DEV),
                cache=torch.zeros(hb.kv_cache_shape(40, 2, 32, 64), dtype=torch.uint8, device=DEV),
                out=torch.zeros((n, 6, 64), dtype=torch.bfloat16, device=DEV))


def test_prompt_at_once_or_token_by_token(gpu):
    """A prompt of 70 tokens in one step gives the rows that 70 steps give."""
    say("prompt against decode")
    whole = step_state(1, [70, 3])
    step(gpu, whole)
    one = step_state(1, [1, 0])
    one["cache"], outs = torch.zeros_like(whole["cache"]), []
    for i in range(70):
        one["qkv"] = whole["qkv"][i:i + 1]
        step(gpu, one)
        torch.cuda.synchronize()
        one["count"] -= one["status"][0]
        one["lens"] = one["kv"].clone()
        outs.append(one["out"].clone())
    got, want = torch.cat(outs).double(), whole["out"][:70].double()
    # two sums of the same terms: each within its tolerance of the exact one
    assert ((got - want).abs() <= 2 * (2.0**-8 * want.abs() + 2.0**-9)).all()


def test_captured_step_replays_like_the_eager_one(gpu):
    say("graph")
    stream = torch.cuda.Stream()
    ctx = hb.Context(0)
    ctx.set_stream(stream.cuda_stream)
    st = step_state(2, [40, 1, 1, 9])
    with torch.cuda.stream(stream):
        step(ctx, st)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(ctx, st)
    for seed in range(3, 7):  # other inputs in the same buffers, eager work between
        new = step_state(seed, [40, 1, 1, 9])
        step(gpu, new)
        torch.cuda.synchronize()
        for name in ("qkv", "lens", "free"):
            st[name].copy_(new[name])
        st["table"].fill_(-1)
        st["cache"].zero_()
        st["out"].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for name in ("out", "cache", "table", "slots", "pos", "cu", "kv"):
            assert torch.equal(st[name], new[name]), name
    ctx.close()


def test_another_stream(gpu):
    """Work ordered on a context's stream alone, while the default stream is busy."""
    say("stream")
    want = step_state(11, [33, 2])
    step(gpu, want)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    ctx = hb.Context(0)
    ctx.set_stream(stream.cuda_stream)
    st = step_state(11, [33, 2])
    torch.cuda.synchronize()
    busy = torch.randn((4096, 4096), device=DEV)
    for _ in range(5):
        busy = busy @ busy * 1e-4
    step(ctx, st)
    stream.synchronize()
    assert torch.equal(st["out"], want["out"]) and torch.equal(st["cache"], want["cache"])
    ctx.close()
