"""Performance cases of the serving operators: attention over a paged cache
held in MXFP4, and what feeds it.

Every case is a plain dict; `kind` names the operator, the other values its
sizes, types and masks:

  plan       block tables, slot maps and positions of a step, from the
             requests' lengths (kv_plan)
  rope       RMS norm of every query and key head and the rotation by
             position, one pass (norm_rope)
  append     K and V rows into the cache as MXFP4, and the stored values
             back out by slot (kv_append, kv_read)
  attention  ragged requests over the paged cache: a new token each, a few,
             or a prompt; prefix mask, window, capped scores (kv_attention)

The cache is uint8 [pages][heads][page / 32][34 D]: a record per 32 tokens of
one head holding K codes (16 D bytes), V codes (16 D), K scales (D), V scales
(D).  With g = 0..3, n, c = 0..15 and `chunk` counting 16-byte pieces:
  K codes   [chunk D/64][g][n][16 B]: lane (g, n) holds, in chunk order,
            columns [g D/4, (g + 1) D/4) of token n and then of token 16 + n
  V codes   [chunk D/64][g][c][16 B]: lane (g, c) holds columns
            [c D/16, (c + 1) D/16) of tokens 4g..4g+3, then 16+4g..16+4g+3
  K scales  [D/32][n][2]: tokens n, 16 + n;  V scales [D/32][g][8 tokens]
Even columns are low nibbles; scales are E8M0 (255: NaN).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6
SECTIONS = {32: (8, 12, 12), 64: (16, 24, 24), 128: (32, 48, 48)}  # time, height, width


def listed():
    return [
        # one decode step of a server with 64 running requests (latency)
        dict(name="plan_decode", kind="plan", batch=64, cached=4096, new=1, page=64),
        # a step that mixes prompts and decodes, 512 requests
        dict(name="plan_mixed", kind="plan", batch=512, cached=8192, new=300, page=32),
        # SmolVLA's decoder heads, 16 tokens, fp32 as hb_linear leaves them (latency)
        dict(name="rope_decode", kind="rope", tokens=16, q_heads=15, k_heads=5, dim=64, rot=64,
             axes=1, pairs="halves", type="float32"),
        # a prompt of image and text tokens, three position axes
        dict(name="rope_prompt", kind="rope", tokens=8192, q_heads=32, k_heads=8, dim=128,
             rot=128, axes=3, pairs="halves", type="bfloat16"),
        # a decode step's new K and V rows (latency)
        dict(name="append_decode", kind="append", tokens=64, heads=8, dim=128, page=64,
             type="bfloat16"),
        # a prompt's K and V, fp32 as the projections leave them
        dict(name="append_prompt", kind="append", tokens=16001, heads=5, dim=64, page=64,
             type="float32"),
        # one robot's step: one token over SmolVLA's 141 + 50 positions
        dict(name="attend_single", kind="attention", batch=1, cached_lo=190, cached_hi=190,
             new_lo=1, new_hi=1, q_heads=15, k_heads=5, dim=64, page=32, prefix=0, window=0,
             cap=0.0, type="float32"),
        # a decode step of 64 requests of 1 to 8 thousand tokens
        dict(name="attend_decode", kind="attention", batch=64, cached_lo=1000, cached_hi=8191,
             new_lo=1, new_hi=1, q_heads=32, k_heads=8, dim=128, page=64, prefix=0, window=0,
             cap=0.0, type="bfloat16"),
        # one request with a very long context
        dict(name="attend_long", kind="attention", batch=1, cached_lo=262146, cached_hi=262146,
             new_lo=1, new_hi=1, q_heads=64, k_heads=8, dim=128, page=128, prefix=0, window=0,
             cap=0.0, type="bfloat16"),
        # SmolVLA's action chunk: 50 rows that see a bidirectional prefix of
        # 141 and each other causally, 32 requests
        dict(name="attend_actions", kind="attention", batch=32, cached_lo=141, cached_hi=177,
             new_lo=50, new_hi=50, q_heads=15, k_heads=5, dim=64, page=32, prefix=141, window=0,
             cap=0.0, type="float32"),
        # prompts of up to 4,096 tokens, some behind a cached part
        dict(name="attend_prompt", kind="attention", batch=3, cached_lo=0, cached_hi=1000,
             new_lo=2500, new_hi=4096, q_heads=32, k_heads=8, dim=128, page=64, prefix=300,
             window=0, cap=0.0, type="bfloat16"),
        # chunks of prompts with a sliding window and capped scores
        dict(name="attend_window", kind="attention", batch=8, cached_lo=500, cached_hi=4000,
             new_lo=100, new_hi=256, q_heads=16, k_heads=4, dim=256, page=64, prefix=0,
             window=1024, cap=50.0, type="float16"),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope", "append", "attention", "attention", "attention"])
    kinds = ["float32", "bfloat16", "float16"]
    if kind == "plan":
        new = _log(rng, 1, 300)
        return dict(kind=kind, batch=_log(rng, 1, min(1000, 150000 // new)),
                    cached=_log(rng, 1, 8192), new=new, page=rng.choice([32, 64, 128]))
    if kind == "rope":
        q, k, d = rng.choice([(15, 5, 64), (12, 12, 64), (32, 8, 128), (16, 1, 128), (8, 4, 256),
                              (6, 2, 96)])
        rot = rng.choice([d, d // 2])
        axes = rng.choice([1, 3]) if rot // 2 in SECTIONS else 1
        return dict(kind=kind, tokens=_log(rng, 1, 8192 * 40 * 64 // ((q + k) * d)), q_heads=q,
                    k_heads=k, dim=d, rot=rot, axes=axes,
                    pairs=rng.choice(["halves", "neighbours"]), type=rng.choice(kinds))
    if kind == "append":
        d = rng.choice([64, 128, 256])
        h = rng.choice([1, 2, 5, 8])
        return dict(kind=kind, tokens=_log(rng, 1, 16000 * 5 * 64 // (h * d)), heads=h, dim=d,
                    page=rng.choice([32, 64, 128]), type=rng.choice(kinds))
    q, k, d = rng.choice([(15, 5, 64), (12, 12, 64), (32, 8, 128), (32, 1, 128), (16, 4, 256),
                          (48, 2, 64)])
    shape = rng.choice(["decode", "few", "prompt"])
    if shape == "decode":
        lo = hi = 1
        batch = _log(rng, 1, 128)
        most = min(131072, (1 << 28) // (k * d * batch))
    elif shape == "few":
        lo, hi = 1, rng.randint(2, 9)
        batch = _log(rng, 1, 32)
        most = min(16384, (1 << 26) // (k * d * batch))
    else:
        hi = _log(rng, 16, 1500)
        lo = rng.randint(hi // 2, hi)
        batch = _log(rng, 1, 6)
        most = 2000
    top = _log(rng, 1, max(1, most))
    return dict(kind=kind, batch=batch, cached_lo=rng.randint(0, top), cached_hi=top, new_lo=lo,
                new_hi=hi, q_heads=q, k_heads=k, dim=d, page=rng.choice([32, 64, 128]),
                prefix=rng.choice([0, 0, rng.randint(1, 600)]),
                window=rng.choice([0, 0, rng.randint(1, 2000)]), cap=rng.choice([0.0, 0.0, 30.0]),
                type=rng.choice(kinds))


# ------------------------------------------------------------------ sizes --

def _ramp(lo, hi, count):
    return [lo + (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _requests(case):
    """(cached, new, prefix) of every request, in an order of its own."""
    b = case["batch"]
    cached = _ramp(case["cached_lo"], case["cached_hi"], b)
    new = _ramp(case["new_hi"], case["new_lo"], b)
    return [(c, n, max(0, case["prefix"] - i % 3)) for i, (c, n) in enumerate(zip(cached, new))]


def _plan_requests(case):
    """(cached, new) of every request: most bring one token, a few many."""
    b = case["batch"]
    cached = _ramp(0, case["cached"], b) if b > 1 else [case["cached"]]
    return [(c, case["new"] if i % 4 == 0 else 1) for i, c in enumerate(cached)]


def _size(case):
    return 4 if case["type"] == "float32" else 2


def work(case):
    kind = case["kind"]
    if kind == "plan":
        reqs, p = _plan_requests(case), case["page"]
        need = sum(-(-(c + n) // p) + (-c // p) for c, n in reqs)
        kept = sum(1 for c, n in reqs if c % p)  # a table entry that new tokens go on filling
        tokens = sum(n for _, n in reqs)
        return {"bytes": 4.0 * (5 * len(reqs) + 2 * need + kept + 2 * tokens), "flops": 0.0}
    if kind == "rope":
        t, h, d = case["tokens"], case["q_heads"] + case["k_heads"], case["dim"]
        return {"bytes": 2.0 * t * h * d * _size(case) + 4.0 * t * case["axes"],
                "flops": t * h * (4.0 * d + 3.0 * case["rot"])}
    if kind == "append":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        rows = 2.0 * t * h * d
        return {"bytes": rows * (2 * _size(case) + 2 * 17 / 32) + 8.0 * t, "flops": 4 * rows}
    pairs = keys = tokens = 0
    w = case["window"]
    for c, n, pre in _requests(case):
        total = c + n
        pos = np.arange(c, total)
        start = np.maximum(0, pos - w + 1) if w else np.zeros(n, np.int64)
        pre = min(pre, total)
        own_keys = pos + 1 - np.maximum(start, np.minimum(pre, pos + 1))
        pairs += int(own_keys.sum()) + pre * n
        first = int(start[0]) if n else total
        keys += total - first + min(pre, first)
        tokens += n
    d, hq, hk = case["dim"], case["q_heads"], case["k_heads"]
    return {"bytes": keys * hk * d * 34 / 32 + 2.0 * tokens * hq * d * _size(case),
            "flops": 4.0 * d * hq * pairs}


# ----------------------------------------------------------------- inputs --

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 32))
    kind = case["kind"]
    state = {"case": case}
    if kind == "plan":
        reqs = [_plan_requests(case)[i] for i in order.permutation(case["batch"])]
        p, b = case["page"], case["batch"]
        cols = -(-(case["cached"] + case["new"]) // p) + 1
        have = [-(-c // p) for c, _ in reqs]
        need = sum(-(-(c + n) // p) for c, n in reqs) - sum(have)
        pages = torch.randperm(sum(have) + need + 64, generator=gen, device=DEV).to(torch.int32)
        at = torch.arange(cols, device=DEV) < _ints(have)[:, None]
        table = torch.full((b, cols), -1, dtype=torch.int32, device=DEV)
        table[at] = pages[:sum(have)]
        tokens = sum(n for _, n in reqs)
        new_ints = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)  # noqa: E731
        state.update(lens=_ints([c for c, _ in reqs]), new=_ints([n for _, n in reqs]),
                     free=pages[sum(have):].clone(), count=_ints([need + 64]), table=table,
                     cu=new_ints(b + 1), kv_lens=new_ints(b), slots=new_ints(tokens + 5),
                     positions=new_ints(tokens + 5), status=new_ints(2))
        return state
    kind_type = TYPES[case["type"]]
    if kind == "rope":
        t, hq, hk, d, rot = (case[n] for n in ("tokens", "q_heads", "k_heads", "dim", "rot"))
        # the projections' output: q, k and v of a token side by side
        qkv = torch.randn((t, hq + 2 * hk, d), generator=gen, device=DEV).to(kind_type)
        pos = torch.randint(0, 131072, (case["axes"], t), generator=gen, device=DEV,
                            dtype=torch.int32)
        exponent = torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot
        gamma = 1 + 0.2 * torch.randn((2, d), generator=gen, device=DEV)
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], positions=pos,
                     inv_freq=100000.0 ** -exponent, gamma_q=gamma[0], gamma_k=gamma[1],
                     sections=SECTIONS[rot // 2] if case["axes"] == 3 else (rot // 2,),
                     q_out=torch.empty((t, hq, d), dtype=kind_type, device=DEV),
                     k_out=torch.empty((t, hk, d), dtype=kind_type, device=DEV))
        return state
    if kind == "append":
        t, h, d, p = (case[n] for n in ("tokens", "heads", "dim", "page"))
        pages = -(-t // p) + 2
        # channels of different size, as keys have them
        k = torch.randn((t, h, d), generator=gen, device=DEV) * torch.exp(
            torch.randn((h, d), generator=gen, device=DEV))
        v = torch.randn((t, h, d), generator=gen, device=DEV)
        slots = torch.randperm(pages, generator=gen, device=DEV)[:, None] * p
        slots = (slots + torch.arange(p, device=DEV)).reshape(-1)[:t].to(torch.int32)
        slots[torch.rand(t, generator=gen, device=DEV) < 0.01] = -1  # padding
        state.update(k=k.to(kind_type), v=v.to(kind_type), slots=slots,
                     cache=torch.zeros((pages, h, p // 32, 34 * d), dtype=torch.uint8, device=DEV),
                     k_out=torch.empty((t, h, d), dtype=kind_type, device=DEV),
                     v_out=torch.empty((t, h, d), dtype=kind_type, device=DEV))
        return state
    reqs = [_requests(case)[i] for i in order.permutation(case["batch"])]
    hq, hk, d, p = (case[n] for n in ("q_heads", "k_heads", "dim", "page"))
    used = [-(-(c + n) // p) for c, n, _ in reqs]
    pages, cols = sum(used) + 3, max(used) + 1
    # codes as normal values encode to them; scales of channels of unequal size
    pool = torch.randn((1 << 16, 32), generator=gen, device=DEV)
    pool = pool / torch.exp2(torch.floor(torch.log2(pool.abs().amax(1, keepdim=True))) - 2)
    pool = _code(pool).reshape(-1, 2)
    pool = pool[:, 0] | pool[:, 1] << 4
    cache = torch.empty((pages, hk, p // 32, 34 * d), dtype=torch.uint8, device=DEV)
    flat = cache.view(-1, 34 * d)
    step = max(1, (1 << 28) // (32 * d))
    for i in range(0, flat.shape[0], step):
        part = flat[i:i + step]
        pick = torch.randint(0, pool.numel(), (part.shape[0], 32 * d), generator=gen, device=DEV,
                             dtype=torch.int32)
        part[:, :32 * d] = pool[pick]
        part[:, 32 * d:] = torch.randint(124, 127, (part.shape[0], 2 * d), generator=gen,
                                         device=DEV, dtype=torch.uint8)
    perm = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(reqs), cols), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(cols, device=DEV) < _ints(used)[:, None]] = perm[:sum(used)]
    tokens = sum(n for _, n, _ in reqs)
    cu = np.concatenate([[0], np.cumsum([n for _, n, _ in reqs])]).tolist()
    q = torch.randn((tokens, hq, d), generator=gen, device=DEV).to(kind_type)
    state.update(q=q, cache=cache, table=table, cu=_ints(cu),
                 kv_lens=_ints([c + n for c, n, _ in reqs]),
                 prefix=_ints([f for _, _, f in reqs]) if case["prefix"] else None,
                 max_new=max(n for _, n, _ in reqs), max_kv=max(c + n for c, n, _ in reqs),
                 scale=d ** -0.5, out=torch.empty_like(q))
    return state


# ------------------------------------------------------------ plain forms --

def _plain_plan(s):
    p, cols, size = s["case"]["page"], s["table"].shape[1], s["slots"].shape[0]
    lens, new = s["lens"].long(), s["new"].long()
    have, pages = (lens + p - 1) // p, (lens + new + p - 1) // p
    ends = torch.cumsum(new, 0)
    fits = (pages <= cols) & (ends <= size)
    need = torch.where(fits, pages - have, 0)
    stop = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (stop <= s["count"]))
    first = stop - need
    # pages from the top of the stack into the table
    col = torch.arange(cols, device=DEV)
    fresh = (col >= have[:, None]) & (col < pages[:, None]) & ok[:, None]
    at = s["count"] - 1 - first[:, None] - (col - have[:, None])
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].shape[0] - 1)], s["table"])
    token = torch.arange(size, device=DEV)
    req = torch.searchsorted(ends, token, right=True)
    real = req < lens.shape[0]
    req = req.clamp(max=lens.shape[0] - 1)
    pos = lens[req] + token - (ends - new)[req]
    page = table[req, (pos // p).clamp(0, cols - 1)].long()
    slot = torch.where(real & ok[req] & (page >= 0), page * p + pos % p, -1)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    status = torch.stack([torch.where(ok, need, 0).sum(), (~ok).sum()])
    return [x.to(torch.int32) for x in (table, cu, torch.where(ok, lens + new, lens), slot,
                                        torch.where(real, pos, -1), status)]


def _plain_norm_rope(x, gamma, cos, sin, rot, pairs, to):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma
    r = y[..., :rot]
    if pairs == "halves":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
    else:
        a, b = r[..., 0::2], r[..., 1::2]
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.cat([a, b], -1) if pairs == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([r, y[..., rot:]], -1).to(to)


def _plain_rope(s):
    case = s["case"]
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=DEV),
                                   torch.tensor(s["sections"], device=DEV),
                                   output_size=case["rot"] // 2)
    angle = s["positions"].double()[axis].T * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    rest = (cos, sin, case["rot"], case["pairs"], s["q"].dtype)
    return [_plain_norm_rope(s["q"], s["gamma_q"], *rest),
            _plain_norm_rope(s["k"], s["gamma_k"], *rest)]


def _code(y):
    """E2M1 codes of y, rounded to nearest even and saturated."""
    m = y.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5)
            + (m >= 3.5) + (m > 5))
    return code | torch.signbit(y).to(torch.uint8) << 3


def _value(code):
    """E2M1 values, fp32."""
    return torch.tensor(FP4 + tuple(-v for v in FP4), device=DEV)[code.int()]


def _plain_encode(x, bad):
    """[t][h][d] -> codes [t][h][d/2] (two to a byte), scale bytes [t][h][d/32]."""
    t, h, d = x.shape
    x = torch.where(bad[..., None], 0.0, x.float()).view(t, h, d // 32, 32)
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, 0).clamp(-126, 125)
    code = _code(x * torch.exp2(-e.double()).unsqueeze(-1)).view(t, h, d // 2, 2)
    return code[..., 0] | code[..., 1] << 4, (e + 127).to(torch.uint8)


def _places(cache, slots, d):
    """Byte offsets of tokens in the cache: K codes, V codes [t][h][d/2], K and V scales
    [t][h][d/32]."""
    pages, heads, groups, size = cache.shape
    slot = slots.long()
    t = slot % 32
    record = slot // (32 * groups) * heads * groups + slot // 32 % groups
    record = (record[:, None] + torch.arange(heads, device=DEV) * groups)[..., None] * size
    t, n, tile = t[:, None, None], t[:, None, None] % 16, t[:, None, None] // 16
    byte, blk = torch.arange(d // 2, device=DEV), torch.arange(d // 32, device=DEV)
    at = tile * (d // 8) + byte % (d // 8)
    k = (at // 16 * 64 + byte // (d // 8) * 16 + n) * 16 + at % 16
    j = t % 4 + 4 * tile
    at = j * (d // 32) + byte % (d // 32)
    v = 16 * d + (at // 16 * 64 + n // 4 * 16 + byte // (d // 32)) * 16 + at % 16
    return (record + k, record + v, record + 32 * d + (blk * 16 + n) * 2 + tile,
            record + 33 * d + (blk * 4 + n // 4) * 8 + j)


def _plain_decode(codes, scales, to=torch.float32):
    t, h, half = codes.shape
    x = torch.stack([_value(codes & 15), _value(codes >> 4)], -1).view(t, h, half // 16, 32)
    e = scales.float().unsqueeze(-1) - 127
    return torch.where(e < 128, x * torch.exp2(e), math.nan).view(t, h, 2 * half).to(to)


def _plain_append(s):
    cache, d = s["cache"], s["k"].shape[-1]
    bad = ~(s["k"].isfinite().all(-1) & s["v"].isfinite().all(-1))
    (kc, ks), (vc, vs) = _plain_encode(s["k"], bad), _plain_encode(s["v"], bad)
    ks = torch.where(bad[..., None], 255, ks)
    inside = s["slots"] >= 0
    flat = torch.cat([cache.view(-1), cache.new_zeros(1)])  # its last byte takes what has no slot
    keep = inside[:, None, None]
    places = [torch.where(keep, p, flat.numel() - 1) for p in _places(cache, s["slots"], d)]
    for at, what in zip(places, (kc, vc, ks, vs)):
        flat[at.reshape(-1)] = what.reshape(-1)
    cache.view(-1).copy_(flat[:-1])
    kc, vc, ks, vs = (flat[at] for at in places)
    return [torch.where(keep, _plain_decode(kc, ks), 0).to(s["k"].dtype),
            torch.where(keep, _plain_decode(vc, vs), 0).to(s["k"].dtype)]


def _plain_gather(s):
    """K and V of every request, fp32 [b][heads][tokens][d]."""
    cache, table = s["cache"], s["table"]
    d, b = s["q"].shape[-1], table.shape[0]
    heads, groups = cache.shape[1:3]
    cols = -(-s["max_kv"] // (32 * groups))
    rec = cache[table[:, :cols].clamp(min=0)].transpose(1, 2)  # [b][heads][cols][groups][34 d]
    lead, c = (b, heads, cols * groups), d // 64
    kc = rec[..., :16 * d].reshape(*lead, c, 4, 16, 16).permute(0, 1, 2, 4, 5, 3, 6)
    kc = kc.reshape(*lead, 4, 16, 2, d // 8).permute(0, 1, 2, 5, 4, 3, 6)
    vc = rec[..., 16 * d:32 * d].reshape(*lead, c, 4, 16, 16).permute(0, 1, 2, 4, 5, 3, 6)
    vc = vc.reshape(*lead, 4, 16, 2, 4, d // 32).permute(0, 1, 2, 5, 3, 6, 4, 7)
    ks = rec[..., 32 * d:33 * d].reshape(*lead, d // 32, 16, 2).permute(0, 1, 2, 5, 4, 3)
    vs = rec[..., 33 * d:].reshape(*lead, d // 32, 4, 2, 4).permute(0, 1, 2, 5, 4, 6, 3)
    rows, tokens = b * heads, cols * groups * 32
    k = _plain_decode(kc.reshape(rows, tokens, d // 2), ks.reshape(rows, tokens, d // 32))
    v = _plain_decode(vc.reshape(rows, tokens, d // 2), vs.reshape(rows, tokens, d // 32))
    return k.view(b, heads, tokens, d), v.view(b, heads, tokens, d)


def _plain_attention(s):
    case, q = s["case"], s["q"]
    tokens, hq, d = q.shape
    k, v = _plain_gather(s)
    b, hk, keys, _ = k.shape
    n, lens = s["cu"].diff(), s["kv_lens"]
    row = torch.arange(s["max_new"], device=DEV)
    at = (s["cu"][:-1, None] + row).clamp(max=tokens - 1)
    rows = q[at].float().view(b, -1, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    x = torch.matmul(rows.reshape(b, hk, -1, d), k.transpose(-1, -2)) * s["scale"]
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    key = torch.arange(keys, device=DEV)
    pos = (lens - n)[:, None, None] + row[:, None]
    see = key <= pos
    if case["window"]:
        see = see & (pos - key < case["window"])
    if s["prefix"] is not None:
        see = see | (key < s["prefix"][:, None, None])
    see = see & (key < lens[:, None, None])
    x = x.view(b, hk, hq // hk, -1, keys).masked_fill(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = x.sum(-1, keepdim=True)
    v = torch.where((key < lens[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(x.view(b, hk, -1, keys), v).view(b, hk, hq // hk, -1, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, -1, hq, d)
    token = torch.arange(tokens, device=DEV)
    req = torch.searchsorted(s["cu"][1:], token, right=True)
    return o[req, token - s["cu"][req]].to(q.dtype)


# -------------------------------------------------------------------- run --

_ctx = None


def _context(hb):
    global _ctx
    if _ctx is None:
        _ctx = hb.Context(torch.cuda.current_device())
        _ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return _ctx


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"plan": _plain_plan, "rope": _plain_rope, "append": _plain_append,
                "attention": _plain_attention}[kind](s)
    import hotarubi_amd as hb
    ctx = _context(hb)
    if kind == "plan":
        hb.kv_plan(lens=s["lens"], new_tokens=s["new"], free_pages=s["free"],
                   free_count=s["count"], table=s["table"], page_size=s["case"]["page"],
                   cu=s["cu"], kv_lens=s["kv_lens"], slots=s["slots"],
                   positions=s["positions"], status=s["status"], ctx=ctx, sync=False)
        return [s["table"], s["cu"], s["kv_lens"], s["slots"], s["positions"], s["status"]]
    if kind == "rope":
        hb.norm_rope(q=s["q"], k=s["k"], positions=s["positions"], inv_freq=s["inv_freq"],
                     q_out=s["q_out"], k_out=s["k_out"], gamma_q=s["gamma_q"],
                     gamma_k=s["gamma_k"], eps=EPS, sections=s["sections"],
                     interleaved=s["case"]["pairs"] == "neighbours", ctx=ctx, sync=False)
        return [s["q_out"], s["k_out"]]
    if kind == "append":
        hb.kv_append(k=s["k"], v=s["v"], slots=s["slots"], cache=s["cache"], ctx=ctx, sync=False)
        hb.kv_read(k=s["k_out"], v=s["v_out"], slots=s["slots"], cache=s["cache"], ctx=ctx,
                   sync=False)
        return [s["k_out"], s["v_out"]]
    hb.kv_attention(q=s["q"], out=s["out"], cache=s["cache"], table=s["table"], cu=s["cu"],
                    kv_lens=s["kv_lens"], max_new=s["max_new"], max_kv=s["max_kv"],
                    scale=s["scale"], prefix=s["prefix"], window=s["case"]["window"],
                    softcap=s["case"]["cap"], ctx=ctx, sync=False)
    return s["out"]


# ------------------------------------------------------------------ exact --

def _exact_plan(s):
    page, cols, size = s["case"]["page"], s["table"].shape[1], s["slots"].shape[0]
    lens, new = s["lens"].tolist(), s["new"].tolist()
    table, free, count = s["table"].cpu().numpy().copy(), s["free"].tolist(), int(s["count"])
    cu, kv, taken, wanted, refused = [0], [], 0, 0, 0
    slots, positions = np.full(size, -1, np.int32), np.full(size, -1, np.int32)
    for b, (have, more) in enumerate(zip(lens, new)):
        total = have + more
        fits = math.ceil(total / page) <= cols and cu[-1] + more <= size
        add = math.ceil(total / page) - math.ceil(have / page) if fits else 0
        ok = fits and (add == 0 or wanted + add <= count)
        for i in range(add if ok else 0):
            table[b, math.ceil(have / page) + i] = free[count - 1 - wanted - i]
        wanted, taken, refused = wanted + add, taken + add * ok, refused + (not ok)
        for i in range(more):
            if cu[-1] + i < size:
                at = have + i
                positions[cu[-1] + i] = at
                if ok and table[b, at // page] >= 0:
                    slots[cu[-1] + i] = table[b, at // page] * page + at % page
        cu.append(cu[-1] + more)
        kv.append(total if ok else have)
    ints = lambda v: np.array(v, np.int32)  # noqa: E731
    return [table, ints(cu), ints(kv), slots, positions, ints([taken, refused])]


def _exact_rope(s):
    half, t = s["case"]["rot"] // 2, s["q"].shape[0]
    angle = torch.empty((t, half), dtype=torch.float64, device=DEV)
    first = 0
    for axis, count in enumerate(s["sections"]):
        angle[:, first:first + count] = torch.outer(s["positions"][axis].double(),
                                                    s["inv_freq"][first:first + count])
        first += count
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    out = []
    for x, gamma in ((s["q"], s["gamma_q"]), (s["k"], s["gamma_k"])):
        x = x.double()
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * gamma.double()
        if s["case"]["pairs"] == "halves":
            z = torch.complex(x[..., :half].clone(), x[..., half:2 * half].clone()) * turn
            x[..., :half], x[..., half:2 * half] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:2 * half:2].clone(), x[..., 1:2 * half:2].clone()) * turn
            x[..., 0:2 * half:2], x[..., 1:2 * half:2] = z.real, z.imag
        out.append(x)
    return out


def _exact_append(s):
    grid = torch.tensor(FP4, dtype=torch.float64, device=DEV)
    out = []
    for x in (s["k"], s["v"]):
        t, h, d = x.shape
        x = x.double().view(t, h, d // 32, 32)
        top = x.abs().amax(-1, keepdim=True)
        e = torch.where(top > 0, torch.floor(torch.log2(top)), 0.0)
        e = torch.where(torch.exp2(e) > top, e - 1, e)
        e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
        unit = torch.exp2((e - 2).clamp(-126, 125))
        m = (x.abs() / unit).clamp(max=6)
        above = torch.bucketize(m, grid).clamp(1, 7)  # grid[above - 1] < m <= grid[above]
        low, high = grid[above - 1], grid[above]
        up = (m - low > high - m) | ((m - low == high - m) & (above % 2 == 0))
        x = torch.where(up, high, low).copysign(x) * unit
        out.append(torch.where(s["slots"][:, None, None] >= 0, x.view(t, h, d), 0.0))
    return out


def _exact_rows(records, d):
    """K and V, float64, of records [..., 34 d] -> [..., 32, d]."""
    t, col = torch.arange(32, device=DEV)[:, None], torch.arange(d, device=DEV)
    n, tile = t % 16, t // 16
    byte = tile * (d // 8) + col % (d // 4) // 2
    k_at = byte // 16 * 1024 + col // (d // 4) * 256 + n * 16 + byte % 16
    byte = (t % 4 + 4 * tile) * (d // 32) + col % (d // 16) // 2
    v_at = 16 * d + byte // 16 * 1024 + n // 4 * 256 + col // (d // 16) * 16 + byte % 16
    k_sc = 32 * d + col // 32 * 32 + n * 2 + tile
    v_sc = 33 * d + col // 32 * 32 + n // 4 * 8 + t % 4 + 4 * tile
    out = []
    for at, sc in ((k_at, k_sc), (v_at, v_sc)):
        code = (records[..., at] >> (col % 2 * 4).to(torch.uint8)) & 15
        exp, man = (code >> 1 & 3).double(), (code & 1).double()
        x = torch.where(exp > 0, torch.exp2(exp - 1) * (1 + man / 2), man / 2)
        scale = records[..., sc].double()
        scale = torch.where(scale == 255, math.nan, torch.exp2(scale - 127))
        out.append(torch.where(code > 7, -x, x) * scale)
    return out


def _exact_attention(s):
    case, d, page = s["case"], s["q"].shape[-1], s["case"]["page"]
    cu, lens = s["cu"].tolist(), s["kv_lens"].tolist()
    group = case["q_heads"] // case["k_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, total in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if not n or not total:
            continue
        pos = (total - n + torch.arange(n, device=DEV))[:, None]
        key = torch.arange(total, device=DEV)
        see = key <= pos
        if case["window"]:
            see &= key > pos - case["window"]
        if s["prefix"] is not None:
            see |= key < s["prefix"][b]
        pages = s["table"][b, :-(-total // page)].long()
        for h in range(case["k_heads"]):
            k, v = (x.reshape(-1, d)[:total] for x in _exact_rows(s["cache"][pages, h], d))
            for i in range(h * group, (h + 1) * group):
                x = s["q"][cu[b]:cu[b + 1], i].double() @ k.T * s["scale"]
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                x = torch.softmax(x.masked_fill(~see, -math.inf), -1)
                out[cu[b]:cu[b + 1], i] = torch.nan_to_num(x) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "append": _exact_append,
            "attention": _exact_attention}[case["kind"]](s)
