"""Performance cases of the serving operators around an 8-bit paged cache.

Every case is a plain dict; `kind` names the operator, the other values its
sizes, types and masks:

  append8    K and V rows into the 8-bit cache, and the stored values of every
             block that they touch back out (kv8_append, kv8_read)
  attend8    ragged requests over the 8-bit cache: prefix mask, window with
             first tokens that stay visible, capped scores (kv8_attention)
  fork       requests that go on from another's tokens: shared pages, a copy of
             the page they write next, in every layer (kv_fork, kv_copy)
  compact    requests that end, and the others' pages moved to the cache's
             front in every layer (kv_free, kv_compact, kv_copy)
  logprobs   log probabilities of given tokens, the entropy, the most likely
             tokens (token_logprobs)

The 8-bit cache is uint8 [pages][heads][page / 32][64 D + 16]: a record per 32
tokens of one head holding K codes (32 D bytes), V codes (32 D), the scale
byte of K, that of V, 14 unused bytes.  With g = 0..3, n, c = 0..15 and `chunk`
counting 16-byte pieces:
  K codes   [chunk D/32][g][n][16 B]: (g, n) holds, in chunk order, columns
            [g D/4, (g + 1) D/4) of token n and then of token 16 + n
  V codes   [chunk D/32][g][c][16 B]: (g, c) holds columns
            [c D/16, (c + 1) D/16), of each tokens 4g..4g+3, then 16+4g..16+4g+3
A value is an E4M3 code times 2^(scale byte - 127), one scale for the record's
K and one for its V: the least exponent within [-117, 119] that has the
largest value at 448 or below (byte 0 while all are zero).  Tokens come into a
record in their order; where a later one needs a larger scale the earlier ones
are rounded to it.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # a decode step's new K and V rows, blocks begun by earlier steps (latency)
        dict(name="append8_decode", kind="append8", batch=64, cached_lo=1, cached_hi=4000,
             new_lo=1, new_hi=1, heads=8, dim=128, page=64, type="bfloat16"),
        # a long prompt's K and V, fp32 as the projections leave them
        dict(name="append8_prompt", kind="append8", batch=1, cached_lo=0, cached_hi=0,
             new_lo=16001, new_hi=16001, heads=5, dim=64, page=64, type="float32"),
        # one robot's step: one token over SmolVLA's 141 + 50 positions (latency)
        dict(name="attend8_single", kind="attend8", batch=1, cached_lo=190, cached_hi=190,
             new_lo=1, new_hi=1, q_heads=15, k_heads=5, dim=64, page=32, prefix=0, window=0,
             sinks=0, cap=0.0, type="float32"),
        # a decode step of 64 requests of 1 to 8 thousand tokens
        dict(name="attend8_decode", kind="attend8", batch=64, cached_lo=1000, cached_hi=8191,
             new_lo=1, new_hi=1, q_heads=32, k_heads=8, dim=128, page=64, prefix=0, window=0,
             sinks=0, cap=0.0, type="bfloat16"),
        # long streams that keep a window and their first four tokens
        dict(name="attend8_sinks", kind="attend8", batch=24, cached_lo=9000, cached_hi=40000,
             new_lo=1, new_hi=3, q_heads=32, k_heads=8, dim=128, page=128, prefix=0, window=4095,
             sinks=4, cap=0.0, type="float16"),
        # prompts of up to 4,096 tokens, some behind a cached part
        dict(name="attend8_prompt", kind="attend8", batch=3, cached_lo=0, cached_hi=1000,
             new_lo=2500, new_hi=4096, q_heads=32, k_heads=8, dim=128, page=64, prefix=300,
             window=0, sinks=0, cap=0.0, type="bfloat16"),
        # four more samples of one answer, SmolVLA's decoder heads (latency)
        dict(name="fork_samples", kind="fork", batch=8, forks=4, lens_lo=30, lens_hi=191,
             page=32, heads=5, dim=64, layers=2),
        # a beam search's step: 96 beams go on from 32 of them
        dict(name="fork_beams", kind="fork", batch=160, forks=96, lens_lo=300, lens_hi=1500,
             page=64, heads=8, dim=128, layers=2),
        # two of eight requests end (latency)
        dict(name="compact_few", kind="compact", batch=8, ended=2, shared=50, lens_lo=30,
             lens_hi=191, spare=9, page=32, heads=5, dim=64, layers=2),
        # half of a full server's requests end
        dict(name="compact_half", kind="compact", batch=512, ended=256, shared=500, lens_lo=500,
             lens_hi=3500, spare=1000, page=64, heads=1, dim=64, layers=1),
        # the answers of a decode step, fp32 as hb_linear leaves them, a third of
        # the vocabulary not allowed
        dict(name="logprobs_decode", kind="logprobs", rows=8, vocab=50001, pad=7, top=20,
             masked=0.3, spread=3.0, scale=1.25, type="float32"),
        # the score of prompts
        dict(name="logprobs_prompt", kind="logprobs", rows=4096, vocab=65537, pad=0, top=5,
             masked=0.0, spread=2.0, scale=1.0, type="bfloat16"),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append8", "append8", "attend8", "attend8", "attend8", "fork", "compact",
                       "logprobs", "logprobs"])
    kinds = ["float32", "bfloat16", "float16"]
    if kind == "append8":
        d = rng.choice([64, 128, 256])
        h = rng.choice([1, 2, 5, 8])
        most = 16001 * 5 * 64 // (h * d)
        batch = _log(rng, 1, min(500, most))
        new = _log(rng, 1, max(1, most // batch))
        return dict(kind=kind, batch=batch, cached_lo=0, cached_hi=_log(rng, 1, 3000),
                    new_lo=max(1, new // 2), new_hi=new, heads=h, dim=d,
                    page=rng.choice([32, 64, 128]), type=rng.choice(kinds))
    if kind == "fork":
        batch = _log(rng, 2, 160)
        lens = _log(rng, 20, 1500)
        return dict(kind=kind, batch=batch, forks=rng.randint(1, max(1, batch * 3 // 5)),
                    lens_lo=lens // 3, lens_hi=lens, page=rng.choice([32, 64, 128]),
                    heads=rng.choice([1, 5, 8]), dim=rng.choice([64, 128]),
                    layers=rng.choice([1, 2]))
    if kind == "compact":
        batch = _log(rng, 2, 300)
        lens = _log(rng, 20, 1500)
        return dict(kind=kind, batch=batch, ended=rng.randint(0, batch), lens_lo=lens // 3,
                    lens_hi=lens, shared=rng.choice([0, lens // 4]), spare=_log(rng, 1, 500),
                    page=rng.choice([32, 64, 128]), heads=rng.choice([1, 2]), dim=64,
                    layers=rng.choice([1, 2]))
    if kind == "logprobs":
        vocab = _log(rng, 100, 200000)
        return dict(kind=kind, rows=_log(rng, 1, min(4096, (1 << 28) // vocab)), vocab=vocab,
                    pad=rng.choice([0, 0, rng.randint(1, 100)]), top=rng.choice([0, 1, 5, 20, 32]),
                    masked=rng.choice([0.0, 0.0, 0.5]), spread=rng.choice([1.0, 3.0, 6.0]),
                    scale=rng.choice([1.0, 0.7, 1.6]), type=rng.choice(kinds))
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
    window = rng.choice([0, 0, rng.randint(1, 2000)])
    return dict(kind=kind, batch=batch, cached_lo=rng.randint(0, top), cached_hi=top, new_lo=lo,
                new_hi=hi, q_heads=q, k_heads=k, dim=d, page=rng.choice([32, 64, 128]),
                prefix=rng.choice([0, 0, rng.randint(1, 600)]), window=window,
                sinks=rng.choice([0, rng.randint(1, 70)]) if window else 0,
                cap=rng.choice([0.0, 0.0, 30.0]), type=rng.choice(kinds))


# ------------------------------------------------------------------ sizes --

def _ramp(lo, hi, count):
    return [lo + (hi - lo) * i // max(1, count - 1) for i in range(count)]


def _requests(case):
    """(cached, new, prefix) of every request, in an order of its own."""
    b = case["batch"]
    cached = _ramp(case["cached_lo"], case["cached_hi"], b)
    new = _ramp(case["new_hi"], case["new_lo"], b)
    prefix = case.get("prefix", 0)
    return [(c, n, max(0, prefix - i % 3)) for i, (c, n) in enumerate(zip(cached, new))]


def _size(case):
    return 4 if case["type"] == "float32" else 2


def _page_bytes(case):
    return case["heads"] * (case["page"] // 32) * (64 * case["dim"] + 16)


def _fork_lens(case):
    """Tokens of every request: those that will be forked to have none."""
    b = case["batch"]
    live = b - case["forks"]
    return _ramp(case["lens_lo"], case["lens_hi"], live) + [0] * (b - live)


def _compact_pages(case):
    """Pages that all requests share at their start, and further ones of each."""
    lens = _ramp(case["lens_lo"], case["lens_hi"], case["batch"])
    shared = min(case["shared"], case["lens_lo"]) // case["page"]
    return lens, shared, [-(-n // case["page"]) - shared for n in lens]


def work(case):
    kind = case["kind"]
    if kind == "append8":
        h, d = case["heads"], case["dim"]
        new = sum(n for _, n, _ in _requests(case))
        old = sum(c % 32 for c, _, _ in _requests(case))
        # rows in, codes and their scales out, the values of every block back
        return {"bytes": 2.0 * h * d * (new * (_size(case) + 1) + (new + old) * (1 + _size(case)))
                + 4.0 * (2 * new + old), "flops": 8.0 * new * h * d}
    if kind == "fork":
        p, lens = case["page"], _fork_lens(case)
        live = case["batch"] - case["forks"]
        shared = copied = 0
        for i in range(case["forks"]):
            n = lens[i % live]
            shared, copied = shared + -(-n // p), copied + (n % p > 0)
        return {"bytes": 8.0 * shared + 2.0 * copied * case["layers"] * _page_bytes(case)
                + 8.0 * case["batch"] + 16.0 * case["forks"], "flops": 0.0}
    if kind == "compact":
        lens, shared, more = _compact_pages(case)
        b, total = case["batch"], shared + sum(more) + case["spare"]
        kept = (shared if case["ended"] < b else 0) + sum(more[case["ended"]:])
        moved = kept * (total - kept) / total  # those behind the front, on average
        return {"bytes": 8.0 * b * (max(more) + shared + 1) + 8.0 * total
                + 2.0 * moved * case["layers"] * _page_bytes(case), "flops": 0.0}
    if kind == "logprobs":
        n = float(case["rows"]) * case["vocab"]
        return {"bytes": n * _size(case) + case["rows"] * (12.0 + 8 * case["top"]),
                "flops": 6 * n}
    pairs = keys = tokens = 0
    w, sinks = case["window"], case["sinks"]
    for c, n, pre in _requests(case):
        total = c + n
        pos = np.arange(c, total)
        start = np.maximum(0, pos - w + 1) if w else np.zeros(n, np.int64)
        first = np.maximum(min(pre, total), np.minimum(sinks, pos + 1))  # keys [0, first)
        pairs += int((pos + 1 - np.maximum(start, np.minimum(first, pos + 1)) + first).sum())
        keys += total - int(start[0]) + min(int(first[-1]), int(start[0]))
        tokens += n
    d, hq, hk = case["dim"], case["q_heads"], case["k_heads"]
    return {"bytes": keys * hk * 2.0 * d + 2.0 * tokens * hq * d * _size(case),
            "flops": 4.0 * d * hq * pairs}


# ----------------------------------------------------------------- inputs --

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _empty(*shape):
    return torch.empty(shape, dtype=torch.int32, device=DEV)


def _records(count, d, gen):
    """Records as normal values are stored: uint8 [count][64 d + 16]."""
    pool = torch.randn((1 << 16, 16), generator=gen, device=DEV) * 100
    pool = pool.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int32)
    flat = torch.zeros((count, 64 * d + 16), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 28) // (64 * d))
    for i in range(0, count, step):
        part = flat[i:i + step]
        pick = torch.randint(0, 1 << 16, (part.shape[0], 4 * d), generator=gen, device=DEV,
                             dtype=torch.int32)
        part[:, :64 * d] = pool[pick].view(part.shape[0], -1).view(torch.uint8)
        # (values of up to 2 to 8)
        part[:, 64 * d:64 * d + 2] = torch.randint(119, 122, (part.shape[0], 2), generator=gen,
                                                   device=DEV, dtype=torch.uint8)
    return flat


def _tables(used, columns, pages, gen):
    """Block table of requests of `used` pages each, and the pages' order."""
    perm = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(used), columns), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(columns, device=DEV) < _ints(used)[:, None]] = perm[:sum(used)]
    return table, perm


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 32))
    state = {"case": case}
    kind = case["kind"]
    if kind == "logprobs":
        r, v, k = case["rows"], case["vocab"], case["top"]
        x = torch.empty((r, v + case["pad"]), dtype=TYPES[case["type"]], device=DEV)
        step = max(1, (1 << 27) // (v + case["pad"]))
        for i in range(0, r, step):
            part = torch.randn((min(step, r - i), v + case["pad"]), generator=gen, device=DEV)
            x[i:i + step] = part * case["spread"]
            if case["masked"]:
                hide = torch.rand(part.shape, generator=gen, device=DEV) < case["masked"]
                x[i:i + step].masked_fill_(hide, -math.inf)
        x = x[:, :v]
        tokens = torch.randint(0, v, (r,), generator=gen, device=DEV)
        # a row's given token is an allowed one; some rows have none
        x[torch.arange(r, device=DEV), tokens] = 1.5
        tokens[torch.rand(r, generator=gen, device=DEV) < 0.1] = -1
        state.update(logits=x, tokens=tokens.to(torch.int32),
                     logprobs=torch.empty(r, device=DEV), entropy=torch.empty(r, device=DEV),
                     top_ids=_empty(r, k), top=torch.empty((r, k), device=DEV))
        return state
    p, d = case["page"], case["dim"]
    if kind == "append8":
        h, type_ = case["heads"], TYPES[case["type"]]
        reqs = [_requests(case)[i] for i in order.permutation(case["batch"])]
        used = [-(-(c + n) // p) for c, n, _ in reqs]
        pages = sum(used) + 3
        table, _ = _tables(used, max(used), pages, gen)
        table = table.cpu().numpy().astype(np.int64)
        slots, read = [], []
        for b, (c, n, _) in enumerate(reqs):
            at = np.arange(c // 32 * 32, c + n)
            at = table[b, at // p] * p + at % p
            slots.append(at[c % 32:])
            read.append(at)
        slots = np.concatenate(slots + [[-1] * 3])  # a padded step
        tokens = len(slots)
        # channels of different size, as keys have them
        k = torch.randn((tokens, h, d), generator=gen, device=DEV) * torch.exp(
            torch.randn((h, d), generator=gen, device=DEV))
        v = torch.randn((tokens, h, d), generator=gen, device=DEV)
        read = _ints(np.concatenate(read))
        state.update(k=k.to(type_), v=v.to(type_), slots=_ints(slots), read=read,
                     cache=_records(pages * h * (p // 32), d, gen).view(pages, h, p // 32, -1),
                     k_out=torch.empty((len(read), h, d), dtype=type_, device=DEV),
                     v_out=torch.empty((len(read), h, d), dtype=type_, device=DEV))
        return state
    if kind == "fork":
        lens = _fork_lens(case)
        b, live = case["batch"], case["batch"] - case["forks"]
        used = [-(-n // p) for n in lens]
        pages = sum(used) + case["forks"] + 5
        row = order.permutation(b)  # where each request's row lies
        table, perm = _tables(used, max(used) + 2, pages, gen)
        table[torch.tensor(row, device=DEV)] = table.clone()
        at = np.empty(b, np.int64)
        at[row] = lens
        state.update(table=table, lens=_ints(at.tolist()),
                     source=_ints([int(row[i % live]) for i in range(case["forks"])]),
                     target=_ints([int(row[live + i]) for i in range(case["forks"])]),
                     free=torch.cat([perm[sum(used):], perm[:sum(used)]]),
                     count=_ints([pages - sum(used)]), lens_out=_empty(b),
                     pairs=_empty(case["forks"], 2), status=_empty(2))
    elif kind == "compact":
        lens, shared, more = _compact_pages(case)
        b = case["batch"]
        pages = shared + sum(more) + case["spare"]
        perm = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        table = torch.full((b, shared + max(more) + 1), -1, dtype=torch.int32, device=DEV)
        table[:, :shared] = perm[:shared]
        table[:, shared:][torch.arange(max(more) + 1, device=DEV) < _ints(more)[:, None]] = \
            perm[shared:shared + sum(more)]
        row = torch.tensor(order.permutation(b), device=DEV)
        lens = _ints(lens)
        free = torch.full((pages,), -1, dtype=torch.int32, device=DEV)
        free[:case["spare"]] = perm[pages - case["spare"]:]
        state.update(table=table[torch.argsort(row)].contiguous(), lens=lens[torch.argsort(row)],
                     rows=row[:case["ended"]].to(torch.int32), free=free,
                     count=_ints([case["spare"]]), kept=_empty(b), freed=_empty(2),
                     table_out=torch.empty_like(table), free_out=torch.empty_like(free),
                     count_out=_empty(1), pairs=_empty(max(1, pages // 2), 2), status=_empty(2))
    if kind in ("fork", "compact"):
        layers, h, g = case["layers"], case["heads"], p // 32
        cache = _records(layers * pages * h * g, d, gen)
        state["cache"] = cache.view(layers, pages, h, g, 64 * d + 16)
        return state
    reqs = [_requests(case)[i] for i in order.permutation(case["batch"])]
    hq, hk = case["q_heads"], case["k_heads"]
    used = [-(-(c + n) // p) for c, n, _ in reqs]
    pages = sum(used) + 3
    cache = _records(pages * hk * (p // 32), d, gen)
    table, _ = _tables(used, max(used) + 1, pages, gen)
    tokens = sum(n for _, n, _ in reqs)
    cu = np.concatenate([[0], np.cumsum([n for _, n, _ in reqs])]).tolist()
    q = torch.randn((tokens, hq, d), generator=gen, device=DEV).to(TYPES[case["type"]])
    state.update(q=q, cache=cache.view(pages, hk, p // 32, 64 * d + 16), table=table, cu=_ints(cu),
                 kv_lens=_ints([c + n for c, n, _ in reqs]),
                 prefix=_ints([f for _, _, f in reqs]) if case["prefix"] else None,
                 max_new=max(n for _, n, _ in reqs), max_kv=max(c + n for c, n, _ in reqs),
                 scale=d ** -0.5, out=torch.empty_like(q))
    return state


# ------------------------------------------------------------ plain forms --

def _places(cache, slots, d):
    """Byte offsets of tokens in the cache: K and V codes [t][h][d]; records [t][h]."""
    pages, heads, groups, size = cache.shape
    slot = slots.long()
    t = slot % 32
    record = slot // (32 * groups) * heads * groups + slot // 32 % groups
    record = record[:, None] + torch.arange(heads, device=DEV) * groups
    col, t = torch.arange(d, device=DEV), t[:, None, None]
    at = t // 16 * (d // 4) + col % (d // 4)
    k = at // 16 * 1024 + col // (d // 4) * 256 + t % 16 * 16 + at % 16
    at = col % (d // 16) * 8 + t % 4 + t // 16 * 4
    v = 32 * d + at // 16 * 1024 + t % 16 // 4 * 256 + col // (d // 16) * 16 + at % 16
    return record[..., None] * size + k, record[..., None] * size + v, record


def _exponent(top):
    """The least e with top <= 448 x 2^e, within [-117, 119]; -127 for zero."""
    m, e = torch.frexp(top)  # m in [0.5, 1)
    e = (e - 9 + (m > 0.875)).clamp(-117, 119)
    return torch.where(top > 0, e, -127)


def _codes(x, e):
    return torch.ldexp(x.double(), -e).clamp(-448, 448).float().to(torch.float8_e4m3fn)


def _stored(codes, scale):
    """Values, fp32, of codes and the scale bytes that go with them."""
    return codes.view(torch.float8_e4m3fn).float() * torch.exp2(scale.double() - 127).float()


def _plain_append8(s):
    cache, d, slots = s["cache"], s["k"].shape[-1], s["slots"]
    heads, size = cache.shape[1], cache.shape[-1]
    there = slots >= 0
    slots = slots[there]
    k, v = s["k"][there].float(), s["v"][there].float()
    bad = ~(k.isfinite().all(-1) & v.isfinite().all(-1))[..., None]
    k_at, v_at, record = _places(cache, slots, d)
    block, of = torch.unique(slots // 32, return_inverse=True)
    first = torch.full_like(block, 32).scatter_reduce_(0, of, (slots % 32).to(block.dtype), "amin")
    all_slots = (block[:, None] * 32 + torch.arange(32, device=DEV)).view(-1)
    places = _places(cache, all_slots, d)
    flat = cache.view(-1)
    rec = places[2].reshape(-1, 32, heads)[:, 0]  # of each block and head
    for x, new_at, old_at, byte in ((k, k_at, places[0], 64 * d), (v, v_at, places[1], 64 * d + 1)):
        x = torch.where(bad, 0.0, x)
        top = torch.zeros((block.numel(), heads), device=DEV).scatter_reduce_(
            0, of[:, None].expand(-1, heads).long(), x.abs().amax(-1), "amax")
        had = torch.where(first[:, None] > 0, flat[rec * size + byte].long(), 0) - 127
        e = torch.maximum(_exponent(top).long(), had)
        old = flat[old_at].reshape(-1, 32, heads, d)
        live = torch.arange(32, device=DEV)[:, None, None] < first[:, None, None, None]
        again = _codes(_stored(old, (had + 127)[:, None, :, None]), e[:, None, :, None])
        grown = live & (e > had)[:, None, :, None]
        flat[old_at.reshape(-1)] = torch.where(grown, again.view(torch.uint8), old).reshape(-1)
        code = _codes(x, e[of][..., None]).view(torch.uint8)
        if byte == 64 * d:
            code = torch.where(bad, 0x7F, code)
        flat[new_at.reshape(-1)] = code.reshape(-1)
        flat[rec.reshape(-1) * size + byte] = (e + 127).reshape(-1).to(torch.uint8)
    k_at, v_at, record = _places(cache, s["read"], d)
    at = record * size + 64 * d
    return [_stored(flat[k_at], flat[at][..., None]).to(s["k"].dtype),
            _stored(flat[v_at], flat[at + 1][..., None]).to(s["k"].dtype)]


def _plain_gather(s):
    """K and V of every request, fp32 [b][heads][tokens][d]."""
    cache, table = s["cache"], s["table"]
    d, b = s["q"].shape[-1], table.shape[0]
    heads, groups = cache.shape[1:3]
    cols = -(-s["max_kv"] // (32 * groups))
    rec = cache[table[:, :cols].clamp(min=0)].transpose(1, 2)  # [b][heads][cols][groups][...]
    lead, c = (b, heads, cols * groups), d // 32
    kc = rec[..., :32 * d].reshape(*lead, c, 4, 16, 16).permute(0, 1, 2, 4, 5, 3, 6)
    kc = kc.reshape(*lead, 4, 16, 2, d // 4).permute(0, 1, 2, 5, 4, 3, 6)
    vc = rec[..., 32 * d:64 * d].reshape(*lead, c, 4, 16, 16).permute(0, 1, 2, 4, 5, 3, 6)
    vc = vc.reshape(*lead, 4, 16, d // 16, 2, 4).permute(0, 1, 2, 6, 3, 7, 4, 5)
    scale = rec[..., 64 * d:64 * d + 2].reshape(*lead, 2, 1, 1)
    tokens = cols * groups * 32
    k = _stored(kc.reshape(*lead, 32, d), scale[..., 0, :, :])
    v = _stored(vc.reshape(*lead, 32, d), scale[..., 1, :, :])
    return k.view(b, heads, tokens, d), v.view(b, heads, tokens, d)


def _plain_attend8(s):
    case, q = s["case"], s["q"]
    tokens, hq, d = q.shape
    k, v = _plain_gather(s)
    b, hk, keys, _ = k.shape
    n, lens = s["cu"].diff(), s["kv_lens"]
    row = torch.arange(s["max_new"], device=DEV)
    at = (s["cu"][:-1, None] + row).clamp(max=tokens - 1)
    rows = q[at].float().view(b, -1, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    x = torch.matmul(rows.reshape(b, hk, -1, d), k.transpose(-1, -2).contiguous()) * s["scale"]
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    key = torch.arange(keys, device=DEV)
    pos = (lens - n)[:, None, None] + row[:, None]
    see = key <= pos
    if case["window"]:
        see = see & ((pos - key < case["window"]) | (key < case["sinks"]))
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


def _copy(cache, pairs):
    """Pages pairs[:, 0] over pages pairs[:, 1], in every layer."""
    pairs = pairs[(pairs >= 0).all(-1)].long()
    cache[:, pairs[:, 1]] = cache[:, pairs[:, 0]]


def _plain_fork(s):
    p, table, lens = s["case"]["page"], s["table"], s["lens"]
    cols = table.shape[1]
    source, target, i = s["source"].long(), s["target"].long(), torch.arange(len(s["source"]))
    repeat = (target[:, None] == target) & (i[:, None] > i).to(DEV)
    n = lens[source].long()
    full, part = n // p, n % p > 0
    fits = ~(target[:, None] == source).any(1) & ~repeat.any(1) & (full + part <= cols)
    need = (fits & part).long()
    stop = need.cumsum(0)
    ok = fits & ((need == 0) | (stop <= s["count"]))
    page = s["free"][(s["count"] - stop).clamp(min=0)]
    col = torch.arange(cols, device=DEV)
    rows = torch.where(col < full[:, None], table[source], table[target])
    rows = torch.where((col == full[:, None]) & part[:, None], page[:, None], rows)
    last = table[source, full.clamp(max=cols - 1)]
    pairs = torch.where((ok & part)[:, None], torch.stack([last, page], 1), -1)
    kept = lens.clone()
    kept[target[ok]] = lens[source[ok]]
    table[target[ok]] = rows[ok]
    _copy(s["cache"], pairs)
    status = torch.stack([need[ok].sum(), (~ok).sum()])
    return [table, kept, pairs, status.to(torch.int32), s["cache"]]


def _live(table, lens, page):
    return torch.arange(table.shape[1], device=DEV) < ((lens + page - 1) // page)[:, None]


def _plain_compact(s):
    page, table, count = s["case"]["page"], s["table"], s["count"]
    pages = s["free"].shape[0]
    # the pages that only requests that end name go back to the stack
    kept = s["lens"].clone()
    kept[s["rows"].long()] = 0
    at = torch.arange(pages, device=DEV)
    live, all_live = _live(table, kept, page), _live(table, s["lens"], page)
    used, was, free = (torch.zeros(pages, dtype=torch.bool, device=DEV) for _ in range(3))
    used[table[live].long()] = True
    was[table[all_live].long()] = True
    free[s["free"][at < count].long()] = True
    freed = (was & ~used & ~free).nonzero().flip(0).flatten()
    stack = s["free"]
    stack[count.long() + torch.arange(len(freed), device=DEV)] = freed.to(torch.int32)
    # the others move to the front
    n = used.sum()
    from_, to = (used & (at >= n)).nonzero().flatten(), (~used & (at < n)).nonzero().flatten()
    map_ = at.clone()
    map_[from_] = to
    moved = torch.where(live, map_[table.clamp(min=0).long()], -1)
    pairs = torch.full(s["pairs"].shape, -1, dtype=torch.int32, device=DEV)
    pairs[:len(from_)] = torch.stack([from_, to], 1).to(torch.int32)
    stack_out = s["free_out"]
    stack_out[:] = -1
    left = pages - n
    stack_out[at < left] = (pages - 1 - at)[at < left].to(torch.int32)
    _copy(s["cache"], pairs)
    ints = lambda *v: torch.tensor([int(x) for x in v], dtype=torch.int32, device=DEV)  # noqa: E731
    return [kept, stack, ints(len(freed), 0), moved.to(torch.int32), stack_out, ints(left), pairs,
            ints(n, len(from_)), s["cache"]]


def _plain_logprobs(s):
    raw, tokens, k = s["logits"].float(), s["tokens"].long(), s["case"]["top"]
    x = raw * s["case"]["scale"]
    d = x - x.amax(-1, keepdim=True)
    p = torch.exp(d)
    total = p.sum(-1, keepdim=True)
    log = torch.log(total)
    entropy = log - torch.where(p > 0, p * d, 0.0).sum(-1, keepdim=True) / total
    given = (d - log).gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    column = torch.arange(raw.shape[1], device=DEV)
    ids = []
    rest = raw.clone() if k else raw
    for _ in range(k):  # ties go to the lowest index
        best = torch.where(rest == rest.amax(-1, keepdim=True), column, raw.shape[1]).amin(-1)
        ids.append(best)
        rest.scatter_(1, best[:, None], -math.inf)
    out = [torch.where(tokens >= 0, given, 0.0), entropy[:, 0]]
    if k:
        ids = torch.stack(ids, 1)
        out += [ids.to(torch.int32), (d - log).gather(1, ids)]
    return out


# -------------------------------------------------------------------- run --

_ctx = None


def _context(hb):
    global _ctx
    if _ctx is None:
        _ctx = hb.Context(torch.cuda.current_device())
        _ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return _ctx


def run(s):
    kind, case = s["case"]["kind"], s["case"]
    if not own:
        return {"append8": _plain_append8, "attend8": _plain_attend8, "fork": _plain_fork,
                "compact": _plain_compact, "logprobs": _plain_logprobs}[kind](s)
    import hotarubi_amd as hb
    ctx = _context(hb)
    if kind == "append8":
        hb.kv8_append(k=s["k"], v=s["v"], slots=s["slots"], cache=s["cache"], ctx=ctx, sync=False)
        hb.kv8_read(k=s["k_out"], v=s["v_out"], slots=s["read"], cache=s["cache"], ctx=ctx,
                    sync=False)
        return [s["k_out"], s["v_out"]]
    if kind == "attend8":
        hb.kv8_attention(q=s["q"], out=s["out"], cache=s["cache"], table=s["table"], cu=s["cu"],
                         kv_lens=s["kv_lens"], max_new=s["max_new"], max_kv=s["max_kv"],
                         scale=s["scale"], prefix=s["prefix"], window=case["window"],
                         sinks=case["sinks"], softcap=case["cap"], ctx=ctx, sync=False)
        return s["out"]
    if kind == "fork":
        hb.kv_fork(table=s["table"], lens=s["lens"], source=s["source"], target=s["target"],
                   free_pages=s["free"], free_count=s["count"], page_size=case["page"],
                   lens_out=s["lens_out"], pairs=s["pairs"], status=s["status"], ctx=ctx,
                   sync=False)
        hb.kv_copy(cache=s["cache"], pairs=s["pairs"], ctx=ctx, sync=False)
        return [s["table"], s["lens_out"], s["pairs"], s["status"], s["cache"]]
    if kind == "compact":
        pages = s["cache"].shape[1]
        hb.kv_free(table=s["table"], lens=s["lens"], rows=s["rows"], pages=pages,
                   free_pages=s["free"], free_count=s["count"], page_size=case["page"],
                   lens_out=s["kept"], status=s["freed"], ctx=ctx, sync=False)
        hb.kv_compact(table=s["table"], lens=s["kept"], pages=pages, page_size=case["page"],
                      table_out=s["table_out"], free_pages=s["free_out"],
                      free_count=s["count_out"], pairs=s["pairs"], status=s["status"], ctx=ctx,
                      sync=False)
        hb.kv_copy(cache=s["cache"], pairs=s["pairs"], ctx=ctx, sync=False)
        return [s["kept"], s["free"], s["freed"], s["table_out"], s["free_out"], s["count_out"],
                s["pairs"], s["status"], s["cache"]]
    top = {"top_ids": s["top_ids"], "top_logprobs": s["top"]} if case["top"] else {}
    hb.token_logprobs(logits=s["logits"], tokens=s["tokens"], logprobs=s["logprobs"],
                      entropy=s["entropy"], scale=case["scale"], ctx=ctx, sync=False, **top)
    return [s["logprobs"], s["entropy"], *top.values()]


# ------------------------------------------------------------------ exact --

def _code_value(code):
    """E4M3 codes as float64."""
    exp, man = (code >> 3 & 15).double(), (code & 7).double()
    x = torch.where(exp > 0, torch.exp2(exp - 7) * (1 + man / 8), man * 2.0 ** -9)
    x = torch.where(code & 127 == 127, math.nan, x)
    return torch.where(code > 127, -x, x)


def _round(x, e):
    """x on the E4M3 grid of scale 2^e, float64: nearest, ties to even."""
    y = (x * torch.exp2(-e)).abs().clamp(max=448)
    step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step * torch.exp2(e)).copysign(x)


def _offsets(d):
    """Byte offsets in a record of K and V codes [32][d]."""
    t, col = torch.arange(32, device=DEV)[:, None], torch.arange(d, device=DEV)
    n, half = t % 16, t // 16
    byte = half * (d // 4) + col % (d // 4)
    k = byte // 16 * 1024 + col // (d // 4) * 256 + n * 16 + byte % 16
    byte = 8 * (col % (d // 16)) + 4 * half + n % 4
    return k, 32 * d + byte // 16 * 1024 + n // 4 * 256 + col // (d // 16) * 16 + byte % 16


def _exact_rows(records, d):
    """K and V, float64, of records [..., 64 d + 16] -> [..., 32, d]."""
    return [_code_value(records[..., at]) * torch.exp2(records[..., 64 * d + i, None, None].double()
                                                       - 127)
            for i, at in enumerate(_offsets(d))]


def _exact_append8(s):
    cache, d, page = s["cache"], s["k"].shape[-1], s["case"]["page"]
    slots, read = s["slots"].cpu().numpy(), s["read"].cpu().numpy()
    heads = cache.shape[1]
    out = [torch.empty((len(read), heads, d), dtype=torch.float64, device=DEV) for _ in range(2)]
    # runs of tokens that fall into one block, and of the slots read back
    cut = lambda a: np.split(np.arange(len(a)), np.nonzero(np.diff(a // 32))[0] + 1)  # noqa: E731
    runs = {int(slots[r[0]]) // 32: r for r in cut(slots) if slots[r[0]] >= 0}
    # a long prompt's whole blocks by themselves, the others one after another
    for where in cut(read):
        block = int(read[where[0]]) // 32
        mine, begin = runs[block], int(slots[runs[block][0]]) % 32
        record = cache[block * 32 // page, :, block % (page // 32)]
        old = _exact_rows(record, d)
        for i, (x, was) in enumerate(zip((s["k"], s["v"]), old)):
            x = x[int(mine[0]):int(mine[-1]) + 1].double()  # [run][heads][d]
            top = x.abs().amax((0, 2))
            e = torch.floor(torch.log2(top)) - 8
            e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
            e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e).clamp(-117, 119)
            if begin:
                e = torch.maximum(e, record[:, 64 * d + i].double() - 127)
            e = e[:, None]
            whole = torch.cat([_round(was[:, :begin].transpose(0, 1), e), _round(x, e)])
            out[i][int(where[0]):int(where[-1]) + 1] = whole[torch.tensor(
                read[where] % 32, device=DEV)]
    return out


def _exact_attend8(s):
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
        see = torch.ones((n, total), dtype=torch.bool, device=DEV)
        if case["window"]:
            see &= (key > pos - case["window"]) | (key < case["sinks"])
        see &= key <= pos
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


def _exact_fork(s):
    page = s["case"]["page"]
    table, lens = s["table"].cpu().numpy().copy(), s["lens"].tolist()
    free, count = s["free"].tolist(), int(s["count"])
    source, target = s["source"].tolist(), s["target"].tolist()
    kept, pairs, wanted, taken, refused = list(lens), [], 0, 0, 0
    before = table.copy()
    for i, (a, b) in enumerate(zip(source, target)):
        whole, rest = divmod(lens[a], page)
        pair = (-1, -1)
        if b in source or b in target[:i] or whole + (rest > 0) > table.shape[1]:
            refused += 1
        elif rest and wanted + 1 > count:
            refused, wanted = refused + 1, wanted + 1
        else:
            table[b, :whole] = before[a, :whole]
            if rest:
                pair = (int(before[a, whole]), free[count - 1 - wanted])
                table[b, whole] = pair[1]
                wanted, taken = wanted + 1, taken + 1
            kept[b] = lens[a]
        pairs.append(pair)
    cache = s["cache"].clone()
    for a, b in pairs:
        if a >= 0:
            cache[:, b] = s["cache"][:, a]
    ints = lambda v: np.array(v, np.int32)  # noqa: E731
    return [table, ints(kept), ints(pairs), ints([taken, refused]), cache]


def _exact_compact(s):
    page, count, pages = s["case"]["page"], int(s["count"]), s["free"].shape[0]
    table, lens, ended = s["table"].tolist(), s["lens"].tolist(), set(s["rows"].tolist())
    free = s["free"].tolist()
    rows = [t[:-(-n // page)] for t, n in zip(table, lens)]
    used = {p for b, r in enumerate(rows) if b not in ended for p in r}
    gone = {p for b in ended for p in rows[b]} - used - set(free[:count])
    free[count:count + len(gone)] = sorted(gone, reverse=True)
    n = len(used)
    moves = list(zip(sorted(p for p in used if p >= n), sorted(set(range(n)) - used)))
    to = dict(moves)
    width = len(table[0])
    table = [[to.get(p, p) for p in r] if b not in ended else [] for b, r in enumerate(rows)]
    table = [r + [-1] * (width - len(r)) for r in table]
    cache = s["cache"].clone()
    if moves:
        a, b = (torch.tensor(x, device=DEV) for x in zip(*moves))
        cache[:, b] = s["cache"][:, a]
    ints = lambda v: np.array(v, np.int32)  # noqa: E731
    return [ints([0 if b in ended else x for b, x in enumerate(lens)]), ints(free),
            ints([len(gone), 0]), ints(table),
            ints(list(range(pages - 1, n - 1, -1)) + [-1] * n), ints([pages - n]),
            ints(moves + [(-1, -1)] * (s["pairs"].shape[0] - len(moves))).reshape(-1, 2),
            ints([n, len(moves)]), cache]


def _exact_logprobs(s):
    x, tokens, k = s["logits"], s["tokens"].tolist(), s["case"]["top"]
    rows = x.shape[0]
    f64 = dict(dtype=torch.float64, device=DEV)
    given, entropy = torch.zeros(rows, **f64), torch.empty(rows, **f64)
    ids = torch.empty((rows, k), dtype=torch.int64, device=DEV)
    top = torch.empty((rows, k), **f64)
    step = max(1, (1 << 25) // x.shape[1])
    for i in range(0, rows, step):
        part = slice(i, i + step)
        raw = x[part].double()
        lp = torch.log_softmax(raw * s["case"]["scale"], -1)
        entropy[part] = -(lp.exp() * lp.clamp(min=-1e6)).sum(-1)
        best = torch.sort(raw, dim=-1, descending=True, stable=True)[1][:, :k]
        ids[part], top[part] = best, lp.gather(1, best)
        for r in range(i, min(rows, i + step)):
            if tokens[r] >= 0:
                given[r] = lp[r - i, tokens[r]]
    return [given, entropy] + ([ids.to(torch.int32), top] if k else [])


def exact(case, seed):
    s = prepare(case, seed)
    return {"append8": _exact_append8, "attend8": _exact_attend8, "fork": _exact_fork,
            "compact": _exact_compact, "logprobs": _exact_logprobs}[case["kind"]](s)
