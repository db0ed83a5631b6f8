"""The 8-bit cache, its pages and a step's log probabilities without a GPU: the
cache's byte layout, scales and visible keys (hb_kv.h, built for the host), and
the refusals of the C and Python entry points, which come before any device
call."""
from __future__ import annotations

import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_kv_host import NoContext, ints, refused

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv8") / "kv8_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so,
                    os.path.join(HERE, "kv8_host.cpp")], check=True)
    lib = C.CDLL(so)
    lib.kv8h_scale.restype = lib.kv8h_walk.restype = C.c_uint32
    return lib


# ---------------------------------------------------------------- layout --

@pytest.mark.parametrize("dim", [64, 128, 256])
def test_layout_is_the_documented_one_and_covers_the_record(host, dim):
    at = (C.c_uint32 * 5)()
    keys, values = set(), set()
    for t in range(32):
        for col in range(dim):
            host.kv8h_offsets(dim, t, col, at)
            # K: chunks of [g][n][16 B]; lane (g, n) = columns of token n, then 16 + n
            g, within = col // (dim // 4), t // 16 * (dim // 4) + col % (dim // 4)
            assert at[0] == within // 16 * 1024 + g * 256 + t % 16 * 16 + within % 16
            # V: lane (g, c) = columns, of each tokens 4g..4g+3, then 16+4g..16+4g+3
            within = col % (dim // 16) * 8 + t % 4 + 4 * (t // 16)
            assert at[1] == (32 * dim + within // 16 * 1024 + t % 16 // 4 * 256
                             + col // (dim // 16) * 16 + within % 16)
            keys.add(at[0])
            values.add(at[1])
    assert keys == set(range(32 * dim)) and values == set(range(32 * dim, 64 * dim))
    assert list(at[2:]) == [64 * dim, 64 * dim + 1, 64 * dim + 16]
    assert hb.kv8_cache_shape(7, 3, 64, dim) == (7, 3, 2, 64 * dim + 16)


def test_scale_is_the_least_that_holds_the_largest_value(host):
    rng = np.random.default_rng(0)
    tops = np.concatenate([
        rng.integers(1, 0x7F800000, 4000).astype(np.uint32),
        np.array([1, 2, 0x7FFFFF, 0x800000, 0x7F7FFFFF, 0x7F600000, 0x7F600001], np.uint32),
        (np.array([1.75 * 2.0**n for n in range(-126, 128)], np.float32).view(np.uint32)),
        (np.array([1.75 * 2.0**n for n in range(-126, 127)], np.float32).view(np.uint32) + 1)])
    for bits in tops.tolist():
        top = float(np.uint32(bits).view(np.float32))
        e = -117
        while top > 448 * 2.0**e and e < 119:
            e += 1
        assert host.kv8h_scale(bits) == e + 127, (hex(bits), top)
    assert host.kv8h_scale(0) == 0


def test_walk_with_sinks_visits_every_record_that_is_seen_once(host):
    rng = np.random.default_rng(1)
    room = (C.c_uint32 * 64)()
    for _ in range(4000):
        total = int(rng.integers(0, 700))
        pos0 = int(rng.integers(-40, total + 1))
        pos1 = min(total - 1, pos0 + int(rng.integers(0, 60))) if total else pos0
        pos1 = max(pos0, pos1)
        window = int(rng.choice([1, 31, 32, 33, 200, 1000]))
        prefix = min(total, int(rng.choice([0, 0, 1, 32, 150, 700])))
        sinks = int(rng.choice([0, 1, 4, 32, 33, 90, 2**32 - 1]))
        n = host.kv8h_walk(pos0, pos1, total, prefix, window, C.c_uint32(sinks), room, 64)
        walk = list(room[:n])
        key = np.arange(total)
        seen = key < prefix
        for pos in range(pos0, pos1 + 1):
            mine = (key <= pos) & ((pos - key < window) | (key < sinks))
            seen |= mine
            lead = host.kv8h_lead(prefix, C.c_uint32(sinks), pos, total)
            assert lead == max(prefix, min(total, sinks, max(0, pos + 1)))
        assert walk == sorted(set(walk))
        assert set(np.unique(key[seen] // 32)) <= set(walk)
        assert all(r * 32 < total for r in walk)


# -------------------------------------------------------------- refusals --

def cache(pages=2, heads=2, page=64, dim=64):
    return torch.zeros(hb.kv8_cache_shape(pages, heads, page, dim), dtype=torch.uint8)


@pytest.mark.parametrize("fn", [hb.kv8_append, hb.kv8_read])
def test_cache_row_refusals(fn):
    def rows(**kw):
        a = dict(k=torch.zeros(5, 2, 64), v=torch.zeros(5, 2, 64), slots=ints(5), cache=cache())
        a.update(kw)
        fn(ctx=NoContext, sync=False, **a)

    refused(rows, "null context")
    refused(lambda: rows(k=torch.zeros(5, 2, 64).int()), "k is torch.int32")
    refused(lambda: rows(v=torch.zeros(4, 2, 64)), "v is")
    refused(lambda: rows(k=torch.zeros(5, 1, 64), v=torch.zeros(5, 1, 64)), "2 heads of 64")
    refused(lambda: rows(slots=ints(4)), "slots")
    refused(lambda: rows(cache=cache().int()), "the cache")
    refused(lambda: rows(cache=cache()[..., :100]), "the cache")
    refused(lambda: rows(cache=torch.zeros(hb.kv_cache_shape(2, 2, 64, 64), dtype=torch.uint8)),
            "64 dim + 16")
    refused(lambda: rows(cache=cache(dim=96), k=torch.zeros(5, 2, 96), v=torch.zeros(5, 2, 96)),
            "cache of head size 96", hb.HB_EUNSUPPORTED)
    refused(lambda: rows(cache=cache(pages=0)), "cache")


def attention(fn=hb.kv8_attention, **kw):
    a = dict(q=torch.zeros(6, 4, 64), out=torch.zeros(6, 4, 64), cache=cache(), table=ints(3, 2),
             cu=ints(4), kv_lens=ints(3), max_new=2, max_kv=128, scale=0.125, prefix=ints(3),
             window=40, sinks=4)
    a.update(kw)
    return fn(ctx=NoContext, sync=False, **a) if fn is hb.kv8_attention else fn(**a)


def test_attention_refusals():
    refused(attention, "null context")
    refused(lambda: attention(q=torch.zeros(6, 3, 64), out=torch.zeros(6, 3, 64)),
            "3 query heads over 2 K/V heads")
    refused(lambda: attention(out=torch.zeros(6, 4, 64).half()), "out")
    refused(lambda: attention(q=torch.zeros(6, 4, 128), out=torch.zeros(6, 4, 128)),
            "q has heads of 128 elements, the cache of 64")
    refused(lambda: attention(cache=torch.zeros(hb.kv_cache_shape(2, 2, 64, 64),
                                                dtype=torch.uint8)), "64 dim + 16")
    for name in ("cu", "kv_lens", "prefix"):
        refused(lambda: attention(**{name: ints(7)}), name)
    for name in ("max_new", "max_kv", "window", "sinks"):
        refused(lambda: attention(**{name: -1}), "out of range")
    for bad in (math.inf, -math.inf, math.nan):
        refused(lambda: attention(scale=bad), "scale")
        refused(lambda: attention(softcap=bad), "softcap")
    refused(lambda: attention(hb.kv8_attention_way, scale=math.nan), "scale")


def test_the_way_of_a_call_is_told_without_running_it():
    def way(batch, new, keys, hq, hk, dim, dtype, **kw):
        q = torch.empty((1, 1, dim), dtype=dtype).expand(batch * new, hq, dim)
        a = dict(q=q, out=q, cache=cache(heads=hk, dim=dim), table=ints(batch, keys // 64 + 1),
                 cu=ints(batch + 1), kv_lens=ints(batch), max_new=new, max_kv=keys, scale=1.0)
        a.update(kw)
        return hb.kv8_attention_way(**a)

    bf16 = torch.bfloat16
    assert way(3, 0, 100, 4, 2, 64, bf16) == ("none", 0, 0, 0)
    kind, tiles, splits, workspace = way(1, 1, 100000, 8, 1, 128, bf16)
    assert (kind, tiles) == ("splits", 1) and workspace == splits * 8 * 132 * 4
    # a window leaves few records to split, sinks a few more
    narrow = way(1, 1, 100000, 8, 1, 128, bf16, window=1024)
    more = way(1, 1, 100000, 8, 1, 128, bf16, window=1024, sinks=1024)
    assert narrow[2] < more[2] < splits


def fork(**kw):
    a = dict(table=ints(3, 5), lens=ints(3), source=ints(2), target=ints(2), free_pages=ints(8),
             free_count=ints(1), page_size=32, lens_out=ints(3), pairs=ints(2, 2), status=ints(2))
    a.update(kw)
    hb.kv_fork(ctx=NoContext, sync=False, **a)


def test_fork_refusals():
    refused(fork, "null context")
    for name, bad in [("table", ints(15)), ("lens", ints(2)), ("source", ints(2).long()),
                      ("target", ints(3)), ("free_count", ints(2)), ("lens_out", ints(2)),
                      ("status", ints(3)), ("pairs", ints(2, 3)), ("free_pages", ints(4, 2))]:
        refused(lambda: fork(**{name: bad}), name)
    refused(lambda: fork(pairs=ints(3, 2)), "3 pairs for 2 forks")
    refused(lambda: fork(page_size=33), "page size 33")
    refused(lambda: fork(source=ints(4), target=ints(4), pairs=ints(4, 2)), "4 forks")
    lens = ints(3)
    refused(lambda: fork(lens=lens, lens_out=lens), "lens_out must not be an input")
    big = ints(65537)
    refused(lambda: fork(table=ints(65537, 1), lens=big, lens_out=ints(65537)), "65537 rows",
            hb.HB_EUNSUPPORTED)


def test_copy_refusals():
    def copy(**kw):
        a = dict(cache=cache(), pairs=ints(3, 2))
        a.update(kw)
        hb.kv_copy(ctx=NoContext, sync=False, **a)

    refused(copy, "null context")
    refused(lambda: copy(cache=cache()[None]), "null context")  # a layer in front
    refused(lambda: copy(cache=cache()[:, :1]), "the cache")
    refused(lambda: copy(cache=cache().int()), "the cache")
    refused(lambda: copy(cache=cache()[0]), "the cache")
    refused(lambda: copy(pairs=ints(3, 2).long()), "pairs")
    refused(lambda: copy(pairs=ints(6)), "pairs")
    refused(lambda: copy(cache=torch.zeros(2, 2, 1, 40, dtype=torch.uint8)[..., :36].clone()),
            "16-byte aligned")


def free(**kw):
    a = dict(table=ints(3, 5), lens=ints(3), rows=ints(1), pages=20, free_pages=ints(20),
             free_count=ints(1), page_size=32, lens_out=ints(3), status=ints(2))
    a.update(kw)
    hb.kv_free(ctx=NoContext, sync=False, **a)


def test_free_refusals():
    refused(free, "null context")
    for name, bad in [("table", ints(15)), ("lens", ints(2)), ("rows", ints(2, 2)),
                      ("free_count", ints(0)), ("lens_out", ints(2)), ("status", ints(1)),
                      ("free_pages", ints(20).long())]:
        refused(lambda: free(**{name: bad}), name)
    refused(lambda: free(page_size=0), "page size 0")
    refused(lambda: free(pages=524289), "524289 pages", hb.HB_EUNSUPPORTED)
    refused(lambda: free(pages=-1), "out of range")
    lens = ints(3)
    refused(lambda: free(lens=lens, lens_out=lens), "lens_out must not be an input")


def compact(**kw):
    a = dict(table=ints(3, 5), lens=ints(3), pages=20, page_size=32, table_out=ints(3, 5),
             free_pages=ints(20), free_count=ints(1), pairs=ints(10, 2), status=ints(2))
    a.update(kw)
    hb.kv_compact(ctx=NoContext, sync=False, **a)


def test_compact_refusals():
    refused(compact, "null context")
    for name, bad in [("lens", ints(4)), ("table_out", ints(3, 4)), ("free_count", ints(2)),
                      ("pairs", ints(10)), ("status", ints(3))]:
        refused(lambda: compact(**{name: bad}), name)
    refused(lambda: compact(free_pages=ints(19)), "room for 19 free pages")
    refused(lambda: compact(pairs=ints(9, 2)), "9 pairs of 20 pages")
    refused(lambda: compact(page_size=16), "page size 16")
    refused(lambda: compact(pages=524289, free_pages=ints(600000), pairs=ints(300000, 2)),
            "524289 pages", hb.HB_EUNSUPPORTED)


def logprobs(**kw):
    a = dict(logits=torch.zeros(3, 50), tokens=ints(3), logprobs=torch.zeros(3),
             entropy=torch.zeros(3), top_ids=ints(3, 4), top_logprobs=torch.zeros(3, 4))
    a.update(kw)
    hb.token_logprobs(ctx=NoContext, sync=False, **a)


def test_logprob_refusals():
    refused(logprobs, "null context")
    none = dict(tokens=None, logprobs=None, entropy=None, top_ids=None, top_logprobs=None)
    refused(lambda: logprobs(**none), "no log probabilities asked for")
    for name in ("tokens", "logprobs", "top_ids", "top_logprobs"):
        refused(lambda: logprobs(**{name: None}), "go together")
    for name, bad in [("logits", torch.zeros(3, 50).int()), ("logits", torch.zeros(150)),
                      ("logits", torch.zeros(50, 3).T), ("tokens", ints(3).long()),
                      ("logprobs", torch.zeros(3).half()), ("entropy", torch.zeros(2)),
                      ("top_ids", ints(3, 0)), ("top_logprobs", torch.zeros(3, 5))]:
        refused(lambda: logprobs(**{name: bad}), name)
    for bad in (0.0, -1.0, math.nan, math.inf, 1e-38):
        refused(lambda: logprobs(scale=bad), "scale")
    refused(lambda: logprobs(top_ids=ints(3, 51), top_logprobs=torch.zeros(3, 51)), "51 of 50")
    refused(lambda: logprobs(logits=torch.zeros(3, 500), top_ids=ints(3, 65),
                             top_logprobs=torch.zeros(3, 65)), "65 most likely", hb.HB_EUNSUPPORTED)
    refused(lambda: logprobs(logits=torch.zeros(3, 0)), "0 tokens")


def test_c_entry_points_refuse_null_and_misaligned_descriptors():
    lib = hb.lib()
    for name in ("hb_kv8_append", "hb_kv8_read", "hb_kv8_attention", "hb_kv_fork", "hb_kv_copy",
                 "hb_kv_free", "hb_kv_compact", "hb_token_logprobs"):
        for fn in (getattr(lib, name), getattr(lib, name + "_async")):
            assert fn(None, None) == hb.HB_EINVAL and hb.last_error() == "null descriptor"
    assert lib.hb_kv8_attention_way(None, None) == hb.HB_EINVAL and hb.last_error() == "null way"
    at = 1 << 20

    def says(fn, desc, text):
        assert fn(None, desc) != hb.HB_OK and text in hb.last_error(), hb.last_error()

    def fork_c(table=at, lens=at, pairs=at, columns=4, stride=4, batch=2):
        return hb.KV_FORK_DESC.pack(table, lens, at, at, at, at, 2 * at, pairs, at, batch, columns,
                                    stride, 32, 1, 5)
    says(lib.hb_kv_fork, fork_c(), "null context")
    says(lib.hb_kv_fork, fork_c(table=0), "null table")
    says(lib.hb_kv_fork, fork_c(table=at + 2), "4-byte aligned")
    says(lib.hb_kv_fork, fork_c(lens=0), "null page argument")
    says(lib.hb_kv_fork, fork_c(pairs=at + 1), "4-byte aligned")
    says(lib.hb_kv_fork, fork_c(stride=3), "3 apart")
    says(lib.hb_kv_fork, fork_c(columns=1 << 31, stride=1 << 31), "table of")

    def copy_c(base=at, page=4112, layer=1 << 20, pages=9, layers=2, count=3, pairs=at):
        return hb.KV_COPY_DESC.pack(base, pairs, page, layer, pages, layers, count)
    says(lib.hb_kv_copy, copy_c(), "null context")
    says(lib.hb_kv_copy, copy_c(base=0), "null cache")
    says(lib.hb_kv_copy, copy_c(base=at + 8), "16-byte aligned")
    says(lib.hb_kv_copy, copy_c(page=4104), "16-byte aligned")
    says(lib.hb_kv_copy, copy_c(layer=4112 * 8), "9 pages of 4112 bytes")
    says(lib.hb_kv_copy, copy_c(pairs=0), "null page argument")
    says(lib.hb_kv_copy, copy_c(count=0, pairs=0), "null context")

    def compact_c(table_out=2 * at, stride=4):
        return hb.KV_COMPACT_DESC.pack(at, at, table_out, at, at, at, at, 2, 4, 4, stride, 32, 8, 8,
                                       4)
    says(lib.hb_kv_compact, compact_c(), "null context")
    says(lib.hb_kv_compact, compact_c(table_out=0), "null table")
    says(lib.hb_kv_compact, compact_c(table_out=at, stride=5), "one table with rows 4 and 5")

    def logprobs_c(logits=at, kind=hb.HB_TYPE_F32, top=2, ids=at, vocab=100):
        return hb.LOGPROBS_DESC.pack(logits, 100, at, at, at, ids, at if ids else 0, kind, 3, vocab,
                                     top, 1.0)
    says(lib.hb_token_logprobs, logprobs_c(), "null context")
    says(lib.hb_token_logprobs, logprobs_c(logits=0), "null logits")
    says(lib.hb_token_logprobs, logprobs_c(logits=at + 2), "aligned")
    says(lib.hb_token_logprobs, logprobs_c(kind=3), "tensor type 3")
    says(lib.hb_token_logprobs, logprobs_c(ids=0), "go together")
    says(lib.hb_token_logprobs, logprobs_c(vocab=1 << 31), "tokens")


def test_calls_of_more_threads_than_a_launch_has_are_refused():
    """2^24 workgroups of 256 are 2^32 threads."""
    lib, at = hb.lib(), 1 << 20

    def says(fn, desc, text):
        assert fn(None, desc) != hb.HB_OK and text in hb.last_error(), hb.last_error()

    def rows_c(tokens, heads):
        return hb.KV_ROWS_DESC.pack(at, 9, heads, 64, 256, at, at, heads * 256, 256, heads * 256,
                                    256, at, hb.HB_TYPE_F16, tokens)
    for fn in (lib.hb_kv8_append, lib.hb_kv8_read):
        says(fn, rows_c((1 << 25) - 1, 8), "null context")
        says(fn, rows_c(1 << 25, 8), "33554432 tokens of 8 heads in one call")
    for fn in (lib.hb_kv_append, lib.hb_kv_read):
        says(fn, rows_c(1 << 25, 8), "null context")

    def logprobs_c(rows):
        return hb.LOGPROBS_DESC.pack(at, 1, at, at, 0, 0, 0, hb.HB_TYPE_F16, rows, 1, 0, 1.0)
    says(lib.hb_token_logprobs, logprobs_c((1 << 24) - 1), "null context")
    says(lib.hb_token_logprobs, logprobs_c(1 << 24), "16777216 rows in one call")

    def copy_c(page, layers):
        return hb.KV_COPY_DESC.pack(at, at, page, 1 << 40, 9, layers, 3)
    says(lib.hb_kv_copy, copy_c(8192 * 1023 + 16, 16383), "null context")
    says(lib.hb_kv_copy, copy_c(8192 * 1023 + 16, 16384), "in 16384 layers in one call")
    says(lib.hb_kv_copy, copy_c(1 << 36, (1 << 32) - 1), "layers in one call")


def test_without_a_context_tensors_must_be_on_a_gpu():
    rows = torch.zeros(5, 2, 64)
    for call, name in [
            (lambda: hb.kv8_append(k=rows, v=rows, slots=ints(5), cache=cache()), "k"),
            (lambda: hb.kv8_read(k=rows, v=rows, slots=ints(5), cache=cache()), "k"),
            (lambda: hb.kv8_attention(q=rows, out=rows, cache=cache(), table=ints(1, 1),
                                      cu=ints(2), kv_lens=ints(1), max_new=5, max_kv=64,
                                      scale=1.0), "q"),
            (lambda: hb.kv_copy(cache=cache(), pairs=ints(1, 2)), "cache"),
            (lambda: hb.token_logprobs(logits=torch.zeros(2, 3), entropy=torch.zeros(2)),
             "logits")]:
        refused(call, f"{name} is on cpu, not on a GPU")
