"""The serving operators without a GPU: the paged cache's byte layout and the
bounds that the kernels apply to block tables, slots and lengths (hb_kv.h,
built for the host), and the refusals of the C and Python entry points, which
come before any device call."""
from __future__ import annotations

import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import hotarubi_amd as hb

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv") / "kv_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so,
                    os.path.join(HERE, "kv_host.cpp")], check=True)
    lib = C.CDLL(so)
    lib.kvh_walk.restype = C.c_uint32
    return lib


# ---------------------------------------------------------------- layout --

@pytest.mark.parametrize("dim", [64, 128, 256])
def test_layout_is_the_documented_one_and_covers_the_record(host, dim):
    at = (C.c_uint32 * 4)()
    codes, scales = set(), set()
    for t in range(32):
        for col in range(0, dim, 2):
            host.kvh_offsets(dim, t, col, at)
            # K: chunks of [g][n][16 B]; lane (g, n) = columns of token n, then 16 + n
            g, within = col // (dim // 4), t // 16 * (dim // 8) + col % (dim // 4) // 2
            assert at[0] == within // 16 * 1024 + g * 256 + t % 16 * 16 + within % 16
            # V: lane (g, c) = columns of tokens 4g..4g+3, then 16+4g..16+4g+3
            g, j, c = t % 16 // 4, t % 4 + 4 * (t // 16), col // (dim // 16)
            within = j * (dim // 32) + col % (dim // 16) // 2
            assert at[1] == 16 * dim + within // 16 * 1024 + g * 256 + c * 16 + within % 16
            codes |= {at[0], at[1]}
            scales |= {at[2], at[3]}
            assert at[2] == 32 * dim + col // 32 * 32 + t % 16 * 2 + t // 16
            assert at[3] == 33 * dim + col // 32 * 32 + t % 16 // 4 * 8 + j
    assert codes == set(range(32 * dim)) and scales == set(range(32 * dim, 34 * dim))


# ---------------------------------------------------------------- bounds --

def test_slots_outside_the_cache_have_no_record(host):
    record, t = C.c_uint64(), C.c_uint32()
    pages, heads, groups = 7, 3, 2
    for slot in list(range(-3, pages * 64 + 70)) + [-2**31, 2**31 - 1]:
        ok = host.kvh_slot(slot, pages, heads, groups, C.byref(record), C.byref(t))
        assert bool(ok) == (0 <= slot < pages * 64)
        if ok:
            assert record.value == slot // 64 * heads * groups + slot // 32 % groups
            assert t.value == slot % 32


def test_bad_pages_have_no_record(host):
    record = C.c_uint64()
    row = np.array([3, -1, 6, 7, 2**31 - 1, -2**31, 0], np.int32)
    ptr = row.ctypes.data_as(C.POINTER(C.c_int32))
    for groups in (1, 2, 3):
        for i in range(0, 12 * groups):
            for head in range(3):
                ok = host.kvh_record(ptr, 7, i, head, 7, 3, groups, C.byref(record))
                col = i // groups
                good = col < 7 and 0 <= row[col] < 7
                assert bool(ok) == good
                if good:
                    want = (int(row[col]) * 3 + head) * groups + i % groups
                    assert record.value == want < 7 * 3 * groups


def test_records_past_32_bits_of_bytes(host):
    record, t = C.c_uint64(), C.c_uint32()
    pages = 60000
    assert host.kvh_slot(pages * 128 - 1, pages, 8, 4, C.byref(record), C.byref(t))
    assert record.value * 34 * 256 > 2**33 and t.value == 31


def test_requests_stay_inside_the_tensors(host):
    rng = np.random.default_rng(0)
    ends = [-2**31, -5, -1, 0, 1, 7, 40, 41, 100, 2**31 - 1]
    out = (C.c_int64 * 5)()
    for _ in range(4000):
        a, b, kv, pre = (int(rng.choice(ends)) for _ in range(4))
        tokens, max_new, keys = (int(rng.choice([0, 1, 7, 40])) for _ in range(3))
        host.kvh_request(a, b, kv, pre, tokens, max_new, C.c_uint64(keys), out)
        first, rows, count, total, prefix = list(out)
        assert 0 <= rows <= max_new and first + rows <= max(tokens, first)
        assert rows == 0 or (first == a and first + rows <= tokens and count == b - a)
        assert 0 <= prefix <= total <= keys


def test_walk_visits_every_record_that_is_seen_once(host):
    rng = np.random.default_rng(1)
    room = (C.c_uint32 * 64)()
    for _ in range(3000):
        total = int(rng.integers(0, 700))
        pos0 = int(rng.integers(-40, 700))
        pos1 = pos0 + int(rng.integers(0, 60))
        window = int(rng.choice([0, 0, 1, 31, 32, 33, 200, 1000]))
        prefix = min(total, int(rng.choice([0, 0, 1, 32, 150, 700])))
        n = host.kvh_walk(pos0, pos1, total, prefix, window, room, 64)
        walk = list(room[:n])
        key = np.arange(total)
        seen = key < prefix
        for pos in range(pos0, pos1 + 1):
            seen |= (key <= pos) & ((pos - key < window) if window else True)
        assert walk == sorted(set(walk))
        assert set(np.unique(key[seen] // 32)) <= set(walk)
        assert all(r * 32 < total for r in walk)


# -------------------------------------------------------------- refusals --

class NoContext:
    """Python's checks on CPU tensors: a context on 'device -1'."""
    handle, device = None, -1


def refused(call, text, code=hb.HB_EINVAL):
    with pytest.raises(hb.HbError) as err:
        call()
    assert text in err.value.message and err.value.code == code, err.value


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def plan(**kw):
    a = dict(lens=ints(3), new_tokens=ints(3), free_pages=ints(8), free_count=ints(1),
             table=ints(3, 5), page_size=32, cu=ints(4), kv_lens=ints(3), slots=ints(9),
             positions=ints(9), status=ints(2))
    a.update(kw)
    hb.kv_plan(ctx=NoContext, sync=False, **a)


def test_plan_refusals():
    refused(plan, "null context")  # everything else is in order
    for name, bad in [("lens", ints(2)), ("new_tokens", ints(3).long()), ("cu", ints(3)),
                      ("kv_lens", ints(3, 1)), ("positions", ints(8)), ("status", ints(1)),
                      ("slots", ints(18)[::2]), ("free_count", ints(2)), ("table", ints(3).float())]:
        refused(lambda: plan(**{name: bad}), name)
    for page in (0, 16, 48):
        refused(lambda: plan(page_size=page), f"page size {page} is not a multiple of 32")
    refused(lambda: plan(page_size=-32), "out of range")
    refused(lambda: plan(table=ints(3, 5)[:, ::2]), "table")
    refused(lambda: plan(table=ints(1, 5).expand(3, 5)), "table rows of 5 entries are 0 apart")
    lens = ints(3)
    refused(lambda: plan(lens=lens, kv_lens=lens), "kv_lens must not be an input")
    plan_0 = dict(lens=ints(0), new_tokens=ints(0), table=ints(0, 5), cu=ints(1), kv_lens=ints(0),
                  slots=ints(0), positions=ints(0), free_pages=ints(0))
    refused(lambda: plan(**plan_0), "null context")


def rope(**kw):
    a = dict(q=torch.zeros(4, 3, 64), positions=ints(1, 4), sections=None,
             inv_freq=torch.zeros(16, dtype=torch.float64), q_out=torch.zeros(4, 3, 64),
             k=torch.zeros(4, 1, 64), k_out=torch.zeros(4, 1, 64), gamma_q=torch.ones(64),
             gamma_k=None, eps=1e-6)
    a.update(kw)
    hb.norm_rope(ctx=NoContext, sync=False, **a)


def test_rope_refusals():
    refused(rope, "null context")
    refused(lambda: rope(q=torch.zeros(4, 3, 64).double()), "q is torch.float64")
    refused(lambda: rope(q_out=torch.zeros(4, 3, 64).half()), "q_out")
    refused(lambda: rope(q_out=torch.zeros(4, 2, 64)), "q_out")
    refused(lambda: rope(k_out=None), "k without k_out")
    refused(lambda: rope(k=torch.zeros(3, 1, 64), k_out=torch.zeros(3, 1, 64)), "k is (3, 1, 64)")
    refused(lambda: rope(q=torch.zeros(4, 64, 3).transpose(1, 2)), "must be neighbours")
    refused(lambda: rope(positions=ints(1, 3)), "positions")
    refused(lambda: rope(positions=torch.zeros(1, 4)), "positions")
    refused(lambda: rope(positions=ints(3, 4), sections=(8, 8)), "sections")
    refused(lambda: rope(positions=ints(2, 4), sections=(8, 7)), "sections of 15 pairs for 16")
    refused(lambda: rope(positions=ints(2, 4), sections=(17, -1)), "out of range")
    refused(lambda: rope(positions=ints(4, 4), sections=(4, 4, 4, 4)), "position axes")
    refused(lambda: rope(inv_freq=torch.zeros(16)), "inv_freq")
    refused(lambda: rope(inv_freq=torch.zeros(33, dtype=torch.float64)), "66 turned elements of a head of 64")
    refused(lambda: rope(gamma_q=torch.ones(32)), "gamma_q")
    refused(lambda: rope(eps=-1.0), "negative eps")
    refused(lambda: rope(eps=float("nan")), "negative eps")
    odd = dict(q=torch.zeros(4, 3, 63), q_out=torch.zeros(4, 3, 63), k=None, gamma_q=None)
    refused(lambda: rope(**odd), "heads of 63 elements", hb.HB_EUNSUPPORTED)


def cache(pages=2, heads=2, page=64, dim=64):
    return torch.zeros(hb.kv_cache_shape(pages, heads, page, dim), dtype=torch.uint8)


@pytest.mark.parametrize("fn", [hb.kv_append, hb.kv_read])
def test_cache_row_refusals(fn):
    def rows(**kw):
        a = dict(k=torch.zeros(5, 2, 64), v=torch.zeros(5, 2, 64), slots=ints(5), cache=cache())
        a.update(kw)
        fn(ctx=NoContext, sync=False, **a)

    refused(rows, "null context")
    refused(lambda: rows(k=torch.zeros(5, 2, 64).int()), "k is torch.int32")
    refused(lambda: rows(v=torch.zeros(5, 2, 64).half()), "v is")
    refused(lambda: rows(v=torch.zeros(4, 2, 64)), "v is")
    refused(lambda: rows(k=torch.zeros(5, 1, 64), v=torch.zeros(5, 1, 64)), "2 heads of 64")
    refused(lambda: rows(slots=ints(4)), "slots")
    refused(lambda: rows(cache=cache().int()), "the cache")
    refused(lambda: rows(cache=cache()[..., :100]), "the cache")
    refused(lambda: rows(cache=cache(dim=96), k=torch.zeros(5, 2, 96), v=torch.zeros(5, 2, 96)),
            "cache of head size 96", hb.HB_EUNSUPPORTED)
    refused(lambda: rows(cache=cache(pages=0)), "cache")


def attention(**kw):
    a = dict(q=torch.zeros(6, 4, 64), out=torch.zeros(6, 4, 64), cache=cache(), table=ints(3, 2),
             cu=ints(4), kv_lens=ints(3), max_new=2, max_kv=128, scale=0.125, prefix=ints(3))
    a.update(kw)
    hb.kv_attention(ctx=NoContext, sync=False, **a)


def test_attention_refusals():
    refused(attention, "null context")
    refused(lambda: attention(q=torch.zeros(6, 3, 64), out=torch.zeros(6, 3, 64)),
            "3 query heads over 2 K/V heads")
    refused(lambda: attention(out=torch.zeros(6, 4, 64).half()), "out")
    refused(lambda: attention(q=torch.zeros(6, 4, 128), out=torch.zeros(6, 4, 128)),
            "q has heads of 128 elements, the cache of 64")
    refused(lambda: attention(q=torch.zeros(6, 256), out=torch.zeros(6, 256)), "q is (6, 256)")
    refused(lambda: attention(cu=ints(3)), "cu")
    refused(lambda: attention(kv_lens=ints(4)), "kv_lens")
    refused(lambda: attention(prefix=ints(2)), "prefix")
    refused(lambda: attention(table=ints(3, 2).long()), "table")
    refused(lambda: attention(max_new=-1), "out of range")
    refused(lambda: attention(max_kv=-1), "out of range")
    refused(lambda: attention(window=-1), "out of range")
    refused(lambda: attention(scale=float("nan")), "scale")
    refused(lambda: attention(softcap=-1.0), "softcap")
    refused(lambda: attention(softcap=float("nan")), "softcap")


def test_c_entry_points_refuse_null_and_misaligned_descriptors():
    lib = hb.lib()
    for name in ("hb_kv_plan", "hb_norm_rope", "hb_kv_append", "hb_kv_read", "hb_kv_attention"):
        for fn in (getattr(lib, name), getattr(lib, name + "_async")):
            assert fn(None, None) == hb.HB_EINVAL and hb.last_error() == "null descriptor"

    def attend(base=1 << 20, q=1 << 20, kind=hb.HB_TYPE_F32, pages=4, heads=2, table=1 << 20,
               columns=4, stride=4, cu=1 << 20, batch=2):
        return lib.hb_kv_attention(None, hb.KV_ATTENTION_DESC.pack(
            base, pages, heads, 64, 64, q, 1 << 21, 256, 64, 256, 64, table, cu, 1 << 20, 0, kind,
            8, 4, batch, columns, stride, 2, 100, 0, 0.1, 0.0))

    assert attend() == hb.HB_EINVAL and hb.last_error() == "null context"
    for kw, text in [(dict(base=0), "null cache"), (dict(base=(1 << 20) + 8), "16-byte aligned"),
                     (dict(q=0), "null attention"), (dict(q=(1 << 20) + 2), "aligned"),
                     (dict(kind=3), "tensor type 3"), (dict(pages=0), "0 pages"),
                     (dict(pages=0xFFFFFFFF, heads=0xFFFFFF00), "query heads"),
                     (dict(pages=0xFFFFFFFF), "2^32 records"), (dict(table=0), "null attention"),
                     (dict(cu=(1 << 20) + 1), "aligned"), (dict(stride=3), "3 apart"),
                     (dict(columns=0x7FFFFFFF, stride=0x7FFFFFFF), "attention of")]:
        assert attend(**kw) == hb.HB_EINVAL, kw
        assert text in hb.last_error() or "records" in hb.last_error(), (kw, hb.last_error())
    # no rows, no launch: only the context is looked at
    assert attend(batch=0, cu=0) == hb.HB_EINVAL and hb.last_error() == "null context"


def test_without_a_context_tensors_must_be_on_a_gpu():
    """A call without `ctx` is ordered on torch's current stream of its
    tensors' device: there is none for host memory."""
    rows = torch.zeros(5, 2, 64)
    for call, name in [
            (lambda: hb.kv_plan(lens=ints(3), new_tokens=ints(3), free_pages=ints(8),
                                free_count=ints(1), table=ints(3, 5), page_size=32, cu=ints(4),
                                kv_lens=ints(3), slots=ints(9), positions=ints(9),
                                status=ints(2)), "lens"),
            (lambda: hb.norm_rope(q=rows, positions=ints(5), q_out=rows,
                                  inv_freq=torch.zeros(8, dtype=torch.float64)), "q"),
            (lambda: hb.kv_append(k=rows, v=rows, slots=ints(5), cache=cache()), "k"),
            (lambda: hb.kv_read(k=rows, v=rows, slots=ints(5), cache=cache()), "k"),
            (lambda: hb.kv_attention(q=rows, out=rows, cache=cache(), table=ints(1, 1), cu=ints(2),
                                     kv_lens=ints(1), max_new=5, max_kv=64, scale=1.0), "q")]:
        refused(call, f"{name} is on cpu, not on a GPU")


def test_scales_and_caps_that_are_not_finite_are_refused():
    for bad in (float("inf"), -float("inf"), float("nan")):
        refused(lambda: attention(scale=bad), "scale")
        refused(lambda: attention(softcap=bad), "softcap")


def test_the_way_of_a_call_is_told_without_running_it():
    """hb_kv_attention_way: sizes alone choose, no address is read (these are
    in host memory), and what a call refuses it refuses."""
    def way(batch, new, keys, hq, hk, dim, dtype, **kw):
        q = torch.empty((1, 1, dim), dtype=dtype).expand(batch * new, hq, dim)
        a = dict(q=q, out=q, cache=cache(heads=hk, dim=dim), table=ints(batch, keys // 64 + 1),
                 cu=ints(batch + 1), kv_lens=ints(batch), max_new=new, max_kv=keys, scale=1.0)
        a.update(kw)
        return hb.kv_attention_way(**a)

    f32, bf16 = torch.float32, torch.bfloat16
    assert way(3, 0, 100, 4, 2, 64, bf16) == ("none", 0, 0, 0)
    assert way(1, 1, 40, 8, 1, 64, f32) == ("splits", 1, 1, 0)
    kind, tiles, splits, workspace = way(1, 1, 100000, 8, 1, 128, bf16)
    assert (kind, tiles) == ("splits", 1) and workspace == splits * 8 * 132 * 4
    kind, tiles, splits, workspace = way(24, 6, 12000, 8, 2, 128, f32)
    assert (kind, tiles) == ("shares", 2) and workspace == (48 + splits) * 24 * 132 * 4
    assert way(24, 60, 130, 32, 8, 64, f32)[:2] == ("rows", 2)
    kind, tiles, _, workspace = way(16, 300, 500, 16, 2, 256, bf16)
    assert (kind, tiles) == ("prompt", 1) and workspace == 16 * 32 * (128 * 256 + 4)
    assert way(16, 300, 500, 16, 2, 256, f32)[0] == "rows"
    refused(lambda: way(1, 1, 40, 8, 1, 64, f32, scale=float("nan")), "scale")
    refused(lambda: way(1, 1, 40, 8, 1, 64, f32, cu=ints(3)), "cu")
    lib = hb.lib()
    assert lib.hb_kv_attention_way(None, None) == hb.HB_EINVAL and hb.last_error() == "null way"
    assert lib.hb_kv_attention_way(None, bytes(hb.KV_WAY.size)) == hb.HB_EINVAL
    assert hb.last_error() == "null descriptor"
