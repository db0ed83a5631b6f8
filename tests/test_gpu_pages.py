"""Pages of a cache that requests share, give back and move, on an MI355X
against plain Python, number for number: forks, freed pages, renumbered caches,
and the copies of both."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, ints, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu


def pages_of(n, page):
    return -(-max(0, n) // page)


# ------------------------------------------------------------------ fork --

def fork_reference(table, lens, source, target, free, count, page):
    table, out, pairs = table.copy(), list(lens), []
    before, batch, cols = table.copy(), *table.shape
    count = max(0, min(count, len(free)))
    wanted = taken = refused = 0
    for i, (s, t) in enumerate(zip(source, target)):
        pair = (-1, -1)
        good = 0 <= s < batch and 0 <= t < batch and t not in source and t not in target[:i]
        n = max(0, lens[s]) if good else 0
        if not good or pages_of(n, page) > cols:
            refused += 1
        else:
            need = n % page > 0
            wanted += need
            if need and wanted > count:
                refused += 1
            else:
                table[t, :n // page] = before[s, :n // page]
                if need:
                    pair = (int(before[s, n // page]), int(free[count - wanted]))
                    table[t, n // page] = pair[1]
                    taken += 1
                out[t] = n
        pairs.append(pair)
    return table, out, pairs, [taken, refused]


def run_fork(gpu, table, lens, source, target, free, count, page):
    t = ints(table)
    out, pairs, status = ints([9] * len(lens)), ints(np.full((len(source), 2), 9)), ints([9, 9])
    hb.kv_fork(table=t, lens=ints(lens), source=ints(source), target=ints(target),
               free_pages=ints(free), free_count=ints([count]), page_size=page, lens_out=out,
               pairs=pairs, status=status, ctx=gpu)
    return t, out, pairs, status


@pytest.mark.parametrize("batch,forks,cols,page,short", [
    (2, 1, 3, 32, 0), (8, 4, 6, 32, 0), (40, 25, 90, 64, 0), (300, 150, 12, 32, -20),
    (700, 600, 5, 32, 0), (9000, 1000, 3, 96, 0), (20000, 400, 2, 32, -100), (65536, 300, 1, 32, 0)])
def test_fork(gpu, batch, forks, cols, page, short):
    say("fork", batch, forks, cols, page, short)
    rng = np.random.default_rng(batch)
    lens = rng.integers(-2, cols * page + 1, batch)
    lens[rng.random(batch) < 0.2] //= page
    lens[rng.random(batch) < 0.05] = cols * page + 1  # past the table
    table = rng.integers(-1, 10000, (batch, cols))
    row = rng.permutation(batch)
    live = max(1, batch - forks) if batch > forks else 1
    source = row[rng.integers(0, live, forks)]
    target = row[batch - forks:]
    if forks > 3:  # targets that are sources, targets twice, rows that are none
        target[1] = source[0]
        target[2] = target[3]
        source[-1] = batch
        target[-2] = -1
    free = rng.permutation(50000)[:forks + 3]
    count = max(0, forks + short)
    args = (table, lens.tolist(), source.tolist(), target.tolist(), free.tolist(), count, page)
    got = run_fork(gpu, *args)
    want = fork_reference(*args)
    for name, g, w in zip(("table", "lens", "pairs", "status"), got, want):
        w = np.asarray(w).reshape(g.shape)
        if name == "lens":  # a row that is no target keeps its number as it is
            w = np.where(np.isin(np.arange(batch), target), w, lens)
        assert np.array_equal(g.cpu().numpy(), w), name


def test_fork_of_nothing(gpu):
    say("fork of nothing")
    table, out, pairs, status = run_fork(gpu, np.array([[4, -1], [5, 6]]), [3, 40], [], [], [], 0, 32)
    assert out.tolist() == [3, 40] and status.tolist() == [0, 0]
    # whole pages ask for no page of their own, a count past the stack is its size
    got = run_fork(gpu, np.array([[4, 7], [5, 6], [-1, -1]]), [64, 0, 5], [0], [1], [], 100, 32)
    assert got[0].tolist() == [[4, 7], [4, 7], [-1, -1]] and got[2].tolist() == [[-1, -1]]
    assert got[1].tolist() == [64, 64, 5] and got[3].tolist() == [0, 0]


def test_fork_with_a_strided_table(gpu):
    say("fork, strided table")
    wide = ints(np.full((3, 9), 55))
    table = wide[:, 2:6]
    table[:] = ints([[1, 2, 3, -1], [-1] * 4, [-1] * 4])
    out, pairs, status = ints([0] * 3), ints(np.zeros((2, 2))), ints([0, 0])
    hb.kv_fork(table=table, lens=ints([70, 0, 0]), source=ints([0, 0]), target=ints([1, 2]),
               free_pages=ints([8, 9]), free_count=ints([2]), page_size=32, lens_out=out,
               pairs=pairs, status=status, ctx=gpu)
    assert table.tolist() == [[1, 2, 3, -1], [1, 2, 9, -1], [1, 2, 8, -1]]
    assert pairs.tolist() == [[3, 9], [3, 8]] and status.tolist() == [2, 0]
    assert (wide[:, :2] == 55).all() and (wide[:, 6:] == 55).all()


# ------------------------------------------------------------------ copy --

@pytest.mark.parametrize("layers,pages,record,count", [
    (1, 3, 16, 1), (1, 5, 4112, 2), (3, 40, 8208, 300), (2, 700, 4112, 350), (1, 9, 34 * 128, 4),
    (5, 6, 40000, 3)])
def test_copy(gpu, layers, pages, record, count):
    """Pairs with holes between them, pages that are none, and one page twice."""
    say("copy", layers, pages, record, count)
    rng = np.random.default_rng(pages)
    cache = torch.randint(0, 256, (layers, pages, 2, 1, record), device=DEV, dtype=torch.uint8)
    perm = rng.permutation(pages)
    pairs = np.full((count, 2), -1, np.int64)
    moves = min(pages // 2, count)
    at = np.sort(rng.permutation(count)[:moves])
    pairs[at] = np.stack([perm[:moves], perm[pages - moves:]], 1)
    if count > 3:
        odd = [i for i in range(count) if i not in set(at.tolist())][:3]
        for i, p in zip(odd, ([pages, 0], [0, pages + 5], [perm[0], perm[0]])):
            pairs[i] = p
    want = cache.clone()
    for a, b in pairs[at]:
        want[:, b] = cache[:, a]
    if layers == 1:
        cache, want = cache[0], want[0]
    guard = torch.full((cache.numel() + 64,), 77, dtype=torch.uint8, device=DEV)
    inner = guard[32:-32].view(cache.shape)
    inner.copy_(cache)
    hb.kv_copy(cache=inner, pairs=ints(pairs), ctx=gpu)
    assert torch.equal(inner, want) and (guard[:32] == 77).all() and (guard[-32:] == 77).all()
    hb.kv_copy(cache=inner, pairs=ints(np.zeros((0, 2))), ctx=gpu)
    assert torch.equal(inner, want)


# --------------------------------------------------------- free, compact --

def names(table, lens, page, rows):
    """The pages that rows name."""
    return {int(p) for b in rows for p in table[b, :pages_of(lens[b], page)] if p >= 0}


def free_reference(table, lens, rows, pages, free, count, page):
    batch = len(lens)
    ends = {r for r in rows if 0 <= r < batch}
    count = max(0, min(count, len(free)))
    in_range = lambda s: {p for p in s if p < pages}  # noqa: E731
    kept = in_range(names(table, lens, page, set(range(batch)) - ends)) | set(free[:count])
    gone = sorted(in_range(names(table, lens, page, ends)) - kept, reverse=True)
    free, room = list(free), len(free) - count
    free[count:count + min(room, len(gone))] = gone[:room]
    return ([0 if b in ends else n for b, n in enumerate(lens)], free,
            [min(room, len(gone)), max(0, len(gone) - room)])


def compact_reference(table, lens, pages, page, free_size, pair_count):
    used = sorted(p for p in names(table, lens, page, range(len(lens))) if p < pages)
    n = len(used)
    holes = sorted(set(range(n)) - set(used))
    moves = list(zip([p for p in used if p >= n], holes))
    to = {p: p for p in used} | dict(moves)
    out = np.full(table.shape, -1)
    for b in range(len(lens)):
        for c in range(min(table.shape[1], pages_of(lens[b], page))):
            out[b, c] = to.get(int(table[b, c]), -1)
    free = list(range(pages - 1, n - 1, -1)) + [-1] * (free_size - pages + n)
    pairs = moves + [(-1, -1)] * (pair_count - len(moves))
    return out, free, [pages - n], np.array(pairs).reshape(-1, 2), [n, len(moves)]


def tables(rng, batch, cols, page, pages, shared=0.2, odd=True):
    lens = rng.integers(0, cols * page + 1, batch)
    lens[rng.random(batch) < 0.2] = 0
    table = np.full((batch, cols), -1, np.int64)
    perm = rng.permutation(pages)
    at = 0
    for b in range(batch):
        for c in range(pages_of(lens[b], page)):
            if at >= pages or rng.random() < shared:
                table[b, c] = perm[rng.integers(0, max(1, at))]
            else:
                table[b, c] = perm[at]
                at += 1
    if odd and batch > 2:  # entries that name no page, lengths that make no sense
        table[1, 0], table[2, -1] = pages + 3, -7
        lens[0], lens[2] = -5, cols * page + 1000
    return table, lens.tolist(), perm[at:].tolist()


SIZES = [(1, 1, 32, 1), (3, 2, 32, 10), (8, 6, 32, 33), (64, 70, 64, 1500), (300, 9, 32, 700),
         (17, 400, 32, 3000), (2000, 3, 96, 4000), (5, 5, 32, 524288), (40, 130, 32, 32 * 64)]


@pytest.mark.parametrize("batch,cols,page,pages", SIZES)
def test_free(gpu, batch, cols, page, pages):
    say("free", batch, cols, page, pages)
    rng = np.random.default_rng(pages)
    table, lens, spare = tables(rng, batch, cols, page, pages)
    rows = rng.integers(-1, batch + 1, max(1, batch // 2)).tolist()
    spare = [p for p in spare[:50]]
    for size, count in ((pages + 5, len(spare)), (len(spare) + 3, len(spare)), (pages + 5, 0)):
        free = spare + [-1] * (size - len(spare))
        out, status = ints([9] * batch), ints([9, 9])
        stack = ints(free)
        hb.kv_free(table=ints(table), lens=ints(lens), rows=ints(rows), pages=pages,
                   free_pages=stack, free_count=ints([count]), page_size=page, lens_out=out,
                   status=status, ctx=gpu)
        want = free_reference(table, lens, rows, pages, free, count, page)
        assert out.tolist() == want[0] and status.tolist() == want[2]
        assert stack.tolist() == want[1]


@pytest.mark.parametrize("batch,cols,page,pages", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(gpu, batch, cols, page, pages, in_place):
    say("compact", batch, cols, page, pages, in_place)
    rng = np.random.default_rng(pages + 1)
    table, lens, _ = tables(rng, batch, cols, page, pages)
    t = ints(table)
    out = t if in_place else ints(np.full((batch, cols + 3), 9))[:, 1:cols + 1]
    free, count = ints([9] * (pages + 2)), ints([9])
    pairs, status = ints(np.full((pages // 2 + 1, 2), 9)), ints([9, 9])
    hb.kv_compact(table=t, lens=ints(lens), pages=pages, page_size=page, table_out=out,
                  free_pages=free, free_count=count, pairs=pairs, status=status, ctx=gpu)
    want = compact_reference(table, lens, pages, page, pages + 2, pages // 2 + 1)
    assert np.array_equal(out.cpu().numpy(), want[0])
    assert free.tolist() == want[1] and count.tolist() == want[2]
    assert np.array_equal(pairs.cpu().numpy(), want[3]) and status.tolist() == want[4]


def test_full_and_empty_caches(gpu):
    say("full and empty caches")
    for lens, pages in (([0, 0], 64), ([64, 64], 4), ([64, 64], 64)):
        table = np.array([[pages - 1, pages - 2], [pages - 3, pages - 4]])
        free, count, pairs, status = ints([9] * pages), ints([9]), ints(np.zeros((32, 2))), ints([0, 0])
        out = ints(np.zeros((2, 2)))
        hb.kv_compact(table=ints(table), lens=ints(lens), pages=pages, page_size=32, table_out=out,
                      free_pages=free, free_count=count, pairs=pairs, status=status, ctx=gpu)
        want = compact_reference(table, lens, pages, 32, pages, 32)
        assert np.array_equal(out.cpu().numpy(), want[0]) and free.tolist() == want[1]
        assert np.array_equal(pairs.cpu().numpy(), want[3]) and status.tolist() == want[4]


def test_pages_in_a_graph(gpu):
    """A captured compaction with its copy, replayed between eager work."""
    say("pages in a graph")
    rng = np.random.default_rng(8)
    batch, cols, page, pages = 64, 20, 32, 900
    table, lens, _ = tables(rng, batch, cols, page, pages, odd=False)
    cache = torch.randint(0, 256, (2, pages, 1, 1, 4112), device=DEV, dtype=torch.uint8)
    t, n = ints(table), ints(lens)
    bufs = dict(table_out=torch.empty_like(t), free_pages=ints([0] * pages), free_count=ints([0]),
                pairs=ints(np.zeros((pages // 2, 2))), status=ints([0, 0]))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    moved = cache.clone()

    def work():
        hb.kv_compact(table=t, lens=n, pages=pages, page_size=page, sync=False, **bufs)
        hb.kv_copy(cache=moved, pairs=bufs["pairs"], sync=False)

    with torch.cuda.stream(stream):
        work()
        torch.cuda.synchronize()
        want = [x.clone() for x in bufs.values()] + [moved.clone()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            work()
    for _ in range(3):
        for x in bufs.values():
            x.fill_(5)
        moved.copy_(cache)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(list(bufs.values()) + [moved], want):
            assert torch.equal(a, b)
        torch.randn((1 << 20,), device=DEV).sum()
