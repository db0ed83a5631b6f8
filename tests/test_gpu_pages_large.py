"""Ends and compactions of the largest tables and caches that are taken, on an
MI355X, number for number against test_gpu_pages' Python sets."""
from __future__ import annotations

import numpy as np
import pytest

import hotarubi_amd as hb
from test_gpu_kv import ints, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401
from test_gpu_pages import compact_reference, free_reference, pytestmark, tables  # noqa: F401

MOST_PAGES, MOST_ROWS = 524288, 65536


@pytest.mark.parametrize("batch,cols,page", [(MOST_ROWS, 9, 32), (260, 2100, 64), (1, 400000, 32)])
def test_free_of_the_largest(gpu, batch, cols, page):
    say("free, the largest", batch, cols, page)
    rng = np.random.default_rng(batch)
    table, lens, spare = tables(rng, batch, cols, page, MOST_PAGES)
    if batch == 1:
        lens = [cols * page]
        table[0] = rng.permutation(MOST_PAGES)[:cols]
        spare = []
    rows = rng.integers(-1, batch + 1, max(1, batch // 2)).tolist() + [0]
    free = spare[:1000] + [-1] * MOST_PAGES
    out, status, stack = ints([9] * batch), ints([9, 9]), ints(free)
    hb.kv_free(table=ints(table), lens=ints(lens), rows=ints(rows), pages=MOST_PAGES,
               free_pages=stack, free_count=ints([len(spare[:1000])]), page_size=page, lens_out=out,
               status=status, ctx=gpu)
    want = free_reference(table, lens, rows, MOST_PAGES, free, len(spare[:1000]), page)
    assert out.tolist() == want[0] and status.tolist() == want[2]
    assert (stack.cpu().numpy() == np.array(want[1])).all()


@pytest.mark.parametrize("batch,cols,page", [(MOST_ROWS + 1, 9, 32), (260, 2100, 64),
                                             (1, 400000, 32)])
def test_compact_of_the_largest(gpu, batch, cols, page):
    say("compact, the largest", batch, cols, page)
    rng = np.random.default_rng(batch)
    table, lens, _ = tables(rng, batch, cols, page, MOST_PAGES)
    if batch == 1:
        lens = [cols * page]
        table[0] = rng.permutation(MOST_PAGES)[:cols]
    t, free, count = ints(table), ints([9] * MOST_PAGES), ints([9])
    pairs, status = ints(np.full((MOST_PAGES // 2, 2), 9)), ints([9, 9])
    hb.kv_compact(table=t, lens=ints(lens), pages=MOST_PAGES, page_size=page, table_out=t,
                  free_pages=free, free_count=count, pairs=pairs, status=status, ctx=gpu)
    want = compact_reference(table, lens, MOST_PAGES, page, MOST_PAGES, MOST_PAGES // 2)
    assert status.tolist() == want[4] and count.tolist() == want[2]
    for got, w in zip((t, free, pairs), (want[0], want[1], want[3])):
        assert (got.cpu().numpy() == np.array(w)).all()
