"""Lists of pages that a call would write without having an address are refused,
whatever the cache's size, without a GPU."""
from __future__ import annotations

import hotarubi_amd as hb


def test_a_free_list_without_an_address():
    lib, at = hb.lib(), 1 << 20

    def compact(pages, free_pages, free_size):
        desc = hb.KV_COMPACT_DESC.pack(at, at, 2 * at, free_pages, at, at, at, 2, 4, 4, 4, 32, pages,
                                       free_size, 4)
        assert lib.hb_kv_compact(None, desc) == hb.HB_EINVAL
        return hb.last_error()

    assert compact(8, at, 8) == compact(0, at, 5) == compact(0, 0, 0) == "null context"
    # entries past the free pages are written too
    assert compact(8, 0, 8) == compact(0, 0, 5) == "null page argument"
