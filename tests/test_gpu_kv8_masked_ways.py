"""Windows with first tokens that stay visible, prefixes and caps over the 8-bit
cache on every way of dividing attention's work that takes them: walks with a
gap, shared out over the requests, in splits that are joined, with one tile of
rows a wave and two.  Each call's way is asserted.  References and tolerances
are test_gpu_kv8's."""
from __future__ import annotations

import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, TYPES, ints, say
from test_gpu_kv8 import build, call, check, ramp
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

#: requests, query heads, K/V heads, window, first tokens; the way, 16-row tiles
#: of a wave, whether there are several splits
SIZES = {
    "rows": (ramp(4, 300, 256), 32, 32, 120, 50, "rows", 1, False),
    "rows, two tiles": (ramp(24, 130, 60), 32, 8, 60, 20, "rows", 2, False),
    "splits, two tiles": (ramp(6, 340, 300), 8, 1, 120, 50, "splits", 2, False),
    "splits, joined": (ramp(12, 3000, 3), 8, 1, 1500, 150, "splits", 1, True),
    "splits, joined, two tiles": (ramp(3, 6000, 130), 8, 1, 4500, 150, "splits", 2, True),
    "shares": (ramp(12, 9000, 2), 16, 8, 6000, 150, "shares", 1, True),
    "shares, two tiles": (ramp(12, 9000, 12), 16, 8, 6000, 150, "shares", 2, True),
    "prompt": (ramp(16, 500, 300), 16, 2, 200, 40, "prompt", None, False),
}


def cases():
    for name in SIZES:
        for dim in (64, 128, 256):
            for dtype in TYPES:
                if "two tiles" in name and dim == 256 or name == "prompt" and dtype is F32:
                    continue
                if name == "rows, two tiles" and (dim, dtype) == (128, F16):
                    continue
                yield pytest.param(name, dim, dtype, id=f"{name}-{dim}-{str(dtype)[6:]}")


@pytest.mark.parametrize("name,dim,dtype", cases())
def test_masks_on_every_way(gpu, name, dim, dtype):
    requests, hq, hk, window, sinks, way, tiles, several = SIZES[name]
    say("masked ways", name, dim, dtype)
    s = build(torch.Generator(device=DEV).manual_seed(dim), requests, 64, hk, dim, dtype, hq)

    def asserted(s, **mask):
        out = torch.empty_like(s["q"])
        kind, of, splits, workspace = call(s, out, None, 1.0, fn=True, **mask)
        assert kind == way and (tiles is None or of == tiles)
        assert (splits > 1) == several and (workspace > 0) == (several or way == "prompt")
        check(gpu, s, **mask)

    asserted(s, window=window, sinks=sinks)
    asserted(s, window=window, sinks=sinks, cap=20.0)
    if name.startswith("shares"):  # (a prefix has the call take all keys for visible)
        s["prefix"] = ints([(0, 70, 300)[b % 3] for b in range(len(requests))])
        asserted(s, window=window, sinks=sinks)
        asserted(s, window=700, sinks=200, cap=3.0)
