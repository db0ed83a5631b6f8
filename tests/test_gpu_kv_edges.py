"""The serving operators on an MI355X where their arguments are unusual: values
that are not finite, sizes at the ends of their range, against plain 64-bit
implementations."""
from __future__ import annotations

import math

import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, HALF, TINY, TYPES, rope_reference, say

pytestmark = pytest.mark.gpu


def same(a, b):
    """torch.equal, with no tensors in a failure's message."""
    return bool(torch.equal(a, b))


# ------------------------------------------------------------------ rope --

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 32, False), (64, 32, True), (96, 48, False),
                                                 (128, 0, False), (30, 14, False), (30, 14, True),
                                                 (64, 64, False)])
def test_rotation_of_infinities_and_nans(gpu, dtype, dim, rot, interleaved):
    """What is not finite stays with its own pair, and past `rot` with its own
    element: the rest of the head comes out as for any other row."""
    say("rope, not finite", dtype, dim, rot, interleaved)
    gen = torch.Generator(device=DEV).manual_seed(dim + rot)
    odd = [math.inf, -math.inf, math.nan]
    x = torch.randn((3 * dim, 2, dim), generator=gen, device=DEV).to(dtype)
    for i in range(3 * dim):  # each element of the head once with each of them
        x[i, 0, i % dim] = odd[i // dim]
        x[i, 1, (i + dim // 2) % dim] = odd[i // dim]
    x[0, :, -1] = -0.0
    half = rot // 2
    pos = torch.randint(1, 5000, (1, 3 * dim), generator=gen, device=DEV, dtype=torch.int32)
    freq = 10000.0 ** -(torch.arange(half, device=DEV, dtype=torch.float64) / max(1, half))
    gamma = 1 + 0.3 * torch.randn((dim,), generator=gen, device=DEV)
    for g in (None, gamma):
        out = torch.empty_like(x)
        hb.norm_rope(q=x, positions=pos, inv_freq=freq, q_out=out, gamma_q=g, eps=1e-5,
                     interleaved=interleaved, ctx=gpu)
        want, size = rope_reference(x, g, pos, freq, (half,), interleaved, 1e-5)
        assert same(out.isnan(), want.isnan())
        assert same(torch.where(out.isinf(), out, 0).double(),
                           torch.where(want.isinf(), want, 0))
        fine = want.isfinite()
        tol = HALF[dtype] * want.abs() + (dim + 16) * 2.0**-24 * size + TINY[dtype]
        assert ((out.double() - want).abs() <= tol)[fine].all()
        if g is None:  # not turned: as they went in, bit for bit where they are numbers
            tail, there = x[..., rot:], ~x[..., rot:].isnan()
            assert same(out[..., rot:][there], tail[there])
            assert same(torch.signbit(out[..., rot:][there]), torch.signbit(tail[there]))
