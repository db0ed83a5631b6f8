"""The serving example (examples/paged_decode.py): steps of ragged requests
through projections, plan, rotation, cache and attention."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

import hotarubi_amd as hb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def test_tokens_one_by_one_give_the_prompt_rows(gpu):
    """The rows of a prompt served at once and token by token.  The cache's
    codes are equal (the same rows, encoded alike); queries, scores and sums
    are fp32 in another order, and MXINT8 activations of the last projection
    may then fall on neighbouring steps: 2^-6 of a row's largest value is
    two of them."""
    import paged_decode as pd
    gen = torch.Generator(device="cuda").manual_seed(2)
    lengths = [45, 3, 33]
    x = torch.randn((sum(lengths), pd.HIDDEN), generator=gen, device="cuda")
    whole = pd.Layer(3, 8, 64, gpu)
    rows = whole.step(x, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 45)
    assert whole.lens.tolist() == lengths and int(whole.free_count) == 8 - (2 + 1 + 2)
    start = [0, 45, 48]
    single = pd.Layer(3, 8, 64, gpu)
    for i in range(45):
        new = [1 if i < n else 0 for n in lengths]
        at = [s + i for s, n in zip(start, lengths) if i < n]
        got = single.step(x[at], torch.tensor(new, dtype=torch.int32, device="cuda"), 1)
        want = rows[at]
        limit = 2.0**-6 * want.abs().amax(-1, keepdim=True)
        assert ((got - want).abs() <= limit).all(), i
    assert single.lens.tolist() == lengths


def test_pages_run_out(gpu):
    """A request that no page is left for is refused and the others go on."""
    import paged_decode as pd
    layer = pd.Layer(2, 2, 64, gpu)
    x = torch.randn((64, pd.HIDDEN), device="cuda")
    layer.step(x, torch.tensor([32, 32], dtype=torch.int32, device="cuda"), 32)
    assert layer.status.tolist() == [2, 0] and int(layer.free_count) == 0
    layer.step(x[:2], torch.tensor([1, 1], dtype=torch.int32, device="cuda"), 1)
    assert layer.status.tolist() == [0, 2] and layer.lens.tolist() == [32, 32]


def test_the_example_runs():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "paged_decode.py"),
                          "--steps", "4"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "us a step" in out.stdout
