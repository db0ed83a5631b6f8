"""The sampling example (examples/sampled_answers.py): prompts, forks, steps,
ends and a compaction on a cache of 8 bits, and the log probabilities of what
was answered."""
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
DEV = "cuda:0"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("mask", [dict(), dict(window=40, sinks=5)])
def test_forks_and_moved_pages_change_no_bit(gpu, mask):
    """A fork given its source's tokens gives its source's rows, and a server
    that compacts between steps the rows of one that does not: page numbers
    enter no sum, and a request's keys are divided by its length alone."""
    import sampled_answers as sa
    lengths = [45, 3, 64, 33]
    gen = torch.Generator(device=DEV).manual_seed(3)
    prompt = torch.randint(0, sa.VOCAB, (sum(lengths),), generator=gen, device=DEV)
    more = torch.randint(0, sa.VOCAB, (6, 8), generator=gen, device=DEV)
    outs = []
    for compact in (False, True):
        server = sa.Server(8, 40, 96, gpu, **mask)
        rows = [server.step(prompt, ints(lengths + [0] * 4), 64)]
        server.fork(ints([0, 1, 2, 3]), ints([4, 5, 6, 7]))
        assert server.status.tolist() == [3, 0]  # 64 tokens are whole pages
        assert server.lens.tolist() == lengths * 2
        if compact:  # the third prompt's pages are its fork's too
            server.end(ints([1]))
            server.compact()
        else:
            server.end(ints([1]))
        for i, tokens in enumerate(more[:3]):
            both = torch.cat([tokens[[0, 2, 3]], tokens[[0, 1, 2, 3]]])
            x = server.step(both, ints([1, 0, 1, 1, 1, 1, 1, 1]), 1)
            assert torch.equal(x[:3], x[[3, 5, 6]])
            rows.append(x)
            if compact and i == 1:
                server.end(ints([0]))
                server.compact()
                live = server.table[server.lens > 0]
                used = int(server.status[0])
                assert int(live.max()) == used - 1 and int(server.free_count) == 40 - used
            elif i == 1:
                server.end(ints([0]))
            if i == 1:
                x = server.step(more[5, 1:7], ints([0, 0, 1, 1, 1, 1, 1, 1]), 1)
                rows.append(x)
                break
        ids, best, entropy, given = server.answers(rows[-1], 5, tokens=ints([4, 5, 6, 7, 8, -1]))
        rows += [ids, best, entropy, given]
        assert (best.diff(dim=-1) <= 0).all() and (entropy > 0).all()
        assert (given[:5] <= best[:5, 0]).all() and given[5] == 0
        server.end(ints(list(range(8))))
        assert int(server.free_count) == 40
        assert sorted(server.free.tolist()) == list(range(40))
        outs.append(rows)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_the_example_runs(gpu):
    done = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "sampled_answers.py"),
                           "--prompts", "3", "--samples", "3", "--steps", "5"],
                          capture_output=True, text=True, timeout=110)
    assert done.returncode == 0, done.stderr[-2000:]
    assert done.stdout.count("answers:") == 2
