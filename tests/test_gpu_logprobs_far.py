"""Log probabilities of logits far apart on an MI355X.  References and tolerances
are test_gpu_logprobs'."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_kv import DEV, TYPES, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401
from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(3, 40), (3, 70001), (1100, 1000)])
@pytest.mark.parametrize("scale", [2.0**-100, 2.0**-20, 0.25, 0.45])
def test_logits_far_apart(gpu, dtype, rows, vocab, scale):
    """Logits whose difference passes the type or fp32, under scales that bring
    the log probability back within it."""
    say("logprobs far apart", dtype, rows, vocab, scale)
    gen = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn((rows, vocab), generator=gen, device=DEV)
    x = torch.where(x.abs() > 1, x.sign() * torch.finfo(dtype).max, 0.0)
    x[:, 5], x[:, 7], x[:, 9] = -torch.finfo(dtype).max, -math.inf, torch.finfo(dtype).max
    x = x.to(dtype)
    tokens = [[5, 7, 9, 0][r % 4] for r in range(rows)]
    check(gpu, x, tokens, min(vocab, 64), scale=scale)
