"""Log probabilities, entropy and the most likely tokens on an MI355X against a
64-bit log softmax and a stable sort.

Tolerances, with e = 2^-24: the sum of the exponentials is off by a rounding a
term of a lane's own (vocab / 64 at most) and 64 for what joins them, and by 4 e
of the mean of |x - max| for the exponents' rounding (the scale's, the product's
and the difference's) and 2 e for the exponential; its logarithm moves by as
much.  A token's log probability has 4 e |x - max| for its own and 3 e of itself
for the last steps.  The entropy's second sum has a rounding a term of the mean
of |x - max| more, and each logarithm and quotient 2 e of itself.  Ids are equal."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import hotarubi_amd as hb
from test_gpu_kv import DEV, TYPES, ints, say
from test_gpu_kv_edges import memory_given_back  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0**-24


def order(x):
    """Columns, the largest first, of equal ones the lowest; a NaN behind -inf."""
    key = torch.where(x.isnan(), -math.inf, x.double() + 0.0)
    first = torch.sort(x.isnan().long(), dim=-1, stable=True)[1]
    return first.gather(1, torch.sort(key.gather(1, first), dim=-1, descending=True,
                                      stable=True)[1])


def check(gpu, x, tokens, top, scale=1.0, ctx=True, entropy=True):
    rows, vocab = x.shape
    out = [torch.full((rows,), 9.0, device=DEV), torch.full((rows,), 9.0, device=DEV)]
    ids = torch.full((rows, top), 9, dtype=torch.int32, device=DEV)
    best = torch.full((rows, top), 9.0, device=DEV)
    kw = dict(logits=x, tokens=ints(tokens), logprobs=out[0], scale=scale)
    if entropy:
        kw["entropy"] = out[1]
    if top:
        kw.update(top_ids=ids, top_logprobs=best)
    hb.token_logprobs(ctx=gpu if ctx else None, **kw)
    raw = x.double()
    y = raw * scale
    odd = (y.isnan() | (y == math.inf)).any(-1)
    empty = ~odd & (y == -math.inf).all(-1)
    plain = ~odd & ~empty
    lp = torch.log_softmax(torch.where(plain[:, None], y, 0.0), -1)
    lp = torch.where(empty[:, None], -math.inf, lp)
    lp = torch.where(odd[:, None], math.nan, lp)
    p = torch.where(plain[:, None], torch.nan_to_num(lp, nan=0.0).exp(), 0.0)
    far = torch.where(plain[:, None], y - y.amax(-1, keepdim=True), 0.0)
    far = torch.where(far.isinf(), 0.0, far.abs())
    mean = (p * far).sum(-1)
    tol_sum = E * (vocab / 64 + 64 + 4 * mean + 2)
    tokens = torch.tensor(tokens, device=DEV)
    at = tokens.clamp(0, vocab - 1)[:, None]

    def near(got, want, tol):
        got = got.double()
        same = (got == want) | (got.isnan() & want.isnan())
        off = torch.where(same, 0.0, (got - want).abs() / tol)
        assert not off.isnan().any() and (off <= 1).all(), off.max()

    want = lp.gather(1, at)[:, 0]
    want = torch.where(tokens < 0, 0.0, torch.where(tokens >= vocab, math.nan, want))
    near(out[0], want, tol_sum + E * (4 * far.gather(1, at)[:, 0] + 3 * want.abs()))
    if entropy:
        want = -(p * torch.where(p > 0, lp, 0.0)).sum(-1)
        want = torch.where(odd, math.nan, want)
        log = lp.amax(-1).abs()  # the sum's logarithm
        near(out[1], want, tol_sum + E * ((vocab / 64 + 70) * mean + 4 * log + 2 * want.abs()))
    if top:
        want = order(x)[:, :top]
        assert torch.equal(ids.long(), want)
        want = lp.gather(1, want)
        near(best, want, tol_sum[:, None] + E * (4 * far.gather(1, ids.long()) + 3 * want.abs()))
    return out[0], out[1], ids, best


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 2, 2), (3, 7, 7), (5, 64, 64), (2, 65, 1), (70, 100, 20), (9, 513, 5),
    (1, 5000, 64), (3, 20011, 20), (1, 131073, 5), (300, 3001, 3), (1100, 1000, 5),
    (1030, 9000, 20), (4100, 300, 1), (600, 33000, 0), (40, 50001, 8)])
def test_sizes(gpu, dtype, rows, vocab, top):
    say("logprobs", dtype, rows, vocab, top)
    gen = torch.Generator(device=DEV).manual_seed(vocab)
    wide = torch.randn((rows, vocab + 3), generator=gen, device=DEV) * 4
    x = wide.to(dtype)[:, 2:2 + vocab]  # rows that begin anywhere
    tokens = np.random.default_rng(rows).integers(-2, vocab, rows)
    tokens[0] = vocab - 1
    if rows > 2:
        tokens[1], tokens[2] = vocab, 2**31 - 1
    check(gpu, x, tokens.tolist(), top, scale=1.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [
    (1100, 1000, 40), (1040, 8000, 64), (4200, 9001, 33), (30, 1025, 25), (300, 3001, 64),
    (2, 200001, 48)])
@pytest.mark.parametrize("ties", [False, True])
def test_many_likeliest(gpu, dtype, rows, vocab, top, ties):
    """Enough of them that most lanes of a wave have one or two; with ties, that
    the lowest columns of many equal logits win."""
    say("logprobs, many likeliest", dtype, rows, vocab, top, ties)
    gen = torch.Generator(device=DEV).manual_seed(top)
    x = (torch.randn((rows, vocab), generator=gen, device=DEV) * 2).to(dtype)
    if ties:
        x = x.round()
    check(gpu, x, np.random.default_rng(top).integers(0, vocab, rows).tolist(), top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [6, 1100])
@pytest.mark.parametrize("vocab", [40, 9001])
def test_odd_rows(gpu, dtype, rows, vocab):
    """Ties, masked tokens, rows of nothing, infinities, NaN of both kinds, zeros
    of both signs, the largest numbers."""
    say("logprobs odd", dtype, rows, vocab)
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x = (torch.randn((rows, vocab), generator=gen, device=DEV) * 3).to(dtype)
    most = torch.finfo(dtype).max
    bits = {F32: (torch.int32, 0x7F800001), BF16: (torch.int16, 0x7F81), F16: (torch.int16, 0x7C01)}
    kind, signalling = bits[dtype]
    for r in range(rows):
        row, what = x[r], r % 15
        if what == 0:
            row[:] = 1.5  # all the same
        elif what == 1:
            row[:] = -math.inf
        elif what == 2:
            row[:] = -math.inf
            row[[3, vocab - 1]] = torch.tensor([2.0, -5.0], device=DEV).to(dtype)
        elif what == 3:
            row[7] = math.inf
        elif what == 4:
            row[[2, 30]] = math.nan
        elif what == 5:
            row[:] = math.nan
            row[[5, 20]] = 1.0
        elif what == 6:
            row.view(kind)[[11, 12, 33]] = signalling
        elif what == 7:
            row[:] = torch.tensor([0.0, -0.0], device=DEV).repeat(vocab)[:vocab].to(dtype)
        elif what == 8:
            row[:] = -most
        elif what == 9:
            row[::2] = row.sort()[0][::2]  # rising
        elif what == 10:
            row[:] = (row.float().round() / 2).to(dtype)  # few values
        elif what == 11:
            row[torch.rand(vocab, generator=gen, device=DEV) < 0.9] = -math.inf
        elif what == 12:
            row[9] = 60.0  # all of the probability
        elif what == 13:
            row[:] = torch.linspace(-9, 9, vocab, device=DEV).to(dtype)
    for top in (0, 1, 5, 40):
        check(gpu, x, [r % vocab for r in range(rows)], top)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales(gpu, dtype):
    say("logprobs scales", dtype)
    x = torch.randn((4, 3000), device=DEV).to(dtype)
    for scale in (2.0**-100, 1e-3, 30.0, 1e4):
        check(gpu, x, [0, 1, -1, 2999], 4, scale=scale)
    check(gpu, x, [0, 1, -1, 2999], 4, entropy=False)
    # 0 rows, and a call that names no context
    check(gpu, x[:0], [], 3)
    check(gpu, x, [0, 1, 2, 3], 3, ctx=False)


def test_without_tokens(gpu):
    say("logprobs without tokens")
    x = torch.randn((5, 700), device=DEV)
    ids, best = ints(np.zeros((5, 3))), torch.empty((5, 3), device=DEV)
    hb.token_logprobs(logits=x, top_ids=ids, top_logprobs=best, ctx=gpu)
    assert torch.equal(ids.long(), order(x)[:, :3])
    entropy = torch.empty(5, device=DEV)
    hb.token_logprobs(logits=x, entropy=entropy, ctx=gpu)
    p = torch.softmax(x.double(), -1)
    assert (entropy - -(p * p.log()).sum(-1)).abs().max() < 1e-5


def test_long_strides(gpu):
    """Rows more than 2^32 elements apart."""
    say("logprobs long strides")
    base = torch.zeros(((1 << 32) + 4000,), dtype=BF16, device=DEV)
    x = base.as_strided((2, 4000), (1 << 32, 1))
    x.copy_(torch.randn((2, 4000), device=DEV))
    check(gpu, x, [17, 3999], 5)


def test_results_do_not_change_and_graphs_replay(gpu):
    say("logprobs in a graph")
    x = torch.randn((3, 60001), device=DEV).to(BF16)
    args = dict(logits=x, tokens=ints([5, 6, 60000]), logprobs=torch.empty(3, device=DEV),
                entropy=torch.empty(3, device=DEV), top_ids=ints(np.zeros((3, 20))),
                top_logprobs=torch.empty((3, 20), device=DEV))
    outs = [args[n] for n in ("logprobs", "entropy", "top_ids", "top_logprobs")]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        hb.token_logprobs(**args)
        torch.cuda.synchronize()
        want = [x.clone() for x in outs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            hb.token_logprobs(sync=False, **args)
    for _ in range(4):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        torch.randn((1 << 20,), device=DEV).sum()
