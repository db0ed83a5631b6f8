"""Answers sampled from shared prompts on a paged cache of 8 bits.

Two attention layers of SmolVLA's decoder size (examples/paged_decode.py) and a
head over a vocabulary serve prompts whose answers are sampled several times:

    prompts    hb_kv_plan -> per layer hb_linear (QKV), hb_norm_rope,
               hb_kv8_append, hb_kv8_attention, hb_linear (O) -> head
    answers    hb_token_logprobs: the likeliest tokens of each prompt
    forks      hb_kv_fork, hb_kv_copy: a request goes on from each of them, on
               the prompt's pages
    steps      as the prompts, a token each; hb_token_logprobs scores the taken
               ones
    ends       hb_kv_free: the least likely answers end; hb_kv_compact,
               hb_kv_copy: the others' pages move to the cache's front

Lengths, tables, free pages and scores stay on the device.

    python examples/sampled_answers.py [--prompts 4] [--samples 4] [--steps 24]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import hotarubi_amd as hb  # noqa: E402
from paged_decode import DEV, DIM, HIDDEN, KV_HEADS, PAGE, Q_HEADS, Linear, _ints  # noqa: E402

LAYERS, VOCAB = 2, 1000


class Server:
    """Layers, head and cache for up to `rows` requests of `most` tokens."""

    def __init__(self, rows: int, pages: int, most: int, ctx, window: int = 0, sinks: int = 0,
                 seed: int = 0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.ctx, self.most, self.pages = ctx, most, pages
        self.mask = dict(window=window, sinks=sinks)
        self.layers = [(Linear((Q_HEADS + 2 * KV_HEADS) * DIM, HIDDEN, gen, ctx),
                        Linear(HIDDEN, Q_HEADS * DIM, gen, ctx)) for _ in range(LAYERS)]
        self.head = Linear(VOCAB, HIDDEN, gen, ctx)
        self.embedding = torch.randn((VOCAB, HIDDEN), generator=gen, device=DEV)
        self.gamma = 1 + 0.1 * torch.randn((2, DIM), generator=gen, device=DEV)
        self.inv_freq = 10000.0 ** -(torch.arange(DIM // 2, device=DEV, dtype=torch.float64)
                                     / (DIM // 2))
        self.cache = torch.zeros((LAYERS, *hb.kv8_cache_shape(pages, KV_HEADS, PAGE, DIM)),
                                 dtype=torch.uint8, device=DEV)
        self.free = torch.arange(pages, dtype=torch.int32, device=DEV)
        self.free_count = _ints(1, fill=pages)
        self.table = _ints(rows, -(-most // PAGE), fill=-1)
        self.lens, self.next_lens = _ints(rows), _ints(rows)
        self.cu, self.status = _ints(rows + 1), _ints(2)

    def step(self, tokens, new, max_new: int):
        """The last layer's rows of `tokens`, new[b] (int32, at most max_new) of
        each request, one request after another."""
        count, ctx = tokens.shape[0], self.ctx
        slots, positions = _ints(count), _ints(count)
        hb.kv_plan(lens=self.lens, new_tokens=new, free_pages=self.free,
                   free_count=self.free_count, table=self.table, page_size=PAGE, cu=self.cu,
                   kv_lens=self.next_lens, slots=slots, positions=positions, status=self.status,
                   ctx=ctx, sync=False)
        x = self.embedding[tokens.long()]
        for (qkv, o), cache in zip(self.layers, self.cache):
            y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
            rows = qkv(y, ctx).view(count, Q_HEADS + 2 * KV_HEADS, DIM)
            q, k, v = rows.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
            hb.norm_rope(q=q, k=k, q_out=q, k_out=k, positions=positions, inv_freq=self.inv_freq,
                         gamma_q=self.gamma[0], gamma_k=self.gamma[1], ctx=ctx, sync=False)
            hb.kv8_append(k=k, v=v, slots=slots, cache=cache, ctx=ctx, sync=False)
            out = torch.empty((count, Q_HEADS, DIM), device=DEV)
            hb.kv8_attention(q=q, out=out, cache=cache, table=self.table, cu=self.cu,
                             kv_lens=self.next_lens, max_new=max_new, max_kv=self.most,
                             scale=DIM ** -0.5, ctx=ctx, sync=False, **self.mask)
            x = x + o(out.view(count, Q_HEADS * DIM), ctx)
        self.free_count -= self.status[0]
        self.lens.copy_(self.next_lens)
        return x

    def answers(self, x, top: int, tokens=None):
        """(likeliest tokens, their log probabilities, entropy, log probabilities
        of `tokens`) of rows x."""
        rows = x.shape[0]
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        logits = self.head(y, self.ctx)
        ids, best = _ints(rows, top), torch.empty((rows, top), device=DEV)
        entropy, given = torch.empty(rows, device=DEV), torch.zeros(rows, device=DEV)
        hb.token_logprobs(logits=logits, tokens=_ints(rows, fill=-1) if tokens is None else tokens,
                          logprobs=given, entropy=entropy, top_ids=ids, top_logprobs=best,
                          scale=0.05, ctx=self.ctx, sync=False)
        return ids, best, entropy, given

    def fork(self, source, target):
        """Requests target[i] (int32) go on from requests source[i]."""
        pairs = _ints(source.shape[0], 2)
        hb.kv_fork(table=self.table, lens=self.lens, source=source, target=target,
                   free_pages=self.free, free_count=self.free_count, page_size=PAGE,
                   lens_out=self.next_lens, pairs=pairs, status=self.status, ctx=self.ctx,
                   sync=False)
        hb.kv_copy(cache=self.cache, pairs=pairs, ctx=self.ctx, sync=False)
        self.free_count -= self.status[0]
        self.lens.copy_(self.next_lens)

    def end(self, rows):
        """Requests `rows` (int32) end."""
        hb.kv_free(table=self.table, lens=self.lens, rows=rows, pages=self.pages,
                   free_pages=self.free, free_count=self.free_count, page_size=PAGE,
                   lens_out=self.next_lens, status=self.status, ctx=self.ctx, sync=False)
        self.free_count += self.status[0]
        self.lens.copy_(self.next_lens)

    def compact(self):
        """The pages in use become the first ones."""
        pairs = _ints(self.pages // 2, 2)
        hb.kv_compact(table=self.table, lens=self.lens, pages=self.pages, page_size=PAGE,
                      table_out=self.table, free_pages=self.free, free_count=self.free_count,
                      pairs=pairs, status=self.status, ctx=self.ctx, sync=False)
        hb.kv_copy(cache=self.cache, pairs=pairs, ctx=self.ctx, sync=False)


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    args.add_argument("--prompts", type=int, default=4)
    args.add_argument("--samples", type=int, default=4)
    args.add_argument("--length", type=int, default=141)
    args.add_argument("--steps", type=int, default=24)
    a = args.parse_args()
    ctx = hb.Context(torch.cuda.current_device())
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    p, n = a.prompts, a.samples
    most, rows = a.length + 2 * a.steps + 1, p * (n + 1)
    server = Server(rows, rows * -(-most // PAGE), most, ctx)
    gen = torch.Generator(device=DEV).manual_seed(1)
    lengths = [max(1, a.length - 5 * b) for b in range(p)]
    prompt = torch.randint(0, VOCAB, (sum(lengths),), generator=gen, device=DEV)
    new = _ints(rows)
    new[:p] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    x = server.step(prompt, new, max(lengths))
    ids, scores, _, _ = server.answers(x[torch.tensor(lengths).cumsum(0).to(DEV) - 1], n)
    source = torch.arange(p, device=DEV, dtype=torch.int32).repeat_interleave(n)
    server.fork(source, torch.arange(p, rows, device=DEV, dtype=torch.int32))
    server.end(torch.arange(p, device=DEV, dtype=torch.int32))  # the prompts themselves
    alive = torch.arange(p, rows, device=DEV)
    tokens, score = ids.flatten(), scores.flatten()
    for half in range(2):
        new = _ints(rows)
        new[alive] = 1
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(a.steps):
            x = server.step(tokens, new, 1)
            ids, scores, _, _ = server.answers(x, 1)
            tokens, score = ids[:, 0], score + scores[:, 0]
        torch.cuda.synchronize()
        us = (time.perf_counter() - start) / a.steps * 1e6
        print(f"{alive.shape[0]} answers: {us:.0f} us a step, {int(server.free_count)} of "
              f"{server.pages} pages free, best {score.max().item():.2f}")
        if half == 0:  # the likelier half goes on
            order = score.argsort(descending=True)[:max(1, alive.shape[0] // 2)].sort()[0]
            gone = torch.ones_like(alive, dtype=torch.bool)
            gone[order] = False
            server.end(alive[gone].to(torch.int32))
            server.compact()
            alive, tokens, score = alive[order], tokens[order], score[order]
    assert int(server.status[1]) == 0


if __name__ == "__main__":
    main()
